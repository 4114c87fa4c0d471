"""The operators of a transformer block around the deformable attention, as measured cases.

rope   rotary positions with several axes (time, height, width) of [B, N, heads * head_dim] tokens
qkn    RMS norm of queries and keys for each head, and the rotation, in one pass
ffn    gated feed-forward block  y = (act(x Wg^T + bg) * (x Wu^T + bu)) Wo^T + bo
clip   global gradient norm over many tensors, and the scaled gradients

A case's `train` says whether its pass is forward and backward (outputs: result and gradients) or
forward alone.  Where `own` is false, run() computes the plain form with elementary torch operations in
float32, rounded once at the end.
"""

import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # one frame of a small video (8 x 16 x 16, 4 heads x 64) as a streamed sampler rotates it: latency
        dict(name="rope_frame_fp32", op="rope", train=False, dtype="fp32", B=1, T=8, H=16, W=16, frame0=5, frames=1, heads=4, d=64,
             at=16, ah=24, aw=24, interleaved=True, tokens=0),
        # training on 2 videos of 64 x 32 x 32 tokens, 16 heads x 72: the benchmark's shape
        dict(name="rope_train_64x32x32", op="rope", train=True, dtype="bf16", B=2, T=64, H=32, W=32, frame0=0, frames=64, heads=16,
             d=72, at=24, ah=24, aw=24, interleaved=True, tokens=0),
        # a single token of the widest model (56 heads x 128) with a position of its own: latency
        dict(name="qkn_token", op="qkn", train=False, dtype="bf16", B=1, T=16, H=16, W=16, frame0=0, frames=1, heads=56, kv=56, d=128,
             at=32, ah=48, aw=48, interleaved=False, tokens=1),
        # training on 64 frames of 64 x 64 tokens, 24 heads x 64: a quarter of the long video
        dict(name="qkn_train_64x64x64", op="qkn", train=True, dtype="bf16", B=1, T=64, H=64, W=64, frame0=0, frames=64, heads=24, kv=24,
             d=64, at=16, ah=24, aw=24, interleaved=False, tokens=0),
        # images and videos of different sizes packed into rows of 5003 tokens, fewer key heads, channels that do not turn
        dict(name="qkn_packed_fp32", op="qkn", train=True, dtype="fp32", B=2, T=32, H=32, W=32, frame0=0, frames=1, heads=16, kv=4, d=72,
             at=16, ah=24, aw=24, interleaved=True, tokens=5003),
        # one token through the 1152-wide block: the weights are read once, latency
        dict(name="ffn_token", op="ffn", train=False, dtype="bf16", M=1, C=1152, F=4608, act="silu", bias=True),
        # one frame and an odd number of register tokens through the 1536-wide block, inference
        dict(name="ffn_frame", op="ffn", train=False, dtype="bf16", M=1027, C=1536, F=6144, act="silu", bias=False),
        # a training step's block at 32 x 32 x 32 tokens, hidden 1152, MLP ratio 4
        dict(name="ffn_train_1152", op="ffn", train=True, dtype="bf16", M=32768, C=1152, F=4608, act="gelu", bias=True),
        # the 33B model's block: 4096 tokens, hidden 7168, MLP ratio 4
        dict(name="ffn_train_7168", op="ffn", train=True, dtype="bf16", M=4096, C=7168, F=28672, act="silu", bias=False),
        # the small float32 configuration (2048 tokens, 256 channels) that parity is checked with
        dict(name="ffn_train_fp32", op="ffn", train=True, dtype="fp32", M=2048, C=256, F=1024, act="gelu", bias=True),
        # every block gradient of a 28-block 1152-wide model, clipped into the flat buffer that goes to the host
        dict(name="clip_blocks", op="clip", clip=True, dtype="bf16", tensors=504, smallest=1152, largest=8128512, spread=7, max_norm=1.0),
        # the resident head and embedding gradients of a small model: latency
        dict(name="norm_head", op="clip", clip=False, dtype="fp32", tensors=11, smallest=16, largest=262144, spread=3, max_norm=1.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _axes(rng, d):
    """Even channel counts (time, height, width) of at most d."""
    r = d if rng.random() < 0.6 else max(6, 2 * int(d * rng.uniform(0.5, 1.0) / 2))
    at = 2 * max(1, int(r * rng.uniform(0.15, 0.4) / 2))
    ah = 2 * max(1, (r - at) // 4)
    return at, ah, r - at - ah


def draw(rng):
    op = rng.choice(["rope", "qkn", "ffn", "ffn", "clip"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if op in ("rope", "qkn"):
        d = rng.choice([32, 40, 64, 72, 80, 96, 128])
        heads = rng.choice([1, 3, 4, 8, 12, 16, 20])
        kv = rng.choice([h for h in (1, 2, 3, 4, 8, 12, 16, 20) if heads % h == 0])
        at, ah, aw = _axes(rng, d)
        B = rng.choice([1, 1, 2, 3])
        most = 4.0e8 / (heads * d * (2 if dtype == "fp32" else 1))
        tokens = _log(rng, 1, min(300000, most) / B)
        H, W = rng.choice([20, 40, _log(rng, 5, 69) | 1]), _log(rng, 4, 70)
        frames = max(1, tokens // (H * W))
        frame0 = rng.choice([0, 0, 1, 5])
        T = frame0 + frames + rng.choice([0, 0, 3])
        case = dict(op=op, train=rng.random() < 0.6, dtype=dtype, B=B, T=T, H=H, W=W, frame0=frame0, frames=frames, heads=heads, d=d, at=at,
                    ah=ah, aw=aw, interleaved=rng.random() < 0.5, tokens=tokens | 1 if rng.random() < 0.4 else 0)
        if op == "qkn":
            case["kv"] = kv
        return case
    if op == "ffn":
        train = rng.random() < 0.6
        C = rng.choice([256, 256, 640, 1152, 1152, 1536, 1600, 2560, 3584, 7168])
        F = int(C * rng.choice([2.5, 3.5, 4]))
        if rng.random() < 0.15:  # widths that no vector or tile divides
            C, F = C - rng.choice([2, 3, 4, 6]), F - rng.choice([1, 4, 10])
        most = (8.0e11 if dtype == "bf16" else 3.0e10) / (C * F)
        M = _log(rng, 1, min(65536, most))
        M = M | 1 if rng.random() < 0.7 else -(-M // 5) * 5
        return dict(op=op, train=train, dtype=dtype, M=M, C=C, F=F, act=rng.choice(["silu", "gelu"]), bias=rng.random() < 0.5)
    tensors = _log(rng, 1, 700)
    largest = _log(rng, 100, min(3.0e7, 2.4e9 / tensors))
    smallest = max(1, int(largest / _log(rng, 1, 10000)))
    return dict(op="clip", clip=rng.random() < 0.7, dtype=dtype, tensors=tensors, smallest=smallest, largest=largest,
                spread=rng.choice([1, 2, 3, 5, 7]), max_norm=rng.choice([0.1, 1.0, 1.0e9]))


def _numels(case):
    """Element counts: a cycle from the smallest to the largest, spread over their logarithm."""
    lo, hi, s = math.log(case["smallest"]), math.log(case["largest"]), case["spread"]
    return [int(round(math.exp(lo + (hi - lo) * (i % s + 1) / s))) if i % s + 1 < s else case["largest"] for i in range(case["tensors"])]


def _rows(case):
    return case["tokens"] if case["tokens"] else case["frames"] * case["H"] * case["W"]


def _table(case, device):
    """float32 [T * at/2 + H * ah/2 + W * aw/2, 2]: cos and sin of position * 10000^(-2i / axis channels)."""
    parts = []
    for size, ch in ((case["T"], case["at"]), (case["H"], case["ah"]), (case["W"], case["aw"])):
        freq = 10000.0 ** (-torch.arange(0, ch, 2, dtype=torch.float64) / ch)
        ang = torch.arange(size, dtype=torch.float64)[:, None] * freq[None]
        parts.append(torch.stack([ang.cos(), ang.sin()], -1).reshape(-1, 2))
    return torch.cat(parts).float().to(device)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)

    def randn(*shape, std=1.0, dtype=None):
        return torch.randn(*shape, generator=gen, device=dev, dtype=dtype or _DT[case["dtype"]]).mul_(std)

    st = {"case": case}
    op = case["op"]
    if op in ("rope", "qkn"):
        B, N, train = case["B"], _rows(case), case["train"]
        st["table"] = _table(case, dev)
        st["index"] = None
        if case["tokens"]:
            st["index"] = torch.stack([torch.randint(0, n, (B, N), generator=gen, device=dev, dtype=torch.int32)
                                       for n in (case["T"], case["H"], case["W"])], -1)
        width = case["heads"] * case["d"]
        if op == "rope":
            st["x"] = randn(B, N, width).requires_grad_(train)
            if train:
                st["dy"] = randn(B, N, width)
        else:
            kw = case["kv"] * case["d"]
            # queries and keys are columns of one projection's output, as the block has them
            qkv = randn(B, N, width + 2 * kw)
            st["q"] = qkv[..., :width].detach().requires_grad_(train)
            st["k"] = qkv[..., width:width + kw].detach().requires_grad_(train)
            st["gq"] = (1 + randn(case["d"], std=0.2, dtype=torch.float32)).to(_DT[case["dtype"]]).requires_grad_(train)
            st["gk"] = (1 + randn(case["d"], std=0.2, dtype=torch.float32)).to(_DT[case["dtype"]]).requires_grad_(train)
            if train:
                st["dq"], st["dk"] = randn(B, N, width), randn(B, N, kw)
    elif op == "ffn":
        M, C, F = case["M"], case["C"], case["F"]
        g = case["train"]
        st["x"] = randn(M, C).requires_grad_(g)
        st["w_in"] = randn(2 * F, C, std=C ** -0.5).requires_grad_(g)
        st["w_out"] = randn(C, F, std=F ** -0.5).requires_grad_(g)
        st["b_in"] = randn(2 * F, std=0.1).requires_grad_(g) if case["bias"] else None
        st["b_out"] = randn(C, std=0.1).requires_grad_(g) if case["bias"] else None
        if g:
            st["dy"] = randn(M, C)
    else:
        sizes = _numels(case)
        st["grads"] = [randn(n, std=1e-3 * (1 + i % 4)) for i, n in enumerate(sizes)]
        st["sizes"] = sizes
        if case["clip"]:
            st["flat"] = torch.empty(sum(sizes), device=dev, dtype=_DT[case["dtype"]])
            st["out"] = list(st["flat"].split(sizes))
    return st


# ---------------------------------------------------------------------------------- plain forms


def _cos_sin(st, dtype=torch.float32):
    """cos and sin [B or 1, N, 1, pairs] of every token and pair."""
    c, table = st["case"], st["table"].to(dtype)
    T, H, W = c["T"], c["H"], c["W"]
    nt, nh, nw = c["at"] // 2, c["ah"] // 2, c["aw"] // 2
    if st["index"] is not None:
        t, h, w = st["index"].long().unbind(-1)
    else:
        n = torch.arange(c["frames"] * H * W, device=table.device)[None]
        t, h, w = c["frame0"] + n // (H * W), n // W % H, n % W
    tt, th, tw = table[:T * nt].view(T, nt, 2), table[T * nt:T * nt + H * nh].view(H, nh, 2), table[T * nt + H * nh:].view(W, nw, 2)
    cs = torch.cat([tt[t], th[h], tw[w]], -2)[:, :, None]
    return cs[..., 0], cs[..., 1]


def _turn(x, cos, sin, interleaved):
    """Rotates the pairs of x [B, N, heads, d]; channels beyond the pairs pass."""
    n = cos.shape[-1]
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if interleaved else (x[..., :n], x[..., n:2 * n])
    y, z = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([y, z], -1).flatten(-2) if interleaved else torch.cat([y, z], -1)
    return torch.cat([turned, x[..., 2 * n:]], -1)


def _plain_rope(st):
    c = st["case"]
    x = st["x"].detach()
    cos, sin = _cos_sin(st)
    shape = (*x.shape[:2], c["heads"], c["d"])
    y = _turn(x.float().view(shape), cos, sin, c["interleaved"]).flatten(2).to(x.dtype)
    if not c["train"]:
        return [y]
    return [y, _turn(st["dy"].float().view(shape), cos, -sin, c["interleaved"]).flatten(2).to(x.dtype)]


def _plain_norm(x, g, dy, cos, sin, heads, c):
    """Result, and with dy the gradients, of one of the two operands."""
    v = x.detach().float().unflatten(-1, (heads, c["d"]))
    w = g.detach().float()
    r = torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-6)
    y = _turn(v * r * w, cos, sin, c["interleaved"]).flatten(2).to(x.dtype)
    if dy is None:
        return [y]
    dn = _turn(dy.float().unflatten(-1, (heads, c["d"])), cos, -sin, c["interleaved"])
    dg = (dn * v * r).sum((0, 1, 2))
    a = dn * w
    dx = r * (a - v * r * r * (a * v).mean(-1, keepdim=True))
    return [y, dx.flatten(2).to(x.dtype), dg.to(g.dtype)]


def _plain_qkn(st):
    c = st["case"]
    cos, sin = _cos_sin(st)
    return [_plain_norm(st["q"], st["gq"], st.get("dq"), cos, sin, c["heads"], c),
            _plain_norm(st["k"], st["gk"], st.get("dk"), cos, sin, c["kv"], c)]


def _plain_ffn(st):
    c, F = st["case"], st["case"]["F"]
    x, w_in, w_out = (st[k].detach().float() for k in ("x", "w_in", "w_out"))
    gu = x @ w_in.t()
    gu = gu + st["b_in"].detach().float() if c["bias"] else gu
    g, u = gu[:, :F], gu[:, F:]
    if c["act"] == "silu":
        s = 1 / (1 + torch.exp(-g))
        a = g * s
    else:
        s = 0.5 * (1 + torch.erf(g * 0.5 ** 0.5))
        a = g * s
    h = a * u
    y = h @ w_out.t()
    y = y + st["b_out"].detach().float() if c["bias"] else y
    dt = st["x"].dtype
    if not c["train"]:
        return {"y": y.to(dt)}
    da = s * (1 + g * (1 - s)) if c["act"] == "silu" else s + g * torch.exp(-0.5 * g * g) * (2 * math.pi) ** -0.5
    dy = st["dy"].float()
    dh = dy @ w_out
    dgu = torch.cat([dh * u * da, dh * a], 1)
    out = {"y": y.to(dt), "dx": (dgu @ w_in).to(dt), "dw_in": (dgu.t() @ x).to(dt), "dw_out": (dy.t() @ h).to(dt)}
    if c["bias"]:
        out |= {"db_in": dgu.sum(0).to(dt), "db_out": dy.sum(0).to(dt)}
    return out


def _plain_clip(st):
    norm = torch.stack([g.float().square().sum() for g in st["grads"]]).sum().sqrt()
    if not st["case"]["clip"]:
        return {"norm": norm}
    scale = (st["case"]["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    return {"norm": norm, "flat": torch.cat([(g.float() * scale).to(g.dtype) for g in st["grads"]])}


# ---------------------------------------------------------------------------------- the framework's calls


def _own(st):
    import megaslide_b200 as msl

    c = st["case"]
    op = c["op"]
    if op == "clip":
        if not c["clip"]:
            return {"norm": msl.grad_norm(st["grads"])}
        return {"norm": msl.clip_grad_norm_(st["grads"], c["max_norm"], out=st["out"]), "flat": st["flat"]}
    if op == "ffn":
        leaves = {k: st[k] for k in ("x", "w_in", "w_out", "b_in", "b_out") if st[k] is not None}
        y = msl.gated_ffn(st["x"], st["w_in"], st["w_out"], st["b_in"], st["b_out"], activation=c["act"])
        if not c["train"]:
            return {"y": y}
        grads = torch.autograd.grad(y, list(leaves.values()), st["dy"])
        return {"y": y, **{"d" + k: g for k, g in zip(leaves, grads)}}
    where = dict(video_shape=(c["T"], c["H"], c["W"]), axes=(c["at"], c["ah"], c["aw"]), interleaved=c["interleaved"], frame0=c["frame0"],
                 index=st["index"])
    if op == "rope":
        y = msl.rope3d(st["x"], st["table"], heads=c["heads"], **where)
        return [y, *torch.autograd.grad(y, st["x"], st["dy"])] if c["train"] else [y]
    q, k = msl.qk_norm_rope(st["q"], st["k"], st["gq"], st["gk"], st["table"], heads=c["heads"], kv_heads=c["kv"], eps=1e-6, **where)
    if not c["train"]:
        return [[q], [k]]
    dq, dk, dgq, dgk = torch.autograd.grad([q, k], [st["q"], st["k"], st["gq"], st["gk"]], [st["dq"], st["dk"]])
    return [[q, dq, dgq], [k, dk, dgk]]


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"rope": _plain_rope, "qkn": _plain_qkn, "ffn": _plain_ffn, "clip": _plain_clip}[state["case"]["op"]](state)


def work(case):
    es = 2 if case["dtype"] == "bf16" else 4
    op = case["op"]
    if op == "clip":
        n = sum(_numels(case))
        return {"bytes": n * es * (2 if case["clip"] else 1) + 4, "flops": n * (3 if case["clip"] else 2)}
    if op == "ffn":
        M, C, F = case["M"], case["C"], case["F"]
        weights, rows = 3 * C * F + ((2 * F + C) if case["bias"] else 0), 2 * M * C
        both = 2 if case["train"] else 1
        return {"bytes": es * both * (weights + rows), "flops": 6 * M * C * F * (3 if case["train"] else 1)}
    tokens = case["B"] * _rows(case)
    table = 4 * (case["T"] * case["at"] + case["H"] * case["ah"] + case["W"] * case["aw"]) + (12 * tokens if case["tokens"] else 0)
    both = 2 if case["train"] else 1
    if op == "rope":
        n = tokens * case["heads"] * case["d"]
        return {"bytes": both * 2 * n * es + table, "flops": both * 3 * n}
    n = tokens * (case["heads"] + case["kv"]) * case["d"]
    return {"bytes": both * 2 * n * es + table, "flops": n * (30 if case["train"] else 8)}


def exact(case, seed):
    """The outputs in float64 from the definitions: rotations as complex products, gradients by automatic differentiation."""
    st = prepare(case, seed)
    op = case["op"]
    if op == "clip":
        total = math.fsum(float(g.double().pow(2).sum()) for g in st["grads"])
        norm = math.sqrt(total)
        out = {"norm": torch.tensor(norm, dtype=torch.float64)}
        if case["clip"]:
            out["flat"] = torch.cat(st["grads"]).double() * min(1.0, case["max_norm"] / (norm + 1e-6))
        return out
    if op == "ffn":
        names = [k for k in ("x", "w_in", "w_out", "b_in", "b_out") if st[k] is not None]
        v = {k: st[k].detach().double().requires_grad_(case["train"]) for k in names}
        y = torch.nn.functional.linear(v["x"], v["w_in"], v.get("b_in"))
        gate, up = y.chunk(2, 1)
        act = torch.nn.functional.silu if case["act"] == "silu" else torch.nn.functional.gelu
        y = torch.nn.functional.linear(act(gate) * up, v["w_out"], v.get("b_out"))
        if not case["train"]:
            return {"y": y}
        grads = torch.autograd.grad(y, [v[k] for k in names], st["dy"].double())
        return {"y": y.detach(), **{"d" + k: g for k, g in zip(names, grads)}}

    T, H, W = case["T"], case["H"], case["W"]
    sizes = [T * case["at"] // 2, H * case["ah"] // 2, W * case["aw"] // 2]
    tabs = [torch.complex(p[:, 0], p[:, 1]).view(n, -1) for p, n in zip(st["table"].double().split(sizes), (T, H, W))]
    if st["index"] is None:
        grid = torch.cartesian_prod(torch.arange(case["frame0"], case["frame0"] + case["frames"]), torch.arange(H), torch.arange(W))
        where = grid.to(st["table"].device)[None]
    else:
        where = st["index"].long()
    turn = torch.cat([tab[where[..., i]] for i, tab in enumerate(tabs)], -1).unsqueeze(2)

    def rotated(v, heads):
        v = v.unflatten(-1, (heads, case["d"]))
        n = turn.shape[-1]
        lead, tail = v[..., :2 * n], v[..., 2 * n:]
        if case["interleaved"]:
            z = torch.view_as_complex(lead.unflatten(-1, (n, 2)).contiguous()) * turn
            lead = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(lead[..., :n], lead[..., n:]) * turn
            lead = torch.cat([z.real, z.imag], -1)
        return torch.cat([lead, tail], -1).flatten(2)

    if op == "rope":
        x = st["x"].detach().double().requires_grad_(case["train"])
        y = rotated(x, case["heads"])
        return [y.detach(), *torch.autograd.grad(y, x, st["dy"].double())] if case["train"] else [y]
    out = []
    for name, heads in (("q", case["heads"]), ("k", case["kv"])):
        x = st[name].detach().double().requires_grad_(case["train"])
        g = st["g" + name].detach().double().requires_grad_(case["train"])
        v = x.unflatten(-1, (heads, case["d"]))
        v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-6) * g
        y = rotated(v.flatten(2), heads)
        out.append([y.detach(), *torch.autograd.grad(y, [x, g], st["d" + name].double())] if case["train"] else [y])
    return out
