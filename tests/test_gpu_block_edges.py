"""The operators around the attention on the GPU where operands share memory, tensors come from inference mode, another
memory order or another default device, and where a trainer's gradients are not finite.  Tolerances as in
test_gpu_block_ops.py: (2 sqrt(K) + 16) roundings of float32 for a product of K terms in the 2-norm, RMS for every rounding
to bfloat16."""

import math

import pytest
import torch
from torch.autograd import forward_ad

import megaslide_b200 as msl
from megaslide_b200 import ops
from megaslide_b200.dit import MegaSlideDiT, VideoDiTConfig
from megaslide_b200.stream import CPUMasterVideoDiT, _HostAdamW
from test_gpu_block_ops import (DTYPES, EPS, HALF, IDS, RMS, _angles, _close, _dev, _ffn_case, _ffn_ref, _positions, _rand,
                                _ref_norm_rope, _within)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shared", ["w_out", "x"])
@pytest.mark.parametrize("dtype,M,D", [(torch.float32, 1000, 512), (torch.float32, 700, 509), (torch.bfloat16, 700, 253)], ids=["fp32", "fp32-odd", "bf16-odd"])
def test_gated_ffn_operands_that_begin_at_one_address(dtype, M, D, shared):
    """w_out or x as the first rows of w_in: the same address, another shape.  The gradient of the shared matrix is the sum
    of two, each within its own tolerance (4 RMS in bf16), rounded once more."""
    w = _rand(1, 2 * D, D, dtype=dtype, std=D ** -0.5).requires_grad_()
    other = _rand(2, D, D, dtype=dtype, std=D ** -0.5).requires_grad_()
    if shared == "w_out":
        x, w_out = _rand(3, M, D, dtype=dtype).requires_grad_(), w[:D]
    else:
        x, w_out = w[:M], other
    dy = _rand(4, x.shape[0], D, dtype=dtype)
    want = list(_ffn_ref(x, w, w_out, None, None, "silu", dy)[:4])
    y = msl.gated_ffn(x, w, w_out)
    got = [y.detach(), *torch.autograd.grad(y, [w, x if shared == "w_out" else other], dy)]
    dw = want[2].clone()
    if shared == "w_out":
        dw[:D] += want[3]
        want = [want[0], dw, want[1]]
    else:
        dw[:M] += want[1]
        want = [want[0], dw, want[3]]
    K = max(2 * D, M)
    for name, a, b, roundings in zip(("y", "shared", "alone"), got, want, (2, 5, 4)):
        _close(a, b, (2 * math.sqrt(K) + 16) * EPS if dtype == torch.float32 else roundings * RMS, name)


@pytest.fixture
def fresh_status():
    """A process that has made no call yet: no status words."""
    kept = [(d, dict(d)) for d in (ops._STATUS, ops._FLAGS)]
    for d, _ in kept:
        d.clear()
    yield
    for d, old in kept:
        d.clear()
        d.update(old)


def test_attention_trains_after_a_first_call_in_inference_mode(fresh_status):
    torch.manual_seed(0)
    m = msl.DeformableSlideAttention3D(64, 4, (3, 3, 3)).cuda()
    x = _rand(1, 2, 24, 64)
    with torch.inference_mode():
        first = m(x, (2, 3, 4)).clone()
    y = m(x.requires_grad_(), (2, 3, 4))
    y.sum().backward()
    assert torch.equal(y.detach(), first) and torch.isfinite(x.grad).all()
    torch.cuda.synchronize()


def test_module_with_rotary_positions_trains_after_a_first_call_in_inference_mode(fresh_status):
    torch.manual_seed(0)
    m = msl.DeformableSlideAttention3D(64, 4, (3, 3, 3), qk_norm=True, rotary_axes=(4, 6, 6)).cuda()
    x = _rand(1, 2, 24, 64)
    with torch.inference_mode():
        first = m(x, (2, 3, 4)).clone()
    y = m(x.requires_grad_(), (2, 3, 4))
    y.sum().backward()
    assert torch.equal(y.detach(), first) and torch.isfinite(x.grad).all()


def test_calls_under_another_default_device(fresh_status):
    """torch.set_default_device does not reach into the host-side buffers of the package."""
    x, w_in, w_out = _rand(1, 3, 16), _rand(2, 16, 16), _rand(3, 16, 8)
    m = msl.DeformableSlideAttention3D(64, 4, (3, 3, 3)).cuda()
    v = _rand(4, 2, 24, 64)
    torch.set_default_device("cuda")
    try:
        y = msl.gated_ffn(x, w_in, w_out)
        z = m(v, (2, 3, 4))
        assert msl.grad_norm([], extra_sumsq=4.0).device.type == "cpu"
    finally:
        torch.set_default_device(None)
    assert torch.equal(msl.gated_ffn(x, w_in, w_out), y) and torch.equal(m(v, (2, 3, 4)), z)
    torch.cuda.synchronize()


@pytest.mark.parametrize("op", ["rope3d", "qk_norm_rope", "gated_ffn"])
def test_forward_mode_derivatives_are_refused(op):
    """No operator has a forward-mode derivative: a tangent is an error, not a result without one.  Without a tangent the
    calls inside a level are the same as outside."""
    x, t = _rand(1, 1, 6, 16), _rand(2, 1, 6, 16)
    table = msl.rotary_table((1, 2, 3), (2, 2, 4), device=_dev())
    w_in, w_out = _rand(3, 16, 16), _rand(4, 16, 8)
    call = {"rope3d": lambda v: msl.rope3d(v, table, video_shape=(1, 2, 3), axes=(2, 2, 4), heads=2),
            "qk_norm_rope": lambda v: msl.qk_norm_rope(v, x, None, None, heads=2)[0],
            "gated_ffn": lambda v: msl.gated_ffn(v, w_in, w_out)}[op]
    want = call(x)
    with forward_ad.dual_level():
        assert torch.equal(call(x), want)
        dual = forward_ad.make_dual(x, t)
        with pytest.raises((RuntimeError, NotImplementedError), match="jvp|forward"):
            call(dual)
        with torch.no_grad():
            with pytest.raises((RuntimeError, NotImplementedError), match="jvp|forward"):
                call(dual)


def test_clip_refuses_results_that_overlap():
    """Blocks write the results in no order: memory that belongs to two of them would be scaled once or twice by chance."""
    t = _rand(1, 400)
    want = t.clone()
    for ts, out in (([t, t], None), ([t[:300], t[100:]], None), ([t[:200]], [t[50:250]]), ([t[:200], t[200:]], [t[200:], t[:200]])):
        with pytest.raises(msl.MslError, match="overlap"):
            msl.clip_grad_norm_(ts, 0.1, out=out)
    torch.cuda.synchronize()
    assert torch.equal(t, want)
    norm = float(msl.grad_norm([t, t]))  # reading twice is no conflict
    assert abs(norm - math.sqrt(2) * float(t.double().norm())) <= 1e-6 * norm
    a, b = torch.empty(400, device=_dev()), torch.empty(400, device=_dev())
    msl.clip_grad_norm_([t, t], 0.1, out=[a, b])
    assert torch.equal(a, b)
    msl.clip_grad_norm_([t[:200], t[200:]], 0.1, out=[t[:200], t[200:]])  # in place, piece by piece
    # neighbours in one buffer, and sources that lie before the results
    flat = torch.zeros(801, device=_dev())
    flat[:400] = want
    msl.clip_grad_norm_([flat[:100], flat[100:400]], 0.1, out=[flat[401:501], flat[501:801]])
    assert torch.equal(flat[:400], want)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_clip_tensors_in_another_memory_order(dtype):
    """Gradients that are dense in an order other than their rows' (a channels-last convolution, a transposed matrix): norm and
    scaling see every element once, whatever the order."""
    conv = _rand(1, 8, 4, 1, 2, 2, dtype=dtype).to(memory_format=torch.channels_last_3d)
    turned = _rand(2, 30, 50, dtype=dtype).t()
    plain = _rand(3, 70, dtype=dtype)
    ts = [conv, turned, plain]
    assert not conv.is_contiguous() and not turned.is_contiguous()
    want = math.sqrt(math.fsum(float(t.double().square().sum()) for t in ts))
    assert abs(float(msl.grad_norm(ts)) - want) <= 1e-6 * want
    before = [t.double().clone() for t in ts]
    limit = want / 4
    outs = [torch.empty_like(t) for t in ts]
    msl.clip_grad_norm_(ts, limit, out=outs)
    norm = msl.clip_grad_norm_(ts, limit)
    assert abs(float(norm) - want) <= 1e-6 * want
    for t, o, b in zip(ts, outs, before):
        ref = b * (limit / (want + 1e-6))
        assert torch.equal(t, o) and torch.all((t.double() - ref).abs() <= (HALF * (dtype == torch.bfloat16) + 2e-6) * ref.abs())
    p = torch.nn.Parameter(torch.zeros(8, 4, 1, 2, 2, device=_dev(), dtype=dtype))
    p.grad = conv
    assert torch.allclose(msl.clip_grad_norm_([p], 1e9), conv.double().norm().float(), rtol=1e-6)


def test_clip_refuses_what_has_no_order():
    base = _rand(1, 6, 10)
    with pytest.raises(ValueError, match="dense"):
        msl.grad_norm([base[:, :5]])  # gaps
    with pytest.raises(ValueError, match="dense"):
        msl.grad_norm([base[:1].expand(6, 10)])  # one row six times
    with pytest.raises(ValueError, match="dense"):
        msl.clip_grad_norm_([base], 1.0, out=[torch.zeros(6, 20, device=_dev())[:, ::2]])
    with pytest.raises(ValueError, match="order"):
        msl.clip_grad_norm_([base], 1.0, out=[torch.zeros(10, 6, device=_dev()).t()])
    with pytest.raises(ValueError, match="order"):
        msl.clip_grad_norm_([base.t()], 1.0, out=[torch.zeros(60, device=_dev())])


def _trainer(fused, max_norm=0.05):
    """A small trainer with gradients put into its buffers: the same for every call."""
    torch.manual_seed(5)
    cfg = VideoDiTConfig(frames=2, in_channels=4, height=8, width=8, patch_size=2, hidden_size=64, num_heads=2, num_layers=3,
                         dsa_kernel_size=(3, 3, 3), checkpoint_interval=2, num_grad_slabs=3, learning_rate=1e-3, weight_decay=0.01,
                         max_grad_norm=max_norm, dtype="float32", device=0, log_interval=0, gated_mlp=True, fused_clip=fused)
    tr = CPUMasterVideoDiT(MegaSlideDiT(cfg), cfg)
    for i in range(tr.num_blocks):
        tr.hgrad[i].normal_(std=1e-2)
        tr.has_grad[i] = True
    for p in tr.res_params:
        p.grad = torch.randn(p.shape).mul_(1e-2).to(p.device)
    return tr


def _step(tr, monkeypatch):
    """(norm, scale handed to the host's updates, resident gradients, parameters) of one optimizer step."""
    scales = []
    update = _HostAdamW.update

    def spy(self, p, g, scale, stage=None):
        scales.append(scale)
        return update(self, p, g, scale, stage=stage)

    monkeypatch.setattr(_HostAdamW, "update", spy)
    for i in range(tr.num_blocks):
        tr.sumsq[i] = float(tr.hgrad[i].double().square().sum())
    norm = tr.optimizer_step()
    params = [p.detach().cpu().clone() for p in tr.get_parameters()]
    assert len(scales) == tr.num_blocks
    return norm, scales, [p.grad.cpu() for p in tr.res_params], params


def test_fused_clip_scales_host_and_resident_gradients_alike(monkeypatch):
    """The norm lies far above its limit: every gradient, on the host and on the GPU, is scaled by the same factor, once."""
    tr = _trainer(True)
    try:
        before = [p.grad.double().cpu() for p in tr.res_params]
        want = math.sqrt(sum(float(g.double().square().sum()) for g in tr.hgrad) + sum(float(g.square().sum()) for g in before))
        assert want > 10 * tr.config.max_grad_norm
        norm, scales, grads, _ = _step(tr, monkeypatch)
        f = tr.config.max_grad_norm / (want + 1e-6)
        assert abs(norm - want) <= 1e-5 * want and all(abs(s - f) <= 1e-5 * f for s in scales)
        for g, b in zip(grads, before):
            assert torch.all((g.double() - b * f).abs() <= 1e-5 * (b * f).abs())
    finally:
        tr.cleanup()


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("where", ["block", "resident"])
def test_fused_clip_with_a_gradient_that_is_not_finite(where, value, monkeypatch):
    """One bad gradient has the same outcome with and without fused_clip, wherever it lies."""
    got = []
    for fused in (False, True):
        tr = _trainer(fused)
        try:
            if where == "block":
                tr.hgrad[1][7] = value
            else:
                tr.res_params[0].grad.view(-1)[3] = value
            got.append(_step(tr, monkeypatch))
            monkeypatch.undo()
        finally:
            tr.cleanup()
    (n0, s0, g0, p0), (n1, s1, g1, p1) = got
    assert (math.isnan(n0) and math.isnan(n1)) or n0 == n1
    assert s0 == s1
    for a, b in zip(g0 + p0, g1 + p1):
        assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a), torch.nan_to_num(b))


@pytest.mark.parametrize("G", [0, 3], ids=["", "extra"])
def test_norm_weights_stay_float32_under_autocast(G, monkeypatch):
    """float32 norm weights reach the kernels beside bf16 tokens as they are, and their gradients, sums in float32, come back
    without a rounding to bf16 on the way."""
    torch.manual_seed(0)
    m = msl.DeformableSlideAttention3D(64, 4, (3, 3, 3), qk_norm=True, rotary_axes=(4, 6, 6)).cuda()
    with torch.no_grad():
        m.q_norm_weight.normal_(1, 0.2)
        m.k_norm_weight.normal_(1, 0.2)
    seen, sums = [], {"q": 0.0, "k": 0.0}
    forward, backward = ops.qk_norm_rope_fwd, ops.qk_norm_rope_bwd

    def fwd(shape, heads, kv, q, k, gq, gk, *a, **kw):
        seen.extend(w for w in (gq, gk) if w is not None)
        return forward(shape, heads, kv, q, k, gq, gk, *a, **kw)

    def bwd(shape, heads, kv, q, k, gq, gk, *a, **kw):
        r = backward(shape, heads, kv, q, k, gq, gk, *a, **kw)
        if kv:
            sums["q"], sums["k"] = sums["q"] + r[2].float(), sums["k"] + r[3].float()
        else:  # the extra keys
            sums["k"] = sums["k"] + r[2].float()
        return r

    monkeypatch.setattr(ops, "qk_norm_rope_fwd", fwd)
    monkeypatch.setattr(ops, "qk_norm_rope_bwd", bwd)
    x = _rand(1, 2, 60, 64).requires_grad_()
    extra = _rand(2, 2, G, 64).requires_grad_() if G else None
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = m(x, (3, 4, 5), extra)
    y.float().square().sum().backward()
    assert len(seen) == (3 if G else 2)
    for w in seen:
        assert any(torch.equal(w.float(), p.detach()) for p in (m.q_norm_weight, m.k_norm_weight))
    for p, s in ((m.q_norm_weight, sums["q"]), (m.k_norm_weight, sums["k"])):
        assert torch.equal(p.grad, s)
        assert not torch.equal(p.grad, p.grad.bfloat16().float())


def _kept_factors(kept, M, F):
    """The kept factors of a bf16 block as float32 [M, 2 F]: the upper 16 bits, then 8 more in rows of F rounded up to 16; the
    last 8 are those 8 again."""
    high = kept[:4 * M * F].view(torch.int16).view(M, 2, F).int() << 16
    low = kept[4 * M * F:].view(M, 2, -1)[..., :F].int()
    return (high | low << 8 | low).view(torch.float32).reshape(M, 2 * F)


@pytest.mark.parametrize("M,C,F", [(1, 9, 30), (40, 77, 203), (130, 253, 635), (200, 1533, 2047)])
def test_gated_ffn_widths_off_vectors_round_the_inner_gradients_once(M, C, F):
    """With one-hot rows of x, dw_in's columns are the gradients of g and u as the kernels hold them: the exact gradient
    of h (a product of C terms) times the kept factor, rounded to bf16 once."""
    x = torch.zeros(M, C, dtype=torch.bfloat16, device=_dev())
    _, w_in, w_out, _, _ = (t.detach() if t is not None else None for t in _ffn_case(M, C, F, torch.bfloat16, "gelu", False))
    rows = min(M, C)
    x[torch.arange(rows), torch.arange(rows)] = 1
    dy = _rand(9, M, C, dtype=torch.bfloat16)
    _, h, kept = ops.gated_ffn_fwd(x, w_in, w_out, activation="gelu", keep=True)
    dw_in = ops.gated_ffn_bwd(x, w_in, w_out, h, kept, dy, activation="gelu", needs=(False, True, False, False, False))[1]
    got = dw_in.t()[:rows].double()
    dh = dy.double() @ w_out.double()
    mag = dy.double().abs() @ w_out.double().abs()
    kd = _kept_factors(kept, M, F).double()
    want = torch.cat([dh * kd[:, :F], dh * kd[:, F:]], 1)[:rows]
    bound = torch.cat([mag * kd[:, :F].abs(), mag * kd[:, F:].abs()], 1)[:rows] * (C + 2) * EPS
    err = (got - want).abs()
    # a result that is nearly halfway between two bf16 numbers may go either way by the sums' own roundings
    assert torch.all(err <= HALF * want.abs() + 2 * bound + 1e-38), float((err / (HALF * want.abs() + 2 * bound + 1e-38)).max())


def _check_product(got, a, b):
    """A product of K terms may be off by 4 EPS of its 2-norm for what the splitting and the accumulators of 32 terms cut
    off, and by the random walk of K / 32 rounded additions to a sum that grows like one (EPS / sqrt(3) each):
    EPS sqrt(K / 192).  What is cut off always pulls a sum towards zero: at most EPS of it, on average, for each of
    the two full-sized additions of an accumulator."""
    want = a.double() @ b.double()
    err = got.double() - want
    assert float(err.norm() / want.norm()) <= (4 + math.sqrt(a.shape[1] / 192)) * EPS
    assert float((err * want.sign()).mean().abs() / want.abs().mean()) <= 2 * EPS


@pytest.mark.parametrize("M", [3, 8, 12, 30, 40, 64])
def test_gated_ffn_float32_few_rows_of_wide_weights_keep_float32(M):
    """Single products of the form that splits the weights on their way."""
    C, F = 4100, 4108
    x, w_in, w_out, b_in, _ = (t.detach() for t in _ffn_case(M, C, F, torch.float32, "silu", True))
    w_in[:F], b_in[:F], b_in[F:] = 0, 40, 0  # silu(40) = 40 and its derivative is 1: the first kept factor is u
    kept = ops.gated_ffn_fwd(x, w_in, w_out, b_in, None, keep=True)[2]
    assert torch.all(kept[:, F:] == 40)
    _check_product(kept[:, :F], x, w_in[F:].t())
    if M > 32:
        return
    w_in = _rand(2, 2 * F, C, std=C ** -0.5)
    dy, ones, h = _rand(9, M, C), torch.ones(M, 2 * F, device=_dev()), torch.zeros(M, F, device=_dev())
    hot = torch.eye(M, C, device=_dev())  # one-hot rows: dw_in's columns are the gradients of g and u
    dx, dw_in = ops.gated_ffn_bwd(hot, w_in, w_out, h, ones, dy, needs=(True, True, False, False, False))[:2]
    dgu = dw_in.t()[:M].contiguous()
    assert torch.equal(dgu[:, :F], dgu[:, F:])
    _check_product(dgu[:, :F], dy, w_out)
    _check_product(dx, dgu, w_in)


@pytest.mark.parametrize("interleaved", [True, False], ids=["interleaved", "split"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("heads,kv,d", [(5, 5, 8), (7, 7, 16), (9, 3, 24), (11, 11, 32), (5, 5, 64), (4, 2, 96), (3, 3, 128), (2, 1, 256)])
def test_qk_norm_rope_heads_of_every_number_of_lanes(heads, kv, d, dtype, interleaved):
    """1 to 32 lanes of 8 channels, powers of two and others, heads that do not fill the last warp; bounds as in
    test_gpu_block_ops.test_qk_norm_rope."""
    vs, axes, B, N = (3, 4, 5), (d // 2, d // 4, d // 4), 2, 60
    table = msl.rotary_table(vs, axes, theta=100.0, device=_dev())
    cos, sin = _angles(table, vs, axes, _positions(vs, 0, N, None, B))
    q, k = _rand(1, B, N, heads * d, dtype=dtype).requires_grad_(), _rand(2, B, N, kv * d, dtype=dtype).requires_grad_()
    gq, gk = (1 + _rand(3, d, std=0.3)).to(dtype).requires_grad_(), (1 + _rand(4, d, std=0.3)).to(dtype).requires_grad_()
    dq, dk = _rand(5, B, N, heads * d, dtype=dtype), _rand(6, B, N, kv * d, dtype=dtype)
    q2, k2 = msl.qk_norm_rope(q, k, gq, gk, table, heads=heads, kv_heads=kv, video_shape=vs, axes=axes, interleaved=interleaved)
    got = torch.autograd.grad([q2, k2], [q, k, gq, gk], [dq, dk])
    half = HALF if dtype == torch.bfloat16 else 0.0
    for y, x, g, dy, nh, dx, dg in ((q2, q, gq, dq, heads, got[0], got[2]), (k2, k, gk, dk, kv, got[1], got[3])):
        w, wm, wdx, wdxm, wdg, wdgm = _ref_norm_rope(x, g, dy, nh, cos, sin, interleaved, 1e-6)
        _within(y.detach(), w, wm, (d / 2 + 16) * EPS, half)
        _within(dx, wdx, wdxm, (2 * d + 32) * EPS, half)
        _within(dg, wdg, wdgm, (d / 2 + 16 + 6 * math.sqrt(B * N * nh)) * EPS, half)


FACTORS = [(1, 64, 72), (5, 72, 200), (16, 256, 640), (17, 264, 328), (300, 256, 1024), (700, 1152, 1000), (1027, 256, 4040), (40, 77, 203), (700, 253, 635)]


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("M,C,F", FACTORS)
def test_gated_ffn_keeps_its_factors_in_24_bits(M, C, F, act):
    """u act'(g) and act(g) as the forward keeps them in bf16, by every form: off by the float32 sums (2 sqrt(C) + 16 EPS of
    the absolute sums, through the activation's slope), the activation's own approximation (2^-15 of its value's scale) and
    the 24th bit (2^-16)."""
    x, w_in, w_out, b_in, b_out = (t.detach() for t in _ffn_case(M, C, F, torch.bfloat16, act, True))
    kept = ops.gated_ffn_fwd(x, w_in, w_out, b_in, b_out, activation=act, keep=True)[2]
    got = _kept_factors(kept, M, F).double()
    gu = x.double() @ w_in.double().t() + b_in.double()
    sums = (2 * math.sqrt(C) + 16) * EPS * (x.double().abs() @ w_in.double().abs().t() + b_in.double().abs())
    g, u, eg, eu = gu[:, :F], gu[:, F:], sums[:, :F], sums[:, F:]
    if act == "silu":
        s = torch.sigmoid(g)
        a, da = g * s, s * (1 + g * (1 - s))
    else:
        s = 0.5 * (1 + torch.erf(g / math.sqrt(2)))
        a, da = g * s, s + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    # |act'| < 1.13 and |act''| < 1 for both
    bound = torch.cat([2 * eg * u.abs() + 1.2 * eu, 1.2 * eg], 1) + 2.0 ** -15 * torch.cat([u.abs() * (da.abs() + 0.5), a.abs() + 0.5 * g.abs()], 1)
    err = (got - torch.cat([u * da, a], 1)).abs()
    assert torch.all(err <= bound + 2.0 ** -16 * got.abs() + 1e-37), float((err / bound).max())


@pytest.mark.parametrize("M,C,F", FACTORS)
def test_gated_ffn_bf16_gradients_have_two_roundings(M, C, F):
    """The gradients of g and u are rounded as operands, then the result: RMS each, and no third one.  (RMS bounds a rounding's
    root mean square at the foot of a binade; over all of it, it is 0.74 of that.  Two make 1.42, three 1.73.)"""
    x, w_in, w_out, _, _ = _ffn_case(M, C, F, torch.bfloat16, "silu", False)
    dy = _rand(9, M, C, dtype=torch.bfloat16)
    y = msl.gated_ffn(x, w_in, w_out)
    dx, dw_in = torch.autograd.grad(y, [x, w_in], dy)
    _, wdx, wdw = _ffn_ref(x, w_in, w_out, None, None, "silu", dy)[:3]
    for name, a, b in (("dx", dx, wdx), ("dw_in", dw_in, wdw)):
        rel = float((a.double() - b).norm() / b.norm())
        assert rel <= 1.5 * 0.74 * RMS, (name, rel)


@pytest.mark.parametrize("C,F", [(64, 96), (61, 75)])
@pytest.mark.parametrize("M", [1, 7, 200])
def test_gated_ffn_kept_factors_that_are_not_finite(M, C, F):
    """NaN and infinities keep what they are through the 24 bits: the row they are in, and no other."""
    x, w_in, w_out, _, _ = (t.detach() if t is not None else None for t in _ffn_case(M, C, F, torch.bfloat16, "silu", False))
    clean = _kept_factors(ops.gated_ffn_fwd(x, w_in, w_out, keep=True)[2], M, F)
    for value in (float("nan"), float("inf")):
        bad = x.clone()
        bad[M - 1, 3] = value
        got = _kept_factors(ops.gated_ffn_fwd(bad, w_in, w_out, keep=True)[2], M, F)
        assert torch.equal(got[:M - 1], clean[:M - 1])
        last = got[M - 1]
        assert torch.isnan(last).all() if math.isnan(value) else not torch.isfinite(last[F:][clean[M - 1, F:].abs() < 1e30]).all()


@pytest.mark.parametrize("dtype,C,F", [(torch.bfloat16, 8, 2056), (torch.bfloat16, 7, 2055), (torch.float32, 8, 2056)], ids=["bf16", "bf16-odd", "fp32"])
def test_gated_ffn_beyond_2_31_elements(dtype, C, F):
    """Hidden values, kept factors and inner gradients of over 2^31 elements: the last rows and, with a gradient in them
    alone, the weights' gradients."""
    M, n = 2 ** 19 + 37, 70
    x = torch.empty(M, C, device=_dev(), dtype=dtype).normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    _, w_in, w_out, b_in, b_out = _ffn_case(1, C, F, dtype, "silu", True)
    x.requires_grad_()
    dy = torch.zeros_like(x)
    dy[-n:] = _rand(9, n, C, dtype=dtype)
    y = msl.gated_ffn(x, w_in, w_out, b_in, b_out)
    got = torch.autograd.grad(y, [x, w_in, w_out, b_in, b_out], dy)
    want = _ffn_ref(x[-n:], w_in, w_out, b_in, b_out, "silu", dy[-n:])
    assert torch.count_nonzero(got[0][:-n]) == 0
    for name, a, b in zip(("y", "dx", "dw_in", "dw_out", "db_in", "db_out"), (y.detach()[-n:], got[0][-n:], *got[1:]), want):
        _close(a, b, (2 * math.sqrt(2 * F) + 16) * EPS if dtype == torch.float32 else (2 if name in ("y", "db_out") else 4) * RMS, name)
