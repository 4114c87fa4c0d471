"""The operators around the attention where the package runs them: DeformableSlideAttention3D(qk_norm, rotary_axes),
MegaSlideDiT with rotary positions, normalised queries and keys and gated blocks, and the CPU-master trainer
with the fused clip.

float32 results of the module are compared with the same attention kernels (checked against the oracle elsewhere)
fed with q and k that plain float64 formulas have normalised and turned: what differs is the rounding of q and k to
float32 (2^-24 each, through a softmax over at most 40 keys of scores of a few units) and the order of the
projections' sums, under 1e-5 together; 1e-4 is allowed, as everywhere for float32 in this package."""

import copy

import pytest
import torch

import megaslide_b200 as msl
from megaslide_b200 import ops
from megaslide_b200.dit import MegaSlideDiT, VideoDiTConfig
from megaslide_b200.stream import CPUMasterVideoDiT

pytestmark = pytest.mark.gpu

RTOL = 1e-4


def _rel(a, b):
    a, b = a.detach(), b.detach()
    return float((a.double() - b.double()).norm() / b.double().norm().clamp_min(1e-30))


def _module(qk_norm, axes, seed=0, C=64, heads=4):
    torch.manual_seed(seed)
    m = msl.DeformableSlideAttention3D(C, heads, (3, 3, 3), qk_norm=qk_norm, rotary_axes=axes, rotary_theta=50.0)
    with torch.no_grad():
        m.offset_net[2].weight.normal_(0, 0.05)
        if qk_norm:
            m.q_norm_weight.normal_(1, 0.2)
            m.k_norm_weight.normal_(1, 0.2)
    return m.cuda()


def _turned(v, w, axes, vs, theta, heads, positions=True):
    """Plain float64 norm (w not None) and rotation of v [B, N, C]."""
    T, H, W = vs
    v = v.double().unflatten(-1, (heads, -1))
    if w is not None:
        v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-6) * w.double()
    if axes is None or not positions:
        return v.flatten(2)
    n = torch.arange(T * H * W, device=v.device)
    ang = []
    for pos, ch in zip((n // (H * W), n // W % H, n % W), axes):
        ang.append(pos[:, None].double() * theta ** (-torch.arange(0, ch, 2, device=v.device, dtype=torch.float64) / max(ch, 1)))
    ang = torch.cat(ang, -1)[None, :, None]
    p = ang.shape[-1]
    a, b = v[..., 0:2 * p:2], v[..., 1:2 * p:2]
    y = torch.stack([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], -1).flatten(-2)
    return torch.cat([y, v[..., 2 * p:]], -1).flatten(2)


OPTIONS = [pytest.param(True, (4, 6, 6), id="norm-rotary"), pytest.param(True, None, id="norm"),
           pytest.param(False, (2, 4, 6), id="rotary-partial")]


@pytest.mark.parametrize("G", [0, 3], ids=["", "extra"])
@pytest.mark.parametrize("qk_norm,axes", OPTIONS)
def test_module_forward_equals_the_plain_preparation(qk_norm, axes, G):
    B, vs, C, heads = 2, (3, 4, 5), 64, 4
    N = 60
    m = _module(qk_norm, axes)
    x = torch.randn(B, N, C, device="cuda")
    extra = torch.randn(B, G, C, device="cuda") if G else None
    with torch.no_grad():
        y = m(x, vs, extra)
        plain = copy.deepcopy(m)
        plain.qk_norm, plain.rotary_axes = False, None
        cap: dict = {}
        plain.capture = cap
        plain(x, vs, extra)
        wq, wk = (m.q_norm_weight, m.k_norm_weight) if qk_norm else (None, None)
        q, k, v = (cap["qkv"][:, i * C:(i + 1) * C].contiguous() for i in range(3))
        q = _turned(q.view(B, N, C), wq, axes, vs, 50.0, heads).float().view(B * N, C)
        k = _turned(k.view(B, N, C), wk, axes, vs, 50.0, heads).float().view(B * N, C)
        ek = ev = None
        if G:
            ek = _turned(m.k_proj(extra), wk, axes, vs, 50.0, heads, positions=False).float().view(B * G, C)
            ev = m.v_proj(extra).view(B * G, C)
        sh = ops.DsaShape(B, *vs, heads, C // heads, (3, 3, 3), extra=G)
        attn, _ = ops.attn_fwd(sh, q, k, v, cap["off"], ek, ev, offset_bias=cap["offset_bias"])
        want = cap["y"] + (attn - cap["attn"]) @ m.out_proj.weight.t()
    assert _rel(y.view(B * N, C), want) <= RTOL
    assert _rel(y.view(B * N, C), cap["y"]) > 10 * RTOL  # the options do something


@pytest.mark.parametrize("G", [0, 3], ids=["", "extra"])
@pytest.mark.parametrize("qk_norm,axes", OPTIONS)
def test_module_gradients_against_differences(qk_norm, axes, G):
    """Given offsets (the sampling positions do not move, so the result is smooth in everything else); central
    differences with step 2^-7: truncation 6e-5 of the third derivative, rounding 2^-20 of the result over the
    step, 2e-3 of the gradient's scale together at most."""
    B, vs, C = 1, (2, 3, 4), 64
    m = _module(qk_norm, axes)
    off = torch.randn(B, 24, 4 * 27 * 3, device="cuda") * 0.5
    x = torch.randn(B, 24, C, device="cuda")
    extra = torch.randn(B, G, C, device="cuda") if G else None
    g = torch.randn(B, 24, C, device="cuda")
    leaves = {"x": x, **({"extra": extra} if G else {}), "q_proj": m.q_proj.weight, "k_proj": m.k_proj.weight}
    if qk_norm:
        leaves |= {"q_norm": m.q_norm_weight, "k_norm": m.k_norm_weight}
    for t in leaves.values():
        t.requires_grad_(True)
    y = m.forward_with_offsets(x, vs, off, extra)
    grads = torch.autograd.grad(y, list(leaves.values()), g)
    step = 2.0 ** -7
    for (name, t), grad in zip(leaves.items(), grads):
        torch.manual_seed(7)
        v = torch.randn_like(t)
        v *= t.detach().norm() / v.norm()  # a step of 2^-7 of the operand
        vals = []
        with torch.no_grad():
            for s in (step, -2 * step, step):
                vals.append(float((m.forward_with_offsets(x, vs, off, extra).double() * g.double()).sum()))
                t.add_(v, alpha=s)
        hi, lo = vals[1], vals[2]
        scale = float(grad.double().norm() * v.double().norm())
        assert abs((hi - lo) / (2 * step) - float((grad.double() * v.double()).sum())) <= 2e-3 * scale, name


def test_options_off_leave_the_module_as_it_was():
    m = msl.DeformableSlideAttention3D(64, 4, (3, 3, 3))
    assert not any("norm" in k for k in m.state_dict())
    with pytest.raises(ValueError, match="rotary_axes"):
        msl.DeformableSlideAttention3D(64, 4, (3, 3, 3), rotary_axes=(8, 8, 8))
    with pytest.raises(ValueError, match="even"):
        msl.DeformableSlideAttention3D(60, 4, (3, 3, 3), qk_norm=True)


def _cfg(dtype, resident):
    return VideoDiTConfig(frames=4, in_channels=4, height=16, width=16, patch_size=2, hidden_size=64, num_heads=2, num_layers=5,
                          dsa_kernel_size=(3, 3, 3), checkpoint_interval=2, num_grad_slabs=3, learning_rate=1e-3,
                          weight_decay=0.01, max_grad_norm=1.0, dtype=dtype, device=0, log_interval=0, qk_norm=True,
                          rotary_axes=(8, 12, 12), gated_mlp=True, fused_clip=True, resident_blocks=resident)


@pytest.mark.parametrize("resident", [False, True], ids=["streamed", "resident"])
@pytest.mark.parametrize("dtype,tol", [("float32", 1e-4), ("bfloat16", 3e-2)])
def test_training_steps_of_a_model_with_every_operator(dtype, tol, resident):
    """Two steps of CPUMasterVideoDiT against the same model trained in place with plain autograd, torch's clipping
    and AdamW (the existing trainer test's form and tolerances)."""
    torch.manual_seed(3)
    cfg = _cfg(dtype, resident)
    model = MegaSlideDiT(cfg)
    with torch.no_grad():
        for b in model.blocks:
            b.attn.offset_net[2].weight.normal_(0, 0.05)
    ref = copy.deepcopy(model).cuda()
    opt = torch.optim.AdamW(ref.parameters(), lr=cfg.learning_rate, betas=(cfg.beta1, cfg.beta2), eps=cfg.eps,
                            weight_decay=cfg.weight_decay)
    trainer = CPUMasterVideoDiT(model, cfg)
    try:
        for step in range(2):
            gen = torch.Generator().manual_seed(step)
            lat = torch.randn(2, cfg.in_channels, cfg.frames, cfg.height, cfg.width, generator=gen)
            noise = torch.randn(lat.shape, generator=gen)
            ts = torch.randint(0, 1000, (2,), generator=gen)
            with torch.autocast("cuda", dtype=torch.bfloat16, enabled=dtype == "bfloat16"):
                pred = ref(lat.cuda(), ts.cuda())
            loss_ref = torch.nn.functional.mse_loss(pred.float(), noise.cuda())
            opt.zero_grad()
            loss_ref.backward()
            norm_ref = float(torch.nn.utils.clip_grad_norm_(ref.parameters(), cfg.max_grad_norm))
            opt.step()
            trainer.zero_grad()
            loss, _ = trainer.forward_and_backward(lat, ts, noise)
            norm = trainer.optimizer_step()
            loss_ref = float(loss_ref.detach())
            assert abs(loss - loss_ref) <= tol * abs(loss_ref), (step, loss, loss_ref)
            assert abs(norm - norm_ref) <= tol * norm_ref, (step, norm, norm_ref)
        if dtype != "float32":
            return
        got = dict(zip([n for n, _ in model.named_parameters()], trainer.get_parameters()))
        for name, p in ref.named_parameters():
            if name.endswith("attn.k_proj.bias"):
                continue
            assert _rel(got[name].detach().float().cpu(), p.detach().float().cpu()) <= tol, name
    finally:
        trainer.cleanup()


def test_gated_mlp_module_and_autocast():
    torch.manual_seed(0)
    m = msl.GatedMLP(96, 160, activation="gelu").cuda()
    x = torch.randn(2, 33, 96, device="cuda", requires_grad=True)
    with torch.no_grad():
        g, u = m.fc1(x).double().chunk(2, -1)
        want = torch.nn.functional.linear(torch.nn.functional.gelu(g) * u, m.fc2.weight.double(), m.fc2.bias.double())
    assert _rel(m(x), want) <= RTOL
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = m(x)
    assert y.dtype == torch.bfloat16 and _rel(y, want) <= 2e-2
    y.float().sum().backward()
    assert x.grad.dtype == torch.float32 and m.fc1.weight.grad.shape == (320, 96)
