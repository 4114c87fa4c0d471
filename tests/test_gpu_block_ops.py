"""The operators around the attention on the GPU (rope3d, qk_norm_rope, gated_ffn, grad_norm, clip_grad_norm_)
against plain float64 implementations of their formulas, forward and backward, at the sizes, layouts and values
where they can go wrong.

Tolerances.  EPS = 2^-24 is float32's rounding, HALF = 2^-8 that of a bfloat16 result (8 significant bits), RMS =
2^-8 / sqrt(3) its root mean square.  Elementwise bounds are sums of the absolute terms of each formula times the
roundings on the way; sums of n terms are allowed 6 standard deviations of a random walk of roundings (6 sqrt(n)
EPS of the absolute sum) where the worst case says nothing.  Matrix products are bounded in the 2-norm: 2 sqrt(K) + 16
roundings in float32; in bfloat16 RMS for each rounded intermediate and the result (forward: h, y; backward: the
kept projections, h, their gradients, the result).
"""

import ctypes
import math
import threading

import pytest
import torch

import megaslide_b200 as msl
from megaslide_b200 import _lib, ops

pytestmark = pytest.mark.gpu

EPS, HALF, RMS = 2.0 ** -24, 2.0 ** -8, 2.0 ** -8 / math.sqrt(3)
DTYPES = [torch.float32, torch.bfloat16]
IDS = ["fp32", "bf16"]


def _dev():
    return torch.device("cuda:0")


def _rand(seed, *shape, dtype=torch.float32, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype).to(_dev())


def _half(dtype):
    return HALF if dtype == torch.bfloat16 else 0.0


# ---------------------------------------------------------------------------------- rotary positions


def _positions(video_shape, frame0, N, index, B):
    T, H, W = video_shape
    if index is not None:
        ix = index.long().reshape(-1, N, 3)
        return ix.expand(B, N, 3) if ix.shape[0] == 1 else ix
    n = torch.arange(N, device=_dev())
    return torch.stack([frame0 + n // (H * W), n // W % H, n % W], -1)[None].expand(B, N, 3)


def _angles(table, video_shape, axes, pos):
    """cos, sin float64 [B, N, 1, pairs]."""
    out, at = [], 0
    for i, (size, ch) in enumerate(zip(video_shape, axes)):
        n = size * ch // 2
        part = table[at:at + n].double().view(size, ch // 2, 2)
        at += n
        out.append(part[pos[..., i]])
    cs = torch.cat(out, -2)[:, :, None]
    return cs[..., 0], cs[..., 1]


def _pairs(v, n, interleaved):
    return (v[..., 0:2 * n:2], v[..., 1:2 * n:2]) if interleaved else (v[..., :n], v[..., n:2 * n])


def _turn(v, cos, sin, interleaved):
    """(rotated float64, sum of the absolute terms)."""
    n = cos.shape[-1]
    a, b = _pairs(v, n, interleaved)
    y, z = a * cos - b * sin, b * cos + a * sin
    m = (a.abs() * cos.abs() + b.abs() * sin.abs(), b.abs() * cos.abs() + a.abs() * sin.abs())

    def join(p, q):
        t = torch.stack([p, q], -1).flatten(-2) if interleaved else torch.cat([p, q], -1)
        return t

    return torch.cat([join(y, z), v[..., 2 * n:]], -1), torch.cat([join(*m), v[..., 2 * n:].abs()], -1)


def _ref_norm_rope(x, g, dy, heads, cos, sin, interleaved, eps):
    """Formulas in float64: (y, its bound's magnitude, dx, magnitude, dg, magnitude)."""
    v = x.detach().double().unflatten(-1, (heads, -1))
    d = v.shape[-1]
    w = g.detach().double() if g is not None else torch.ones(d, device=x.device, dtype=torch.float64)
    r = 1 / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)
    y, ym = _turn(v * r * w, cos, sin, interleaved)
    if dy is None:
        return y.flatten(2), ym.flatten(2)
    dn, dm = _turn(dy.double().unflatten(-1, (heads, -1)), cos, -sin, interleaved)
    dg, dgm = (dn * v * r).sum((0, 1, 2)), (dm * (v * r).abs()).sum((0, 1, 2))
    a, am = dn * w, dm * w.abs()
    dx = r * (a - v * r * r * (a * v).mean(-1, keepdim=True))
    dxm = r * (am + v.abs() * r * r * (am * v.abs()).mean(-1, keepdim=True))
    return y.flatten(2), ym.flatten(2), dx.flatten(2), dxm.flatten(2), dg, dgm


def _within(got, want, magnitude, relative, half):
    err = (got.double() - want).abs()
    lim = relative * magnitude + half * (want.abs() + relative * magnitude) + 1e-30
    worst = float((err / lim).max()) if err.numel() else 0.0
    assert torch.isfinite(got.float()).all() or not torch.isfinite(want).all()
    assert worst <= 1.0, worst


ROTARY = [
    # B, (T, H, W), frame0, frames, heads, kv_heads, head_dim, axes
    pytest.param(1, (1, 1, 1), 0, 1, 1, 1, 2, (2, 0, 0), id="one-token-one-pair"),
    pytest.param(2, (5, 3, 7), 0, 5, 3, 3, 64, (16, 24, 24), id="odd-video"),
    pytest.param(1, (6, 4, 5), 2, 3, 16, 16, 72, (24, 24, 24), id="head-72-frame0"),
    pytest.param(3, (4, 2, 3), 0, 4, 8, 2, 72, (16, 24, 24), id="grouped-partial"),
    pytest.param(1, (2, 5, 4), 0, 2, 5, 1, 128, (32, 48, 48), id="head-128-one-key-head"),
    pytest.param(2, (3, 4, 4), 1, 1, 4, 4, 80, (22, 28, 30), id="axes-inside-a-vector"),
    pytest.param(1, (2, 3, 3), 0, 2, 7, 7, 6, (2, 2, 2), id="head-6"),
    pytest.param(1, (2, 3, 3), 0, 2, 2, 2, 98, (20, 30, 40), id="head-98"),
    pytest.param(2, (2, 3, 3), 0, 2, 2, 1, 256, (64, 96, 96), id="head-256"),
    pytest.param(1, (2, 3, 3), 0, 2, 3, 3, 100, (0, 40, 40), id="two-axes"),
]


@pytest.mark.parametrize("interleaved", [True, False], ids=["interleaved", "split"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("B,vs,frame0,frames,heads,kv,d,axes", ROTARY)
def test_rope3d(B, vs, frame0, frames, heads, kv, d, axes, dtype, interleaved):
    N = frames * vs[1] * vs[2]
    table = msl.rotary_table(vs, axes, theta=100.0, device=_dev())
    cos, sin = _angles(table, vs, axes, _positions(vs, frame0, N, None, B))
    x, dy = _rand(1, B, N, heads * d, dtype=dtype).requires_grad_(), _rand(2, B, N, heads * d, dtype=dtype)
    kw = dict(video_shape=vs, axes=axes, heads=heads, interleaved=interleaved, frame0=frame0)
    y = msl.rope3d(x, table, **kw)
    (dx,) = torch.autograd.grad(y, x, dy)
    assert y.dtype == dtype and dx.dtype == dtype
    for got, src, s in ((y, x, sin), (dx, dy, -sin)):
        want, mag = _turn(src.detach().double().unflatten(-1, (heads, d)), cos, s, interleaved)
        _within(got.detach(), want.flatten(2), mag.flatten(2), 4 * EPS, _half(dtype))
    # the gradient against differences: the rotation is linear, so they are exact but for rounding
    v = _rand(3, B, N, heads * d, dtype=dtype)
    with torch.no_grad():
        change = (msl.rope3d(v, table, **kw).double() * dy.double()).sum()
    terms = (v.double() * dy.double()).abs().sum()
    assert abs(float(change - (v.double() * dx.double()).sum())) <= float(terms) * 2 * (8 * EPS + 2 * _half(dtype))


@pytest.mark.parametrize("interleaved", [True, False], ids=["interleaved", "split"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("B,vs,frame0,frames,heads,kv,d,axes", ROTARY)
def test_qk_norm_rope(B, vs, frame0, frames, heads, kv, d, axes, dtype, interleaved):
    N = frames * vs[1] * vs[2]
    table = msl.rotary_table(vs, axes, theta=100.0, device=_dev())
    cos, sin = _angles(table, vs, axes, _positions(vs, frame0, N, None, B))
    q, k = _rand(1, B, N, heads * d, dtype=dtype).requires_grad_(), _rand(2, B, N, kv * d, dtype=dtype).requires_grad_()
    gq, gk = (1 + _rand(3, d, std=0.3)).to(dtype).requires_grad_(), (1 + _rand(4, d, std=0.3)).to(dtype).requires_grad_()
    dq, dk = _rand(5, B, N, heads * d, dtype=dtype), _rand(6, B, N, kv * d, dtype=dtype)
    q2, k2 = msl.qk_norm_rope(q, k, gq, gk, table, heads=heads, kv_heads=kv, video_shape=vs, axes=axes,
                              interleaved=interleaved, frame0=frame0)
    got = torch.autograd.grad([q2, k2], [q, k, gq, gk], [dq, dk])
    for y, x, g, dy, nh, dx, dg in ((q2, q, gq, dq, heads, got[0], got[2]), (k2, k, gk, dk, kv, got[1], got[3])):
        w, wm, wdx, wdxm, wdg, wdgm = _ref_norm_rope(x, g, dy, nh, cos, sin, interleaved, 1e-6)
        _within(y.detach(), w, wm, (d / 2 + 16) * EPS, _half(dtype))
        _within(dx, wdx, wdxm, (2 * d + 32) * EPS, _half(dtype))
        _within(dg, wdg, wdgm, (d / 2 + 16 + 6 * math.sqrt(B * N * nh)) * EPS, _half(dtype))


def test_qk_norm_rope_gradient_against_differences():
    B, vs, heads, d, axes = 1, (2, 3, 2), 2, 12, (4, 4, 4)
    N = 12
    table = msl.rotary_table(vs, axes, theta=10.0, device=_dev())
    args = [_rand(1, B, N, heads * d), _rand(2, B, N, heads * d), 1 + _rand(3, d, std=0.2), 1 + _rand(4, d, std=0.2)]
    out = [_rand(5, B, N, heads * d).double(), _rand(6, B, N, heads * d).double()]

    def f(a):
        with torch.no_grad():
            r = msl.qk_norm_rope(*a, table, heads=heads, video_shape=vs, axes=axes)
        return float(sum((x.double() * o).sum() for x, o in zip(r, out)))

    leaves = [a.clone().requires_grad_() for a in args]
    r = msl.qk_norm_rope(*leaves, table, heads=heads, video_shape=vs, axes=axes)
    grads = torch.autograd.grad(list(r), leaves, [o.float() for o in out])
    step = 2.0 ** -8
    for i, g in enumerate(grads):
        v = _rand(10 + i, *g.shape)
        hi = f([a + step * v if j == i else a for j, a in enumerate(args)])
        lo = f([a - step * v if j == i else a for j, a in enumerate(args)])
        # truncation ~ step^2 of the scale; rounding: the results' 2^-22 relative over 2 step
        scale = float(g.double().norm() * v.double().norm())
        assert abs((hi - lo) / (2 * step) - float((g.double() * v.double()).sum())) <= scale * 2e-3


@pytest.mark.parametrize("per_sample", [True, False], ids=["index-per-sample", "index-shared"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_positions_from_an_index(dtype, per_sample):
    B, N, vs, axes, heads, kv, d = 3, 37, (9, 5, 11), (8, 12, 12), 6, 3, 40
    g = torch.Generator().manual_seed(0)
    ix = torch.stack([torch.randint(0, s, (B, N) if per_sample else (N,), generator=g) for s in vs], -1).int().to(_dev())
    table = msl.rotary_table(vs, axes, device=_dev())
    cos, sin = _angles(table, vs, axes, _positions(vs, 0, N, ix, B))
    q, k = _rand(1, B, N, heads * d, dtype=dtype).requires_grad_(), _rand(2, B, N, kv * d, dtype=dtype).requires_grad_()
    dq, dk = _rand(5, B, N, heads * d, dtype=dtype), _rand(6, B, N, kv * d, dtype=dtype)
    kw = dict(video_shape=vs, axes=axes, heads=heads, index=ix)
    want, mag = _turn(q.detach().double().unflatten(-1, (heads, d)), cos, sin, True)
    _within(msl.rope3d(q.detach(), table, **kw), want.flatten(2), mag.flatten(2), 4 * EPS, _half(dtype))
    q2, k2 = msl.qk_norm_rope(q, k, None, None, table, kv_heads=kv, **kw)
    gq, gk = torch.autograd.grad([q2, k2], [q, k], [dq, dk])
    for y, x, dy, nh, dx in ((q2, q, dq, heads, gq), (k2, k, dk, kv, gk)):
        w, wm, wdx, wdxm, _, _ = _ref_norm_rope(x, None, dy, nh, cos, sin, True, 1e-6)
        _within(y.detach(), w, wm, (d / 2 + 16) * EPS, _half(dtype))
        _within(dx, wdx, wdxm, (2 * d + 32) * EPS, _half(dtype))
    msl.check_status()


def test_norm_without_rotation_and_empty_rows():
    dev = _dev()
    x = _rand(1, 2, 5, 3 * 40)
    x[0, 1] = 0
    q2, k2 = msl.qk_norm_rope(x, x, None, None, heads=3)
    w, wm = _ref_norm_rope(x, None, None, 3, torch.ones(2, 5, 1, 0, device=dev), torch.zeros(2, 5, 1, 0, device=dev), True, 1e-6)
    _within(q2, w, wm, (40 / 2 + 16) * EPS, 0.0)
    assert torch.equal(q2, k2) and torch.count_nonzero(q2[0, 1]) == 0  # a zero head stays zero
    # eps = 0: a zero head has no direction, as the formula says; its neighbours are not touched
    q0, _ = msl.qk_norm_rope(x, x, None, None, heads=3, eps=0.0)
    assert torch.isnan(q0[0, 1]).all() and torch.isfinite(q0[0, 0]).all() and torch.isfinite(q0[0, 2]).all()
    # no tokens: empty results, zero gradients of the weights
    e = torch.empty(2, 0, 80, device=dev, requires_grad=True)
    g = torch.ones(40, device=dev, requires_grad=True)
    t = msl.rotary_table((2, 2, 2), (8, 8, 8), device=dev)
    a, b = msl.qk_norm_rope(e, e, g, g, t, heads=2, video_shape=(2, 2, 2), axes=(8, 8, 8))
    assert a.shape == (2, 0, 80)
    (dg,) = torch.autograd.grad([a, b], g, [torch.empty_like(a), torch.empty_like(b)])
    assert torch.equal(dg, torch.zeros_like(dg))
    assert msl.rope3d(e.detach(), t, video_shape=(2, 2, 2), axes=(8, 8, 8), heads=2).shape == (2, 0, 80)


def test_values_that_are_not_finite_stay_in_their_head():
    vs, axes, heads, d = (2, 2, 3), (8, 12, 12), 4, 32
    table = msl.rotary_table(vs, axes, device=_dev())
    x = _rand(1, 1, 12, heads * d)
    clean = msl.qk_norm_rope(x, x, None, None, table, heads=heads, video_shape=vs, axes=axes)[0]
    bad = x.clone()
    bad[0, 3, d + 5], bad[0, 7, 2 * d] = float("nan"), float("inf")
    got = msl.qk_norm_rope(bad, bad, None, None, table, heads=heads, video_shape=vs, axes=axes)[0].view(1, 12, heads, d)
    assert torch.isnan(got[0, 3, 1]).all() and torch.isnan(got[0, 7, 2, :].sum())
    keep = torch.ones(1, 12, heads, dtype=torch.bool, device=_dev())
    keep[0, 3, 1] = keep[0, 7, 2] = False
    assert torch.equal(got[keep], clean.view(1, 12, heads, d)[keep])


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_rotary_strides_in_place_and_alignment(dtype):
    """q and k as columns of a qkv buffer, in place; a buffer whose rows start off any vector's boundary; a sample
    stride that no row view has."""
    vs, axes, heads, kv, d = (2, 3, 4), (8, 12, 12), 4, 2, 32
    B, N = 2, 24
    table = msl.rotary_table(vs, axes, device=_dev())
    kw = dict(video_shape=vs, axes=axes, heads=heads)
    q, k = _rand(1, B, N, heads * d, dtype=dtype), _rand(2, B, N, kv * d, dtype=dtype)
    gq, gk = 1 + _rand(3, d, std=0.3), 1 + _rand(4, d, std=0.3)
    want_q, want_k = msl.qk_norm_rope(q, k, gq, gk, table, kv_heads=kv, **kw)
    for shift, width in ((0, heads * d + 2 * kv * d), (1, heads * d + kv * d + 3)):
        buf = torch.zeros(B, N, width, dtype=dtype, device=_dev())
        bq, bk = buf[..., shift:shift + heads * d], buf[..., shift + heads * d:shift + (heads + kv) * d]
        bq.copy_(q), bk.copy_(k)
        a, b = msl.qk_norm_rope(bq, bk, gq, gk, table, kv_heads=kv, **kw)
        assert torch.allclose(a, want_q, rtol=2 * HALF if dtype == torch.bfloat16 else 8 * EPS, atol=1e-6)
        assert torch.allclose(b, want_k, rtol=2 * HALF if dtype == torch.bfloat16 else 8 * EPS, atol=1e-6)
        sh = ops.RotaryShape(B, N, vs, axes, d)
        rows = buf.view(B * N, width)
        rq, rk = rows[:, shift:shift + heads * d], rows[:, shift + heads * d:shift + (heads + kv) * d]
        ops.qk_norm_rope_fwd(sh, heads, kv, rq, rk, gq, gk, 1e-6, table, q_out=rq, k_out=rk)
        assert torch.equal(rq.reshape(B, N, -1), a) and torch.equal(rk.reshape(B, N, -1), b)
    t = q.transpose(0, 1).contiguous().transpose(0, 1)  # samples interleaved in memory
    assert torch.equal(msl.rope3d(t, table, **kw), msl.rope3d(q, table, **kw))


def test_weight_gradients_are_the_same_on_every_run():
    vs, axes, heads, d = (4, 32, 32), (16, 24, 24), 8, 64
    table = msl.rotary_table(vs, axes, device=_dev())
    q, k = (_rand(i, 1, 4096, heads * d, dtype=torch.bfloat16).requires_grad_() for i in (1, 2))
    g = torch.ones(d, device=_dev(), requires_grad=True)
    runs = []
    for _ in range(3):
        r = msl.qk_norm_rope(q, k, g, g, table, heads=heads, video_shape=vs, axes=axes)
        runs.append(torch.autograd.grad([r[0], r[1]], g, [q.detach(), k.detach()])[0])
    assert torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])


def test_index_outside_its_axis_is_reported():
    vs, axes = (3, 4, 5), (4, 4, 4)
    table = msl.rotary_table(vs, axes, device=_dev())
    x = _rand(1, 1, 2, 16)
    ix = torch.tensor([[1, 2, 3], [1, 4, 3]], dtype=torch.int32, device=_dev())
    msl.rope3d(x, table, video_shape=vs, axes=axes, heads=1, index=ix)
    with pytest.raises(msl.MslError, match="outside its axis"):
        msl.check_status()
    msl.check_status()  # reported once; the context is fine
    ix[1, 1] = 3
    y = msl.rope3d(x, table, video_shape=vs, axes=axes, heads=1, index=ix)
    assert torch.isfinite(y).all()
    msl.check_status()


def test_rotary_rows_beyond_2_31_elements():
    heads, d = 16, 64
    N = 2 ** 21 + 5  # 2^31 + 5120 elements, 4.3 GB
    x = torch.zeros(1, N, heads * d, dtype=torch.bfloat16, device=_dev())
    x[0, -5:] = _rand(1, 5, heads * d, dtype=torch.bfloat16)
    axes = (32, 0, 0)
    table = msl.rotary_table((5, 1, 1), axes, device=_dev())
    ix = torch.zeros(N, 3, dtype=torch.int32, device=_dev())
    ix[-5:, 0] = torch.arange(5)
    y = msl.rope3d(x, table, video_shape=(5, 1, 1), axes=axes, heads=heads, index=ix)
    tail = msl.rope3d(x[:, -5:].contiguous(), table, video_shape=(5, 1, 1), axes=axes, heads=heads)
    assert torch.equal(y[:, -5:], tail) and torch.count_nonzero(y[:, :-5]) == 0


# ---------------------------------------------------------------------------------- gated feed-forward block


def _ffn_ref(x, w_in, w_out, b_in, b_out, act, dy):
    """Formulas in float64: y, dx, dw_in, dw_out, db_in, db_out."""
    x, w_in, w_out, dy = (t.detach().double() for t in (x, w_in, w_out, dy))
    F = w_out.shape[1]
    gu = x @ w_in.t() + (b_in.detach().double() if b_in is not None else 0)
    g, u = gu[:, :F], gu[:, F:]
    if act == "silu":
        s = torch.sigmoid(g)
        a, da = g * s, s * (1 + g * (1 - s))
    else:
        s = 0.5 * (1 + torch.erf(g / math.sqrt(2)))
        a, da = g * s, s + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    h = a * u
    y = h @ w_out.t() + (b_out.detach().double() if b_out is not None else 0)
    dh = dy @ w_out
    dgu = torch.cat([dh * u * da, dh * a], 1)
    return y, dgu @ w_in, dgu.t() @ x, dy.t() @ h, dgu.sum(0), dy.sum(0)


def _close(got, want, tol, what):
    assert torch.isfinite(got.float()).all(), what
    err = got.double() - want
    rel = float(err.norm() / want.norm().clamp_min(1e-30))
    assert rel <= tol, (what, rel, tol)
    worst = float(err.abs().max() / (want.abs() + want.square().mean().sqrt()).max().clamp_min(1e-30))
    assert worst <= 8 * tol, (what, worst, tol)


def _ffn_case(M, C, F, dtype, act, bias, seed=0):
    x = _rand(seed + 1, M, C, dtype=dtype).requires_grad_()
    w_in = _rand(seed + 2, 2 * F, C, dtype=dtype, std=C ** -0.5).requires_grad_()
    w_out = _rand(seed + 3, C, F, dtype=dtype, std=F ** -0.5).requires_grad_()
    b_in = _rand(seed + 4, 2 * F, dtype=dtype, std=0.3).requires_grad_() if bias else None
    b_out = _rand(seed + 5, C, dtype=dtype, std=0.3).requires_grad_() if bias else None
    return x, w_in, w_out, b_in, b_out


def _ffn_check_all(M, C, F, dtype, act, bias):
    x, w_in, w_out, b_in, b_out = _ffn_case(M, C, F, dtype, act, bias)
    dy = _rand(9, M, C, dtype=dtype)
    y = msl.gated_ffn(x, w_in, w_out, b_in, b_out, activation=act)
    leaves = [t for t in (x, w_in, w_out, b_in, b_out) if t is not None]
    got = [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    want = _ffn_ref(x, w_in, w_out, b_in, b_out, act, dy)[:len(got)]
    K = max(C, 2 * F, M)
    names = ("y", "dx", "dw_in", "dw_out", "db_in", "db_out")
    for name, a, b in zip(names, got, want):
        tol = (2 * math.sqrt(K) + 16) * EPS if dtype == torch.float32 else (2 if name in ("y", "db_out") else 4) * RMS
        assert a.dtype == dtype
        _close(a, b, tol, name)
    with torch.no_grad():  # the form that keeps nothing gives the same result
        assert torch.equal(msl.gated_ffn(x, w_in, w_out, b_in, b_out, activation=act), y)
    msl.check_status()


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("M,C,F", [(1, 8, 8), (1, 64, 160), (3, 256, 640), (17, 72, 200), (33, 128, 136), (127, 256, 384), (129, 264, 256),
                                   (300, 256, 1024), (64, 1, 1), (5, 30, 75), (70, 130, 61), (200, 100, 250)])
def test_gated_ffn(M, C, F, dtype, act):
    _ffn_check_all(M, C, F, dtype, act, bias=act == "gelu")


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("M,C,F,bias", [(700, 1150, 2301, True), (333, 640, 1604, False), (2048, 256, 1024, True), (9249, 253, 1020, True),
                                        (40, 1533, 6143, False), (1000, 1001, 1600, True)])
def test_gated_ffn_widths_that_no_vector_divides(M, C, F, bias, dtype, act):
    """Widths off any vector's or tile's multiple, large enough for the tensor cores: float32 as three planes, bf16 as
    padded copies, sums of the last tiles cut along k."""
    _ffn_check_all(M, C, F, dtype, act, bias)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("M,C,F,bias", [(1, 1152, 4608, True), (8, 1152, 2880, False), (1027, 1536, 3840, False), (2500, 640, 1600, True)])
def test_gated_ffn_sizes(M, C, F, bias, dtype):
    _ffn_check_all(M, C, F, dtype, "silu", bias)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 7, 8, 9, 13, 16, 17])
def test_gated_ffn_few_rows(M, dtype):
    """Single tokens up to the first size beyond their form, k that no warp's loads divide, and a long k."""
    for C, F, bias in ((72, 200, True), (1160, 392, False), (64, 9000, True), (8, 8, False), (1152, 1228, True), (64, 75, True), (77, 64, True)):
        _ffn_check_all(M, C, F, dtype, "gelu", bias)


@pytest.mark.parametrize("M", [8, 9, 16])
def test_gated_ffn_few_rows_of_wide_weights(M):
    """Weights beyond the size up to which 9 to 16 rows go by rows."""
    _ffn_check_all(M, 4104, 4096, torch.bfloat16, "silu", True)


@pytest.mark.parametrize("M,C,F", [(1, 1152, 4608), (6, 2560, 1000), (13, 640, 2240), (16, 100, 70), (17, 250, 639), (30, 1152, 2880), (65, 640, 1600),
                                   (100, 77, 1531)])
def test_gated_ffn_float32_few_rows(M, C, F):
    """The CUDA-core form: 16 and 64 rows a tile, shares of k, widths off its vectors."""
    _ffn_check_all(M, C, F, torch.float32, "silu", True)


@pytest.mark.parametrize("M", [1, 3, 12, 30, 50, 64, 65])
def test_gated_ffn_float32_few_rows_of_wide_weights(M):
    """Weights of 64 MB: split on the way to the tensor cores, up to 64 rows; columns and k off the blocks' multiples."""
    _ffn_check_all(M, 4100, 4108, torch.float32, "gelu", True)


def test_gated_ffn_float32_wide_weights_off_16_bytes():
    """The same weights with rows of x that no 16-byte copy reads, and with weights at an odd address, go another way."""
    M, C, F = 12, 4100, 4108
    x, w_in, w_out, b_in, b_out = (t.detach() for t in _ffn_case(M, C, F, torch.float32, "silu", True))
    want = msl.gated_ffn(x, w_in, w_out, b_in, b_out)
    padded = torch.zeros(M, C + 1, device=_dev())
    padded[:, :C] = x.reshape(M, C)
    flat = torch.cat([torch.zeros(1, device=_dev()), w_in.reshape(-1)])
    tol = 2 * (2 * math.sqrt(F) + 16) * EPS
    _close(msl.gated_ffn(padded[:, :C], w_in, w_out, b_in, b_out), want.reshape(M, C).double(), tol, "x")
    _close(msl.gated_ffn(x, flat[1:].view(2 * F, C), w_out, b_in, b_out), want.double(), tol, "w_in")


def test_gated_ffn_without_rows():
    x, w_in, w_out, b_in, b_out = _ffn_case(0, 64, 96, torch.bfloat16, "silu", True)
    y = msl.gated_ffn(x, w_in, w_out, b_in, b_out)
    assert y.shape == (0, 64)
    for g in torch.autograd.grad(y, [x, w_in, w_out, b_in, b_out], torch.empty_like(y)):
        assert torch.count_nonzero(g) == 0


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_gated_ffn_some_gradients_and_strides(dtype):
    """Each subset of gradients a caller may ask for; x and dy as columns of wider buffers, 3-D, off any alignment."""
    M, C, F = 60, 96, 160
    x, w_in, w_out, b_in, b_out = _ffn_case(M, C, F, dtype, "silu", True)
    dy = _rand(9, M, C, dtype=dtype)
    y = msl.gated_ffn(x, w_in, w_out, b_in, b_out)
    full = torch.autograd.grad(y, [x, w_in, w_out, b_in, b_out], dy)
    for i, leaf in enumerate((x, w_in, w_out, b_in, b_out)):
        args = [t.detach() for t in (x, w_in, w_out, b_in, b_out)]
        args[i] = leaf
        (g,) = torch.autograd.grad(msl.gated_ffn(*args), leaf, dy)
        assert torch.equal(g, full[i])
    tol = (2 * math.sqrt(2 * F) + 16) * EPS if dtype == torch.float32 else 4 * RMS
    for shift in (0, 1, 8):
        wide = torch.zeros(4, 15, C + 24, dtype=dtype, device=_dev())
        wide[..., shift:shift + C] = x.detach().view(4, 15, C)
        xs = wide[..., shift:shift + C].requires_grad_()
        dys = torch.zeros(4, 15, C + 24, dtype=dtype, device=_dev())
        dys[..., shift:shift + C] = dy.view(4, 15, C)
        ys = msl.gated_ffn(xs, w_in, w_out, b_in, b_out)
        _close(ys.detach().view(M, C), y.detach().double(), 2 * tol, "y")
        got = torch.autograd.grad(ys, [xs, w_in], dys[..., shift:shift + C])
        _close(got[0].reshape(M, C), full[0].double(), 2 * tol, "dx")
        _close(got[1], full[1].double(), 2 * tol, "dw_in")


def test_gated_ffn_weights_inside_a_packed_buffer():
    """Weights at any element of a flat buffer, as the CPU-master trainer packs them: results as from weights of
    their own, within the rounding of sums in another order."""
    M, C, F = 700, 256, 512
    x, w_in, w_out, b_in, b_out = (t.detach() for t in _ffn_case(M, C, F, torch.bfloat16, "silu", True))
    dy = _rand(9, M, C, dtype=torch.bfloat16)

    def run(*ws):
        leaves = [x.clone().requires_grad_(), *(w.requires_grad_() for w in ws)]
        y = msl.gated_ffn(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    want = run(w_in.clone(), w_out.clone(), b_in.clone(), b_out.clone())
    for first in (1, 2, 4):
        flat = torch.cat([torch.zeros(first, dtype=torch.bfloat16, device=_dev())] + [t.reshape(-1) for t in (w_in, w_out, b_in, b_out)])
        views, at = [], first
        for t in (w_in, w_out, b_in, b_out):
            views.append(flat[at:at + t.numel()].view(t.shape).detach())
            at += t.numel()
        for name, a, b in zip(("y", "dx", "dw_in", "dw_out", "db_in", "db_out"), run(*views), want):
            _close(a, b.double(), 2 * RMS, name)


@pytest.mark.parametrize("M,C,F,x_ld", [(40, 16, 32, 17), (40, 15, 32, 16), (3, 16, 32, 17), (3, 15, 32, 16)])
def test_gated_ffn_entry_refuses_rows_off_16_bytes_without_room(M, C, F, x_ld):
    """A C caller that leaves unaligned at 0 gets an error for such rows, and nothing is written; odd widths say
    it by themselves."""
    lib = _lib.load()
    x = torch.zeros(M, x_ld, device=_dev(), dtype=torch.bfloat16)
    w_in, w_out = (torch.zeros(n, device=_dev(), dtype=torch.bfloat16) for n in (2 * F * C, C * F))
    h, y = (torch.full((M, n), 7.0, device=_dev(), dtype=torch.bfloat16) for n in (F, C))
    g = _lib.FfnGeometry(M, C, F, _lib.MSL_DTYPE_BF16, 0, 0)
    io = _lib.FfnIO(x=x.data_ptr(), x_ld=x_ld, w_in=w_in.data_ptr(), w_out=w_out.data_ptr(), h=h.data_ptr(), y=y.data_ptr(), y_ld=C)
    need = lib.msl_gated_ffn_workspace_bytes(ctypes.byref(g), 0)
    ws = torch.empty(max(need, 1), device=_dev(), dtype=torch.uint8)
    rc = lib.msl_gated_ffn_fwd(ctypes.byref(g), ctypes.byref(io), ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    if C % 8:
        assert rc == _lib.MSL_OK and not bool(y.any())
    else:
        assert rc == _lib.MSL_ERR_INVALID and b"unaligned" in lib.msl_last_error()
        assert bool((y == 7).all()) and bool((h == 7).all())


def test_gated_ffn_gradient_against_differences():
    M, C, F = 6, 16, 24
    args = [t.detach() for t in _ffn_case(M, C, F, torch.float32, "gelu", True)]
    dy = _rand(9, M, C)
    for act in ("silu", "gelu"):
        leaves = [a.clone().requires_grad_() for a in args]
        grads = torch.autograd.grad(msl.gated_ffn(*leaves, activation=act), leaves, dy)

        def f(a):
            with torch.no_grad():
                return float((msl.gated_ffn(*a, activation=act).double() * dy.double()).sum())

        step = 2.0 ** -8
        for i, g in enumerate(grads):
            v = _rand(20 + i, *g.shape)
            hi = f([a + step * v if j == i else a for j, a in enumerate(args)])
            lo = f([a - step * v if j == i else a for j, a in enumerate(args)])
            scale = float(g.double().norm() * v.double().norm())
            assert abs((hi - lo) / (2 * step) - float((g.double() * v.double()).sum())) <= scale * 4e-3, (act, i)


def test_gated_ffn_on_another_stream_and_repeated():
    x, w_in, w_out, b_in, b_out = _ffn_case(500, 256, 512, torch.bfloat16, "silu", True)
    dy = _rand(9, 500, 256, dtype=torch.bfloat16)

    def once():
        y = msl.gated_ffn(x, w_in, w_out, b_in, b_out)
        return [y.detach(), *torch.autograd.grad(y, [x, w_in, w_out, b_in, b_out], dy)]

    want = once()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = once()
    s.synchronize()
    for a, b, c in zip(want, got, once()):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_gated_ffn_not_finite_rows_stay_rows():
    x, w_in, w_out, _, _ = (t.detach() if t is not None else None for t in _ffn_case(140, 64, 96, torch.bfloat16, "silu", False))
    clean = msl.gated_ffn(x, w_in, w_out)
    bad = x.clone()
    bad[3, 7], bad[139, 0] = float("nan"), float("inf")
    got = msl.gated_ffn(bad, w_in, w_out)
    assert torch.isnan(got[3]).all() and not torch.isfinite(got[139]).all()
    keep = [i for i in range(140) if i not in (3, 139)]
    assert torch.equal(got[keep], clean[keep])


# ---------------------------------------------------------------------------------- gradient norm and clipping


def _sumsq(ts):
    return math.fsum(float(t.double().square().sum()) for t in ts)


def _tensors(sizes, dtype, seed=0, std=0.1):
    kinds = DTYPES if dtype is None else [dtype]
    return [_rand(seed + i, n, dtype=kinds[i % len(kinds)], std=std) for i, n in enumerate(sizes)]


SIZES = [
    pytest.param([1], id="one-element"),
    pytest.param([0, 5, 0, 0, 3], id="empty-ones"),
    pytest.param([7, 8191, 8192, 8193, 1, 16385], id="chunk-edges"),
    pytest.param([1152, 4608, 300007, 16, 1152 * 40], id="block"),
    pytest.param([3] * 2000 + [100003], id="two-thousand"),
]


@pytest.mark.parametrize("dtype", [*DTYPES, None], ids=[*IDS, "mixed"])
@pytest.mark.parametrize("sizes", SIZES)
def test_grad_norm_and_clip(sizes, dtype):
    ts = _tensors(sizes, dtype)
    want = math.sqrt(_sumsq(ts))
    n = sum(sizes)
    tol = (8 + 6 * math.sqrt(min(n, 8192))) * EPS
    assert abs(float(msl.grad_norm(ts)) - want) <= tol * want
    both = math.sqrt(_sumsq(ts) + 2.25)
    assert abs(float(msl.grad_norm(ts, extra_sumsq=2.25)) - both) <= tol * both
    for limit in (want / 3, want * 2, 0.0):
        flat = {d: torch.full((sum(t.numel() for t in ts if t.dtype == d) + 1,), 9.0, dtype=d, device=_dev()) for d in DTYPES}
        at = {d: 1 for d in DTYPES}  # results start off any vector's boundary
        out = []
        for t in ts:
            out.append(flat[t.dtype][at[t.dtype]:at[t.dtype] + t.numel()])
            at[t.dtype] += t.numel()
        norm = msl.clip_grad_norm_(ts, limit, out=out)
        assert abs(float(norm) - want) <= tol * want
        f = min(1.0, limit / (want + 1e-6))
        for t, o in zip(ts, out):
            assert torch.all((o.double() - t.double() * f).abs() <= (_half(t.dtype) + tol + 4 * EPS) * t.double().abs() * f + 1e-38)
        assert all(float(v[0]) == 9.0 for v in flat.values())
        same = [t.clone() for t in ts]
        again = msl.clip_grad_norm_(same, limit)
        assert torch.equal(again, norm) and all(torch.equal(a, b) for a, b in zip(same, out))


def test_clip_alignments():
    """Sources and results at every offset from a 16-byte boundary."""
    for dtype, per in ((torch.bfloat16, 8), (torch.float32, 4)):
        base = _rand(1, 9000 + per, dtype=dtype)
        for i in range(per):
            src = base[i:i + 8500 + i]
            want = math.sqrt(_sumsq([src]))
            for j in range(per):
                dst = torch.zeros(9000 + per, dtype=dtype, device=_dev())
                norm = msl.clip_grad_norm_([src], 1.0, out=[dst[j:j + 8500 + i]])
                assert abs(float(norm) - want) <= 1e-6 * want
                ref = src.double() / (want + 1e-6)
                assert torch.all((dst[j:j + 8500 + i].double() - ref).abs() <= (_half(dtype) + 1e-6) * ref.abs())
                assert torch.count_nonzero(dst[:j]) == 0 and torch.count_nonzero(dst[j + 8500 + i:]) == 0


def test_clip_parameters_and_values_that_are_not_finite():
    ps = [torch.nn.Parameter(torch.zeros(n, device=_dev())) for n in (40, 50, 60)]
    ps[0].grad, ps[2].grad = _rand(1, 40), _rand(2, 60)
    want = torch.nn.utils.get_total_norm([ps[0].grad, ps[2].grad])
    before = ps[2].grad.clone()
    norm = msl.clip_grad_norm_(ps, 0.5)
    assert torch.allclose(norm, want) and torch.allclose(ps[2].grad, before * (0.5 / (want + 1e-6)), rtol=1e-5)
    g = _rand(3, 1000)
    g[17] = float("inf")
    t = g.clone()
    assert math.isinf(float(msl.clip_grad_norm_([t], 1.0)))
    assert math.isnan(float(t[17])) and torch.count_nonzero(t[:17]) == 0
    g[17] = float("nan")
    t = g.clone()
    assert math.isnan(float(msl.clip_grad_norm_([t], 1.0))) and torch.isnan(t).all()


def test_norm_beyond_2_31_elements_and_on_another_stream():
    t = torch.full((2 ** 31 + 5,), 0.5, dtype=torch.bfloat16, device=_dev())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        norm = msl.grad_norm([t])
    s.synchronize()
    want = 0.5 * math.sqrt(2 ** 31 + 5)
    assert abs(float(norm) - want) <= 4 * EPS * want


# ------------------------------------------------------------------------------------------ with threads and autograd

@pytest.mark.parametrize("C", [64, 61])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_first_call_of_a_thread(dtype, C):
    """A thread whose first contact with the GPU is a call of the gated block, all its memory from torch's cache (as
    autograd's thread may be), gets the same results."""
    M, F = 300, 128
    x, w_in, w_out, b_in, b_out = (t.detach() for t in _ffn_case(M, C, F, dtype, "silu", True))
    dy = _rand(9, M, C, dtype=dtype)
    y, h, kept = ops.gated_ffn_fwd(x, w_in, w_out, b_in, b_out, keep=True)

    def forward():
        return ops.gated_ffn_fwd(x, w_in, w_out, b_in, b_out, keep=True)

    def backward():
        return ops.gated_ffn_bwd(x, w_in, w_out, h, kept, dy, b_in, b_out)

    for call in (forward, backward):
        want = [t.clone() for t in call()]
        torch.cuda.synchronize()
        got, errors = [], []

        def run():
            try:
                got.extend(call())
            except Exception as e:  # raised again where pytest sees it
                errors.append(e)

        thread = threading.Thread(target=run)
        thread.start()
        thread.join()
        assert not errors, errors
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)



def test_second_derivatives_are_refused():
    """The backward passes are kernels without a derivative of their own: asking for one is an error, not a term that
    is silently missing."""
    x = _rand(1, 1, 6, 16).requires_grad_()
    table = msl.rotary_table((1, 2, 3), (2, 2, 4), device=_dev())
    w = torch.ones(8, device=_dev(), requires_grad=True)
    w_in, w_out = _rand(2, 16, 16).requires_grad_(), _rand(3, 16, 8).requires_grad_()
    for y in (msl.rope3d(x, table, video_shape=(1, 2, 3), axes=(2, 2, 4), heads=2),
              msl.qk_norm_rope(x, x, w, w, heads=2)[0], msl.gated_ffn(x, w_in, w_out)):
        dx, = torch.autograd.grad((y * y).sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            (dx * dx).sum().backward()


def test_clipping_counts_as_a_write():
    """A tensor that autograd has saved and the clipping then scales is noticed by autograd."""
    a = torch.ones(64, device=_dev(), requires_grad=True)
    g = torch.full((64,), 2.0, device=_dev())
    y = (a * g).sum()
    msl.clip_grad_norm_([g], 1.0)
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward()
    b, c = torch.ones(64, device=_dev()), torch.empty(64, device=_dev())
    y = (a * b).sum() + (a * c).sum()
    msl.clip_grad_norm_([b], 1.0, out=[c])
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_calls_in_a_cuda_graph(dtype):
    """A step over all operators, forward and backward, captured once and replayed on other inputs, equals the calls."""
    M, C, F, vs, axes = 60, 64, 96, (3, 4, 5), (4, 4, 8)
    x = _rand(1, 1, M, C, dtype=dtype).requires_grad_()
    w_in, w_out = _rand(2, 2 * F, C, dtype=dtype, std=0.1).requires_grad_(), _rand(3, C, F, dtype=dtype, std=0.1).requires_grad_()
    weight = _rand(4, 16).add_(2).requires_grad_()
    table = msl.rotary_table(vs, axes, device=_dev())

    def step():
        kw = dict(video_shape=vs, axes=axes, heads=4)
        q, k = msl.qk_norm_rope(x, msl.rope3d(x, table, **kw), weight, weight, table, **kw)
        grads = torch.autograd.grad(msl.gated_ffn(q + k, w_in, w_out), (x, w_in, w_out, weight), torch.ones_like(x))
        grads = [g.clone() for g in grads]
        return [msl.clip_grad_norm_(grads, 0.5), *grads, msl.gated_ffn(x[:, :1].detach(), w_in.detach(), w_out.detach())]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (5, 6):
        with torch.no_grad():
            x.copy_(_rand(seed, 1, M, C, dtype=dtype))
        graph.replay()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)
