"""The operators around the attention without a GPU: what the module keeps between calls, host-side buffers, and refusals
that come before any CUDA call."""

import ctypes
from contextlib import nullcontext

import pytest
import torch

import megaslide_b200 as msl
from megaslide_b200 import _lib, clip, ops
from oracle import sampled


def _module(**kw):
    return msl.DeformableSlideAttention3D(64, 4, (3, 3, 3), **{**dict(qk_norm=True, rotary_axes=(4, 6, 6)), **kw})


def test_table_made_in_inference_mode_serves_training():
    m, cpu = _module(), torch.device("cpu")
    with torch.inference_mode():
        first = m._table((2, 3, 4), cpu)
    t = m._table((2, 3, 4), cpu)
    assert t is first and not t.is_inference()
    assert torch.equal(t, msl.rotary_table((2, 3, 4), (4, 6, 6)))


def test_table_follows_the_module_attributes():
    m, cpu = _module(), torch.device("cpu")
    before = m._table((2, 3, 4), cpu)
    m.rotary_theta = 5.0
    assert torch.equal(m._table((2, 3, 4), cpu), msl.rotary_table((2, 3, 4), (4, 6, 6), 5.0))
    m.rotary_axes = (2, 4, 4)
    assert torch.equal(m._table((2, 3, 4), cpu), msl.rotary_table((2, 3, 4), (2, 4, 4), 5.0))
    m.rotary_axes, m.rotary_theta = (4, 6, 6), 10000.0
    assert torch.equal(m._table((2, 3, 4), cpu), before)


def test_table_under_another_default_device():
    """torch.set_default_device does not reach the table's own arithmetic."""
    half = [torch.tensor([0.0, 0.5]), torch.zeros(1), torch.zeros(1)]
    want = msl.rotary_table((2, 1, 1), (2, 0, 0), positions=half), msl.rotary_table((2, 3, 4), (4, 6, 6))
    with torch.device("meta"):
        got = msl.rotary_table((2, 1, 1), (2, 0, 0), positions=half), msl.rotary_table((2, 3, 4), (4, 6, 6))
    for a, b in zip(got, want):
        assert a.device.type == "cpu" and torch.equal(a, b)


def test_table_that_requires_a_gradient_is_refused():
    """The operators give no gradient of the table: a learned one must not be left without, silently."""
    x = torch.zeros(1, 24, 64)
    kw = dict(video_shape=(2, 3, 4), axes=(4, 6, 6), heads=4)
    table = msl.rotary_table((2, 3, 4), (4, 6, 6)).requires_grad_()
    for call in (lambda t: msl.rope3d(x, t, **kw), lambda t: msl.qk_norm_rope(x, x, None, None, t, **kw)):
        with pytest.raises(ValueError, match="gradient"):
            call(table)
        with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
            call(table)
        with pytest.raises(RuntimeError, match="CUDA"):
            call(table.detach())


@pytest.mark.parametrize("src,dst,numel,bf16,text", [
    ([4096, 4096], [4096, 4096], [10, 10], 0, "result of tensor"),  # the same tensor twice, in place
    ([4096, 8192], [4096, 4100], [10, 10], 0, "result of tensor"),
    ([4096, 8192], [4132, 8192], [10, 10], 0, "source of tensor 0"),  # its own source, shifted
    ([4096, 4136], [4136, 4096], [10, 10], 0, "source of tensor"),  # exchanged
    ([4096, 4116], [4096, 8192], [10, 10], 1, None),  # neighbours in bf16, one in place
    ([4096, 4136], [4096, 4136], [10, 10], 0, None),
    ([4096, 4096, 4100], [8192, 9000, 16384], [10, 0, 10], 0, None),  # sources may share, a tensor without elements is nowhere
    ([4096, 4136], [4056, 4176], [10, 10], 0, None),  # a result on either side of the sources
], ids=str)
def test_clip_entry_refuses_overlapping_results(src, dst, numel, bf16, text):
    """Checked before any launch: too small a workspace stops the calls that pass."""
    n = len(src)
    vp, i64, i32 = ctypes.c_void_p * n, ctypes.c_int64 * n, ctypes.c_int32 * n
    lib = _lib.load()
    rc = lib.msl_grad_clip(vp(*src), vp(*dst), i64(*numel), i32(*[bf16] * n), n, 0.0, 1.0, 16, 16, 0, None)
    if text is None:
        assert rc == _lib.MSL_ERR_WORKSPACE
    else:
        assert rc == _lib.MSL_ERR_INVALID and text in lib.msl_last_error().decode()
    assert lib.msl_grad_norm(vp(*src), i64(*numel), i32(*[bf16] * n), n, 0.0, 16, 16, 0, None) == _lib.MSL_ERR_WORKSPACE


def test_dense_in_any_order():
    t = torch.zeros(2, 3, 4, 5)
    for d in (t, t.permute(2, 0, 3, 1), t.transpose(0, 3), t[:1], t[:, :, :1, :1].contiguous().transpose(1, 2), torch.zeros(()), torch.zeros(3, 0).t()):
        assert ops._dense(d)
    for d in (t[:, 1:], t[..., ::2], t[:1, :, :, :1], torch.zeros(1, 5).expand(3, 5), torch.zeros(20).as_strided((4, 5), (3, 1))):
        assert not ops._dense(d)


@pytest.fixture
def launches(monkeypatch):
    """The functions of ops on CPU tensors, up to the point of the launch: what they would have launched."""
    seen = []
    monkeypatch.setattr(ops, "_need_cuda", lambda *ts: None)
    monkeypatch.setattr(ops, "_on", lambda dev: nullcontext())
    monkeypatch.setattr(ops, "_call", lambda name, dev, fn: seen.append(name) or 0)
    monkeypatch.setattr(ops, "_flag", lambda dev, status: None)
    return seen


def test_rotary_functions_refuse_operands_beyond_the_geometry(launches):
    sh, table = ops.RotaryShape(2, 24, (2, 3, 4), (4, 6, 6), 16), msl.rotary_table((2, 3, 4), (4, 6, 6))
    x, few, narrow, half = torch.zeros(48, 64), torch.zeros(47, 64), torch.zeros(48, 63), torch.zeros(48, 64, dtype=torch.bfloat16)
    wide = torch.zeros(48, 200)[:, :64]
    w = torch.ones(16)

    def forward(q=x, k=x, **kw):
        return ops.qk_norm_rope_fwd(sh, 4, 4, q, k, w, w, 1e-6, table, **kw)

    def backward(q=x, k=x, dq_out=x, dk_out=x, **kw):
        return ops.qk_norm_rope_bwd(sh, 4, 4, q, k, w, w, dq_out, dk_out, 1e-6, table, **kw)

    for good in (lambda: ops.rope3d(sh, 4, x, table), lambda: ops.rope3d(sh, 4, wide, table, out=wide), lambda: ops.rope3d(sh, 3, x, table),
                 forward, lambda: forward(wide, wide, q_out=wide, k_out=x), backward, lambda: backward(dq=wide, dk=wide),
                 lambda: forward(x.view(2, 24, 64), x.view(2, 24, 64))):
        good()
    assert len(launches) == 8
    for bad, error in ((few, ValueError), (narrow, ValueError), (half, TypeError)):
        calls = [lambda: ops.rope3d(sh, 4, x, table, out=bad)]
        calls += [lambda nm=nm: forward(**{nm: bad}) for nm in ("k", "q_out", "k_out")]
        calls += [lambda nm=nm: backward(**{nm: bad}) for nm in ("k", "dq_out", "dk_out", "dq", "dk")]
        if bad is not half:
            calls += [lambda: ops.rope3d(sh, 4, bad, table), lambda: forward(q=bad, k=bad)]
        for call in calls:
            with pytest.raises(error):
                call()
    with pytest.raises(ValueError):
        ops.rope3d(sh, 5, x, table)
    assert len(launches) == 8


def test_gated_backward_refuses_operands_beyond_the_geometry(launches):
    M, C, F = 6, 16, 24
    x, w_in, w_out, dy = torch.zeros(M, C), torch.zeros(2 * F, C), torch.zeros(C, F), torch.zeros(M, C)
    h, kept = torch.zeros(M, F), torch.zeros(M, 2 * F)

    def call(**kw):
        a = {**dict(h=h, kept=kept, dy=dy), **kw}
        return ops.gated_ffn_bwd(x, w_in, w_out, a["h"], a["kept"], a["dy"])

    call()
    call(dy=torch.zeros(M, 40)[:, :C])
    assert len(launches) == 2
    for nm, t in (("h", h), ("kept", kept), ("dy", dy)):
        for bad in (t[:-1], t[:, :-1].contiguous(), torch.zeros(M, t.shape[1] + 1)):
            with pytest.raises(ValueError, match=nm):
                call(**{nm: bad})
        with pytest.raises(TypeError, match=nm):
            call(**{nm: t.bfloat16()})
    with pytest.raises(ValueError, match="h must"):
        call(h=torch.zeros(M, F + 8)[:, :F])
    assert len(launches) == 2


def test_status_word_of_a_caller_is_checked():
    dev = torch.device("cpu")
    assert ops._flag(dev, torch.zeros(1, dtype=torch.int32)) != 0
    for bad in (torch.zeros(1), torch.zeros(0, dtype=torch.int32), torch.zeros(1, dtype=torch.int32, device="meta")):
        with pytest.raises(ValueError, match="status"):
            ops._flag(dev, bad)


def test_flag_loses_no_bit_that_is_set_while_it_is_read(monkeypatch):
    """A kernel that is still running reports between the host's look at the word and its clearing it."""
    flag = object.__new__(ops.HostFlag)
    flag.index = None

    class Word:
        value, running = 0, False

        def __getitem__(self, i):
            v, self.value = self.value, self.value | (_lib.MSL_STATUS_TIMEOUT if self.running else 0)
            self.running = False
            return v

        def __setitem__(self, i, v):
            self.value = v

    flag._view = word = Word()
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device=None: setattr(word, "running", False))
    flag.poll()
    word.value, word.running = _lib.MSL_STATUS_ROTARY_INDEX, True
    texts = []
    for _ in range(2):
        try:
            flag.poll()
        except msl.MslError as e:
            texts.append(str(e))
    assert "outside its axis" in " ".join(texts) and "did not complete" in " ".join(texts)
    assert word.value == 0
    flag.poll()


@pytest.mark.parametrize("dim,hidden,text", [((1 << 21) + 1, 8, "dim is over 2^21"), (8, (1 << 20) + 1, "hidden is over 2^20")])
def test_ffn_entry_names_the_limit_it_checks(dim, hidden, text):
    lib = _lib.load()
    g = _lib.FfnGeometry(4, dim, hidden, 0, 0)
    io = _lib.FfnIO(x=16, x_ld=dim, w_in=16, w_out=16, h=16, y=16, y_ld=dim)
    assert lib.msl_gated_ffn_fwd(ctypes.byref(g), ctypes.byref(io), None, 0, None) == _lib.MSL_ERR_UNSUPPORTED
    assert lib.msl_last_error().decode().endswith(text)


@pytest.mark.parametrize("kw", [dict(rotary_axes=None), dict(qk_norm=False)], ids=["norm", "rotary"])
def test_sampled_check_refuses_options_that_the_oracle_does_not_restate(kw):
    """It would compare the attention of normalised, turned q and k with that of the projections."""
    with pytest.raises(ValueError, match="qk_norm and rotary_axes"):
        sampled.check(_module(**kw), {}, (2, 3, 4), batch=1, dtype=torch.float32)


def test_leaves_that_require_gradients_stand_for_them():
    """As torch's clip_grad_norm_ has it: a leaf is a parameter whether or not it is a Parameter, and it is not the weights
    that are scaled."""
    plain, leaf, bare = torch.ones(3), torch.ones(4, requires_grad=True), torch.ones(5, requires_grad=True)
    param, frozen = torch.nn.Parameter(torch.ones(6)), torch.nn.Parameter(torch.ones(7), requires_grad=False)
    leaf.grad, param.grad = torch.zeros(4), torch.zeros(6)
    result = leaf * 2  # no leaf: itself
    got = clip._list([plain, leaf, None, bare, param, frozen, result])
    for a, b in zip(got, (plain, leaf.grad, param.grad, result), strict=True):
        assert a is b
    assert clip._list(leaf)[0] is leaf.grad and clip._list(bare) == []


def test_ffn_entry_wants_the_low_bytes_beside_bf16_factors():
    lib = _lib.load()
    g = _lib.FfnGeometry(4, 8, 16, _lib.MSL_DTYPE_BF16, 0)
    io = _lib.FfnIO(x=16, x_ld=8, w_in=16, w_out=16, h=16, y=16, y_ld=8, kept=16)
    assert lib.msl_gated_ffn_fwd(ctypes.byref(g), ctypes.byref(io), None, 0, None) == _lib.MSL_ERR_INVALID
    assert "kept_low" in lib.msl_last_error().decode()
    io = _lib.FfnIO(x=16, x_ld=8, w_in=16, w_out=16, h=16, kept=16, dx=16, dx_ld=8, dy=16, dy_ld=8, dgu=16)
    assert lib.msl_gated_ffn_bwd(ctypes.byref(g), ctypes.byref(io), None, 0, None) == _lib.MSL_ERR_INVALID
    assert "kept_low" in lib.msl_last_error().decode()
    assert ops._kept_bytes(3, 17) == (204, 204 + 2 * 3 * 32)
