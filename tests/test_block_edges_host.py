"""The operators around the attention without a GPU: what the module keeps between calls, host-side buffers, and refusals
that come before any CUDA call."""

import ctypes

import pytest
import torch

import megaslide_b200 as msl
from megaslide_b200 import _lib, ops


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
