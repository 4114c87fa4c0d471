"""The operators around the attention without a GPU: the table of positions, the refusals of their arguments (in
Python and at the C entry points, before any CUDA call), and the structs' layouts."""

import ctypes
import math
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

import megaslide_b200 as msl
from megaslide_b200 import _lib, ops, rotary

HEADER = Path(__file__).resolve().parent.parent / "include" / "megaslide_b200.h"


def test_rotary_table_values():
    t = msl.rotary_table((3, 2, 4), (4, 2, 6), theta=50.0)
    assert t.shape == (3 * 2 + 2 * 1 + 4 * 3, 2) and t.dtype == torch.float32
    for p in range(3):
        for i in range(2):
            a = p * 50.0 ** (-2 * i / 4)
            assert abs(float(t[p * 2 + i, 0]) - math.cos(a)) < 1e-7 and abs(float(t[p * 2 + i, 1]) - math.sin(a)) < 1e-7
    a = 3 * 50.0 ** (-4 / 6)
    assert abs(float(t[6 + 2 + 3 * 3 + 2, 1]) - math.sin(a)) < 1e-7
    half = msl.rotary_table((2, 1, 1), (2, 0, 0), positions=[torch.tensor([0.0, 0.5]), torch.zeros(1), torch.zeros(1)])
    assert half.shape == (2, 2) and abs(float(half[1, 0]) - math.cos(0.5)) < 1e-7
    with pytest.raises(ValueError, match="even"):
        msl.rotary_table((2, 2, 2), (3, 2, 2))
    with pytest.raises(ValueError, match="positions"):
        msl.rotary_table((2, 2, 2), (2, 2, 2), positions=[torch.zeros(3), torch.zeros(2), torch.zeros(2)])


def test_cpu_tensors_are_refused():
    x = torch.zeros(1, 8, 16)
    t = msl.rotary_table((2, 2, 2), (4, 4, 4))
    with pytest.raises(RuntimeError, match="CUDA"):
        msl.rope3d(x, t, video_shape=(2, 2, 2), axes=(4, 4, 4), heads=1)
    with pytest.raises(RuntimeError, match="CUDA"):
        msl.qk_norm_rope(x, x, None, None, heads=1)
    with pytest.raises(RuntimeError, match="CUDA"):
        msl.gated_ffn(x, torch.zeros(8, 16), torch.zeros(16, 4))
    with pytest.raises(RuntimeError, match="CUDA"):
        msl.grad_norm([x])


def test_python_refusals():
    x = torch.zeros(1, 8, 16)
    with pytest.raises(ValueError, match="heads"):
        msl.rope3d(x, x, video_shape=(2, 2, 2), axes=(4, 4, 4), heads=3)
    with pytest.raises(ValueError, match="heads"):
        msl.rope3d(x[0], x, video_shape=(2, 2, 2), axes=(4, 4, 4), heads=1)
    with pytest.raises(ValueError, match="activation"):
        msl.GatedMLP(8, 16, activation="tanh")
    with pytest.raises(ValueError, match="max_norm"):
        msl.clip_grad_norm_([x], -1.0)
    with pytest.raises(ValueError, match="extra_sumsq"):
        msl.grad_norm([x], extra_sumsq=float("nan"))
    assert float(msl.grad_norm([], extra_sumsq=9.0)) == 3.0
    shape = ops.RotaryShape(1, 8, (2, 2, 2), (4, 4, 4), 16)
    dev = torch.device("cpu")
    with pytest.raises(ValueError, match="table"):
        ops._check_positions(shape, torch.zeros(5, 2), None, dev)
    table = msl.rotary_table((2, 2, 2), (4, 4, 4))
    with pytest.raises(ValueError, match="index"):
        ops._check_positions(shape, table, torch.zeros(8, 3), dev)
    with pytest.raises(ValueError, match="names 5 tokens"):
        ops._check_positions(shape, table, torch.zeros(5, 3, dtype=torch.int32), dev)
    assert ops._check_positions(shape, table, torch.zeros(8, 3, dtype=torch.int32), dev) == 8


def test_gated_mlp_parameters():
    m = msl.GatedMLP(8, 20)
    assert {k: tuple(v.shape) for k, v in m.state_dict().items()} == {
        "fc1.weight": (40, 8), "fc1.bias": (40,), "fc2.weight": (8, 20), "fc2.bias": (8,)}


def test_row_views():
    """Tokens whose rows lie at one stride are used as they are, others are copied."""
    x = torch.zeros(2, 3, 10)
    assert rotary._as_rows(x) is x and ops._ld(x, "x") == 10
    cols = torch.zeros(2, 3, 30)[..., 10:20]
    assert rotary._as_rows(cols) is cols and ops._ld(cols, "x") == 30
    swapped = torch.zeros(3, 2, 10).transpose(0, 1)
    assert rotary._as_rows(swapped).is_contiguous()
    with pytest.raises(ValueError, match="one stride"):
        ops._ld(swapped, "x")
    spread = torch.zeros(2, 1, 10).expand(2, 4, 10)  # one row for every token of a sample
    assert rotary._as_rows(spread).is_contiguous() and rotary._as_rows(torch.zeros(1, 1, 10).expand(1, 4, 10)).stride(1) == 10
    assert ops._ld(rotary._as_rows(torch.zeros(1, 0, 10)), "x") == 10


def _err():
    return _lib.load().msl_last_error().decode()


def _rot(**kw):
    base = dict(rows=8, tokens=8, frames=2, height=2, width=2, frame0=0, axis_t=4, axis_h=4, axis_w=4, head_dim=16, interleaved=1, dtype=0)
    base.update(kw)
    return _lib.RotaryGeometry(**base)


@pytest.mark.parametrize("kw,text", [
    (dict(head_dim=15), "even"), (dict(axis_t=3), "even"), (dict(axis_t=10), "more than head_dim"), (dict(rows=-1), "rows"),
    (dict(frames=0), "frames"), (dict(dtype=5), "dtype"), (dict(frame0=-1), "frame0"), (dict(frame0=1), "outside the table"),
    (dict(tokens=7), "whole frames"),
])
def test_rotary_entry_refuses(kw, text):
    g = _rot(**kw)
    assert _lib.load().msl_rope3d(ctypes.byref(g), 1, 16, 16, 16, None, 0, 0, 16, 16, None, None) == _lib.MSL_ERR_INVALID
    assert text in _err()


def test_rotary_entry_refuses_operands():
    lib = _lib.load()
    g = _rot()
    assert lib.msl_rope3d(None, 1, 16, 16, 16, None, 0, 0, 16, 16, None, None) == _lib.MSL_ERR_INVALID
    assert lib.msl_rope3d(ctypes.byref(g), 1, 16, 15, 16, None, 0, 0, 16, 16, None, None) == _lib.MSL_ERR_INVALID and "stride" in _err()
    assert lib.msl_rope3d(ctypes.byref(g), 1, 16, 16, None, None, 0, 0, 16, 16, None, None) == _lib.MSL_ERR_INVALID and "table" in _err()
    assert lib.msl_rope3d(ctypes.byref(_rot(head_dim=258)), 1, 16, 258, 16, None, 0, 0, 16, 258, None, None) == _lib.MSL_ERR_UNSUPPORTED
    io = _lib.QkNormIO(q=16, q_ld=16, q_out=16, q_out_ld=16, heads=1, kv_heads=1, eps=1e-6)
    assert lib.msl_qk_norm_rope_fwd(ctypes.byref(g), ctypes.byref(io), None) == _lib.MSL_ERR_INVALID and "k is required" in _err()
    io.eps = -1.0
    assert lib.msl_qk_norm_rope_fwd(ctypes.byref(g), ctypes.byref(io), None) == _lib.MSL_ERR_INVALID and "eps" in _err()
    io.eps, io.heads = 0.0, 0
    assert lib.msl_qk_norm_rope_fwd(ctypes.byref(g), ctypes.byref(io), None) == _lib.MSL_ERR_INVALID and "heads" in _err()
    assert lib.msl_qk_norm_rope_fwd(ctypes.byref(g), None, None) == _lib.MSL_ERR_INVALID
    io = _lib.QkNormIO(q=16, q_ld=16, heads=1, kv_heads=0, eps=1e-6, dq_out=16, dq_out_ld=16, dq=16, dq_ld=16, dq_weight=16)
    assert lib.msl_qk_norm_rope_bwd_workspace_bytes(ctypes.byref(g), ctypes.byref(io)) > 0
    assert lib.msl_qk_norm_rope_bwd(ctypes.byref(g), ctypes.byref(io), None, 0, None) == _lib.MSL_ERR_WORKSPACE


@pytest.mark.parametrize("kw,code,text", [
    (dict(rows=-1), _lib.MSL_ERR_INVALID, "rows"), (dict(dim=0), _lib.MSL_ERR_INVALID, "dim"), (dict(dtype=3), _lib.MSL_ERR_INVALID, "dtype"),
    (dict(activation=7), _lib.MSL_ERR_INVALID, "activation"), (dict(hidden=1 << 21), _lib.MSL_ERR_UNSUPPORTED, "2^20"),
    (dict(rows=2**31 - 255), _lib.MSL_ERR_UNSUPPORTED, "2^31"),
])
def test_ffn_entry_refuses(kw, code, text):
    g = _lib.FfnGeometry(**{**dict(rows=4, dim=8, hidden=16, dtype=0, activation=0), **kw})
    io = _lib.FfnIO(x=16, x_ld=8, w_in=16, w_out=16, h=16, y=16, y_ld=8)
    assert _lib.load().msl_gated_ffn_fwd(ctypes.byref(g), ctypes.byref(io), None, 0, None) == code
    assert text in _err()


def test_ffn_entry_refuses_operands():
    lib = _lib.load()
    g = _lib.FfnGeometry(4, 8, 16, 0, 0)
    io = _lib.FfnIO(x=16, x_ld=7, w_in=16, w_out=16, h=16, y=16, y_ld=8)
    assert lib.msl_gated_ffn_fwd(ctypes.byref(g), ctypes.byref(io), None, 0, None) == _lib.MSL_ERR_INVALID and "stride" in _err()
    io = _lib.FfnIO(x=16, x_ld=8, w_out=16, h=16, y=16, y_ld=8)
    assert lib.msl_gated_ffn_fwd(ctypes.byref(g), ctypes.byref(io), None, 0, None) == _lib.MSL_ERR_INVALID and "w_in" in _err()
    io = _lib.FfnIO(x=16, x_ld=8, w_in=16, w_out=16, h=16, dx=16, dx_ld=8, dy=16, dy_ld=8, dgu=16)
    assert lib.msl_gated_ffn_bwd(ctypes.byref(g), ctypes.byref(io), None, 0, None) == _lib.MSL_ERR_INVALID and "gu" in _err()
    io = _lib.FfnIO(h=16, dw_out=16, dy=16, dy_ld=8, db_out=16)
    assert lib.msl_gated_ffn_bwd(ctypes.byref(g), ctypes.byref(io), None, 0, None) == _lib.MSL_ERR_WORKSPACE


def test_grad_norm_entry_refuses():
    lib = _lib.load()
    one = (ctypes.c_int64 * 1)(10)
    f32, bad = (ctypes.c_int32 * 1)(0), (ctypes.c_int32 * 1)(9)
    ptr, odd = (ctypes.c_void_p * 1)(16), (ctypes.c_void_p * 1)(18)

    def norm(src=ptr, numel=one, dt=f32, count=1, extra=0.0, out=16, ws=16, n=1 << 20):
        return lib.msl_grad_norm(src, numel, dt, count, extra, out, ws, n, None)

    assert norm(count=-1) == _lib.MSL_ERR_INVALID
    assert norm(dt=bad) == _lib.MSL_ERR_INVALID and "dtype" in _err()
    assert norm(src=odd) == _lib.MSL_ERR_INVALID and "aligned" in _err()
    assert norm(src=(ctypes.c_void_p * 1)(None)) == _lib.MSL_ERR_INVALID and "NULL" in _err()
    assert norm(numel=(ctypes.c_int64 * 1)(-1)) == _lib.MSL_ERR_INVALID
    assert norm(extra=-1.0) == _lib.MSL_ERR_INVALID and "extra" in _err()
    assert norm(out=None) == _lib.MSL_ERR_INVALID
    assert norm(n=0) == _lib.MSL_ERR_WORKSPACE
    assert lib.msl_grad_clip(ptr, ptr, one, f32, 1, 0.0, -1.0, 16, 16, 1 << 20, None) == _lib.MSL_ERR_INVALID and "max_norm" in _err()


STRUCTS = {
    "msl_rotary_geometry": _lib.RotaryGeometry,
    "msl_qk_norm_io": _lib.QkNormIO,
    "msl_ffn_geometry": _lib.FfnGeometry,
    "msl_ffn_io": _lib.FfnIO,
}


def test_struct_layouts_match_header(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void) {"]
    for cname, py in STRUCTS.items():
        lines.append(f'printf("{cname} size %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in py._fields_]
    lines.append("return 0; }")
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines))
    subprocess.run([cc, str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines():
        s, f, v = line.split()
        assert int(v) == (ctypes.sizeof(STRUCTS[s]) if f == "size" else getattr(STRUCTS[s], f).offset), (s, f)
