"""Torch-tensor wrappers over the C ABI (include/megaslide_b200.h).

Each function takes CUDA tensors, checks shapes / dtypes / devices on the host, passes raw
pointers, row strides and the current CUDA stream to libmegaslide_b200.so, and raises
``MslError`` (a RuntimeError) on any error code.  Nothing here computes on the CPU.
"""

from __future__ import annotations

import ctypes
import math
from contextlib import contextmanager, nullcontext
from dataclasses import dataclass
from operator import attrgetter
from typing import List, Optional, Tuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import DsaBwdIO, DsaFwdIO, DsaGeometry, DwconvGeometry

_DTYPES = {torch.float32: _lib.MSL_DTYPE_F32, torch.bfloat16: _lib.MSL_DTYPE_BF16}


def dtype_code(dt: torch.dtype) -> int:
    try:
        return _DTYPES[dt]
    except KeyError:
        raise TypeError(f"megaslide_b200 supports float32 and bfloat16 activations, got {dt}") from None


def takes_derivatives(*ts) -> bool:
    """Whether a call goes through its autograd function: an operand requires a gradient, or a level of forward mode is
    open (a tangent asks for no gradient; the function refuses it, where the kernel alone would lose it)."""
    if forward_ad._current_level >= 0:
        return True
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return True
    return False


def once_only(backward):
    """torch's once_differentiable, an error where a second derivative is taken, at its cost (a few microseconds) only
    where a graph of the backward is recorded."""
    guarded = once_differentiable(backward)

    def run(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return run


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _rows(t: torch.Tensor, name: str) -> int:
    """Row stride (elements) of a [rows, cols] matrix view with unit column stride."""
    if t.dim() != 2 or (t.stride(1) != 1 and t.size(1) > 1):
        raise ValueError(f"{name} must be a row-major 2-D view, got shape {tuple(t.shape)} strides {t.stride()}")
    return t.stride(0) if t.size(0) > 1 else max(t.stride(0), t.size(1))


def _stream(dev: torch.device) -> int:
    return torch.cuda.current_stream(dev).cuda_stream


_TIMER: Optional[List] = None


@contextmanager
def kernel_timer():
    """Records a (entry point name, start event, end event) triple around every C-ABI call made
    inside the block, on the stream the kernels are launched on.  Used by bench.py to time the
    kernels live (synchronise before reading the events)."""
    global _TIMER
    prev, _TIMER = _TIMER, []
    try:
        yield _TIMER
    finally:
        _TIMER = prev


def _call(name: str, dev: torch.device, fn):
    if _TIMER is None:
        return fn()
    s = torch.cuda.Event(enable_timing=True)
    e = torch.cuda.Event(enable_timing=True)
    stream = torch.cuda.current_stream(dev)
    s.record(stream)
    rc = fn()
    e.record(stream)
    _TIMER.append((name, s, e))
    return rc


class StatusWord:
    """The per-device status word the attention kernels OR their MSL_STATUS_* bits into (device int32),
    read back without stalling the host: after every call an asynchronous copy into pinned memory is
    enqueued with an event, and the next call (poll) reads that copy once its event has completed.  A
    halo miss or a timed-out TMA wait (results not valid) raises MslError there, at most one call late;
    check() reads the word synchronously.  MSL_STATUS_TC_RANGE is informational (the kernels computed
    such tiles with the CUDA-core gather)."""

    BAD = _lib.MSL_STATUS_HALO_MISS | _lib.MSL_STATUS_TIMEOUT

    def __init__(self, device: torch.device):
        with torch.inference_mode(False):  # both outlive the call that makes them, which may be in inference mode
            self.word = torch.zeros(1, dtype=torch.int32, device=device)
            self.host = torch.zeros(1, dtype=torch.int32, device="cpu").pin_memory()
        self.event: Optional[torch.cuda.Event] = None
        self.seen = 0  # every bit observed so far (TC_RANGE included)

    def post(self) -> None:
        with torch.cuda.device(self.word.device):
            self.host.copy_(self.word, non_blocking=True)
            self.event = torch.cuda.Event()
            self.event.record()

    def _raise_if_bad(self, v: int) -> None:
        self.seen |= v
        if v & self.BAD:
            self.word.zero_()
            what = []
            if v & _lib.MSL_STATUS_HALO_MISS:
                what.append("a sample corner fell outside the K/V frames the call was given (halo miss)")
            if v & _lib.MSL_STATUS_TIMEOUT:
                what.append("a tensor-core CTA's TMA copies did not complete within a second")
            raise _lib.MslError("msl_dsa_attn", _lib.MSL_ERR_CUDA,
                                "a previous attention call produced invalid results: " + "; ".join(what))

    def poll(self) -> None:
        if self.event is not None and self.event.query():
            self.event = None
            self._raise_if_bad(int(self.host[0]))

    def check(self) -> int:
        """Synchronous: raises on a bad bit (and clears the word), else returns the word's bits
        (MSL_STATUS_TC_RANGE once a tile took the CUDA-core fallback)."""
        self.event = None
        v = int(self.word.item())
        self._raise_if_bad(v)
        return v


_STATUS: dict = {}


def status_word(device: torch.device) -> StatusWord:
    """The process-wide StatusWord of a CUDA device."""
    key = torch.device(device).index if torch.device(device).index is not None else torch.cuda.current_device()
    sw = _STATUS.get(key)
    if sw is None:
        sw = _STATUS[key] = StatusWord(torch.device("cuda", key))
    return sw


class HostFlag:
    """The status word of the operators around the attention (rotary positions, feed-forward): one pinned host
    word per device that their kernels write only when something went wrong, so a good call costs nothing.
    The next call that finds a bit set waits for the device, so that no kernel sets another one while the word is
    cleared, and raises MslError (the failed calls' results are not valid)."""

    def __init__(self, index: Optional[int] = None):
        self.index = index
        self.word = torch.zeros(1, dtype=torch.int32, device="cpu").pin_memory()
        self.ptr = self.word.data_ptr()
        self._view = self.word.numpy()

    def poll(self) -> None:
        if self._view[0]:
            if not torch.cuda.is_current_stream_capturing():
                torch.cuda.synchronize(self.index)
            v = self._view[0]
            self._view[0] = 0
            what = []
            if v & _lib.MSL_STATUS_ROTARY_INDEX:
                what.append("a rotary position index was outside its axis (msl_rope3d, msl_qk_norm_rope)")
            if v & _lib.MSL_STATUS_TIMEOUT:
                what.append("operand copies of a matrix product did not complete within seconds (msl_gated_ffn)")
            raise _lib.MslError("a previous call", _lib.MSL_ERR_CUDA, "its results are not valid: " + "; ".join(what))


_FLAGS: dict = {}


def host_flag(device: torch.device) -> HostFlag:
    """The process-wide HostFlag of a CUDA device."""
    f = _FLAGS.get(device.index)
    if f is None:
        f = _FLAGS[device.index] = HostFlag(device.index)
    return f


def check_status(device=None) -> int:
    """Synchronously checks the kernels' status words of `device` (default: current): raises MslError if a call
    produced invalid results, else returns the attention kernels' informational bits seen so far."""
    dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
    bits = status_word(dev).check()
    torch.cuda.synchronize(dev)
    for index, flag in _FLAGS.items():
        if index == (dev.index if dev.index is not None else torch.cuda.current_device()):
            flag.poll()
    return bits


def _need_cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise RuntimeError("megaslide_b200 operands must be CUDA tensors (no CPU fallback)")


@dataclass(frozen=True)
class DsaShape:
    """Geometry of one deformable-attention call (mirrors ``msl_dsa_geometry``)."""

    batch: int
    frames: int
    height: int
    width: int
    heads: int
    head_dim: int
    kernel: Tuple[int, int, int]
    extra: int = 0
    q_frame0: int = 0
    q_frames: Optional[int] = None
    kv_frame0: int = 0
    kv_frames: Optional[int] = None
    softmax_scale: Optional[float] = None
    offset_scale: float = 1.0
    dropout_p: float = 0.0
    dropout_seed: int = 0
    algo: int = 0  # 0 auto, 1 CUDA-core gather, 2 tensor-core envelope

    @property
    def taps(self) -> int:
        return self.kernel[0] * self.kernel[1] * self.kernel[2]

    @property
    def q_rows(self) -> int:
        return (self.q_frames if self.q_frames is not None else self.frames) * self.height * self.width

    @property
    def kv_rows(self) -> int:
        return (self.kv_frames if self.kv_frames is not None else self.frames) * self.height * self.width

    def geometry(self, dtype: torch.dtype) -> DsaGeometry:
        kt, kh, kw = self.kernel
        scale = self.softmax_scale if self.softmax_scale is not None else 1.0 / math.sqrt(self.head_dim)
        return DsaGeometry(
            self.batch, self.frames, self.height, self.width, self.heads, self.head_dim, kt, kh, kw, self.extra,
            self.q_frame0, self.q_frames if self.q_frames is not None else self.frames,
            self.kv_frame0, self.kv_frames if self.kv_frames is not None else self.frames,
            dtype_code(dtype), float(scale), float(self.offset_scale), float(self.dropout_p),
            int(self.dropout_seed) & 0xFFFFFFFFFFFFFFFF, int(self.algo))


def wants_probs(shape: DsaShape, dtype: torch.dtype) -> bool:
    """Host-side pre-check for the tensor-core backward, which needs two outputs of the tensor-core
    forward (``probs``, ``saved``): bf16, at most 256 extra keys, head_dim a multiple of 8 in [16, 128],
    algo not forced to the CUDA-core gather.  The library makes the final decision (alignment,
    shared-memory plan)."""
    return (dtype == torch.bfloat16 and shape.extra <= 256 and shape.algo != _lib.MSL_ALGO_SIMT
            and shape.head_dim % 8 == 0 and 16 <= shape.head_dim <= 128)


def probs_buffer(shape: DsaShape, device) -> torch.Tensor:
    """float32 [B, nh, q_rows, K] buffer for the forward's per-sample softmax weights."""
    return torch.empty(shape.batch, shape.heads, shape.q_rows, shape.taps, device=device, dtype=torch.float32)


def saved_buffer(shape: DsaShape, dtype: torch.dtype, device) -> torch.Tensor:
    """uint8 buffer (msl_dsa_saved_bytes) for the tensor-core forward's per-sample records and tile
    envelopes, which the tensor-core backward reads instead of recomputing the sample coordinates."""
    g = shape.geometry(dtype)
    n = int(_lib.load().msl_dsa_saved_bytes(ctypes.byref(g)))
    if n <= 0:
        raise ValueError("invalid geometry for the saved buffer")
    return torch.empty(n, device=device, dtype=torch.uint8)


def saved_buffers(shape: DsaShape, dtype: torch.dtype, device) -> Tuple[torch.Tensor, torch.Tensor]:
    """(probs, saved): the tensor-core forward's outputs that the tensor-core backward needs."""
    return probs_buffer(shape, device), saved_buffer(shape, dtype, device)


def _check_saved(shape: DsaShape, dtype: torch.dtype, saved: torch.Tensor) -> None:
    g = shape.geometry(dtype)
    n = int(_lib.load().msl_dsa_saved_bytes(ctypes.byref(g)))
    if saved.dtype != torch.uint8 or saved.numel() < n or not saved.is_contiguous():
        raise ValueError(f"saved must be a contiguous uint8 tensor of at least {n} bytes (saved_buffer)")


def _check_probs(shape: DsaShape, probs: torch.Tensor) -> None:
    want = (shape.batch, shape.heads, shape.q_rows, shape.taps)
    if probs.dtype != torch.float32 or tuple(probs.shape) != want or not probs.is_contiguous():
        raise ValueError(f"probs must be a contiguous float32 tensor of shape {want}")


def _check_offset_bias(bias: Optional[torch.Tensor], n: int) -> None:
    if bias is not None and (bias.dtype != torch.float32 or bias.numel() != n or not bias.is_contiguous()):
        raise ValueError(f"offset_bias must be a contiguous float32 tensor of {n} elements")


def attn_fwd(shape: DsaShape, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, offsets: torch.Tensor,
             ek: Optional[torch.Tensor] = None, ev: Optional[torch.Tensor] = None,
             out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
             status: Optional[torch.Tensor] = None,
             probs: Optional[torch.Tensor] = None,
             saved: Optional[torch.Tensor] = None,
             offset_bias: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Deformable gather attention forward.

    q: [B*q_rows, >=C] row view; k, v: [B*kv_rows, >=C]; offsets: float32 [B*q_rows, >=nh*K*3];
    ek, ev: [B*G, >=C] or None.  Returns (out [B*q_rows, C], lse float32 [B, nh, q_rows]).
    probs, saved (optional, see saved_buffers): filled with the per-sample softmax weights and the
    per-sample records for the tensor-core backward; the call raises MslError(MSL_ERR_UNSUPPORTED)
    when the tensor-core forward does not apply to these operands.  offset_bias (float32 [nh*K*3]):
    added to every offsets row before use (offsets + bias, one float32 rounding).
    """
    _need_cuda(q, k, v, offsets, ek, ev, offset_bias)
    _check_offset_bias(offset_bias, shape.heads * shape.taps * 3)
    C = shape.heads * shape.head_dim
    dt = q.dtype
    if offsets.dtype != torch.float32:
        raise TypeError("offsets must be float32")
    if out is None:
        out = torch.empty(shape.batch * shape.q_rows, C, device=q.device, dtype=dt)
    if lse is None:
        lse = torch.empty(shape.batch, shape.heads, shape.q_rows, device=q.device, dtype=torch.float32)
    io = DsaFwdIO(_ptr(q), _rows(q, "q"), _ptr(k), _rows(k, "k"), _ptr(v), _rows(v, "v"),
                  _ptr(offsets), _rows(offsets, "offsets"), _ptr(ek), _ptr(ev),
                  _rows(ek, "ek") if ek is not None else 0, _ptr(out), _rows(out, "out"), _ptr(lse), _ptr(status))
    if probs is not None:
        _need_cuda(probs)
        _check_probs(shape, probs)
        io.probs = _ptr(probs)
    if saved is not None:
        _need_cuda(saved)
        _check_saved(shape, dt, saved)
        io.saved = _ptr(saved)
    io.offset_bias = _ptr(offset_bias)
    g = shape.geometry(dt)
    with torch.cuda.device(q.device):
        rc = _call("msl_dsa_attn_fwd", q.device,
                   lambda: _lib.load().msl_dsa_attn_fwd(ctypes.byref(g), ctypes.byref(io), _stream(q.device)))
    _lib.check("msl_dsa_attn_fwd", rc)
    return out, lse


def attn_bwd(shape: DsaShape, q, k, v, offsets, out, lse, dout, *, ek=None, ev=None, dq=None, dk=None, dv=None,
             dk_acc=None, dv_acc=None, doffsets=None, dek=None, dev=None, workspace=None, status=None, probs=None,
             saved=None, doff_dtype=torch.float32, offset_bias=None):
    """Deformable gather attention backward.

    Without dk_acc: dK/dV are written to dk/dv (allocated if None) in q's dtype, float32
    accumulators live in ``workspace`` (allocated if None).  With dk_acc/dv_acc (float32 views):
    dK/dV are ACCUMULATED there.  Returns (dq, dk, dv, doffsets, dek, dev); dk/dv are the
    accumulators in accumulate mode.  probs, saved: the tensor-core forward's outputs for these operands
    (attn_fwd(probs=..., saved=...)); with both, the tensor-core backward runs where it applies.
    doffsets (or doff_dtype when it is allocated here) is float32 or bf16 (the float32 gradient rounded
    to nearest even).  offset_bias: the forward's.
    """
    _need_cuda(q, k, v, offsets, out, lse, dout, ek, ev, offset_bias)
    _check_offset_bias(offset_bias, shape.heads * shape.taps * 3)
    C = shape.heads * shape.head_dim
    dt = q.dtype
    dev_ = q.device
    rows_q = shape.batch * shape.q_rows
    rows_kv = shape.batch * shape.kv_rows
    if dq is None:
        dq = torch.empty(rows_q, C, device=dev_, dtype=dt)
    accumulate = dk_acc is not None
    if not accumulate:
        if dk is None:
            dk = torch.empty(rows_kv, C, device=dev_, dtype=dt)
        if dv is None:
            dv = torch.empty(rows_kv, C, device=dev_, dtype=dt)
    if doffsets is None:
        doffsets = torch.empty(rows_q, shape.heads * shape.taps * 3, device=dev_, dtype=doff_dtype)
    if doffsets.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError("doffsets must be float32 or bfloat16")
    if shape.extra > 0:
        if dek is None:
            dek = torch.empty(shape.batch * shape.extra, C, device=dev_, dtype=torch.float32)
        if dev is None:
            dev = torch.empty(shape.batch * shape.extra, C, device=dev_, dtype=torch.float32)
    g = shape.geometry(dt)
    lib = _lib.load()
    need = int(lib.msl_dsa_attn_bwd_workspace_bytes(ctypes.byref(g), 1 if accumulate else 0))
    if need and (workspace is None or workspace.numel() < need):
        workspace = torch.empty(need, device=dev_, dtype=torch.uint8)
    io = DsaBwdIO(
        _ptr(q), _rows(q, "q"), _ptr(k), _rows(k, "k"), _ptr(v), _rows(v, "v"),
        _ptr(offsets), _rows(offsets, "offsets"), _ptr(ek), _ptr(ev), _rows(ek, "ek") if ek is not None else 0,
        _ptr(out), _rows(out, "out"), _ptr(lse), _ptr(dout), _rows(dout, "dout"),
        _ptr(dq), _rows(dq, "dq"),
        None if accumulate else _ptr(dk), None if accumulate else _ptr(dv),
        0 if accumulate else _rows(dk, "dk"),
        _ptr(dk_acc), _ptr(dv_acc), _rows(dk_acc, "dk_acc") if accumulate else 0,
        _ptr(doffsets), _rows(doffsets, "doffsets"), _ptr(dek), _ptr(dev), _ptr(status))
    io.doff_dtype = dtype_code(doffsets.dtype)
    io.offset_bias = _ptr(offset_bias)
    if probs is not None:
        _need_cuda(probs)
        _check_probs(shape, probs)
        io.probs = _ptr(probs)
    if saved is not None:
        _need_cuda(saved)
        _check_saved(shape, dt, saved)
        io.saved = _ptr(saved)
    with torch.cuda.device(dev_):
        rc = _call("msl_dsa_attn_bwd", dev_,
                   lambda: lib.msl_dsa_attn_bwd(ctypes.byref(g), ctypes.byref(io), _ptr(workspace) if need else None,
                                                need, _stream(dev_)))
    _lib.check("msl_dsa_attn_bwd", rc)
    if accumulate:
        dk, dv = dk_acc, dv_acc
    return dq, dk, dv, doffsets, dek, dev


@dataclass(frozen=True)
class ConvShape:
    """Geometry of a depthwise conv call (mirrors ``msl_dwconv_geometry``)."""

    batch: int
    frames: int
    height: int
    width: int
    channels: int
    kernel: Tuple[int, int, int]
    in_frame0: int = 0
    in_frames: Optional[int] = None
    out_frame0: int = 0
    out_frames: Optional[int] = None
    zero_outside: bool = False  # input frames outside the window read as zero (sharded adjoint)

    def geometry(self, dtype: torch.dtype) -> DwconvGeometry:
        kt, kh, kw = self.kernel
        return DwconvGeometry(self.batch, self.frames, self.height, self.width, self.channels, kt, kh, kw,
                              self.in_frame0, self.in_frames if self.in_frames is not None else self.frames,
                              self.out_frame0, self.out_frames if self.out_frames is not None else self.frames,
                              dtype_code(dtype), 1 if self.zero_outside else 0)

    @property
    def out_rows(self) -> int:
        return self.batch * (self.out_frames if self.out_frames is not None else self.frames) * self.height * self.width


def conv_weight_kc(w: torch.Tensor) -> torch.Tensor:
    """nn.Conv3d depthwise weight [C, 1, kt, kh, kw] -> float32 tap-major [kt*kh*kw, C]."""
    C = w.shape[0]
    return w.detach().reshape(C, -1).t().contiguous().float()


def dwconv_fwd(shape: ConvShape, x: torch.Tensor, weight_kc: torch.Tensor, bias: Optional[torch.Tensor] = None,
               bias2: Optional[torch.Tensor] = None, epilogue: int = _lib.MSL_EPI_NONE,
               aux: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
               out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """y = epilogue(depthwise_conv(x) + bias [+ bias2]); x/y [rows, >=C] row views.  y (and aux)
    have ``out_dtype`` (default: x's dtype)."""
    _need_cuda(x, weight_kc, bias, bias2, aux)
    for t, nm in ((weight_kc, "weight"), (bias, "bias"), (bias2, "bias2")):
        if t is not None and (t.dtype != torch.float32 or not t.is_contiguous()):
            raise TypeError(f"{nm} must be a contiguous float32 tensor")
    if out is None:
        out = torch.empty(shape.out_rows, shape.channels, device=x.device, dtype=out_dtype or x.dtype)
    if aux is not None and aux.dtype != out.dtype:
        raise TypeError("aux must have the output's dtype")
    g = shape.geometry(x.dtype)
    with torch.cuda.device(x.device):
        rc = _call("msl_dwconv3d_fwd", x.device, lambda: _lib.load().msl_dwconv3d_fwd(
            ctypes.byref(g), _ptr(x), _rows(x, "x"), _ptr(weight_kc), _ptr(bias), _ptr(bias2), int(epilogue),
            _ptr(aux), _rows(aux, "aux") if aux is not None else 0, _ptr(out), _rows(out, "y"),
            dtype_code(out.dtype), _stream(x.device)))
    _lib.check("msl_dwconv3d_fwd", rc)
    return out


def dwconv_bwd_data(shape: ConvShape, dy: torch.Tensor, weight_kc: torch.Tensor,
                    out: Optional[torch.Tensor] = None, accumulate: bool = False) -> torch.Tensor:
    """dx = conv_transpose(dy); the geometry's input window is dy's frames, output is dx's.
    accumulate=True adds into ``out`` (float32) instead: dx += conv_transpose(dy)."""
    _need_cuda(dy, weight_kc)
    if accumulate:
        if out is None or out.dtype != torch.float32:
            raise TypeError("accumulate=True needs a float32 out")
    elif out is None:
        out = torch.empty(shape.out_rows, shape.channels, device=dy.device, dtype=dy.dtype)
    g = shape.geometry(dy.dtype)
    name = "msl_dwconv3d_bwd_data_acc" if accumulate else "msl_dwconv3d_bwd_data"
    with torch.cuda.device(dy.device):
        rc = _call(name, dy.device, lambda: getattr(_lib.load(), name)(
            ctypes.byref(g), _ptr(dy), _rows(dy, "dy"), _ptr(weight_kc), _ptr(out), _rows(out, "dx"),
            _stream(dy.device)))
    _lib.check(name, rc)
    return out


def dwconv_bwd_weight(shape: ConvShape, dy: torch.Tensor, x: torch.Tensor, dweight_kc: torch.Tensor,
                      dbias: Optional[torch.Tensor] = None) -> None:
    """dweight_kc [K, C] += sum dy * shifted x ; dbias [C] += sum dy (float32, accumulated)."""
    _need_cuda(dy, x, dweight_kc, dbias)
    g = shape.geometry(x.dtype)
    with torch.cuda.device(dy.device):
        rc = _call("msl_dwconv3d_bwd_weight", dy.device, lambda: _lib.load().msl_dwconv3d_bwd_weight(
            ctypes.byref(g), _ptr(dy), _rows(dy, "dy"), dtype_code(dy.dtype), _ptr(x), _rows(x, "x"),
            _ptr(dweight_kc), _ptr(dbias), _stream(dy.device)))
    _lib.check("msl_dwconv3d_bwd_weight", rc)


def offsets_absmax(offsets: torch.Tensor, heads: int, taps: int, offset_scale: float = 1.0,
                   out: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Per-axis max |(offset + bias) * offset_scale| -> float32[3] on the device (channel 0, 1, 2)."""
    _need_cuda(offsets, bias)
    _check_offset_bias(bias, heads * taps * 3)
    if out is None:
        out = torch.zeros(3, device=offsets.device, dtype=torch.float32)
    with torch.cuda.device(offsets.device):
        rc = _lib.load().msl_offsets_absmax(_ptr(offsets), offsets.shape[0], _rows(offsets, "offsets"), _ptr(bias),
                                            heads, taps,
                                            float(offset_scale), _ptr(out), _stream(offsets.device))
    _lib.check("msl_offsets_absmax", rc)
    return out


def convert_f32(src: torch.Tensor, dst: torch.Tensor) -> torch.Tensor:
    _need_cuda(src, dst)
    with torch.cuda.device(src.device):
        rc = _lib.load().msl_convert_f32(_ptr(src), _rows(src, "src"), _ptr(dst), _rows(dst, "dst"),
                                         dtype_code(dst.dtype), src.shape[0], src.shape[1], _stream(src.device))
    _lib.check("msl_convert_f32", rc)
    return dst


_HERE = nullcontext()
# the handle alone (current_stream() builds an object, 2 us a call), and the device without asking whether CUDA has started
_raw_stream, _current = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice


def _on(dev: torch.device):
    """Context that makes `dev` current; nothing to do where it is."""
    return _HERE if dev.index == _current() else torch.cuda.device(dev)


def _ld(t: torch.Tensor, name: str) -> int:
    """Row stride (elements) of rows of t.shape[-1]: of contiguous tensors of any shape, of row views [rows, C] and of
    [B, N, C] whose samples follow one another at the rows' stride."""
    if t.is_contiguous():
        return t.shape[-1]
    if t.dim() == 3:
        B, N, C = t.shape
        sb, sn, sc = t.stride()
        if (sc == 1 or C == 1) and (B == 1 or N == 1 or sb == N * sn):
            ld = sn if N > 1 else sb
            if ld >= C:
                return ld
        raise ValueError(f"{name} must be rows at one stride, got shape {tuple(t.shape)} strides {t.stride()}")
    return _rows(t, name)


def _extent(t: torch.Tensor, name: str, rows: int, width: int) -> int:
    """Row stride of an operand; refuses one that is not `rows` rows of at least `width` elements: the kernels go by the
    call's geometry and would read or write beyond it."""
    shape = t.shape
    if not shape or shape[-1] < width or t.numel() != rows * shape[-1]:
        raise ValueError(f"{name} must be {rows} rows of {width} elements, got {tuple(shape)}")
    return shape[-1] if t.is_contiguous() else _ld(t, name)


def _operand(t: torch.Tensor, name: str, rows: int, width: int, dtype: torch.dtype, dev: torch.device) -> int:
    """The same, and refuses one that is not of the call's type and on its device."""
    if t.dtype != dtype:
        raise TypeError(f"{name} must have the call's dtype {dtype}, got {t.dtype}")
    if t.device != dev:
        raise RuntimeError(f"{name} must be on the call's CUDA device {dev}, got {t.device}")
    return _extent(t, name, rows, width)


def _result(t: Optional[torch.Tensor], name: str, like: torch.Tensor, rows: int, width: int) -> Tuple[torch.Tensor, int]:
    """A call's result and its row stride: the caller's tensor, checked, or a new one of like's rows."""
    if t is None:
        return torch.empty(*like.shape[:-1], width, device=like.device, dtype=like.dtype), width
    return t, _operand(t, name, rows, width, like.dtype, like.device)


class RotaryShape:
    """Geometry of a rotary call (``msl_rotary_geometry``): `tokens` of each of `batch` samples, the table's extents
    (frames, height, width), the channels each axis turns, the heads' width."""

    __slots__ = ("batch", "tokens", "rows", "video_shape", "axes", "head_dim", "table_pairs", "_geom")

    def __init__(self, batch: int, tokens: int, video_shape: Tuple[int, int, int], axes: Tuple[int, int, int], head_dim: int,
                 frame0: int = 0, interleaved: bool = True):
        t, h, w = video_shape
        at, ah, aw = axes
        self.batch, self.tokens, self.video_shape, self.axes, self.head_dim = batch, tokens, video_shape, axes, head_dim
        self.rows = batch * tokens
        self.table_pairs = (t * at + h * ah + w * aw) // 2
        self._geom = _lib.RotaryGeometry(batch * tokens, tokens or 1, t, h, w, frame0, at, ah, aw, head_dim, 1 if interleaved else 0, 0)

    def geometry(self, dtype: torch.dtype) -> "_lib.RotaryGeometry":
        self._geom.dtype = dtype_code(dtype)
        return self._geom


def _check_positions(shape: RotaryShape, table: Optional[torch.Tensor], index: Optional[torch.Tensor], dev: torch.device) -> int:
    """Checks a rotary call's table and index; returns the rows of the index (0 without one)."""
    if table is None:
        return 0
    if table.dtype != torch.float32 or table.numel() != 2 * shape.table_pairs or not table.is_contiguous():
        raise ValueError(f"table must be a contiguous float32 tensor of {shape.table_pairs} (cos, sin) pairs (rotary_table), "
                         f"got {tuple(table.shape)} {table.dtype}")
    if table.device != dev:
        raise RuntimeError("table must be on the tokens' CUDA device")
    if index is None:
        return 0
    if index.dtype != torch.int32 or not index.is_contiguous() or index.shape[-1:] != (3,):
        raise ValueError(f"index must be a contiguous int32 tensor [..., tokens, 3], got {tuple(index.shape)} {index.dtype}")
    rows = index.numel() // 3
    if rows not in (shape.tokens, shape.batch * shape.tokens):
        raise ValueError(f"index names {rows} tokens, the call has {shape.tokens} in each of {shape.batch} samples")
    if index.device != dev:
        raise RuntimeError("index must be on the tokens' CUDA device")
    return rows


def _flag(dev: torch.device, status: Optional[torch.Tensor]) -> int:
    """Address a kernel reports to: the caller's device word, or the device's HostFlag (which raises here if an
    earlier call has reported)."""
    if status is not None:
        if status.dtype != torch.int32 or status.numel() < 1 or status.device != dev:
            raise ValueError(f"status must be an int32 word on {dev}, got {status.numel()} of {status.dtype} on {status.device}")
        return status.data_ptr()
    f = _FLAGS.get(dev.index) or host_flag(dev)
    f.poll()
    return f.ptr


def rope3d(shape: RotaryShape, heads: int, x: torch.Tensor, table: torch.Tensor, index: Optional[torch.Tensor] = None,
           inverse: bool = False, out: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotates the heads of x [rows, >= heads*head_dim] (row view; or [B, N, C] at one row stride) by their tokens' positions; ``inverse`` turns
    back, which is the backward pass.  ``out`` may be x.  status: a device word for MSL_STATUS_ROTARY_INDEX in
    place of the device's HostFlag."""
    _need_cuda(x, table, index)
    dev = x.device
    index_rows = _check_positions(shape, table, index, dev)
    width = heads * shape.head_dim
    x_ld = _extent(x, "x", shape.rows, width)
    out, out_ld = _result(out, "out", x, shape.rows, width)
    g = shape.geometry(x.dtype)
    flag = _flag(dev, status) if index is not None else None
    with _on(dev):
        rc = _call("msl_rope3d", dev, lambda: _lib.load().msl_rope3d(
            ctypes.byref(g), heads, x.data_ptr(), x_ld, table.data_ptr(), _ptr(index), index_rows, 1 if inverse else 0,
            out.data_ptr(), out_ld, flag, _raw_stream(dev.index)))
    _lib.check("msl_rope3d", rc)
    return out


def _qk_io(shape: RotaryShape, heads: int, kv_heads: int, q, k, q_weight, k_weight, eps, table, index, status) -> "_lib.QkNormIO":
    _need_cuda(q, k, q_weight, k_weight, table, index)
    dev = q.device
    q_ld = _extent(q, "q", shape.rows, heads * shape.head_dim)
    k_ld = _operand(k, "k", shape.rows, kv_heads * shape.head_dim, q.dtype, dev) if kv_heads else 0
    wdt = torch.float32
    for w, nm in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if w is None:
            continue
        if w.numel() != shape.head_dim or not w.is_contiguous():
            raise ValueError(f"{nm} must be a contiguous tensor of head_dim = {shape.head_dim} elements, got {tuple(w.shape)}")
        if w.device != dev:
            raise RuntimeError(f"{nm} must be on q's CUDA device")
        wdt = w.dtype
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        raise TypeError("q_weight and k_weight must have the same dtype")
    return _lib.QkNormIO(
        q.data_ptr(), q_ld, _ptr(k) if kv_heads else None, k_ld, _ptr(q_weight), _ptr(k_weight),
        None, 0, None, 0, _ptr(table), _ptr(index), _check_positions(shape, table, index, dev),
        _flag(dev, status) if index is not None else None, heads, kv_heads, dtype_code(wdt), eps)


def qk_norm_rope_fwd(shape: RotaryShape, heads: int, kv_heads: int, q: torch.Tensor, k: Optional[torch.Tensor],
                     q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor], eps: float = 1e-6,
                     table: Optional[torch.Tensor] = None, index: Optional[torch.Tensor] = None,
                     q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None,
                     status: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """RMS norm of every head of q [rows, >= heads*head_dim] and k [rows, >= kv_heads*head_dim] (row views) times
    the weights (None = ones), then the rotation (none without a table).  q_out / k_out may be q / k; kv_heads = 0
    takes q alone.  status as in rope3d."""
    io = _qk_io(shape, heads, kv_heads, q, k, q_weight, k_weight, eps, table, index, status)
    dev = q.device
    q_out, io.q_out_ld = _result(q_out, "q_out", q, shape.rows, heads * shape.head_dim)
    io.q_out = q_out.data_ptr()
    if kv_heads:
        k_out, io.k_out_ld = _result(k_out, "k_out", k, shape.rows, kv_heads * shape.head_dim)
        io.k_out = k_out.data_ptr()
    g = shape.geometry(q.dtype)
    with _on(dev):
        rc = _call("msl_qk_norm_rope_fwd", dev, lambda: _lib.load().msl_qk_norm_rope_fwd(
            ctypes.byref(g), ctypes.byref(io), _raw_stream(dev.index)))
    _lib.check("msl_qk_norm_rope_fwd", rc)
    return q_out, k_out


def qk_norm_rope_bwd(shape: RotaryShape, heads: int, kv_heads: int, q, k, q_weight, k_weight, dq_out, dk_out, eps: float = 1e-6,
                     table=None, index=None, dq=None, dk=None, weight_grads: bool = True, status=None):
    """Backward of qk_norm_rope_fwd: (dq, dk, dq_weight, dk_weight); the weights' gradients are None for weights
    that are None and where ``weight_grads`` is false.  dq / dk may be dq_out / dk_out."""
    io = _qk_io(shape, heads, kv_heads, q, k, q_weight, k_weight, eps, table, index, status)
    _need_cuda(dq_out, dk_out)
    dev = q.device
    width = heads * shape.head_dim
    io.dq_out, io.dq_out_ld = dq_out.data_ptr(), _operand(dq_out, "dq_out", shape.rows, width, q.dtype, dev)
    dq, io.dq_ld = _result(dq, "dq", q, shape.rows, width)
    io.dq = dq.data_ptr()
    if kv_heads:
        width = kv_heads * shape.head_dim
        io.dk_out, io.dk_out_ld = dk_out.data_ptr(), _operand(dk_out, "dk_out", shape.rows, width, q.dtype, dev)
        dk, io.dk_ld = _result(dk, "dk", k, shape.rows, width)
        io.dk = dk.data_ptr()
    dgq = torch.empty_like(q_weight) if weight_grads and q_weight is not None else None
    dgk = torch.empty_like(k_weight) if weight_grads and k_weight is not None and kv_heads else None
    io.dq_weight, io.dk_weight = _ptr(dgq), _ptr(dgk)
    g = shape.geometry(q.dtype)
    lib = _lib.load()
    with _on(dev):
        need = int(lib.msl_qk_norm_rope_bwd_workspace_bytes(ctypes.byref(g), ctypes.byref(io)))
        ws = torch.empty(need, device=dev, dtype=torch.uint8) if need else None
        rc = _call("msl_qk_norm_rope_bwd", dev, lambda: lib.msl_qk_norm_rope_bwd(
            ctypes.byref(g), ctypes.byref(io), _ptr(ws), need, _raw_stream(dev.index)))
    _lib.check("msl_qk_norm_rope_bwd", rc)
    return dq, dk, dgq, dgk


_ACTIVATIONS = {"silu": _lib.MSL_ACT_SILU, "gelu": _lib.MSL_ACT_GELU}


def activation_code(name: str) -> int:
    try:
        return _ACTIVATIONS[name]
    except KeyError:
        raise ValueError(f"activation must be one of {sorted(_ACTIVATIONS)}, got {name!r}") from None


def _ffn_check(x, w_in, w_out, b_in, b_out) -> Tuple[int, int, int]:
    """(rows, dim, hidden) of a gated feed-forward call, its operands checked."""
    _need_cuda(x, w_in, w_out, b_in, b_out)
    C = x.shape[-1]
    M = x.numel() // C if C else 0
    if w_in.dim() != 2 or w_in.shape[0] % 2 or w_in.shape[1] != C:
        raise ValueError(f"w_in must be [2 * hidden, {C}], got {tuple(w_in.shape)}")
    F = w_in.shape[0] // 2
    if tuple(w_out.shape) != (C, F):
        raise ValueError(f"w_out must be {(C, F)}, got {tuple(w_out.shape)}")
    dev, dt = x.device, x.dtype
    for t, n, nm in ((w_in, 0, "w_in"), (w_out, 0, "w_out"), (b_in, 2 * F, "b_in"), (b_out, C, "b_out")):
        if t is None:
            continue
        if n and (t.dim() != 1 or t.numel() != n):
            raise ValueError(f"{nm} must be [{n}], got {tuple(t.shape)}")
        if t.dtype != dt:
            raise TypeError(f"{nm} must have x's dtype {dt}, got {t.dtype}")
        if not t.is_contiguous():
            raise ValueError(f"{nm} must be contiguous")
        if t.device != dev:
            raise RuntimeError(f"{nm} must be on x's CUDA device")
    return M, C, F


def _unaligned(*operands) -> int:
    """1 where an operand's address is no multiple of 16 bytes (views into packed buffers, say)."""
    return 1 if any(t is not None and t.data_ptr() & 15 for t in operands) else 0


def _kept_bytes(M: int, F: int) -> Tuple[int, int]:
    """Bytes of the kept factors of a bf16 block: the upper 16 bits [M, 2, F], and with the low 8 [M, 2, F rounded up to
    16] after them."""
    return 4 * M * F, 4 * M * F + 2 * M * ((F + 15) // 16 * 16)


def gated_ffn_fwd(x: torch.Tensor, w_in: torch.Tensor, w_out: torch.Tensor, b_in: Optional[torch.Tensor] = None,
                  b_out: Optional[torch.Tensor] = None, activation: str = "silu", keep: bool = False,
                  status: Optional[torch.Tensor] = None):
    """Gated feed-forward block on x [rows, >= dim] (row view).  Returns (y, h, kept): h [rows, hidden] the gated
    product, kept what the backward needs (u act'(g), then act(g)) where ``keep``, else None: [rows, 2 * hidden] in float32, in
    bf16 bytes that hold 24 bits of each.  status: a device word for MSL_STATUS_TIMEOUT in place of the device's HostFlag."""
    M, C, F = _ffn_check(x, w_in, w_out, b_in, b_out)
    dev, dt = x.device, x.dtype
    x_ld = _ld(x, "x")
    px, pi, po, pbi, pbo = x.data_ptr(), w_in.data_ptr(), w_out.data_ptr(), _ptr(b_in), _ptr(b_out)
    off = (px | pi | po | (pbi or 0) | (pbo or 0)) & 15 or x_ld % 8
    g = _lib.FfnGeometry(M, C, F, dtype_code(dt), activation_code(activation), 1 if off else 0)
    h = torch.empty(M, F, device=dev, dtype=dt)
    kept = low = None
    if keep and dt == torch.float32:
        kept = torch.empty(M, 2 * F, device=dev, dtype=dt)
    elif keep:
        high, both = _kept_bytes(M, F)
        kept = torch.empty(both, device=dev, dtype=torch.uint8)
        low = kept.data_ptr() + high
    y = torch.empty(x.shape, device=dev, dtype=dt)
    io = _lib.FfnIO(px, x_ld, pi, pbi, po, pbo, h.data_ptr(), _ptr(kept), y.data_ptr(), C)
    io.status, io.kept_low = _flag(dev, status), low
    lib = _lib.load()
    with _on(dev):
        need = int(lib.msl_gated_ffn_workspace_bytes(ctypes.byref(g), 0))
        ws = torch.empty(need, device=dev, dtype=torch.uint8) if need else None
        rc = _call("msl_gated_ffn_fwd", dev, lambda: lib.msl_gated_ffn_fwd(
            ctypes.byref(g), ctypes.byref(io), _ptr(ws), need, _raw_stream(dev.index)))
    _lib.check("msl_gated_ffn_fwd", rc)
    return y, h, kept


def gated_ffn_bwd(x, w_in, w_out, h, kept, dy, b_in=None, b_out=None, activation: str = "silu",
                  needs=(True, True, True, True, True), status: Optional[torch.Tensor] = None):
    """Backward of gated_ffn_fwd(keep=True): (dx, dw_in, dw_out, db_in, db_out); ``needs`` says which are computed
    (the others, and those of biases that are None, are None)."""
    M, C, F = _ffn_check(x, w_in, w_out, b_in, b_out)
    _need_cuda(h, kept, dy)
    dev, dt = x.device, x.dtype
    high, both = _kept_bytes(M, F)
    rows = [(h, "h", M, F, dt), (dy, "dy", M, C, dt), (kept, "kept", M, 2 * F, dt) if dt == torch.float32 else (kept, "kept", 1, both, torch.uint8)]
    for t, nm, n, width, kind in rows:
        _operand(t, nm, n, width, kind, dev)
        if nm != "dy" and (t.shape[-1] != width or not t.is_contiguous()):
            raise ValueError(f"{nm} must be contiguous rows of {width} elements, got shape {tuple(t.shape)} strides {t.stride()}")
    if dy.shape[-1] != C:
        raise ValueError(f"dy must have rows of {C} elements, got {tuple(dy.shape)}")
    needs = (needs[0], needs[1], needs[2], needs[3] and b_in is not None, needs[4] and b_out is not None)
    dx = torch.empty(x.shape, device=dev, dtype=dt) if needs[0] else None
    dw_in = torch.empty_like(w_in) if needs[1] else None
    dw_out = torch.empty_like(w_out) if needs[2] else None
    db_in = torch.empty_like(b_in) if needs[3] else None
    db_out = torch.empty_like(b_out) if needs[4] else None
    dgu = torch.empty(M, 2 * F, device=dev, dtype=dt) if needs[0] or needs[1] or needs[3] else None
    x_ld, dy_ld = _ld(x, "x"), _ld(dy, "dy")
    g = _lib.FfnGeometry(M, C, F, dtype_code(dt), activation_code(activation), _unaligned(x, w_in, w_out, dy, h, kept) or int((x_ld | dy_ld) % 8 != 0))
    io = _lib.FfnIO(x.data_ptr(), x_ld, w_in.data_ptr(), None, w_out.data_ptr(), None, h.data_ptr(), kept.data_ptr(), None, 0,
                    dy.data_ptr(), dy_ld, _ptr(dgu), _ptr(dx), C, _ptr(dw_in), _ptr(dw_out), _ptr(db_in), _ptr(db_out),
                    _flag(dev, status), kept.data_ptr() + high if dt == torch.bfloat16 else None)
    lib = _lib.load()
    with _on(dev):
        need = int(lib.msl_gated_ffn_workspace_bytes(ctypes.byref(g), 1))
        ws = torch.empty(need, device=dev, dtype=torch.uint8) if need else None
        rc = _call("msl_gated_ffn_bwd", dev, lambda: lib.msl_gated_ffn_bwd(
            ctypes.byref(g), ctypes.byref(io), _ptr(ws), need, _raw_stream(dev.index)))
    _lib.check("msl_gated_ffn_bwd", rc)
    return dx, dw_in, dw_out, db_in, db_out


_dtype_of, _device_of = attrgetter("dtype"), attrgetter("device")
_numel_of, _ptr_of, _is_whole = torch.Tensor.numel, torch.Tensor.data_ptr, torch.Tensor.is_contiguous


def _dense(t: torch.Tensor) -> bool:
    """Whether the elements fill their memory without gaps and none twice, in whatever order of the axes."""
    n = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz > 1):
        if stride != n:
            return False
        n *= size
    return True


def _one_device(ts: List[torch.Tensor], dev: torch.device, name: str) -> bool:
    """Checks device and density of the tensors of a list; whether all lie in the order of their axes."""
    if set(map(_device_of, ts)) != {dev} or dev.type != "cuda":
        raise RuntimeError(f"every {name} must be on the same CUDA device (no CPU fallback)")
    whole = all(map(_is_whole, ts))
    if not whole:
        for i, t in enumerate(ts):
            if not (_is_whole(t) or _dense(t)):
                raise ValueError(f"{name} {i} must be dense, got shape {tuple(t.shape)} strides {t.stride()}")
    return whole


def grad_norm(src: List[torch.Tensor], dst: Optional[List[torch.Tensor]] = None, max_norm: float = 0.0,
              extra_sumsq: float = 0.0) -> torch.Tensor:
    """sqrt(extra_sumsq + the sum of squares of every element of the CUDA tensors `src`, each dense in any order of its
    axes), a 0-dim float32 tensor; with ``dst`` also dst[i] = src[i] * min(1, max_norm / (norm + 1e-6)) (dst[i] in src[i]'s
    order; it may be src[i])."""
    if not src:
        raise ValueError("no tensors")
    n = len(src)
    dev = src[0].device
    whole = _one_device(src, dev, "tensor")
    dtypes = list(map(_dtype_of, src))
    sizes = list(map(_numel_of, src))
    if dst is not None and dst is not src:
        if len(dst) != n:
            raise ValueError(f"{n} tensors, but {len(dst)} to write")
        whole = _one_device(dst, dev, "out") and whole
        if list(map(_dtype_of, dst)) != dtypes or list(map(_numel_of, dst)) != sizes:
            raise ValueError("every out must have its tensor's dtype and size")
        if not whole:
            for i, (a, b) in enumerate(zip(src, dst)):
                if not (_is_whole(a) and _is_whole(b)) and (a.shape != b.shape or a.stride() != b.stride()):
                    raise ValueError(f"out {i} must lie in its tensor's order: strides {a.stride()}, got {b.stride()}")
    codes = {d: dtype_code(d) for d in set(dtypes)}
    numel = (ctypes.c_int64 * n)(*sizes)
    codes_arr = (ctypes.c_int32 * n)(*[codes[d] for d in dtypes])
    ptrs = (ctypes.c_void_p * n)(*map(_ptr_of, src))
    norm = torch.empty((), device=dev, dtype=torch.float32)
    lib = _lib.load()
    with _on(dev):
        need = int(lib.msl_grad_norm_workspace_bytes(numel, n))
        ws = torch.empty(need, device=dev, dtype=torch.uint8)
        if dst is None:
            name = "msl_grad_norm"
            rc = _call(name, dev, lambda: lib.msl_grad_norm(ptrs, numel, codes_arr, n, extra_sumsq, norm.data_ptr(), ws.data_ptr(),
                                                            need, _raw_stream(dev.index)))
        else:
            name = "msl_grad_clip"
            outs = ptrs if dst is src else (ctypes.c_void_p * n)(*map(_ptr_of, dst))
            rc = _call(name, dev, lambda: lib.msl_grad_clip(ptrs, outs, numel, codes_arr, n, extra_sumsq, max_norm,
                                                            norm.data_ptr(), ws.data_ptr(), need, _raw_stream(dev.index)))
    _lib.check(name, rc)
    return norm
