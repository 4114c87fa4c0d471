"""Rotary positions with several axes (time, height, width), alone and together with the RMS norm of
queries and keys for each head, on the kernels of csrc/rotary.cu.

    table = rotary_table((T, H, W), (24, 24, 24), device=x.device)
    y = rope3d(x, table, video_shape=(T, H, W), axes=(24, 24, 24), heads=16)
    q, k = qk_norm_rope(q, k, q_weight, k_weight, table, video_shape=(T, H, W), axes=(24, 24, 24), heads=16)

Tokens are [B, N, heads * head_dim] in the order n = (t*H + h)*W + w, as everywhere in this package; q and k may
be columns of one qkv buffer.  `frame0` places a call's first token at a later frame of the table (a rank's
frames of a sharded volume, a streamed frame); `index` (int32 [B, N, 3] or [N, 3]) gives each token its
own three positions instead (packed images and videos, single tokens); a position outside its axis is reported by a
later call or by check_status.  float32 or bfloat16; the
statistics, the rotation and the weights' gradients are computed in float32 and rounded once.
"""

from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch
from torch import Tensor

from . import ops

Int3 = Tuple[int, int, int]


def rotary_table(video_shape: Int3, axes: Int3, theta: float = 10000.0, positions: Optional[Sequence[Tensor]] = None,
                 device=None) -> Tensor:
    """The (cos, sin) table of a video's positions: float32 [T*at/2 + H*ah/2 + W*aw/2, 2].

    axes = (at, ah, aw): the channels of a head that turn with the time, the row and the column, each even.  Pair i
    of an axis of `a` channels turns by position * theta^(-2i/a).  positions: three 1-D tensors of T, H and W
    positions (any real numbers: fractions for another resolution, say) in place of 0, 1, 2, ..."""
    parts = []
    for i, (size, ch) in enumerate(zip(video_shape, axes)):
        if size < 1 or ch < 0 or ch % 2:
            raise ValueError(f"extents must be >= 1 and axes even, got {tuple(video_shape)} and {tuple(axes)}")
        if positions is None:
            pos = torch.arange(size, dtype=torch.float64, device="cpu")
        else:
            pos = positions[i].detach().to("cpu", torch.float64)
            if tuple(pos.shape) != (size,):
                raise ValueError(f"positions[{i}] must be [{size}], got {tuple(pos.shape)}")
        freq = theta ** (-torch.arange(0, ch, 2, dtype=torch.float64, device="cpu") / max(ch, 1))
        angle = pos[:, None] * freq[None]
        parts.append(torch.stack([angle.cos(), angle.sin()], -1).reshape(-1, 2))
    return torch.cat(parts).float().to(device if device is not None else "cpu").contiguous()


def _as_rows(x: Tensor) -> Tensor:
    """[B, N, C] tokens whose rows lie at one stride: x, or a copy where its strides have none."""
    if x.is_contiguous():
        return x
    B, N, C = x.shape
    sb, sn, sc = x.stride()
    if (sc == 1 or C == 1) and (B == 1 or N == 1 or sb == N * sn) and (sn if N > 1 else sb) >= C:
        return x
    return x.contiguous()


def _check_tokens(name: str, x: Tensor, heads: int) -> int:
    """head_dim of tokens [B, N, heads * head_dim]."""
    if x.dim() != 3 or heads < 1 or x.shape[2] % heads:
        raise ValueError(f"{name} must be [B, N, heads * head_dim] with heads = {heads}, got {tuple(x.shape)}")
    if not x.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor (no CPU fallback)")
    ops.dtype_code(x.dtype)
    return x.shape[2] // heads


def _check_table(table: Optional[Tensor]) -> None:
    if table is not None and table.requires_grad and torch.is_grad_enabled():
        raise ValueError("table requires a gradient, which the rotation does not compute: detach it")


class _Call:
    """What a call's backward needs besides its tensors."""

    __slots__ = ("shape", "heads", "kv_heads", "eps")

    def __init__(self, shape: ops.RotaryShape, heads: int, kv_heads: int = 0, eps: float = 0.0):
        self.shape, self.heads, self.kv_heads, self.eps = shape, heads, kv_heads, eps


def _rotate(call: _Call, x: Tensor, table: Tensor, index: Optional[Tensor], inverse: bool) -> Tensor:
    return ops.rope3d(call.shape, call.heads, _as_rows(x), table, index, inverse)


class Rope3DFunction(torch.autograd.Function):
    """Rotation; its backward turns the gradient back."""

    @staticmethod
    def forward(ctx, call: _Call, x, table, index):
        ctx.call = call
        ctx.save_for_backward(table, index)
        return _rotate(call, x, table, index, False)

    @staticmethod
    @ops.once_only
    def backward(ctx, dy):
        table, index = ctx.saved_tensors
        return None, _rotate(ctx.call, dy, table, index, True), None, None


def rope3d(x: Tensor, table: Tensor, *, video_shape: Int3, axes: Int3, heads: int, interleaved: bool = True, frame0: int = 0,
           index: Optional[Tensor] = None) -> Tensor:
    """Turns the heads of x [B, N, heads * head_dim] by their tokens' positions (rotary_table).

    The first at/2 pairs of a head turn with the time, the next ah/2 with the row, the last aw/2 with the column;
    channels beyond at + ah + aw pass.  Pair p is channels (2p, 2p+1) (interleaved) or (p, p + (at+ah+aw)/2).
    Differentiable in x."""
    _check_table(table)
    d = _check_tokens("x", x, heads)
    call = _Call(ops.RotaryShape(x.shape[0], x.shape[1], tuple(video_shape), tuple(axes), d, frame0, interleaved), heads)
    if ops.takes_derivatives(x):
        return Rope3DFunction.apply(call, x, table, index)
    return _rotate(call, x, table, index, False)


def _norm_rotate(call: _Call, q, k, q_weight, k_weight, table, index):
    return ops.qk_norm_rope_fwd(call.shape, call.heads, call.kv_heads, _as_rows(q), _as_rows(k), q_weight, k_weight, call.eps,
                                table, index)


class QKNormRopeFunction(torch.autograd.Function):
    """Norm and rotation; the backward reads q and k again and keeps nothing else."""

    @staticmethod
    def forward(ctx, call: _Call, q, k, q_weight, k_weight, table, index):
        ctx.call = call
        ctx.save_for_backward(q, k, q_weight, k_weight, table, index)
        return _norm_rotate(call, q, k, q_weight, k_weight, table, index)

    @staticmethod
    @ops.once_only
    def backward(ctx, dq_out, dk_out):
        q, k, q_weight, k_weight, table, index = ctx.saved_tensors
        c = ctx.call
        dq, dk, dgq, dgk = ops.qk_norm_rope_bwd(c.shape, c.heads, c.kv_heads, _as_rows(q), _as_rows(k), q_weight, k_weight,
                                                _as_rows(dq_out), _as_rows(dk_out), c.eps, table, index,
                                                weight_grads=ctx.needs_input_grad[3] or ctx.needs_input_grad[4])
        return None, dq, dk, dgq, dgk, None, None


def qk_norm_rope(q: Tensor, k: Tensor, q_weight: Optional[Tensor], k_weight: Optional[Tensor], table: Optional[Tensor] = None, *,
                 heads: int, kv_heads: Optional[int] = None, eps: float = 1e-6, video_shape: Optional[Int3] = None,
                 axes: Int3 = (0, 0, 0), interleaved: bool = True, frame0: int = 0,
                 index: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
    """RMS norm of every head of q [B, N, heads * head_dim] and k [B, N, kv_heads * head_dim] (kv_heads: heads by
    default, fewer for grouped heads), times the weights [head_dim] that the heads share (None = ones), then the
    rotation of rope3d (none without a table), in one pass.  Differentiable in q, k and the weights."""
    _check_table(table)
    kv_heads = heads if kv_heads is None else kv_heads
    d = _check_tokens("q", q, heads)
    if _check_tokens("k", k, kv_heads) != d or k.shape[:2] != q.shape[:2]:
        raise ValueError(f"k must be [{q.shape[0]}, {q.shape[1]}, {kv_heads} * {d}], got {tuple(k.shape)}")
    if k.device != q.device:
        raise RuntimeError("k must be on q's CUDA device")
    if table is not None and video_shape is None:
        raise ValueError("a table needs video_shape and axes")
    if table is None:
        video_shape, axes, index, frame0 = (1, 1, 1), (0, 0, 0), None, 0
    call = _Call(ops.RotaryShape(q.shape[0], q.shape[1], tuple(video_shape), tuple(axes), d, frame0, interleaved), heads, kv_heads,
                 float(eps))
    if ops.takes_derivatives(q, k, q_weight, k_weight):
        return QKNormRopeFunction.apply(call, q, k, q_weight, k_weight, table, index)
    return _norm_rotate(call, q, k, q_weight, k_weight, table, index)
