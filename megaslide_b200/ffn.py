"""Gated feed-forward block on the kernels of csrc/gated_ffn.cu.

    y = (act(x Wg^T + bg) * (x Wu^T + bu)) w_out^T + b_out,   w_in = [Wg; Wu]

Both projections, their biases, the activation and the product are one kernel; the second projection is another.
For the backward the first also writes two factors of every hidden element, u act'(g) and act(g); the backward is one
kernel for the gradients of the projections (dy w_out, times the two factors) and one for each of dx, dw_in and
dw_out.  float32 or bfloat16 operands, float32 sums; the intermediate results are rounded to the operands' type,
in which the next product reads them.  (float32, and widths that are no multiple of 8, take a few more kernels.)
"""

from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn
from torch import Tensor

from . import ops


def _rows_of(x: Tensor) -> Tensor:
    """[..., C] whose rows lie at one stride: x, a row view of it, or a copy where its strides have none."""
    if x.is_contiguous():
        return x
    x2 = x.reshape(-1, x.shape[-1])
    if (x2.stride(1) != 1 and x2.shape[1] > 1) or (x2.shape[0] > 1 and x2.stride(0) < x2.shape[1]):
        x2 = x2.contiguous()
    return x2


class GatedFFNFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_in, w_out, b_in, b_out, activation):
        x2 = _rows_of(x)
        y, h, kept = ops.gated_ffn_fwd(x2, w_in, w_out, b_in, b_out, activation, keep=True)
        ctx.save_for_backward(x2, w_in, w_out, b_in, b_out, h, kept)
        ctx.activation = activation
        ctx.x_shape = x.shape
        return y if y.shape == x.shape else y.view(x.shape)

    @staticmethod
    @ops.once_only
    def backward(ctx, dy):
        x2, w_in, w_out, b_in, b_out, h, kept = ctx.saved_tensors
        dx, dw_in, dw_out, db_in, db_out = ops.gated_ffn_bwd(x2, w_in, w_out, h, kept, _rows_of(dy), b_in, b_out, ctx.activation,
                                                             needs=ctx.needs_input_grad[:5])
        return dx.view(ctx.x_shape) if dx is not None and dx.shape != ctx.x_shape else dx, dw_in, dw_out, db_in, db_out, None


def gated_ffn(x: Tensor, w_in: Tensor, w_out: Tensor, b_in: Optional[Tensor] = None, b_out: Optional[Tensor] = None,
              activation: str = "silu") -> Tensor:
    """y [..., dim] of x [..., dim]; w_in [2 * hidden, dim] holds the gate's rows, then the other's; w_out [dim, hidden];
    activation "silu" or "gelu" (erf form).  One dtype (float32 or bfloat16) for all.  Differentiable in everything."""
    if not x.is_cuda:
        raise RuntimeError("x must be a CUDA tensor (no CPU fallback)")
    if x.dim() < 1:
        raise ValueError("x must be [..., dim]")
    ops.dtype_code(x.dtype)
    if ops.takes_derivatives(x, w_in, w_out, b_in, b_out):
        return GatedFFNFunction.apply(x, w_in, w_out, b_in, b_out, activation)
    y = ops.gated_ffn_fwd(_rows_of(x), w_in, w_out, b_in, b_out, activation)[0]
    return y if y.shape == x.shape else y.view(x.shape)


class GatedMLP(nn.Module):
    """The gated block as a module: fc1 (2 * intermediate_size rows: gate, then the other) and fc2, as nn.Linear
    parameters.  Under CUDA autocast to bfloat16 it computes in bfloat16, like nn.Linear.  dropout acts on the result alone:
    the hidden values stay inside the kernels (MLP in dit.py drops out both)."""

    def __init__(self, hidden_size: int, intermediate_size: int, dropout: float = 0.0, activation: str = "silu"):
        super().__init__()
        ops.activation_code(activation)
        self.fc1 = nn.Linear(hidden_size, 2 * intermediate_size)
        self.fc2 = nn.Linear(intermediate_size, hidden_size)
        self.dropout = nn.Dropout(dropout)
        self.activation = activation

    def forward(self, x: Tensor) -> Tensor:
        p = (x, self.fc1.weight, self.fc2.weight, self.fc1.bias, self.fc2.bias)
        if torch.is_autocast_enabled("cuda") and torch.get_autocast_dtype("cuda") == torch.bfloat16:
            p = tuple(t.to(torch.bfloat16) for t in p)
        return self.dropout(gated_ffn(*p, activation=self.activation))
