"""Global gradient norm over many tensors and clipping on the kernels of csrc/grad_norm.cu: two launches for the
norm or for norm and scaling of up to 896 tensors with elements, one or two more for every further 896, and no wait for
the GPU."""

from __future__ import annotations

import math
from operator import attrgetter
from typing import Iterable, List, Optional, Sequence, Union

import torch
from torch import Tensor
from torch.autograd.graph import increment_version

from . import ops

_requires_grad = attrgetter("requires_grad")
Tensors = Union[Tensor, Iterable[Optional[Tensor]]]


def _list(tensors: Tensors) -> List[Tensor]:
    """The tensors of a call; of parameters, and of other leaves that require gradients, their gradients, where they have
    one."""
    ts = [tensors] if isinstance(tensors, Tensor) else tensors
    # plain tensors first: isinstance of Parameter runs a check in Python
    ts = [t if type(t) is Tensor else t.grad if isinstance(t, torch.nn.Parameter) else t for t in ts if t is not None]
    ts = [t for t in ts if t is not None]
    if any(map(_requires_grad, ts)):
        ts = [t.grad if t.requires_grad and t.is_leaf else t for t in ts]
        ts = [t for t in ts if t is not None]
    return ts


def _check(extra_sumsq: float) -> float:
    if not extra_sumsq >= 0:
        raise ValueError(f"extra_sumsq must be >= 0, got {extra_sumsq}")
    return float(extra_sumsq)


def grad_norm(tensors: Tensors, extra_sumsq: float = 0.0) -> Tensor:
    """2-norm of all elements of the tensors together (float32 or bfloat16, dense in any order of the axes, on one CUDA
    device; parameters and other leaves that require gradients stand for their gradients), as a 0-dim float32 tensor
    on their device.  extra_sumsq: a sum of squares held elsewhere (on the host, on other ranks) that belongs to the
    norm.  Without tensors the norm of extra_sumsq alone, on the CPU.  Like torch's, it records no derivative."""
    ts = _list(tensors)
    extra = _check(extra_sumsq)
    if not ts:
        return torch.tensor(math.sqrt(extra), device="cpu")
    return ops.grad_norm(ts, extra_sumsq=extra)


def clip_grad_norm_(tensors: Tensors, max_norm: float, *, out: Optional[Sequence[Tensor]] = None,
                    extra_sumsq: float = 0.0) -> Tensor:
    """Scales the tensors (as in grad_norm, gradients of parameters) by min(1, max_norm / (norm + 1e-6)) and returns the
    norm before that; nothing waits for the GPU.  out: tensors of the same dtypes, sizes and order that receive the
    result in place of the tensors themselves (slices of one flat buffer, say).  Results share memory with nothing but
    their own tensor, in place: a tensor twice in the list is refused (MslError).  A norm that is not finite reaches the
    results as the formula says (an infinite norm: zeros, and NaN for its infinite elements)."""
    if not max_norm >= 0:
        raise ValueError(f"max_norm must be >= 0, got {max_norm}")
    ts = _list(tensors)
    extra = _check(extra_sumsq)
    if not ts:
        return torch.tensor(math.sqrt(extra), device="cpu")
    out = ts if out is None else list(out)
    norm = ops.grad_norm(ts, out, float(max_norm), extra)
    increment_version(out)  # the kernel wrote them behind autograd's back
    return norm
