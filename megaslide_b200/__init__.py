"""megaslide_b200 — B200-native (sm_100a) 3D Deformable Slide Attention for MegaSlide-DiT.

``DeformableSlideAttention3D`` is a drop-in for ``infinity.video.attention.DeformableSlideAttention3D``
(same constructor, forward signature and parameter names) whose forward and backward run on the
hand-written kernels of ``libmegaslide_b200.so`` (C ABI in ``include/megaslide_b200.h``).  Around it stand the
operators of the rest of a transformer block's step: rotary positions over time, height and width (``rope3d``),
the norm of queries and keys with that rotation (``qk_norm_rope``), the gated feed-forward block (``gated_ffn``,
``GatedMLP``) and the global gradient norm with clipping (``clip_grad_norm_``).
"""

from . import ops
from .ops import check_status
from ._lib import MslError, launch_count, library_path
from .attention import DeformableSlideAttention3D, DSA3DFunction
from .clip import clip_grad_norm_, grad_norm
from .ffn import GatedMLP, gated_ffn
from .rotary import qk_norm_rope, rope3d, rotary_table

__all__ = ["DeformableSlideAttention3D", "DSA3DFunction", "MslError", "ops", "launch_count", "library_path",
           "check_status", "rotary_table", "rope3d", "qk_norm_rope", "gated_ffn", "GatedMLP", "grad_norm", "clip_grad_norm_"]
__version__ = "0.1.0"
