"""Layer norm of token rows with the modulation of an adaLN block in the same pass: what the reference's block computes with
torch modules in front of its attention and of its feed-forward part (models/rope_dit_transformer_2d.py:295-337, 581-711)."""
from __future__ import annotations

from typing import Optional

import torch

from ..._lib import current_lib


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *,
               scale: Optional[torch.Tensor] = None, shift: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """((x - mean) * rsqrt(var + eps) * weight + bias) * (1 + scale) + shift, statistics over the last dimension.

    x is (..., C) in bf16, fp16 or fp32, C at most 8192; weight and bias are (C,); scale and shift are (B, C) for an x of
    (B, ..., C), one row for each sample.  Any of the four may be left out; each has x's dtype or fp32.  Everything is computed
    in fp32 and rounded once.  Differentiable in all five (once: there is no second derivative)."""
    lib = current_lib()
    return lib.host.layer_norm(lib.host_library, x, weight, bias, scale, shift, float(eps))
