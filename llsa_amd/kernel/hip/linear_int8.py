"""The linear layer in 8-bit integers, for sampling: weights as whole numbers with a scale for each channel out, rows brought to whole numbers
with a scale each on the way in."""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from ..._lib import current_lib
from .linear import _activation


def quantize_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """x (..., K) of bf16, fp16 or fp32 -> (q, scale): q (..., K) int8, scale (...) fp32, with scale = max |x| / 127 over a row and q = x / scale to the
    nearest whole number, halves to even.  A row of zeros has a scale of zero; one that holds an infinity or a NaN a scale of NaN and q of zero.  What
    linear_int8 takes as weight (N, K) and, for rows that several layers read, as x.  No gradient."""
    lib = current_lib()
    return lib.host.quantize_rows(lib.host_library, x)


def linear_int8(x: Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]], weight: torch.Tensor, scale: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                activation: Optional[str] = None, gate: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
                dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """residual + gate * activation(x @ (scale * weight).T + bias), the product in 8-bit integers.

    x is (..., K) of bf16 or fp16, which quantize_rows brings to 8 bits here, or its result (q, scales) for such an x; weight (N, K) int8 and scale (N,) fp32
    (quantize_rows of a linear layer's weight), bias (N,), gate (B, N) for an x of (B, ..., K), one row for each sample, residual (..., N).  The result, bias,
    gate and residual have x's dtype, or `dtype` (bf16 or fp16) where x is a pair.  K is at most 131072.  The sums are exact, what follows them is fp32,
    rounded once.  No gradient: tensors that want one are refused outside torch.no_grad()."""
    lib = current_lib()
    pair = isinstance(x, (tuple, list))
    if pair and len(x) != 2:
        raise ValueError(f"linear_int8: x must be a tensor or the pair that quantize_rows returns (got {len(x)} entries)")
    if pair and dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"linear_int8: dtype must be torch.bfloat16 or torch.float16 (got {dtype})")
    rows, scales = x if pair else (x, None)
    return lib.host.linear_int8(lib.host_library, rows, scales, weight, scale, bias, _activation(activation), gate, residual, dtype)
