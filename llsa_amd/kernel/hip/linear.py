"""Linear layers of a transformer block with what follows them in the same pass (models/rope_dit_transformer_2d.py:180-260, 581-711,
torch modules in the reference): bias, activation, the gate of an adaLN block and the residual stream."""
from __future__ import annotations

from typing import Optional

import torch

from ..._lib import current_lib

ACTIVATIONS = {None: 0, "silu": 1, "gelu": 2, "gelu_tanh": 3}          # LLSA_ACT_* of include/llsa_hip.h


def _activation(name: Optional[str]) -> int:
    if name not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {', '.join(repr(a) for a in ACTIVATIONS)} (got {name!r})")
    return ACTIVATIONS[name]


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *, activation: Optional[str] = None,
           gate: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """residual + gate * activation(x @ weight.T + bias).

    x is (..., K), weight (N, K), bias (N,), gate (B, N) for an x of (B, ..., K), one row for each sample, residual (..., N); all of
    them bf16 or all fp16.  activation: None, "silu", "gelu" (erf) or "gelu_tanh".  Sums in fp32; the forward rounds once, the
    backward, besides its results, what its products take in: the gradient behind gate and activation (or gate * weight in its place),
    and x @ weight.T + bias where it is kept.  Differentiable in all five (once); the backward keeps x, weight and, with an
    activation (or a gate that wants a gradient, on samples of less than 2 K rows), x @ weight.T + bias."""
    lib = current_lib()
    return lib.host.linear(lib.host_library, x, weight, bias, _activation(activation), gate, residual)


def feed_forward(x: torch.Tensor, w_in: torch.Tensor, b_in: Optional[torch.Tensor], w_out: torch.Tensor,
                 b_out: Optional[torch.Tensor] = None, *, activation: str = "gelu_tanh", gate: Optional[torch.Tensor] = None,
                 residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """residual + gate * (activation(x @ w_in.T + b_in) @ w_out.T + b_out).

    x is (..., C), w_in (F, C), b_in (F,), w_out (N, F), b_out (N,), gate (B, N) for an x of (B, ..., C), residual (..., N); all of
    them bf16 or all fp16.  Sums in fp32; the hidden rows are rounded to that type between the two products, and so are what the backward keeps of them
    and their gradient.  Differentiable in all seven (once)."""
    lib = current_lib()
    return lib.host.feed_forward(lib.host_library, x, w_in, b_in, w_out, b_out, _activation(activation), gate, residual)
