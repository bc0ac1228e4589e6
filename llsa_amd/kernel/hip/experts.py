"""Rows that choose their weights: a router, products with an expert's weights for each run of rows, and the feed-forward block made of both."""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from ..._lib import current_lib
from .linear import _activation


class Routing(NamedTuple):
    """Which experts every token goes to, as route_tokens returns it.  A slot is token * experts_per_token + choice.

    weights  (..., k) fp32     of the chosen experts, 0 where there is none
    experts  (..., k) int32    or -1
    order    (tokens * k) int32   the slots sorted by expert and then by number, -1 behind the last
    offsets  (experts + 1) int32  places offsets[e] .. offsets[e + 1] - 1 of order are expert e's
    places   (..., k) int32    of every slot in order, or -1"""
    weights: torch.Tensor
    experts: torch.Tensor
    order: torch.Tensor
    offsets: torch.Tensor
    places: torch.Tensor


def route_tokens(logits: torch.Tensor, experts_per_token: int, *, normalize: bool = True) -> Routing:
    """The `experts_per_token` experts with the largest logits of every token, and the order in which the experts' products take the rows.

    logits is (..., experts) of bf16, fp16 or fp32, 1 to 256 experts, of which a token takes 1 to 16.  Equal logits go to the lowest index; -inf is never chosen
    (a token of nothing but -inf, padding, goes nowhere, and one with too few others to fewer); a NaN counts as the largest number.  weights = exp(logit - max) / sum, over the
    chosen ones (normalize) or over all of the token's, in fp32 and differentiable (once); the backward keeps logits and experts.  A token with a NaN or an infinite
    logit has weights of NaN.  Nothing is copied to the host; the results do not depend on the order of atomics."""
    lib = current_lib()
    return Routing(*lib.host.route_tokens(lib.host_library, logits, experts_per_token, normalize))


def grouped_linear(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor, bias: Optional[torch.Tensor] = None, *, activation: Optional[str] = None) -> torch.Tensor:
    """activation(x @ weight[e].T + bias[e]) for rows offsets[e] .. offsets[e + 1] - 1 of x.

    x is (rows, K), weight (experts, N, K), bias (experts, N), all bf16 or all fp16; offsets (experts + 1) int32 on x's device, which stays there: experts may have any
    number of rows, none among them, and rows that no expert has (in front of the first or behind the last) come out as zeros, as does their gradient.  Offsets are
    held to 0 .. rows and made not to fall.  1 to 256 experts.  activation: None, "silu", "gelu" (erf) or "gelu_tanh".  Sums in fp32; besides the results, the backward rounds the
    gradient behind the activation, whose slopes it keeps in 16 bits: off by up to 2^-15, and where they are small, far below zero, by up to a 2^-8th part of themselves
    (below 2^-19, a 2^-11th above).  Differentiable in x, weight and bias (once)."""
    lib = current_lib()
    return lib.host.grouped_linear(lib.host_library, x, weight, offsets, bias, _activation(activation))


def expert_feed_forward(x: torch.Tensor, routing: Routing, w_in: torch.Tensor, b_in: Optional[torch.Tensor], w_out: torch.Tensor, b_out: Optional[torch.Tensor] = None, *,
                        activation: str = "gelu_tanh", gate: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """residual + gate * sum over a token's experts e of weight_e * (activation(x @ w_in[e].T + b_in[e]) @ w_out[e].T + b_out[e]).

    x is (..., C), routing what route_tokens returned for logits (..., experts) of the same tokens, w_in (experts, F, C), b_in (experts, F), w_out (experts, N, F),
    b_out (experts, N), gate (B, N) for an x of (B, ..., C), residual (..., N); all but the routing bf16 or all fp16.  A token without an expert gets its residual, and
    nothing comes from places in front of offsets[0] or behind the last of the offsets.
    Sums in fp32, each expert's result among them; the hidden rows and the gradients of either product's result (weight * gate * its own) are rounded to that type,
    which in fp16 wants a scaled loss, and the backward keeps the activation's slopes in
    16 bits as grouped_linear does.  Differentiable in x, routing.weights, the weights and biases, gate and residual (once)."""
    lib = current_lib()
    weights, experts, order, offsets, places = routing
    return lib.host.expert_feed_forward(lib.host_library, x, weights, experts, order, offsets, places, w_in, b_in, w_out, b_out, _activation(activation), gate, residual)
