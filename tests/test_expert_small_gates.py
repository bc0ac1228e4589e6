"""Gradients of the routed block in fp16 whose gates lie far from 1, as those of an adaLN-zero block do while it trains.  dout comes scaled, as a loss scaler leaves it."""
import contextlib

import pytest
import torch

import llsa_amd
from emu_util import emu_lib
from llsa_amd._lib import override_library_for_tests

FP16 = torch.float16


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def dev(request):
    with contextlib.ExitStack() as stack:
        if request.param == "cpu":
            stack.enter_context(override_library_for_tests(emu_lib()))
        yield torch.device(request.param)


@pytest.mark.parametrize("size", [1e-3, 1e-4, 1e-6])
def test_small_gates(dev, size):
    """Roundings of 2^-12 in the mean (half a step is 2^-11 at most); dx, dW_in and db_in come through three at most (weight * gate * dout, dz, their own): below 2^-11 as
    a root mean square.  Twice that, as their sums also take in the roundings of the products in fp32."""
    g = torch.Generator().manual_seed(1)
    r = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).to(FP16)
    B, T, n, k, C, F = 2, 70, 3, 2, 40, 72
    t = [r(B, T, C), r(n, F, C, std=C ** -0.5), r(n, F, std=0.3), r(n, C, F, std=F ** -0.5), r(n, C, std=0.3), r(B, C, std=size)]
    logits, dout = r(B, T, n), r(B, T, C, std=2.0 ** 10)
    leaves = [v.to(dev).requires_grad_() for v in t]
    routing = llsa_amd.route_tokens(logits.to(dev), k)
    weights = routing.weights.requires_grad_()
    y = llsa_amd.expert_feed_forward(leaves[0], routing, *leaves[1:5], gate=leaves[5])
    got = torch.autograd.grad(y, leaves + [weights], dout.to(dev))
    x, w1, b1, w2, b2, gate, w = v64 = [v.detach().double().cpu().requires_grad_() for v in t + [weights]]
    z = torch.einsum("btc,efc->btef", x, w1) + b1
    h = z * torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (z + 0.044715 * z ** 3))
    each = torch.einsum("btef,ecf->btec", h, w2) + b2
    y64 = gate[:, None] * (w[..., None] * each.gather(2, routing.experts.cpu().long()[..., None].expand(B, T, k, C))).sum(2)
    for name, a, b in zip(("x", "w_in", "b_in", "w_out", "b_out", "gate", "weights"), got, torch.autograd.grad(y64, v64, dout.double())):
        off = (a.double().cpu() - b).norm() / b.norm()
        assert torch.isfinite(a).all() and off <= 2.0 ** -10, (name, off.item())
