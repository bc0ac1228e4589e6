"""Slopes of the activations far from zero, where SiLU's is small but not nothing: dx of a layer of one weight of 1 is dout * act'(x)."""
import contextlib

import pytest
import torch

import llsa_amd
from emu_util import emu_lib
from llsa_amd._lib import override_library_for_tests

ACTS = {"silu": lambda t: t * torch.sigmoid(t), "gelu": lambda t: t * 0.5 * torch.erfc(-t / 2 ** 0.5),
        "gelu_tanh": lambda t: t * torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (t + 0.044715 * t ** 3))}


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def dev(request):
    with contextlib.ExitStack() as stack:
        if request.param == "cpu":
            stack.enter_context(override_library_for_tests(emu_lib()))
        yield torch.device(request.param)


@pytest.mark.parametrize("dtype,scale", [(torch.bfloat16, 1.0), (torch.bfloat16, 2.0 ** 40), (torch.float16, 2.0 ** 15)])
@pytest.mark.parametrize("act", list(ACTS))
def test_slopes_of_far_arguments(dev, act, dtype, scale):
    z = torch.tensor([-3e38, -1e4, -300.0, -129.0, -128.0, -127.0, -100.0, -80.0, -50.0, -30.0, -20.0, -17.0, 17.0, 20.0, 30.0, 100.0, 128.0, 1e4, 3e38]).clamp(-6e4, 6e4)
    x = z[:, None].to(dtype).to(dev).requires_grad_()
    one = torch.ones(1, 1, dtype=dtype, device=dev)
    dout = torch.full((len(z), 1), scale, dtype=dtype, device=dev)
    for feed in (False, True):                                # the slope on the way out of dx of a layer behind it, and in a pass of its own
        y = llsa_amd.feed_forward(x, one, None, one, activation=act) if feed else llsa_amd.linear(x, one, activation=act)
        d, = torch.autograd.grad(y, x, dout)
        v = x.detach().double().cpu().requires_grad_()
        ref, = torch.autograd.grad(ACTS[act](v).sum(), v)
        ref = torch.nan_to_num(ref) * scale                   # (0 * inf of the formula's own derivative at the farthest)
        u = torch.finfo(dtype).eps / 2
        # dz and dx rounded once each; in fp32 exp2 of an argument of up to 185 whose last step is 2^-17; a subnormal exponential counts as nothing (2^-126 of |z|)
        bound = 2 * u * (1 + u) * ref.abs() + 2.0 ** -15 * ref.abs() + 128 * scale * 2.0 ** -126 + (torch.finfo(dtype).tiny * u if dtype == torch.float16 else 0)
        off = (d.double().cpu() - ref).abs()
        assert (off <= bound).all(), (z[(off > bound)[:, 0]], d[(off > bound).to(dev)], ref[off > bound])
