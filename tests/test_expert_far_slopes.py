"""Slopes of the activations as grouped_linear and expert_feed_forward keep them for their backward, down to the smallest: one row, one weight of 1, so that dx is
dout * act'(x), and a bias whose gradient is the sum of a few of those."""
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


def _slopes(act, x):
    v = x.detach().double().cpu().requires_grad_()
    return torch.nan_to_num(torch.autograd.grad(ACTS[act](v).sum(), v)[0])      # (0 * inf of the formula's own derivative at the farthest)


def _kept(act, s):
    """What a kept slope may be off by: half a step of 2^-14; of negative ones above -2^-4 half a step of ten bits and, above -2^-19, of seven.  Before it is kept: exp2 of an
    argument of up to 185, whose last step is 2^-17, and a few operations of fp32 next to 1; the normal distribution's tail is a rational approximation whose share of z's
    bell is off by up to 2.2e-4 < 2^-12 of the slope for every z below -3, and by 1.5e-7 / 2 anywhere."""
    size = s.abs()
    small = (s < 0) & (size < 2.0 ** -4 * (1 + 2.0 ** -10))
    kept = torch.where(small, torch.where(size < 2.0 ** -19 * (1 + 2.0 ** -7), 2.0 ** -8, 2.0 ** -11) * size, torch.full_like(s, 2.0 ** -15))
    made = (2.0 ** -15 + (2.0 ** -12 if act == "gelu" else 0)) * size + torch.where(small & (size < 2.0 ** -7), 0.0, 2.0 ** -20)
    return kept * (1 + 2.0 ** -11) + made + 128 * 2.0 ** -126


def _outputs(form, x, act, bias=None):
    one = torch.ones(1, 1, 1, dtype=x.dtype, device=x.device)
    if form == "grouped":
        return llsa_amd.grouped_linear(x, one, torch.tensor([0, x.shape[0]], dtype=torch.int32, device=x.device), bias, activation=act)
    return llsa_amd.expert_feed_forward(x, llsa_amd.route_tokens(torch.zeros_like(x), 1), one, bias, one, activation=act)


@pytest.mark.parametrize("dtype,scale", [(torch.bfloat16, 1.0), (torch.bfloat16, 2.0 ** 40), (torch.float16, 64.0), (torch.float16, 2.0 ** 15)])
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("form", ["grouped", "block"])
def test_slopes(dev, act, dtype, scale, form):
    far = [-3e38, -1e4, -300.0, -129.0, -128.0, -127.0, -100.0, -80.0, -50.0, -30.0, 12.0, 17.0, 30.0, 128.0, 1e4, 3e38]
    z = torch.cat([torch.tensor(far), torch.linspace(-24, 6, 241)]).clamp(-6e4, 6e4)
    x = z[:, None].to(dtype).to(dev).requires_grad_()
    d, = torch.autograd.grad(_outputs(form, x, act), x, torch.full_like(x, scale))
    s = _slopes(act, x)
    ref, u = s * scale, torch.finfo(dtype).eps / 2
    # dz and dx rounded once each
    bound = scale * _kept(act, s) * (1 + u) ** 2 + 2 * u * (1 + u) * ref.abs() + (2 * torch.finfo(dtype).tiny * u if dtype == torch.float16 else 0)
    off = (d.double().cpu() - ref).abs()
    assert (off <= bound).all(), (x[(off > bound).to(dev)], d[(off > bound).to(dev)], ref[off > bound])


@pytest.mark.parametrize("act,z", [("gelu", -5.0), ("gelu_tanh", -5.0), ("silu", -14.0), ("silu", -11.0)])
@pytest.mark.parametrize("form", ["grouped", "block"])
def test_a_bias_far_below_zero(dev, act, z, form):
    """Eight rows that all lie there: the unit's gradient is what leads out again."""
    x = (z + 0.125 * torch.arange(8.0)[:, None] / 8).half().to(dev).requires_grad_()
    bias = torch.zeros(1, 1, dtype=torch.float16, device=dev).requires_grad_()
    d, = torch.autograd.grad(_outputs(form, x, act, bias), bias, torch.full_like(x, 64.0))
    s, u = _slopes(act, x), 2.0 ** -11
    ref = 64 * s.sum()
    assert ref != 0
    assert (d.double().cpu() - ref).abs() <= 64 * _kept(act, s).sum() * (1 + u) ** 2 + 2 * u * (1 + u) * ref.abs() + 9 * 2.0 ** -25


def test_no_number_stays_one(dev):
    """The slope of a NaN is a NaN; those of the rows beside it are what they were."""
    for form in ("grouped", "block"):
        x = torch.linspace(-9, 2, 16)[:, None].to(torch.bfloat16).to(dev)
        bad = x.clone()
        bad[5] = float("nan")
        got = []
        for v in (x, bad):
            v = v.requires_grad_()
            got.append(torch.autograd.grad(_outputs(form, v, "silu"), v, torch.ones_like(v))[0])
        keep = [i for i in range(16) if i != 5]
        assert got[1][5].isnan().all() and torch.equal(got[0][keep], got[1][keep])
