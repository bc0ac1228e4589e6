"""layer_norm of fp32 rows whose values lie close together far from zero: what the mean is off by must stay small beside their spread, not beside their size."""
import contextlib

import pytest
import torch

import llsa_amd
from block_cases import E, within
from emu_util import emu_lib
from llsa_amd._lib import override_library_for_tests


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def dev(request):
    with contextlib.ExitStack() as stack:
        if request.param == "cpu":
            stack.enter_context(override_library_for_tests(emu_lib()))
        yield torch.device(request.param)


@pytest.mark.parametrize("value,C", [(0.1, 777), (3.7, 384), (1234.567, 777), (-0.3, 5), (1e-30, 333), (7.7e30, 1000), (0.1, 8191), (0.7, 2048)])
def test_rows_of_one_value(dev, value, C):
    """Nothing is left of them but the bias and the shift, however small eps is."""
    x = torch.full((2, 3, C), value, device=dev).requires_grad_()
    w, b, sc, sh = (torch.randn(s, generator=torch.Generator().manual_seed(i)).to(dev) for i, s in enumerate(((C,), (C,), (2, C), (2, C))))
    y = llsa_amd.layer_norm(x, eps=1e-12)
    assert not y.any()
    dx, = torch.autograd.grad(y, x, torch.randn(x.shape, generator=torch.Generator().manual_seed(9)).to(dev))
    assert torch.isfinite(dx).all()
    y = llsa_amd.layer_norm(x, w, b, scale=sc, shift=sh, eps=1e-12)
    want = torch.addcmul(sh[:, None].double(), b.double(), 1 + sc[:, None].double()).expand_as(y)
    assert ((y.double() - want).abs() <= 2 * E * ((b * (1 + sc[:, None])).abs() + want.abs())).all()


@pytest.mark.parametrize("offset,spread", [(1000.0, 1e-2), (-300.0, 1.0), (1e5, 3.0), (0.3, 1.0)])
@pytest.mark.parametrize("C", [777, 384, 40, 2049, 8192])
def test_rows_far_from_zero(dev, C, offset, spread):
    g = torch.Generator().manual_seed(C)
    r = lambda *s: torch.randn(*s, generator=g)
    x, w, dout = (r(2, 3, C) * spread + offset), r(C), r(2, 3, C)
    leaves = [x.to(dev).requires_grad_(), w.to(dev).requires_grad_()]
    y = llsa_amd.layer_norm(*leaves, eps=1e-12)
    dx, dw = torch.autograd.grad(y, leaves, dout.to(dev))
    x64, w64, d64 = x.double().requires_grad_(), w.double().requires_grad_(), dout.double()
    d = x64 - x64.mean(-1, keepdim=True)
    rstd = (d.square().mean(-1, keepdim=True) + 1e-12).rsqrt()
    h = d * rstd
    ref = h * w64
    rx, rw = torch.autograd.grad(ref, [x64, w64], d64)
    with torch.no_grad():
        d, rstd, h, w64, ref = (t.detach() for t in (d, rstd, h, w64, ref))
        c = 48 * E                                            # a lane adds up to 32 values, then up to 10 halvings
        # the first mean is off by c |x|; differences from it are exact (values and mean within a factor of two) or off by E of them; their mean by c of theirs
        far = d.abs() + c * x.double().abs().mean(-1, keepdim=True)
        dh = rstd * (2 * E * far + c * far.mean(-1, keepdim=True)) + 3 * c * h.abs()
        within(y.detach().cpu(), ref, (dh + 6 * E * h.abs()) * w64.abs(), "y")
        gw = d64 * w64
        gh, dgh = (gw * h).abs().mean(-1, keepdim=True), (gw.abs() * dh).mean(-1, keepdim=True)
        bound = rstd * (8 * E * gw.abs() + c * gw.abs().mean(-1, keepdim=True) + h.abs() * (c * gh + dgh) + dh * gh + 4 * E * gh * h.abs())
        within(dx.cpu(), rx, bound + 4 * c * rx.abs(), "dx")
        within(dw.cpu(), rw, (d64.abs() * dh + 32 * E * (d64 * h).abs()).sum((0, 1)), "dweight")
