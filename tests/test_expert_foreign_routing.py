"""A routing of a caller's own whose offsets do not cover its places: a token gets nothing from a place that no expert has, whatever lies in memory that was never
written.  (torch fills what it allocates with NaN here.)"""
import contextlib

import pytest
import torch

import llsa_amd
from emu_util import emu_lib
from llsa_amd._lib import override_library_for_tests

BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def dev(request):
    with contextlib.ExitStack() as stack:
        if request.param == "cpu":
            stack.enter_context(override_library_for_tests(emu_lib()))
        yield torch.device(request.param)


@pytest.fixture
def no_numbers_in_new_memory():
    before = torch.are_deterministic_algorithms_enabled(), torch.is_deterministic_algorithms_warn_only_enabled(), torch.utils.deterministic.fill_uninitialized_memory
    torch.use_deterministic_algorithms(True, warn_only=True)
    torch.utils.deterministic.fill_uninitialized_memory = True
    yield
    torch.use_deterministic_algorithms(before[0], warn_only=before[1])
    torch.utils.deterministic.fill_uninitialized_memory = before[2]


def _runs(offsets, rows):
    """begin of the first run and end of the last: offsets are held to 0 .. rows and made not to fall"""
    o = offsets.cpu().long().clamp(0, rows)
    return int(o[0]), int(o.max())


def _check(dev, dtype, B, T, n, k, C, F, N, cut):
    g = torch.Generator().manual_seed(T + C)
    r = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).to(dtype).to(dev).requires_grad_()
    x, w_in, b_in, w_out, b_out = r(B, T, C), r(n, F, C, std=C ** -0.5), r(n, F), r(n, N, F, std=F ** -0.5), r(n, N)
    gate, residual, dout = r(B, N), r(B, T, N), r(B, T, N).detach()
    routing = llsa_amd.route_tokens(torch.randn(B, T, n, generator=g).to(dev), k)
    rows = B * T * k
    bad = cut(routing.offsets.clone(), rows)
    first, end = _runs(bad, rows)
    assert (first, end) != (0, rows)
    held = (routing.places >= first) & (routing.places < end)

    def run(places):
        weights = routing.weights.detach().requires_grad_()
        y = llsa_amd.expert_feed_forward(x, routing._replace(weights=weights, offsets=bad, places=places), w_in, b_in, w_out, b_out, gate=gate, residual=residual)
        return [y.detach()] + list(torch.autograd.grad(y, [x, weights, w_in, b_in, w_out, b_out, gate, residual], dout))

    got, want = run(routing.places), run(torch.where(held, routing.places, -torch.ones_like(routing.places)))
    names = ("y", "x", "weights", "w_in", "b_in", "w_out", "b_out", "gate", "residual")
    for name, a, b in zip(names, got, want):
        assert torch.isfinite(a).all() and torch.equal(a, b), name
    none = ~held.any(-1)
    if none.any():
        assert torch.equal(got[0][none], residual.detach()[none]) and not got[1][none].any()
    assert not got[2][~held].any()


CUTS = {"front": lambda o, rows: o.clamp(min=rows // 3), "back": lambda o, rows: o.clamp(max=rows // 2), "both": lambda o, rows: o.clamp(rows // 4, 3 * rows // 4), "none": lambda o, rows: o * 0 + rows,
        "negative": lambda o, rows: o - 5, "shifted": lambda o, rows: o + 7}


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("cut", list(CUTS))
def test_places_without_an_expert(dev, no_numbers_in_new_memory, cut, dtype):
    if dev.type == "cuda" or dtype == BF16:                   # (the emulation takes seconds for either)
        _check(dev, dtype, 2, 19, 4, 2, 24, 40, 24, CUTS[cut])
    if dev.type == "cuda" or dtype == FP16:
        _check(dev, dtype, 1, 33, 3, 1, 13, 21, 9, CUTS[cut])


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,n,k,C,F,N", [(1, 700, 4, 2, 136, 264, 136), (2, 8190, 8, 2, 264, 520, 264), (2, 20000, 8, 2, 384, 384, 384), (2, 20000, 8, 2, 320, 320, 320), (1, 40960, 2, 1, 1040, 2048, 1024)])
@pytest.mark.parametrize("cut", ["front", "back", "both", "none"])
def test_places_without_an_expert_in_larger_tiles(no_numbers_in_new_memory, cut, B, T, n, k, C, F, N):
    """The other kernels of the products: tiles of several sizes, weights in registers on the way to fp32."""
    _check(torch.device("cuda"), BF16, B, T, n, k, C, F, N, CUTS[cut])
