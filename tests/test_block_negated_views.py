"""Tensors that torch holds with their sign flipped (the imaginary part of a conjugate is a view whose memory has the other sign): what layer_norm, linear and
feed_forward read is their value."""
import contextlib

import pytest
import torch

import llsa_amd
from emu_util import emu_lib
from llsa_amd._lib import override_library_for_tests


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def dev(request):
    with contextlib.ExitStack() as stack:
        if request.param == "cpu":
            stack.enter_context(override_library_for_tests(emu_lib()))
        yield torch.device(request.param)


def _inputs(op, dev):
    g = torch.Generator().manual_seed(0)
    r = lambda *s: (torch.randn(*s, generator=g) * 0.5).to(torch.float32 if op == "norm" else torch.float16).to(dev)
    B, T, C, F = 2, 9, 24, 40
    if op == "norm":
        return {"x": r(B, T, C), "weight": r(C), "bias": r(C), "scale": r(B, C), "shift": r(B, C)}
    if op == "linear":
        return {"x": r(B, T, C), "weight": r(F, C), "bias": r(F), "gate": r(B, F), "residual": r(B, T, F)}
    return {"x": r(B, T, C), "w_in": r(F, C), "b_in": r(F), "w_out": r(C, F), "b_out": r(C), "gate": r(B, C), "residual": r(B, T, C)}


def _call(op, t):
    if op == "norm":
        return llsa_amd.layer_norm(t["x"], t["weight"], t["bias"], scale=t["scale"], shift=t["shift"])
    if op == "linear":
        return llsa_amd.linear(t["x"], t["weight"], t["bias"], activation="silu", gate=t["gate"], residual=t["residual"])
    return llsa_amd.feed_forward(t["x"], t["w_in"], t["b_in"], t["w_out"], t["b_out"], gate=t["gate"], residual=t["residual"])


@pytest.mark.parametrize("op", ["norm", "linear", "ffn"])
@pytest.mark.parametrize("adjacent", [False, True])
def test_negated_views(dev, op, adjacent):
    plain = _inputs(op, dev)
    leaves = {n: v.clone().requires_grad_() for n, v in plain.items()}
    y = _call(op, leaves)
    dout = torch.randn(y.shape, generator=torch.Generator().manual_seed(1)).to(y.dtype).to(dev)
    want = [y.detach()] + list(torch.autograd.grad(y, list(leaves.values()), dout))

    def negated(v):
        w = torch._neg_view(-v) if adjacent else torch.complex(torch.zeros_like(v, dtype=torch.float32), -v.float()).to(torch.complex64 if v.dtype == torch.float32 else torch.complex32).conj().imag
        assert w.is_neg() and torch.equal(w, v)
        return w

    for name in list(plain) + ["dout"]:
        t = {n: v.clone().requires_grad_() for n, v in plain.items()}
        if name != "dout":
            t[name] = negated(plain[name]).requires_grad_()
        got = _call(op, t)
        got = [got.detach()] + list(torch.autograd.grad(got, list(t.values()), negated(dout) if name == "dout" else dout))
        for i, (a, b) in enumerate(zip(want, got)):
            assert torch.equal(a, b), (name, i)
