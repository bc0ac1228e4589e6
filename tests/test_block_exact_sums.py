"""Gradients that can be held to equality or to the roundings of their own sums: inputs that share memory, differences of an operator that is linear in each of its inputs, and the
gradients behind the scores of the small DiT where every block is selected."""
import contextlib

import pytest
import torch

import llsa_amd
import test_block_in_dit
from emu_util import emu_lib
from llsa_amd._lib import override_library_for_tests
from llsa_amd.caller import dit as D

BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def dev(request):
    with contextlib.ExitStack() as stack:
        if request.param == "cpu":
            stack.enter_context(override_library_for_tests(emu_lib()))
        yield torch.device(request.param)


def _whole(g, dev, *shape, low=-1, high=1):
    return torch.randint(low, high + 1, shape, generator=g).to(FP16).to(dev)


def _linear(t):
    return llsa_amd.linear(t["x"], t["weight"], t["bias"], gate=t["gate"], residual=t["residual"])


@pytest.mark.parametrize("B,T", [(3, 5), (1, 15), (2, 50)])
def test_expanded_inputs_exactly(dev, B, T):
    """Whole numbers: every sum is below 2^11, where fp16 holds them all.  Rows: at most 40 * 2 * 100; but weights, gates and dout of -1, 0, 1 (gate 1, 2), each zero
    one time in three: the largest here are below 1000, which the test checks."""
    g = torch.Generator().manual_seed(T)
    K, N = 24, 40
    leaf = {"x": _whole(g, dev, 1, 1, K), "weight": _whole(g, dev, N, K), "bias": _whole(g, dev, N), "gate": _whole(g, dev, 1, N, low=1, high=2), "residual": _whole(g, dev, 1, 1, N)}
    leaf = {n: v.requires_grad_() for n, v in leaf.items()}
    wide = {n: v.expand(B, T, v.shape[-1]) if v.dim() == 3 else v.expand(B, N) if n == "gate" else v for n, v in leaf.items()}
    dout = _whole(g, dev, B, T, N)
    got = torch.autograd.grad(_linear(wide), list(leaf.values()), dout)
    ref = {n: v.detach().double().requires_grad_() for n, v in leaf.items()}
    w = {n: v.expand(B, T, v.shape[-1]) if v.dim() == 3 else v.expand(B, N) if n == "gate" else v for n, v in ref.items()}
    y = w["residual"] + w["gate"][:, None] * (w["x"] @ w["weight"].t() + w["bias"])
    for n, a, b in zip(leaf, got, torch.autograd.grad(y, list(ref.values()), dout.double())):
        assert b.abs().max() < 2048 and torch.equal(a.double(), b), n


@pytest.mark.parametrize("op", ["norm", "ffn"])
def test_expanded_inputs_within_their_sums(dev, op):
    """The gradient of a shared row is the sum of the rows' gradients, which autograd adds in the gradient's type: 15 roundings of half a step of sums no larger than that
    of the magnitudes."""
    from test_block_contract import _call, _inputs
    base = _inputs(op, dev, B=1, T=1)
    leaf = {n: v.detach().requires_grad_() for n, v in base.items()}
    wide = {n: v.expand(3, 5, v.shape[-1]) if v.dim() == 3 else v.expand(3, v.shape[-1]) if n in ("gate", "scale", "shift") else v for n, v in leaf.items()}
    copied = {n: v.detach().contiguous().requires_grad_() for n, v in wide.items()}
    y, z = _call(op, wide), _call(op, copied)
    dout = torch.randn(y.shape, generator=torch.Generator().manual_seed(3)).to(BF16).to(dev)
    each = torch.autograd.grad(z, list(copied.values()), dout)
    for n, a, b in zip(leaf, torch.autograd.grad(y, list(leaf.values()), dout), each):
        if b.shape == a.shape:
            assert torch.equal(a, b), n
        else:
            b = b.double()
            assert ((a.double() - b.sum_to_size(a.shape)).abs() <= 15 * 2.0 ** -8 * b.abs().sum_to_size(a.shape)).all(), n


@pytest.mark.parametrize("T", [9, 50])
def test_linear_against_differences_exactly(dev, T):
    """linear without an activation is linear in each input: with whole numbers the difference of two of its outputs along a step is the gradient's product with that step, to the
    last bit (|y| below 2 * 2 * 17 + 2, gradients below 2^11)."""
    g = torch.Generator().manual_seed(T)
    B, K, N = 2, 16, 24
    t = {"x": _whole(g, dev, B, T, K), "weight": _whole(g, dev, N, K), "bias": _whole(g, dev, N), "gate": _whole(g, dev, B, N, low=1, high=2), "residual": _whole(g, dev, B, T, N)}
    dout = _whole(g, dev, B, T, N)
    leaves = {n: v.clone().requires_grad_() for n, v in t.items()}
    grads = dict(zip(t, torch.autograd.grad(_linear(leaves), list(leaves.values()), dout)))
    for n, v in t.items():
        for first in range(5):
            step = torch.zeros_like(v)
            step.view(-1)[first::5] = 1
            change = ((_linear({**t, n: v + step}).double() - _linear(t).double()) * dout.double()).sum()
            assert change == (grads[n].double() * step.double()).sum(), (n, first)


def _compare_all(dev, B, **cfg):
    """The step of test_block_in_dit with every block selected: the gradients of q, k and their norms too are off by the roundings alone, 5 % as there.  A bias' gradient is
    the sum over rows whose entries in dW's columns are of order 1, so its error is one column's of dW: 5 % of dW / C^0.5, beside its own 5 %."""
    torch.manual_seed(3)
    plain = D.PixelDiT(**cfg).to(dev)
    fused = D.PixelDiT(fused_layers=True, **cfg).to(dev)
    fused.load_state_dict(plain.state_dict())
    g = torch.Generator().manual_seed(0)
    side = cfg["sample_size"]
    batch = [t.to(dev) for t in (torch.randn(B, 3, side, side, generator=g).clamp(-1, 1), torch.randn(B, 3, side, side, generator=g), torch.randint(0, 1000, (B,), generator=g))]
    (_, grads), (_, ref) = test_block_in_dit._step(fused, batch), test_block_in_dit._step(plain, batch)
    seen = 0
    for n, r in ref.items():
        if not any(t in n for t in ("to_q.", "to_k.", "norm_q_weight", "norm_k_weight")):
            continue
        seen += 1
        size = r.norm()
        if n.endswith("bias"):
            size = size + ref[n[:-4] + "weight"].norm() / r.numel() ** 0.5
        assert size > 0 and (grads[n] - r).norm() <= 5e-2 * size, (n, ((grads[n] - r).norm() / size).item())
    assert seen == 6 * cfg["num_layers"]


def test_scores_gradients_in_dit(dev):
    _compare_all(dev, 1, num_attention_heads=1, num_layers=1, sample_size=32, levels=1, sparse_topk=64)


@pytest.mark.gpu
def test_scores_gradients_in_a_larger_dit():
    _compare_all(torch.device("cuda"), 3, num_attention_heads=3, num_layers=2, sample_size=32, levels=1, sparse_topk=64)
