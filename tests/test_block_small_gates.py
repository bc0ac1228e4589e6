"""Gradients of gated layers in fp16 whose gates and weights lie far from 1, as those of an adaLN-zero block do while it trains: on samples long enough
that the backward puts the gate into the weights and on shorter ones alike.  dout comes scaled, as a loss scaler leaves it."""
import contextlib

import pytest
import torch

import llsa_amd
from block_cases import E, half_step, least, within
from emu_util import emu_lib
from llsa_amd._lib import override_library_for_tests

FP16 = torch.float16
U, LO = half_step(FP16), least(FP16)


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def dev(request):
    with contextlib.ExitStack() as stack:
        if request.param == "cpu":
            stack.enter_context(override_library_for_tests(emu_lib()))
        yield torch.device(request.param)


def _check_dx(dev, T, K, N, gate, weight=None, dout_scale=1024.0, seed=0):
    g = torch.Generator().manual_seed(seed)
    B = gate.shape[0]
    r = lambda *s: torch.randn(*s, generator=g)
    x, w = r(B, T, K).to(FP16), (r(N, K) * K ** -0.5).to(FP16) if weight is None else weight.to(FP16)
    gate, dout = gate.to(FP16), (r(B, T, N) * dout_scale).to(FP16)
    leaf = x.to(dev).requires_grad_()
    y = llsa_amd.linear(leaf, w.to(dev), gate=gate.to(dev))
    dx, = torch.autograd.grad(y, leaf, dout.to(dev))
    d, ga, w64 = dout.double(), gate.double()[:, None], w.double()
    ref, mag = (d * ga) @ w64, (d.abs() * ga.abs()) @ w64.abs()
    if T >= 2 * K:
        # gate * w rounded once; what lies 2^-28 below the largest of its column and sample by half a step of that size, 2^-39 of the largest
        rounded = U * mag + d.abs().sum(-1, keepdim=True) * 2.0 ** -39 * (ga[:, 0].abs()[:, :, None] * w64.abs()[None]).amax(1)[:, None]
    else:
        rounded = U * mag + LO * w64.abs().sum(0)             # dout * gate rounded once
    within(dx.cpu(), ref, rounded * (1 + 2 * U) + (N + 32) * E * mag + U * ref.abs() + LO, "dx")


@pytest.mark.parametrize("T", [95, 96])                       # 2 K = 96: the gate in the rows, and in the weights
@pytest.mark.parametrize("size", [1e-2, 1e-4, 1e-5, 1e-6])
def test_linear_dx_of_small_gates(dev, T, size):
    _check_dx(dev, T, 48, 40, torch.randn(2, 40, generator=torch.Generator().manual_seed(1)) * size)


def test_linear_dx_of_gates_of_many_sizes(dev):
    """Samples of small, ordinary, vanishing and large gates beside each other, and a sample with all of them."""
    n = torch.randn(6, 40, generator=torch.Generator().manual_seed(2))
    gates = n * torch.tensor([1e-6, 1.0, 0.0, 300.0, 1e-4, 1.0])[:, None]
    gates[5, ::3] *= 1e-5
    _check_dx(dev, 70, 24, 40, gates, dout_scale=1.0)
    _check_dx(dev, 70, 21, 35, gates[:, :35], dout_scale=1.0)


def test_linear_dx_of_weights_of_many_sizes(dev):
    """gate * w beyond the largest fp16, and weights that are small themselves."""
    g = torch.Generator().manual_seed(3)
    w = torch.randn(40, 24, generator=g) * torch.logspace(-4, 3, 24)
    _check_dx(dev, 50, 24, 40, torch.randn(2, 40, generator=g) * torch.tensor([[1e-5], [100.0]]), w, dout_scale=2.0 ** -6)


def test_linear_dx_where_a_weight_is_not_finite(dev):
    """An infinity or a NaN stays in the columns that read it."""
    g = torch.Generator().manual_seed(4)
    x, w, gate = torch.randn(2, 50, 24, generator=g).to(FP16), torch.randn(40, 24, generator=g).to(FP16), (torch.randn(2, 40, generator=g) * 1e-3).to(FP16)
    dout = torch.randn(2, 50, 40, generator=g).to(FP16).to(dev)

    def dx(w):
        leaf = x.to(dev).requires_grad_()
        return torch.autograd.grad(llsa_amd.linear(leaf, w.to(dev), gate=gate.to(dev)), leaf, dout)[0].cpu()

    plain = dx(w)
    for bad in (float("inf"), float("nan")):
        v = w.clone()
        v[7, 5] = bad
        got = dx(v)
        assert not torch.isfinite(got[..., 5]).any()
        got[..., 5] = plain[..., 5]
        assert torch.equal(got, plain)


def _check_ffn(dev, B, T, C, F, size, act="gelu_tanh"):
    """Every rounding of 2^-12 in the mean (half a step is 2^-11 at most); dx, dW_in and db_in come through four at most (gate * w, z, dz, their own): 2^-11 as
    a root mean square.  Twice that, as their sums also take in the roundings of the products in fp32."""
    g = torch.Generator().manual_seed(C)
    r = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).to(FP16)
    t = [r(B, T, C), r(F, C, std=C ** -0.5), r(F, std=0.3), r(C, F, std=F ** -0.5), r(C, std=0.3), r(B, C, std=size)]
    dout = r(B, T, C, std=2.0 ** 10)
    leaves = [v.to(dev).requires_grad_() for v in t]
    got = torch.autograd.grad(llsa_amd.feed_forward(*leaves[:5], activation=act, gate=leaves[5]), leaves, dout.to(dev))
    x, w1, b1, w2, b2, gate = (v.double().to(dev).requires_grad_() for v in t)
    z = x.reshape(-1, C) @ w1.t() + b1
    h = z * torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (z + 0.044715 * z ** 3))
    y = gate[:, None] * (h @ w2.t() + b2).view(B, T, C)
    ref = torch.autograd.grad(y, [x, w1, b1, w2, b2, gate], dout.double().to(dev))
    for name, a, b in zip(("x", "w_in", "b_in", "w_out", "b_out", "gate"), got, ref):
        a = a.double()
        # (the gate's gradient is not made smaller by its gate: sums over 3301 rows of dout around 2^10 are of the order of 3301^0.5 2^10 = 58833, beside fp16's
        # largest value, 65504.  Beyond 65520 an infinity is what they round to; within a rounding error of that, either.)
        far = b.abs() > 65504
        assert torch.isfinite(a[~far]).all() and (a[b.abs() > 65520 * (1 + 2.0 ** -9)] * b[b.abs() > 65520 * (1 + 2.0 ** -9)] == torch.inf).all(), name
        off = (a - b)[~far].norm() / b[~far].norm()
        assert off <= 2.0 ** -10, (name, off.item())


@pytest.mark.parametrize("T", [143, 144])                     # 2 F = 144
@pytest.mark.parametrize("size", [1e-4, 1e-6])
def test_feed_forward_of_small_gates(dev, T, size):
    _check_ffn(dev, 2, T, 40, 72, size)


@pytest.mark.gpu
@pytest.mark.parametrize("T,K,N", [(3301, 1536, 384), (4099, 1600, 320), (2070, 1032, 264), (1100, 136, 520)])
def test_large_linear_dx_of_small_gates(T, K, N):
    """Each kernel of dx with weights of each sample: in registers, and the tiles."""
    gates = torch.randn(3, N, generator=torch.Generator().manual_seed(5)) * torch.tensor([1e-6, 1e-4, 1.0])[:, None]
    _check_dx(torch.device("cuda"), T, K, N, gates)


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,C,F", [(3, 3301, 384, 1536), (2, 2085, 264, 1040)])
def test_large_feed_forward_of_small_gates(B, T, C, F):
    _check_ffn(torch.device("cuda"), B, T, C, F, 1e-5)


def test_c_calls_check_scales():
    """Gated weights in fp16 need room for their scales, and dx takes scales with such weights alone; nothing is launched."""
    import ctypes as C
    from llsa_amd._lib import LIB_PATH, Lib, LinearArgs
    lib = Lib(LIB_PATH)
    bad = lambda fn, a: fn(C.byref(a), None) != 0 and b"scales" in lib.last_error_string()
    a = LinearArgs()
    a.M, a.N, a.K, a.dtype, a.per_sample = 8, 8, 8, 2, 4
    a.w = a.gate = a.out = a.dz = 1 << 20
    a.ldw = a.ldo = a.lddz = a.s_gate = 8
    assert bad(lib.linear_gate_rows, a)
    a.scales = 8 + (1 << 20)
    assert bad(lib.linear_gate_rows, a)
    assert bad(lib.linear_dx, a)                              # (one set of weights for all rows)
    a.s_w = 64
    assert bad(lib.linear_dx, a)                              # (not aligned)
    a.scales, a.dtype = 1 << 20, 0
    assert bad(lib.linear_dx, a)                              # (bf16)
