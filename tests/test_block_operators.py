"""layer_norm, linear and feed_forward against their formulas in 64 bits: forward and every gradient, element by element, within bounds that
follow from the roundings.  On the CPU through the x86 build of the kernels, on the GPU through the library, where larger sizes run too."""
import contextlib

import pytest
import torch

import llsa_amd
from block_cases import check_layers, check_norm
from emu_util import emu_lib
from llsa_amd._lib import override_library_for_tests

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def dev(request):
    with contextlib.ExitStack() as stack:
        if request.param == "cpu":
            stack.enter_context(override_library_for_tests(emu_lib()))
        yield torch.device(request.param)


class Draw:
    def __init__(self, dev, dtype, seed):
        self.g, self.dev, self.dtype = torch.Generator().manual_seed(seed), dev, dtype

    def __call__(self, *shape, std=1.0, mean=0.0, dtype=None):
        return (torch.randn(*shape, generator=self.g) * std + mean).to(dtype or self.dtype).to(self.dev).requires_grad_()


def norm_inputs(dev, dtype, shape, affine, mod, vector=None, seed=0):
    r, C, B = Draw(dev, dtype, seed), shape[-1], shape[0]
    v = dict(dtype=vector or dtype)
    x = r(*shape, mean=0.5)
    w, b = (r(C, std=0.2, mean=1.0, **v), r(C, std=0.2, **v)) if affine else (None, None)
    sc, sh = (r(B, C, std=0.3, **v), r(B, C, std=0.3, **v)) if mod else (None, None)
    return x, w, b, sc, sh, r(*shape).detach()


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("shape,affine,mod", [((2, 5, 384), False, True), ((3, 7, 40), True, False), ((1, 1, 8), True, True), ((2, 3, 13), True, True), ((4, 1), False, False),
                                              ((2, 2, 3, 130), False, True), ((9, 520), True, False)])
def test_norm(dev, dtype, shape, affine, mod):
    check_norm(*norm_inputs(dev, dtype, shape, affine, mod))


@pytest.mark.parametrize("C", [128, 256, 400, 512, 640, 1024, 1500, 2048, 2304, 4096, 6000, 8192])
def test_norm_channels(dev, C):
    """Every number of lanes and pieces a row is held in."""
    check_norm(*norm_inputs(dev, BF16, (2, 3, C), True, True, seed=C))


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_norm_vectors_in_32_bits(dev, dtype):
    check_norm(*norm_inputs(dev, dtype, (2, 9, 72), True, True, vector=FP32))


def layer_inputs(dev, dtype, B, T, K, N, bias, gate, residual, seed=0):
    r = Draw(dev, dtype, seed)
    x, w = r(B, T, K), r(N, K, std=K ** -0.5)
    return (x, w, r(N, std=0.3) if bias else None, r(B, N, std=0.3, mean=0.5) if gate else None, r(B, T, N) if residual else None, r(B, T, N).detach())


def check_linear(dev, dtype, B, T, K, N, act=None, bias=True, gate=False, residual=False, seed=0):
    x, w, b, g, res, dout = layer_inputs(dev, dtype, B, T, K, N, bias, gate, residual, seed)
    return check_layers(x, [(w, b, act)], g, res, dout, lambda: llsa_amd.linear(x, w, b, activation=act, gate=g, residual=res))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("act", [None, "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("gate,residual", [(False, False), (True, True)])
def test_linear(dev, dtype, act, gate, residual):
    check_linear(dev, dtype, 2, 19, 72, 88, act, gate=gate, residual=residual)


@pytest.mark.parametrize("B,T,K,N", [(1, 1, 1, 1), (3, 1, 8, 8), (1, 7, 5, 3), (2, 33, 64, 64), (1, 65, 130, 67), (2, 64, 200, 129), (1, 130, 33, 200)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_linear_sizes(dev, dtype, B, T, K, N):
    check_linear(dev, dtype, B, T, K, N, "gelu_tanh", gate=True, residual=True, seed=K)
    check_linear(dev, dtype, B, T, K, N, None, bias=False, seed=N)


@pytest.mark.parametrize("B,T,K,N", [(2, 40, 16, 24), (3, 130, 40, 33), (1, 70, 8, 5), (70, 9, 4, 3)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_linear_gate_in_the_weights(dev, dtype, B, T, K, N):
    """Samples long enough that the backward gates the weights instead of the rows."""
    check_linear(dev, dtype, B, T, K, N, None, gate=True, residual=True, seed=K)
    check_linear(dev, dtype, B, T, K, N, None, bias=False, gate=True, seed=N)


@pytest.mark.parametrize("dtype,act", [(BF16, "silu"), (FP16, None)])
def test_linear_tiles(dev, dtype, act):
    """More than a workgroup of few rows for each CU: the smallest tiles."""
    check_linear(dev, dtype, 2, 515, 8, 500, act, gate=act is None, residual=True)


def check_ffn(dev, dtype, B, T, C, F, act="gelu_tanh", bias=True, gate=True, residual=True, N=None, seed=0):
    r = Draw(dev, dtype, seed)
    N = N or C
    x, w1, w2 = r(B, T, C), r(F, C, std=C ** -0.5), r(N, F, std=F ** -0.5)
    b1, b2 = (r(F, std=0.3), r(N, std=0.3)) if bias else (None, None)
    g, res, dout = r(B, N, std=0.3, mean=0.5) if gate else None, r(B, T, N) if residual else None, r(B, T, N).detach()
    return check_layers(x, [(w1, b1, act), (w2, b2, None)], g, res, dout, lambda: llsa_amd.feed_forward(x, w1, b1, w2, b2, activation=act, gate=g, residual=res))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_feed_forward(dev, dtype, act):
    check_ffn(dev, dtype, 2, 21, 40, 72, act)


@pytest.mark.parametrize("B,T,C,F,N", [(1, 1, 1, 1, 1), (2, 3, 7, 13, 5), (1, 66, 24, 130, 24), (3, 22, 65, 65, 9)])
def test_feed_forward_sizes(dev, B, T, C, F, N):
    check_ffn(dev, BF16, B, T, C, F, N=N, seed=F)
    check_ffn(dev, FP16, B, T, C, F, "silu", bias=False, gate=False, residual=False, N=N, seed=C)


@pytest.mark.parametrize("B,T,C,F,N", [(2, 80, 24, 40, 24), (3, 66, 9, 33, 7)])
def test_feed_forward_gate_in_the_weights(dev, B, T, C, F, N):
    check_ffn(dev, BF16, B, T, C, F, N=N, seed=F)
    check_ffn(dev, FP16, B, T, C, F, "gelu", bias=False, N=N, seed=C)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("B,T,K,N", [(3, 5459, 136, 264), (3, 32765, 40, 120), (1, 4090, 1032, 4090), (2, 2046, 1032, 4088), (5, 1639, 320, 1025), (3, 1531, 77, 333)])
def test_large_tiles(dtype, B, T, K, N):
    """Sizes at which the larger tiles are taken, with edges inside them in every direction: each activation once."""
    dev = torch.device("cuda")
    for act, gate, residual in ((None, True, True), ("gelu_tanh", False, True), ("silu", True, False), ("gelu", False, False)):
        check_linear(dev, dtype, B, T, K, N, act, gate=gate, residual=residual, seed=N)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("B,T,C,F", [(3, 32765, 40, 120), (2, 8190, 264, 520), (4, 1021, 1032, 4088)])
def test_large_feed_forward(dtype, B, T, C, F):
    for act in ("gelu_tanh", "gelu", "silu"):
        check_ffn(torch.device("cuda"), dtype, B, T, C, F, act, seed=F)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("B,T,K,N", [(3, 3221, 384, 1472), (2, 20011, 384, 320), (7, 1639, 320, 1184), (33, 289, 384, 1536), (3, 3301, 1536, 384), (2, 4099, 1600, 320)])
def test_weights_in_registers(dtype, B, T, K, N):
    """Many rows and a contraction of 320 or 384, forward (K) or back (N): a last tile that overlaps the one before it, columns that end inside a
    workgroup's, samples that begin anywhere, weights of each sample."""
    dev = torch.device("cuda")
    for act, gate, residual in ((None, True, True), ("gelu_tanh", False, True), ("silu", True, False), ("gelu", False, False), (None, False, False)):
        check_linear(dev, dtype, B, T, K, N, act, gate=gate, residual=residual, seed=N)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("B,T,C,F", [(3, 3301, 384, 1536), (1, 8211, 320, 1600), (35, 257, 384, 1536)])
def test_feed_forward_weights_in_registers(dtype, B, T, C, F):
    for act in ("gelu_tanh", "gelu", "silu"):
        check_ffn(torch.device("cuda"), dtype, B, T, C, F, act, seed=F)


@pytest.mark.gpu
def test_weights_in_registers_of_slices():
    """Rows inside wider ones: the same bits as contiguous rows."""
    r = Draw(torch.device("cuda"), BF16, 7)
    x, w, res, g = r(2, 4111, 400).detach(), r(1536, 424).detach(), r(2, 4111, 1552).detach(), r(2, 1536).detach()
    xs, ws, rs = x[..., 8:392], w[:, 16:400], res[..., 8:1544]
    a = llsa_amd.linear(xs, ws, None, activation="silu", gate=g, residual=rs)
    assert torch.equal(a, llsa_amd.linear(xs.contiguous(), ws.contiguous(), None, activation="silu", gate=g, residual=rs.contiguous()))
