"""Every form that the kernels of layer_norm, linear and feed_forward are compiled in, against 64 bits element by element: channels by which a row is spread over lanes and
pieces, whole and odd, in each type; tiles of few rows; the tiles of dx behind each activation and of odd rows."""
import contextlib

import pytest
import torch

from block_cases import check_norm
from emu_util import emu_lib
from llsa_amd._lib import override_library_for_tests
from test_block_operators import check_ffn, check_linear, norm_inputs

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def dev(request):
    with contextlib.ExitStack() as stack:
        if request.param == "cpu":
            stack.enter_context(override_library_for_tests(emu_lib()))
        yield torch.device(request.param)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("C", [128, 200, 384, 504, 1000, 1504, 2048, 4000, 6000, 8000])
def test_norm_rows(dev, dtype, C):
    """16, 64 and 256 lanes a row, one to four pieces each, in pieces of 16 bytes and value by value."""
    for c in (C, C - 3):
        check_norm(*norm_inputs(dev, dtype, (2, 5, c), True, True, seed=c))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("M", [9, 23, 41])
@pytest.mark.parametrize("act", [None, "silu", "gelu", "gelu_tanh"])
def test_few_rows(dev, dtype, M, act):
    """One, two and four tiles of sixteen rows; whole pieces and odd rows."""
    for K, N in ((136, 72), (77, 35)):
        check_linear(dev, dtype, 1, M, K, N, act, gate=True, residual=True, seed=K)
        if act is not None:
            check_ffn(dev, dtype, 1, M, K, N, act, seed=N)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("B,T,C,F", [(2, 1021, 40, 504), (2, 4090, 40, 1016), (2, 4090, 40, 1400)])
def test_back_through_activations(dtype, B, T, C, F):
    """Tiles of 64 x 64, 128 x 128 and 192 x 128."""
    for act in ("silu", "gelu", "gelu_tanh"):
        check_ffn(torch.device("cuda"), dtype, B, T, C, F, act, gate=False, seed=F)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("B,T,K,N", [(2, 1021, 503, 40), (2, 4090, 1015, 40), (2, 4090, 1399, 40)])
def test_back_to_odd_rows(dtype, B, T, K, N):
    """The same tiles where rows of dx are no whole pieces; the gate in the rows and in the weights."""
    for gate in (True, False):
        check_linear(torch.device("cuda"), dtype, B, T, K, N, None, gate=gate, seed=K)
