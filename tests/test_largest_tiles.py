"""linear and feed_forward at sizes that take the tiles of 256 x 256, forward and back, against 64 bits element by element.  By the rule of tiles_for (linear.hip): forward
6138 rows of 2056 > 2056 are 216 such tiles, one round of 1.8 + 220 / 2056 = 1.91, against 2 of 128 x 128 and 2.6 of 192 x 128; back 6138 of 2056 (216) and 12270 of 1032
(240) are one round of 1.8 against 2 and 2.76.  A trace of the kernels shows them."""
import pytest
import torch

from test_block_operators import check_ffn, check_linear

BF16, FP16 = torch.bfloat16, torch.float16


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("B,T,K,N", [(3, 2046, 2056, 2056), (3, 2046, 2051, 2055)])
def test_forward_and_back(dtype, B, T, K, N):
    """Each activation, gates of samples that end inside a tile, residual, kept z; odd rows (2055) take the form for any alignment, back (2051) too."""
    for act, gate, residual in ((None, True, True), ("gelu_tanh", False, True), ("silu", True, False), ("gelu", False, False), (None, False, False)):
        check_linear(torch.device("cuda"), dtype, B, T, K, N, act, gate=gate, residual=residual, seed=N)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("B,T,K,N", [(5, 2454, 1032, 264), (5, 2454, 1029, 261), (1, 12270, 1032, 264)])
def test_back_with_weights_of_each_sample(dtype, B, T, K, N):
    """Samples of 2 K rows and more: the gate in the weights.  The last tiles of a sample end inside it."""
    check_linear(torch.device("cuda"), dtype, B, T, K, N, None, gate=True, residual=True, seed=N)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("act", ["gelu_tanh", "gelu", "silu"])
@pytest.mark.parametrize("gate", [True, False])
def test_feed_forward_back(dtype, act, gate):
    """dx multiplied by act'(z), with weights of each sample and without."""
    check_ffn(torch.device("cuda"), dtype, 5, 2454, 264, 1032, act, gate=gate, seed=3)
