"""Every compiled form of the experts' products that smaller sizes do not reach, against 64 bits element by element: weights in registers (contractions of 320 and 384, blocks of
columns that are full and that leave waves idle, runs that are empty, rows without an expert, each way out) and tiles of 256 x 256.  llsa_experts_form says that a size takes
the form it is listed for; so does the same rule in the linear layer in 8-bit integers, in words."""
import pytest
import torch

import llsa_amd
from expert_cases import check_experts, check_grouped
from llsa_amd._lib import LIB_PATH, Lib

BF16, FP16 = torch.bfloat16, torch.float16
T256, RESIDENT = 6, 7
pad8 = lambda n: (n + 7) // 8 * 8

# runs, channels in and out, forms of the forward and of dx (None: any)
GROUPED = [([5000, 0, 7001, 4400], 384, 1536, RESIDENT, None), ([9000, 1, 7500], 320, 1184, RESIDENT, None), ([0, 16500, 3], 384, 1472, RESIDENT, None),
           ([30000, 0, 36001, 5], 320, 320, RESIDENT, RESIDENT), ([66001], 384, 384, RESIDENT, RESIDENT), ([16385, 0, 401], 1536, 384, None, RESIDENT), ([16385, 402], 1184, 320, None, RESIDENT),
           ([6500, 0, 5188], 2048, 1032, T256, None), ([6500, 0, 5188], 2051, 1030, T256, None), ([9001, 11300], 520, 264, None, T256)]
# samples, tokens, experts, choices, channels in, hidden, out; forms of both products, of their gradients' (hidden rows, x)
BLOCKS = [(2, 20000, 4, 2, 384, 384, 384, RESIDENT, RESIDENT, RESIDENT, RESIDENT), (2, 20000, 4, 2, 320, 320, 320, RESIDENT, RESIDENT, RESIDENT, RESIDENT),
          (1, 9300, 4, 2, 320, 1184, 320, RESIDENT, None, RESIDENT, None), (1, 9300, 4, 2, 384, 1472, 384, RESIDENT, None, RESIDENT, None), (1, 6100, 4, 2, 264, 2048, 1032, None, T256, None, None),
          (1, 6100, 4, 2, 2048, 1032, 264, T256, None, None, None), (2, 10001, 2, 1, 520, 264, 72, None, None, None, T256)]


def _forms_of_grouped(counts, K, N, front=13, tail=300):
    form, rows, E = Lib(LIB_PATH).experts_form, sum(counts) + front + tail, len(counts)
    return form(rows, E, N, pad8(K), 0, 0, int(N % 8 == 0)), form(rows, E, K, N, 1, 0, int(K % 8 == 0))


def _forms_of_block(B, T, n, k, C, F, N):
    form, rows = Lib(LIB_PATH).experts_form, B * T * k
    return form(rows, n, F, pad8(C), 0, 0, 1), form(rows, n, N, pad8(F), 0, 0, 1), form(rows, n, F, N, 1, 1, 1), form(rows, n, C, F, 1, 0, 1)


@pytest.mark.parametrize("counts,K,N,fwd,dx", GROUPED)
def test_which_form_products_take(counts, K, N, fwd, dx):
    for want, got in zip((fwd, dx), _forms_of_grouped(counts, K, N)):
        assert want is None or want == got


@pytest.mark.parametrize("case", BLOCKS)
def test_which_form_blocks_take(case):
    for want, got in zip(case[7:], _forms_of_block(*case[:7])):
        assert want is None or want == got


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("counts,K,N", [c[:3] for c in GROUPED])
def test_grouped(dtype, counts, K, N):
    """Each activation, with kept slopes and without, rows in front of the first run and behind the last."""
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(K + N)
    r = lambda *s, std=1.0: (torch.randn(*s, generator=g, device=dev) * std).to(dtype).requires_grad_()
    offsets = torch.tensor([13] + counts).cumsum(0).to(torch.int32).to(dev)
    rows, E = int(offsets[-1]) + 300, len(counts)
    for act in (None, "gelu_tanh", "silu", "gelu"):
        x, w, b = r(rows, K), r(E, N, K, std=K ** -0.5), r(E, N, std=0.3) if act != "silu" else None
        out, _ = check_grouped(x, w, offsets, b, act, r(rows, N).detach())
        with torch.no_grad():
            assert torch.equal(llsa_amd.grouped_linear(x, w, offsets, b, activation=act), out)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("B,T,n,k,C,F,N", [c[:7] for c in BLOCKS])
def test_block(dtype, B, T, n, k, C, F, N):
    """Tokens without an expert, an expert without a token; gate and residual, and neither."""
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(C + F)
    r = lambda *s, std=1.0: (torch.randn(*s, generator=g, device=dev) * std).to(dtype).requires_grad_()
    for act, extra in (("gelu_tanh", True), ("silu", False), ("gelu", True)):
        x, logits = r(B, T, C), r(B, T, n).detach()
        logits[:, ::7] = -float("inf")
        if extra and n > 2:
            logits[..., 1] = -float("inf")
        routing = llsa_amd.route_tokens(logits, k)
        routing.weights.requires_grad_()
        w1, w2 = r(n, F, C, std=C ** -0.5), r(n, N, F, std=F ** -0.5)
        b1, b2, gate, residual = (r(n, F, std=0.3), r(n, N, std=0.3), r(B, N), r(B, T, N)) if extra else (None,) * 4
        out, _ = check_experts(x, routing, w1, b1, w2, b2, act, gate, residual, r(B, T, N).detach())
        with torch.no_grad():
            assert torch.equal(llsa_amd.expert_feed_forward(x, routing, w1, b1, w2, b2, activation=act, gate=gate, residual=residual), out)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("B,T,K,N", [(3, 2046, 4096, 2056), (3, 2046, 4090, 2051)])
def test_8_bits_in_tiles_of_256(dtype, B, T, K, N):
    """6138 rows of 4096 > 2056 are 216 tiles of 256 x 256, one round of 1.8 + 220 / 2048 = 1.91, against 2 of 128 x 128 and 2.6 of 192 x 128; odd columns take the form for any
    alignment."""
    from test_linear_int8 import run
    for act, gate, residual in ((None, True, True), ("gelu_tanh", False, True), ("silu", True, False), ("gelu", False, False)):
        run(torch.device("cuda"), dtype, B, T, K, N, act, gate=gate, residual=residual, seed=N)
