"""The router, the products by expert and the routed feed-forward block against their formulas in 64 bits: whole numbers have to be equal, everything else
stays within bounds that follow from the roundings.  On the CPU through the x86 build of the kernels, on the GPU through the library, where larger sizes run too."""
import contextlib

import pytest
import torch

import llsa_amd
from emu_util import emu_lib
from expert_cases import check_experts, check_grouped, check_route
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

    def __call__(self, *shape, std=1.0, mean=0.0, dtype=None, grad=True):
        return (torch.randn(*shape, generator=self.g) * std + mean).to(dtype or self.dtype).to(self.dev).requires_grad_(grad)


# ---------------------------------------------------------------------------------------
# the router
# ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("M,n,k", [(1, 1, 1), (1, 8, 2), (37, 8, 2), (50, 5, 3), (65, 16, 4), (33, 9, 9), (40, 64, 8), (21, 61, 16), (19, 256, 5), (13, 100, 2), (70, 2, 2)])
def test_route(dev, dtype, normalize, M, n, k):
    r = Draw(dev, dtype, M + n)
    check_route(r(M, n), k, normalize, r(M, k, dtype=FP32, grad=False))


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("M,n,k", [(2100, 8, 2), (1500, 5, 4), (700, 70, 7)])
def test_route_in_chunks(dev, normalize, M, n, k):
    """More slots than one workgroup places: a launch that counts, another that places."""
    r = Draw(dev, BF16, M)
    check_route(r(M, n), k, normalize, r(M, k, dtype=FP32, grad=False))


def test_route_equal_logits(dev):
    for n, k in ((8, 3), (16, 5), (64, 9), (256, 16)):
        check_route(torch.zeros(9, n, device=dev).requires_grad_(), k, True, torch.randn(9, k).to(dev))
        g = torch.Generator().manual_seed(n)
        check_route((torch.randint(0, 3, (33, n), generator=g).float() * torch.where(torch.rand(33, n, generator=g) < 0.3, -0.0, 1.0)).to(dev).requires_grad_(), k, False, torch.randn(33, k).to(dev))


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("n", [6, 16, 40, 90])
def test_route_masks(dev, normalize, n):
    """Rows with nothing, with one expert, with fewer than k; the type's lowest values, which may be chosen."""
    r = Draw(dev, BF16, n)
    l = r(24, n, grad=False)
    l[0] = l[23] = -float("inf")
    l[1, 1:] = -float("inf")
    l[2, :n - 2] = -float("inf")
    l[3, 2:] = torch.finfo(BF16).min
    l[4] = torch.finfo(BF16).min
    l[5:12][torch.rand(7, n, generator=r.g).to(dev) < 0.7] = -float("inf")
    check_route(l.requires_grad_(), 4, normalize, r(24, 4, dtype=FP32, grad=False))
    out = llsa_amd.route_tokens(torch.full((7, n), -float("inf"), device=dev), 3, normalize=normalize)
    assert not out.weights.any() and (out.experts == -1).all() and (out.order == -1).all() and (out.places == -1).all() and not out.offsets.any()


def test_route_no_numbers(dev):
    """A NaN counts as the largest number; the weights of such a row, and of one with an infinity, are NaN, those of others are what they were."""
    r = Draw(dev, FP32, 3)
    for n in (8, 16, 64, 200):
        l = r(12, n, grad=False)
        plain = llsa_amd.route_tokens(l, 2)
        bad = l.clone()
        bad[3, 5], bad[7, 2], bad[7, 6], bad[9, 1] = float("nan"), float("nan"), float("nan"), float("inf")
        out = llsa_amd.route_tokens(bad, 2)
        assert out.experts[3, 0] == 5 and out.experts[7].tolist() == [2, 6] and out.experts[9, 0] == 1
        assert out.weights[[3, 7, 9]].isnan().all()
        keep = [i for i in range(12) if i not in (3, 7, 9)]
        assert torch.equal(out.weights[keep], plain.weights[keep]) and torch.equal(out.experts[keep], plain.experts[keep])
        assert sorted(out.order.tolist()) == list(range(24))


@pytest.mark.gpu
@pytest.mark.parametrize("M,n,k", [(131072, 8, 2), (40000, 64, 8), (20001, 256, 16), (9999, 61, 3)])
def test_large_route(M, n, k):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(M)
    l = torch.randn(M, n, device=dev, generator=g)
    out = llsa_amd.route_tokens(l, k)
    v, i = torch.sort(l, dim=-1, descending=True, stable=True)
    assert torch.equal(out.experts.long(), i[:, :k])
    by, order = torch.sort(i[:, :k].reshape(-1), stable=True)
    assert torch.equal(out.order.long(), order) and torch.equal(out.offsets.long(), torch.searchsorted(by, torch.arange(n + 1, device=dev)))
    assert torch.equal(out.places.reshape(-1)[order].long(), torch.arange(M * k, device=dev))
    assert (out.weights.double() - torch.softmax(v[:, :k].double(), -1)).abs().max() < 2.0 ** -20


# ---------------------------------------------------------------------------------------
# products by expert
# ---------------------------------------------------------------------------------------
def grouped(dev, dtype, counts, K, N, act=None, bias=True, front=0, tail=0, seed=0):
    r = Draw(dev, dtype, seed)
    offsets = torch.tensor([front] + counts).cumsum(0).to(torch.int32).to(dev)
    rows = int(offsets[-1]) + tail
    x, w, b = r(rows, K), r(len(counts), N, K, std=K ** -0.5), r(len(counts), N, std=0.3) if bias else None
    return check_grouped(x, w, offsets, b, act, r(rows, N, grad=False))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("act", [None, "silu", "gelu", "gelu_tanh"])
def test_grouped(dev, dtype, act):
    grouped(dev, dtype, [7, 0, 19, 1], 40, 72, act, tail=3)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("counts,K,N,front,tail", [([1], 1, 1, 0, 0), ([0, 0, 1, 0], 8, 8, 0, 0), ([5, 3, 9], 13, 7, 2, 4), ([33, 17], 64, 64, 0, 0), ([70, 1, 66], 130, 67, 0, 1),
                                                  ([0, 0], 16, 24, 0, 9), ([20, 30, 10, 0, 40], 72, 33, 17, 0), ([130], 24, 40, 0, 0), ([2] * 70, 16, 16, 1, 1), ([1] * 256, 8, 9, 0, 0)])
def test_grouped_sizes(dev, dtype, counts, K, N, front, tail):
    if dev.type == "cpu" and len(counts) > 100:
        pytest.skip("minutes in the emulation, where every lane of a scan is a fiber")
    grouped(dev, dtype, counts, K, N, "gelu_tanh", front=front, tail=tail, seed=K)
    grouped(dev, dtype, counts, K, N, None, bias=False, front=front, tail=tail, seed=N)


@pytest.mark.parametrize("dtype,act", [(BF16, "silu"), (FP16, None)])
def test_grouped_tiles(dev, dtype, act):
    """More rows than a workgroup of few rows for each CU: the smallest tiles; rows of an expert in several pieces."""
    grouped(dev, dtype, [700, 0, 515, 65], 16, 500, act, tail=70)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("counts,K,N", [([5000, 77, 0, 9001, 1], 136, 264), ([40000, 30001, 27011], 48, 120), ([3000, 5001, 4100], 1032, 1030), ([4090, 4096, 257, 1, 3000], 1032, 1024),
                                       ([2000, 1639, 8], 320, 1025), ([1531] * 7, 77, 333), ([400] * 60 + [0, 3, 1, 9], 256, 512), ([50] * 64, 520, 264), ([8192] * 3, 2048, 2048)])
def test_grouped_large(dtype, counts, K, N):
    """Sizes at which the larger tiles are taken, forward and back, with edges inside them in every direction: each activation once."""
    dev = torch.device("cuda")
    for act in (None, "gelu_tanh", "silu", "gelu"):
        grouped(dev, dtype, counts, K, N, act, front=13 if act else 0, tail=300 if act else 0, seed=N)


def test_grouped_offsets_out_of_order(dev):
    """A caller's offsets: beyond the rows, negative, falling.  They are held to the rows and made not to fall."""
    r = Draw(dev, BF16, 5)
    for offsets in ([-5, 4, 3, 30], [0, 50, 20, 12], [7, 2, 1, 0], [3, 3, 3, 1 << 30], [-(1 << 31), 0, (1 << 31) - 1, 5]):
        check_grouped(r(24, 16), r(3, 24, 16), torch.tensor(offsets, dtype=torch.int32, device=dev), r(3, 24), "silu", r(24, 24, grad=False))


# ---------------------------------------------------------------------------------------
# the routed feed-forward block
# ---------------------------------------------------------------------------------------
def routed(dev, dtype, B, T, n, k, C, F, act="gelu_tanh", bias=True, gate=True, residual=True, N=None, seed=0, mask=None, normalize=True):
    r = Draw(dev, dtype, seed)
    N = N or C
    x, logits = r(B, T, C), r(B, T, n, grad=False)
    if mask is not None:
        logits = mask(logits)
    routing = llsa_amd.route_tokens(logits, k, normalize=normalize)
    routing.weights.requires_grad_()
    w1, w2 = r(n, F, C, std=C ** -0.5), r(n, N, F, std=F ** -0.5)
    b1, b2 = (r(n, F, std=0.3), r(n, N, std=0.3)) if bias else (None, None)
    return check_experts(x, routing, w1, b1, w2, b2, act, r(B, N, std=0.3, mean=0.5) if gate else None, r(B, T, N) if residual else None, r(B, T, N, grad=False))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_experts(dev, dtype, act):
    routed(dev, dtype, 2, 21, 4, 2, 40, 72, act)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("B,T,n,k,C,F,N", [(1, 1, 1, 1, 1, 1, 1), (2, 3, 3, 2, 7, 13, 5), (1, 66, 4, 3, 24, 130, 24), (3, 22, 2, 2, 65, 65, 9), (1, 1, 8, 2, 24, 40, 16), (1, 40, 70, 5, 16, 24, 16)])
def test_experts_sizes(dev, dtype, B, T, n, k, C, F, N):
    routed(dev, dtype, B, T, n, k, C, F, N=N, seed=F)
    routed(dev, dtype, B, T, n, k, C, F, "silu", bias=False, gate=False, residual=False, N=N, seed=C, normalize=False)


def test_experts_masks(dev):
    """Tokens without an expert, experts without a token, tokens with fewer experts than the others."""
    def mask(l):
        l[0, :5] = -float("inf")
        l[1, :, 2] = -float("inf")
        l[0, :, 2] = -float("inf")
        l[1, 3, 1:] = -float("inf")
        return l
    out, got = routed(dev, BF16, 2, 17, 4, 2, 24, 40, mask=mask)
    out, got = routed(dev, FP16, 2, 17, 4, 3, 24, 40, mask=mask, gate=False, residual=False)
    assert not out[0, :5].any() and not got["x"][0, :5].any() and not got["weights"][0, :5].any() and not got["w_in"][2].any()
    routed(dev, BF16, 2, 9, 3, 2, 16, 24, mask=lambda l: torch.full_like(l, -float("inf")))


def test_experts_tiles(dev):
    """All tokens to one of them: more rows than a workgroup of few rows for each CU."""
    routed(dev, BF16, 1, 1030, 2, 1, 24, 264, mask=lambda l: l * torch.tensor([1.0, 0.0], device=l.device).to(l.dtype) + torch.tensor([9.0, 0.0], device=l.device).to(l.dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("B,T,n,k,C,F", [(3, 5459, 5, 2, 136, 264), (2, 8190, 8, 2, 264, 520), (4, 1021, 7, 3, 333, 1001), (8, 700, 64, 4, 128, 512), (2, 20000, 8, 2, 384, 1536), (3, 2049, 2, 1, 1032, 2048)])
def test_experts_large(dtype, B, T, n, k, C, F):
    for act, extra in (("gelu_tanh", True), ("gelu", False), ("silu", True)):
        routed(torch.device("cuda"), dtype, B, T, n, k, C, F, act, gate=extra, residual=extra, bias=extra, seed=F)


def test_router_and_experts_together(dev):
    """Gradients of the logits through the block, against differences of the definition in 64 bits."""
    r = Draw(dev, BF16, 11)
    x, logits, w1, b1, w2, b2 = r(2, 9, 16), r(2, 9, 4), r(4, 24, 16, std=0.3), r(4, 24, std=0.3), r(4, 16, 24, std=0.3), r(4, 16, std=0.3)
    dout = r(2, 9, 16, grad=False)
    routing = llsa_amd.route_tokens(logits, 2)
    y = llsa_amd.expert_feed_forward(x, routing, w1, b1, w2, b2, activation="silu")
    got, = torch.autograd.grad(y, logits, dout)
    v = [t.detach().double().cpu() for t in (x, w1, b1, w2, b2)]
    chosen = torch.zeros(2, 9, 4, dtype=torch.bool).scatter_(2, routing.experts.cpu().long(), True)

    def value(l):
        p = torch.softmax(torch.where(chosen, l, -float("inf")), -1)
        h = torch.nn.functional.silu(torch.einsum("btc,efc->btef", v[0], v[1]) + v[2])
        y = torch.einsum("btef,enf->bten", h, v[3]) + v[4]
        return ((p[..., None] * y).sum(2) * dout.double().cpu()).sum((1, 2)), y
    l = logits.detach().double().cpu()
    y64 = value(l)[1]
    size = (y64.abs() * dout.double().cpu().abs()[:, :, None]).sum(-1).amax(-1)       # of what a weight's gradient is a sum of
    step = 1e-4
    for t in range(9):
        for e in range(4):
            d = torch.zeros_like(l)
            d[:, t, e] = step
            diff = (value(l + d)[0] - value(l - d)[0]) / (2 * step)
            # (six roundings of half a step, 2^-8, on the way to a weight's gradient, in the worst case all of one sign; the differences' own error is far below)
            assert ((got[:, t, e].double().cpu() - diff).abs() <= 6 * 2.0 ** -8 * size[:, t] + 2.0 ** -8 * diff.abs() + 1e-6).all()
