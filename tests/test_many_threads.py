"""Rows of which there are so many that one launch, which has fewer than 2^32 threads, does not take them: a token a sample, long rows of 8-bit integers, a router's logits."""
import pytest
import torch

import llsa_amd

BF16 = torch.bfloat16


def _room(gigabytes):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < gigabytes << 30:
        pytest.skip(f"needs {gigabytes} GB")


@pytest.mark.gpu
def test_samples_of_the_routed_block():
    """The gradients of weights and gate take a workgroup of 256 for every sample.  A contraction of 8 is one matrix instruction in every kernel, and what is added to it are zeros, so
    that a few of the rows by themselves have the same bits."""
    _room(16)
    dev = torch.device("cuda")
    B, n = (1 << 24) + 3, 2
    g = torch.Generator(device=dev).manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, device=dev, dtype=BF16)
    x, gate, dout, logits = r(B, 1, 8), r(B, 8), r(B, 1, 8), r(B, 1, n)
    w_in, b_in, w_out, b_out = r(n, 8, 8), r(n, 8), r(n, 8, 8), r(n, 8)

    def run(pick):
        v = [t[pick].requires_grad_() for t in (x, gate, logits)]
        routing = llsa_amd.route_tokens(v[2], 1, normalize=False)
        y = llsa_amd.expert_feed_forward(v[0], routing, w_in, b_in, w_out, b_out, gate=v[1])
        return [y.detach()] + list(torch.autograd.grad(y, [*v, routing.weights], dout[pick]))

    every = run(slice(None))
    some = torch.tensor([0, 1, (1 << 24) - 2, (1 << 24) - 1, 1 << 24, B - 1], device=dev)
    for name, a, b in zip(("y", "x", "gate", "logits", "weights"), every, run(some)):
        assert torch.equal(a[some], b), name
        assert torch.isfinite(a).all(), name


@pytest.mark.gpu
def test_long_rows_to_8_bits():
    _room(120)
    dev = torch.device("cuda")
    rows, K = (1 << 24) + 5, 1544                             # (a workgroup a row)
    x = torch.zeros(rows, K, dtype=BF16, device=dev)
    some = torch.tensor([0, (1 << 24) - 2, (1 << 24) - 1, 1 << 24, rows - 1], device=dev)
    x[some] = torch.randn(5, K, generator=torch.Generator(device=dev).manual_seed(2), device=dev, dtype=BF16)
    q, s = llsa_amd.quantize_rows(x)
    part_q, part_s = llsa_amd.quantize_rows(x[some])
    assert torch.equal(q[some], part_q) and torch.equal(s[some], part_s) and int((s != 0).sum()) == 5


@pytest.mark.gpu
def test_logits_of_a_router():
    _room(150)
    dev = torch.device("cuda")
    M, n = 1 << 28, 65                                        # (sixteen threads a token)
    logits = torch.zeros(M, n, dtype=torch.float16, device=dev)
    some = torch.tensor([0, (1 << 28) - 17, (1 << 28) - 16, M - 1], device=dev)
    logits[some] = torch.randn(4, n, generator=torch.Generator(device=dev).manual_seed(3), device=dev, dtype=torch.float16)

    def run(l):
        l = l.requires_grad_()
        r = llsa_amd.route_tokens(l, 1, normalize=False)
        weights, experts = r.weights.detach(), r.experts
        return weights, experts, torch.autograd.grad(r.weights, l, torch.ones_like(weights))[0]

    every, part = run(logits), run(logits.detach()[some])
    for name, a, b in zip(("weights", "experts", "logits"), every, part):
        assert torch.equal(a[some], b), name
    # (equal logits: p = 1 / 65, its gradient p (1 - p) at the chosen one, the first, and -p^2 elsewhere)
    a = every[2][1 << 27]
    assert abs(a[0].item() - 64 / 65 ** 2) <= 2.0 ** -16 and (a[1:].float() + 65.0 ** -2).abs().max() <= 2.0 ** -21
