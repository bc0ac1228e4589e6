"""Gradients of the experts' weights out of chunks of rows: what the sums on the way take of memory, and runs that begin, end and go on at the chunks' borders."""
import contextlib

import pytest
import torch

from emu_util import emu_lib
from expert_cases import check_grouped
from llsa_amd._lib import LIB_PATH, Lib, override_library_for_tests

BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def dev(request):
    with contextlib.ExitStack() as stack:
        if request.param == "cpu":
            stack.enter_context(override_library_for_tests(emu_lib()))
        yield torch.device(request.param)


@pytest.mark.parametrize("rows,E,N,K", [(65536, 256, 2048, 7168), (4096, 256, 2048, 2048), (16384, 64, 2048, 2048), (16384, 256, 384, 1536), (100, 256, 1536, 384), (262144, 8, 1536, 384),
                                        (1 << 20, 256, 1024, 1024)])
def test_memory_of_the_sums(rows, E, N, K):
    """Besides a row of sums for each expert and chunk there are only the gradients of experts that a chunk cuts, two of each at most: chunks of 256 rows and more, and no more of them
    than four rounds of the chip's workgroups (2048 of tiles of 128 x 128 at least, 4096 of 64 x 64)."""
    got = Lib(LIB_PATH).experts_dw_workspace_bytes(rows, E, N, K)
    tiles = -(-N // 192) * -(-K // 128)
    chunks = min(max(1, rows // 256), 1 + 4 * 1024 // tiles) + 1
    assert 0 < got <= 4 * (2 * (chunks - 1) * N * K + (chunks + E) * N * -(-K // 64))
    if rows <= 512:
        assert got <= 4 * (1 + E) * N * -(-K // 64)           # one chunk cuts no one


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("counts", [[320] * 6 + [80], [319, 1, 321, 0, 640, 3, 716], [2000], [5, 0, 1990, 5], [1, 2, 3, 314, 0, 0, 320, 700, 1, 1, 658], [0, 640, 0, 640, 0, 640, 80, 0], [40] * 50])
def test_runs_at_the_borders(dev, counts, dtype):
    """2000 rows of 16 and 24 channels are seven chunks of 320; memory that nothing wrote holds NaN."""
    before = torch.are_deterministic_algorithms_enabled(), torch.is_deterministic_algorithms_warn_only_enabled(), torch.utils.deterministic.fill_uninitialized_memory
    torch.use_deterministic_algorithms(True, warn_only=True)
    torch.utils.deterministic.fill_uninitialized_memory = True
    try:
        g = torch.Generator().manual_seed(len(counts))
        r = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).to(dtype).to(dev)
        both = ((0, 0), (70, 9))                              # (the emulation takes seconds for either)
        for front, tail in both if dev.type == "cuda" else both[:1] if dtype == BF16 else both[1:]:
            rows, E = sum(counts) + front + tail, len(counts)
            offsets = torch.tensor([front] + counts).cumsum(0).to(torch.int32).to(dev)
            check_grouped(r(rows, 24).requires_grad_(), r(E, 16, 24, std=0.2).requires_grad_(), offsets, r(E, 16).requires_grad_(), None, r(rows, 16))
    finally:
        torch.use_deterministic_algorithms(before[0], warn_only=before[1])
        torch.utils.deterministic.fill_uninitialized_memory = before[2]


@pytest.mark.gpu
def test_many_experts_of_few_rows():
    """256 experts share 4096 rows of 2048 and 1024 channels: the step asks for its results, and little more."""
    import llsa_amd
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=g, device=dev).to(BF16)
    x, w = r(4096, 1024).requires_grad_(), (r(256, 2048, 1024) * 0.03).requires_grad_()
    offsets = (torch.arange(257, device=dev) * 16).to(torch.int32)
    y = llsa_amd.grouped_linear(x, w, offsets)
    dout = torch.ones_like(y)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    start = torch.cuda.memory_allocated()
    dw, = torch.autograd.grad(y, w, dout)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - start <= dw.numel() * 2 + (600 << 20)     # (as one slab of fp32 for each expert: 2 GB and more)
    for e in (0, 101, 255):
        ref = dout[16 * e:16 * e + 16].double().t() @ x.detach()[16 * e:16 * e + 16].double()
        # (sums of 16, which bf16 rounds once)
        assert ((dw[e].double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -18 * x.detach()[16 * e:16 * e + 16].double().abs().sum(0)).all()
