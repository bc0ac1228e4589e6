"""The C ABI's products into rows of any alignment and distance, at sizes where aligned ones take the kernel that keeps the weights in registers: it stores 16 bytes at a
time, so that others have to take the tiles."""
import ctypes as C

import pytest
import torch

from llsa_amd._lib import LIB_PATH, ExpertsArgs, Lib

RESIDENT = 7                                                  # LLSA_EXPERTS_RESIDENT


@pytest.mark.parametrize("rows,E,N,K", [(16384, 8, 1536, 384), (65536, 4, 384, 384), (65536, 1, 320, 320), (32768, 3, 704, 320)])
@pytest.mark.parametrize("back", [0, 1])
def test_weights_in_registers_take_whole_stores(rows, E, N, K, back):
    form = Lib(LIB_PATH).experts_form
    assert form(rows, E, N, K, back, 0, 1) == RESIDENT and 3 <= form(rows, E, N, K, back, 0, 0) < RESIDENT
    assert form(0, E, N, K, back, 0, 1) == -1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,number", [(torch.bfloat16, 0), (torch.float16, 2)])
@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("shift,extra", [(1, 0), (0, 3), (5, 1), (8, 4)])
def test_any_out(dtype, number, back, shift, extra):
    """out begins `shift` elements in, its rows are N + extra apart; what lies between and around them stays."""
    dev = torch.device("cuda")
    rows, E, N, K = 16384, 3, 1536, 384
    g = torch.Generator(device=dev).manual_seed(shift + extra)
    x, w = torch.randn(rows, K, generator=g, device=dev).to(dtype), (torch.randn(E, *((K, N) if back else (N, K)), generator=g, device=dev) * K ** -0.5).to(dtype)
    offsets = torch.tensor([13, 5000, 5000, rows - 77], dtype=torch.int32, device=dev)
    lib = Lib(LIB_PATH)

    def run(shift, ld):
        room = torch.full((rows * ld + 16,), 7.0, dtype=dtype, device=dev)
        a = ExpertsArgs()
        a.w, a.offsets, a.rows, a.tokens, a.k, a.E, a.dtype, a.gaps = w.data_ptr(), offsets.data_ptr(), rows, rows, 1, E, number, 1
        a.out, a.ldo = room.data_ptr() + 2 * shift, ld
        if back:
            a.dz, a.lddz, a.ldw, a.N, a.K = x.data_ptr(), K, N, K, N
            assert lib.experts_dx(C.byref(a), torch.cuda.current_stream().cuda_stream) == 0
        else:
            a.x, a.ldx, a.ldw, a.N, a.K = x.data_ptr(), K, K, N, K
            assert lib.experts_fwd(C.byref(a), torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        assert (room[:shift] == 7).all() and (room[shift + rows * ld:] == 7).all()
        at = room[shift:shift + rows * ld].view(rows, ld)
        assert (at[:, N:] == 7).all()
        return at[:, :N].float()

    plain, got = run(0, N), run(shift, N + extra)
    # (two sums of the same K products in fp32, each off by up to K * 2^-24 of the sum of their magnitudes, which is no larger than the product of the vectors' lengths; rounded once each)
    size = x.float().norm(dim=1).max() * w.float().norm(dim=1 if back else 2).max()
    assert ((got - plain).abs() <= torch.finfo(dtype).eps * plain.abs() + 2 * K * 2.0 ** -24 * size).all() and not got[:13].any() and not got[rows - 77:].any() and got[13:5000].any()
