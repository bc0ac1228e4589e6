"""quantize_rows and linear_int8 against their definition in 64 bits.  Whole numbers have to be equal; results stay within bounds that follow from the
roundings (the sums are exact, what follows them is fp32, the result is rounded once)."""
import contextlib

import pytest
import torch

import llsa_amd
from block_cases import E, FAST, SLOPE, act64, half_step, least, per_sample, within
from emu_util import emu_lib
from llsa_amd._lib import override_library_for_tests

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def dev(request):
    with contextlib.ExitStack() as stack:
        if request.param == "cpu":
            stack.enter_context(override_library_for_tests(emu_lib()))
        yield torch.device(request.param)


def step64(x):
    """max |x| / 127 to the nearest fp32: 24 bits over 7, which a rounding to 53 bits in between does not change"""
    return (x.double().abs().amax(-1) / 127).float()


def quantized64(x):
    x = x.detach().cpu()
    s = step64(x)
    d = torch.where(s > 0, s, torch.ones_like(s)).double()[..., None]
    return torch.where(s[..., None] > 0, torch.round(x.double() / d), 0.0).to(torch.int8), s


def rows(dev, dtype, *shape, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std * (torch.rand(*shape[:-1], 1, generator=g) * 3 + 0.05)).to(dtype).to(dev)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("K", [1, 7, 16, 40, 128, 130, 256, 300, 384, 520, 1024, 1030, 1536, 2100, 4096, 9000])
def test_quantize_rows(dev, dtype, K):
    """Every number of lanes and pieces a row is held in; odd lengths."""
    x = rows(dev, dtype, 2, 9, K, seed=K)
    q, s = llsa_amd.quantize_rows(x)
    ref, rs = quantized64(x)
    assert q.dtype == torch.int8 and s.dtype == FP32 and q.shape == x.shape and s.shape == x.shape[:-1]
    assert torch.equal(s.cpu(), rs) and torch.equal(q.cpu(), ref)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_quantize_halves(dev, dtype):
    """Quotients at and next to a half: halves of the largest value (63.5 steps of the unrounded scale), and scales that are powers of two, where halves are exact."""
    top = torch.arange(1, 129).float() * 3
    x = torch.stack([top, top / 2, -top / 2, top / 254 * 3, top * 0.25, -top], 1)
    half = torch.tensor([[127.0] + [k + 0.5 for k in range(0, 126)] + [-(k + 0.5) for k in range(0, 126)]])
    for v in (x, x * 2.0 ** -10, half, half * 2.0 ** -7, half * 64):
        v = v.to(dtype).to(dev)
        q, s = llsa_amd.quantize_rows(v)
        ref, rs = quantized64(v)
        assert torch.equal(s.cpu(), rs) and torch.equal(q.cpu(), ref)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_quantize_extremes(dev, dtype):
    """Rows of zeros, of the least and the largest numbers, one value alone; rows that hold what is no number."""
    f = torch.finfo(dtype)
    x = torch.zeros(8, 40, dtype=dtype)
    x[1, 3] = f.smallest_normal
    x[2] = torch.linspace(-1, 1, 40).to(dtype) * f.smallest_normal
    x[3] = (torch.linspace(-1, 1, 40).double() * f.max).to(dtype)
    x[4, 7] = -f.max
    x[5, 5], x[5, 6] = float("nan"), 1
    x[6, 5], x[6, 6] = float("inf"), 1
    x[7, 39] = -float("inf")
    q, s = (t.cpu() for t in llsa_amd.quantize_rows(x.to(dev)))
    ref, rs = quantized64(x[:5])
    assert torch.equal(s[:5], rs) and torch.equal(q[:5], ref)
    assert s[5:].isnan().all() and not q[5:].any()
    if dtype != FP32:                                         # (numbers below the smallest normal one; a scale of fp32 has room for those of 16 bits)
        x = torch.zeros(3, 24, dtype=dtype)
        x[0, 1] = f.smallest_normal * f.eps
        x[1, :12] = torch.arange(12).to(dtype) * f.smallest_normal * f.eps
        x[2, :12] = -x[1, :12] * 5
        q, s = (t.cpu() for t in llsa_amd.quantize_rows(x.to(dev)))
        ref, rs = quantized64(x)
        assert torch.equal(s, rs) and torch.equal(q, ref)


def layer(dev, dtype, B, T, K, N, bias, gate, residual, seed=0):
    g = torch.Generator().manual_seed(seed + 1)
    r = lambda *s, std=1.0, mean=0.0: (torch.randn(*s, generator=g) * std + mean).to(dtype).to(dev)
    w, ws = quantized64(torch.randn(N, K, generator=g) * K ** -0.5)
    return (rows(dev, dtype, B, T, K, seed=seed), w.to(dev), ws.to(dev), r(N, std=0.3) if bias else None, r(B, N, std=0.3, mean=0.5) if gate else None,
            r(B, T, N) if residual else None)


def check(x, w, ws, b, gate, res, act, got):
    dtype = x.dtype
    where = x.device if x.numel() * w.shape[0] > 1 << 26 else torch.device("cpu")
    c = lambda t: None if t is None else t.detach().double().to(where)
    q, s = quantized64(x)
    p = (c(q).reshape(-1, x.shape[-1]) @ c(w).t()).reshape(*x.shape[:-1], -1) * c(s)[..., None] * c(ws)
    z = p if b is None else p + c(b)
    # the sum to fp32, two products, the bias: half a step each
    a, da = act64(act, z), SLOPE * (3.1 * E * p.abs() + E * z.abs()) + (FAST * (act64(act, z).abs() + z.abs()) if act else 0)
    y = a if gate is None else per_sample(c(gate), x) * a
    dy = da if gate is None else per_sample(c(gate).abs(), x) * da
    ref = y if res is None else y + c(res)
    within(got.to(where), ref, dy + 2.1 * E * (y.abs() + ref.abs()) + half_step(dtype) * (ref.abs() + dy) + least(dtype), "out")


def run(dev, dtype, B, T, K, N, act=None, bias=True, gate=False, residual=False, seed=0):
    x, w, ws, b, g, r = layer(dev, dtype, B, T, K, N, bias, gate, residual, seed)
    y = llsa_amd.linear_int8(x, w, ws, b, activation=act, gate=g, residual=r)
    assert y.dtype == dtype and y.shape == (B, T, N)
    check(x, w, ws, b, g, r, act, y)
    pair = llsa_amd.linear_int8(llsa_amd.quantize_rows(x), w, ws, b, activation=act, gate=g, residual=r, dtype=dtype)
    assert torch.equal(pair, y)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("act", [None, "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("gate,residual", [(False, False), (True, True)])
def test_linear_int8(dev, dtype, act, gate, residual):
    run(dev, dtype, 2, 19, 80, 88, act, gate=gate, residual=residual)


@pytest.mark.parametrize("B,T,K,N", [(1, 1, 1, 1), (3, 1, 16, 8), (1, 7, 5, 3), (2, 33, 128, 64), (1, 65, 130, 67), (2, 64, 400, 129), (1, 130, 33, 200), (1, 17, 1100, 40)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_sizes(dev, dtype, B, T, K, N):
    run(dev, dtype, B, T, K, N, "gelu_tanh", gate=True, residual=True, seed=K)
    run(dev, dtype, B, T, K, N, None, bias=False, seed=N)


def test_tiles(dev):
    """More than a workgroup of few rows for each CU: the smallest tiles."""
    run(dev, BF16, 2, 515, 16, 500, "silu", residual=True)
    run(dev, FP16, 2, 515, 200, 504, None, gate=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("B,T,K,N", [(3, 5459, 136, 264), (3, 32765, 48, 120), (1, 4090, 1040, 4090), (2, 2046, 1040, 4088), (5, 1639, 384, 1025), (1, 8190, 392, 4344), (3, 1531, 777, 333)])
def test_large_tiles(dtype, B, T, K, N):
    dev = torch.device("cuda")
    for act, gate, residual in ((None, True, True), ("gelu_tanh", False, True), ("silu", True, False), ("gelu", False, False)):
        run(dev, dtype, B, T, K, N, act, gate=gate, residual=residual, seed=N)


def test_largest_sums(dev):
    """Sums of 32 bits at their limit, weights of -128 among them."""
    K = 131072
    x = torch.ones(2, K, dtype=BF16, device=dev)
    x[1] = -1
    w = torch.full((3, K), 127, dtype=torch.int8, device=dev)
    w[1] = -128
    w[2, ::2] = -127
    y = llsa_amd.linear_int8(x, w, torch.ones(3, device=dev))
    step = step64(x.cpu())[0].double()
    ref = torch.tensor([[127.0 * K, -128.0 * K, 0], [-127.0 * K, 128.0 * K, 0]], dtype=torch.float64) * step * 127
    assert ((y.double().cpu() - ref).abs() <= ref.abs() * (half_step(BF16) + 4 * E)).all()


@pytest.mark.parametrize("K,T", [(40, 9), (48, 7)])
def test_rows_that_are_no_numbers(dev, K, T):
    """Quantised beforehand, and (up to sixteen rows, a multiple of sixteen long) in one launch with the product."""
    x, w, ws, b, g, r = layer(dev, BF16, 2, T, K, 24, True, True, True)
    plain = llsa_amd.linear_int8(x, w, ws, b, gate=g, residual=r)
    for bad in (float("nan"), float("inf"), -float("inf")):
        v = x.clone()
        v[1, 4, 3] = bad
        got = llsa_amd.linear_int8(v, w, ws, b, gate=g, residual=r)
        keep = torch.ones(2, T, dtype=torch.bool)
        keep[1, 4] = False
        assert torch.equal(got[keep.to(dev)], plain[keep.to(dev)]) and got[1, 4].isnan().all()
    v = x.clone()
    v[0, 2] = 0
    zero = llsa_amd.linear_int8(v, w, ws, b)[0, 2]
    assert torch.equal(zero, b)


def _layouts(v):
    yield torch.cat([v.new_zeros(1), v.reshape(-1)])[1:].view(v.shape)
    if v.dim() > 1:
        yield v.transpose(-1, -2).contiguous().transpose(-1, -2)
        yield torch.cat([v, v], -1)[..., :v.shape[-1]]
        yield torch.cat([v, v[..., :3]], -1)[..., :v.shape[-1]]
    if v.dim() > 2:
        yield v.transpose(0, 1).contiguous().transpose(0, 1)
        yield torch.stack([v, v], 2)[:, :, 1]
    if v.is_floating_point():
        yield torch.complex(torch.zeros_like(v, dtype=FP32), -v.float()).conj().imag if v.dtype == FP32 else v


@pytest.mark.parametrize("K,N", [(48, 40), (21, 13)])
def test_layouts(dev, K, N):
    names = ("x", "weight", "scale", "bias", "gate", "residual")
    given = dict(zip(names, layer(dev, BF16, 2, 7, K, N, True, True, True)))
    call = lambda t: llsa_amd.linear_int8(t["x"], t["weight"], t["scale"], t["bias"], activation="gelu", gate=t["gate"], residual=t["residual"])
    plain = call(given)
    for name in names:
        for v in _layouts(given[name]):
            assert torch.equal(v, given[name])
            assert torch.equal(call({**given, name: v}), plain), name
    q, s = llsa_amd.quantize_rows(given["x"])
    for v in _layouts(q):
        assert torch.equal(call({**given, "x": (v, s)}), plain)
    for v in _layouts(s):
        assert torch.equal(call({**given, "x": (q, v)}), plain)
    for v in _layouts(given["x"]):
        a, b = llsa_amd.quantize_rows(v)
        assert torch.equal(a, q) and torch.equal(b, s)
    assert torch.equal(llsa_amd.linear_int8(given["x"][0, 0], given["weight"], given["scale"]), llsa_amd.linear_int8(given["x"], given["weight"], given["scale"])[0, 0])


def test_no_rows(dev):
    x, w, ws, *_ = layer(dev, BF16, 2, 3, 16, 8, False, False, False)
    assert llsa_amd.linear_int8(x[:, :0], w, ws).shape == (2, 0, 8)
    q, s = llsa_amd.quantize_rows(x[:0])
    assert q.shape == (0, 3, 16) and s.shape == (0, 3)
    assert llsa_amd.linear_int8((q, s), w, ws).shape == (0, 3, 8)


def test_refusals(dev):
    x, w, ws, b, g, r = layer(dev, BF16, 2, 3, 16, 8, True, True, True)
    call = llsa_amd.linear_int8
    for bad, match in ((dict(x=x.float()), "bf16 or fp16"), (dict(x=x[..., :15]), "weight must be"), (dict(weight=w.float()), "int8"), (dict(scale=ws.half()), "float32"),
                       (dict(scale=ws[:7]), "scale must be"), (dict(bias=b.float()), "dtype"), (dict(bias=b[:7]), "bias must be"), (dict(gate=g[:1]), "gate must be"),
                       (dict(residual=r[:, :2]), "residual must be"), (dict(activation="relu"), "activation"), (dict(x=(x, ws)), "int8"), (dict(x=(w,)), "pair"),
                       (dict(x=(w[None, :, :], ws)), "scales of x"), (dict(x=(w, ws), dtype=torch.float32), "dtype"), (dict(weight=w[0]), "weight must be")):
        t = {"x": x, "weight": w, "scale": ws, "bias": b, "gate": g, "residual": r, **bad}
        if isinstance(t["x"], tuple):
            t.update(bias=None, gate=None, residual=None)
        with pytest.raises((ValueError, NotImplementedError), match=match):
            call(**t)
    for t in (x, b, g, r, ws):
        t.requires_grad_()
        with pytest.raises(NotImplementedError, match="no gradient"):
            call(x, w, ws, b, gate=g, residual=r)
        with torch.no_grad():
            call(x, w, ws, b, gate=g, residual=r)
        t.requires_grad_(False)
    with pytest.raises(NotImplementedError, match="no gradient"):
        llsa_amd.quantize_rows(x.clone().requires_grad_())
    with pytest.raises(NotImplementedError, match="131072"):
        call(torch.zeros(1, 131073, dtype=BF16, device=dev), torch.zeros(1, 131073, dtype=torch.int8, device=dev), ws[:1])
    with pytest.raises(NotImplementedError):
        llsa_amd.quantize_rows(x.double())
    with pytest.raises(ValueError):
        llsa_amd.quantize_rows(x[0, 0, 0])
    with pytest.raises(RuntimeError, match="functorch"):
        torch.func.vmap(lambda t: call(t, w, ws))(x)
    with pytest.raises(RuntimeError, match="torch.jit.trace"):
        torch.jit.trace(lambda t: call(t, w, ws), (x,), check_trace=False)


def test_cpu_tensors_are_refused():
    x, w, ws, *_ = layer(torch.device("cpu"), BF16, 2, 3, 16, 8, False, False, False)
    for f in (lambda: llsa_amd.linear_int8(x, w, ws), lambda: llsa_amd.quantize_rows(x)):
        with pytest.raises(RuntimeError, match="AMD GPU"):
            f()


@pytest.mark.gpu
def test_streams_and_graphs():
    dev = torch.device("cuda")
    x, w, ws, b, g, r = layer(dev, BF16, 2, 300, 777, 333, True, True, True)
    call = lambda v: llsa_amd.linear_int8(v, w, ws, b, activation="silu", gate=g, residual=r)
    plain = call(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call(x)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, plain)
    held = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        call(held)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = call(held)
    for k in range(4):
        held.copy_(x * (k + 1))
        graph.replay()
        assert torch.equal(out, call(x * (k + 1)))
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """Rows and results whose last element lies beyond 2^32 bytes."""
    dev = torch.device("cuda")
    M, K, N = 300001, 32, 8192                                # out: 4.9 GB
    g = torch.Generator(device=dev).manual_seed(3)
    x = torch.randn(M, K, generator=g, device=dev).to(BF16)
    w, ws = quantized64(torch.randn(N, K))
    w, ws = w.to(dev), ws.to(dev)
    y = llsa_amd.linear_int8(x, w, ws)
    for m in (0, 131071, 262143, 262145, M - 1):
        assert torch.equal(y[m], llsa_amd.linear_int8(x[m:m + 1], w, ws)[0])
