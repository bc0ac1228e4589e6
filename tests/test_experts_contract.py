"""What route_tokens, grouped_linear and expert_feed_forward owe their callers beside the numbers: refusals, autograd's rules, memory in any layout, empty inputs,
a caller's own routing, streams, threads, captured graphs, offsets beyond 32 bits."""
import contextlib
import threading

import pytest
import torch
import torch.autograd.forward_ad as fwAD

import llsa_amd
from emu_util import emu_lib
from llsa_amd._lib import override_library_for_tests

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
OPS = ["route", "grouped", "experts"]


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def dev(request):
    with contextlib.ExitStack() as stack:
        if request.param == "cpu":
            stack.enter_context(override_library_for_tests(emu_lib()))
        yield torch.device(request.param)


def _inputs(op, dev, dtype=BF16, B=2, T=9, n=4, C=24, F=40, grad=True, seed=0):
    """name -> tensor; all but the offsets differentiable"""
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, dt=dtype: (torch.randn(*s, generator=g) * 0.5).to(dt).to(dev).requires_grad_(grad)
    if op == "route":
        return {"logits": r(B, T, n)}
    if op == "grouped":
        cuts = torch.tensor([0, 3, 3, 11, B * T - 2][:n + 1] if n == 4 and B * T >= 13 else [0] * n + [B * T], dtype=torch.int32, device=dev)
        return {"x": r(B * T, C), "weight": r(n, F, C), "bias": r(n, F), "offsets": cuts}
    return {"x": r(B, T, C), "logits": r(B, T, n), "w_in": r(n, F, C), "b_in": r(n, F), "w_out": r(n, C, F), "b_out": r(n, C), "gate": r(B, C), "residual": r(B, T, C)}


def _call(op, t, act="silu"):
    if op == "route":
        return llsa_amd.route_tokens(t["logits"], 2, normalize=False).weights
    if op == "grouped":
        return llsa_amd.grouped_linear(t["x"], t["weight"], t["offsets"], t.get("bias"), activation=act)
    return llsa_amd.expert_feed_forward(t["x"], llsa_amd.route_tokens(t["logits"], 2), t["w_in"], t.get("b_in"), t["w_out"], t.get("b_out"), activation=act or "gelu", gate=t.get("gate"),
                                        residual=t.get("residual"))


def _leaves(t):
    return {n: v for n, v in t.items() if v.is_floating_point()}


def _dout(y):
    return torch.randn(y.shape, generator=torch.Generator().manual_seed(77)).to(y.dtype).to(y.device)


def _grads(op, t, act="silu", dout=None):
    y = _call(op, t, act)
    return [y.detach()] + list(torch.autograd.grad(y, list(_leaves(t).values()), _dout(y) if dout is None else dout))


def _same(a, b):
    assert len(a) == len(b)
    for i, (x, y) in enumerate(zip(a, b)):
        assert x.shape == y.shape and x.dtype == y.dtype and torch.equal(x, y), i


@pytest.mark.parametrize("op", OPS)
def test_tangents_and_transforms_are_refused(dev, op):
    for name in _leaves(_inputs(op, dev)):
        t = _inputs(op, dev, grad=False)
        with fwAD.dual_level():
            t[name] = fwAD.make_dual(t[name], torch.ones_like(t[name]))
            with pytest.raises(NotImplementedError, match="jvp"):
                _call(op, t)
    t = _inputs(op, dev, grad=False)
    name = "logits" if op == "route" else "x"
    call = lambda v: _call(op, {**t, name: v})
    for transform in (lambda: torch.func.vmap(call)(t[name][None]), lambda: torch.func.grad(lambda v: call(v).float().sum())(t[name])):
        with pytest.raises(RuntimeError, match="functorch transforms"):
            transform()
    with pytest.raises(RuntimeError, match="torch.jit.trace"):
        torch.jit.trace(call, (t[name],), check_trace=False)


@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("C,F", [(24, 40), (13, 21)])
def test_saved_tensors(dev, op, C, F):
    """Hooks that keep copies elsewhere and give them back unaligned, save_on_cpu, and both kinds of checkpoint change no bit."""
    from torch.utils.checkpoint import checkpoint
    make = lambda: _inputs(op, dev, C=C, F=F)

    def pack(t):
        room = torch.empty(t.numel() + 1, dtype=t.dtype)
        room[1:] = t.detach().reshape(-1).cpu()
        return room, t.shape

    plain = _grads(op, make())
    for ctx in (torch.autograd.graph.saved_tensors_hooks(pack, lambda p: p[0].to(dev)[1:].view(p[1])), torch.autograd.graph.save_on_cpu()):
        t = make()
        with ctx:
            y = _call(op, t)
        _same(plain, [y.detach()] + list(torch.autograd.grad(y, list(_leaves(t).values()), _dout(y))))
    for reentrant in (False, True):
        t = make()
        y = checkpoint(lambda *a: _call(op, dict(zip(t, a))), *t.values(), use_reentrant=reentrant)
        y.backward(_dout(y))
        _same(plain[1:], [v.grad for v in _leaves(t).values()])


@pytest.mark.parametrize("op", OPS)
def test_rules_of_autograd(dev, op):
    t = _inputs(op, dev)
    y = _call(op, t)
    y.sum().backward()
    with pytest.raises(RuntimeError, match="second time"):
        y.sum().backward()
    with pytest.raises(NotImplementedError, match="second derivative"):
        torch.autograd.grad(_call(op, t).sum(), list(_leaves(t).values()), create_graph=True)
    for name in {"route": ["logits"], "grouped": ["weight", "offsets"], "experts": ["logits", "w_in", "w_out", "gate"]}[op]:
        t = _inputs(op, dev)
        y = _call(op, t)
        with torch.no_grad():
            t[name].add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
    with pytest.raises(RuntimeError, match="another tensor"):
        with torch.autograd.graph.saved_tensors_hooks(lambda a: a, lambda a: a.reshape(-1)[:1]):
            y = _call(op, _inputs(op, dev))
        y.sum().backward()
    with torch.no_grad():
        assert not _call(op, _inputs(op, dev)).requires_grad


@pytest.mark.parametrize("op", ["grouped", "experts"])
@pytest.mark.parametrize("act", [None, "gelu_tanh"])
def test_gradients_that_are_asked_for(dev, op, act):
    """Any one of the inputs may be the only one that wants a gradient, or the only one that does not."""
    whole = dict(zip(["y"] + list(_leaves(_inputs(op, dev))), _grads(op, _inputs(op, dev), act)))
    for name in _leaves(_inputs(op, dev)):
        for alone in (True, False):
            t = _inputs(op, dev)
            for n, v in _leaves(t).items():
                v.requires_grad_((n == name) == alone)
            y = _call(op, t, act)
            wanted = [n for n, v in t.items() if v.requires_grad]
            assert torch.equal(y, whole["y"])
            _same([whole[n] for n in wanted], torch.autograd.grad(y, [t[n] for n in wanted], _dout(y)))
    for name in ("bias", "b_in", "b_out", "gate", "residual"):
        t = _inputs(op, dev)
        if name in t:
            del t[name]
            _grads(op, t, act)


def test_inference_takes_the_same_way(dev):
    """Without a backward few rows are gathered on their way into LDS; the results are the same bits."""
    for n, T in ((4, 9), (2, 70), (1, 3)):
        t = _inputs("experts", dev, n=max(n, 2), T=T)
        with torch.no_grad():
            y = _call("experts", t)
        assert torch.equal(y, _call("experts", t).detach())


def _layouts(v):
    """The same values in other layouts of memory"""
    yield torch.cat([v.new_zeros(1), v.reshape(-1)])[1:].view(v.shape)
    if v.dim() > 1:
        yield v.transpose(-1, -2).contiguous().transpose(-1, -2)
        yield torch.cat([v, v], -1)[..., :v.shape[-1]]
        yield torch.cat([v, v[..., :3]], -1)[..., :v.shape[-1]]
    if v.dim() > 2:
        yield v.transpose(0, 1).contiguous().transpose(0, 1)
        yield torch.stack([v, v], 2)[:, :, 1]
        yield torch.cat([v, v], 1)[:, :v.shape[1]]


@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("C,F", [(24, 40), (13, 21)])
def test_layouts(dev, op, C, F):
    make = lambda: _inputs(op, dev, C=C, F=F)
    plain = _grads(op, make())
    for name, v in make().items():
        for w in _layouts(v.detach()):
            t = make()
            assert torch.equal(w, v)
            t[name] = w.detach().requires_grad_(v.requires_grad)
            for i, (a, b) in enumerate(zip(plain, _grads(op, t))):
                assert torch.equal(a, b), (name, w.stride(), i)
    for w in _layouts(_dout(plain[0])):
        _same(plain, _grads(op, make(), dout=w))


def test_negated_views(dev):
    """Values of views that torch negates on reading"""
    neg = lambda v: torch.complex(torch.zeros_like(v, dtype=FP32), -v.float()).conj().imag
    l = torch.randn(2, 9, 4, device=dev)
    assert neg(l).is_neg()
    _same(list(llsa_amd.route_tokens(l, 2)), list(llsa_amd.route_tokens(neg(l), 2)))
    t = _inputs("experts", dev, grad=False)
    r = llsa_amd.route_tokens(l, 2)
    call = lambda r: llsa_amd.expert_feed_forward(t["x"], r, t["w_in"], None, t["w_out"])
    assert torch.equal(call(r), call(r._replace(weights=neg(r.weights))))


def test_expanded_inputs(dev):
    """One expert's weights for all, one row for all tokens: read as they are, gradients summed by autograd."""
    base = _inputs("experts", dev, B=1, T=1, n=1)
    logits = _inputs("experts", dev)["logits"].detach()
    wide = lambda v, n: v.expand(2, 9, v.shape[-1]) if n in ("x", "residual") else v.expand(2, v.shape[-1]) if n == "gate" else v.expand(4, *v.shape[1:])
    shared = {n: v.detach().requires_grad_() for n, v in base.items() if n != "logits"}
    copied = {n: wide(v, n).detach().contiguous().requires_grad_() for n, v in shared.items()}
    y = _call("experts", {**{n: wide(v, n) for n, v in shared.items()}, "logits": logits})
    z = _call("experts", {**copied, "logits": logits})
    assert torch.equal(y, z)
    dout = _dout(y)
    for n, a, b in zip(shared, torch.autograd.grad(y, list(shared.values()), dout), torch.autograd.grad(z, list(copied.values()), dout)):
        b = b.float()
        # (autograd adds up to 18 of them in bf16: as many half steps, 2^-8, of sums no larger than that of the magnitudes)
        assert ((a.float() - b.sum_to_size(a.shape)).abs() <= 18 * 2.0 ** -8 * b.abs().sum_to_size(a.shape) + 1e-6).all(), n
    one = torch.ones((), dtype=BF16, device=dev).expand_as(y)
    _same(torch.autograd.grad(_call("experts", {**copied, "logits": logits}), list(copied.values()), one),
          torch.autograd.grad(_call("experts", {**copied, "logits": logits}), list(copied.values()), one.contiguous()))


@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("B,T", [(0, 3), (2, 0)])
def test_no_rows(dev, op, B, T):
    t = _inputs(op, dev, B=B, T=T)
    got = _grads(op, t)
    assert got[0].numel() == 0
    for v, g in zip(_leaves(t).values(), got[1:]):
        assert g.shape == v.shape and not g.any()
    r = llsa_amd.route_tokens(torch.zeros(B, T, 5, device=dev), 3)
    assert r.weights.shape == r.places.shape == (B, T, 3) and r.order.shape == (0,) and not r.offsets.any() and r.offsets.shape == (6,)


def test_a_callers_routing(dev):
    """Weights of the caller's own; numbers that are out of range are held to it or skipped, and what else there is stays as it was."""
    t = _inputs("experts", dev, grad=False)
    r = llsa_amd.route_tokens(t["logits"], 2)
    call = lambda r: llsa_amd.expert_feed_forward(t["x"], r, t["w_in"], t["b_in"], t["w_out"], t["b_out"])
    plain = call(r)
    twice = call(r._replace(weights=r.weights * 2))
    assert torch.equal(twice.float(), (plain.float() * 2).to(BF16).float())
    assert not call(r._replace(weights=torch.zeros_like(r.weights))).any()
    wild = lambda v: torch.where(torch.arange(v.numel(), device=dev).view(v.shape) % 3 == 0, torch.full_like(v, (1 << 31) - 1), torch.full_like(v, -(1 << 31)))
    for bad in (dict(order=wild(r.order)), dict(offsets=wild(r.offsets)), dict(places=wild(r.places)), dict(order=wild(r.order), offsets=wild(r.offsets), places=wild(r.places))):
        x = t["x"].detach().requires_grad_()
        w = r.weights.detach().requires_grad_()
        y = llsa_amd.expert_feed_forward(x, r._replace(weights=w, **bad), t["w_in"], t["b_in"], t["w_out"], t["b_out"])
        assert y.shape == plain.shape
        torch.autograd.grad(y, [x, w], _dout(y))
        if list(bad) == ["places"]:
            assert not y.any()
    some = r.places.clone()
    some[0, 3] = -1
    got = call(r._replace(places=some))
    keep = torch.ones(2, 9, dtype=torch.bool)
    keep[0, 3] = False
    assert torch.equal(got[keep.to(dev)], plain[keep.to(dev)]) and not got[0, 3].any()


def test_what_is_in_a_row_stays_there(dev):
    """Infinities and NaN in one token, and rows of the lowest values."""
    for op in ("grouped", "experts"):
        t = _inputs(op, dev, T=9, grad=False)
        plain = _call(op, t)
        for bad in (float("nan"), float("inf"), -float("inf"), torch.finfo(BF16).min):
            t = _inputs(op, dev, T=9, grad=False)
            row = (4,) if op == "grouped" else (1, 4)
            t["x"][row + (3,)] = bad
            got = _call(op, t)
            keep = torch.ones(plain.shape[:-1], dtype=torch.bool)
            keep[row] = False
            assert torch.equal(got[keep.to(dev)], plain[keep.to(dev)])
            if bad != bad:
                assert got[row].isnan().all()


def test_refusals(dev):
    t = _inputs("grouped", dev, grad=False)
    for bad, match in ((dict(x=t["x"].float()), "bf16 or fp16"), (dict(x=t["x"][None]), "x must be"), (dict(x=t["x"][:, :23]), "weight must be"), (dict(weight=t["weight"][0]), "weight must be"),
                       (dict(weight=t["weight"].half()), "dtype"), (dict(offsets=t["offsets"].long()), "int32"), (dict(offsets=t["offsets"][:4]), "offsets must be"), (dict(bias=t["bias"][:2]), "bias must be"),
                       (dict(bias=t["bias"].float()), "dtype"), (dict(activation="relu"), "activation"), (dict(weight=t["weight"].repeat(65, 1, 1), offsets=torch.zeros(261, dtype=torch.int32, device=dev)), "256 experts")):
        with pytest.raises((ValueError, NotImplementedError), match=match):
            llsa_amd.grouped_linear(**{**t, **bad})
    l = torch.zeros(3, 8, device=dev)
    for bad, match in ((dict(logits=l.double()), "bf16, fp16 or fp32"), (dict(experts_per_token=0), "experts_per_token"), (dict(experts_per_token=9), "experts_per_token"),
                       (dict(logits=torch.zeros(3, 257, device=dev)), "256 experts"), (dict(logits=torch.zeros((), device=dev)), "experts"), (dict(logits=torch.zeros(3, 0, device=dev)), "experts"),
                       (dict(logits=torch.zeros(2, 64, device=dev), experts_per_token=17), "experts_per_token")):
        with pytest.raises((ValueError, NotImplementedError), match=match):
            llsa_amd.route_tokens(**{"logits": l, "experts_per_token": 2, **bad})
    t = _inputs("experts", dev, grad=False)
    r = llsa_amd.route_tokens(t.pop("logits"), 2)
    full = {**t, "routing": r}
    for bad, match in ((dict(x=t["x"].float()), "bf16 or fp16"), (dict(x=t["x"][..., :23]), "w_in must be"), (dict(w_out=t["w_out"][:3]), "w_out must be"), (dict(w_out=t["w_out"][..., :39]), "w_out must be"),
                       (dict(b_in=t["b_in"][:, :3]), "b_in must be"), (dict(b_out=t["b_out"].half()), "dtype"), (dict(gate=t["gate"][:1]), "gate must be"), (dict(residual=t["residual"][:, :2]), "residual must be"),
                       (dict(activation=None), "needs an activation"), (dict(x=t["x"][:, :8], residual=None), "routing"), (dict(routing=r._replace(weights=r.weights.to(BF16))), "float32"),
                       (dict(routing=r._replace(weights=r.weights[:1])), "routing.weights"), (dict(routing=r._replace(order=r.order.long())), "int32"), (dict(routing=r._replace(order=r.order[1:])), "routing.order"),
                       (dict(routing=r._replace(offsets=r.offsets[1:])), "routing.offsets"), (dict(routing=r._replace(places=r.places[..., :1])), "routing.places"),
                       (dict(routing=r._replace(experts=r.experts[..., :1])), "routing.experts")):
        with pytest.raises((ValueError, NotImplementedError), match=match):
            llsa_amd.expert_feed_forward(**{**full, **bad})


def test_cpu_tensors_are_refused():
    for op in OPS:
        with pytest.raises(RuntimeError, match="AMD GPU"):
            _call(op, _inputs(op, torch.device("cpu")))


def test_the_entry_points_check():
    """Rejected before a kernel is launched: no GPU needed."""
    import ctypes as C
    from llsa_amd._lib import ExpertsArgs, Int8Args, LIB_PATH, Lib, QuantizeArgs, RouteArgs
    lib = Lib(LIB_PATH)
    none = C.c_void_p()
    for f in (lib.route_tokens, lib.route_tokens_bwd, lib.experts_gather, lib.experts_fwd, lib.experts_dx, lib.experts_dw, lib.experts_combine, lib.experts_dweights, lib.quantize_rows, lib.linear_int8):
        assert f(None, none) != 0
    r = RouteArgs()
    r.E, r.k, r.M = 8, 2, 4
    assert lib.route_tokens(C.byref(r), none) != 0 and b"logits" in lib.last_error_string()
    for E, k, M in ((0, 1, 1), (257, 1, 1), (8, 0, 1), (8, 9, 1), (32, 17, 1), (8, 2, 1 << 28)):
        r.E, r.k, r.M = E, k, M
        assert lib.route_tokens(C.byref(r), none) != 0
    a = ExpertsArgs()
    a.rows, a.tokens, a.k, a.E, a.N, a.K = 16, 16, 1, 2, 8, 8
    assert lib.experts_fwd(C.byref(a), none) != 0 and b"offsets" in lib.last_error_string()
    a.offsets = 16
    for f, text in ((lib.experts_fwd, b"16-byte aligned"), (lib.experts_dx, b"16-byte aligned"), (lib.experts_dw, b"16-byte aligned"), (lib.experts_gather, b"order"), (lib.experts_combine, b"16-byte"),
                    (lib.experts_dweights, b"places")):
        assert f(C.byref(a), none) != 0 and text in lib.last_error_string(), text
    a.rows = (1 << 28) + 1
    assert lib.experts_fwd(C.byref(a), none) != 0
    q = QuantizeArgs()
    q.rows, q.K = 4, 16
    assert lib.quantize_rows(C.byref(q), none) != 0
    i = Int8Args()
    i.M, i.N, i.K = 4, 8, 131073
    assert lib.linear_int8(C.byref(i), none) != 0 and b"131072" in lib.last_error_string()
    assert lib.experts_dw_workspace_bytes(100, 4, 8, 8) > 0 and lib.experts_dw_workspace_bytes(0, 4, 8, 8) == 0 and lib.route_workspace_bytes(100, 8, 2) == 0 < lib.route_workspace_bytes(100000, 8, 2)


@pytest.mark.gpu
def test_streams_and_threads():
    dev = torch.device("cuda")
    for op in OPS:
        plain = _grads(op, _inputs(op, dev, T=300, C=72, F=136))
        results, errors = [None] * 4, []

        def work(i):
            try:
                stream = torch.cuda.Stream()
                with torch.cuda.stream(stream):
                    for _ in range(3):
                        results[i] = _grads(op, _inputs(op, dev, T=300, C=72, F=136))
                stream.synchronize()
            except Exception as e:                            # noqa: BLE001
                errors.append(e)
        threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not errors
        for r in results:
            _same(plain, r)


@pytest.mark.gpu
@pytest.mark.parametrize("op,size", [("route", {}), ("grouped", {}), ("experts", {}), ("experts", dict(B=4, T=800, n=8, C=384, F=768))])
def test_captured_steps(op, size):
    """Forward and backward in one graph, replayed with other inputs, with eager work between the replays; two graphs that run one after the other."""
    dev = torch.device("cuda")
    t = _inputs(op, dev, **size)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            _grads(op, t)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    y = _call(op, t)
    dout = _dout(y)
    del y
    graphs, captured = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for g in graphs:
        with torch.cuda.graph(g):
            captured.append(_grads(op, t, dout=dout))
    for seed in (1, 2, 3):
        new = _inputs(op, dev, seed=seed, **size)
        with torch.no_grad():
            for n, v in new.items():
                t[n].copy_(v)
        eager = [v.clone() for v in _grads(op, new, dout=dout)]
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for c in captured:
            _same(eager, c)


@pytest.mark.gpu
def test_the_same_bits_every_time():
    dev = torch.device("cuda")
    t = _inputs("experts", dev, B=4, T=3000, n=8, C=384, F=768)
    first = _grads("experts", t)
    for _ in range(3):
        _same(first, _grads("experts", t))


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """Rows, results and hidden rows whose last element lies beyond 2^32 bytes."""
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(1)
    rows, K, N = 300001, 32, 8192                             # 4.9 GB
    x, w = torch.randn(rows, K, generator=g, device=dev).to(BF16), torch.randn(3, N, K, generator=g, device=dev).to(BF16)
    offsets = torch.tensor([0, 100, 290000, rows], dtype=torch.int32, device=dev)
    y = llsa_amd.grouped_linear(x, w, offsets)
    at = lambda m: 0 if m < 100 else 1 if m < 290000 else 2
    for m in (0, 99, 100, 262143, 262145, 289999, 290000, rows - 1):
        assert torch.equal(y[m], llsa_amd.linear(x[m:m + 1], w[at(m)])[0])
    del y
    tokens, n = 200001, 4                                     # hidden rows: 6.6 GB
    x, logits = torch.randn(tokens, 32, generator=g, device=dev).to(BF16), torch.randn(tokens, n, generator=g, device=dev)
    w1, w2 = torch.randn(n, N, 32, generator=g, device=dev).to(BF16), (torch.randn(n, 32, N, generator=g, device=dev) * 0.01).to(BF16)
    x.requires_grad_()
    y = llsa_amd.expert_feed_forward(x, llsa_amd.route_tokens(logits, 2), w1, None, w2)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    pick = torch.tensor([0, 100000, 131073, 199999, tokens - 1], device=dev)
    xs = x.detach()[pick].requires_grad_()
    ys = llsa_amd.expert_feed_forward(xs, llsa_amd.route_tokens(logits[pick], 2), w1, None, w2)
    ds, = torch.autograd.grad(ys, xs, torch.ones_like(ys))
    # (other tiles add up in another order: sums of 8192 in fp32, 2^-11 of the sum of magnitudes at the worst, and two roundings to bf16 on the way)
    for a, b in ((y[pick], ys), (dx[pick], ds)):
        assert (a.float() - b.float()).abs().max() <= 2.0 ** -5 * b.float().abs().max()
