"""What layer_norm, linear and feed_forward owe their callers beside the numbers: refusals, autograd's rules, memory in any layout, empty inputs, streams,
threads, captured graphs, offsets beyond 32 bits."""
import contextlib
import threading

import pytest
import torch
import torch.autograd.forward_ad as fwAD

import llsa_amd
from emu_util import emu_lib
from llsa_amd._lib import override_library_for_tests

BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def dev(request):
    with contextlib.ExitStack() as stack:
        if request.param == "cpu":
            stack.enter_context(override_library_for_tests(emu_lib()))
        yield torch.device(request.param)


def _inputs(op, dev, dtype=BF16, B=2, T=7, C=24, F=40, grad=True, seed=0):
    """name -> tensor, in the order of the call"""
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: (torch.randn(*s, generator=g) * 0.5).to(dtype).to(dev).requires_grad_(grad)
    if op == "norm":
        return {"x": r(B, T, C), "weight": r(C), "bias": r(C), "scale": r(B, C), "shift": r(B, C)}
    if op == "linear":
        return {"x": r(B, T, C), "weight": r(F, C), "bias": r(F), "gate": r(B, F), "residual": r(B, T, F)}
    return {"x": r(B, T, C), "w_in": r(F, C), "b_in": r(F), "w_out": r(C, F), "b_out": r(C), "gate": r(B, C), "residual": r(B, T, C)}


def _call(op, t, act="gelu_tanh"):
    if op == "norm":
        return llsa_amd.layer_norm(t["x"], t.get("weight"), t.get("bias"), scale=t.get("scale"), shift=t.get("shift"))
    if op == "linear":
        return llsa_amd.linear(t["x"], t["weight"], t.get("bias"), activation=act, gate=t.get("gate"), residual=t.get("residual"))
    return llsa_amd.feed_forward(t["x"], t["w_in"], t.get("b_in"), t["w_out"], t.get("b_out"), activation=act, gate=t.get("gate"), residual=t.get("residual"))


OPS = ["norm", "linear", "ffn"]


def _grads(op, t, act="gelu_tanh", dout=None):
    y = _call(op, t, act)
    dout = torch.randn(y.shape, generator=torch.Generator().manual_seed(77)).to(y.dtype).to(y.device) if dout is None else dout
    return [y.detach()] + list(torch.autograd.grad(y, list(t.values()), dout))


def _same(a, b):
    assert len(a) == len(b)
    for i, (x, y) in enumerate(zip(a, b)):
        assert x.shape == y.shape and x.dtype == y.dtype and torch.equal(x, y), i


@pytest.mark.parametrize("op", OPS)
def test_tangents_and_transforms_are_refused(dev, op):
    names = list(_inputs(op, dev))
    for name in names:
        t = _inputs(op, dev, grad=False)
        with fwAD.dual_level():
            t[name] = fwAD.make_dual(t[name], torch.ones_like(t[name]))
            with pytest.raises(NotImplementedError, match="jvp"):
                _call(op, t)
    t = _inputs(op, dev, grad=False)
    for transform in (lambda f: torch.func.vmap(f)(t["x"][None]), lambda f: torch.func.grad(lambda x: f(x).float().sum())(t["x"])):
        with pytest.raises(RuntimeError, match="functorch transforms"):
            transform(lambda x: _call(op, {**t, "x": x}))
    with pytest.raises(RuntimeError, match="torch.jit.trace"):
        torch.jit.trace(lambda x: _call(op, {**t, "x": x}), (t["x"],), check_trace=False)


@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("C,F,T", [(24, 40, 7), (13, 21, 7), (8, 8, 50)])
def test_saved_tensors(dev, op, C, F, T):
    """Hooks that keep copies elsewhere and give them back unaligned, save_on_cpu, and both kinds of checkpoint change no bit."""
    from torch.utils.checkpoint import checkpoint
    make = lambda: _inputs(op, dev, T=T, C=C, F=F)

    def pack(t):
        room = torch.empty(t.numel() + 1, dtype=t.dtype)
        room[1:] = t.detach().reshape(-1).cpu()
        return room, t.shape

    plain = _grads(op, make(), None if op == "linear" else "silu")
    for ctx in (torch.autograd.graph.saved_tensors_hooks(pack, lambda p: p[0].to(dev)[1:].view(p[1])), torch.autograd.graph.save_on_cpu()):
        t = make()
        with ctx:
            y = _call(op, t, None if op == "linear" else "silu")
        dout = torch.randn(y.shape, generator=torch.Generator().manual_seed(77)).to(y.dtype).to(dev)
        _same(plain, [y.detach()] + list(torch.autograd.grad(y, list(t.values()), dout)))
    t = make()
    y = checkpoint(lambda *a: _call(op, dict(zip(t, a)), None if op == "linear" else "silu"), *t.values(), use_reentrant=False)
    dout = torch.randn(y.shape, generator=torch.Generator().manual_seed(77)).to(y.dtype).to(dev)
    _same(plain, [y.detach()] + list(torch.autograd.grad(y, list(t.values()), dout)))
    t = make()
    checkpoint(lambda *a: _call(op, dict(zip(t, a)), None if op == "linear" else "silu"), *t.values(), use_reentrant=True).backward(dout)
    _same(plain[1:], [v.grad for v in t.values()])


@pytest.mark.parametrize("op", OPS)
def test_rules_of_autograd(dev, op):
    t = _inputs(op, dev)
    y = _call(op, t)
    y.sum().backward()
    with pytest.raises(RuntimeError, match="second time"):
        y.sum().backward()
    y = _call(op, t)
    with pytest.raises(NotImplementedError, match="second derivative"):
        torch.autograd.grad(y.sum(), list(t.values()), create_graph=True)
    t = _inputs(op, dev)
    y = _call(op, t)
    with torch.no_grad():
        t["x"].add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with pytest.raises(RuntimeError, match="another tensor"):
        with torch.autograd.graph.saved_tensors_hooks(lambda a: a, lambda a: a.reshape(-1)[:1]):
            y = _call(op, _inputs(op, dev))
        y.sum().backward()
    with torch.no_grad():
        assert not _call(op, _inputs(op, dev)).requires_grad


@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("T,act", [(7, "gelu_tanh"), (50, None), (90, "silu")])
def test_gradients_that_are_asked_for(dev, op, T, act):
    """Any one of the inputs may be the only one that wants a gradient, or the only one that does not."""
    if op == "ffn" and act is None:
        act = "gelu"
    whole = dict(zip(["y"] + list(_inputs(op, dev)), _grads(op, _inputs(op, dev, T=T), act)))
    for name in _inputs(op, dev):
        for alone in (True, False):
            t = _inputs(op, dev, T=T)
            for n, v in t.items():
                v.requires_grad_((n == name) == alone)
            y = _call(op, t, act)
            dout = torch.randn(y.shape, generator=torch.Generator().manual_seed(77)).to(y.dtype).to(dev)
            wanted = [n for n, v in t.items() if v.requires_grad]
            assert torch.equal(y, whole["y"])
            _same([whole[n] for n in wanted], torch.autograd.grad(y, [t[n] for n in wanted], dout))


def _layouts(v):
    """The same values in other layouts of memory"""
    yield "offset", torch.cat([v.new_zeros(1), v.reshape(-1)])[1:].view(v.shape)
    if v.dim() > 1:
        yield "columns", v.transpose(-1, -2).contiguous().transpose(-1, -2)
        wide = torch.cat([v, v.new_full(v.shape, 7)], -1)
        yield "slice", wide[..., :v.shape[-1]]
        odd = torch.cat([v, v.new_full(v.shape[:-1] + (3,), 7)], -1)
        yield "odd slice", odd[..., :v.shape[-1]]
    if v.dim() > 2:
        yield "middle", v.transpose(0, 1).contiguous().transpose(0, 1)
        yield "rows apart", torch.stack([v, v], 2)[:, :, 1]
        yield "part of longer samples", torch.cat([v, v], 1)[:, :v.shape[1]]


@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("C,F", [(24, 40), (13, 21)])
def test_layouts(dev, op, C, F):
    make = lambda: _inputs(op, dev, C=C, F=F)
    for act in (None, "gelu") if op == "linear" else ("gelu",):
        plain = _grads(op, make(), act)
        for name, v in make().items():
            for kind, w in _layouts(v.detach()):
                t = make()
                assert torch.equal(w, v)
                t[name] = w.detach().requires_grad_()
                got = _grads(op, t, act)
                for i, (a, b) in enumerate(zip(plain, got)):
                    assert torch.equal(a, b), (name, kind, i)
        for kind, w in _layouts(torch.randn(plain[0].shape, generator=torch.Generator().manual_seed(77)).to(BF16).to(dev)):
            _same(plain, _grads(op, make(), act, dout=w))


@pytest.mark.parametrize("op", OPS)
def test_expanded_inputs(dev, op):
    """One row of memory for several: read as it is, and its gradient is the sum of theirs."""
    base = _inputs(op, dev, B=1, T=1)
    leaf = {n: v.detach().requires_grad_() for n, v in base.items()}
    wide = {n: v.expand(3, 5, v.shape[-1]) if v.dim() == 3 else v.expand(3, v.shape[-1]) if n in ("gate", "scale", "shift") else v for n, v in leaf.items()}
    copied = {n: v.detach().contiguous().requires_grad_() for n, v in wide.items()}
    y, z = _call(op, wide), _call(op, copied)
    assert torch.equal(y, z)
    dout = torch.randn(y.shape, generator=torch.Generator().manual_seed(3)).to(BF16).to(dev)
    for n, a, b in zip(leaf, torch.autograd.grad(y, list(leaf.values()), dout), torch.autograd.grad(z, list(copied.values()), dout)):
        b = b.sum_to_size(a.shape) if b.dtype != BF16 or a.shape == b.shape else b.float().sum_to_size(a.shape)
        # (autograd adds up to 15 rows in bf16: 15 roundings of half a step, 2^-8, of sums no larger than that of the magnitudes)
        size = b.abs().max() + dout.float().abs().max()
        assert (a.float() - b.float()).abs().max() <= 16 * 2 ** -8 * max(1.0, size.item()) * 4, n
    one = torch.ones((), dtype=BF16, device=dev).expand_as(y)                # a gradient out of a sum: no memory of its own
    _same(torch.autograd.grad(_call(op, copied), list(copied.values()), one), torch.autograd.grad(_call(op, copied), list(copied.values()), one.contiguous()))


@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("B,T", [(0, 3), (2, 0)])
def test_no_rows(dev, op, B, T):
    t = _inputs(op, dev, B=B, T=T)
    got = _grads(op, t)
    assert got[0].shape[:2] == (B, T)
    for v, g in zip(t.values(), got[1:]):
        assert g.shape == v.shape and not g.any()
    with torch.no_grad():
        assert _call(op, t).shape[:2] == (B, T)


def test_plain_shapes(dev):
    """Without samples: single vectors, matrices, more dimensions."""
    g = torch.Generator().manual_seed(1)
    x, w = (torch.randn(s, generator=g).to(BF16).to(dev) for s in ((2, 3, 4, 16), (8, 16)))
    rows = llsa_amd.linear(x.reshape(-1, 16), w)
    assert torch.equal(llsa_amd.linear(x, w), rows.view(2, 3, 4, 8))
    assert torch.equal(llsa_amd.linear(x[0, 0, 0], w), rows[0])
    n = llsa_amd.layer_norm(x)
    assert torch.equal(llsa_amd.layer_norm(x.reshape(-1, 16)), n.view(-1, 16)) and torch.equal(llsa_amd.layer_norm(x[0, 0, 0]), n[0, 0, 0])
    gate = torch.randn(2, 8, generator=g).to(BF16).to(dev)
    each = llsa_amd.linear(x.reshape(2, 12, 16), w, gate=gate)
    assert torch.equal(llsa_amd.linear(x, w, gate=gate), each.view(2, 3, 4, 8))
    per_row = llsa_amd.linear(x.reshape(-1, 16), w, gate=gate.repeat_interleave(12, 0))
    assert torch.equal(per_row.view(2, 12, 8), each)


def test_what_is_in_a_row_stays_there(dev):
    """Infinities and NaN in one row, and rows of the lowest values."""
    for op in OPS:
        t = _inputs(op, dev, T=9, grad=False)
        plain = _call(op, t)
        for bad in (float("nan"), float("inf"), -float("inf"), torch.finfo(BF16).min):
            t = _inputs(op, dev, T=9, grad=False)
            t["x"][1, 4, 3] = bad
            got = _call(op, t)
            keep = torch.ones(2, 9, dtype=torch.bool)
            keep[1, 4] = False
            assert torch.equal(got[keep.to(dev)], plain[keep.to(dev)])
            if bad != bad:
                assert got[1, 4].isnan().all()
    x = torch.full((1, 4, 40), 3.0, device=dev).to(BF16)                      # rows without any variance
    y = llsa_amd.layer_norm(x.requires_grad_())
    assert not y.any()
    assert torch.isfinite(torch.autograd.grad(y, x, torch.ones_like(y))[0]).all()


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_far_arguments_of_activations(dev, act):
    """act and act' where the activation is 0 or the identity to the last bit."""
    z = torch.tensor([-1e4, -300.0, -40.0, -17.0, -16.0, 16.0, 17.0, 40.0, 300.0, 1e4])
    x = z[:, None].to(BF16).to(dev).requires_grad_()
    w = torch.ones(1, 1, device=dev).to(BF16)
    y = llsa_amd.linear(x, w, activation=act)
    d, = torch.autograd.grad(y, x, torch.ones_like(y))
    v = x.detach().double().cpu().requires_grad_()
    ref = {"silu": lambda t: t * torch.sigmoid(t), "gelu": lambda t: t * 0.5 * torch.erfc(-t / 2 ** 0.5),
           "gelu_tanh": lambda t: t * torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (t + 0.044715 * t ** 3))}[act](v)
    rd, = torch.autograd.grad(ref.sum(), v)
    # half a step of bf16, and 2^-20 of |z| (of 1) for the activation (its slope) in fp32
    assert ((y.double().cpu() - ref.detach()).abs() <= 2.0 ** -8 * ref.detach().abs() + 2.0 ** -20 * v.detach().abs()).all()
    assert ((d.double().cpu() - rd).abs() <= 2.0 ** -8 * rd.abs() + 2.0 ** -18).all()


def test_refusals(dev):
    other = torch.device("meta")
    for op in OPS:
        good = _inputs(op, dev, grad=False)
        for name, v in good.items():
            with pytest.raises(ValueError, match="one device" if name != "x" else "one device"):
                _call(op, {**good, name: v.to(other)})
            wrong = {"x": None, "w_out": (24, 41), "w_in": (40, 25), "weight": (25,) if op == "norm" else (40, 25)}.get(name, tuple(v.shape[:-1]) + (v.shape[-1] + 1,))
            if wrong is not None:
                with pytest.raises(ValueError, match=name):
                    _call(op, {**good, name: torch.zeros(wrong, dtype=BF16, device=dev)})
            if op != "norm" and name != "x":
                with pytest.raises(ValueError, match="dtype"):
                    _call(op, {**good, name: v.float()})
        for dtype in (torch.float64, torch.int32, torch.float8_e4m3fn) + ((torch.float32,) if op != "norm" else ()):
            with pytest.raises(NotImplementedError, match=f"got {dtype}"):
                _call(op, {n: v.to(dtype) for n, v in good.items()})
        for name in set(good) & {"gate", "scale", "shift"}:
            with pytest.raises(ValueError):
                _call(op, {**good, name: torch.zeros(3, good[name].shape[-1], dtype=BF16, device=dev)})
    t = _inputs("norm", dev, grad=False)
    with pytest.raises(ValueError, match="torch.float32"):
        llsa_amd.layer_norm(t["x"], t["weight"].half())
    with pytest.raises(ValueError, match="samples"):
        llsa_amd.layer_norm(t["x"][0, 0], scale=t["scale"])
    with pytest.raises(NotImplementedError, match="8192"):
        llsa_amd.layer_norm(torch.zeros(2, 8193, device=dev))
    with pytest.raises(NotImplementedError, match="channels"):
        llsa_amd.layer_norm(torch.zeros(2, 0, device=dev))
    t = _inputs("linear", dev, grad=False)
    with pytest.raises(ValueError, match="activation"):
        llsa_amd.linear(t["x"], t["weight"], activation="relu6")
    with pytest.raises(ValueError, match="weight"):
        llsa_amd.linear(t["x"], t["weight"][0])
    with pytest.raises(ValueError, match="weight"):
        llsa_amd.linear(t["x"], t["weight"][:0])
    with pytest.raises(ValueError, match="samples"):
        llsa_amd.linear(t["x"][0, 0], t["weight"], gate=t["gate"])
    with pytest.raises(ValueError, match="activation"):
        llsa_amd.feed_forward(t["x"], t["weight"], None, t["weight"].t().contiguous(), activation=None)
    if dev.type == "cuda":
        with pytest.raises(RuntimeError, match="AMD GPU only"):
            llsa_amd.linear(t["x"].cpu(), t["weight"].cpu())


def test_c_calls_are_checked():
    """The C entry points reject what the kernels could not take, and launch nothing."""
    import ctypes as C
    from llsa_amd._lib import LIB_PATH, LayerNormArgs, Lib, LinearArgs, PadJob
    lib = Lib(LIB_PATH)
    bad = lambda fn, a, text: (fn(C.byref(a), None) != 0 and text in lib.last_error_string())
    a = LinearArgs()
    assert bad(lib.linear_fwd, a, b"bad sizes") and bad(lib.linear_dx, a, b"bad sizes") and bad(lib.linear_dw, a, b"bad sizes")
    a.M, a.N, a.K, a.dtype = 8, 8, 8, 1
    assert bad(lib.linear_fwd, a, b"bf16 or fp16")
    a.dtype, a.act = 0, 9
    assert bad(lib.linear_fwd, a, b"activation")
    a.act = 0
    a.x = a.w = a.out = a.dz = a.dz_out = a.dout = a.workspace = 1 << 20
    a.ldx = a.ldw = a.ldo = a.lddz = a.lddout = 8
    for field, value in (("x", 8 + (1 << 20)), ("ldx", 12), ("ldw", 4), ("ldx", 1 << 24), ("K", 7)):
        keep, _ = getattr(a, field), setattr(a, field, value)
        assert bad(lib.linear_fwd, a, b"16-byte aligned"), field
        setattr(a, field, keep)
    a.gate = 1 << 20
    assert bad(lib.linear_fwd, a, b"rows of a sample") and bad(lib.linear_dz, a, b"rows of a sample") and bad(lib.linear_dw, a, b"whole samples")
    a.per_sample = 3
    assert bad(lib.linear_dw, a, b"whole samples") and bad(lib.linear_gate_rows, a, b"whole samples")
    a.gate, a.per_sample, a.lddz = None, 8, 4
    assert bad(lib.linear_dx, a, b"padded") and bad(lib.linear_dw, a, b"padded") and bad(lib.linear_dz, a, b"padded")
    a.lddz, a.M = 8, (1 << 31) - 1
    assert bad(lib.linear_fwd, a, b"bad sizes")
    a.M, a.act = 8, 1
    assert bad(lib.linear_dz, a, b"z is needed")
    n = LayerNormArgs()
    assert bad(lib.layer_norm_fwd, n, b"channels")
    n.C, n.rows, n.per_sample = 8, 5, 3
    assert bad(lib.layer_norm_fwd, n, b"rows of a sample")
    n.per_sample, n.dtype = 5, 7
    assert bad(lib.layer_norm_fwd, n, b"bf16, fp16 or fp32")
    n.dtype, n.vtype = 0, 2
    assert bad(lib.layer_norm_fwd, n, b"rows' type")
    n.vtype = 0
    n.x = n.y = 1 << 20
    assert bad(lib.layer_norm_bwd, n, b"statistics")
    n.dy = n.stats = n.dweight = 1 << 20
    assert bad(lib.layer_norm_bwd, n, b"workspace")
    jobs = (PadJob * 2)()
    assert lib.pad_rows(jobs, 0, None) != 0 and lib.pad_rows(jobs, 5, None) != 0 and lib.pad_rows(jobs, 2, None) != 0
    assert lib.linear_dw_workspace_bytes(0, 1, 8, 8) == 0 and lib.layer_norm_bwd_workspace_bytes(8, 8, 9000) == 0


def test_a_run_of_them(dev):
    """The block they are made for: norm, gated projection onto the residual stream, norm, feed-forward, against 64 bits."""
    g = torch.Generator().manual_seed(5)
    B, T, C = 2, 33, 40
    r = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).to(BF16)
    t = [r(B, T, C), r(B, 6 * C, std=0.3), r(C, C, std=C ** -0.5), r(C, std=0.1), r(4 * C, C, std=C ** -0.5), r(4 * C, std=0.1), r(C, 4 * C, std=(4 * C) ** -0.5), r(C, std=0.1)]
    dout = r(B, T, C)

    def block(x, mod, w, b, w1, b1, w2, b2, ops):
        sh1, sc1, g1, sh2, sc2, g2 = mod.chunk(6, 1)
        h = ops.layer_norm(x, scale=sc1, shift=sh1, eps=1e-6)
        x = ops.linear(h, w, b, gate=g1, residual=x)
        h = ops.layer_norm(x, scale=sc2, shift=sh2, eps=1e-6)
        return ops.feed_forward(h, w1, b1, w2, b2, gate=g2, residual=x)

    class Ops64:
        @staticmethod
        def layer_norm(x, scale, shift, eps):
            d = x - x.mean(-1, keepdim=True)
            return d * (d.square().mean(-1, keepdim=True) + eps).rsqrt() * (1 + scale[:, None]) + shift[:, None]

        @staticmethod
        def linear(x, w, b, gate, residual):
            return residual + gate[:, None] * (x @ w.t() + b)

        @staticmethod
        def feed_forward(x, w1, b1, w2, b2, gate, residual):
            z = x @ w1.t() + b1
            return residual + gate[:, None] * ((z * torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (z + 0.044715 * z ** 3))) @ w2.t() + b2)

    got = [v.to(dev).requires_grad_() for v in t]
    y = block(*got, llsa_amd)
    grads = torch.autograd.grad(y, got, dout.to(dev))
    ref = [v.double().requires_grad_() for v in t]
    ry = block(*ref, Ops64)
    rgrads = torch.autograd.grad(ry, ref, dout.double())
    # at most a dozen roundings of bf16 (2^-9 in the mean) between an input and any of these: 12^0.5 2^-9 = 0.7 %; held to twice that
    for a, b in zip((y,) + grads, (ry,) + rgrads):
        a, b = a.detach().double().cpu(), b.detach()
        assert (a - b).norm() <= 1.5e-2 * b.norm()


def test_against_differences(dev):
    """Gradients against differences of the operator's own outputs: layer_norm in fp32; linear, which is linear in each of its inputs without an activation."""
    g = torch.Generator().manual_seed(9)
    r = lambda *s: torch.randn(*s, generator=g).to(dev)
    x, w, b, sc, sh = (v.requires_grad_() for v in (r(2, 5, 24), r(24), r(24), r(2, 24), r(2, 24)))
    f = lambda *a: llsa_amd.layer_norm(a[0], a[1], a[2], scale=a[3], shift=a[4], eps=1e-3)
    leaves, dout = [x, w, b, sc, sh], r(2, 5, 24)
    grads = torch.autograd.grad(f(*leaves), leaves, dout)
    for i, v in enumerate(leaves):
        d, h = r(*v.shape), 2.0 ** -6
        moved = lambda s: [u.detach() + s * h * d if j == i else u.detach() for j, u in enumerate(leaves)]
        slope = ((f(*moved(1)).double() - f(*moved(-1)).double()) * dout.double()).sum() / (2 * h)
        # the difference quotient's own error: h^2 times a third derivative (rows of 24 values of order 1), and rounding 2^-24 / h
        assert abs(slope - (grads[i].double() * d.double()).sum()) <= 2e-3 * (grads[i].double() * d.double()).abs().sum() + 1e-4
    t = {n: v.float() for n, v in _inputs("linear", dev, B=2, T=50, C=16, F=24, grad=False).items()}
    ints = {n: torch.randint(-3, 4, v.shape, generator=g).to(dev).to(BF16).requires_grad_() for n, v in t.items()}
    dout = torch.randint(-1, 2, (2, 50, 24), generator=g).to(dev).to(BF16)
    call = lambda q: llsa_amd.linear(q["x"], q["weight"], q["bias"], gate=q["gate"], residual=q["residual"])
    grads = dict(zip(ints, torch.autograd.grad(call(ints), list(ints.values()), dout)))
    for n, v in ints.items():                                 # whole numbers: outputs below 2^8 in 16 bits, so most differences are exact; sums of 2400 roundings of half a step else
        step = torch.zeros_like(v)
        step.view(-1)[:: 7] = 1
        q = {k: u.detach() for k, u in ints.items()}
        up = (call({**q, n: q[n] + step}).double() * dout.double()).sum() - (call(q).double() * dout.double()).sum()
        size = (call(q).double() * dout.double()).abs().sum()
        want = (grads[n].double() * step.double()).sum()
        assert abs(up - want) <= 2 * 2.0 ** -8 * size + 2.0 ** -8 * (grads[n].double() * step.double()).abs().sum(), n


# ---------------------------------------------------------------------------------------
# on the GPU only
# ---------------------------------------------------------------------------------------
SHAPES = [dict(B=2, T=7, C=24, F=40), dict(B=2, T=700, C=384, F=1536), dict(B=3, T=331, C=77, F=130)]


@pytest.mark.gpu
@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("shape", SHAPES)
def test_same_bits_again_on_another_stream_and_in_threads(op, shape):
    dev = torch.device("cuda")
    plain = _grads(op, _inputs(op, dev, **shape))
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        for _ in range(3):
            _same(plain, _grads(op, _inputs(op, dev, **shape)))
    stream.synchronize()
    failed = []

    def work():
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    _same(plain, _grads(op, _inputs(op, dev, **shape)))
                torch.cuda.current_stream().synchronize()
        except BaseException as e:                            # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work) for _ in range(3)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not failed, failed


@pytest.mark.gpu
@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_in_a_captured_graph(op, shape):
    """Two graphs that share a pool, replayed in turn with new inputs and eager work in between."""
    dev = torch.device("cuda")
    t = _inputs(op, dev, grad=False, **shape)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.no_grad():
        _call(op, t)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for act in ("gelu_tanh", "silu"):
        graph = torch.cuda.CUDAGraph()
        with torch.no_grad(), torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            outs.append(_call(op, t, act))
        graphs.append(graph)
    for seed in (1, 2, 3):
        for n, v in _inputs(op, dev, grad=False, seed=seed, **shape).items():
            t[n].copy_(v)
        for i, act in ((0, "gelu_tanh"), (1, "silu")):
            with torch.no_grad():
                eager = _call(op, t, act)
            graphs[i].replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[i], eager)


@pytest.mark.gpu
@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("shape", SHAPES)
def test_training_step_in_a_captured_graph(op, shape):
    """Forward and backward captured once nothing of the warm-up lives, replayed with new inputs and eager work in between."""
    dev = torch.device("cuda")
    t = _inputs(op, dev, **shape)
    dout = torch.randn(_call(op, t).shape, generator=torch.Generator().manual_seed(77)).to(BF16).to(dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            _grads(op, t, dout=dout)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = _grads(op, t, dout=dout)
    for seed in (1, 2, 3):
        new = _inputs(op, dev, seed=seed, **shape)
        with torch.no_grad():
            for n, v in new.items():
                t[n].copy_(v)
        eager = _grads(op, new, dout=dout)
        graph.replay()
        torch.cuda.synchronize()
        _same(eager, captured)


@pytest.mark.gpu
@pytest.mark.parametrize("op", OPS)
def test_capture_with_gradients_alive_is_refused(op):
    """Leaves whose gradients belong to a graph that still lives: a captured forward that would record their backward is an error, and the same without
    gradients is none."""
    dev = torch.device("cuda")
    t = _inputs(op, dev)
    alive = _call(op, t)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="another graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            _call(op, t)
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        out = _call(op, t)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, alive)


@pytest.mark.gpu
def test_rows_beyond_32_bits():
    """Row numbers times their length beyond 2^31 elements, in every tensor of rows."""
    dev = torch.device("cuda")
    M, C, N = (1 << 21) + 37, 1032, 8
    x = torch.zeros(M, C, device=dev, dtype=BF16)
    at = torch.tensor([0, 1, M // 2, M - 70, M - 1], device=dev)
    g = torch.Generator().manual_seed(2)
    x[at] = torch.randn(len(at), C, generator=g).to(BF16).to(dev)
    w = (torch.randn(N, C, generator=g) * C ** -0.5).to(BF16).to(dev)
    assert x.numel() > 1 << 31
    few = x[at]
    assert torch.equal(llsa_amd.layer_norm(x)[at], llsa_amd.layer_norm(few))
    y = llsa_amd.linear(x.requires_grad_(), w.requires_grad_(), activation="silu")
    ref = few.double() @ w.detach().double().t()
    ref = ref * torch.sigmoid(ref)
    assert ((y.detach()[at].double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -12).all()      # half a step, and 1032 additions of order 1 in fp32
    dout = torch.zeros(M, N, device=dev, dtype=BF16)
    dout[at] = 1
    dx, dw = torch.autograd.grad(y, [x, w], dout)
    xs, ws = few.detach().clone().requires_grad_(), w.detach().clone().requires_grad_()
    sx, sw = torch.autograd.grad(llsa_amd.linear(xs, ws, activation="silu"), [xs, ws], torch.ones(len(at), N, device=dev, dtype=BF16))
    # the same products in another order of their sums: fp32, then one rounding each
    assert ((dx[at].double() - sx.double()).abs() <= 2 * 2.0 ** -8 * sx.abs() + 2.0 ** -10).all()
    assert ((dw.double() - sw.double()).abs() <= 2 * 2.0 ** -8 * sw.abs() + 2.0 ** -10).all()
    back = llsa_amd.linear(y.detach(), w.detach().t().contiguous())           # rows of 1032 out
    assert torch.equal(back[at], llsa_amd.linear(y.detach()[at.repeat(20)], w.detach().t().contiguous())[:len(at)])


def test_c_calls_check_distances():
    """Rows so far apart that a kernel's 32-bit offsets would not hold, and a gate for part of a sample."""
    import ctypes as C
    from llsa_amd._lib import LIB_PATH, Lib, LinearArgs
    lib = Lib(LIB_PATH)
    bad = lambda fn, a, text: (fn(C.byref(a), None) != 0 and text in lib.last_error_string())
    a = LinearArgs()
    a.M, a.N, a.K = 8, 8, 8
    a.x = a.w = a.out = a.dz = a.workspace = a.residual = 1 << 20
    a.ldx = a.ldw = a.ldo = a.lddz = a.ldr = 8
    for field in ("ldr", "ldo"):
        for value in ((1 << 23) + 8, -8):
            setattr(a, field, value)
            assert bad(lib.linear_fwd, a, b"apart"), field
        setattr(a, field, 8)
    a.gate = 1 << 20
    for per_sample in (3, 1 << 32):
        a.per_sample = per_sample
        assert bad(lib.linear_fwd, a, b"whole samples")
    a.gate, a.ldo = None, (1 << 23) + 8
    assert bad(lib.linear_dx, a, b"apart") and bad(lib.linear_dw, a, b"output")


def test_residual_of_distant_rows(dev):
    K, N, far = 16, 24, (1 << 23) + 8
    g = torch.Generator().manual_seed(5)
    draw = lambda *s: torch.randn(*s, generator=g).bfloat16().to(dev)
    x, w, res = draw(3, K), draw(N, K), draw(3, N)
    wide = torch.empty(2 * far + N, dtype=torch.bfloat16, device=dev).as_strided((3, N), (far, 1))
    wide.copy_(res)
    assert torch.equal(llsa_amd.linear(x, w, residual=wide), llsa_amd.linear(x, w, residual=res))
    w2, short = draw(N, N), dict(activation="silu")
    assert torch.equal(llsa_amd.feed_forward(x, w, None, w2, residual=wide, **short), llsa_amd.feed_forward(x, w, None, w2, residual=res, **short))


@pytest.mark.gpu
def test_norm_of_many_samples():
    """More samples than a grid has rows, each with a scale and shift of its own."""
    B, C = 70001, 24
    g = torch.Generator().manual_seed(6)
    x, scale, shift, dout = (torch.randn(*s, generator=g).cuda() for s in ((B, 1, C), (B, C), (B, C), (B, 1, C)))
    w = torch.randn(C, generator=g).cuda()
    leaves = [t.requires_grad_() for t in (x, w, scale, shift)]
    got = torch.autograd.grad(llsa_amd.layer_norm(x, w, scale=scale, shift=shift), leaves, dout)
    l64 = [t.detach().double().requires_grad_() for t in leaves]
    d = l64[0] - l64[0].mean(-1, keepdim=True)
    h = d * (d.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    ref = torch.autograd.grad(h * l64[1] * (1 + l64[2][:, None]) + l64[3][:, None], l64, dout.double())
    # in fp32: a few roundings an element; the weight's gradient adds up 70001 rows one after another, 70001 * 2^-24 of the sum of magnitudes
    for a, b, bound in zip(got, ref, (2e-5, None, 2e-5, 1e-6)):
        if bound is None:
            sums = (dout.double() * (h * (1 + l64[2][:, None])).detach()).abs().sum((0, 1))
            assert ((a - b).abs() <= (B + 64) * 2.0 ** -24 * sums).all()
        else:
            assert (a - b).norm() <= bound * b.norm()
