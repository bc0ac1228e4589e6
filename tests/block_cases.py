"""The operators around the attention (layer_norm, linear, feed_forward) against their formulas in 64 bits, with bounds on every element that
follow from the roundings: u = finfo(dtype).eps / 2 for each value written in 16 bits, and n * 2^-24 times the sum of magnitudes for n additions in fp32.
Below the smallest normal number a step does not shrink any more: a rounding there is off by up to `least` = finfo(dtype).tiny * u (fp16: 2^-14 * 2^-11 = 2^-25)."""
import torch

import llsa_amd

E = 2.0 ** -24                                                # half a step of fp32
FAST = 2.0 ** -20                                             # activations: exp2 and reciprocal of the hardware (1 ulp each) and a handful of fp32 operations
SLOPE, CURVE = 1.2, 1.0                                       # |act'| <= 1.13, |act''| <= 0.8 of all three activations


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):
    return torch.finfo(dtype).tiny * half_step(dtype)


def act64(name, z):
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return z * 0.5 * torch.erfc(-z / 2 ** 0.5)
    if name == "gelu_tanh":
        return z * torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (z + 0.044715 * z ** 3))
    return z


def per_sample(t, x):
    """(B, C) against (B, ..., C)"""
    return t.reshape(t.shape[0], *([1] * (x.dim() - 2)), t.shape[1])


def within(got, ref, bound, what):
    got = got.double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    off = (got - ref).abs() - bound
    assert torch.isfinite(got).all(), f"{what}: not finite"
    if off.numel():
        worst = off.argmax()
        assert off.max() <= 0, f"{what}: {got.flatten()[worst].item()} instead of {ref.flatten()[worst].item()}, bound {bound.expand_as(ref).flatten()[worst].item():.3g}"


def norm64(x, weight, bias, scale, shift, eps):
    d = x - x.mean(-1, keepdim=True)
    h = d * (d.square().mean(-1, keepdim=True) + eps).rsqrt()
    n = h if weight is None else h * weight
    n = n if bias is None else n + bias
    y = n if scale is None else n * (1 + per_sample(scale, x))
    return h, n, y if shift is None else y + per_sample(shift, x)


def check_norm(x, weight, bias, scale, shift, dout, eps=1e-5):
    """All inputs leaves (or None) on the device; forward, then the gradients of all of them."""
    named = [(n, t) for n, t in (("x", x), ("weight", weight), ("bias", bias), ("scale", scale), ("shift", shift)) if t is not None]
    y = llsa_amd.layer_norm(x, weight, bias, scale=scale, shift=shift, eps=eps)
    assert y.dtype == x.dtype and y.shape == x.shape
    got = dict(zip([n for n, _ in named], torch.autograd.grad(y, [t for _, t in named], dout)))
    leaf = {n: t.detach().double().cpu().requires_grad_() for n, t in named}
    v = lambda n: leaf.get(n)
    x64, C, u, lo = leaf["x"], x.shape[-1], half_step(x.dtype), least(x.dtype)
    h, n, ref = norm64(x64, v("weight"), v("bias"), v("scale"), v("shift"), eps)
    d64 = dout.double().cpu()
    grads = dict(zip(leaf, torch.autograd.grad(ref, list(leaf.values()), d64)))
    with torch.no_grad():
        h, n, ref = h.detach(), n.detach(), ref.detach()
        c = 48 * E                                            # a lane adds up to 32 values, then up to 10 halvings
        one = torch.ones((), dtype=torch.float64)
        rstd = (x64.var(-1, unbiased=False, keepdim=True) + eps).rsqrt()
        dh = rstd * (c * x64.abs().mean(-1, keepdim=True) + 2 * E * x64.abs()) + 3 * c * h.abs()
        up = (v("weight").abs() if "weight" in leaf else one) * (1 + per_sample(v("scale").abs(), x64) if "scale" in leaf else one)
        add = (v("bias").abs() if "bias" in leaf else 0 * one) * (1 + per_sample(v("scale").abs(), x64) if "scale" in leaf else one)
        within(y.detach().cpu(), ref, up * dh + 6 * E * (up * h.abs() + add + ref.abs()) + u * ref.abs() + lo, "y")
        g, gh = d64.abs() * up, (d64 * h).abs() * up
        dgh = g * dh
        bound = rstd * (6 * E * g + c * g.mean(-1, keepdim=True) + h.abs() * (c * gh.mean(-1, keepdim=True) + dgh.mean(-1, keepdim=True)) + dh * gh.mean(-1, keepdim=True))
        within(got["x"].cpu(), grads["x"], bound + (4 * c + u) * grads["x"].abs() + 4 * E * rstd * (g + gh.mean(-1, keepdim=True) * h.abs()) + lo, "dx")
        rows = x64.numel() // C
        flat = lambda t: t.reshape(-1, C)
        S1, S2, dS2 = d64.abs(), (d64 * h).abs(), d64.abs() * dh
        many = (rows + 16) * E
        scale_up = (1 + per_sample(v("scale").abs(), x64)) if "scale" in leaf else one
        if "weight" in leaf:
            uw = half_step(weight.dtype)
            within(got["weight"].cpu(), grads["weight"], flat(scale_up * (dS2 + many * S2)).sum(0) + uw * grads["weight"].abs() + least(weight.dtype), "dweight")
        if "bias" in leaf:
            within(got["bias"].cpu(), grads["bias"], flat(scale_up * many * S1).sum(0) + half_step(bias.dtype) * grads["bias"].abs() + least(bias.dtype), "dbias")
        each = lambda t: t.reshape(t.shape[0], -1, C).sum(1)
        if "scale" in leaf:
            w, b = (v("weight").abs() if "weight" in leaf else one), (v("bias").abs() if "bias" in leaf else 0 * one)
            within(got["scale"].cpu(), grads["scale"], each(w * (dS2 + many * S2) + b * many * S1) + half_step(scale.dtype) * grads["scale"].abs() + least(scale.dtype), "dscale")
        if "shift" in leaf:
            within(got["shift"].cpu(), grads["shift"], each(many * S1) + half_step(shift.dtype) * grads["shift"].abs() + least(shift.dtype), "dshift")
    return y, got


def _layer_bounds(x, w, b, act, dh):
    """z of a layer and its bound, from inputs h (fp64) with bound dh: (z, dz, a, da), a before its rounding."""
    K = w.shape[1]
    mag = x.abs() @ w.abs().t() + (b.abs() if b is not None else 0)
    z = x @ w.t() + (b if b is not None else 0)
    dz = dh @ w.abs().t() + (K + 4) * E * mag
    a = act64(act, z)
    return z, dz, a, SLOPE * dz + (FAST * (a.abs() + z.abs()) if act else 0)


def check_layers(x, layers, gate, residual, dout, call):
    """layers: [(weight, bias or None, activation or None)] one after another; call() runs the operator.  All leaves on the device."""
    named = [("x", x)] + [(f"{n}{i}", t) for i, (w, b, _) in enumerate(layers) for n, t in (("weight", w), ("bias", b)) if t is not None]
    named += [(n, t) for n, t in (("gate", gate), ("residual", residual)) if t is not None]
    named = [(n, t) for n, t in named if t.requires_grad]
    out = call()
    u, lo = half_step(x.dtype), least(x.dtype)
    got = dict(zip([n for n, _ in named], torch.autograd.grad(out, [t for _, t in named], dout)))
    where = x.device if x.numel() * layers[0][0].shape[0] > 1 << 26 else torch.device("cpu")
    c = lambda t: None if t is None else t.detach().double().to(where)
    # forward
    h, steps = c(x).reshape(-1, x.shape[-1]), []
    dh = torch.zeros_like(h)
    for i, (w, b, act) in enumerate(layers):
        z, dz, a, da = _layer_bounds(h, c(w), c(b), act, dh)
        steps.append((h, dh, z, dz, a, da))
        last = i == len(layers) - 1
        h, dh = a, da if last else da + u * (a.abs() + da)    # (the hidden rows are rounded, the output is not yet)
    N = layers[-1][0].shape[0]
    T = h.shape[0] // x.shape[0] if gate is not None else 1
    rep = c(gate).repeat_interleave(T, 0) if gate is not None else torch.ones(1, dtype=torch.float64, device=where)
    res = c(residual).reshape(-1, N) if residual is not None else torch.zeros(1, dtype=torch.float64, device=where)
    ref = res + rep * h
    within(out.detach().to(where).reshape(-1, N), ref, rep.abs() * dh + 4 * E * (res.abs() + (rep * h).abs()) + u * (ref.abs() + rep.abs() * dh) + lo, "out")
    # backward
    d = c(dout).reshape(-1, N)
    if residual is not None and residual.requires_grad:
        assert torch.equal(got["residual"], dout)
    M = d.shape[0]
    if gate is not None and gate.requires_grad:
        y, dy = h, dh
        zs = steps[-1]
        # (act(z) is taken of the z that was kept in 16 bits)
        dy = dy + SLOPE * (u * (zs[2].abs() + zs[3]) + lo) + FAST * zs[2].abs()
        each = lambda t: t.reshape(x.shape[0], -1, N).sum(1)
        r = each(d * y)
        within(got["gate"].to(where), r, each(d.abs() * dy + (T + 32) * E * (d * y).abs()) * (1 + u) + u * r.abs() + lo, "dgate")
    g, dg = d * rep, E * (d * rep).abs()
    rounded = gate is not None
    for i in range(len(layers) - 1, -1, -1):
        w, b, act = layers[i]
        hh, dhh, z, dz, a, da = steps[i]
        if act:
            slope_ref = torch.autograd.functional.jvp(lambda t: act64(act, t), z, torch.ones_like(z))[1]
            off = CURVE * (dz + u * (z.abs() + dz) + lo) + FAST
            dg = dg * SLOPE + g.abs() * off
            g = g * slope_ref
            rounded = True
        if rounded:
            dg = dg + u * (g.abs() + dg) + lo
        more = lambda n: (n + 32) * E
        if f"weight{i}" in got:
            r = g.t() @ hh
            bound = dg.t() @ (hh.abs() + dhh) + g.abs().t() @ dhh + more(M) * (g.abs().t() @ hh.abs())
            within(got[f"weight{i}"].to(where), r, bound * (1 + u) + u * r.abs() + lo, f"dweight{i}")
        if f"bias{i}" in got:
            r = g.sum(0)
            within(got[f"bias{i}"].to(where), r, (dg.sum(0) + more(M) * g.abs().sum(0)) * (1 + u) + u * r.abs() + lo, f"dbias{i}")
        wc = c(w)
        # (a gate in the weights is rounded there: gate * w instead of dout * gate, u of each product either way, but at least `lo` for each weight)
        small = lo * (d.abs() if gate is not None and i == len(layers) - 1 else g.abs()).sum(1, keepdim=True)
        dg, g = dg @ wc.abs() + more(wc.shape[0]) * (g.abs() @ wc.abs()) + small, g @ wc
        rounded = False
    if "x" in got:
        within(got["x"].to(where).reshape(g.shape), g, dg * (1 + u) + u * g.abs() + lo, "dx")
    return out, got
