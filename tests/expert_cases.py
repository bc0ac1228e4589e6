"""route_tokens, grouped_linear and expert_feed_forward against their formulas in 64 bits, with bounds on every element that follow from the roundings
(the notation of block_cases: u = half a step of the 16-bit type for each value written in it, n * 2^-24 of the sum of magnitudes for n additions in fp32)."""
import torch

import llsa_amd
from block_cases import CURVE, E, FAST, SLOPE, act64, half_step, least, within


def more(n):
    return (n + 32) * E


KEPT = 2.0 ** -15                                             # half a step of a kept act'(z)


def slope64(act, z):
    return torch.autograd.functional.jvp(lambda t: act64(act, t), z, torch.ones_like(z))[1] if act else torch.ones_like(z)


# ---------------------------------------------------------------------------------------
# the router
# ---------------------------------------------------------------------------------------
def chosen64(logits, k):
    """experts (M, k), -1 where there is none: the largest first, of equal ones the lowest index; a NaN above every number, -inf never"""
    out = torch.full((logits.shape[0], k), -1, dtype=torch.int32)
    for m, row in enumerate(logits.double().tolist()):
        key = [(float("inf"), 1) if v != v else (v, 0) for v in row]
        order = sorted((i for i in range(len(row)) if row[i] != float("-inf")), key=lambda i: (-key[i][0], -key[i][1], i))
        for j, e in enumerate(order[:k]):
            out[m, j] = e
    return out


def plan64(experts, n):
    flat = experts.reshape(-1).tolist()
    runs = [[s for s, e in enumerate(flat) if e == x] for x in range(n)]
    order = [s for r in runs for s in r]
    places = [-1] * len(flat)
    for p, s in enumerate(order):
        places[s] = p
    offsets = [0]
    for r in runs:
        offsets.append(offsets[-1] + len(r))
    t = lambda v: torch.tensor(v, dtype=torch.int32)
    return t(order + [-1] * (len(flat) - len(order))), t(offsets), t(places).reshape(experts.shape)


def check_plan(r, logits, k):
    """The whole numbers of a routing."""
    n = logits.shape[-1]
    flat = logits.detach().cpu().reshape(-1, n)
    experts = chosen64(flat, k)
    order, offsets, places = plan64(experts, n)
    for name, got, want in (("experts", r.experts.reshape(-1, k), experts), ("order", r.order, order), ("offsets", r.offsets, offsets), ("places", r.places.reshape(-1, k), places)):
        assert got.dtype == torch.int32 and torch.equal(got.cpu(), want), name
    assert r.weights.shape == r.experts.shape == r.places.shape == (*logits.shape[:-1], k)
    return experts


def check_route(logits, k, normalize, dweights=None):
    n = logits.shape[-1]
    r = llsa_amd.route_tokens(logits, k, normalize=normalize)
    experts = check_plan(r, logits, k)
    l = logits.detach().double().cpu().reshape(-1, n).requires_grad_()
    taken = torch.zeros(l.shape, dtype=torch.bool)
    for j in range(k):
        has = experts[:, j] >= 0
        taken[has, experts[has, j].long()] = True
    over = taken if normalize else l > -float("inf")
    top = torch.where(over, l, -1e300).amax(-1, keepdim=True).detach()
    e = torch.where(over, torch.exp(torch.where(over, l - top, 0.0)), 0.0)
    total = e.sum(-1, keepdim=True)
    p = torch.where(over, e / torch.where(total > 0, total, 1.0), 0.0)
    w = torch.where(experts >= 0, torch.where(taken, p, 0.0).gather(1, experts.clamp(min=0).long()), 0.0)
    # exp2 of a product that is rounded, once for each logit, and expf itself; a sum of up to n; a division
    far = torch.where(over, (l.detach() - top).abs(), 0.0).clamp(max=110).amax(-1, keepdim=True)
    rel = E * (4 * far + 16 + 2 * n)
    within(r.weights.detach().cpu().reshape(-1, k), w.detach(), rel * w.detach() + 2.0 ** -126, "weights")
    if dweights is None:
        return r
    d, = torch.autograd.grad(r.weights, logits, dweights)
    ref, = torch.autograd.grad(w, l, dweights.double().cpu().reshape(-1, k))
    g = torch.zeros(l.shape, dtype=torch.float64)
    for j in range(k):
        has = experts[:, j] >= 0
        g[has, experts[has, j].long()] = dweights.double().cpu().reshape(-1, k)[has, j]
    pd = torch.where(taken | (torch.tensor(not normalize) & over), p.detach(), 0.0)
    size = pd * (g.abs() + (g.abs() * torch.where(taken, p.detach(), 0.0)).sum(-1, keepdim=True))
    within(d.cpu().reshape(-1, n), ref, (2.5 * rel + 8 * E + k * E) * size + half_step(logits.dtype) * ref.abs() + least(logits.dtype), "dlogits")
    return r


# ---------------------------------------------------------------------------------------
# products by expert
# ---------------------------------------------------------------------------------------
def runs_of(offsets, rows):
    """begin and end of every expert's rows: held to 0 .. rows, not falling"""
    at, out = 0, []
    o = offsets.cpu().tolist()
    for a, b in zip(o, o[1:]):
        at = max(at, min(max(a, 0), rows))
        end = max(at, min(max(b, 0), rows))
        out.append((at, end))
        at = end
    return out


def check_grouped(x, weight, offsets, bias, act, dout):
    """All of them leaves (offsets aside) on the device; forward and every gradient."""
    named = [(n, t) for n, t in (("x", x), ("weight", weight), ("bias", bias)) if t is not None]
    out = llsa_amd.grouped_linear(x, weight, offsets, bias, activation=act)
    got = dict(zip([n for n, _ in named], torch.autograd.grad(out, [t for _, t in named], dout)))
    where = x.device if x.numel() * weight.shape[1] > 1 << 26 else torch.device("cpu")
    c = lambda t: t.detach().double().to(where)
    u, lo, (rows, K), N = half_step(x.dtype), least(x.dtype), x.shape, weight.shape[1]
    held = torch.zeros(rows, dtype=torch.bool)
    for e, (a, b) in enumerate(runs_of(offsets, rows)):
        held[a:b] = True
        xe, we, d = c(x[a:b]), c(weight[e]), c(dout[a:b])
        be = c(bias[e]) if bias is not None else torch.zeros(N, dtype=torch.float64, device=where)
        z = xe @ we.t() + be
        dz = (K + 4) * E * (xe.abs() @ we.abs().t() + be.abs())
        v = act64(act, z)
        dv = SLOPE * dz + (FAST * (v.abs() + z.abs()) if act else 0)
        within(out[a:b].detach().to(where), v, dv + u * (v.abs() + dv) + lo, f"out, expert {e}")
        g, dg = d * slope64(act, z), 0 * d
        if act:
            dg = d.abs() * (CURVE * dz + FAST + KEPT)
            dg = dg + E * g.abs() + u * (g.abs() + dg) + lo
        n = b - a
        r = g.t() @ xe
        within(got["weight"][e].to(where), r, (dg.t() @ xe.abs() + more(n) * (g.abs().t() @ xe.abs())) * (1 + u) + u * r.abs() + lo, f"dweight, expert {e}")
        if bias is not None:
            r = g.sum(0)
            within(got["bias"][e].to(where), r, (dg.sum(0) + more(n) * g.abs().sum(0)) * (1 + u) + u * r.abs() + lo, f"dbias, expert {e}")
        r = g @ we
        within(got["x"][a:b].to(where), r, (dg @ we.abs() + more(N) * (g.abs() @ we.abs())) * (1 + u) + u * r.abs() + lo, f"dx, expert {e}")
    assert not out[~held.to(out.device)].any() and not got["x"][~held.to(out.device)].any()
    return out, got


def check_experts(x, routing, w_in, b_in, w_out, b_out, act, gate, residual, dout):
    """All leaves (routing.weights among them) on the device; forward and every gradient."""
    weights = routing.weights
    named = [(n, t) for n, t in (("x", x), ("weights", weights), ("w_in", w_in), ("b_in", b_in), ("w_out", w_out), ("b_out", b_out), ("gate", gate), ("residual", residual)) if t is not None]
    out = llsa_amd.expert_feed_forward(x, routing, w_in, b_in, w_out, b_out, activation=act, gate=gate, residual=residual)
    got = dict(zip([n for n, _ in named], torch.autograd.grad(out, [t for _, t in named], dout)))
    where = x.device if x.numel() * w_in.shape[1] > 1 << 25 else torch.device("cpu")
    c = lambda t: t.detach().double().to(where)
    u, lo = half_step(x.dtype), least(x.dtype)
    n_experts, F, C = w_in.shape
    N, k = w_out.shape[1], weights.shape[-1]
    xs, ws, ids = c(x).reshape(-1, C), c(weights).reshape(-1, k), routing.experts.detach().to(where).reshape(-1, k)
    M = xs.shape[0]
    zero = lambda *s: torch.zeros(*s, dtype=torch.float64, device=where)
    per_row = lambda t: t.repeat_interleave(M // x.shape[0], 0)
    gt = per_row(c(gate)) if gate is not None else torch.ones(1, 1, dtype=torch.float64, device=where)
    d = c(dout).reshape(M, N)
    G = d * gt
    s, ds, size = zero(M, N), zero(M, N), zero(M, N)
    dx, ddx, dp, ddp = zero(M, C), zero(M, C), zero(M, k), zero(M, k)
    for e in range(n_experts):
        tok, j = torch.nonzero(ids == e, as_tuple=True)
        n = tok.numel()
        xe, w, w1, w2 = xs[tok], ws[tok, j][:, None], c(w_in[e]), c(w_out[e])
        b1 = c(b_in[e]) if b_in is not None else zero(F)
        b2 = c(b_out[e]) if b_out is not None else zero(N)
        z = xe @ w1.t() + b1
        dz = (C + 4) * E * (xe.abs() @ w1.abs().t() + b1.abs())
        a = act64(act, z)
        da = SLOPE * dz + FAST * (a.abs() + z.abs())
        h, dh = a, da + u * (a.abs() + da) + lo               # (the hidden rows are rounded)
        y = h @ w2.t() + b2
        dy = dh @ w2.abs().t() + (F + 4) * E * (h.abs() @ w2.abs().t() + b2.abs())
        s.index_add_(0, tok, w * y)
        ds.index_add_(0, tok, w * dy)
        size.index_add_(0, tok, (w * y).abs())
        # backward
        dp[tok, j] = (G[tok] * y).sum(1)
        ddp[tok, j] = (G[tok].abs() * dy).sum(1) + more(N) * (G[tok] * y).abs().sum(1)
        ge = w * G[tok]
        dge = (2 * E + u) * ge.abs() + lo                     # (dout with weight and gate is rounded)
        t = ge @ w2
        dt = dge @ w2.abs() + more(N) * (ge.abs() @ w2.abs())
        g = t * slope64(act, z)
        dg = dt * SLOPE + t.abs() * (CURVE * dz + FAST + KEPT) + 2 * E * g.abs()
        dg = dg + u * (g.abs() + dg) + lo
        r = ge.t() @ h
        within(got["w_out"][e].to(where), r, (dge.t() @ (h.abs() + dh) + ge.abs().t() @ dh + more(n) * (ge.abs().t() @ h.abs())) * (1 + u) + u * r.abs() + lo, f"dw_out, expert {e}")
        if b_out is not None:
            r = ge.sum(0)
            within(got["b_out"][e].to(where), r, (dge.sum(0) + more(n) * ge.abs().sum(0)) * (1 + u) + u * r.abs() + lo, f"db_out, expert {e}")
        r = g.t() @ xe
        within(got["w_in"][e].to(where), r, (dg.t() @ xe.abs() + more(n) * (g.abs().t() @ xe.abs())) * (1 + u) + u * r.abs() + lo, f"dw_in, expert {e}")
        if b_in is not None:
            r = g.sum(0)
            within(got["b_in"][e].to(where), r, (dg.sum(0) + more(n) * g.abs().sum(0)) * (1 + u) + u * r.abs() + lo, f"db_in, expert {e}")
        r = g @ w1
        b = dg @ w1.abs() + more(F) * (g.abs() @ w1.abs())
        dx.index_add_(0, tok, r)
        ddx.index_add_(0, tok, b + k * E * (r.abs() + b))
    ds = ds + k * E * size
    res = c(residual).reshape(M, N) if residual is not None else zero(1, 1)
    ref = res + gt * s
    within(out.detach().to(where).reshape(M, N), ref, gt.abs() * ds + 3 * E * (res.abs() + (gt * s).abs()) + u * (ref.abs() + gt.abs() * ds) + lo, "out")
    within(got["x"].to(where).reshape(M, C), dx, ddx * (1 + u) + u * dx.abs() + lo, "dx")
    within(got["weights"].to(where).reshape(M, k), dp, ddp + E * dp.abs(), "dweights")
    if gate is not None:
        T = M // x.shape[0]
        each = lambda t: t.reshape(x.shape[0], -1, N).sum(1)
        r = each(d * s)
        b = each(d.abs() * ds + (T + 32) * E * d.abs() * size)
        within(got["gate"].to(where), r, b * (1 + u) + u * r.abs() + lo, "dgate")
    if residual is not None:
        assert torch.equal(got["residual"], dout)
    return out, got
