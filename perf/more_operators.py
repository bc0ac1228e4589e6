"""Further forms of the linear layer and the feed-forward block, as plain cases: rows that choose their weights (a router, products
with an expert's weights for each run of rows, the feed-forward block made of both; sampling and training), and the linear layer in
8-bit integers (sampling).

A case: {"op": "route" | "grouped" | "experts" | "int8", "mode": "infer" | "train", "dtype": "bf16" | "fp16" | "fp32" (route only), ...} and for

  route    "M" tokens, "E" experts, "k" of them for each token, "normalize": the chosen ones' weights add up to one, "masked": some
           tokens are padding (no expert at all), and some have few experts to choose from
  grouped  "R" rows in runs of "E" experts, "tail": rows behind the last run, "K" channels in, "N" out, "act", "bias"
  experts  "B" samples of "T" tokens, "E", "k", "C" channels, "F" hidden ones, "act", "gate": a factor for each sample and channel, "residual"
  int8     "B", "T", "K", "N", "act", "bias", "gate", "residual"; weights in 8 bits with a scale for each channel, the rows are
           brought to 8 bits, with a scale each, on the way

Formulas, for a row l of logits, a row x of a sample b:

  route    the k largest l_i (equal ones: lowest index first; -inf is never chosen, and leaves -1 in its place);
           w_i = exp(l_i - max l) / sum, the sum over the chosen ones (normalize) or over all; 0 where there is none
           order: the numbers token * k + j of what was chosen, by expert and then by number, -1 behind the last; offsets (E + 1): where each
           expert's begin in it; places (token, j): where that number stands in it, or -1
  grouped  y = act(W_e x + bias_e) for rows offsets[e] .. offsets[e + 1] - 1, 0 for rows that no expert has
  experts  y = residual + gate_b * sum over the chosen e of w_e (W_out,e act(W_in,e x + b_in,e) + b_out,e)
  int8     s = max |x| / 127, q = x / s rounded to the nearest whole number (halves to even),  y = residual + gate_b * act(s s_n sum q q_n + bias)
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _route(name, mode, dtype, M, E, k, normalize=True, masked=False):
    return {"name": name, "op": "route", "mode": mode, "dtype": dtype, "M": M, "E": E, "k": k, "normalize": normalize, "masked": masked}


def _grouped(name, mode, dtype, R, E, K, N, act="", bias=True, tail=0):
    return {"name": name, "op": "grouped", "mode": mode, "dtype": dtype, "R": R, "E": E, "K": K, "N": N, "act": act, "bias": bias, "tail": tail}


def _experts(name, mode, dtype, B, T, E, k, C, F, act="gelu_tanh", gate=False, residual=False):
    return {"name": name, "op": "experts", "mode": mode, "dtype": dtype, "B": B, "T": T, "E": E, "k": k, "C": C, "F": F, "act": act, "gate": gate,
            "residual": residual}


def _int8(name, dtype, B, T, K, N, act="", bias=True, gate=False, residual=False):
    return {"name": name, "op": "int8", "mode": "infer", "dtype": dtype, "B": B, "T": T, "K": K, "N": N, "act": act, "bias": bias, "gate": gate,
            "residual": residual}


def listed():
    return [
        # the router of one block while one image of 32 x 32 pixels is sampled: two of eight experts for each token
        _route("route_infer_1k", "infer", "bf16", 1024, 8, 2),
        # many small experts in the training step of batch 8 of 128 x 128 pixels, logits in 32 bits, padded images among the batch
        _route("route_train_many", "train", "fp32", 131072, 64, 8, normalize=False, masked=True),
        # one vector for each of 8 images, two experts each: the weights of the experts that are hit, and hardly any rows
        _grouped("grouped_infer_rows", "infer", "bf16", 16, 8, 384, 1536, act="silu"),
        # odd sizes all round, rows behind the last run (a buffer that is not full)
        _grouped("grouped_train_odd", "train", "fp16", 4593, 7, 777, 333, act="gelu", tail=61),
        # generic square products, bound by the matrix units
        _grouped("grouped_train_wide", "train", "bf16", 16384, 8, 2048, 2048, bias=False),
        # the routed feed-forward block while one small image is sampled
        _experts("experts_infer_1k", "infer", "bf16", 1, 1024, 8, 2, 384, 1536, gate=True, residual=True),
        # the routed feed-forward block in the DiT-S training step: batch 8 of 128 x 128 pixels
        _experts("experts_train_layer", "train", "bf16", 8, 16384, 8, 2, 384, 1536, gate=True, residual=True),
        # odd token, channel and expert counts, another activation
        _experts("experts_train_odd", "train", "fp16", 3, 1531, 5, 3, 333, 1001, act="silu", residual=True),
        # the layer that makes the six modulation vectors of a block while 8 images are sampled: all weights, eight rows
        _int8("int8_infer_rows", "bf16", 8, 1, 384, 2304),
        # odd sizes all round
        _int8("int8_infer_odd", "fp16", 3, 1531, 777, 333, act="gelu", residual=True),
        # the second layer of the feed-forward block while 8 images of 128 x 128 pixels are sampled: gated, onto the residual stream
        _int8("int8_infer_layer", "bf16", 8, 16384, 1536, 384, gate=True, residual=True),
        # a generic square projection, bound by the matrix units
        _int8("int8_infer_wide", "bf16", 1, 8192, 4096, 4096),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def _channels(rng, hi):
    """Multiples of 64, of 8, and any count at all."""
    step = rng.choice([64, 64, 8, 1])
    return step * _log_int(rng, max(1, 16 // step), hi // step)


def draw(rng):
    op = rng.choice(["route", "grouped", "grouped", "experts", "experts", "int8", "int8"])
    mode = rng.choice(["infer", "train", "train"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16"])
    act = rng.choice(["", "silu", "gelu", "gelu_tanh"])
    E = rng.choice([8, 16, 64, rng.randint(2, 64)])
    k = rng.randint(2, min(E, 8))                             # (one alone has a weight of one, whatever its logit is)
    if op == "route":
        c = _route("", mode, rng.choice([dtype, "fp32"]), _log_int(rng, 1, 131072), E, k, rng.random() < 0.6, rng.random() < 0.4)
        rows, most = "M", {"bytes": 0.2e9, "flops": 1e15}
    elif op == "grouped":
        c = _grouped("", mode, dtype, _log_int(rng, 1, 65536), E, _channels(rng, 2048), _channels(rng, 2048), act, rng.random() < 0.8)
        c["tail"] = rng.choice([0, 0, rng.randint(0, c["R"] // 4)])
        rows, most = "R", {"bytes": 0.9e9, "flops": 0.41e12}
    elif op == "experts":
        C = _channels(rng, 1024)
        c = _experts("", mode, dtype, rng.randint(1, 8), _log_int(rng, 1, 16384), E, min(k, 4), C, rng.choice([4 * C, 2 * C, _channels(rng, 2048)]),
                     act or "gelu_tanh", rng.random() < 0.6, rng.random() < 0.8)
        rows, most = "T", {"bytes": 0.8e9, "flops": 1.8e12}
    else:
        c = _int8("", dtype, rng.randint(1, 8), _log_int(rng, 1, 16384), _channels(rng, 4096), _channels(rng, 4096), act, rng.random() < 0.8, rng.random() < 0.3,
                  rng.random() < 0.4)
        rows, most = "T", {"bytes": 0.7e9, "flops": 0.27e12}
    del c["name"]
    while any(work(c)[n] > most[n] for n in most):
        if c.get("B", 1) > 1:
            c["B"] -= 1
        elif c[rows] > 1:
            c[rows] = c[rows] * 2 // 3
        elif c["E"] > 2:                                      # (the weights alone are too much)
            c["E"] = c["E"] * 2 // 3
            c["k"] = min(c["k"], c["E"]) if "k" in c else 0
        else:
            break
    if "tail" in c:
        c["tail"] = min(c["tail"], c["R"])
        c.pop("k", None)
    return c


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------
def _small_integers(w):
    """A weight (N, K) as it is kept for sampling: whole numbers from -127 to 127, and a scale for each channel out."""
    scale = w.float().abs().amax(-1) / 127
    return torch.round(w.double() / scale.double()[:, None]).to(torch.int8), scale


def prepare(case, seed):
    dev, dtype = torch.device("cuda"), DTYPES[case["dtype"]]
    gen = torch.Generator(device=dev).manual_seed(seed)
    train = case["mode"] == "train"

    def normal(*shape, std=1.0, mean=0.0):
        return (torch.randn(*shape, device=dev, generator=gen) * std + mean).to(dtype).requires_grad_(train)

    def weight(*shape):                                       # as a linear layer starts: uniform, 1 / sqrt(fan in)
        return ((torch.rand(*shape, device=dev, generator=gen) * 2 - 1) / math.sqrt(shape[-1])).to(dtype).requires_grad_(train)

    s = {"case": case}
    if case["op"] == "route":
        M, E = case["M"], case["E"]
        logits = torch.randn(M, E, device=dev, generator=gen) + torch.randn(E, device=dev, generator=gen) * 0.5      # some experts are liked better
        if case["masked"]:
            logits[torch.rand(M, device=dev, generator=gen) < 0.1] = -math.inf
            few = torch.rand(M, device=dev, generator=gen) < 0.1
            logits = torch.where(few[:, None] & (torch.rand(M, E, device=dev, generator=gen) < 0.8), -math.inf, logits)
        s["logits"] = logits.to(dtype).requires_grad_(train)
        if train:
            s["dweights"] = torch.randn(M, case["k"], device=dev, generator=gen)
        return s
    if case["op"] == "grouped":
        R, E, K, N = case["R"], case["E"], case["K"], case["N"]
        liked = torch.softmax(torch.randn(E, device=dev, generator=gen) * 0.5, 0)
        chosen = torch.multinomial(liked, max(1, R - case["tail"]), replacement=True, generator=gen)[:R - case["tail"]]
        counts = (chosen[:, None] == torch.arange(E, device=dev)).sum(0)
        s["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
        s["x"], s["weight"] = normal(R, K), weight(E, N, K)
        if case["bias"]:
            s["bias"] = normal(E, N, std=0.1)
        if train:
            s["dout"] = torch.randn(R, N, device=dev, generator=gen).to(dtype)
        return s
    B, T = case["B"], case["T"]
    if case["op"] == "experts":
        E, out, F = case["E"], case["C"], case["F"]
        s["x"] = normal(B, T, out)
        liked = torch.randn(E, device=dev, generator=gen) * 0.5
        s["logits"] = (torch.randn(B, T, E, device=dev, generator=gen) + liked).to(dtype).requires_grad_(train)
        s["w_in"], s["b_in"], s["w_out"], s["b_out"] = weight(E, F, out), normal(E, F, std=0.1), weight(E, out, F), normal(E, out, std=0.1)
    else:
        K, out = case["K"], case["N"]
        s["x"] = normal(B, T, K) * (torch.rand(B, T, 1, device=dev, generator=gen) * 3 + 0.1).to(dtype)       # rows of different sizes
        s["weight"], s["scale"] = _small_integers(weight(out, K))
        if case["bias"]:
            s["bias"] = normal(out, std=0.1)
    if case["gate"]:
        s["gate"] = normal(B, out, std=0.3, mean=0.5)
    if case["residual"]:
        s["residual"] = normal(B, T, out)
    if train:
        s["dout"] = torch.randn(B, T, out, device=dev, generator=gen).to(dtype)
    return s


def _leaves(s):
    """What a training step wants the gradients of, by name."""
    names = ["logits", "x", "weight", "bias", "w_in", "b_in", "w_out", "b_out", "gate", "residual"]
    return [(n, s[n]) for n in names if n in s]


# ---------------------------------------------------------------------------------------
# plain forms: elementary operations in 32 bits (64 where a whole number hangs on them)
# ---------------------------------------------------------------------------------------
def _act(name, z):
    """act(z) and act'(z)."""
    if name == "silu":
        g = 1 / (1 + torch.exp(-z))
        return z * g, g * (1 + z * (1 - g))
    if name == "gelu":
        p = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * p, p + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    return z, torch.ones_like(z)


def _choose(logits, k, normalize):
    """Of fp32 logits (M, E): the experts (M, k) or -1, their weights, and all probabilities."""
    values, index = torch.sort(logits, dim=-1, descending=True, stable=True)
    there = values[:, :k] > -math.inf
    top = torch.where(values[:, :1] > -math.inf, values[:, :1], torch.zeros_like(values[:, :1]))
    e, all_e = torch.exp(values[:, :k] - top), torch.exp(logits - top)
    total = (e if normalize else all_e).sum(-1, keepdim=True)
    total = torch.where(total > 0, total, torch.ones_like(total))
    return torch.where(there, index[:, :k], torch.full_like(index[:, :k], -1)), e / total, all_e / total


def _plan(experts, E):
    """order, offsets and places of the chosen experts (M, k)."""
    flat = experts.reshape(-1)
    by = torch.where(flat >= 0, flat, torch.full_like(flat, E))
    ordered, number = torch.sort(by, stable=True)
    counts = (by[None] == torch.arange(E, device=by.device)[:, None]).sum(1)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    places = torch.empty_like(number)
    places[number] = torch.arange(number.numel(), device=by.device)
    order = torch.where(ordered < E, number, torch.full_like(number, -1))
    places = torch.where(flat >= 0, places, torch.full_like(places, -1))
    return order.to(torch.int32), offsets.to(torch.int32), places.reshape(experts.shape).to(torch.int32)


def _logits_back(g, w, p, experts, normalize):
    """The logits' gradient out of the weights' gradient g."""
    gw = torch.where(experts >= 0, g * w, torch.zeros_like(w))
    total = gw.sum(-1, keepdim=True)
    dl = torch.zeros_like(p) if normalize else -p * total
    return dl.scatter_add(1, experts.clamp(min=0), torch.where(experts >= 0, gw - w * total if normalize else gw, torch.zeros_like(gw)))


def _plain_route(s):
    c = s["case"]
    experts, w, p = _choose(s["logits"].detach().float(), c["k"], c["normalize"])
    order, offsets, places = _plan(experts, c["E"])
    out = {"weights": w, "experts": experts.to(torch.int32), "order": order, "offsets": offsets, "places": places}
    if c["mode"] == "train":
        out["logits"] = _logits_back(s["dweights"], w, p, experts, c["normalize"]).to(s["logits"].dtype)
    return out


def _plain_grouped(s):
    c, dtype = s["case"], s["x"].dtype
    x, w = s["x"].detach(), s["weight"].detach()
    train = c["mode"] == "train"
    at = s["offsets"].tolist()
    y = x.new_zeros(c["R"], c["N"])
    got = {"y": y}
    if train:
        got["x"], got["weight"] = torch.zeros_like(x), torch.zeros_like(w)
        if c["bias"]:
            got["bias"] = torch.zeros_like(s["bias"].detach())
    for e in range(c["E"]):
        r = slice(at[e], at[e + 1])
        xe, we = x[r].float(), w[e].float()
        z = xe @ we.t()
        if c["bias"]:
            z = z + s["bias"].detach()[e].float()
        a, da = _act(c["act"], z)
        y[r] = a.to(dtype)
        if train:
            g = s["dout"][r].float() * da
            got["x"][r], got["weight"][e] = (g @ we).to(dtype), (g.t() @ xe).to(dtype)
            if c["bias"]:
                got["bias"][e] = g.sum(0).to(dtype)
    return got


def _plain_experts(s):
    c, dtype = s["case"], s["x"].dtype
    train, E, M, C = c["mode"] == "train", c["E"], c["B"] * c["T"], c["C"]
    one = lambda n: s[n].detach().float()
    x = one("x").reshape(M, C)
    experts, w, p = _choose(one("logits").reshape(M, E), c["k"], True)
    per_token = lambda t: t.repeat_interleave(c["T"], 0)
    total = torch.zeros_like(x)
    kept = []
    for e in range(E):
        token, j = torch.nonzero(experts == e, as_tuple=True)
        z = x[token] @ one("w_in")[e].t() + one("b_in")[e]
        a, da = _act(c["act"], z)
        y = a @ one("w_out")[e].t() + one("b_out")[e]
        we = w[token, j][:, None]
        total.index_add_(0, token, we * y)
        kept.append((token, j, a, da, y, we) if train else None)
    out = total * per_token(one("gate")) if c["gate"] else total
    if c["residual"]:
        out = out + one("residual").reshape(M, C)
    got = {"y": out.reshape(s["x"].shape).to(dtype)}
    if not train:
        return got
    g = s["dout"].float().reshape(M, C)
    if c["residual"]:
        got["residual"] = s["dout"]
    if c["gate"]:
        got["gate"] = (g * total).reshape(c["B"], c["T"], C).sum(1).to(dtype)
        g = g * per_token(one("gate"))
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    for n in ("w_in", "b_in", "w_out", "b_out"):
        got[n] = torch.empty_like(s[n].detach())
    for e, (token, j, a, da, y, we) in enumerate(kept):
        ge = g[token]
        dw[token, j] = (ge * y).sum(-1)
        ge = ge * we
        got["w_out"][e], got["b_out"][e] = (ge.t() @ a).to(dtype), ge.sum(0).to(dtype)
        ge = (ge @ one("w_out")[e]) * da
        got["w_in"][e], got["b_in"][e] = (ge.t() @ x[token]).to(dtype), ge.sum(0).to(dtype)
        dx.index_add_(0, token, ge @ one("w_in")[e])
    got["x"] = dx.reshape(s["x"].shape).to(dtype)
    got["logits"] = _logits_back(dw, w, p, experts, True).reshape(s["logits"].shape).to(dtype)
    return got


def _plain_int8(s):
    c, x = s["case"], s["x"]
    scale = x.float().abs().amax(-1, keepdim=True) / 127
    q = torch.where(scale > 0, torch.round(x.double() / torch.where(scale > 0, scale, 1).double()), 0.0)
    z = (q @ s["weight"].double().t()).float() * scale * s["scale"]
    if c["bias"]:
        z = z + s["bias"].float()
    y, _ = _act(c["act"], z)
    if c["gate"]:
        y = y * s["gate"].float()[:, None]
    if c["residual"]:
        y = y + s["residual"].float()
    return {"y": y.to(x.dtype)}


# ---------------------------------------------------------------------------------------
# the framework's operators, as a user calls them
# ---------------------------------------------------------------------------------------
def _own(s):
    """Outputs, and the one that gradients come back to."""
    import llsa_amd
    c = s["case"]
    if c["op"] == "route":
        r = llsa_amd.route_tokens(s["logits"], c["k"], normalize=c["normalize"])
        return {"weights": r.weights, "experts": r.experts, "order": r.order, "offsets": r.offsets, "places": r.places}, r.weights
    if c["op"] == "grouped":
        y = llsa_amd.grouped_linear(s["x"], s["weight"], s["offsets"], s.get("bias"), activation=c["act"] or None)
    elif c["op"] == "experts":
        r = llsa_amd.route_tokens(s["logits"], c["k"])
        y = llsa_amd.expert_feed_forward(s["x"], r, s["w_in"], s["b_in"], s["w_out"], s["b_out"], activation=c["act"], gate=s.get("gate"),
                                         residual=s.get("residual"))
    else:
        y = llsa_amd.linear_int8(s["x"], s["weight"], s["scale"], s.get("bias"), activation=c["act"] or None, gate=s.get("gate"), residual=s.get("residual"))
    return {"y": y}, y


PLAIN = {"route": _plain_route, "grouped": _plain_grouped, "experts": _plain_experts, "int8": _plain_int8}


def run(state):
    c = state["case"]
    if not own:
        with torch.no_grad():
            return PLAIN[c["op"]](state)
    if c["mode"] == "infer":
        with torch.no_grad():
            return _own(state)[0]
    leaves = _leaves(state)
    out, y = _own(state)
    grads = torch.autograd.grad(y, [t for _, t in leaves], state["dweights"] if c["op"] == "route" else state["dout"])
    return {**{n: t.detach() for n, t in out.items()}, **{n: g for (n, _), g in zip(leaves, grads)}}


def work(case):
    es, train = 4 if case["dtype"] == "fp32" else 2, case["mode"] == "train"
    E = case.get("E", 1)
    if case["op"] == "route":
        M, k = case["M"], case["k"]
        # logits in; weights, experts, order and places out; back: the weights' gradient in, the logits' out
        return {"bytes": es * M * E + 16 * M * k + 4 * (E + 1) + ((4 * M * k + es * M * E) if train else 0), "flops": M * E * (6 if train else 4)}
    if case["op"] == "grouped":
        R, K, N = case["R"], case["K"], case["N"]
        hit = max(1, min(E, R - case["tail"]))
        weights, rows, flops = (N * K + (N if case["bias"] else 0)), R * (K + N), 2 * (R - case["tail"]) * N * K
        # of the weights those that are hit in; back: dout in, dx out, all gradients of weights out
        return {"bytes": es * (rows * (2 if train else 1) + weights * (hit + (E if train else 0))), "flops": flops * (3 if train else 1)}
    M = case["B"] * case["T"]
    if case["op"] == "experts":
        C, F, k = case["C"], case["F"], case["k"]
        small = case["B"] * C if case["gate"] else 0
        weights, rows = 2 * C * F + C + F, M * (2 * C + E + (C if case["residual"] else 0))
        if train:                                             # dout in, the gradients of x and the logits out (the residual's is dout itself)
            rows += M * (2 * C + E)
        return {"bytes": es * (rows + weights * (min(E, M * k) + (E if train else 0)) + small * (2 if train else 1)), "flops": 4 * M * k * C * F * (3 if train else 1)}
    K, N = case["K"], case["N"]
    rows = M * (K + N + (N if case["residual"] else 0)) + (N if case["bias"] else 0) + (case["B"] * N if case["gate"] else 0)
    return {"bytes": es * rows + N * K + 4 * N, "flops": 2 * M * N * K}


# ---------------------------------------------------------------------------------------
# the definition in 64 bits, differentiated by autograd
# ---------------------------------------------------------------------------------------
ACTS = {"": lambda z: z, "silu": lambda z: z * torch.sigmoid(z), "gelu": lambda z: z * 0.5 * torch.erfc(-z / 2 ** 0.5),
        "gelu_tanh": lambda z: z * torch.sigmoid(2 * (2 / math.pi) ** 0.5 * (z + 0.044715 * z ** 3))}


def _exact_choice(logits, k, normalize):
    """Which experts (M, E) and with what weights, differentiable; chosen one after another."""
    left, taken = logits.detach().clone(), torch.zeros_like(logits, dtype=torch.bool)
    experts = []
    for _ in range(k):
        best = left.max(-1, keepdim=True).values
        first = ((left == best) & (best > -math.inf)).double()
        first = first * (first.cumsum(-1) == 1)               # of equal ones the first
        experts.append(torch.where(first.sum(-1) > 0, first.argmax(-1), -1))
        taken |= first > 0
        left = left.masked_fill(first > 0, -math.inf)
    over = taken if normalize else logits > -math.inf
    top = logits.detach().masked_fill(~over, -1e300).amax(-1, keepdim=True)
    e = torch.where(over, torch.exp(torch.where(over, logits - top, 0.0)), 0.0)
    total = e.sum(-1, keepdim=True)
    return torch.stack(experts, 1), torch.where(taken, e / torch.where(total > 0, total, 1.0), 0.0)


def exact(case, seed):
    s = prepare(case, seed)
    train = case["mode"] == "train"
    v = {n: t.detach().double().requires_grad_(train) for n, t in _leaves(s)} if case["op"] != "int8" else {}
    act = ACTS[case.get("act", "")]
    if case["op"] == "route":
        M, E, k = case["M"], case["E"], case["k"]
        experts, w = _exact_choice(v["logits"], k, case["normalize"])
        there = experts >= 0
        weights = torch.where(there, w.gather(1, experts.clamp(min=0)), 0.0)
        numbers = torch.arange(M * k, device=experts.device).reshape(M, k)
        runs = [numbers[experts == e] for e in range(E)]
        order = torch.cat(runs)
        places = torch.full((M * k,), -1, device=order.device)
        places[order] = torch.arange(order.numel(), device=order.device)
        offsets = torch.tensor([0] + [r.numel() for r in runs]).cumsum(0).to(order.device)
        order = torch.cat([order, order.new_full((M * k - order.numel(),), -1)])
        got = {"weights": weights.detach(), "experts": experts.to(torch.int32), "order": order.to(torch.int32), "offsets": offsets.to(torch.int32),
               "places": places.reshape(M, k).to(torch.int32)}
        if train:
            got["logits"] = torch.autograd.grad(weights, v["logits"], s["dweights"].double())[0]
        return got
    if case["op"] == "grouped":
        row = torch.arange(case["R"], device=s["offsets"].device)
        y = torch.zeros(case["R"], case["N"], device=row.device, dtype=torch.float64)
        for e in range(case["E"]):
            mine = torch.nonzero((row >= s["offsets"][e]) & (row < s["offsets"][e + 1]))[:, 0]
            z = torch.matmul(v["x"][mine], v["weight"][e].transpose(0, 1))
            y = y.index_copy(0, mine, act(z + v["bias"][e] if case["bias"] else z))
    elif case["op"] == "experts":
        M, C = case["B"] * case["T"], case["C"]
        x = v["x"].reshape(M, C)
        experts, w = _exact_choice(v["logits"].reshape(M, case["E"]), case["k"], True)
        y = torch.zeros(M, C, device=x.device, dtype=torch.float64)
        for e in range(case["E"]):
            token = torch.nonzero((experts == e).any(1))[:, 0]
            h = act(torch.matmul(x[token], v["w_in"][e].transpose(0, 1)) + v["b_in"][e])
            y = y.index_add(0, token, w[token, e, None] * (torch.matmul(h, v["w_out"][e].transpose(0, 1)) + v["b_out"][e]))
        y = y.reshape(s["x"].shape)
        if case["gate"]:
            y = v["gate"].unsqueeze(1) * y
        if case["residual"]:
            y = y + v["residual"]
    else:
        x = s["x"].double()
        step = (x.abs().max(-1, keepdim=True).values.float() / 127).double()
        q = torch.where(step > 0, (x / torch.where(step > 0, step, 1.0)).round(), 0.0)
        z = step * s["scale"].double() * torch.matmul(q, s["weight"].double().transpose(0, 1))
        y = act(z + s["bias"].double() if case["bias"] else z)
        if case["gate"]:
            y = s["gate"].double().unsqueeze(1) * y
        if case["residual"]:
            y = s["residual"].double() + y
    got = {"y": y.detach()}
    if train:
        got.update(zip(v, torch.autograd.grad(y, list(v.values()), s["dout"].double())))
    return got
