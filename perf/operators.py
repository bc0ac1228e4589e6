"""The operators around the attention of a transformer block, as plain cases: the layer norm with the modulation that the
timestep gives it, the linear layer with bias, activation, gate and residual in one pass, and the feed-forward block made of
two of them; forward alone (sampling) and forward + backward (training).

A case: {"op": "norm" | "linear" | "ffn", "mode": "infer" | "train", "dtype": "bf16" | "fp16" | "fp32" (norm only), "B", "T":
samples and tokens of each, ...} and for

  norm     "C" channels, "affine": a weight and a bias for each channel, "mod": scale and shift for each sample and channel
  linear   "K" channels in, "N" channels out, "act": "" | "silu" | "gelu" | "gelu_tanh", "bias", "gate": a factor for each sample
           and channel out, "residual": added to the result
  ffn      "C" channels, "F" hidden channels, "act", "gate", "residual" as above

Formulas, for a row x of a sample b (all sums over channels):

  norm     n = (x - mean(x)) / sqrt(mean((x - mean(x))^2) + eps) * weight + bias,   y = n * (1 + scale_b) + shift_b
  linear   y = residual + gate_b * act(W x + bias)
  ffn      y = residual + gate_b * (W_out act(W_in x + b_in) + b_out)
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


def _norm(name, mode, dtype, B, T, C, affine=False, mod=False):
    return {"name": name, "op": "norm", "mode": mode, "dtype": dtype, "B": B, "T": T, "C": C, "affine": affine, "mod": mod}


def _linear(name, mode, dtype, B, T, K, N, act="", bias=True, gate=False, residual=False):
    return {"name": name, "op": "linear", "mode": mode, "dtype": dtype, "B": B, "T": T, "K": K, "N": N, "act": act, "bias": bias,
            "gate": gate, "residual": residual}


def _ffn(name, mode, dtype, B, T, C, F, act="gelu_tanh", gate=False, residual=False):
    return {"name": name, "op": "ffn", "mode": mode, "dtype": dtype, "B": B, "T": T, "C": C, "F": F, "act": act, "gate": gate,
            "residual": residual}


def listed():
    return [
        # the norm in front of the attention while one image of 32 x 32 pixels is sampled: a launch, hardly any work
        _norm("norm_infer_1k", "infer", "bf16", 1, 1024, 384, mod=True),
        # the same norm in the DiT-S training step: batch 8 of 128 x 128 pixels
        _norm("norm_train_layer", "train", "bf16", 8, 16384, 384, mod=True),
        # rows of an odd length, in 32 bits, with weights of its own
        _norm("norm_train_odd", "train", "fp32", 3, 1531, 777, affine=True),
        # wide rows in half precision, weights and modulation
        _norm("norm_train_wide", "train", "fp16", 2, 4096, 2048, affine=True, mod=True),
        # the first layer of the timestep embedding: one row for each image of the batch
        _linear("linear_infer_rows", "infer", "bf16", 8, 1, 256, 384, act="silu"),
        # the layer that makes the six modulation vectors of a block, in training: all weights, eight rows
        _linear("linear_train_rows", "train", "bf16", 8, 1, 384, 2304),
        # the attention's output projection in the training step: gated, onto the residual stream
        _linear("linear_train_layer", "train", "bf16", 8, 16384, 384, 384, gate=True, residual=True),
        # odd sizes all round
        _linear("linear_train_odd", "train", "fp16", 3, 1531, 777, 333, act="gelu", residual=True),
        # a generic square projection, bound by the matrix units
        _linear("linear_infer_wide", "infer", "bf16", 1, 8192, 4096, 4096),
        # the feed-forward block while one small image is sampled
        _ffn("ffn_infer_1k", "infer", "bf16", 1, 1024, 384, 1536, gate=True, residual=True),
        # the feed-forward block of the DiT-S training step
        _ffn("ffn_train_layer", "train", "bf16", 8, 16384, 384, 1536, gate=True, residual=True),
        # odd token and channel counts, another activation
        _ffn("ffn_train_odd", "train", "fp16", 3, 1531, 333, 1001, act="silu", residual=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def _channels(rng, hi):
    """Multiples of 64, of 8, and any count at all."""
    step = rng.choice([64, 64, 8, 1])
    return step * _log_int(rng, max(1, 16 // step), hi // step)


def draw(rng):
    op = rng.choice(["norm", "linear", "linear", "ffn", "ffn"])
    mode = rng.choice(["infer", "train", "train"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16"])
    B, T = rng.randint(1, 8), _log_int(rng, 1, 16384)
    if op == "norm":
        kind = rng.choice([(True, False), (False, True), (False, True), (True, True), (False, False)])
        c = _norm("", mode, rng.choice([dtype, dtype, "fp32"]), B, T, _channels(rng, 4096), *kind)
        most = {"bytes": 0.6e9, "flops": 1e15}
    elif op == "linear":
        c = _linear("", mode, dtype, B, T, _channels(rng, 4096), _channels(rng, 4096), rng.choice(["", "", "silu", "gelu", "gelu_tanh"]),
                    rng.random() < 0.8, rng.random() < 0.3, rng.random() < 0.4)
        most = {"bytes": 0.7e9, "flops": 0.27e12}
    else:
        C = _channels(rng, 1024)
        c = _ffn("", mode, dtype, B, T, C, rng.choice([4 * C, 2 * C, _channels(rng, 2048)]), rng.choice(["gelu_tanh", "gelu_tanh", "gelu", "silu"]),
                 rng.random() < 0.6, rng.random() < 0.8)
        most = {"bytes": 0.7e9, "flops": 0.9e12}
    del c["name"]
    while any(work(c)[k] > most[k] for k in most) and (c["B"] > 1 or c["T"] > 1):
        if c["B"] > 1:
            c["B"] -= 1
        else:
            c["T"] = c["T"] * 2 // 3
    return c


def prepare(case, seed):
    dev, dtype = torch.device("cuda"), DTYPES[case["dtype"]]
    gen = torch.Generator(device=dev).manual_seed(seed)
    train = case["mode"] == "train"
    B, T = case["B"], case["T"]

    def normal(*shape, std=1.0, mean=0.0):
        return (torch.randn(*shape, device=dev, generator=gen) * std + mean).to(dtype).requires_grad_(train)

    def weight(n, k):                                         # as a linear layer starts: uniform, 1 / sqrt(fan in)
        return ((torch.rand(n, k, device=dev, generator=gen) * 2 - 1) / math.sqrt(k)).to(dtype).requires_grad_(train)

    s = {"case": case}
    if case["op"] == "norm":
        C = case["C"]
        s["x"] = normal(B, T, C, mean=0.3)
        if case["affine"]:
            s["weight"], s["bias"] = normal(C, std=0.1, mean=1.0), normal(C, std=0.1)
        if case["mod"]:
            s["scale"], s["shift"] = normal(B, C, std=0.2), normal(B, C, std=0.2)
        out = C
    elif case["op"] == "linear":
        K, out = case["K"], case["N"]
        s["x"], s["weight"] = normal(B, T, K), weight(out, K)
        if case["bias"]:
            s["bias"] = normal(out, std=0.1)
    else:
        out, F = case["C"], case["F"]
        s["x"], s["w_in"], s["b_in"], s["w_out"], s["b_out"] = normal(B, T, out), weight(F, out), normal(F, std=0.1), weight(out, F), normal(out, std=0.1)
    if case["op"] != "norm" and case["gate"]:
        s["gate"] = normal(B, out, std=0.3, mean=0.5)
    if case["op"] != "norm" and case["residual"]:
        s["residual"] = normal(B, T, out)
    if train:
        s["dout"] = torch.randn(B, T, out, device=dev, generator=gen).to(dtype)
    return s


def _leaves(s):
    """What a training step wants the gradients of, by name."""
    names = ["x", "weight", "bias", "scale", "shift", "w_in", "b_in", "w_out", "b_out", "gate", "residual"]
    return [(n, s[n]) for n in names if n in s]


# ---------------------------------------------------------------------------------------
# plain forms: elementary operations in 32 bits
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


def _plain_norm(s):
    c = s["case"]
    x = s["x"].detach().float()
    one = lambda n: s[n].detach().float() if n in s else None
    w, b, sc, sh = one("weight"), one("bias"), one("scale"), one("shift")
    d = x - x.mean(-1, keepdim=True)
    r = 1 / torch.sqrt((d * d).mean(-1, keepdim=True) + EPS)
    h = d * r
    n = h * w + b if w is not None else h
    y = n * (1 + sc[:, None]) + sh[:, None] if sc is not None else n
    out = {"y": y.to(s["x"].dtype)}
    if c["mode"] == "infer":
        return out
    g = s["dout"].float()
    if sc is not None:
        out["scale"], out["shift"] = (g * n).sum(1).to(s["scale"].dtype), g.sum(1).to(s["shift"].dtype)
        g = g * (1 + sc[:, None])
    if w is not None:
        out["weight"], out["bias"] = (g * h).sum((0, 1)).to(s["weight"].dtype), g.sum((0, 1)).to(s["bias"].dtype)
        g = g * w
    out["x"] = (r * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))).to(s["x"].dtype)
    return out


def _plain_layers(s):
    """Both kinds of linear layers, as one chain of (weight, bias, activation)."""
    c, dtype = s["case"], s["x"].dtype
    train = c["mode"] == "train"
    layers = [("weight", "bias", c["act"])] if c["op"] == "linear" else [("w_in", "b_in", c["act"]), ("w_out", "b_out", "")]
    one = lambda n: s[n].detach().float() if n in s else None
    h = one("x").reshape(c["B"] * c["T"], -1)
    kept = []
    for wn, bn, act in layers:
        z = h @ one(wn).t()
        if bn in s:
            z = z + one(bn)
        a, da = _act(act, z)
        kept.append((h, da))
        h = a
    y = h.reshape(c["B"], c["T"], -1)
    out = y * one("gate")[:, None] if "gate" in s else y
    if "residual" in s:
        out = out + one("residual")
    got = {"y": out.to(dtype)}
    if not train:
        return got
    g = s["dout"].float()
    if "residual" in s:
        got["residual"] = s["dout"]
    if "gate" in s:
        got["gate"] = (g * y).sum(1).to(dtype)
        g = g * one("gate")[:, None]
    g = g.reshape(c["B"] * c["T"], -1)
    for (wn, bn, act), (h, da) in zip(layers[::-1], kept[::-1]):
        if act:
            g = g * da
        got[wn] = (g.t() @ h).to(dtype)
        if bn in s:
            got[bn] = g.sum(0).to(dtype)
        g = g @ one(wn)
    got["x"] = g.reshape(s["x"].shape).to(dtype)
    return got


# ---------------------------------------------------------------------------------------
# the framework's operators, as a user calls them
# ---------------------------------------------------------------------------------------
def _own(s):
    import llsa_amd
    c = s["case"]
    if c["op"] == "norm":
        return llsa_amd.layer_norm(s["x"], s.get("weight"), s.get("bias"), scale=s.get("scale"), shift=s.get("shift"), eps=EPS)
    if c["op"] == "linear":
        return llsa_amd.linear(s["x"], s["weight"], s.get("bias"), activation=c["act"] or None, gate=s.get("gate"), residual=s.get("residual"))
    return llsa_amd.feed_forward(s["x"], s["w_in"], s["b_in"], s["w_out"], s["b_out"], activation=c["act"], gate=s.get("gate"),
                                 residual=s.get("residual"))


def run(state):
    if not own:
        with torch.no_grad():
            return _plain_norm(state) if state["case"]["op"] == "norm" else _plain_layers(state)
    if state["case"]["mode"] == "infer":
        with torch.no_grad():
            return {"y": _own(state)}
    leaves = _leaves(state)
    y = _own(state)
    grads = torch.autograd.grad(y, [t for _, t in leaves], state["dout"])
    return {"y": y.detach(), **{n: g for (n, _), g in zip(leaves, grads)}}


def work(case):
    es, train = 4 if case["dtype"] == "fp32" else 2, case["mode"] == "train"
    B, M = case["B"], case["B"] * case["T"]
    if case["op"] == "norm":
        C = case["C"]
        small = (2 * C if case["affine"] else 0) + (2 * B * C if case["mod"] else 0)
        # forward: x in, y out; backward besides: dy in, dx out, the gradients of the small inputs out
        return {"bytes": es * (M * C * (4 if train else 2) + small * (2 if train else 1)), "flops": (16 if train else 6) * M * C}
    if case["op"] == "linear":
        K, N = case["K"], case["N"]
        weights = N * K + (N if case["bias"] else 0)
        macs = M * N * K
    else:
        K = N = case["C"]
        weights = 2 * case["F"] * N + case["F"] + N
        macs = 2 * M * N * case["F"]
    small = weights + (B * N if case["gate"] else 0)
    rows = M * K + M * N + (M * N if case["residual"] else 0)
    if train:                                                 # dout in, dx out, the residual's gradient is dout itself
        rows += M * N + M * K
    return {"bytes": es * (rows + small * (2 if train else 1)), "flops": 2 * macs * (3 if train else 1)}


# ---------------------------------------------------------------------------------------
# the definition in 64 bits, differentiated by autograd
# ---------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    v = {n: t.detach().double().requires_grad_(case["mode"] == "train") for n, t in _leaves(s)}
    per_sample = lambda t: t.unsqueeze(1)
    acts = {"": lambda z: z, "silu": lambda z: z * torch.sigmoid(z), "gelu": lambda z: z * 0.5 * torch.erfc(-z / 2 ** 0.5),
            "gelu_tanh": lambda z: z * torch.sigmoid(2 * (2 / math.pi) ** 0.5 * (z + 0.044715 * z ** 3))}
    if case["op"] == "norm":
        x = v["x"]
        mean = x.sum(-1, keepdim=True) / case["C"]
        var = ((x - mean) ** 2).sum(-1, keepdim=True) / case["C"]
        y = (x - mean) * (var + EPS) ** -0.5
        if case["affine"]:
            y = y * v["weight"] + v["bias"]
        if case["mod"]:
            y = y + y * per_sample(v["scale"]) + per_sample(v["shift"])
    else:
        if case["op"] == "linear":
            y = torch.matmul(v["x"], v["weight"].transpose(0, 1))
            y = acts[case["act"]](y + v["bias"] if case["bias"] else y)
        else:
            h = acts[case["act"]](torch.matmul(v["x"], v["w_in"].transpose(0, 1)) + v["b_in"])
            y = torch.matmul(h, v["w_out"].transpose(0, 1)) + v["b_out"]
        if case["gate"]:
            y = per_sample(v["gate"]) * y
        if case["residual"]:
            y = y + v["residual"]
    got = {"y": y.detach()}
    if case["mode"] == "train":
        got.update(zip(v, torch.autograd.grad(y, list(v.values()), s["dout"].double())))
    return got
