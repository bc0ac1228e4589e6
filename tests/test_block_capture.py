"""Captured training steps that use a leaf more than once: x in three projections, a weight that is tied to another layer's, a block that runs twice.  Its
gradients' accumulator is then alive when the second call comes, and belongs to the graph that is being captured."""
import pytest
import torch

import llsa_amd

BF16 = torch.bfloat16


def _leaves(seed, B=2, T=50, C=24, F=40):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: (torch.randn(*s, generator=g) * 0.5).to(BF16).cuda().requires_grad_()
    return {"x": r(B, T, C), "wq": r(F, C), "wk": r(F, C), "wv": r(F, C), "w1": r(F, C), "b1": r(F), "w2": r(C, F), "n": r(C), "gate": r(B, C)}


def _projections(t):
    q, k, v = (llsa_amd.linear(t["x"], t[n]) for n in ("wq", "wk", "wv"))
    return q * k + v


def _tied(t):
    return llsa_amd.linear(llsa_amd.linear(t["x"], t["wq"], activation="silu"), t["wk"].t()) + llsa_amd.linear(t["x"], t["wk"]) @ t["wq"]


def _twice(t):
    x = t["x"]
    for _ in range(2):
        h = llsa_amd.layer_norm(x, t["n"], scale=t["gate"])
        x = llsa_amd.feed_forward(h, t["w1"], t["b1"], t["w2"], gate=t["gate"], residual=x)
    return x


def _step(f, t, how):
    y = f(t)
    dout = torch.ones_like(y)
    used = [v for n, v in t.items() if n in {_projections: ("x", "wq", "wk", "wv"), _tied: ("x", "wq", "wk"), _twice: ("x", "w1", "b1", "w2", "n", "gate")}[f]]
    if how == "grad":
        return [y.detach()] + list(torch.autograd.grad(y, used, dout))
    for v in used:
        v.grad = None
    y.backward(dout)
    return [y.detach()] + [v.grad for v in used]


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["grad", "backward"])
@pytest.mark.parametrize("f", [_projections, _tied, _twice])
def test_leaves_that_are_used_twice(f, how):
    t = _leaves(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            _step(f, t, how)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for v in t.values():
        v.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = _step(f, t, how)
    for seed in (1, 2, 3):
        new = _leaves(seed)
        with torch.no_grad():
            for n, v in new.items():
                t[n].copy_(v)
        eager = [v.clone() for v in _step(f, new, how)]
        graph.replay()
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(eager, captured)):
            assert torch.equal(a, b), i


@pytest.mark.gpu
def test_an_accumulator_of_another_stream_is_refused():
    """Alive since a forward on a stream of its own, and by the capture's own stream: the first is an error, the second none."""
    t = _leaves(0)
    other, own = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for stream in (other, own):
        with torch.cuda.stream(stream):
            alive = _projections(t)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        if stream is other:
            with pytest.raises(RuntimeError, match="another graph"), torch.cuda.graph(graph, stream=own):
                _projections(t)
        else:
            with torch.cuda.graph(graph, stream=own):
                y = _projections(t)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y.detach(), alive.detach())
            del y
        del alive
