"""Weights that PixelDiT.quantize_for_sampling() keeps in 8-bit integers follow the weights they were made of: loaded, replaced, written to, cast, moved, copied, saved."""
import contextlib
import copy
import io

import pytest
import torch

import llsa_amd
from emu_util import emu_lib
from llsa_amd._lib import override_library_for_tests
from llsa_amd.caller import dit as D

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def dev(request):
    with contextlib.ExitStack() as stack:
        if request.param == "cpu":
            stack.enter_context(override_library_for_tests(emu_lib()))
        yield torch.device(request.param)


def _layer(dev, dtype=FP32, seed=0):
    torch.manual_seed(seed)
    layer = torch.nn.Linear(48, 40).to(dev, dtype)
    D.keep_in_8_bits(layer)
    return layer


def _x(dev, dtype=BF16):
    return torch.randn(2, 9, 48, generator=torch.Generator().manual_seed(5)).to(dtype).to(dev)


def _is_of_its_weight(layer, x):
    """The layer's result is that of its present weight, quantised."""
    with torch.no_grad():
        q, s = llsa_amd.quantize_rows(layer.weight)
        want = llsa_amd.linear_int8(x, q, s, layer.bias.to(x.dtype))
        for _ in range(2):
            assert torch.equal(D.project(layer, x), want)
            assert torch.equal(D.project(layer, x, llsa_amd.quantize_rows(x)), want)
    return want


def _load(layer):
    layer.load_state_dict({n: v * 2 - 0.1 for n, v in layer.state_dict().items()})


def _assign(layer):
    layer.load_state_dict({n: v * 2 - 0.1 for n, v in layer.state_dict().items()}, assign=True)


def _step(layer):
    for p in layer.parameters():
        p.grad = torch.randn(p.shape, generator=torch.Generator().manual_seed(3)).to(p)
    torch.optim.AdamW(layer.parameters(), lr=0.1).step()


def _write(layer):
    with torch.no_grad():
        layer.weight[3, 5] += 17


def _write_detached(layer):
    layer.weight.detach().mul_(torch.linspace(1, 3, 48).to(layer.weight))


def _replace(layer):
    layer.weight = torch.nn.Parameter(layer.weight.detach() + 1)


def _replace_data(layer):
    layer.weight.data = layer.weight.data + 1


@pytest.mark.parametrize("change", [_load, _assign, _step, _write, _write_detached, _replace, _replace_data], ids=lambda f: f.__name__)
def test_weights_that_change(dev, change):
    layer, x = _layer(dev), _x(dev)
    before = _is_of_its_weight(layer, x)
    for _ in range(2):
        change(layer)
        after = _is_of_its_weight(layer, x)
        assert not torch.equal(before, after)
        before = after


@pytest.mark.parametrize("first,then", [(FP32, [BF16]), (FP32, [FP16, FP32]), (FP32, [BF16, FP32, BF16]), (BF16, [BF16]), (FP16, [FP16, FP32])])
def test_casts(dev, first, then):
    layer = _layer(dev, first)
    _is_of_its_weight(layer, _x(dev))
    for t in then:
        layer = layer.to(t)
        _is_of_its_weight(layer, _x(dev, BF16 if t == FP32 else t))


def test_memory_that_is_used_again(dev):
    """Another weight where the old one lay, written to as often."""
    layer, x = _layer(dev), _x(dev)
    _is_of_its_weight(layer, x)
    for k in range(4):
        value = torch.randn(40, 48, generator=torch.Generator().manual_seed(k))
        layer.weight = None
        layer.weight = torch.nn.Parameter(value.to(dev))
        _is_of_its_weight(layer, x)


def test_copies_and_files(dev):
    layer, x = _layer(dev), _x(dev)
    want = _is_of_its_weight(layer, x)
    other = copy.deepcopy(layer)
    file = io.BytesIO()
    torch.save(layer, file)
    file.seek(0)
    loaded = torch.load(file, weights_only=False)             # (what was written above)
    assert set(layer.state_dict()) == {"weight", "bias"}
    for v in (other, loaded):
        assert torch.equal(_is_of_its_weight(v, x), want)
        _write(v)
        assert not torch.equal(_is_of_its_weight(v, x), want) and torch.equal(_is_of_its_weight(layer, x), want)


def test_weights_of_inference_mode(dev):
    with torch.inference_mode():
        layer = _layer(dev)
        x = _x(dev)
        _is_of_its_weight(layer, x)
        layer.weight = torch.nn.Parameter(layer.weight * 2)
        _is_of_its_weight(layer, x)
    layer = _layer(dev)
    with torch.inference_mode():
        _is_of_its_weight(layer, _x(dev))
    _write(layer)
    _is_of_its_weight(layer, _x(dev))


def test_nothing_is_made_twice(dev, monkeypatch):
    layer, x = _layer(dev), _x(dev)
    made = []
    monkeypatch.setattr(D, "quantize_rows", lambda v: made.append(v.shape) or llsa_amd.quantize_rows(v))
    where = layer.weight_q.data_ptr(), layer.weight_scale.data_ptr()
    with torch.no_grad():
        for _ in range(3):
            D.project(layer, x)
        assert not made
        _write(layer)
        for _ in range(3):
            D.project(layer, x)
    assert made == [(40, 48)] and where == (layer.weight_q.data_ptr(), layer.weight_scale.data_ptr())


def _sample(model, dev):
    g = torch.Generator().manual_seed(0)
    images, t = torch.randn(1, 3, 32, 32, generator=g).to(dev), torch.tensor([300], device=dev)
    with torch.no_grad(), torch.autocast(device_type=dev.type, dtype=BF16):
        return model(images, t)


def test_a_model(dev):
    """Loaded weights are sampled with at once; quantize_for_sampling(False) gives the model back as it was."""
    make = lambda seed: torch.manual_seed(seed) and D.PixelDiT(num_attention_heads=1, num_layers=1, sample_size=32, levels=1, sparse_topk=8, fused_layers=True).to(dev)
    a, b = make(1), make(2)
    assert a.quantize_for_sampling() is a
    a.load_state_dict(b.state_dict())
    got = _sample(a, dev)
    assert torch.equal(got, _sample(b.quantize_for_sampling(), dev))
    if dev.type == "cpu":
        return                                                # (the emulation takes 13 s for each pass)
    plain = _sample(b.quantize_for_sampling(False), dev)
    assert not torch.equal(got, plain)
    assert a.quantize_for_sampling(False) is a and torch.equal(_sample(a, dev), plain)
    assert not any("weight_" in n for n, _ in a.named_buffers())
    a.quantize_for_sampling(False)
    with torch.autocast(device_type=dev.type, dtype=BF16):
        a(torch.zeros(1, 3, 32, 32, device=dev), torch.tensor([3], device=dev)).float().sum().backward()
    assert a.transformer_blocks[0].ff_in.weight.grad is not None


@pytest.mark.gpu
def test_captured_samples():
    """A graph reads the integers where they lie, so that it follows once they have been made again; one captured while they were out of date makes them itself."""
    dev = torch.device("cuda")
    layer, x = _layer(dev), _x(dev)

    def capture():
        graph = torch.cuda.CUDAGraph()
        with torch.no_grad(), torch.cuda.graph(graph):
            out = D.project(layer, x)
        return graph, out

    _is_of_its_weight(layer, x)
    torch.cuda.synchronize()
    graphs = [capture()]
    _write(layer)
    torch.cuda.synchronize()
    graphs.append(capture())
    for k in range(3):
        _write_detached(layer)
        want = _is_of_its_weight(layer, x)
        for graph, out in graphs:
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want), k
