"""The small DiT with experts in its feed-forward blocks, and with weights in 8-bit integers: the operators together, as a model calls them."""
import math

import pytest
import torch
import torch.nn.functional as F

import llsa_amd
from emu_util import emu_lib
from llsa_amd._lib import override_library_for_tests
from llsa_amd.caller import dit as D


def _model(dev, side, layers=1, heads=1, **cfg):
    torch.manual_seed(3)
    return D.PixelDiT(num_attention_heads=heads, num_layers=layers, sample_size=side, levels=1, sparse_topk=8, fused_layers=True, **cfg).to(dev)


def _batch(dev, B, side):
    g = torch.Generator().manual_seed(0)
    return [t.to(dev) for t in (torch.randn(B, 3, side, side, generator=g).clamp(-1, 1), torch.randn(B, 3, side, side, generator=g), torch.randint(0, 1000, (B,), generator=g))]


def _plain_experts(self, x, gate, residual):
    """What Experts.forward does, in torch's operations in fp32, on the bf16 values that it is given."""
    rows = x.float()
    logits = rows @ self.router.weight.to(x.dtype).float().t()
    w_in, b_in, w_out, b_out = (p.to(x.dtype).float() for p in (self.w_in, self.b_in, self.w_out, self.b_out))
    chosen = torch.zeros(logits.shape, dtype=torch.bool, device=x.device)
    with torch.no_grad():                                     # (by the logits that the model itself rounds to bf16)
        chosen.scatter_(-1, llsa_amd.route_tokens(llsa_amd.linear(x, self.router.weight.to(x.dtype)), self.experts_per_token).experts.long(), True)
    p = torch.softmax(torch.where(chosen, logits, torch.full_like(logits, -math.inf)), -1)
    y = 0
    for e in range(logits.shape[-1]):
        y = y + p[..., e, None] * (F.gelu(rows @ w_in[e].t() + b_in[e], approximate="tanh") @ w_out[e].t() + b_out[e])
    return (residual.float() + gate.float().unsqueeze(1) * y).to(x.dtype)


def _step(model, batch):
    model.zero_grad(set_to_none=True)
    loss = D.FlowMatchingStep(model).loss(*batch)
    loss.backward()
    return loss.item(), {n: p.grad.detach().clone() for n, p in model.named_parameters() if p.grad is not None}


def _compare(dev, B, side, monkeypatch, **cfg):
    model, batch = _model(dev, side, num_experts=4, **cfg), _batch(dev, B, side)
    loss, grads = _step(model, batch)
    with monkeypatch.context() as m:
        m.setattr(D.Experts, "forward", _plain_experts)
        ref_loss, ref = _step(model, batch)
    assert set(grads) == set(ref) and any("router" in n for n in ref) and any("w_out" in n for n in ref)
    # The blocks' rows are rounded to bf16 on one side and not on the other.  A chain of n roundings of u = 2^-9 (rms of a half step's 2^-8 and less) is off
    # by about sqrt(n) u: below 5 % for the few hundred of either side.
    assert abs(loss - ref_loss) <= 1e-2 * abs(ref_loss), (loss, ref_loss)
    for n, r in ref.items():
        # (what acts only through scores also sees which of two nearly equal blocks or experts was chosen)
        if any(t in n for t in ("to_q.", "to_k.", "norm_q_weight", "norm_k_weight")):
            assert torch.isfinite(grads[n]).all()
            continue
        err = ((grads[n] - r).norm() / r.norm().clamp_min(1e-12)).item()
        assert err <= 5e-2, f"gradient of {n} differs by rel-L2 {err:.3e}"


def test_experts_emulated(monkeypatch):
    with override_library_for_tests(emu_lib()):
        _compare(torch.device("cpu"), 1, 32, monkeypatch)


@pytest.mark.gpu
@pytest.mark.parametrize("B,heads,side", [(2, 1, 32), (3, 2, 64)])
def test_experts_gpu(B, heads, side, monkeypatch):
    _compare(torch.device("cuda:0"), B, side, monkeypatch, layers=2, heads=heads)


def test_experts_need_fused_layers():
    with pytest.raises(ValueError, match="fused_layers"):
        D.PixelDiT(num_attention_heads=1, num_layers=1, sample_size=32, levels=1, num_experts=4)
    with pytest.raises(ValueError, match="fused_layers"):
        D.PixelDiT(num_attention_heads=1, num_layers=1, sample_size=32, levels=1).quantize_for_sampling()


@pytest.mark.gpu
def test_experts_optimise():
    """A few AdamW steps run, and every parameter moves."""
    model = _model("cuda", 64, layers=2, heads=2, num_experts=8)
    before = {n: p.detach().clone() for n, p in model.named_parameters()}
    step, batch = D.FlowMatchingStep(model, lr=1e-3), _batch("cuda", 2, 64)
    for _ in range(3):
        assert torch.isfinite(step(*batch))
    for n, p in model.named_parameters():
        assert torch.isfinite(p).all() and not torch.equal(p, before[n]), n


def _sample(model, dev, B, side):
    images, _, t = _batch(dev, B, side)
    with torch.no_grad(), torch.autocast(device_type=images.device.type, dtype=torch.bfloat16):
        return model(images, t).float()


def _check_8_bits(dev, B, side, **cfg):
    model = _model(dev, side, **cfg)
    plain = _sample(model, dev, B, side)
    model.quantize_for_sampling()
    for p in model.parameters():
        p.requires_grad_(False)
    got = _sample(model, dev, B, side)
    assert torch.isfinite(got).all() and not torch.equal(got, plain)
    # Either operand of a projection is off by up to half a step, 1/254 of its row's largest value, uniformly: rms of 1/254/sqrt(3), which for rows of a normal or
    # uniform distribution, whose largest values are up to 4 times their rms, is 0.9 % of them.  Two operands, six projections a block on top of one another, each a part of
    # the residual stream: below sqrt(12 layers) * 0.9 % of the result.
    layers = cfg.get("layers", 1)
    assert (got - plain).norm() <= math.sqrt(12 * layers) * 0.009 * plain.norm()


def test_8_bits_emulated():
    with override_library_for_tests(emu_lib()):
        _check_8_bits(torch.device("cpu"), 1, 32)


@pytest.mark.gpu
@pytest.mark.parametrize("cfg", [dict(), dict(num_experts=4)])
def test_8_bits_gpu(cfg):
    _check_8_bits(torch.device("cuda:0"), 2, 64, layers=2, heads=2, **cfg)
