"""The small DiT with its norms, linear layers and feed-forward blocks by this package's operators (fused_layers=True) against the same
model with torch's: one flow-matching step, loss and every parameter's gradient."""
import pytest
import torch

from emu_util import emu_lib
from llsa_amd._lib import override_library_for_tests
from llsa_amd.caller import dit as D


def _step(model, batch):
    model.zero_grad(set_to_none=True)
    loss = D.FlowMatchingStep(model).loss(*batch)
    loss.backward()
    return loss.item(), {n: p.grad.detach().clone() for n, p in model.named_parameters() if p.grad is not None}


def _compare(dev, B, **cfg):
    torch.manual_seed(3)
    plain = D.PixelDiT(**cfg).to(dev)
    fused = D.PixelDiT(fused_layers=True, **cfg).to(dev)
    fused.load_state_dict(plain.state_dict())
    g = torch.Generator().manual_seed(0)
    side = cfg["sample_size"]
    batch = [t.to(dev) for t in (torch.randn(B, 3, side, side, generator=g).clamp(-1, 1), torch.randn(B, 3, side, side, generator=g), torch.randint(0, 1000, (B,), generator=g))]
    (loss, grads), (ref_loss, ref) = _step(fused, batch), _step(plain, batch)
    assert set(grads) == set(ref)
    # Both sides round activations and gradients to bf16 between layers, the plain one more often.  A chain of n roundings of u = 2^-9 (rms of a
    # half step's 2^-8 and less) is off by about sqrt(n) u: below 5 % for the few hundred of either side.
    assert abs(loss - ref_loss) <= 1e-2 * abs(ref_loss), (loss, ref_loss)
    for n, r in ref.items():
        # (what acts only through the scores also sees which of two nearly equal blocks was chosen)
        if any(t in n for t in ("to_q.", "to_k.", "norm_q_weight", "norm_k_weight")):
            assert torch.isfinite(grads[n]).all()
            continue
        err = ((grads[n] - r).norm() / r.norm().clamp_min(1e-12)).item()
        assert err <= 5e-2, f"gradient of {n} differs by rel-L2 {err:.3e}"


def test_fused_layers_emulated():
    with override_library_for_tests(emu_lib()):
        _compare(torch.device("cpu"), 1, num_attention_heads=1, num_layers=1, sample_size=32, levels=1, sparse_topk=8)


@pytest.mark.gpu
@pytest.mark.parametrize("B,heads,levels,side", [(1, 1, 1, 32), (3, 2, 1, 64), (2, 2, 2, 128)])
def test_fused_layers_gpu(B, heads, levels, side):
    _compare(torch.device("cuda:0"), B, num_attention_heads=heads, num_layers=2, sample_size=side, levels=levels, sparse_topk=8)


@pytest.mark.gpu
def test_fused_layers_optimise():
    """A few AdamW steps run, and every parameter moves."""
    torch.manual_seed(0)
    model = D.PixelDiT(num_attention_heads=2, num_layers=2, sample_size=64, levels=1, fused_layers=True).to("cuda")
    before = {n: p.detach().clone() for n, p in model.named_parameters()}
    step = D.FlowMatchingStep(model, lr=1e-3)
    g = torch.Generator().manual_seed(0)
    batch = [t.cuda() for t in (torch.randn(2, 3, 64, 64, generator=g), torch.randn(2, 3, 64, 64, generator=g), torch.randint(0, 1000, (2,), generator=g))]
    for _ in range(3):
        assert torch.isfinite(step(*batch))
    for n, p in model.named_parameters():
        assert torch.isfinite(p).all() and not torch.equal(p, before[n]), n
