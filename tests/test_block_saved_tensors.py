"""Saved-tensor hooks that give back something else than they were given: layer_norm, linear and feed_forward read the sizes and the type of what they
saved from their own node, so each single one is an error and none is read."""
import contextlib

import pytest
import torch

import llsa_amd
from emu_util import emu_lib
from llsa_amd._lib import override_library_for_tests

BF16 = torch.bfloat16


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def dev(request):
    with contextlib.ExitStack() as stack:
        if request.param == "cpu":
            stack.enter_context(override_library_for_tests(emu_lib()))
        yield torch.device(request.param)


def _calls(dev, T):
    """name -> a forward of leaves; T = 50 rows a sample: gates in the weights, T = 9: in the rows.  Odd channels: padded copies are saved."""
    g = torch.Generator().manual_seed(0)
    r = lambda *s, dtype=BF16: torch.randn(*s, generator=g).to(dtype).to(dev).requires_grad_()
    return {
        "norm": lambda: llsa_amd.layer_norm(r(2, T, 24), r(24), r(24), scale=r(2, 24), shift=r(2, 24)),
        "norm plain": lambda: llsa_amd.layer_norm(r(2, T, 24)),
        "norm fp32 vectors": lambda: llsa_amd.layer_norm(r(2, T, 24), r(24, dtype=torch.float32), r(24)),
        "linear plain": lambda: llsa_amd.linear(r(2, T, 24), r(40, 24)),
        "linear odd": lambda: llsa_amd.linear(r(2, T, 23), r(39, 23), r(39)),
        "linear gated": lambda: llsa_amd.linear(r(2, T, 24), r(40, 24), r(40), gate=r(2, 40), residual=r(2, T, 40)),
        "linear activated": lambda: llsa_amd.linear(r(2, T, 24), r(40, 24), r(40), activation="silu", gate=r(2, 40)),
        "ffn": lambda: llsa_amd.feed_forward(r(2, T, 24), r(16, 24), r(16), r(24, 16), r(24), gate=r(2, 24), residual=r(2, T, 24)),
        "ffn odd": lambda: llsa_amd.feed_forward(r(2, T, 23), r(15, 23), None, r(23, 15)),
    }


CHANGES = {
    "other type": lambda t: t.double() if t.dtype == torch.float32 else t.float(),
    "same size, other type": lambda t: t.view(torch.int32 if t.dtype == torch.float32 else torch.float16),
    "part": lambda t: t[:1] if t.shape[0] > 1 else t[..., :1],
    "part of the last dimension": lambda t: t[..., :-1],
    "other shape": lambda t: t.reshape(-1) if t.dim() > 1 else t[None],
    "other device": lambda t: t.to("meta") if t.device.type == "cpu" else t.cpu(),
    "sparse": lambda t: t.to_sparse(),
}


@pytest.mark.parametrize("T", [9, 50])
@pytest.mark.parametrize("name", list(_calls(torch.device("cpu"), 9)))
def test_changed_saved_tensors_are_refused(dev, name, T):
    """Each saved tensor by itself, each way to change it."""
    seen = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: seen.append(t) or t, lambda t: t):
        y = _calls(dev, T)[name]()
    y.sum().backward()                                        # (the hooks alone change nothing)
    assert seen
    for i in range(len(seen)):
        for what, change in CHANGES.items():
            count = iter(range(len(seen)))
            with torch.autograd.graph.saved_tensors_hooks(lambda t: (next(count), t), lambda p: change(p[1]) if p[0] == i else p[1]):
                y = _calls(dev, T)[name]()
            # (whole numbers in the place of a leaf, torch itself refuses)
            with pytest.raises(RuntimeError, match="another tensor than it was given|Only Tensors of floating point"):
                y.sum().backward()
                raise AssertionError(f"saved tensor {i} of {tuple(seen[i].shape)}: {what} was taken")
