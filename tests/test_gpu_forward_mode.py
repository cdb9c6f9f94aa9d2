"""Forward-mode derivatives: the training operators have none, and say so instead of
returning a result without its tangent."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from tcfp_amd.attention import packed_attention
from tcfp_amd.loss import linear_cross_entropy
from tcfp_amd.rotary import rotary_embedding, rotary_frequencies

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def calls(dev):
    """{operator: (its differentiable inputs, the call)}."""
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(6, h, 64, generator=g).to(BF16).to(dev) for h in (4, 2, 2))
    pos, freqs = torch.arange(6, device=dev), rotary_frequencies(64, device=dev)
    at = torch.tensor([0, 2, 6], dtype=torch.int32, device=dev)
    h, w = (torch.randn(n, 64, generator=g).to(BF16).to(dev) for n in (6, 10))
    t = torch.arange(6, device=dev)
    return {
        "rotary": ((q, k), lambda q, k: rotary_embedding(q, k, pos, freqs)),
        "rotary of q": ((q,), lambda q: rotary_embedding(q, None, pos, freqs)),
        "attention": ((q, k, v), lambda *x: packed_attention(*x, at, max_len=4)),
        "mean": ((h, w), lambda *x: linear_cross_entropy(*x, t)),
        "each": ((h, w), lambda *x: linear_cross_entropy(*x, t, reduction="none")),
    }


@pytest.mark.parametrize("grad_mode", [True, False])
@pytest.mark.parametrize("wants", [True, False])
@pytest.mark.parametrize("name", ["rotary", "rotary of q", "attention", "mean", "each"])
def test_a_tangent_is_refused(dev, name, wants, grad_mode):
    inputs, call = calls(dev)[name]
    for i in range(len(inputs)):
        x = [y.clone().requires_grad_(wants) for y in inputs]
        with torch.set_grad_enabled(grad_mode), fwAD.dual_level():
            x[i] = fwAD.make_dual(x[i], torch.ones_like(x[i]))
            with pytest.raises(RuntimeError):
                call(*x)
        # (and what has none is answered as before, inside a level too)
        with torch.no_grad():
            want = call(*inputs)
            with fwAD.dual_level():
                got = call(*inputs)
        for a, b in zip(*((y if isinstance(y, tuple) else (y,)) for y in (got, want))):
            assert (a is None) == (b is None) and (a is None or torch.equal(a, b))


@pytest.mark.parametrize("name", ["rotary", "attention", "mean", "each"])
def test_transforms_are_refused(dev, name):
    inputs, call = calls(dev)[name]
    with pytest.raises(RuntimeError):
        torch.func.jvp(call, inputs, tuple(torch.ones_like(x) for x in inputs))
