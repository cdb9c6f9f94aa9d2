"""Cross entropy of a linear head: gradients of tokens that are left out."""
import pytest
import torch

from tcfp_amd import loss as L
from test_gpu_loss import Exact, inputs, within

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.mark.parametrize("huge", [1e38, 3e38])
def test_a_gradient_of_a_token_left_out(dev, huge):
    """Whatever it is, it does not count: the others' gradients keep their bits."""
    h, w, t = inputs(dev, 90, 64, 300, seed=21, ignored=0.3)
    up = torch.randn(90, generator=torch.Generator().manual_seed(22)).to(dev) * 1e-3
    up[t == -100] = huge
    hg, wg = h.clone().requires_grad_(), w.clone().requires_grad_()
    dh, dw = torch.autograd.grad(L.linear_cross_entropy(hg, wg, t, reduction="none"), (hg, wg), up)
    e = Exact(h, w, t, up, made=False)
    within(dh, e.dh, e.dh_tol, "dh")
    within(dw, e.dw, e.dw_tol, "dw")
