"""Cross entropy of a linear head: gradients of tokens that are left out, rows far apart."""
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


def test_rows_far_apart(dev):
    """The last token's hidden state of each long sequence, a weight inside a wide matrix."""
    h, w, t = inputs(dev, 3, 64, 5, seed=23)
    far = torch.zeros(3, (1 << 22) + 8, dtype=BF16, device=dev)[:, 8:72]
    far.copy_(h)
    wide = torch.zeros(5, 1 << 23, dtype=BF16, device=dev)[:, :64]
    wide.copy_(w)
    want = L.linear_cross_entropy(h, w, t, reduction="none")
    a, b = h.clone().requires_grad_(), w.clone().requires_grad_()
    grads = torch.autograd.grad(L.linear_cross_entropy(a, b, t), (a, b))
    for x, y in ((far, w), (h, wide), (far, wide)):
        assert torch.equal(L.linear_cross_entropy(x, y, t, reduction="none"), want)
        x, y = x.detach().requires_grad_(), y.detach().requires_grad_()
        got = torch.autograd.grad(L.linear_cross_entropy(x, y, t), (x, y))
        assert all(torch.equal(p, q) for p, q in zip(got, grads))
