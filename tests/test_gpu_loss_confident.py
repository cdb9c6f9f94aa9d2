"""Cross entropy where a token's class is almost certain, at logits of any size.

Every hidden state is a unit vector, so that a logit is one value of the weight: what
is compared here starts from the same logits on both sides.  Besides its target's
class a token has one rival at `gap` below the largest, and all others so far below
that their exponentials are 0.

Tolerances.  The sum of exponentials relative to the largest is 1 + e^-gap, rounded to
fp32, 2^-24 for each of its two terms; its logarithm and the largest logit's distance
from the target's (0, or gap) are off by a few roundings of themselves: a loss within
2^-22 + 2^-20 of itself, never below 0.  The gradient of the target's logit is
exp(-loss) - 1, off by what the loss is off by, 2^-22 and 2^-20 of itself, and rounded to bf16, 2^-8 of
itself.  The rival's probability is formed from lse, which is rounded to fp32, 2^-24 of it,
and takes a few roundings more of arguments of that size (2^-21 in all, and 2^-20), fp16 in
between (2^-11, and 2^-25 of 2^-15 at least), and bf16.  Results are rounded once
more, and once again if the loss's gradient is no power of two; here it is 1."""
import math

import pytest
import torch

from tcfp_amd import loss as L

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
HALF = 2.0**-8
KINDS = 16  # of tokens

# largest logit, and how far below it the rival is: both as bf16 has them
TOPS = (8.0, 30.0, 100.0, 2000.0)
GAPS = {8.0: (4.0, 6.0, 8.0, 12.0), 30.0: (8.0, 12.0, 16.0, 20.0), 100.0: (8.0, 10.0, 12.0, 16.0),
        2000.0: (8.0, 16.0, 24.0, 32.0)}


class Case:
    """`copies` tokens of each kind; token t has the unit vector t % KINDS."""

    def __init__(self, dev, copies, d, vocab, rival_is_target=False):
        g = torch.Generator().manual_seed(vocab)
        pairs = [(top, gap) for top in TOPS for gap in GAPS[top]]
        assert len(pairs) == KINDS
        w = torch.zeros(vocab, d, dtype=torch.float64)
        first, second = [], []
        for i, (top, gap) in enumerate(pairs):
            a, b = torch.randperm(vocab, generator=g)[:2].tolist()
            w[:, i] = top - 304.0 if top < 1000 else -top
            w[a, i], w[b, i] = top, top - gap
            first.append(a), second.append(b)
        self.w = w.to(BF16)
        assert torch.equal(self.w.double()[first, range(KINDS)], w[first, range(KINDS)])
        assert torch.equal(self.w.double()[second, range(KINDS)], w[second, range(KINDS)])
        assert float((self.w.double()[:, :KINDS].sort(0).values[-3] - w.amax(0)[:KINDS]).max()) < -250
        n = copies * KINDS
        kind = torch.arange(n) % KINDS
        h = torch.zeros(n, d, dtype=BF16)
        h[range(n), kind] = 1.0
        target = torch.tensor(second if rival_is_target else first)
        other = torch.tensor(first if rival_is_target else second)
        gap = torch.tensor([p[1] for p in pairs], dtype=torch.float64)
        top = torch.tensor([p[0] for p in pairs], dtype=torch.float64)
        self.copies, self.kind, self.target, self.other = copies, kind, target, other
        rare = torch.log1p(torch.exp(-gap))
        self.loss = rare + (gap if rival_is_target else 0.0)  # of a kind
        self.loss_tol = 2.0**-22 + 2.0**-20 * self.loss
        self.at_target = torch.expm1(-self.loss)
        self.at_other = -self.at_target
        self.lse = top + rare
        self.h, self.w, self.t = h.to(dev), self.w.to(dev), target[kind].to(dev)

    def check_losses(self, losses):
        x = losses.detach().double().cpu()
        assert (x >= 0).all()
        err = (x - self.loss[self.kind]).abs() / self.loss_tol[self.kind]
        assert (err <= 1).all(), (float(err.max()), self.kind[err.argmax()])

    def check_grads(self, dh, dw, made, each=None, what=""):
        """dw has the logits' gradients themselves, `copies` equal ones in a sum."""
        dw = dw.detach().double().cpu()
        each = torch.ones(KINDS, dtype=torch.float64) if each is None else each
        i = torch.arange(KINDS)
        out = HALF + 2.0**-20  # (the sum of equal values: rounded fp32 additions)
        for at, want, off in (
                (self.target, self.at_target, 2.0**-22 + 2.0**-20 * self.at_target.abs()),
                (self.other, self.at_other,
                 (2.0**-20 + 2.0**-21 * self.lse + (2.0**-11 if made else 0.0)) * self.at_other +
                 (2.0**-40 if made else 0.0))):
            tol = (HALF * want.abs() + (1 + HALF) * off)
            tol = (out * want.abs() + (1 + out) * tol) * each.abs() * self.copies
            want = want * each * self.copies
            err = (dw[at, i] - want).abs() / tol
            assert (err <= 1).all(), (what, float(err.max()), int(err.argmax()))
            # dh = g W: of the token's own column the target's value times its g, and
            # the other's
        got = dh.detach().double().cpu()
        w = self.w.double().cpu()
        a, b = w[self.target, i], w[self.other, i]
        want = (self.at_target * a + self.at_other * b) * each
        off = 2.0**-22 + (2.0**-20 + HALF) * self.at_target.abs()
        off = off * a.abs() + ((2.0**-20 + 2.0**-21 * self.lse + 2.0**-11 + HALF) * self.at_other +
                               2.0**-40) * b.abs()
        tol = (HALF * want.abs() + (1 + HALF) * 1.01 * off * each.abs())
        err = (got[range(len(self.kind)), self.kind] - want[self.kind]).abs() / tol[self.kind]
        assert (err <= 1).all(), (what, float(err.max()), int(self.kind[err.argmax()]))


# (tiles of 128 and of 256, one and many of them along the classes)
SHAPES = [(1, 16, 40), (1, 64, 300), (4, 64, 5000), (128, 1024, 8192)]


@pytest.mark.parametrize("rival", [False, True])
@pytest.mark.parametrize("copies,d,vocab", SHAPES)
def test_losses(dev, copies, d, vocab, rival):
    print(f"[confident] losses {copies} {d} {vocab}", flush=True)
    c = Case(dev, copies, d, vocab, rival)
    losses, _ = L.linear_cross_entropy_forward(c.h, c.w, c.t)
    c.check_losses(losses)
    assert torch.equal(L.linear_cross_entropy(c.h, c.w, c.t, reduction="none"), losses)
    want, room = (float(x.sum()) * copies for x in (c.loss, c.loss_tol))
    total = L.linear_cross_entropy(c.h, c.w, c.t, reduction="sum")
    assert abs(float(total) - want) <= room + 2.0**-24 * want


@pytest.mark.parametrize("how", ["sum", "again", "each", "apart"])
@pytest.mark.parametrize("rival", [False, True])
@pytest.mark.parametrize("copies,d,vocab", SHAPES)
def test_gradients(dev, copies, d, vocab, rival, how):
    print(f"[confident] gradients {copies} {d} {vocab} {how}", flush=True)
    c = Case(dev, copies, d, vocab, rival)
    h, w = c.h.clone().requires_grad_(), c.w.clone().requires_grad_()
    each = None
    if how in ("sum", "again"):
        out = L.linear_cross_entropy(h, w, c.t, reduction="sum")
        if how == "again":
            torch.autograd.grad(out, (h, w), retain_graph=True)
        dh, dw = torch.autograd.grad(out, (h, w))
    elif how == "each":
        out = L.linear_cross_entropy(h, w, c.t, reduction="none")
        each = 2.0 ** (torch.arange(KINDS, dtype=torch.float64) % 3)
        dh, dw = torch.autograd.grad(out, (h, w), each.float()[c.kind].to(dev))
    else:
        losses, lse = L.linear_cross_entropy_forward(c.h, c.w, c.t)
        dh, dw = L.linear_cross_entropy_backward(torch.ones((), device=dev), c.h, c.w, c.t, lse,
                                                 losses=losses)
    c.check_grads(dh, dw, how == "sum", each, (how, copies, vocab))


def test_losses_may_be_changed(dev):
    """Every token's loss is the caller's own, as it was: the backward does not read it."""
    c = Case(dev, 1, 64, 300)
    got = []
    for change in (False, True):
        h = c.h.clone().requires_grad_()
        losses = L.linear_cross_entropy(h, c.w, c.t, reduction="none")
        total = losses.mul_(2.0).sum() if change else (losses * 2.0).sum()
        got.append(torch.autograd.grad(total, h)[0])
    assert torch.equal(*got)


def test_gradients_at_large_logits(dev):
    """Logits of some +-2000 that are sums of products, in both ways of making gradients
    (tolerances: the loss's own tests, and exponentials below 2^-126, which fp32 has not:
    so much a token of each logit's gradient)."""
    from test_gpu_loss import Exact, inputs, within

    h, w, t = inputs(dev, 33, 64, 500, seed=9, spread=500.0)
    for reduction in ("sum", "none"):
        hg, wg = h.clone().requires_grad_(), w.clone().requires_grad_()
        out = L.linear_cross_entropy(hg, wg, t, reduction=reduction)
        dh, dw = torch.autograd.grad(out, (hg, wg), torch.ones_like(out))
        e = Exact(h, w, t, torch.ones(33), made=reduction == "sum")
        within(dh, e.dh, e.dh_tol + 2.0**-126 * float(w.abs().double().sum()), "dh")
        within(dw, e.dw, e.dw_tol + 2.0**-126 * float(h.abs().double().sum()), "dw")
    assert math.isfinite(float(dh.double().norm()))


def test_losses_refused(dev):
    c = Case(dev, 1, 64, 300)
    losses, lse = L.linear_cross_entropy_forward(c.h, c.w, c.t)
    one = torch.ones((), device=dev)
    for exc, bad in ((ValueError, losses[:5]), (ValueError, losses.double()),
                     (RuntimeError, losses.cpu())):
        with pytest.raises(exc):
            L.linear_cross_entropy_backward(one, c.h, c.w, c.t, lse, losses=bad)
