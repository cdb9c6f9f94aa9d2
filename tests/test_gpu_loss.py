"""Cross entropy of a linear head and its gradients against the formulas in 64 bits.

Tolerances (per element).  A sum of n products in fp32 is within n 2^-23 of the sum
of their sizes (each of n additions off by half a step, or a whole one where the
matrix cores cut bits off): a logit within dz = D 2^-23 sum |h w|.  A softmax
probability is then off by 2 dz + 2^-20 of itself (both exponentials, their
arguments and the sum of V terms, which is within V 2^-24 of itself), a loss by
twice the largest dz and 2^-22 of the sizes it is a difference of.  The arguments of a
probability's exponentials are rounded, 2^-23 of log p in all.  The gradient of a logit
is off by 2^-23 at the target (p - 1) and rounded to bf16, 2^-8 of itself, and so is each
result.  Where the forward makes the gradients (a sum or mean) the exponentials are
rounded to fp16 in between, 2^-11 of themselves and 2^-40 at least (2^-25 of 2^-15 of the
largest probability of 256 classes, 1 at most), and the results are rounded once more when the loss's gradient is not 1."""
import math

import pytest
import torch

from tcfp_amd import loss as L

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
HALF = 2.0**-8


def inputs(dev, tokens, d, vocab, seed=0, ignored=0.0, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(tokens, d, generator=g).to(BF16).to(dev)
    w = (torch.randn(vocab, d, generator=g) * (spread / math.sqrt(d))).to(BF16).to(dev)
    t = torch.randint(0, vocab, (tokens,), generator=g)
    if ignored:
        t[torch.rand(tokens, generator=g) < ignored] = -100
    return h, w, t.to(dev)


class Exact:
    """Losses, gradients and how far each may be off, in 64 bits on the CPU."""

    def __init__(self, h, w, t, grad=None, ignore=-100, made=True):
        h, w, t = h.detach().double().cpu(), w.detach().double().cpu(), t.cpu()
        d, v = h.shape[1], w.shape[0]
        z = h @ w.t()
        dz = d * 2.0**-23 * (h.abs() @ w.abs().t())
        self.kept = t != ignore
        at = t.clamp(min=0)[:, None]
        self.lse = torch.logsumexp(z, 1)
        picked = z.gather(1, at)[:, 0]
        self.losses = (self.lse - picked) * self.kept
        top = dz.amax(1)
        self.lse_tol = top + 2.0**-21 + v * 2.0**-24 + 2.0**-22 * self.lse.abs()
        self.losses_tol = self.lse_tol + top + 2.0**-22 * (self.lse.abs() + picked.abs())
        if grad is None:
            return
        grad = grad.double().cpu() * self.kept
        p = torch.exp(z - self.lse[:, None])
        g = p.clone()
        g.scatter_add_(1, at, torch.full_like(picked, -1.0)[:, None])
        g *= grad[:, None]
        eps = (dz + self.lse_tol[:, None] + 2.0**-20 + 2.0**-23 * (z - self.lse[:, None]).abs() +
               (2.0**-11 if made else 0.0))
        off = eps * p + (2.0**-40 if made else 0.0)
        off.scatter_add_(1, at, torch.full_like(picked, 2.0**-23)[:, None])
        g_tol = HALF * g.abs() + (1 + HALF) * off * grad.abs()[:, None]
        self.dh = g @ w
        self.dw = g.t() @ h
        n = h.shape[0]
        out = 2 * HALF + HALF * HALF if made else HALF
        self.dh_tol = out * self.dh.abs() + (1 + out) * (g_tol + v * 2.0**-23 * g.abs()) @ w.abs()
        self.dw_tol = out * self.dw.abs() + (1 + out) * (g_tol + n * 2.0**-23 * g.abs()).t() @ h.abs()


def within(got, want, tol, what):
    err = (got.detach().double().cpu() - want).abs()
    assert got.shape == want.shape
    assert (err <= tol).all(), (what, float((err / tol.clamp(min=1e-300)).max()))


SHAPES = [(1, 8, 1), (1, 64, 5), (3, 72, 100), (64, 256, 256), (65, 128, 257), (130, 264, 1001),
          (300, 64, 129), (17, 1000, 4100), (512, 512, 2048), (1100, 88, 130), (5, 40, 33000)]


@pytest.mark.parametrize("tokens,d,vocab", SHAPES)
def test_losses(dev, tokens, d, vocab):
    print(f"[loss] forward {tokens} {d} {vocab}", flush=True)
    h, w, t = inputs(dev, tokens, d, vocab, ignored=0.2 if tokens > 3 else 0.0)
    e = Exact(h, w, t)
    losses, lse = L.linear_cross_entropy_forward(h, w, t)
    assert losses.dtype == lse.dtype == torch.float32
    within(losses, e.losses, e.losses_tol, "losses")
    within(lse, e.lse, e.lse_tol, "lse")
    assert torch.equal(L.linear_cross_entropy(h, w, t, reduction="none"), losses)
    total = L.linear_cross_entropy(h, w, t, reduction="sum")
    mean = L.linear_cross_entropy(h, w, t)
    s = float(e.losses.sum())
    room = float(e.losses_tol.sum()) + 2.0**-24 * abs(s)
    assert abs(float(total) - s) <= room
    count = int(e.kept.sum())
    assert abs(float(mean) - s / count) <= room / count


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("tokens,d,vocab", SHAPES)
def test_gradients(dev, tokens, d, vocab, reduction):
    print(f"[loss] backward {tokens} {d} {vocab} {reduction}", flush=True)
    h, w, t = inputs(dev, tokens, d, vocab, seed=1, ignored=0.2 if tokens > 3 else 0.0)
    h.requires_grad_()
    w.requires_grad_()
    out = L.linear_cross_entropy(h, w, t, reduction=reduction)
    if reduction == "none":
        up = torch.randn(tokens, generator=torch.Generator().manual_seed(2)).to(dev)
    else:
        up = torch.tensor(1.75, device=dev)
    dh, dw = torch.autograd.grad(out, (h, w), up)
    each = up.double().cpu().expand(tokens)
    if reduction == "mean":
        each = each / int((t != -100).sum())
    e = Exact(h, w, t, each, made=reduction != "none")
    assert dh.dtype == dw.dtype == BF16
    within(dh, e.dh, e.dh_tol, "dh")
    within(dw, e.dw, e.dw_tol, "dw")
    assert not dh[(t == -100)].any()


def check_on_gpu(h, w, t, reduction):
    """Losses and gradients of larger sizes, held against 64 bits on the GPU by the same
    tolerances (a logit's with one bound for all)."""
    dev, (tokens, d), vocab = h.device, h.shape, w.shape[0]
    h.requires_grad_()
    w.requires_grad_()
    out = L.linear_cross_entropy(h, w, t, reduction=reduction)
    up = torch.ones_like(out)
    if reduction == "none":
        up = torch.randn(tokens, generator=torch.Generator().manual_seed(5)).to(dev)
    dh, dw = torch.autograd.grad(out, (h, w), up)
    hd, wd = h.detach().double(), w.detach().double()
    kept = t != -100
    z = torch.mm(hd, wd.t().contiguous())
    dz = d * 2.0**-23 * float(torch.mm(hd.abs(), wd.abs().t().contiguous()).max())
    lse = torch.logsumexp(z, 1)
    rows = torch.arange(tokens, device=dev)
    at = t.clamp(min=0)
    losses = (lse - z[rows, at]) * kept
    each = 2 * dz + 2.0**-21 + vocab * 2.0**-24 + 2.0**-21 * float(z.abs().max())
    if reduction == "none":
        assert ((out.detach().double() - losses).abs() <= each).all()
    else:
        n = int(kept.sum()) if reduction == "mean" else 1
        assert abs(float(out.detach()) - float(losses.sum()) / n) <= each * tokens / n + 1e-6 * float(losses.sum()) / n
    scale = up.double().expand(tokens) * kept
    if reduction == "mean":
        scale = scale / kept.sum()
    p = torch.exp(z - lse[:, None])
    del z
    eps = 2 * dz + vocab * 2.0**-24 + 2.0**-20 + 2.0**-21 * float(lse.abs().max())
    made = reduction != "none"
    off = eps + (2.0**-11 if made else 0.0)
    tol = (off * p + 2.0**-23 + (2.0**-25 if made else 0.0)) * (1 + HALF)
    p[rows, at] -= 1.0
    tol = (tol + HALF * p.abs()) * scale.abs()[:, None]
    p *= scale[:, None]
    for got, want, room in (
            (dh, torch.mm(p, wd), torch.mm(tol + vocab * 2.0**-23 * p.abs(), wd.abs())),
            (dw, torch.mm(p.t().contiguous(), hd),
             torch.mm((tol + tokens * 2.0**-23 * p.abs()).t().contiguous(), hd.abs()))):
        err = (got.double() - want).abs()
        room = HALF * want.abs() + (1 + HALF) * room
        assert (err <= room).all(), float((err / room.clamp(min=1e-300)).max())
    assert not dh[~kept].any()


@pytest.mark.parametrize("reduction", ["sum", "none"])
def test_runs_of_classes_add_up(dev, reduction):
    """More tokens x classes than a run's workspace: 70000 x 4100 x 2 bytes in three
    runs where every token's loss has a gradient; the sum's gradients come with the
    forward."""
    tokens, d, vocab = 70000, 16, 4100
    nb = L._hip.lib().tcfp_linear_cross_entropy_backward_workspace_bytes(tokens, vocab, d, 1, 1)
    assert nb < 2 * tokens * vocab  # g as a whole would take more
    check_on_gpu(*inputs(dev, tokens, d, vocab, seed=3), reduction)


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("tokens,d,vocab", [
    # enough tiles of 256 for every product, ragged; dh's; dW's, its contraction split;
    # runs whose dh is added up in tiles of 256; few tokens on many classes
    (2045, 2040, 8191), (4090, 4096, 500), (16384, 2048, 2040), (16384, 1024, 8448),
    (60, 1032, 20000)])
def test_large_tiles(dev, tokens, d, vocab, reduction):
    print(f"[loss] large {tokens} {d} {vocab} {reduction}", flush=True)
    check_on_gpu(*inputs(dev, tokens, d, vocab, seed=14, ignored=0.05), reduction)


def test_the_largest_workspace(dev):
    """1 GiB of exponentials and no more: beyond, and for more classes than a
    descriptor reaches, the logits are formed twice."""
    size = L._hip.lib().tcfp_linear_cross_entropy_train_workspace_bytes
    assert size(16320, 32768, 64, 1, 1) < 1 << 31 and size(16385, 32768, 64, 1, 1) == 0
    assert size(4, 1 << 20, 64, 1, 1) > 0 and size(4, (1 << 20) + 1, 64, 1, 1) == 0
    assert size(16320, 32768, 64, 1, 1) > 0 and size(524281, 8, 64, 1, 1) == 0
    assert size(524280, 256, 64, 1, 1) > 0
    h, w, t = inputs(dev, 3, 8, (1 << 20) + 3, seed=12, spread=8.0)
    t[1] = (1 << 20) + 2
    h.requires_grad_()
    w.requires_grad_()
    dh, dw = torch.autograd.grad(L.linear_cross_entropy(h, w, t, reduction="sum"), (h, w))
    e = Exact(h, w, t, torch.ones(3), made=False)
    within(dh, e.dh, e.dh_tol, "dh")
    within(dw, e.dw, e.dw_tol, "dw")


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_a_second_backward(dev, reduction):
    """Of a kept graph: the first one is handed what the forward made, the second forms
    the logits again."""
    h, w, t = inputs(dev, 90, 64, 700, seed=13, ignored=0.2)
    h.requires_grad_()
    w.requires_grad_()
    out = L.linear_cross_entropy(h, w, t, reduction=reduction)
    up = torch.full_like(out, 0.3)
    e = Exact(h, w, t, (up if reduction == "none" else up / int((t != -100).sum())).expand(90))
    for _ in range(3):
        dh, dw = torch.autograd.grad(out, (h, w), up, retain_graph=True)
        within(dh, e.dh, e.dh_tol, "dh")
        within(dw, e.dw, e.dw_tol, "dw")


@pytest.mark.parametrize("which", ["hidden", "weight"])
def test_one_gradient_alone(dev, which):
    h, w, t = inputs(dev, 70, 64, 300, seed=4)
    h.requires_grad_(which == "hidden")
    w.requires_grad_(which == "weight")
    L.linear_cross_entropy(h, w, t).backward()
    a, b = h.detach().clone().requires_grad_(), w.detach().clone().requires_grad_()
    both = torch.autograd.grad(L.linear_cross_entropy(a, b, t), (a, b))
    if which == "hidden":
        assert torch.equal(h.grad, both[0]) and w.grad is None
    else:
        assert torch.equal(w.grad, both[1]) and h.grad is None
    # the same without autograd
    lse = L.linear_cross_entropy_forward(h, w, t)[1]
    e = Exact(h, w, t, torch.full((70,), 1 / 70), made=False)
    dh, dw = L.linear_cross_entropy_backward(
        torch.tensor(1.0, device=dev), h.detach(), w.detach(), t, lse,
        count=torch.tensor(70.0, device=dev), need_hidden_grad=which == "hidden",
        need_weight_grad=which == "weight")
    if which == "hidden":
        within(dh, e.dh, e.dh_tol, "dh")
        assert dw is None
    else:
        within(dw, e.dw, e.dw_tol, "dw")
        assert dh is None


def test_gradient_against_differences(dev):
    """Along directions on which h +- e d and w +- e d are exact in bf16: what the
    difference differs from the 64-bit gradient by (its third order) is known, the
    rest are the losses' and the gradients' tolerances."""
    g = torch.Generator().manual_seed(5)
    tokens, d, vocab, e = 20, 32, 40, 1 / 16
    h = (torch.randint(-16, 17, (tokens, d), generator=g) / 16).to(BF16).to(dev)
    w = (torch.randint(-8, 9, (vocab, d), generator=g) / 16).to(BF16).to(dev)
    t = torch.randint(0, vocab, (tokens,), generator=g).to(dev)
    for leaf in ("h", "w"):
        x = h if leaf == "h" else w
        move = (torch.randint(-1, 2, x.shape, generator=g) * e).to(BF16).to(dev)
        pairs = [(h + s * move, w) if leaf == "h" else (h, w + s * move) for s in (1, -1)]
        exact = [Exact(*p, t) for p in pairs]
        slope = sum(s * L.linear_cross_entropy(*p, t, reduction="sum").double().cpu()
                    for s, p in zip((1, -1), pairs)) / 2
        want = sum(s * x.losses.sum() for s, x in zip((1, -1), exact)) / 2
        room = sum(float(x.losses_tol.sum()) + 2.0**-24 * float(x.losses.sum()) for x in exact)
        assert abs(float(slope - want)) <= room
        a, b = h.clone().requires_grad_(), w.clone().requires_grad_()
        grads = torch.autograd.grad(L.linear_cross_entropy(a, b, t, reduction="sum"), (a, b))
        ref = Exact(h, w, t, torch.ones(tokens))
        got, right, tol = ((grads[0], ref.dh, ref.dh_tol) if leaf == "h"
                           else (grads[1], ref.dw, ref.dw_tol))
        step = move.double().cpu()
        third = abs(float((right * step).sum() - want))
        assert abs(float((got.double().cpu() * step).sum() - slope)) <= (
            third + room + float((tol * step.abs()).sum()))


def test_strides_and_leading_axes(dev):
    h, w, t = inputs(dev, 24, 64, 50, seed=6)
    want = L.linear_cross_entropy(h, w, t, reduction="none")
    wide = torch.zeros(24, 96, dtype=BF16, device=dev)
    wide[:, 16:80] = h
    tall = torch.zeros(50, 80, dtype=BF16, device=dev)
    tall[:, 8:72] = w
    assert torch.equal(L.linear_cross_entropy(wide[:, 16:80], tall[:, 8:72], t, reduction="none"), want)
    assert torch.equal(L.linear_cross_entropy(wide[:, 16:80].clone()[:, :], tall[:, 8:72], t,
                                              reduction="none"), want)
    odd = torch.zeros(24 * 64 + 1, dtype=BF16, device=dev)[1:].view(24, 64)
    odd.copy_(h)
    assert torch.equal(L.linear_cross_entropy(odd, w.t().contiguous().t(), t, reduction="none"), want)
    three = L.linear_cross_entropy(h.view(2, 12, 64), w, t.view(2, 12), reduction="none")
    assert torch.equal(three, want.view(2, 12))
    a = h.view(2, 12, 64).clone().requires_grad_()
    (grad,) = torch.autograd.grad(L.linear_cross_entropy(a, w, t.view(2, 12)), a)
    b = h.clone().requires_grad_()
    (flat,) = torch.autograd.grad(L.linear_cross_entropy(b, w, t), b)
    assert torch.equal(grad.view(24, 64), flat)
    one = L.linear_cross_entropy(h[0], w, t[0], reduction="none")
    assert one.shape == () and torch.equal(one, want[0])


def test_targets_left_out_and_outside(dev):
    h, w, t = inputs(dev, 12, 64, 50, seed=7)
    t[:] = -100
    assert math.isnan(float(L.linear_cross_entropy(h, w, t)))
    assert float(L.linear_cross_entropy(h, w, t, reduction="sum")) == 0.0
    hg, wg = h.clone().requires_grad_(), w.clone().requires_grad_()
    for reduction in ("sum", "mean", "none"):
        out = L.linear_cross_entropy(hg, wg, t, reduction=reduction)
        dh, dw = torch.autograd.grad(out, (hg, wg), torch.ones_like(out))
        assert not dh.any() and not dw.any()
    t = torch.arange(12, device=dev)
    t[3], t[5] = 50, -7
    losses = L.linear_cross_entropy(h, w, t, reduction="none")
    bad = torch.zeros(12, dtype=torch.bool)
    bad[[3, 5]] = True
    assert torch.equal(torch.isnan(losses).cpu(), bad)
    (dh,) = torch.autograd.grad(L.linear_cross_entropy(hg, w, t, reduction="sum"), hg)
    assert torch.equal(torch.isnan(dh).any(1).cpu(), bad)
    # another index to leave out, one of the classes
    t = torch.arange(12, device=dev) % 3
    losses = L.linear_cross_entropy(h, w, t, ignore_index=1, reduction="none")
    assert torch.equal(losses == 0, t == 1)


def test_what_is_not_finite(dev):
    h, w, t = inputs(dev, 40, 64, 300, seed=8)
    h = h.clone()
    h[7, 3] = math.nan
    h[9] = 1e38  # logits of both signs past fp32
    losses = L.linear_cross_entropy(h, w, t, reduction="none")
    bad = torch.zeros(40, dtype=torch.bool)
    bad[[7, 9]] = True
    assert torch.equal(~torch.isfinite(losses).cpu(), bad)
    # what a token that is left out holds reaches no other token's loss or gradient
    t2 = t.clone()
    t2[[7, 9]] = -100
    hg = h.clone().requires_grad_()
    loss = L.linear_cross_entropy(hg, w, t2)
    assert math.isfinite(float(loss.detach()))
    (dh,) = torch.autograd.grad(loss, hg)
    assert torch.isfinite(dh).all() and not dh[[7, 9]].any()


def test_large_logits(dev):
    """Logits of some +-2000: exponentials only of differences."""
    h, w, t = inputs(dev, 33, 64, 500, seed=9, spread=500.0)
    e = Exact(h, w, t, torch.ones(33))
    within(L.linear_cross_entropy(h, w, t, reduction="none"), e.losses, e.losses_tol, "losses")


@pytest.mark.parametrize("how", ["mean", "sum", "again", "each"])
@pytest.mark.parametrize("tokens,d,vocab", [(255, 64, 3000), (255, 1024, 300)])
def test_tokens_do_not_share_a_rounding(dev, tokens, d, vocab, how):
    """1 / 255 lies half a step of bf16 from the nearest value: a factor that is rounded
    with every target's gradient would be 2^-8 off for all of them.  The results' own
    rounding is 2^-8 / sqrt(12) to 2^-8 / sqrt(3) of them, 1.7e-3 for even mantissas, and
    the other factors' average out; the target's probability less 1 is off by 2^-9 at most."""
    h, w, t = inputs(dev, tokens, d, vocab, seed=19)
    hg, wg = h.clone().requires_grad_(), w.clone().requires_grad_()
    factor = torch.full((), 1 / 255, device=dev)
    if how in ("mean", "again"):
        out = L.linear_cross_entropy(hg, wg, t)
        if how == "again":
            torch.autograd.grad(out, (hg, wg), retain_graph=True)
        got = torch.autograd.grad(out, (hg, wg))
    elif how == "sum":
        out = L.linear_cross_entropy(hg, wg, t, reduction="sum")
        torch.autograd.grad(out, (hg, wg), retain_graph=True)
        got = torch.autograd.grad(out, (hg, wg), factor)
    else:
        out = L.linear_cross_entropy(hg, wg, t, reduction="none")
        got = torch.autograd.grad(out, (hg, wg), factor.expand(tokens))
    e = Exact(h, w, t, torch.full((tokens,), 1 / 255))
    for x, want in zip(got, (e.dh, e.dw)):
        off = (x.double().cpu() - want).norm() / want.norm()
        assert off <= 2.6e-3, float(off)


@pytest.mark.parametrize("reduction", ["sum", "none"])
@pytest.mark.parametrize("tokens", [40, 600])
def test_rare_classes_keep_their_gradients(dev, tokens, reduction):
    """Classes that are 2^-15 to 2^-26 as likely as the likeliest of their tile."""
    h, w, t = inputs(dev, tokens, 64, 702, seed=17, spread=0.5)
    h[:, 0] = 1.0
    w[:, 0] = 0.0
    w[::3, 0] = -14.0
    t = t // 3 * 3 + 1  # (none of them a target)
    hg, wg = h.clone().requires_grad_(), w.clone().requires_grad_()
    out = L.linear_cross_entropy(hg, wg, t, reduction=reduction)
    dh, dw = torch.autograd.grad(out, (hg, wg), torch.ones_like(out))
    e = Exact(h, w, t, torch.ones(tokens), made=reduction == "sum")
    within(dh, e.dh, e.dh_tol, "dh")
    within(dw, e.dw, e.dw_tol, "dw")
    # (of these inputs, on the CPU: what may be off is far below what is there)
    assert e.dw[::3].norm() > 16 * e.dw_tol[::3].norm()


def test_no_tokens(dev):
    h = torch.zeros(0, 64, dtype=BF16, device=dev).requires_grad_()
    w = torch.ones(50, 64, dtype=BF16, device=dev).requires_grad_()
    t = torch.zeros(0, dtype=torch.int64, device=dev)
    assert L.linear_cross_entropy(h, w, t, reduction="none").shape == (0,)
    loss = L.linear_cross_entropy(h, w, t, reduction="sum")
    assert float(loss.detach()) == 0.0
    dh, dw = torch.autograd.grad(loss, (h, w))
    assert dh.shape == (0, 64) and not dw.any()
    assert math.isnan(float(L.linear_cross_entropy(h, w, t)))


def test_bits_repeat_and_streams(dev):
    h, w, t = inputs(dev, 700, 264, 1500, seed=10, ignored=0.1)
    h.requires_grad_()
    w.requires_grad_()

    def once():
        loss = L.linear_cross_entropy(h, w, t)
        return (loss.detach(), *torch.autograd.grad(loss, (h, w)))

    want = once()
    assert all(torch.equal(a, b) for a, b in zip(once(), want))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = once()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_graph(dev):
    h, w, t = inputs(dev, 300, 128, 600, seed=11)
    x = h.clone()
    _, lse0 = L.linear_cross_entropy_forward(x, w, t)
    one = torch.tensor(1.0, device=dev)

    def both():
        losses, lse = L.linear_cross_entropy_forward(x, w, t)
        return (losses, *L.linear_cross_entropy_backward(one, x, w, t, lse))

    both()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for i in range(3):
        x.copy_(h * (i + 1))
        eager = both()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager))


def test_graph_of_a_training_forward(dev):
    """The forward that makes gradients, captured and replayed; both ways of taking the
    mean (up to 1024 tokens and more)."""
    for tokens in (300, 1500):
        h, w, t = inputs(dev, tokens, 128, 600, seed=15, ignored=0.1)
        x = h.clone()
        leaf = x.detach().requires_grad_()  # (shares x's memory)
        L.linear_cross_entropy(leaf, w, t)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = L.linear_cross_entropy(leaf, w, t).detach()
        for i in range(3):
            x.copy_(h * (i + 1))
            eager = L.linear_cross_entropy(x, w, t)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, eager)


def test_graph_of_a_backward_alone(dev):
    """Replays give the gradients again, each time."""
    h, w, t = inputs(dev, 60, 64, 300, seed=18)
    by = torch.full((), 0.3, device=dev)
    leaves = h.clone().requires_grad_(), w.clone().requires_grad_()
    want = torch.autograd.grad(L.linear_cross_entropy(*leaves, t), leaves, by)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # (leaves of its own, first used on its stream)
        own = h.clone().requires_grad_(), w.clone().requires_grad_()
        loss = L.linear_cross_entropy(*own, t)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = torch.autograd.grad(loss, own, by, retain_graph=True)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(rel_equal(x, y) for x, y in zip(got, want))


def test_in_place_on_the_loss(dev):
    h, w, t = inputs(dev, 9, 64, 50, seed=16)
    h.requires_grad_()
    loss = L.linear_cross_entropy(h, w, t)
    (want,) = torch.autograd.grad(loss, h, retain_graph=True)
    loss /= 4  # (a power of two: nothing is rounded)
    loss.backward()
    assert rel_equal(h.grad, want / 4)


def rel_equal(a, b):
    """Equal but for bf16 roundings of what was formed twice (see the module's head)."""
    a, b = a.double(), b.double()
    return bool(((a - b).norm() <= 3 * HALF * b.norm()).item())


def test_refusals(dev):
    h, w, t = inputs(dev, 4, 64, 10)
    for exc, args in [
            (TypeError, (h.float(), w, t)), (TypeError, (h, w.float(), t)),
            (TypeError, (h, w, t.int())), (ValueError, (h, w[:, :32], t)),
            (ValueError, (h, w[0], t)), (ValueError, (h, w, t[:3])), (ValueError, (h, w[:0], t)),
            (ValueError, (h[:, :60].contiguous(), w[:, :60].contiguous(), t)),
            (RuntimeError, (h.cpu(), w, t)), (RuntimeError, (h, w, t.cpu()))]:
        with pytest.raises(exc):
            L.linear_cross_entropy(*args)
    with pytest.raises(ValueError):
        L.linear_cross_entropy(h, w, t, reduction="max")
    lse = torch.zeros(4, device=dev)
    g = torch.ones(4, device=dev)
    for args in [(g[:3], h, w, t, lse), (g.double(), h, w, t, lse), (g, h, w, t, lse[:3])]:
        with pytest.raises(ValueError):
            L.linear_cross_entropy_backward(*args)
    a = h.clone().requires_grad_()
    (grad,) = torch.autograd.grad(L.linear_cross_entropy(a, w, t), a, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()
