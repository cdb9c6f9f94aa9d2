"""The training operators in calls around them: recomputed forwards, tensors saved
elsewhere, threads, inputs that share memory, losses of every token in a graph."""
import threading

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from tcfp_amd.attention import packed_attention
from tcfp_amd.loss import linear_cross_entropy
from tcfp_amd.rotary import rotary_embedding, rotary_frequencies

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
HEADS, KV, DIM, VOCAB, LENS = 4, 2, 64, 300, (130, 1, 69)
TOKENS = sum(LENS)


class Step:
    def __init__(self, dev, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.x = torch.randn(TOKENS, (HEADS + 2 * KV) * DIM, generator=g).to(BF16).to(dev)
        self.w = (torch.randn(VOCAB, HEADS * DIM, generator=g) / 16).to(BF16).to(dev)
        self.t = torch.randint(0, VOCAB, (TOKENS,), generator=g).to(dev)
        self.t[3] = -100
        self.at = torch.tensor([0, 130, 131, 200], dtype=torch.int32, device=dev)
        self.pos = torch.arange(TOKENS, device=dev)
        self.freqs = rotary_frequencies(DIM, device=dev)

    def attended(self, x):
        q, k, v = x.unflatten(1, (-1, DIM)).split((HEADS, KV, KV), 1)
        q, k = rotary_embedding(q, k, self.pos, self.freqs)
        return packed_attention(q, k, v, self.at, max_len=TOKENS).flatten(1)

    def loss(self, x, w, reduction="mean"):
        return linear_cross_entropy(self.attended(x), w, self.t, reduction=reduction)

    def run(self, loss=None, reduction="mean"):
        x, w = self.x.clone().requires_grad_(), self.w.clone().requires_grad_()
        out = (loss or self.loss)(x, w, reduction)
        return (out.detach(), *torch.autograd.grad(out, (x, w), torch.full_like(out, 0.5)))


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("reentrant", [False, True])
def test_recomputed(dev, reentrant, reduction):
    s = Step(dev)
    want = s.run(reduction=reduction)
    got = s.run(lambda x, w, r: checkpoint(s.loss, x, w, r, use_reentrant=False), reduction)
    assert same(got, want)
    if reentrant:  # (which takes .backward() alone)
        x, w = s.x.clone().requires_grad_(), s.w.clone().requires_grad_()
        out = checkpoint(s.loss, x, w, reduction, use_reentrant=True)
        out.backward(torch.full_like(out, 0.5))
        assert same((out.detach(), x.grad, w.grad), want)


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_saved_on_the_host(dev, reduction):
    s = Step(dev)
    want = s.run(reduction=reduction)
    with torch.autograd.graph.save_on_cpu():
        got = s.run(reduction=reduction)
    assert same(got, want)


def test_threads(dev):
    """Each thread on a stream of its own, with inputs of its own."""
    steps = [Step(dev, seed) for seed in range(4)]
    want = [s.run() for s in steps]
    torch.cuda.synchronize()
    got, errors = [None] * 4, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    got[i] = steps[i].run()
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # (shown by the test itself)
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    assert all(same(a, b) for a, b in zip(got, want))


def test_one_tensor_as_all_three(dev):
    g = torch.Generator().manual_seed(5)
    x0 = torch.randn(40, 2, DIM, generator=g).to(BF16).to(dev)
    at = torch.tensor([0, 15, 40], dtype=torch.int32, device=dev)
    go = torch.randn(40, 2, DIM, generator=g).to(BF16).to(dev)
    apart = [x0.clone().requires_grad_() for _ in range(3)]
    o = packed_attention(*apart, at, max_len=25)
    dq, dk, dv = torch.autograd.grad(o, apart, go)
    x = x0.clone().requires_grad_()
    p = packed_attention(x, x, x, at, max_len=25)
    (dx,) = torch.autograd.grad(p, x, go)
    assert torch.equal(o, p)
    want = dq.double() + dk.double() + dv.double()
    # (two additions in bf16, each rounded)
    room = 2.0**-7 * (dq.double().abs() + dk.double().abs() + dv.double().abs())
    assert ((dx.double() - want).abs() <= room).all()


def test_a_head_that_is_its_own_input(dev):
    """hidden and weight one tensor: the sum of both gradients."""
    w0 = (torch.randn(48, 64, generator=torch.Generator().manual_seed(6)) / 4).to(BF16).to(dev)
    t = torch.arange(48, device=dev)
    a, b = w0.clone().requires_grad_(), w0.clone().requires_grad_()
    da, db = torch.autograd.grad(linear_cross_entropy(a, b, t), (a, b))
    c = w0.clone().requires_grad_()
    (dc,) = torch.autograd.grad(linear_cross_entropy(c, c, t), c)
    room = 2.0**-8 * (da.double().abs() + db.double().abs())
    assert ((dc.double() - da.double() - db.double()).abs() <= room).all()


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_inputs_changed_before_the_backward(dev, reduction):
    """What was saved and then changed is an error of the engine, not another gradient."""
    s = Step(dev)
    for change in ("hidden", "weight", "out"):
        y = s.attended(s.x).clone().requires_grad_()
        w = s.w.clone().requires_grad_()
        if change == "out":
            x = s.x.clone().requires_grad_()
            o = s.attended(x)
            with torch.no_grad():
                o.mul_(2)
            with pytest.raises(RuntimeError, match="inplace"):
                torch.autograd.grad(o, x, torch.ones_like(o))
            continue
        out = linear_cross_entropy(y, w, s.t, reduction=reduction)
        with torch.no_grad():
            (y if change == "hidden" else w).mul_(2)
        with pytest.raises(RuntimeError, match="inplace"):
            torch.autograd.grad(out, (y, w), torch.ones_like(out))


@pytest.mark.parametrize("reduction", ["sum", "none"])
def test_a_captured_step_of_every_token(dev, reduction):
    """Replays are the eager step, also as hidden states, targets and the losses' own
    gradients change."""
    s = Step(dev)
    x0, t0 = s.x.clone(), s.t.clone()
    up = torch.full((TOKENS,) if reduction == "none" else (), 0.75, device=dev)

    def step():
        x, w = s.x.detach().requires_grad_(), s.w.detach().requires_grad_()
        out = s.loss(x, w, reduction)
        return (out.detach(), *torch.autograd.grad(out, (x, w), up))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step()
    for i in range(3):
        s.x.copy_(x0 * (1 + i / 4))
        s.t.copy_((t0 + i).clamp(max=VOCAB - 1).masked_fill(t0 < 0, -100))
        up.mul_(0.5 + i)
        want = step()
        torch.cuda.synchronize()
        for _ in range(2):
            graph.replay()
            torch.cuda.synchronize()
            assert same(got, want)


def test_a_batch_of_gradients_is_refused(dev):
    s = Step(dev)
    x, w = s.x.clone().requires_grad_(), s.w.clone().requires_grad_()
    for out, leaf in ((s.attended(x), x), (s.loss(x, w), w)):
        ups = torch.ones(2, *out.shape, dtype=out.dtype, device=dev)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(out, leaf, ups, is_grads_batched=True)
