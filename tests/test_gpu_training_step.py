"""The training operators together, as a decoder's step uses them: rotary positions,
attention within packed sequences, cross entropy of the head.

Tolerance of whole steps: on the way from a loss to a gradient a value is rounded to
bf16 at most twelve times (turned q and k, P, the attention's result and hidden states,
g, dh, dS, dq or dk and their turn, the cast in front), each time by 2^-8 of itself at
most, and the norms of what they are multiplied with are the same on both sides: 12 *
2^-8 = 0.047 of a gradient's norm."""
import copy
import importlib.util
from pathlib import Path

import pytest
import torch
import torch.nn.functional as F

from tcfp_amd.attention import PagedKVCache, packed_attention
from tcfp_amd.loss import linear_cross_entropy
from tcfp_amd.rotary import rotary_embedding, rotary_frequencies

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
STEP = 12 * 2.0**-8


def rel(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    return float((a - b).norm() / b.norm())


def plain_rotary(q, k, positions, freqs, interleaved=False):
    angle = positions.double()[:, None, None] * freqs
    c, s = torch.cos(angle), torch.sin(angle)

    def turn(x):
        half = len(freqs)
        a, b = x[..., :half].double(), x[..., half:2 * half].double()
        return torch.cat((a * c - b * s, a * s + b * c, x[..., 2 * half:].double()), -1)

    return turn(q), turn(k)


def plain_attention(q, k, v, starts, max_len=None, window=0):
    group = q.shape[1] // k.shape[1]
    out = []
    starts = starts.tolist()
    for a, b in zip(starts, starts[1:]):
        n = b - a
        Q, K, V = (x[a:b].double().transpose(0, 1) for x in (q, k, v))
        K, V = (x.repeat_interleave(group, 0) for x in (K, V))
        s = torch.matmul(Q, K.transpose(1, 2).contiguous()) / q.shape[2]**0.5
        seen = torch.ones(n, n, dtype=torch.bool, device=q.device).tril()
        if window:
            seen = seen.triu(1 - window)
        out.append(torch.matmul(torch.softmax(s.masked_fill(~seen, float("-inf")), -1), V).transpose(0, 1))
    return torch.cat(out)


def plain_loss(hidden, weight, targets):
    z = hidden.double().flatten(0, -2) @ weight.double().t()
    return F.cross_entropy(z, targets.flatten())


@pytest.mark.parametrize("window", [0, 30])
def test_a_step_of_a_layer_and_its_head(dev, window):
    """Projection -> turn -> attention -> projection -> loss, ragged sequences, a token
    left out, against the same in 64 bits."""
    g = torch.Generator().manual_seed(0)
    lens, d, heads, kv, dim, vocab = [70, 1, 130, 33], 256, 4, 2, 64, 500
    starts = torch.tensor([0, 70, 71, 201, 234], dtype=torch.int32, device=dev)
    tokens = 234
    pos = torch.cat([torch.arange(n) for n in lens]).to(dev)
    freqs = rotary_frequencies(dim, device=dev)
    x = torch.randn(tokens, d, generator=g).to(dev)
    wq = (torch.randn((heads + 2 * kv) * dim, d, generator=g) / d**0.5).to(dev)
    wo = (torch.randn(d, heads * dim, generator=g) / d**0.5).to(dev)
    wv = (torch.randn(vocab, d, generator=g) / d**0.5).to(dev)
    t = torch.randint(0, vocab, (tokens,), generator=g).to(dev)
    t[5] = -100

    def run(dtype, turn, attend, loss):
        leaves = [y.detach().to(dtype).requires_grad_() for y in (x, wq, wo, wv)]
        a, b, c, e = leaves
        qkv = a @ b.t()
        low = qkv.to(BF16) if dtype == torch.float32 else qkv
        q = low[:, :heads * dim].unflatten(1, (heads, dim))
        k = low[:, heads * dim:(heads + kv) * dim].unflatten(1, (kv, dim))
        v = low[:, (heads + kv) * dim:].unflatten(1, (kv, dim))
        q, k = turn(q, k, pos, freqs)
        o = attend(q, k, v, starts, max_len=130, window=window)
        y = o.flatten(1).to(dtype) @ c.t() + a
        if dtype == torch.float32:
            y, e = y.to(BF16), e.to(BF16)
        out = loss(y, e, t)
        return (out, *torch.autograd.grad(out, leaves))

    got = run(torch.float32, rotary_embedding, packed_attention, linear_cross_entropy)
    want = run(torch.float64, plain_rotary, plain_attention, plain_loss)
    assert abs(float(got[0] - want[0])) <= STEP * float(want[0])
    for name, a, b in zip(("x", "wq", "wo", "wv"), got[1:], want[1:]):
        print(f"[step] {name} {rel(a, b):.2e}", flush=True)
        assert rel(a, b) < STEP, name


def test_turned_keys_in_the_cache(dev):
    """Serving: keys are turned before they are cached, queries before they attend, in
    chunks and token by token, against attention over all of them at once."""
    g = torch.Generator().manual_seed(1)
    n, heads, kv, dim = 50, 4, 2, 64
    freqs = rotary_frequencies(dim, factor=4.0, trained_length=32, device=dev)
    q = torch.randn(n, heads, dim, generator=g).to(BF16).to(dev)
    k, v = (torch.randn(n, kv, dim, generator=g).to(BF16).to(dev) for _ in range(2))
    pos = torch.arange(n, device=dev)
    tq, tk = rotary_embedding(q, k, pos, freqs)
    want = packed_attention(tq, tk, v, torch.tensor([0, n], dtype=torch.int32, device=dev), max_len=n)
    cache = PagedKVCache(1, 8, kv, dim, page_size=16, device=dev)
    seq, at, got = cache.open(), 0, []
    for m in (20, 1, 1, 25, 3):
        batch = cache.extend([seq], [m])
        a, b = rotary_embedding(q[at:at + m], k[at:at + m], pos[at:at + m], freqs)
        cache.write(0, b, v[at:at + m], batch)
        got.append(cache.attend(0, a, batch))
        at += m
    # (E4M3 keys and values: half a step of 2^-4 of each, some 2.5e-2 of a vector's norm)
    assert rel(torch.cat(got), want) < 0.1


@pytest.fixture
def example():
    path = Path(__file__).resolve().parent.parent / "examples" / "generate.py"
    spec = importlib.util.spec_from_file_location("generate_example_step", path)
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    return ex


@pytest.mark.parametrize("rotary", [False, True])
def test_the_example_s_gradients(dev, example, monkeypatch, rotary):
    """One step of the example's decoder against the same layers around plain
    operators.  (Block-scaled linears and norms are the same on both sides; their codes
    jump where an input differs by a rounding, 2^-4 of single values, so two layers' worth
    of that are allowed on top.)"""
    torch.manual_seed(0)
    model = example.Decoder(layers=1, rotary=rotary).to(dev)
    data = example.patterns(4, 65, torch.Generator().manual_seed(2)).to(dev)
    names = [n for n, _ in model.named_parameters()]

    def grads():
        m = copy.deepcopy(model)  # (a forward pass moves its layers' error feedback on)
        loss = m.loss(data[:, :-1], data[:, 1:])
        return loss, torch.autograd.grad(loss, list(m.parameters()))

    loss, got = grads()
    monkeypatch.setattr(example, "rotary_embedding", plain_rotary)
    monkeypatch.setattr(example, "packed_attention",
                        lambda q, k, v, starts, max_len: plain_attention(q, k, v, starts).to(BF16))
    monkeypatch.setattr(example, "linear_cross_entropy", lambda h, w, t: plain_loss(h, w, t).float())
    plain, want = grads()
    assert abs(float(loss - plain)) <= STEP * float(plain)
    for n, a, b in zip(names, got, want):
        print(f"[example] {n} {rel(a, b):.2e}", flush=True)
        assert rel(a, b) < STEP + 2 * 2.0**-5, n


def test_the_example_serves_what_it_trains_with_turns(dev, example):
    torch.manual_seed(0)
    model = example.Decoder(rotary=True).to(dev)
    example.train(model, 3, batch=4)
    server = example.Server(model, pages=64)
    rows = example.patterns(3, 40, torch.Generator().manual_seed(1))
    seqs = [server.cache.open() for _ in rows]
    a = server.step(seqs, [r.tolist() for r in rows]).reshape(3, 40, -1)
    with torch.no_grad():
        full = model(rows.to(dev))
    # (as for learned positions: the cache's E4M3 keys and values)
    assert rel(a, full) < 0.1
    with pytest.raises(ValueError, match="256 positions"):
        server.step(seqs, [[1] * 217, [1], [1]])


def test_a_captured_step(dev):
    """Forward and backward through all three in one graph: every replay is the eager
    step, bit for bit, also between eager steps, and as the sequences change."""
    heads, kv_heads, dim, vocab = 4, 2, 64, 300
    lens = (130, 1, 69)
    tokens = sum(lens)
    g = torch.Generator().manual_seed(31)
    x0 = torch.randn(tokens, (heads + 2 * kv_heads) * dim, generator=g).to(BF16).to(dev)
    w0 = (torch.randn(vocab, heads * dim, generator=g) / 16).to(BF16).to(dev)
    targets = torch.randint(0, vocab, (tokens,), generator=g).to(dev)
    at = torch.tensor([0, 130, 131, 200], dtype=torch.int32, device=dev)
    pos = torch.arange(tokens, device=dev)
    freqs = rotary_frequencies(dim, device=dev)
    by = torch.full((), 0.3, device=dev)

    def step(x, w):
        x, w = x.detach().requires_grad_(), w.detach().requires_grad_()  # (sharing memory)
        q, k, v = x.unflatten(1, (-1, dim)).split((heads, kv_heads, kv_heads), 1)
        q, k = rotary_embedding(q, k, pos, freqs)
        y = packed_attention(q, k, v, at, max_len=tokens)
        loss = linear_cross_entropy(y.flatten(1), w, targets)
        return (loss.detach(), *torch.autograd.grad(loss, (x, w), by))

    x, w = x0.clone(), w0.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step(x, w)
    for i, starts in enumerate(([0, 130, 131, 200], [0, 10, 190, 200], [0, 0, 200, 200])):
        x.copy_(x0 * (1 + i / 4))
        w.copy_(w0 * (1 - i / 4))
        at.copy_(torch.tensor(starts, dtype=torch.int32))
        want = step(x, w)
        torch.cuda.synchronize()
        for _ in range(2):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def room(gib):
    if torch.cuda.mem_get_info()[0] < gib << 30:
        pytest.skip(f"needs {gib} GiB of GPU memory")


def test_attention_past_32_bits(dev):
    """More than 2^32 values of q: its last sequence as if it were alone (the others are
    zeros), turned and attended, with gradients."""
    room(90)
    heads, dim, n, tokens = 128, 128, 200, 270000
    g = torch.Generator(device=dev).manual_seed(41)
    part = [torch.randn(n, h, dim, device=dev, dtype=BF16, generator=g) for h in (heads, 1, 1, heads)]
    pos = torch.arange(tokens, device=dev) % 4000
    freqs = rotary_frequencies(dim, device=dev)

    def run(q, k, v, go, pos, starts):
        q, k, v = (x.requires_grad_() for x in (q, k, v))
        a, b = rotary_embedding(q, k, pos, freqs)
        at = torch.tensor(starts, dtype=torch.int32, device=dev)
        o = packed_attention(a, b, v, at, max_len=n, window=64)
        return (o.detach()[-n:], *(x[-n:] for x in torch.autograd.grad(o, (q, k, v), go)))

    whole = []
    for x in part:
        whole.append(torch.zeros(tokens, *x.shape[1:], dtype=BF16, device=dev))
        whole[-1][-n:] = x
    assert whole[0].numel() > 2**32
    got = run(*whole, pos, [*range(0, tokens - n + 1, n), tokens])
    want = run(*part, pos[-n:], [0, n])
    for x, y in zip(got, want):
        # (how many parts a group's heads make is by the number of tiles)
        torch.testing.assert_close(x, y, rtol=3 * 2.0**-8, atol=2e-4 * float(y.abs().max()))


def test_loss_past_32_bits(dev):
    """More than 2^32 values of the hidden states, in a row and with gradients; the last
    tokens as if they were alone (the others are left out)."""
    room(60)
    tokens, d, vocab, n = 2_200_000, 2048, 96, 500
    g = torch.Generator(device=dev).manual_seed(42)
    part = torch.randn(n, d, device=dev, dtype=BF16, generator=g)
    w = (torch.randn(vocab, d, device=dev, generator=g) / 32).to(BF16)
    targets = torch.randint(0, vocab, (n,), device=dev, generator=g)
    h = torch.zeros(tokens, d, dtype=BF16, device=dev)
    h[-n:] = part
    t = torch.full((tokens,), -100, device=dev)
    t[-n:] = targets
    assert h.numel() > 2**32

    def run(h, w, t):
        h, w = h.requires_grad_(), w.detach().requires_grad_()
        loss = linear_cross_entropy(h, w, t)
        dh, dw = torch.autograd.grad(loss, (h, w))
        return loss.detach(), dh[-n:], dw

    got, want = run(h, w, t), run(part, w, targets)
    assert abs(float(got[0] - want[0])) <= 2.0**-20 * float(want[0])
    # (alone the logits' gradients come from fp16: each side's roundings, a sum's order)
    for x, y in zip(got[1:], want[1:]):
        assert rel(x, y) <= 4 * 2.0**-8
