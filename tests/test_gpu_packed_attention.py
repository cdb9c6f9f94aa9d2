"""Attention within packed sequences and its gradients against the formulas in 64
bits.

Tolerances (per element).  A sum of n products in fp32 is within n 2^-23 of the sum
of their sizes.  A score is off by ds = scale D 2^-23 sum |q k|, a weight p by 2 max
ds + 2^-20 + n 2^-23 of itself (eps); p is rounded to bf16, 2^-8 of itself, before it
meets v or dO, and so is dS = p (dP - delta) before it meets k or q; delta comes from
the rounded output; every result is rounded to bf16 once more."""
import math

import pytest
import torch

from tcfp_amd import attention as A

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
HALF = 2.0**-8
SUM = 2.0**-23


def visible(nq, nk, causal, window):
    p = torch.arange(nq)[:, None] + nk - nq
    j = torch.arange(nk)[None, :]
    seen = torch.ones(nq, nk, dtype=torch.bool)
    if causal:
        seen &= j <= p
    if window:
        seen &= j > p - window
    return seen


def exact(q, k, v, go, starts, kstarts, scale, causal, window):
    """{name: (value, tolerance)} in 64 bits on the CPU."""
    q, k, v = (x.detach().double().cpu() for x in (q, k, v))
    go = torch.zeros_like(q) if go is None else go.detach().double().cpu()
    out = {n: (torch.zeros_like(x), torch.zeros_like(x))
           for n, x in (("o", q), ("dq", q), ("dk", k), ("dv", v))}
    group, dim = q.shape[1] // k.shape[1], q.shape[2]
    for b in range(len(starts) - 1):
        a, z, ka, kz = starts[b], starts[b + 1], kstarts[b], kstarts[b + 1]
        nq, nk = z - a, kz - ka
        if nq == 0:
            continue
        seen = visible(nq, nk, causal, window)
        some = seen.any(1)
        for h in range(q.shape[1]):
            g = h // group
            Q, K, V, G = q[a:z, h], k[ka:kz, g], v[ka:kz, g], go[a:z, h]
            s = scale * Q @ K.t()
            p = torch.softmax(s.masked_fill(~seen, -math.inf), 1) * some[:, None]
            p = torch.nan_to_num(p, nan=0.0) * seen
            ds_ = abs(scale) * dim * SUM * (Q.abs() @ K.abs().t())
            ds_ = (ds_ * seen).amax(1, keepdim=True) if nk else torch.zeros(nq, 1)
            eps = 2 * ds_ + 2.0**-20 + nk * SUM + s.abs() * 2.0**-22
            o = p @ V
            o_tol = HALF * o.abs() + (1 + HALF) * ((HALF + 1.01 * eps + nk * SUM) * p) @ V.abs()
            out["o"][0][a:z, h] = o
            out["o"][1][a:z, h] = o_tol
            dp = G @ V.t()
            delta = (G * o).sum(1, keepdim=True)
            dp_off = dim * SUM * (G.abs() @ V.abs().t()) + (G.abs() * (o_tol + 2 * dim * SUM * o.abs())).sum(1, keepdim=True)
            t = p * (dp - delta)
            t_tol = p * ((1.01 * eps) * (dp - delta).abs() + 1.01 * dp_off)
            t_tol = t_tol * (1 + HALF) + HALF * t.abs()
            out["dq"][0][a:z, h] = scale * t @ K
            out["dq"][1][a:z, h] = abs(scale) * ((1 + HALF) * (t_tol + nk * SUM * t.abs()) @ K.abs())
            out["dk"][0][ka:kz, g] += scale * t.t() @ Q
            out["dk"][1][ka:kz, g] += abs(scale) * (1 + HALF) * (t_tol + group * nq * SUM * t.abs()).t() @ Q.abs()
            out["dv"][0][ka:kz, g] += p.t() @ G
            out["dv"][1][ka:kz, g] += (1 + HALF) * ((HALF + 1.01 * eps + group * nq * SUM) * p).t() @ G.abs()
    for n in ("dq", "dk", "dv"):
        out[n][1].add_(HALF * out[n][0].abs())
    return out


def within(got, want, what):
    value, tol = want
    assert got.dtype == BF16 and got.shape == value.shape, what
    err = (got.detach().double().cpu() - value).abs()
    bad = ~(err <= tol + 1e-30)
    assert not bad.any(), (what, int(bad.sum()), float((err / (tol + 1e-30)).max()),
                           bad.nonzero()[0].tolist())


def inputs(dev, lens, heads, kv_heads, dim, key_lens=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    kstarts = starts
    if key_lens is not None:
        kstarts = [0]
        for n in key_lens:
            kstarts.append(kstarts[-1] + n)
    q = (torch.randn(starts[-1], heads, dim, generator=g) * 1.5).to(BF16).to(dev)
    kv = torch.randn(kstarts[-1], 2 * kv_heads * dim, generator=g).to(BF16).to(dev)
    k, v = (x.unflatten(1, (kv_heads, dim)) for x in kv.chunk(2, 1))
    go = torch.randn(starts[-1], heads, dim, generator=g).to(BF16).to(dev)
    return q, k, v, go, starts, kstarts


def i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def run(dev, q, k, v, go, starts, kstarts, *, scale=None, causal=True, window=0, max_len=None):
    q, k, v = (x.detach().requires_grad_() for x in (q, k, v))
    longest = max([b - a for a, b in zip(starts, starts[1:])], default=0)
    how = dict(max_len=longest if max_len is None else max_len, scale=scale, causal=causal, window=window)
    if kstarts is not starts:
        how["key_start"] = i32(kstarts, dev)
        how["max_key_len"] = max([b - a for a, b in zip(kstarts, kstarts[1:])], default=0)
    o = A.packed_attention(q, k, v, i32(starts, dev), **how)
    with torch.no_grad():
        plain = A.packed_attention(q, k, v, i32(starts, dev), **how)
    assert torch.equal(plain.view(torch.int16), o.detach().view(torch.int16))
    return (o.detach(), *torch.autograd.grad(o, (q, k, v), go))


def compare(dev, q, k, v, go, starts, kstarts, **how):
    got = run(dev, q, k, v, go, starts, kstarts, **how)
    how.pop("max_len", None)
    scale = how.pop("scale", None)
    want = exact(q, k, v, go, starts, kstarts, q.shape[2]**-0.5 if scale is None else scale,
                 how.get("causal", True), how.get("window", 0))
    for n, x in zip(("o", "dq", "dk", "dv"), got):
        within(x, want[n], n)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lens,heads,kv_heads", [
    ([1], 1, 1), ([2, 1, 3], 2, 1), ([31, 32, 33], 2, 2), ([63, 64, 65], 4, 1), ([127, 128, 129], 3, 3),
    ([200, 0, 1, 77], 4, 2), ([300], 6, 2), ([513], 1, 1), ([5] * 40, 8, 8)])
def test_causal(dev, dim, lens, heads, kv_heads):
    print(f"[packed] causal {lens} {heads} {kv_heads} {dim}", flush=True)
    compare(dev, *inputs(dev, lens, heads, kv_heads, dim))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window", [0, 1, 17, 64, 100, 1 << 40])
def test_masks(dev, dim, causal, window):
    print(f"[packed] masks {dim} {causal} {window}", flush=True)
    compare(dev, *inputs(dev, [150, 3, 260], 2, 1, dim, seed=1), causal=causal, window=window)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window", [0, 20])
def test_keys_of_their_own(dev, dim, causal, window):
    """Longer than the queries (a chunk behind what is there), shorter (queries that
    see nothing), none at all, and keys that no query has."""
    print(f"[packed] keys {dim} {causal} {window}", flush=True)
    compare(dev, *inputs(dev, [40, 70, 5, 0, 33], 4, 2, dim, [200, 20, 0, 90, 33], seed=2),
            causal=causal, window=window)


@pytest.mark.parametrize("scale", [0.3, -0.2, 0.0, 1e-3])
def test_scales(dev, scale):
    compare(dev, *inputs(dev, [70, 30], 2, 2, 64, seed=3), scale=scale)


@pytest.mark.parametrize("heads,kv_heads", [(8, 1), (6, 1), (7, 7)])
def test_few_keys_share_out_the_heads(dev, heads, kv_heads):
    """Few tiles of keys: the group's heads are dealt to workgroups whose parts are
    joined."""
    compare(dev, *inputs(dev, [140, 60], heads, kv_heads, 128, seed=4))


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_short_sequences_are_as_exact_as_their_results(dev, dim):
    """Bounds up to 256: dQ and dK are off by their own rounding, 2^-8 / sqrt(12) to
    2^-8 / sqrt(3) of a value (1.7e-3 over even mantissas), and by what P's rounding
    left in delta, a third of that; with dS rounded as well, by 2.4e-3."""
    lens = [1 + i * 37 % 256 for i in range(12)] + [256, 255, 64, 65]
    q, k, v, go, starts, _ = inputs(dev, lens, 4, 2, dim, seed=22)
    got = run(dev, q, k, v, go, starts, starts)
    want = exact(q, k, v, go, starts, starts, dim**-0.5, True, 0)
    for n, y in zip(("dq", "dk"), got[1:]):
        value = want[n][0]
        off = (y.double().cpu() - value).norm() / value.norm()
        assert off <= 2.1e-3, (n, float(off))


def test_bounds_that_are_too_small(dev):
    data = inputs(dev, [300, 10, 150], 2, 1, 64, seed=5)
    want = {short: run(dev, *data, max_len=200 if short else 300) for short in (False, True)}
    for bound in (0, 1, 130, 100000):
        got = run(dev, *data, max_len=bound)
        # (the heads are shared out by the bound: the parts' sums have another order; and
        # up to 256 it says how many bits of dS there are)
        assert torch.equal(got[0], want[False][0])
        assert torch.equal(got[1], want[bound <= 256][1])
    compare(dev, *data, max_len=1)


def test_many_short_sequences_under_a_far_bound(dev):
    """Keys of their own without a bound: all keys of the batch for every sequence."""
    lens = [1 + i % 3 for i in range(700)]
    keys = [1 + i % 5 for i in range(700)]
    q, k, v, go, starts, kstarts = inputs(dev, lens, 2, 1, 64, keys, seed=20)
    x = [y.detach().requires_grad_() for y in (q, k, v)]
    o = A.packed_attention(*x, i32(starts, dev), max_len=10**9, key_start=i32(kstarts, dev))
    got = (o.detach(), *torch.autograd.grad(o, x, go))
    want = exact(q, k, v, go, starts, kstarts, 0.125, True, 0)
    for n, y in zip(("o", "dq", "dk", "dv"), got):
        within(y, want[n], n)


def test_more_tiles_than_workgroups(dev):
    """Sequences times heads times tiles past what a launch holds (4 million workgroups):
    one long sequence among many of one token."""
    long, heads = 15000, 8
    lens = [1] * 2500 + [long] + [1] * 2499
    q, k, v, go, starts, _ = inputs(dev, lens, heads, heads, 64, seed=21)
    got = run(dev, q, k, v, go, starts, starts, window=200)
    at = slice(2500, 2500 + long)
    q, k, v, go = (x[at] for x in (q, k, v, go))
    want = run(dev, q, k, v, go, [0, long], [0, long], window=200)
    for x, y in zip(got, want):
        # (the same values, but for dK and dV's sums if they are split another way)
        torch.testing.assert_close(x[at], y, rtol=3 * HALF, atol=2e-4 * float(y.abs().max()))


def test_rows_outside_the_sequences(dev):
    q, k, v, go, _, _ = inputs(dev, [100], 4, 2, 64, seed=6)
    q, k, v, go = (x.clone() for x in (q, k, v, go))
    for x in (q, k, v, go):
        x[:10] = math.nan
        x[90:] = math.nan
    starts = [10, 40, 90]
    got = run(dev, q, k, v, go, starts, starts)
    for x in got:
        assert not x[:10].any() and not x[90:].any()
    inner = run(dev, q[10:90], k[10:90], v[10:90], go[10:90], [0, 30, 80], [0, 30, 80])
    want = exact(q[10:90], k[10:90], v[10:90], go[10:90], [0, 30, 80], [0, 30, 80], 0.125, True, 0)
    for n, x, y in zip(("o", "dq", "dk", "dv"), got, inner):
        within(x[10:90], want[n], n)
        assert torch.equal(x[10:90], y)


def test_what_is_not_finite_stays_in_its_sequence(dev):
    q, k, v, go, starts, _ = inputs(dev, [70, 50, 90], 2, 1, 64, seed=7)
    clean = run(dev, q, k, v, go, starts, starts)
    for name in ("q", "k", "v", "go"):
        x = {"q": q, "k": k, "v": v, "go": go}
        x = {n: y.clone() for n, y in x.items()}
        x[name][80, 0, 5] = math.nan
        x[name][85, 0, 7] = math.inf
        got = run(dev, x["q"], x["k"], x["v"], x["go"], starts, starts)
        for a, b in zip(got, clean):
            assert torch.equal(a[:70], b[:70]) and torch.equal(a[120:], b[120:]), name
        # (and what cannot see the token is as it was: queries in tiles before it)
        assert not torch.isfinite(torch.cat([y[70:120].flatten() for y in got])).all()


def test_large_scores(dev):
    q, k, v, go, starts, _ = inputs(dev, [90], 2, 2, 64, seed=8)
    compare(dev, q * 16, k * 16, v, go, starts, starts)


def test_strides(dev):
    q, k, v, go, starts, _ = inputs(dev, [33, 20], 4, 2, 64, seed=9)
    want = run(dev, q, k, v, go, starts, starts)
    qkv = torch.zeros(53, 8 * 64 + 8, dtype=BF16, device=dev)
    qs, ks, vs = (qkv[:, a * 64:b * 64].unflatten(1, (b - a, 64)) for a, b in ((0, 4), (4, 6), (6, 8)))
    qs.copy_(q), ks.copy_(k), vs.copy_(v)
    assert all(torch.equal(a, b) for a, b in zip(run(dev, qs, ks, vs, go, starts, starts), want))
    swapped = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v, go)]
    assert all(torch.equal(a, b) for a, b in zip(run(dev, *swapped, starts, starts), want))
    odd = [torch.empty(x.numel() + 1, dtype=BF16, device=dev)[1:].view(x.shape).copy_(x)
           for x in (q, k, v, go)]
    assert all(torch.equal(a, b) for a, b in zip(run(dev, *odd, starts, starts), want))
    # the gradient of a sum: one value for all, strides of 0
    a = [x.detach().requires_grad_() for x in (q, k, v)]
    o = A.packed_attention(*a, i32(starts, dev), max_len=33)
    got = torch.autograd.grad(o.sum(), a)
    ones = run(dev, q, k, v, torch.ones_like(go), starts, starts)
    assert all(torch.equal(x, y) for x, y in zip(got, ones[1:]))


def test_one_token_of_odd_strides(dev):
    q = torch.randn(64, 2, 1).to(BF16).to(dev).permute(2, 1, 0)
    k = torch.randn(1, 1, 64).to(BF16).to(dev)
    v = torch.randn(1, 3, 64).to(BF16).to(dev)[:, 1:2]
    o = A.packed_attention(q, k, v, i32([0, 1], dev), max_len=1)
    assert torch.equal(o, v.expand(1, 2, 64))


def test_single_gradients(dev):
    q, k, v, go, starts, _ = inputs(dev, [40], 2, 1, 64, seed=10)
    want = run(dev, q, k, v, go, starts, starts)[1:]
    for i in range(3):
        x = [y.detach().requires_grad_(j == i) for j, y in enumerate((q, k, v))]
        o = A.packed_attention(*x, i32(starts, dev), max_len=40)
        (got,) = torch.autograd.grad(o, x[i], go)
        assert torch.equal(got, want[i])


def test_gradient_against_differences(dev):
    """Along directions on which x +- e d is exact in bf16; the difference's third
    order is known from the formula, the rest are the results' tolerances."""
    g = torch.Generator().manual_seed(11)
    n, e = 40, 1 / 16
    x = {a: (torch.randint(-16, 17, (n, 2 if a in ("q", "go") else 1, 64), generator=g) / 16).to(BF16)
         for a in ("q", "k", "v", "go")}
    starts = [0, 15, n]
    base = exact(x["q"], x["k"], x["v"], x["go"], starts, starts, 0.125, True, 0)
    got = run(dev, *(x[a].to(dev) for a in ("q", "k", "v", "go")), starts, starts)
    for i, a in enumerate(("q", "k", "v")):
        move = (torch.randint(-1, 2, x[a].shape, generator=g) * e).to(BF16)
        slope, formula, room = 0.0, 0.0, 0.0
        for s in (1, -1):
            y = {**x, a: x[a] + s * move}
            o = run(dev, *(y[b].to(dev) for b in ("q", "k", "v", "go")), starts, starts)[0]
            want, tol = exact(y["q"], y["k"], y["v"], y["go"], starts, starts, 0.125, True, 0)["o"]
            go = x["go"].double()
            slope += s * float((o.double().cpu() * go).sum()) / 2
            formula += s * float((want * go).sum()) / 2
            room += float((tol * go.abs()).sum()) / 2
        value, tol = base["d" + a]
        step = move.double()
        third = abs(float((value * step).sum()) - formula)
        assert abs(slope - formula) <= room
        assert abs(float((got[1 + i].double().cpu() * step).sum()) - slope) <= (
            third + room + float((tol * step.abs()).sum()))


def test_bits_repeat_and_streams(dev):
    data = inputs(dev, [200, 90, 130], 8, 2, 128, seed=12)
    want = run(dev, *data)
    assert all(torch.equal(a, b) for a, b in zip(run(dev, *data), want))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run(dev, *data)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_graph(dev):
    """Forward and backward captured, replayed over other values and lengths."""
    q, k, v, go, starts, _ = inputs(dev, [100, 60, 40], 4, 2, 64, seed=13)
    x, at = q.clone(), i32(starts, dev)

    def both():
        o, low, lse = A.packed_attention_forward(x, k, v, at, max_len=150)
        return (o, *A.packed_attention_backward(go, x, k, v, o, low, lse, at, max_len=150))

    both()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for i, other in enumerate(([0, 100, 160, 200], [0, 10, 150, 200], [5, 50, 51, 190])):
        x.copy_(q * (1 + i / 4))
        at.copy_(i32(other, dev))
        eager = both()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager))


def test_nothing(dev):
    q = torch.zeros(0, 2, 64, dtype=BF16, device=dev)
    k = torch.zeros(0, 1, 64, dtype=BF16, device=dev)
    for starts in ([0], [0, 0, 0]):
        got = run(dev, q, k, k, q, starts, starts)
        assert [x.shape[0] for x in got] == [0, 0, 0, 0]
    # queries without any key, keys without any query
    q1 = torch.ones(5, 2, 64, dtype=BF16, device=dev)
    got = run(dev, q1, k, k, q1, [0, 5], [0, 0])
    assert not got[0].any() and not got[1].any()
    k1 = torch.ones(5, 1, 64, dtype=BF16, device=dev)
    got = run(dev, q, k1, k1, q, [0, 0], [0, 5])
    assert not got[2].any() and not got[3].any()


def test_refusals(dev):
    q, k, v, go, starts, _ = inputs(dev, [6], 4, 2, 64)
    at = i32(starts, dev)

    def call(q=q, k=k, v=v, at=at, **kw):
        return A.packed_attention(q, k, v, at, **{"max_len": 6, **kw})

    for exc, kw in [
            (TypeError, dict(q=q.float())), (TypeError, dict(k=k.half())), (TypeError, dict(v=v.float())),
            (TypeError, dict(at=at.long())), (ValueError, dict(q=q[0])),
            (ValueError, dict(q=q[..., :32], k=k[..., :32], v=v[..., :32])),
            (ValueError, dict(q=q[:, :3])), (ValueError, dict(v=v[:, :1])), (ValueError, dict(k=k[:5], v=v[:5])),
            (ValueError, dict(at=at[None])), (ValueError, dict(at=at[:1])), (ValueError, dict(max_len=-1)),
            (ValueError, dict(max_key_len=-1)), (ValueError, dict(window=-1)),
            (ValueError, dict(scale=math.inf)), (ValueError, dict(scale=math.nan)),
            (TypeError, dict(key_start=at.long())), (ValueError, dict(key_start=i32([0, 3, 6], dev))),
            (RuntimeError, dict(q=q.cpu())), (RuntimeError, dict(at=at.cpu()))]:
        with pytest.raises(exc):
            call(**kw)
    o, low, lse = A.packed_attention_forward(q, k, v, at, max_len=6)
    for exc, args in [(ValueError, (go[:5], q, k, v, o, low, lse)),
                      (ValueError, (go, q, k, v, o, low, lse[:3])),
                      (TypeError, (go.float(), q, k, v, o, low, lse)),
                      (ValueError, (go, q, k, v, o[:5], low, lse)),
                      (TypeError, (go, q, k, v, o, low.float(), lse)),
                      (ValueError, (go, q, k, v, o, low[:5], lse))]:
        with pytest.raises(exc):
            A.packed_attention_backward(*args, at, max_len=6)
    a = q.clone().requires_grad_()
    (grad,) = torch.autograd.grad(call(q=a), a, go, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()
