"""Rotary positions against the rotation in 64 bits.

Tolerance (per element, of a pair of size r = A (|a| + |b|)): the angle, formed in
64 bits, is rounded to fp32 as at most half a turn (2^-26 turns, 2^-23.3 radians);
sin and cos are good to 2 ulp (2^-23), each product and the sum are rounded once
(3 * 2^-24): under 2^-21 r in all.  A bf16 result is rounded by 2^-8 of itself at
most, an fp32 one by 2^-24."""
import math

import pytest
import torch

from tcfp_amd import rotary as R

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def turned(x, positions, freqs, interleaved, amplitude=1.0, inverse=False):
    """(result, sum of the pair's sizes) in 64 bits."""
    half = len(freqs)
    angle = positions.double().cpu()[:, None, None] * freqs.double().cpu()
    c, s = torch.cos(angle), torch.sin(angle) * (-1.0 if inverse else 1.0)
    y = x.detach().double().cpu()
    part = y[..., :2 * half]
    a, b = ((part[..., 0::2], part[..., 1::2]) if interleaved
            else (part[..., :half], part[..., half:]))
    p, q, r = amplitude * (a * c - b * s), amplitude * (a * s + b * c), amplitude * (a.abs() + b.abs())

    def back(u, v):
        return torch.stack((u, v), -1).flatten(-2) if interleaved else torch.cat((u, v), -1)

    rest = y[..., 2 * half:]
    return torch.cat((back(p, q), rest), -1), torch.cat((back(r, r), torch.zeros_like(rest)), -1)


def check(got, x, *args, **kw):
    want, size = turned(x, *args, **kw)
    step = torch.finfo(x.dtype).eps / 2
    err = (got.detach().double().cpu() - want).abs()
    assert got.dtype == x.dtype and got.shape == x.shape and got.is_contiguous()
    assert (err <= step * want.abs() + (1 + step) * 2.0**-21 * size).all(), float(err.max())


def inputs(dev, tokens, heads, kv_heads, dim, dtype, far, seed=0):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(tokens, (heads + 2 * kv_heads) * dim, generator=g).to(dtype).to(dev)
    q = qkv[:, :heads * dim].unflatten(1, (heads, dim))
    k = qkv[:, heads * dim:(heads + kv_heads) * dim].unflatten(1, (kv_heads, dim))
    return q, k, torch.randint(0, far, (tokens,), generator=g).to(dev)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rotary", [
    (1, 32, 8, 128, 128), (3, 4, 4, 64, 32), (1023, 2, 1, 64, 64), (1030, 3, 1, 128, 16),
    (5, 2, 2, 80, 20), (7, 1, 1, 10, 6), (2, 2, 1, 256, 256), (1025, 1, 1, 34, 2),
    (2, 1, 1, 4096, 4096)])
def test_against_64_bits(dev, dtype, interleaved, tokens, heads, kv_heads, dim, rotary):
    print(f"[rotary] {tokens} {heads} {kv_heads} {dim} {rotary} {interleaved} {dtype}", flush=True)
    q, k, pos = inputs(dev, tokens, heads, kv_heads, dim, dtype, 100000)
    f = R.rotary_frequencies(rotary, device=dev)
    qo, ko = R.rotary_embedding(q, k, pos, f, interleaved=interleaved, amplitude=1.25)
    check(qo, q, pos, f, interleaved, 1.25)
    check(ko, k, pos, f, interleaved, 1.25)
    qi, none = R.rotary_embedding(q, None, pos, f, interleaved=interleaved, inverse=True)
    assert none is None
    check(qi, q, pos, f, interleaved, 1.0, True)


@pytest.mark.parametrize("far", [1 << 20, 1 << 31, 1 << 40])
def test_far_positions_keep_their_angle(dev, far):
    """Of position * freq the whole turns are dropped in 64 bits: up to 2^31 the
    angle is as good as a near one's, at 2^40 2^-53 of 2^40 radians are left."""
    q, k, pos = inputs(dev, 64, 2, 1, 64, F32, 1000)
    pos = pos + (far - 1000)
    f = R.rotary_frequencies(64, device=dev)
    qo, _ = R.rotary_embedding(q, k, pos, f)
    want, size = turned(q, pos, f, False)
    off = 2.0**-21 + 4 * far * 2.0**-53
    assert ((qo.double().cpu() - want).abs() <= 2.0**-24 * want.abs() + off * size).all()


def test_rows_that_are_not_aligned(dev):
    for dtype in (F32, BF16):
        base = torch.randn(9, 3 * 64 + 1).to(dtype).to(dev)
        q = base[:, 1:].unflatten(1, (3, 64))
        pos = torch.arange(9, device=dev)
        f = R.rotary_frequencies(64, device=dev)
        qo, _ = R.rotary_embedding(q, None, pos, f)
        check(qo, q, pos, f, False)
        t = torch.randn(3, 9, 64).to(dtype).to(dev).transpose(0, 1)  # heads outermost
        check(R.rotary_embedding(t, None, pos, f)[0], t, pos, f, False)
        one = torch.randn(1, 64, 3).to(dtype).to(dev).transpose(1, 2)  # dim not contiguous
        check(R.rotary_embedding(one, None, pos[3:4], f)[0], one, pos[3:4], f, False)


def test_no_tokens_and_no_heads(dev):
    f = R.rotary_frequencies(8, device=dev)
    pos = torch.zeros(0, dtype=torch.int64, device=dev)
    q, k = R.rotary_embedding(torch.zeros(0, 2, 8, device=dev), torch.zeros(0, 1, 8, device=dev),
                              pos, f)
    assert q.shape == (0, 2, 8) and k.shape == (0, 1, 8)
    q, _ = R.rotary_embedding(torch.zeros(3, 0, 8, device=dev), None,
                              torch.zeros(3, dtype=torch.int64, device=dev), f)
    assert q.shape == (3, 0, 8)


def test_what_is_not_finite_stays_in_its_pair(dev):
    q, _, pos = inputs(dev, 4, 2, 1, 64, F32, 1000)
    q = q.clone()
    q[1, 1, 3] = math.nan
    q[2, 0, 60] = math.inf
    f = R.rotary_frequencies(64, device=dev)
    out, _ = R.rotary_embedding(q, None, pos, f)
    bad = torch.zeros(4, 2, 64, dtype=torch.bool)
    bad[1, 1, [3, 35]] = True
    bad[2, 0, [60, 28]] = True
    assert torch.equal(~torch.isfinite(out).cpu(), bad)


@pytest.mark.parametrize("which", ["both", "q", "k"])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gradients_turn_back(dev, dtype, which):
    q, k, pos = inputs(dev, 33, 4, 2, 64, dtype, 5000)
    q, k = q.detach(), k.detach()
    q.requires_grad_(which != "k")
    k.requires_grad_(which != "q")
    f = R.rotary_frequencies(32, device=dev)
    qo, ko = R.rotary_embedding(q, k, pos, f, interleaved=True, amplitude=0.5)
    gq, gk = torch.randn_like(qo), torch.randn_like(ko)
    want = [x for x in (q, k) if x.requires_grad]
    got = list(torch.autograd.grad((qo, ko), want, (gq, gk)))
    if which != "k":
        check(got.pop(0), gq, pos, f, True, 0.5, True)
    if which != "q":
        check(got.pop(0), gk, pos, f, True, 0.5, True)


def test_gradient_against_differences(dev):
    """The map is linear: its difference along any direction is its value there, and
    <g, R x> = <R^T g, x>."""
    q, _, pos = inputs(dev, 20, 2, 1, 64, F32, 5000)
    q = q.detach().clone().requires_grad_()
    f = R.rotary_frequencies(64, device=dev)
    out, _ = R.rotary_embedding(q, None, pos, f)
    g, d = torch.randn_like(out), torch.randn_like(out)
    g = g.detach().requires_grad_()
    (grad,) = torch.autograd.grad(out, q, g, create_graph=True)
    with torch.no_grad():
        up, _ = R.rotary_embedding(q + d, None, pos, f)
        down, _ = R.rotary_embedding(q - d, None, pos, f)
        lhs = ((up.double() - down.double()) * g.double()).sum() / 2
        rhs = (grad.double() * d.double()).sum()
        # every value within 2^-20 of its pair's size: the sum of what they can make up
        room = 2.0**-19 * (2 * g.double().abs().sum() * (q.abs() + d.abs()).max())
        assert abs(float(lhs - rhs)) <= float(room)
    # and the gradient's own gradient is the map again
    (twice,) = torch.autograd.grad(grad, g, d)
    assert torch.equal(twice, R.rotary_embedding(d, None, pos, f)[0])


def test_side_stream_and_graph(dev):
    q, k, pos = inputs(dev, 40, 4, 2, 64, BF16, 5000)
    f = R.rotary_frequencies(64, device=dev)
    want = R.rotary_embedding(q, k, pos, f)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = R.rotary_embedding(q, k, pos, f)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    x = q.clone()
    with torch.cuda.graph(graph):
        out = R.rotary_embedding(x, k, pos, f)
    for i in range(3):
        x.copy_(q * (i + 1))
        eager = R.rotary_embedding(x, k, pos, f)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager))


def test_refusals(dev):
    q, k, pos = inputs(dev, 4, 2, 1, 64, BF16, 100)
    f = R.rotary_frequencies(64, device=dev)
    for exc, args in [
            (TypeError, (q.half(), None, pos, f)), (TypeError, (q, k.float(), pos, f)),
            (TypeError, (q, k, pos.int(), f)), (TypeError, (q, k, pos, f.float())),
            (ValueError, (q[0], None, pos, f)), (ValueError, (q, k[:3], pos, f)),
            (ValueError, (q, k[..., :32], pos, f)), (ValueError, (q, k, pos[:3], f)),
            (ValueError, (q[..., :32], None, pos, f)), (ValueError, (q, k, pos, f[:0])),
            (RuntimeError, (q, k, pos.cpu(), f)), (RuntimeError, (q.cpu(), None, pos, f))]:
        with pytest.raises(exc):
            R.rotary_embedding(*args)
