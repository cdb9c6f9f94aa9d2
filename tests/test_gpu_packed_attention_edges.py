"""Attention within packed sequences: queries that see nothing beside values that are not
finite, and the bits that out_low keeps."""
import math

import pytest
import torch

from tcfp_amd import attention as A
from test_gpu_packed_attention import i32, inputs, run

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("name", ["k", "v", "go"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("bound", [90, 300])
def test_a_query_that_sees_nothing(dev, dim, name, value, bound):
    """Zeros and a zero gradient, whatever the keys, values and gradients hold that
    others of its tile see: 70 queries on 20 keys, of which the first 50 see none."""
    q, k, v, go, starts, kstarts = inputs(dev, [90, 70, 33], 4, 2, dim, [90, 20, 33], seed=31)
    x = {"q": q, "k": k.clone(), "v": v.clone(), "go": go.clone()}
    x[name][(140 if name == "go" else 95), :, 3] = value
    got = run(dev, x["q"], x["k"], x["v"], x["go"], starts, kstarts, max_len=bound)
    assert not got[0][90:140].any(), "out"
    assert not got[1][90:140].any(), "dq"
    clean = run(dev, q, k, v, go, starts, kstarts, max_len=bound)
    for a, b in zip(got, clean):  # (the neighbours)
        n = 110 if a.shape[1] == 2 else 160
        assert torch.equal(a[:90], b[:90]) and torch.equal(a[n:], b[n:])
    # without autograd: the statistic says so too
    _, low, lse = A.packed_attention_forward(
        x["q"], x["k"], x["v"], i32(starts, dev), max_len=bound, key_start=i32(kstarts, dev))
    assert not low[90:140].any() and (lse[:, 90:140] == math.inf).all()


def test_the_bits_that_rounding_left(dev):
    """Two keys alike: every weight is 1/2, and out is the mean of two values, of which
    out and out_low together have sixteen bits: within 2^-8 of bf16's last place, 2^-15 of
    the value (half of that but where half a last place is left, 128 of an int8 that
    ends at 127; and the weights' and sums' fp32 roundings, 2^-20)."""
    g = torch.Generator().manual_seed(32)
    n = 40
    q = torch.randn(2 * n, 2, 64, generator=g).to(BF16).to(dev)
    k = torch.randn(n, 1, 64, generator=g).to(BF16).repeat_interleave(2, 0).to(dev)
    v = torch.randn(2 * n, 1, 64, generator=g).to(BF16).to(dev)
    at = torch.arange(0, 2 * n + 1, 2, dtype=torch.int32, device=dev)
    out, low, _ = A.packed_attention_forward(q, k, v, at, max_len=2, causal=False)
    bits = (out.view(torch.int16).int() << 16) + (low.int() << 8)
    got = bits.view(torch.float32).double()
    want = (v.double().view(n, 2, 1, 64).mean(1, keepdim=True).expand(n, 2, 2, 64)).reshape(got.shape)
    assert ((got - want).abs() <= (2.0**-15 + 2.0**-20) * want.abs()).all()
    assert ((out.double() - want).abs() > 2.0**-10 * want.abs()).any()  # (there was something left)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("name", ["q", "k", "v", "go"])
def test_tiles_that_cannot_see_it_are_as_they_were(dev, dim, name):
    """A value that is not finite is not met by tiles of 128 rows that lie wholly before
    it (queries, of a key) or behind it (keys, of a query)."""
    q, k, v, go, starts, _ = inputs(dev, [300], 2, 1, dim, seed=33)
    x = {"q": q, "k": k.clone(), "v": v.clone(), "go": go}
    x = {n: y.clone() for n, y in x.items()}
    at = 250 if name in ("k", "v") else 50
    x[name][at, 0, 5] = math.nan
    got = run(dev, x["q"], x["k"], x["v"], x["go"], starts, starts)
    clean = run(dev, q, k, v, go, starts, starts)
    for i, (a, b) in enumerate(zip(got, clean)):
        if name in ("k", "v") and i < 2:  # out, dq
            assert torch.equal(a[:128], b[:128])
        elif name in ("q", "go") and i >= 2:  # dk, dv
            assert torch.equal(a[128:], b[128:])
    assert not all(torch.isfinite(a).all() for a in got)
