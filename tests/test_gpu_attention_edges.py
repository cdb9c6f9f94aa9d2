"""Paged attention at the edges of its arguments, against the same plain
implementation in 64 bits and with the same tolerance as the rest."""
import sys

import pytest
import torch

from tcfp_amd import attention as A
from test_gpu_attention import DECODE, MIXED, Batch, _mask, _values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lens", [DECODE, MIXED, [(1, 5000)], [(300, 2000), (1, 3000)]])
def test_a_window_past_every_key(dev, dim, lens):
    """None, by the bits of the call without one."""
    print(f"[attend] window {dim} {lens}", flush=True)
    b = Batch(dev, lens, 6, 2, dim, 16, seed=23)
    want = b.attend()
    b.check(want)
    for window in (1 << 30, 1 << 40, sys.maxsize):
        assert torch.equal(b.attend(window=window), want)
    bound = b.attend(max_query_len=1 << 30)
    assert torch.equal(b.attend(max_query_len=sys.maxsize), bound)
    b.check(bound)


# Batches for every form of launch: (lens, heads, K/V heads) of few rows whole,
# few rows in parts that a wave or four join, more than a wave's and a workgroup's
# sequences, small tiles, tiles of eight waves on 128 and 256 rows, split keys.
FORMS = {
    "few-whole": ([(1, 100), (2, 60), (0, 5), (1, 1)], 4, 2),
    "few-one": ([(1, 3000)], 4, 2),
    "few-parts": ([(4, 900), (3, 1200), (2, 2)], 8, 2),
    "few-70": ([(1, 20 + 9 * i) for i in range(70)], 4, 2),
    "few-300": ([(4 if i % 3 else 0, 300 + (i * 53) % 500) for i in range(300)], 2, 1),
    "small": ([(40, 100), (90, 90)], 2, 2),
    "prompts": ([(500, 500), (0, 3), (77, 200)], 16, 4),
    "paired": ([(900, 900)], 12, 6),
    "wide": ([(200, 1000), (150, 700)], 4, 2),
    "split": ([(90, 6000), (40, 40), (57, 4097)], 3, 3),
}


def _expected_nan(b, bad, causal, window, rows):
    """[rows, heads, dim]: which outputs see a NaN; bad [slots, kv_heads, dim]."""
    out = torch.zeros(rows, b.heads, b.dim, dtype=torch.bool, device=bad.device)
    for s, (n, total) in enumerate(b.lens):
        if n:
            seen = _mask(n, total, causal, window, bad.device)
            for x in b.holes.get(s, ()):
                seen[:, x] = False
            hit = torch.stack([seen.float() @ bad[b.slots[s], h].float()
                               for h in range(bad.shape[1])], 1) > 0
            out[b.at[s]:b.at[s + 1]] = hit.repeat_interleave(b.group, 1)
    return out


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 150), (False, 0), (False, 40)])
def test_nan_in_a_column_of_v(dev, dim, form, causal, window):
    """A NaN in one column of a cached value reaches that column of the rows that
    see it: no other column, no other row, whatever the launch."""
    lens, heads, kv_heads = FORMS[form]
    print(f"[attend] nan {form} {dim} {causal} {window}", flush=True)
    page = 16
    b = Batch(dev, lens, heads, kv_heads, dim, page, seed=24)
    b.holes = {}
    kw = dict(causal=causal, window=window)
    clean = b.attend(**kw)
    g = torch.Generator().manual_seed(25)
    codes = b.pool[1].view(torch.uint8)
    kept = codes.clone()
    for tries in range(3):
        codes.copy_(kept)
        for s, (n, total) in enumerate(lens):
            # near the ends of what is seen, and anywhere
            spots = [total - 1, max(total - n, 0), max(total - n - window, 0)]
            spots += torch.randint(0, max(total, 1), (2,), generator=g).tolist()
            for j in spots[tries:tries + 3]:
                if j < total:
                    slot = int(b.slots[s][j])
                    h = int(torch.randint(0, kv_heads, (), generator=g))
                    d = int(torch.randint(0, dim, (), generator=g))
                    codes[slot // page, h, slot % page, d] = 0x7F if j % 2 else 0xFF
        bad = _values(b.pool)[1].isnan()
        got = b.attend(**kw)
        want = _expected_nan(b, bad, causal, window, got.shape[0])
        assert torch.equal(got.isnan(), want)
        assert torch.equal(got[~want], clean[~want])


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("form", ["few-one", "prompts", "paired", "wide", "split"])
def test_nan_in_a_column_of_v_beside_a_hole(dev, dim, form):
    """The same where pages are missing, so that every step is looked at."""
    lens, heads, kv_heads = FORMS[form]
    print(f"[attend] nan and hole {form} {dim}", flush=True)
    page = 16
    b = Batch(dev, lens, heads, kv_heads, dim, page, seed=26)
    b.table[0, 3:6] = -1
    b.holes = {0: [slice(48, 96)]}
    clean = b.attend()
    codes = b.pool[1].view(torch.uint8)
    for j, d in ((0, 3), (47, 60), (60, 10), (96, dim - 1), (lens[0][1] // 2, 33),
                 (lens[0][1] - 1, 0)):
        slot = int(b.slots[0][j])
        codes[slot // page, kv_heads - 1, slot % page, d] = 0x7F
    bad = _values(b.pool)[1].isnan()
    got = b.attend()
    want = _expected_nan(b, bad, True, 0, got.shape[0])
    assert torch.equal(got.isnan(), want) and want.any()
    assert torch.equal(got[~want], clean[~want])


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("lead,tail", [(3, 0), (0, 2), (5, 37)])
def test_rows_of_no_sequence(dev, dim, form, lead, tail):
    """Rows of q before the first sequence and behind the last: zeros."""
    lens, heads, kv_heads = FORMS[form]
    print(f"[attend] lead {form} {dim} {lead} {tail}", flush=True)
    b = Batch(dev, lens, heads, kv_heads, dim, 16, seed=27)
    n = b.q.shape[0]
    rows = torch.randn(lead + n + tail, heads, dim, device=dev).bfloat16()
    rows[lead:lead + n] = b.q
    # (values where the output may be allocated)
    old = [torch.full_like(rows, 7.0) for _ in range(3)]
    del old
    got = A.paged_attention(rows, *b.pool, b.table, b.seq_lens, b.starts + lead,
                            max_query_len=max(x for x, _ in lens))
    assert (got[:lead] == 0).all() and (got[lead + n:] == 0).all()
    b.check(got[lead:lead + n])


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("form", FORMS)
def test_scale_of_zero(dev, dim, form):
    """The mean of the values that a row sees."""
    lens, heads, kv_heads = FORMS[form]
    b = Batch(dev, lens, heads, kv_heads, dim, 16, seed=28)
    b.check(b.attend(scale=0.0), scale=0.0)
    b.check(b.attend(scale=0.0, window=50), scale=0.0, window=50)


def test_a_gradient_is_refused_and_not_lost(dev):
    """There is no backward pass: the result stays in the graph, and the pass that
    reaches it raises."""
    b = Batch(dev, [(3, 20)], 4, 2, 64, 16, seed=29)
    want = b.attend()
    assert not want.requires_grad
    b.q = b.q.clone().requires_grad_(True)
    got = b.attend()
    assert got.requires_grad and torch.equal(got.detach(), want)
    with pytest.raises(NotImplementedError, match="no backward"):
        got.float().sum().backward()
    with torch.no_grad():
        got = b.attend()
        assert not got.requires_grad and torch.equal(got, want)
    with torch.inference_mode():
        assert torch.equal(b.attend(), want)


@pytest.mark.parametrize("sequences", [3, 70, 300])
def test_sequences_whose_rows_overlap(dev, sequences):
    """Starts that go back: no batch of the operator, but nothing is read or
    written out of place for them, and the batches after it are as ever."""
    print(f"[attend] overlap {sequences}", flush=True)
    lens = [(4, 300 + (b * 53) % 700) for b in range(sequences)]
    b = Batch(dev, lens, 4, 2, 64, 16, seed=30)
    want = b.attend()
    b.check(want)
    kept = b.starts.clone()
    b.starts = torch.where(torch.arange(sequences + 1, device=dev) % 3 == 1, kept + 7, kept)
    assert b.attend().shape == want.shape
    b.starts = kept
    assert torch.equal(b.attend(), want)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_queries_that_are_not_finite(dev, dim, form, value):
    """NaN in every column of that token and head (an infinite score less the
    largest is NaN), the bits of the others as ever."""
    lens, heads, kv_heads = FORMS[form]
    print(f"[attend] q {value} {form} {dim}", flush=True)
    b = Batch(dev, lens, heads, kv_heads, dim, 16, seed=31)
    clean = b.attend()
    bad = torch.zeros(b.q.shape[0], heads, dtype=torch.bool, device=dev)
    for s, (n, _) in enumerate(lens):
        if n:
            bad[b.at[s] + n // 2, s % heads] = True
    b.q[..., 5] = torch.where(bad, torch.tensor(value, dtype=b.q.dtype, device=dev), b.q[..., 5])
    got = b.attend()
    assert got[bad].isnan().all()
    assert torch.equal(got[~bad], clean[~bad])


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("form", FORMS)
def test_scores_of_hundreds(dev, dim, form):
    """A scale of 1.  Beside the two roundings to bf16 (2^-8 of sum p |v| and of the
    result) a score is off by what its products lose: the matrix instruction keeps
    no bit under 2^-13 of the largest of eight, so seven lose up to 2^-13 of it
    each, of either sign: for products of random size some 2^-17 of sum |q k| (one
    standard deviation of dim / 8 such groups), 2^-14 asked.  A weight changes by
    that of itself, and so does the sum they are divided by."""
    lens, heads, kv_heads = FORMS[form]
    print(f"[attend] scale 1 {form} {dim}", flush=True)
    b = Batch(dev, lens, heads, kv_heads, dim, 16, seed=32, q_size=3.0)
    got = b.attend(scale=1.0).double()
    k, v = _values(b.pool)
    for s, (n, total) in enumerate(lens):
        if not n:
            continue
        seen = _mask(n, total, True, 0, dev)
        for h in range(heads):
            q = b.q[b.at[s]:b.at[s + 1], h].double()
            kh, vh = (t[b.slots[s], h // b.group] for t in (k, v))
            score = (q @ kh.t()).masked_fill(~seen, float("-inf"))
            p = torch.softmax(score, 1)
            want, size = p @ vh, p @ vh.abs()
            lost = 2**-14 * (q.abs() @ kh.abs().t()).masked_fill(~seen, 0).amax(1, keepdim=True)
            err = (got[b.at[s]:b.at[s + 1], h] - want).abs()
            # (1e-30: weights under fp32's smallest, as in the other tests)
            assert (err <= 2**-8 * (size + want.abs()) + 2 * lost * size + 1e-30).all()
