"""Paged attention at the edges of its arguments, against the same plain
implementation in 64 bits and with the same tolerance as the rest."""
import sys

import pytest
import torch

from tcfp_amd import attention as A
from test_gpu_attention import DECODE, MIXED, Batch

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
