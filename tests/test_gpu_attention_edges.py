"""Paged attention at the edges of its arguments, against the same plain
implementation in 64 bits and with the same tolerance as the rest."""
import sys

import pytest
import torch

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
