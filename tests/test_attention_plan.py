"""The attention's launch plan, through the size of its workspace (host code: no
GPU needed)."""
import pytest

from tcfp_amd import _hip

HUGE = (1 << 30, 1 << 40, 2**62, 2**63 - 200, 2**63 - 1)
# tokens, heads, K/V heads, columns, sequences, max_query_len, max_seq_len
BATCHES = [(4, 8, 2, 128, 4, 1, 8192), (4, 8, 2, 64, 4, 1, 200), (100, 8, 2, 128, 4, 25, 8192),
           (300, 4, 4, 64, 2, 200, 9000), (64, 6, 1, 256, 1, 64, 4000),
           (2048, 8, 8, 128, 1, 2048, 2048)]


def _bytes(*args):
    return _hip.load_library().tcfp_paged_attention_workspace_bytes(*args)


@pytest.mark.parametrize("batch", BATCHES)
def test_a_window_past_every_key_is_none(batch):
    want = _bytes(*batch, 0)
    for window in HUGE:
        assert _bytes(*batch, window) == want


@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("window", [0, 500])
def test_bounds_past_every_length(batch, window):
    tokens, heads, kv_heads, dim, sequences, _, longest = batch
    want = _bytes(tokens, heads, kv_heads, dim, sequences, 1 << 30, longest, window)
    for bound in HUGE:
        assert _bytes(tokens, heads, kv_heads, dim, sequences, bound, longest, window) == want
    want = _bytes(tokens, heads, kv_heads, dim, sequences, 7, 1 << 30, window)
    for bound in HUGE:
        assert _bytes(tokens, heads, kv_heads, dim, sequences, 7, bound, window) == want
