"""How many sequences and heads packed attention takes, at the C entry (no GPU needed:
what is refused is refused before anything is launched)."""
import pytest

from test_training_ops import packed_call, status, PTR


@pytest.mark.parametrize("batch,heads,kv", [
    (65535, 257, 257), (65535, 512, 8), (32768, 512, 512), (65535, 65535, 1)])
def test_past_a_grid(batch, heads, kv):
    shape = status("tcfp_scale_bf16", PTR, 7, PTR, 0, PTR, None)
    # (with no tokens nothing is launched; what the sizes allow is answered)
    assert packed_call(batch=batch, heads=heads, kv=kv, tokens=0) == shape
    assert packed_call(batch=batch, heads=heads, kv=kv) == shape


@pytest.mark.parametrize("batch,heads,kv", [
    (65535, 256, 256), (65535, 256, 32), (32767, 512, 512), (1, 65535, 1), (255, 65535, 65535)])
def test_up_to_it(batch, heads, kv):
    assert packed_call(batch=batch, heads=heads, kv=kv, tokens=0) == "ok"
