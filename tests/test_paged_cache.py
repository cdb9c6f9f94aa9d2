"""The page lists of PagedKVCache (no GPU needed: the tensors stay on the CPU)
and what its ops refuse there."""
import pytest
import torch

from tcfp_amd import attention as A
from tcfp_amd import norm


def _cache(pages=8, page_size=16):
    return A.PagedKVCache(2, pages, 2, 64, page_size=page_size, device="cpu")


def test_a_step_describes_its_tokens():
    c = _cache()
    a, b = c.open(), c.open()
    s = c.extend([a, b], [17, 3])
    assert s.seq_lens.tolist() == [17, 3] and s.query_start.tolist() == [0, 17, 20]
    assert s.max_query_len == 17 and s.max_seq_len == 17
    assert s.slots.dtype == torch.int64 and s.page_table.dtype == torch.int32
    for row, n, at in ((0, 17, 0), (1, 3, 17)):
        pages = s.page_table[row].tolist()
        want = [pages[j // 16] * 16 + j % 16 for j in range(n)]
        assert s.slots[at:at + n].tolist() == want
    s = c.extend([b, a], [14, 0])
    assert s.seq_lens.tolist() == [17, 17] and s.query_start.tolist() == [0, 14, 14]
    pages = s.page_table[0].tolist()
    assert s.slots.tolist() == [pages[j // 16] * 16 + j % 16 for j in range(3, 17)]
    assert c.length(b) == 17 and c.free_pages == 4


def test_pages_are_given_back_and_never_shared():
    c = _cache(pages=6)
    seqs = [c.open() for _ in range(3)]
    for n in (1, 10, 7, 14):
        s = c.extend(seqs, [n] * 3)
        used = s.page_table[s.page_table >= 0].tolist()
        assert len(used) == len(set(used))
    assert c.free_pages == 0
    before = c.length(seqs[0])
    with pytest.raises(RuntimeError, match="free pages"):
        c.extend(seqs, [1, 0, 0])
    assert c.length(seqs[0]) == before
    c.close(seqs[1])
    assert c.free_pages == 2
    c.extend([seqs[0]], [1])
    assert c.free_pages == 1
    with pytest.raises(KeyError):
        c.length(seqs[1])


def test_empty_step():
    c = _cache()
    s = c.extend([], [])
    assert s.slots.shape == (0,) and s.page_table.shape == (0, 1)
    assert s.query_start.tolist() == [0]


@pytest.mark.parametrize("kw,match", [
    (dict(page_size=24), "page_size"), (dict(page_size=8), "page_size"), (dict(dim=96), "head"),
    (dict(pages=0), "at least one"), (dict(layers=0), "at least one")])
def test_refused_caches(kw, match):
    args = {"layers": 1, "pages": 1, "kv_heads": 1, "dim": 64, "device": "cpu", **kw}
    with pytest.raises(ValueError, match=match):
        A.PagedKVCache(**args)


def test_refused_steps():
    c = _cache()
    a = c.open()
    for seqs, counts in (([a], [1, 2]), ([a, a], [1, 1]), ([a], [-1])):
        with pytest.raises(ValueError, match="one count"):
            c.extend(seqs, counts)
    with pytest.raises(KeyError):
        c.extend([99], [1])


def test_cpu_tensors_are_refused():
    c = _cache()
    a = c.open()
    s = c.extend([a], [2])
    x = torch.zeros(2, 2, 64)
    with pytest.raises(RuntimeError, match="only on the GPU"):
        c.write(0, x, x, s)
    with pytest.raises(RuntimeError, match="only on the GPU"):
        c.read(0, a)
    with pytest.raises(RuntimeError, match="only on the GPU"):
        c.attend(0, x.bfloat16(), s)
    y, w = torch.zeros(2, 64), torch.ones(64)
    for f in (norm.rms_norm, norm.rms_norm_quantize):
        with pytest.raises(RuntimeError, match="only on the GPU"):
            f(y, w)
    with pytest.raises(RuntimeError, match="only on the GPU"):
        norm.rms_norm_backward(y, y, torch.ones(2), w)
