"""The paged 8-bit K/V cache and attention over it, against plain
implementations in 64 bits.

Tolerance of the attention (per element): the result's rounding to bf16 is
2^-9 of it, and weights rounded to bf16 before the second product add 2^-9 of
sum_j p_j |v_j| at most; scores in fp32 of magnitude up to some 60 are off by
60 * 2^-22, which changes a weight by 2e-5 of itself.  2^-8 of both sizes is
asked."""
import math

import pytest
import torch

from tcfp_amd import attention as A
from tcfp_amd import kernels as K

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
E4M3 = torch.float8_e4m3fn


def _pool(dev, pages, heads, page, dim, fill=0):
    codes = [torch.full((pages, heads, page, dim), fill, dtype=torch.uint8, device=dev).view(E4M3)
             for _ in range(2)]
    exps = [torch.zeros(pages, heads, page, dtype=torch.int8, device=dev) for _ in range(2)]
    return (*codes, *exps)


def _values(pool):
    """[slots, heads, dim] in 64 bits of K and V."""
    out = []
    for c, e in ((pool[0], pool[2]), (pool[1], pool[3])):
        x = c.double() * torch.exp2(e.double())[..., None]
        out.append(x.transpose(1, 2).reshape(-1, x.shape[1], x.shape[3]))
    return out


# ---------------------------------------------------------------- the cache


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("tokens,heads,page", [(1, 1, 16), (5, 3, 16), (130, 8, 64), (77, 2, 256)])
def test_cache_write_is_the_block_quantisation_of_a_head(dev, dim, dtype, tokens, heads, page):
    print(f"[cache] write {tokens} {heads} {dim} {page} {dtype}", flush=True)
    g = torch.Generator().manual_seed(0)
    pages = -(-tokens // page) + 2
    # slices of a projection's output, of values of all sizes
    qkv = torch.randn(tokens, 4 * heads * dim, generator=g)
    qkv = (qkv * torch.exp(3 * torch.randn(tokens, 1, generator=g))).to(dtype).to(dev)
    k, v = (qkv[:, i * heads * dim:(i + 1) * heads * dim].unflatten(1, (heads, dim))
            for i in (1, 3))
    slots = torch.randperm(pages * page, generator=g)[:tokens].to(dev)
    pool = _pool(dev, pages, heads, page, dim, fill=3)
    A.kv_cache_write(k, v, *pool, slots)
    for x, c, e in ((k, pool[0], pool[2]), (v, pool[1], pool[3])):
        at, off = slots // page, slots % page
        flat = x.float().reshape(tokens * heads, dim)
        if dim == 256:  # the block of a head, by the rule in 64 bits
            amax = flat.abs().amax(1).clamp(min=1e-12)
            e0 = torch.log2((amax / 448.0).double()).float().ceil()
            q0 = (flat * torch.exp2(-e0)[:, None]).clamp(-448, 448).to(E4M3)
            e0 = e0.to(torch.int8)
        else:
            q0, e0 = K.block_quantize_fp8(flat, dim)
        assert torch.equal(c.view(torch.uint8)[at, :, off].reshape(-1, dim),
                           q0.view(torch.uint8))
        assert torch.equal(e[at, :, off].flatten(), e0.flatten())
        untouched = torch.ones(pages * page, dtype=torch.bool, device=dev)
        untouched[slots] = False
        rest = c.view(torch.uint8).transpose(1, 2).reshape(pages * page, -1)[untouched]
        assert (rest == 3).all()
    for out in (F32, BF16):
        rk, rv = A.kv_cache_read(*pool, slots, out_dtype=out)
        wk, wv = (t[slots] for t in _values(pool))
        assert rk.dtype == out and torch.equal(rk.double(), wk) and torch.equal(rv.double(), wv)


def test_cache_slots_outside_the_pool_and_empty_calls(dev):
    pool = _pool(dev, 2, 2, 16, 64, fill=1)
    x = torch.randn(4, 2, 64, device=dev)
    slots = torch.tensor([-1, 5, 32, 1 << 40], device=dev)
    A.kv_cache_write(x, x, *pool, slots)
    k, v = A.kv_cache_read(*pool, slots)
    assert (k[[0, 2, 3]] == 0).all() and (v[[0, 2, 3]] == 0).all() and (k[1] != 0).any()
    flat = pool[0].view(torch.uint8).transpose(1, 2).reshape(32, -1)
    assert (flat[:5] == 1).all() and (flat[6:] == 1).all()
    A.kv_cache_write(x[:0], x[:0], *pool, slots[:0])
    assert A.kv_cache_read(*pool, slots[:0])[0].shape == (0, 2, 64)
    none = _pool(dev, 0, 2, 16, 64)
    A.kv_cache_write(x, x, *none, slots)
    assert (A.kv_cache_read(*none, slots)[0] == 0).all()


def test_cache_values_that_are_not_finite(dev):
    pool = _pool(dev, 1, 1, 16, 64)
    x = torch.randn(3, 1, 64, device=dev)
    x[0, 0, 3], x[1, 0, 5], x[2] = float("nan"), float("-inf"), 0.0
    y = x.clone()
    y[0, 0, 3], y[1, 0, 5] = 0.0, 0.0
    slots = torch.arange(3, device=dev)
    A.kv_cache_write(x, y, *pool, slots)
    k, v = A.kv_cache_read(*pool, slots, out_dtype=F32)
    bad = ~x.isfinite()
    assert k[bad].isnan().all() and torch.equal(k[~bad], v[~bad])
    assert (k[2] == 0).all()


def test_cache_of_more_than_2_gib(dev):
    """Pages whose codes lie past 2^31 bytes (2^32 from the first)."""
    heads, page, dim = 8, 64, 128
    pages = (1 << 32) // (heads * page * dim) + 3
    pool = tuple(torch.empty(s, dtype=t, device=dev) for s, t in
                 ([((pages, heads, page, dim), E4M3)] * 2 + [((pages, heads, page), torch.int8)] * 2))
    g = torch.Generator().manual_seed(1)
    n = 100
    k, v = (torch.randn(n, heads, dim, generator=g).to(dev) for _ in range(2))
    table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device=dev)
    j = torch.arange(n, device=dev)
    slots = table[0].long()[j // page] * page + j % page
    A.kv_cache_write(k, v, *pool, slots)
    rk, rv = A.kv_cache_read(*pool, slots, out_dtype=F32)
    assert ((rk - k).abs() <= 2**-4 * k.abs() + 2**-9).all()
    q = torch.randn(40, 16, dim, generator=g).bfloat16().to(dev)
    lens = torch.tensor([n], dtype=torch.int32, device=dev)
    for nq in (1, 3, 40):
        starts = torch.tensor([0, nq], dtype=torch.int32, device=dev)
        got = A.paged_attention(q[:nq], *pool, table, lens, starts, max_query_len=nq)
        for h in range(16):
            _check(got[:, h], q[:nq, h], rk[:, h // 2], rv[:, h // 2],
                   _mask(nq, n, True, 0, dev), dim**-0.5)


# -------------------------------------------------------------- attention


def _mask(nq, nk, causal, window, dev):
    pos = torch.arange(nk - nq, nk, device=dev)[:, None]
    j = torch.arange(nk, device=dev)[None]
    seen = torch.ones(nq, nk, dtype=torch.bool, device=dev)
    if causal:
        seen &= j <= pos
    if window:
        seen &= j > pos - window
    return seen


def _check(got, q, k, v, seen, scale):
    """One sequence and head: [n, dim], [n, dim], [len, dim] x 2, [n, len]."""
    q, k, v = (t.double() for t in (q, k, v))
    s = (q @ k.t()) * scale
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(1, keepdim=True) if s.shape[1] else s.new_zeros(s.shape[0], 1)
    p = torch.exp(s - top.masked_fill(top == -math.inf, 0.0))
    p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
    want, size = p @ v, p @ v.abs()
    err = (got.double() - want).abs()
    assert torch.isfinite(got.float()).all()
    bad = err > 2**-8 * (size + want.abs()) + 1e-30
    assert not bad.any(), (int(bad.sum()), float((err / (size + 1e-30)).max()))


class Batch:
    """Sequences of ``lens`` (new tokens, tokens in all) over a pool whose
    unused places hold NaN codes."""

    def __init__(self, dev, lens, heads, kv_heads, dim, page, seed=0, q_size=2.0):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.dim, self.heads, self.group = lens, dim, heads, heads // kv_heads
        need = [-(-n // page) for _, n in lens]
        pages = sum(need) + 2
        order = torch.randperm(pages, generator=g).tolist()
        self.pool = _pool(dev, pages, kv_heads, page, dim, fill=0x7F)
        self.table = torch.full((len(lens), max([*need, 1])), -1, dtype=torch.int32)
        self.slots = []
        for b, n in enumerate(need):
            self.table[b, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
            j = torch.arange(lens[b][1])
            self.slots.append((self.table[b].long()[j // page] * page + j % page).to(dev))
        self.table = self.table.to(dev)
        total = sum(n for _, n in lens)
        kv = torch.randn(2, total, kv_heads, dim, generator=g)
        kv *= torch.exp(0.5 * torch.randn(2, total, kv_heads, 1, generator=g))
        if total:
            A.kv_cache_write(*kv.to(dev), *self.pool, torch.cat(self.slots))
        starts = [0]
        for n, _ in lens:
            starts.append(starts[-1] + n)
        self.starts = torch.tensor(starts, dtype=torch.int32, device=dev)
        self.seq_lens = torch.tensor([n for _, n in lens], dtype=torch.int32, device=dev)
        self.q = (q_size * torch.randn(starts[-1], heads, dim, generator=g)).bfloat16().to(dev)
        self.at = starts

    def attend(self, **kw):
        kw = {"max_query_len": max([n for n, _ in self.lens] or [0]), **kw}
        return A.paged_attention(self.q, *self.pool, self.table, self.seq_lens, self.starts, **kw)

    def check(self, got, causal=True, window=0, scale=None):
        scale = self.dim**-0.5 if scale is None else scale
        k, v = _values(self.pool)
        assert got.shape == self.q.shape and got.dtype == BF16
        for b, (n, total) in enumerate(self.lens):
            if not n:
                continue
            rows = slice(self.at[b], self.at[b + 1])
            seen = _mask(n, total, causal, window, got.device)
            for h in range(self.heads):
                kh, vh = (t[self.slots[b], h // self.group] for t in (k, v))
                _check(got[rows, h], self.q[rows, h], kh, vh, seen, scale)


DECODE = [(1, 1), (1, 2), (1, 15), (1, 16), (1, 17), (1, 63), (1, 64), (1, 65), (1, 500),
          (1, 1025)]
MIXED = [(1, 40), (0, 33), (17, 17), (130, 300), (3, 3), (64, 64), (5, 700), (65, 129)]


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 4), (8, 2), (6, 2), (5, 1), (16, 1),
                                            (40, 1)])
def test_one_new_token(dev, dim, heads, kv_heads):
    print(f"[attend] decode {dim} {heads} {kv_heads}", flush=True)
    b = Batch(dev, DECODE, heads, kv_heads, dim, 16)
    b.check(b.attend())


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (8, 2), (3, 1), (16, 1)])
@pytest.mark.parametrize("page", [16, 64])
def test_ragged_chunks(dev, dim, heads, kv_heads, page):
    print(f"[attend] ragged {dim} {heads} {kv_heads} {page}", flush=True)
    b = Batch(dev, MIXED, heads, kv_heads, dim, page, seed=1)
    b.check(b.attend())


@pytest.mark.parametrize("lens", [[(2, 9), (2, 300)], [(4, 1000)], [(7, 64), (16, 333)],
                                  [(33, 1500)], [(256, 256)], [(300, 2000), (1, 3000)]])
@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (8, 1)])
def test_lengths(dev, lens, heads, kv_heads):
    print(f"[attend] {lens} {heads} {kv_heads}", flush=True)
    b = Batch(dev, lens, heads, kv_heads, 128, 32, seed=2)
    b.check(b.attend())


@pytest.mark.parametrize("sequences", [2, 63, 65, 300, 520])
def test_many_sequences(dev, sequences):
    """More sequences than a wave or a workgroup looks at in one go, some
    without new tokens, their keys cut into runs that span sequences."""
    print(f"[attend] {sequences} sequences", flush=True)
    for new in (1, 3):
        lens = [(new if b % 7 else 0, 1 + (b * 37) % 290) for b in range(sequences)]
        lens = [(n, max(n, total)) for n, total in lens]
        b = Batch(dev, lens, 4, 2, 64, 16, seed=14)
        b.check(b.attend())
        b.check(b.attend(max_seq_len=40))
    lens = [(40, 40 + b % 11) if b % 5 else (1, 9) for b in range(min(sequences, 100))]
    b = Batch(dev, lens, 4, 2, 64, 16, seed=15)
    b.check(b.attend())


@pytest.mark.parametrize("heads,kv_heads", [(6, 2), (5, 1), (8, 8)])
@pytest.mark.parametrize("sequences", [60, 250])
def test_many_rows_of_split_items(dev, heads, kv_heads, sequences):
    """So many rows that one wave each joins their parts, in numbers of heads
    that fill its workgroups and that do not."""
    print(f"[attend] {sequences} x {heads}", flush=True)
    new = 4 if sequences == 60 else 1
    lens = [(new if b % 9 else 0, 300 + (b * 53) % 700) for b in range(sequences)]
    b = Batch(dev, lens, heads, kv_heads, 128, 16, seed=19)
    b.check(b.attend())


def test_heads_of_256_in_few_and_many_rows(dev):
    """More than 16 rows of an item, and more than 1024 rows of split items."""
    for lens, heads, kv_heads in (([(1, 700), (1, 3), (1, 2050)], 24, 1), ([(5, 900)], 20, 4),
                                  ([(2, 600 + 7 * i) for i in range(70)], 8, 2)):
        print(f"[attend] 256 {len(lens)} {heads} {kv_heads}", flush=True)
        b = Batch(dev, lens, heads, kv_heads, 256, 16, seed=22)
        b.check(b.attend())
        b.check(b.attend(window=100), window=100)


def test_long_sequences(dev):
    """Keys cut into more runs than the card has places for, and a window."""
    for lens, heads in (([(1, 40000)], 4), ([(2, 30000), (1, 5), (1, 9000)], 8),
                        ([(70, 20000)], 2)):
        print(f"[attend] {lens}", flush=True)
        b = Batch(dev, lens, heads, 1, 64, 64, seed=16)
        b.check(b.attend())
        b.check(b.attend(window=7000), window=7000)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,kv_heads", [(3, 3), (6, 2), (16, 2)])
@pytest.mark.parametrize("window", [0, 900])
def test_prompts_whose_keys_are_split(dev, dim, heads, kv_heads, window):
    """Long contexts in front of few tiles of rows, beside sequences that do
    not reach the second run of keys and rows that a hole leaves with none of
    a run."""
    lens = [(90, 6000), (40, 40), (1, 3000), (57, 4097)]
    print(f"[attend] split {dim} {heads} {kv_heads} {window}", flush=True)
    b = Batch(dev, lens, heads, kv_heads, dim, 32, seed=18)
    b.check(b.attend(window=window), window=window)
    b.check(b.attend(causal=False, window=window), False, window)
    b.table[0, 10:160] = -1  # keys 320 ... 5119
    got = b.attend(window=window)
    k, v = _values(b.pool)
    seen = _mask(90, 6000, True, window, dev)
    seen[:, 320:5120] = False
    group = heads // kv_heads
    for h in range(heads):
        kh, vh = (t[b.slots[0], h // group] for t in (k, v))
        _check(got[:90, h], b.q[:90, h], kh, vh, seen, dim**-0.5)


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64), (256, 32)])
@pytest.mark.parametrize("lens,heads,kv_heads", [([(1100, 1100)], 8, 8), ([(300, 460)], 6, 2), ([(900, 1000)], 32, 8),
                                                 ([(700, 700), (0, 30), (1, 40), (511, 513)], 9, 9)])
def test_long_prompts_of_few_tiles(dev, dim, page, lens, heads, kv_heads):
    """Tiles whose steps two groups of waves share, with a window, a hole and
    keys that only one of the groups sees."""
    print(f"[attend] {lens} {heads} {kv_heads} {dim}", flush=True)
    b = Batch(dev, lens, heads, kv_heads, dim, page, seed=20)
    b.check(b.attend())
    for window in (1, 65, 600):
        b.check(b.attend(window=window), window=window)
    b.check(b.attend(causal=False), False)
    n, total = lens[0]
    hole = slice(64 // page, 448 // page)
    b.table[0, hole] = -1
    got = b.attend()
    k, v = _values(b.pool)
    seen = _mask(n, total, True, 0, dev)
    seen[:, 64:448] = False
    for h in range(heads):
        kh, vh = (t[b.slots[0], h // (heads // kv_heads)] for t in (k, v))
        _check(got[:n, h], b.q[:n, h], kh, vh, seen, dim**-0.5)


@pytest.mark.parametrize("dim,heads", [(64, 24), (128, 24), (256, 10)])
def test_nan_in_long_prompts_of_few_tiles(dev, dim, heads):
    """A NaN of a cached key or value reaches the rows and heads that see it
    and no other."""
    n, page = 700, 16
    b = Batch(dev, [(n, n)], heads, heads // 2, dim, page, seed=21)
    want = b.attend()
    b.check(want)
    for which in (0, 1):
        for at in (650, 130, 3):
            codes = b.pool[which].view(torch.uint8)
            slot = int(b.slots[0][at])
            keep = codes[slot // page, :, slot % page].clone()
            codes[slot // page, 0, slot % page, 7] = 0x7F
            got = b.attend()
            codes[slot // page, :, slot % page] = keep
            assert torch.equal(got[:at], want[:at]) and torch.equal(got[:, 2:], want[:, 2:])
            assert got[at:, :2, 7].float().isnan().all()


@pytest.mark.parametrize("page", [16, 32, 128, 256, 1024])
def test_page_sizes(dev, page):
    b = Batch(dev, [(1, 5), (1, 700), (1, 1500)], 8, 2, 64, page, seed=3)
    b.check(b.attend())
    b = Batch(dev, [(20, 1100), (70, 90)], 4, 2, 64, page, seed=3)
    b.check(b.attend())


@pytest.mark.parametrize("causal,window", [(True, 1), (True, 7), (True, 64), (True, 1000),
                                           (False, 0), (False, 20)])
@pytest.mark.parametrize("lens", [DECODE, MIXED])
def test_masks(dev, causal, window, lens):
    print(f"[attend] mask {causal} {window}", flush=True)
    b = Batch(dev, lens, 6, 2, 64, 16, seed=4)
    b.check(b.attend(causal=causal, window=window), causal, window)


def test_scale_and_large_scores(dev):
    """Scores far apart: all the weight on a few keys."""
    b = Batch(dev, MIXED + DECODE, 4, 2, 128, 16, seed=5, q_size=8.0)
    b.check(b.attend())
    b.check(b.attend(scale=0.01), scale=0.01)
    b.check(b.attend(scale=-0.05), scale=-0.05)
    assert torch.isfinite(b.attend(scale=0.0).float()).all()


@pytest.mark.parametrize("bound", [1, 100, 5000])
def test_bounds_that_do_not_fit(dev, bound):
    """max_query_len and max_seq_len size the launch; lengths past them are
    answered all the same."""
    b = Batch(dev, MIXED + DECODE, 4, 2, 64, 16, seed=6)
    want = b.attend()
    b.check(b.attend(max_query_len=bound, max_seq_len=bound))
    b.check(b.attend(max_seq_len=bound))
    b.check(want)


def test_rows_that_see_nothing(dev):
    """Sequences without tokens, more new tokens than tokens, rows of q that
    belong to no sequence: zeros, and the others as ever."""
    for nq in (1, 4, 60):
        b = Batch(dev, [(nq, 100), (nq, 90)], 4, 2, 64, 16, seed=7)
        want = b.attend()
        b.check(want)
        b.seq_lens = torch.tensor([0, 90], dtype=torch.int32, device=dev)
        got = b.attend()
        assert (got[:nq] == 0).all() and torch.equal(got[nq:], want[nq:])
        if nq > 2:
            b.seq_lens = torch.tensor([nq - 2, 90], dtype=torch.int32, device=dev)
            got = b.attend()
            assert (got[:2] == 0).all() and (got[2:nq] != 0).any()
            assert torch.equal(got[nq:], want[nq:])
            got = b.attend(causal=False, window=1)
            assert (got[:2] != 0).any()
        more = torch.cat([b.q, b.q])
        got = A.paged_attention(more, *b.pool, b.table, b.seq_lens, b.starts, max_query_len=nq)
        assert (got[2 * nq:] == 0).all() and torch.equal(got[nq:2 * nq], want[nq:])


def test_pages_that_were_given_up(dev):
    """Pages outside the pool are not seen; with a window that does not reach
    them nothing changes."""
    for nq in (1, 5, 40):
        b = Batch(dev, [(nq, 400)], 4, 2, 64, 16, seed=8)
        want = b.attend(window=64)
        kept = b.table.clone()
        b.table[0, :10] = torch.tensor([-1, 10**6] * 5, dtype=torch.int32, device=dev)
        assert torch.equal(b.attend(window=64), want)
        # without the window: the first 160 keys are not there
        k, v = _values(b.pool)
        seen = _mask(nq, 400, True, 0, dev)[:, 160:]
        got = b.attend()
        for h in range(4):
            kh, vh = (t[b.slots[0][160:], h // 2] for t in (k, v))
            _check(got[:, h], b.q[:, h], kh, vh, seen, 64**-0.5)
        b.table[:] = -1
        assert (b.attend() == 0).all()
        b.table = kept[:, :3].contiguous()  # a table that ends before the sequence
        got = b.attend()
        seen = _mask(nq, 400, True, 0, dev)[:, :48]
        for h in range(4):
            kh, vh = (t[b.slots[0][:48], h // 2] for t in (k, v))
            _check(got[:, h], b.q[:, h], kh, vh, seen, 64**-0.5)


def test_nan_in_masked_places(dev):
    """A key or value that is not finite reaches the tokens that see it and no
    other."""
    for nq, at in ((30, 380), (3, 398), (100, 330)):
        b = Batch(dev, [(nq, 400)], 4, 2, 64, 16, seed=9)
        want = b.attend()
        for which in (0, 1):
            codes = b.pool[which].view(torch.uint8)
            slot = int(b.slots[0][at])
            keep = codes[slot // 16, :, slot % 16].clone()
            codes[slot // 16, 0, slot % 16, 5] = 0x7F
            got = b.attend()
            first = at - (400 - nq)  # the first new token that sees it
            assert torch.equal(got[:first], want[:first])
            assert torch.equal(got[:, 2:], want[:, 2:])
            seeing = got[first:, :2].float().isnan()
            assert seeing[..., 5].all() and (which == 1 or seeing.all())
            # and with a window that has passed it
            got = b.attend(window=8)
            codes[slot // 16, :, slot % 16] = keep
            ref = b.attend(window=8)
            assert torch.equal(got[first + 8:], ref[first + 8:])
            assert torch.equal(got[:first], ref[:first])


@pytest.mark.parametrize("dim,window", [(64, 0), (64, 300), (128, 0), (128, 300)])
def test_nan_and_missing_pages_among_many_rows(dev, dim, window):
    """The same two among more rows than a small tile has, in front of long
    contexts (the eight-wave kernel)."""
    nq, total, page = 200, 1000, 16
    b = Batch(dev, [(nq, total), (150, 700)], 4, 2, dim, page, seed=17)
    want = b.attend(window=window)
    b.check(want, window=window)
    for which in (0, 1):
        for at in (total - 150, 500, 3):
            codes = b.pool[which].view(torch.uint8)
            slot = int(b.slots[0][at])
            keep = codes[slot // page, :, slot % page].clone()
            codes[slot // page, 0, slot % page, 7] = 0x7F
            got = b.attend(window=window)
            codes[slot // page, :, slot % page] = keep
            pos = torch.arange(total - nq, total, device=dev)
            sees = pos >= at
            if window:
                sees &= pos < at + window
            assert torch.equal(got[:nq][~sees], want[:nq][~sees])
            assert torch.equal(got[:, 2:], want[:, 2:]) and torch.equal(got[nq:], want[nq:])
            assert got[:nq][sees][:, :2, 7].float().isnan().all()
    b.table[0, :40] = -1  # the first 640 keys
    got = b.attend(window=window)
    assert torch.equal(got[nq:], want[nq:])
    k, v = _values(b.pool)
    seen = _mask(nq, total, True, window, dev)[:, 640:]
    for h in range(4):
        kh, vh = (t[b.slots[0][640:], h // 2] for t in (k, v))
        _check(got[:nq, h], b.q[:nq, h], kh, vh, seen, dim**-0.5)
    b.table[0, 50] = 10**6  # and a hole inside
    got = b.attend(window=window)
    keep = torch.ones(total - 640, dtype=torch.bool, device=dev)
    keep[160:176] = False
    for h in range(4):
        kh, vh = (t[b.slots[0][640:], h // 2] for t in (k, v))
        _check(got[:nq, h], b.q[:nq, h], kh, vh, seen & keep, dim**-0.5)


def test_strides(dev):
    """Queries as a slice of the QKV projection, the page table as a slice."""
    b = Batch(dev, MIXED + DECODE, 6, 2, 64, 16, seed=10)
    want = b.attend()
    wide = torch.randn(b.q.shape[0], 10 * 64, device=dev).bfloat16()
    wide[:, 64:64 * 7] = b.q.flatten(1)
    b.q = wide[:, 64:64 * 7].unflatten(1, (6, 64))
    table = torch.full((b.table.shape[0], b.table.shape[1] + 5), -1, dtype=torch.int32, device=dev)
    table[:, :b.table.shape[1]] = b.table
    b.table = table[:, :b.table.shape[1]]
    assert torch.equal(b.attend(), want)
    odd = torch.zeros(b.q.shape[0], 6, 65, dtype=BF16, device=dev)
    odd[..., 1:] = b.q
    b.q = odd[..., 1:]
    assert torch.equal(b.attend(), want)
    b.q = want.transpose(0, 1).contiguous().transpose(0, 1)  # heads outermost
    b.check(b.attend())


def test_empty_calls(dev):
    b = Batch(dev, [(0, 5), (0, 0)], 4, 2, 64, 16)
    assert b.attend().shape == (0, 4, 64)
    q = torch.zeros(0, 4, 64, dtype=BF16, device=dev)
    i = torch.zeros(1, dtype=torch.int32, device=dev)
    out = A.paged_attention(q, *b.pool, b.table[:0], i[:0], i, max_query_len=0)
    assert out.shape == (0, 4, 64)


def test_same_bits_each_time_and_on_another_stream(dev):
    for lens in (DECODE, MIXED, [(1, 6000)], [(9, 4000)]):
        b = Batch(dev, lens, 8, 2, 128, 16, seed=11)
        want = b.attend()
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            got = [b.attend() for _ in range(3)]
        torch.cuda.synchronize()
        for x in got:
            assert torch.equal(x, want)


def test_graph_whose_sequences_grow(dev):
    """A captured write and attention, replayed as the lengths on the device
    grow, against the eager result of every step."""
    heads, kv_heads, dim, page, steps = 8, 2, 64, 16, 6
    b = Batch(dev, [(1, 30 + steps), (1, 500 + steps)], heads, kv_heads, dim, page, seed=12)
    full = b.seq_lens.clone()
    g = torch.Generator().manual_seed(13)
    qkv = torch.zeros(2, (heads + 2 * kv_heads) * dim, dtype=BF16, device=dev)
    lens, slots = full.clone(), torch.full((2,), -1, dtype=torch.int64, device=dev)
    q, k, v = (t.unflatten(1, (-1, dim)) for t in
               qkv.split([heads * dim, kv_heads * dim, kv_heads * dim], 1))

    def step(pool):
        A.kv_cache_write(k, v, *pool, slots)
        return A.paged_attention(q, *pool, b.table, lens, b.starts, max_query_len=1)

    eager = tuple(t.clone() for t in b.pool)
    step(b.pool)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(b.pool)
    for i in range(steps):
        qkv.copy_(torch.randn(qkv.shape, generator=g).bfloat16())
        lens.copy_(full - steps + i + 1)
        at = (lens - 1).long()
        slots.copy_(b.table.long().gather(1, (at // page)[:, None])[:, 0] * page + at % page)
        graph.replay()
        want = step(eager)
        torch.cuda.synchronize()
        assert torch.equal(out, want), i


def test_refusals(dev):
    b = Batch(dev, [(3, 20)], 4, 2, 64, 16)
    kc, vc, ke, ve = b.pool
    x = torch.zeros(2, 2, 64, device=dev)
    s = torch.arange(2, device=dev)
    with pytest.raises(RuntimeError, match="only on the GPU"):
        A.kv_cache_write(x.cpu(), x, *b.pool, s)
    with pytest.raises(TypeError, match="slots must be torch.int64"):
        A.kv_cache_write(x, x, *b.pool, s.int())
    with pytest.raises(ValueError, match="slots must have shape"):
        A.kv_cache_write(x, x, *b.pool, s[:1])
    with pytest.raises(ValueError, match="k must have shape"):
        A.kv_cache_write(x[:, :1], x, *b.pool, s)
    with pytest.raises(TypeError, match="one dtype"):
        A.kv_cache_write(x, x.bfloat16(), *b.pool, s)
    with pytest.raises(ValueError, match="tokens"):
        A.kv_cache_write(x, x[:1], *b.pool, s)
    with pytest.raises(TypeError, match="unsupported input dtype"):
        A.kv_cache_write(x.half(), x.half(), *b.pool, s)
    with pytest.raises(TypeError, match="cache codes"):
        A.kv_cache_read(kc.view(torch.uint8), vc, ke, ve, s)
    with pytest.raises(TypeError, match="cache exponents"):
        A.kv_cache_read(kc, vc, ke.view(torch.uint8), ve, s)
    with pytest.raises(ValueError, match="one shape"):
        A.kv_cache_read(kc, vc[:1], ke, ve, s)
    with pytest.raises(ValueError, match="exponents must have shape"):
        A.kv_cache_read(kc, vc, ke[:1], ve, s)
    with pytest.raises(ValueError, match="contiguous"):
        A.kv_cache_read(kc.transpose(1, 2).contiguous().transpose(1, 2), vc, ke, ve, s)
    with pytest.raises(ValueError, match="head dimension"):
        A.kv_cache_read(*_pool(dev, 1, 1, 16, 96), s)
    with pytest.raises(ValueError, match="page_size"):
        A.kv_cache_read(*_pool(dev, 1, 1, 24, 64), s)
    with pytest.raises(ValueError, match="page_size"):
        A.kv_cache_read(*_pool(dev, 1, 1, 8, 64), s)
    with pytest.raises(TypeError, match="unsupported output dtype"):
        A.kv_cache_read(*b.pool, s, out_dtype=torch.float16)
    args = (b.q, *b.pool, b.table, b.seq_lens, b.starts)

    def attend(i=None, v=None, **kw):
        a = list(args)
        if i is not None:
            a[i] = v
        return A.paged_attention(*a, **{"max_query_len": 3, **kw})

    with pytest.raises(TypeError, match="q must be torch.bfloat16"):
        attend(0, b.q.float())
    with pytest.raises(ValueError, match="q must have shape"):
        attend(0, b.q[..., :32])
    with pytest.raises(ValueError, match="multiple of the cache's"):
        attend(0, b.q[:, :3])
    with pytest.raises(TypeError, match="page_table must be torch.int32"):
        attend(5, b.table.long())
    with pytest.raises(ValueError, match="page_table must be 2-D"):
        attend(5, b.table[0])
    with pytest.raises(ValueError, match="seq_lens must have shape"):
        attend(6, b.starts)
    with pytest.raises(ValueError, match="query_start must have shape"):
        attend(7, b.seq_lens)
    with pytest.raises(RuntimeError, match="only on the GPU"):
        attend(7, b.starts.cpu())
    with pytest.raises(ValueError, match="window"):
        attend(window=-1)
    with pytest.raises(ValueError, match="negative"):
        attend(max_query_len=-1)
