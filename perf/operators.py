"""What the speed of the decoder operators is measured on.

The operators that stand between the linear layers of a decoder which is
trained and served with FP8 codes:

* ``norm``  -- residual addition and root-mean-square norm whose output is
  E4M3 codes with block scales, as the block dual GEMM reads them (forward),
  and the gradients of its input and weight (``norm_grad``).
* ``write`` / ``read`` -- the K/V cache: new keys and values quantised as they
  are written into the pages of their sequences (E4M3 codes, one power-of-two
  exponent per token and head), and cached tokens read back.
* ``attend`` -- attention of a chunk of new tokens of every sequence of a
  batch (one token when generating, a prompt or a part of one otherwise) over
  the paged cache, causal, heads in groups that share a K/V head.

The plain forms are elementary torch operations in fp32, rounded once at the
end.  Block scales are measured in the fp32-multiplier format (448 / amax):
the power-of-two exponents are whole numbers, which the last bit of a sum of
squares flips where an amax lies on a binade's edge; both formats are the same
work.  Cache exponents depend on no sum and are compared as they are.

Sizes: d_model 4096 with 8192 tokens and the small transformer's heads (4 of
64) are the repository's own; the others are generic.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_E4M3 = torch.float8_e4m3fn
_MAX = 448.0
_EPS = 1e-6
_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp32": 4}


def _norm(kind, tokens, d, dtype, residual, block, name=None):
    c = {"kind": kind, "tokens": tokens, "d": d, "dtype": dtype, "residual": residual,
         "block": block}
    return c if name is None else {"name": name, **c}


def _cache(kind, tokens, kv_heads, dim, page, dtype, name=None):
    c = {"kind": kind, "tokens": tokens, "kv_heads": kv_heads, "dim": dim, "page": page,
         "dtype": dtype}
    return c if name is None else {"name": name, **c}


def _attend(batch, new, context, heads, kv_heads, dim, page, window=0, name=None):
    c = {"kind": "attend", "batch": batch, "new": new, "context": context, "heads": heads,
         "kv_heads": kv_heads, "dim": dim, "page": page, "window": window}
    return c if name is None else {"name": name, **c}


def listed():
    return [
        # one generated token in front of a 4096-wide layer: latency only
        _norm("norm", 1, 4096, "bf16", True, 64, name="norm-1"),
        # a training or prompt batch of 8192 tokens, residual stream in bf16
        _norm("norm", 8192, 4096, "bf16", True, 64, name="norm-8192"),
        # a short last batch in fp32 without a residual (a model's first
        # norm), a width that is no power of two
        _norm("norm", 1000, 1056, "fp32", False, 32, name="norm-1000"),
        # the backward pass of the training batch, the residual's gradient added
        _norm("norm_grad", 8192, 4096, "bf16", True, 64, name="norm-grad-8192"),
        # the backward pass of the short batch
        _norm("norm_grad", 1000, 1056, "fp32", False, 32, name="norm-grad-1000"),
        # 64 sequences generating: one token each into the cache
        _cache("write", 64, 8, 128, 64, "bf16", name="write-64"),
        # a batch of prompts into the cache, keys and values as the block
        # GEMM's fp32 output holds them
        _cache("write", 8000, 8, 128, 64, "fp32", name="write-8000"),
        # cached sequences read back, to move them or attend to them elsewhere
        _cache("read", 30011, 8, 128, 16, "bf16", name="read-30011"),
        # one sequence generating on the small transformer: the smallest call
        _attend(1, 1, 127, 4, 4, 64, 16, name="attend-1"),
        # 64 sequences of up to 8192 tokens generating: the cache is read once
        _attend(64, 1, 8191, 32, 8, 128, 64, name="attend-64"),
        # ragged prompts of up to 1000 tokens, nothing cached before them
        _attend(6, 1000, 0, 16, 16, 64, 32, name="attend-prompt-1000"),
        # chunks of 2048 tokens of two long prompts, up to 14336 tokens cached
        # before: the largest
        _attend(2, 2048, 14336, 32, 8, 128, 64, name="attend-chunk-2048"),
    ]


def _log(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def _int(rng, lo, hi):
    return int(round(_log(rng, lo, hi)))


def draw(rng):
    kind = rng.choice(["norm", "norm_grad", "write", "read", "attend", "attend", "attend"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if kind in ("norm", "norm_grad"):
        block = rng.choice([32, 64, 128])
        d = block * max(1, int(round(_log(rng, 256, 8192) / block)))
        return _norm(kind, _int(rng, 1, 4096), d, dtype, rng.random() < 0.7, block)
    page = rng.choice([16, 32, 64, 128])
    dim = rng.choice([64, 128, 128, 256])
    if kind in ("write", "read"):
        return _cache(kind, _int(rng, 1, 16384), rng.choice([1, 2, 4, 8]), dim, page, dtype)
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 8])
    window = rng.choice([0, 0, 0, _int(rng, 64, 2048)])
    how = rng.random()
    if how < 0.5:  # generating
        batch, new, context = _int(rng, 1, 64), 1, _int(rng, 16, 8192)
    elif how < 0.65:  # a few tokens at a time (drafts to be checked)
        batch, new, context = _int(rng, 1, 16), rng.randint(2, 16), _int(rng, 64, 8192)
    else:  # prompts, or chunks of them
        batch, new = _int(rng, 1, 4), _int(rng, 17, 2048)
        context = rng.choice([0, _int(rng, 64, 8192)])
    return _attend(batch, new, context, heads, kv_heads, dim, page, window)


def _lengths(case):
    """(new tokens, tokens in the cache with them) of each sequence: the first
    has the case's sizes, the others between a quarter of them and all."""
    rng = random.Random(case["batch"] * 1000003 + case["new"] * 1009 + case["context"])
    got = []
    for b in range(case["batch"]):
        f = 1.0 if b == 0 else rng.uniform(0.25, 1.0)
        n = case["new"] if case["new"] <= 16 else max(1, int(case["new"] * f))
        got.append((n, n + int(case["context"] * f)))
    return got


# ---------------------------------------------------------------- the inputs


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=gen, device="cuda").to(dtype)

    kind = case["kind"]
    s = {"case": case}
    if kind in ("norm", "norm_grad"):
        m, d, dt = case["tokens"], case["d"], _DT[case["dtype"]]
        # a residual stream: some channels are far larger than the others
        chan = torch.exp(0.5 * torch.randn(d, generator=gen, device="cuda"))
        s["x"] = (randn(m, d) * chan).to(dt)
        s["r"] = (randn(m, d) * chan).to(dt) if case["residual"] else None
        s["w"] = 1.0 + 0.1 * randn(d)
        if kind == "norm_grad":
            # what the forward kept: the sum in its own type, and 1 / rms
            s["h"] = s.pop("x")
            hf = s["h"].float()
            s["rstd"] = torch.rsqrt((hf * hf).mean(-1) + _EPS)
            s["gy"] = (randn(m, d) * 1e-3).to(dt)
            s["gh"] = (s.pop("r").float() * 1e-3).to(dt) if case["residual"] else None
        return s
    hkv, dim, page = case["kv_heads"], case["dim"], case["page"]
    if kind == "write":
        t, dt = case["tokens"], _DT[case["dtype"]]
        pages = -(-t // page) + 3
        s["pool"] = _pool(pages, hkv, page, dim, None)
        # K and V as the QKV projection leaves them: slices of one matrix
        kv = randn(t, (2 + 2) * hkv * dim, dtype=dt)
        s["k"] = kv[:, 2 * hkv * dim:3 * hkv * dim].unflatten(1, (hkv, dim))
        s["v"] = kv[:, 3 * hkv * dim:].unflatten(1, (hkv, dim))
        s["slots"] = _slots(t, pages, page, gen)
        return s
    if kind == "read":
        t = case["tokens"]
        pages = -(-t // page) + 3
        s["pool"] = _pool(pages, hkv, page, dim, gen)
        s["slots"] = _slots(t, pages, page, gen)
        return s
    lens = _lengths(case)
    need = [-(-total // page) for _, total in lens]
    pages = sum(need) + 2
    s["pool"] = _pool(pages, hkv, page, dim, gen)
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros(len(lens), max(need), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    starts = [0]
    for n, _ in lens:
        starts.append(starts[-1] + n)
    s["table"] = table
    s["seq_lens"] = torch.tensor([total for _, total in lens], dtype=torch.int32, device="cuda")
    s["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    s["max_new"] = max(n for n, _ in lens)
    s["max_len"] = max(total for _, total in lens)
    hq = case["heads"]
    # the queries are a slice of the QKV projection's output too; scores of
    # a trained model are spread wider than those of unit vectors
    qkv = randn(starts[-1], (hq + 2 * hkv) * dim, dtype=torch.float32) * 2.0
    s["q"] = qkv.to(torch.bfloat16)[:, :hq * dim].unflatten(1, (hq, dim))
    return s


def _pool(pages, hkv, page, dim, gen):
    """(k_codes, v_codes, k_exps, v_exps) of a cache, empty or of random keys
    and values of varying size."""
    made = []
    for _ in range(2):
        if gen is None:
            codes = torch.zeros(pages, hkv, page, dim, dtype=torch.uint8, device="cuda").view(_E4M3)
            exps = torch.zeros(pages, hkv, page, dtype=torch.int8, device="cuda")
        else:
            x = torch.randn(pages, hkv, page, dim, generator=gen, device="cuda")
            x *= torch.exp(0.3 * torch.randn(pages, hkv, page, 1, generator=gen, device="cuda"))
            codes, exps = _quantise(x)
            del x
        made.append((codes, exps))
    (kc, ke), (vc, ve) = made
    return kc, vc, ke, ve


def _slots(tokens, pages, page, gen):
    """Places of `tokens` tokens, in pages of any order."""
    n = -(-tokens // page)
    at = torch.randperm(pages, generator=gen, device="cuda")[:n]
    slots = at[:, None] * page + torch.arange(page, device="cuda")
    return slots.reshape(-1)[:tokens].contiguous()


# ----------------------------------------------------------- the plain forms


def _quantise(x):
    """E4M3 codes of the last axis and its power-of-two exponents."""
    ratio = x.abs().amax(-1).clamp(min=1e-12) / _MAX
    # the logarithm correctly rounded to fp32: taken in 64 bits
    e = torch.log2(ratio.double()).float().ceil().clamp(min=-126.0)
    codes = (x * torch.exp2(-e)[..., None]).clamp(-_MAX, _MAX).to(_E4M3)
    return codes, e.to(torch.int8)


def _plain_norm(s):
    c = s["case"]
    x = s["x"].float()
    if s["r"] is not None:
        x = x + s["r"].float()
    rstd = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
    y = (x * rstd * s["w"]).unflatten(1, (-1, c["block"]))
    mul = y.abs().amax(-1).clamp(min=1e-12).reciprocal() * _MAX
    codes = (y * mul[..., None]).clamp(-_MAX, _MAX).to(_E4M3).flatten(1)
    h = x.to(s["x"].dtype) if s["r"] is not None else s["x"]
    return {"codes": codes, "scales": (1.0 / mul).t().contiguous(), "h": h,
            "rstd": rstd.flatten()}


def _plain_norm_grad(s):
    gy, xh = s["gy"].float(), s["h"].float() * s["rstd"][:, None]
    g = gy * s["w"]
    dx = s["rstd"][:, None] * (g - xh * (g * xh).mean(-1, keepdim=True))
    if s["gh"] is not None:
        dx = dx + s["gh"].float()
    return {"dx": dx.to(s["h"].dtype), "dw": (gy * xh).sum(0)}


def _plain_write(s):
    page = s["case"]["page"]
    kc, vc, ke, ve = s["pool"]
    at, off = s["slots"] // page, s["slots"] % page
    for x, codes, exps in ((s["k"], kc, ke), (s["v"], vc, ve)):
        q, e = _quantise(x.float())
        codes.view(torch.uint8)[at, :, off] = q.view(torch.uint8)
        exps[at, :, off] = e
    return {"k": kc, "v": vc, "k_exps": ke, "v_exps": ve}


def _gather(codes, exps, at, off, dtype):
    x = codes.view(torch.uint8)[at, :, off].view(_E4M3).to(dtype)
    return x * torch.exp2(exps[at, :, off].to(dtype))[..., None]


def _plain_read(s):
    page, dt = s["case"]["page"], _DT[s["case"]["dtype"]]
    kc, vc, ke, ve = s["pool"]
    at, off = s["slots"] // page, s["slots"] % page
    return {"k": _gather(kc, ke, at, off, torch.float32).to(dt),
            "v": _gather(vc, ve, at, off, torch.float32).to(dt)}


def _visible(s, new, total):
    """[batch, max new, max length]: which keys a query sees."""
    w = s["case"]["window"]
    i = torch.arange(s["max_new"], device="cuda")[None, :, None]
    j = torch.arange(s["max_len"], device="cuda")[None, None, :]
    pos = (total - new)[:, None, None] + i
    seen = (j <= pos) & (j < total[:, None, None]) & (i < new[:, None, None])
    return seen & (j > pos - w) if w else seen


def _plain_attend(s):
    c = s["case"]
    hq, hkv, dim, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    group, nb, nq, nk = hq // hkv, c["batch"], s["max_new"], s["max_len"]
    kc, vc, ke, ve = s["pool"]
    new, total = s["starts"].diff(), s["seq_lens"]
    j = torch.arange(nk, device="cuda")
    at, off = s["table"][:, j // page].long(), (j % page).expand(nb, nk)
    k = _gather(kc, ke, at, off, torch.float32).permute(0, 2, 3, 1).contiguous()
    v = _gather(vc, ve, at, off, torch.float32).permute(0, 2, 1, 3).contiguous()
    rows = s["starts"][:-1, None] + torch.arange(nq, device="cuda")
    q = s["q"].float()[rows.clamp(max=s["q"].shape[0] - 1).long()]
    q = q.view(nb, nq, hkv, group, dim).permute(0, 2, 3, 1, 4).reshape(nb, hkv, group * nq, dim)
    p = torch.matmul(q, k).mul_(dim**-0.5).view(nb, hkv, group, nq, nk)
    p.masked_fill_(~_visible(s, new, total)[:, None, None], float("-inf"))
    top = p.amax(-1, keepdim=True)
    p = p.sub_(top.masked_fill_(top == float("-inf"), 0.0)).exp_()
    total_p = p.sum(-1).clamp_(min=1e-30)
    o = torch.matmul(p.view(nb, hkv, group * nq, nk), v).view(nb, hkv, group, nq, dim)
    o = (o / total_p[..., None]).permute(0, 3, 1, 2, 4).reshape(nb * nq, hq, dim)
    t = torch.arange(s["q"].shape[0], device="cuda")
    b = torch.searchsorted(s["starts"], t, right=True) - 1
    return o[b * nq + t - s["starts"][b]].to(s["q"].dtype)


_PLAIN = {"norm": _plain_norm, "norm_grad": _plain_norm_grad, "write": _plain_write,
          "read": _plain_read, "attend": _plain_attend}


# ------------------------------------------------------ the framework's calls


def _own(s):
    from tcfp_amd import attention, norm

    c = s["case"]
    kind = c["kind"]
    if kind == "norm":
        codes, scales, h, rstd = norm.rms_norm_quantize(
            s["x"], s["w"], s["r"], eps=_EPS, block_size=c["block"], scale_format="fp32")
        return {"codes": codes, "scales": scales, "h": h, "rstd": rstd}
    if kind == "norm_grad":
        dx, dw = norm.rms_norm_backward(s["gy"], s["h"], s["rstd"], s["w"], s["gh"])
        return {"dx": dx, "dw": dw}
    if kind == "write":
        kc, vc, ke, ve = s["pool"]
        attention.kv_cache_write(s["k"], s["v"], kc, vc, ke, ve, s["slots"])
        return {"k": kc, "v": vc, "k_exps": ke, "v_exps": ve}
    if kind == "read":
        k, v = attention.kv_cache_read(*s["pool"], s["slots"], out_dtype=_DT[c["dtype"]])
        return {"k": k, "v": v}
    return attention.paged_attention(
        s["q"], *s["pool"], s["table"], s["seq_lens"], s["starts"], max_query_len=s["max_new"],
        max_seq_len=s["max_len"], window=c["window"])


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["kind"]](state)


def work(case):
    kind = case["kind"]
    if kind in ("norm", "norm_grad"):
        m, d, b = case["tokens"], case["d"], _BYTES[case["dtype"]]
        if kind == "norm":
            # x (and the residual, and their sum), codes, scales, 1 / rms
            per = d * (b * (3 if case["residual"] else 1) + 1) + d // case["block"] * 4 + 4
            return {"bytes": m * per + 4 * d, "flops": 6 * m * d}
        # the gradient of y, h, (the gradient of h,) dx; 1 / rms; w and dw
        return {"bytes": m * (d * b * (4 if case["residual"] else 3) + 4) + 8 * d,
                "flops": 9 * m * d}
    hkv, dim = case["kv_heads"], case["dim"]
    if kind in ("write", "read"):
        b = _BYTES[case["dtype"]]
        return {"bytes": 2 * case["tokens"] * hkv * (dim * (b + 1) + 1) + 8 * case["tokens"],
                "flops": 2 * case["tokens"] * hkv * dim}
    hq, w = case["heads"], case["window"]
    pairs = keys = tokens = pages = 0
    for new, total in _lengths(case):
        tokens += new
        before = total - new
        if w:
            full = max(0, min(new, w - 1 - before))  # queries that see all before them
            pairs += full * before + full * (full + 1) // 2 + (new - full) * w
            seen = min(total, new + w - 1)
        else:
            pairs += new * before + new * (new + 1) // 2
            seen = total
        keys += seen
        pages += -(-seen // case["page"])
    return {"bytes": 4 * tokens * hq * dim + 2 * keys * hkv * (dim + 1) + 4 * pages,
            "flops": 4 * pairs * hq * dim}


# ------------------------------------------------------- the same in 64 bits


def _round_e4m3(x):
    """x (64 bits, within +-448) rounded to the nearest E4M3 value, ties to even."""
    _, e = torch.frexp(x)
    step = torch.exp2((e.double() - 1).clamp(min=-6.0) - 3.0)
    return torch.round(x / step) * step


def _exact_quantise(x):
    amax = x.abs().amax(-1).clamp(min=1e-12)
    e = torch.ceil(torch.log2(amax / _MAX)).clamp(min=-126.0)
    return _round_e4m3((x * torch.exp2(-e)[..., None]).clamp(-_MAX, _MAX))


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "norm":
        x = s["x"].double() + (s["r"].double() if s["r"] is not None else 0.0)
        rstd = 1.0 / torch.sqrt(x.square().mean(1) + _EPS)
        y = (x * rstd[:, None] * s["w"].double()).reshape(x.shape[0], -1, case["block"])
        step = y.abs().amax(2).clamp(min=1e-12) / _MAX
        codes = _round_e4m3((y / step[..., None]).clamp(-_MAX, _MAX)).reshape(x.shape)
        return {"codes": codes, "scales": step.t().contiguous(), "h": x, "rstd": rstd}
    if kind == "norm_grad":
        h, gy, rstd = s["h"].double(), s["gy"].double(), s["rstd"].double()[:, None]
        g = gy * s["w"].double()
        d = h.shape[1]
        dx = rstd * g - h * rstd**3 * (g * h).sum(1, keepdim=True) / d
        if s["gh"] is not None:
            dx = dx + s["gh"].double()
        return {"dx": dx, "dw": (gy * h * rstd).sum(0)}
    page = case["page"]
    if kind == "write":
        pages, hkv, _, dim = s["pool"][0].shape
        out = {"k_exps": None, "v_exps": None}
        for name in ("k", "v"):
            flat = torch.zeros(pages * page, hkv, dim, dtype=torch.float64, device="cuda")
            flat[s["slots"]] = _exact_quantise(s[name].double())
            out[name] = flat.reshape(pages, page, hkv, dim).transpose(1, 2).contiguous()
        return out
    kc, vc, ke, ve = s["pool"]

    def whole(codes, exps):  # [tokens of the pool, heads, dim]
        x = codes.double() * torch.exp2(exps.double())[..., None]
        return x.transpose(1, 2).reshape(-1, x.shape[1], x.shape[3])

    if kind == "read":
        return {"k": whole(kc, ke)[s["slots"]], "v": whole(vc, ve)[s["slots"]]}
    # one sequence and one query head at a time
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    group, w = case["heads"] // case["kv_heads"], case["window"]
    starts, lens = s["starts"].tolist(), s["seq_lens"].tolist()
    k, v = whole(kc, ke), whole(vc, ve)
    for b, total in enumerate(lens):
        lo, hi = starts[b], starts[b + 1]
        j = torch.arange(total, device="cuda")
        at = s["table"][b].long()[j // page] * page + j % page
        kb, vb = k[at], v[at]
        ahead = j[None, :] - torch.arange(total - (hi - lo), total, device="cuda")[:, None]
        hidden = ahead > 0
        if w:
            hidden |= ahead <= -w
        for h in range(case["heads"]):
            kh, vh = kb[:, h // group].contiguous(), vb[:, h // group].contiguous()
            score = torch.mm(s["q"][lo:hi, h].double(), kh.t()) / math.sqrt(case["dim"])
            score[hidden] = -math.inf
            out[lo:hi, h] = torch.mm(torch.softmax(score, 1), vh)
    return out
