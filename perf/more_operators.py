"""What the speed of a decoder's training operators is measured on.

What a training step of a decoder takes between and behind its linear layers
and norms:

* ``rope``   -- rotary positions of queries and keys (both layouts, a part of
  the head, frequencies stretched for long contexts), forward, and with the
  gradients of both.
* ``attend`` -- attention within packed sequences of different lengths, heads
  in groups that share a K/V head, causal, with and without a window: forward
  (a prompt, an evaluation), and with the gradients of queries, keys, values.
* ``loss``   -- softmax cross entropy of a linear head over a vocabulary,
  without keeping the logits: every token's loss (an evaluation), and the mean
  loss with the gradients of the hidden states and of the head's weight.

The plain forms are elementary torch operations in fp32 (the rotation's angles
in fp64), rounded once at the end.

Sizes: the small transformer's (4 heads of 64, d_model 256, vocabulary 256, 32
sequences of 128) and d_model 4096 with 8192 tokens are the repository's own;
the others are generic.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp32": 4}
_IGNORE = -100


def _rope(tokens, heads, kv_heads, dim, rotary, interleaved, stretch, far, dtype, train, name=None):
    c = {"kind": "rope", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
         "rotary": rotary, "interleaved": interleaved, "stretch": stretch, "far": far,
         "dtype": dtype, "train": train}
    return c if name is None else {"name": name, **c}


def _attend(batch, length, heads, kv_heads, dim, window, train, even=False, name=None):
    c = {"kind": "attend", "batch": batch, "length": length, "heads": heads,
         "kv_heads": kv_heads, "dim": dim, "window": window, "train": train, "even": even}
    return c if name is None else {"name": name, **c}


def _loss(tokens, d, vocab, ignored, train, name=None):
    c = {"kind": "loss", "tokens": tokens, "d": d, "vocab": vocab, "ignored": ignored,
         "train": train}
    return c if name is None else {"name": name, **c}


def listed():
    return [
        # one generated token, far into its sequence: latency only
        _rope(1, 32, 8, 128, 128, False, 1.0, 30000, "bf16", False, name="rope-1"),
        # a training batch of 8192 tokens, forward and backward
        _rope(8192, 32, 8, 128, 128, False, 1.0, 8192, "bf16", True, name="rope-8192"),
        # a long prompt in fp32, pairs side by side, half of each head rotated,
        # frequencies stretched to 16 times the trained length
        _rope(4001, 16, 16, 64, 32, True, 16.0, 131072, "fp32", False, name="rope-long-4001"),
        # the small transformer's training batch: 32 sequences of 128
        _attend(32, 128, 4, 4, 64, 0, True, even=True, name="attend-small"),
        # ragged prompts of up to 1000 tokens, nothing trained
        _attend(6, 1000, 32, 8, 128, 0, False, name="attend-prompt-1000"),
        # documents of up to 4096 tokens packed into a training batch
        _attend(4, 4096, 32, 8, 128, 0, True, name="attend-packed-4096"),
        # a long sequence whose layers look back 1000 tokens
        _attend(1, 8192, 16, 16, 64, 1000, True, name="attend-window-8192"),
        # a long sequence whose layers see all of it
        _attend(1, 8192, 32, 8, 128, 0, True, name="attend-8192"),
        # the small transformer's loss: few classes, a short contraction
        _loss(4096, 256, 256, 0.0, True, name="loss-256"),
        # 64 tokens scored against a whole vocabulary: the weight is read once
        _loss(64, 4096, 32768, 0.0, False, name="loss-score-64"),
        # a short batch, an odd vocabulary, padding left out
        _loss(1000, 1056, 50001, 0.1, True, name="loss-50001"),
        # a training batch of 8192 tokens: the largest
        _loss(8192, 4096, 32768, 0.0, True, name="loss-8192"),
    ]


def _log(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def _int(rng, lo, hi):
    return int(round(_log(rng, lo, hi)))


def draw(rng):
    kind = rng.choice(["rope", "attend", "attend", "loss", "loss"])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4])
    dim = rng.choice([64, 128, 128])
    if kind == "rope":
        rotary = rng.choice([dim, dim, dim // 2, dim // 4])
        return _rope(_int(rng, 1, 8192), heads, kv_heads, dim, rotary, rng.random() < 0.5,
                     rng.choice([1.0, 4.0, 16.0]), _int(rng, 100, 200000),
                     rng.choice(["bf16", "bf16", "fp32"]), rng.random() < 0.6)
    if kind == "attend":
        batch = _int(rng, 1, 16)
        # (no more pairs of tokens and heads than the longest listed sequence)
        most = min(8192.0, math.sqrt(1.4e9 / (batch * heads)))
        return _attend(batch, _int(rng, 1, most), heads, kv_heads, dim,
                       rng.choice([0, 0, _int(rng, 16, 2048)]), rng.random() < 0.7)
    tokens, d = _int(rng, 1, 8192), 8 * _int(rng, 8, 512)
    return _loss(tokens, d, _int(rng, 100, 64000 if tokens * d < 1 << 23 else 32000),
                 rng.choice([0.0, 0.1]), rng.random() < 0.7)


def _lengths(case):
    """The sequences' lengths: the first has the case's, the others between a
    quarter of it and all."""
    rng = random.Random(case["batch"] * 1000003 + case["length"])
    return [case["length"] if b == 0 or case["even"] else
            max(1, int(case["length"] * rng.uniform(0.25, 1.0))) for b in range(case["batch"])]


# ---------------------------------------------------------------- the inputs


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def randn(*shape, dtype=torch.float32, std=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * std).to(dtype)

    kind = case["kind"]
    s = {"case": case}
    if kind == "rope":
        t, hq, hkv, dim = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        dt = _DT[case["dtype"]]
        # queries and keys as the QKV projection leaves them: slices of a matrix
        qkv = randn(t, (hq + 2 * hkv) * dim, dtype=dt)
        s["q"] = qkv[:, :hq * dim].unflatten(1, (hq, dim))
        s["k"] = qkv[:, hq * dim:(hq + hkv) * dim].unflatten(1, (hkv, dim))
        s["positions"] = torch.randint(0, case["far"], (t,), generator=gen, device="cuda")
        s["freqs"] = _frequencies(case["rotary"], case["stretch"]).cuda()
        if case["train"]:
            s["q"], s["k"] = s["q"].detach().requires_grad_(), s["k"].detach().requires_grad_()
            s["gq"], s["gk"] = randn(t, hq, dim, dtype=dt), randn(t, hkv, dim, dtype=dt)
        return s
    if kind == "attend":
        hq, hkv, dim = case["heads"], case["kv_heads"], case["dim"]
        lens = _lengths(case)
        starts = [0]
        for n in lens:
            starts.append(starts[-1] + n)
        t = starts[-1]
        s["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
        s["max_len"] = max(lens)
        # queries and keys come rotated, each a tensor of its own, values as a
        # slice of the projection; scores of a trained model are spread wider
        # than those of unit vectors
        s["q"] = randn(t, hq, dim, dtype=torch.bfloat16, std=1.5)
        s["k"] = randn(t, hkv, dim, dtype=torch.bfloat16)
        qkv = randn(t, (hq + 2 * hkv) * dim, dtype=torch.bfloat16)
        s["v"] = qkv[:, (hq + hkv) * dim:].unflatten(1, (hkv, dim))
        if case["train"]:
            for n in ("q", "k", "v"):
                s[n] = s[n].detach().requires_grad_()
            s["go"] = randn(t, hq, dim, dtype=torch.bfloat16, std=1e-2)
        return s
    t, d, v = case["tokens"], case["d"], case["vocab"]
    s["h"] = randn(t, d, dtype=torch.bfloat16)
    s["w"] = randn(v, d, dtype=torch.bfloat16, std=2.0 / math.sqrt(d))
    s["targets"] = torch.randint(0, v, (t,), generator=gen, device="cuda")
    if case["ignored"]:
        out = torch.rand(t, generator=gen, device="cuda") < case["ignored"]
        out[0] = False  # (a mean needs a token)
        s["targets"].masked_fill_(out, _IGNORE)
    if case["train"]:
        s["h"], s["w"] = s["h"].requires_grad_(), s["w"].requires_grad_()
    return s


def _frequencies(rotary, stretch, base=10000.0, trained=8192, slow=1.0, fast=32.0):
    """Radians a position of each pair, fp64.  Stretched for a context of
    ``stretch`` times the trained one: pairs that turn fewer than ``slow`` times
    within the trained length are slowed down by it, those that turn more than
    ``fast`` times keep their pace, those between are blended."""
    f = base ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)
    if stretch == 1.0:
        return f
    turns = trained * f / (2 * math.pi)
    keep = ((turns - slow) / (fast - slow)).clamp(0.0, 1.0)
    return f * (keep + (1.0 - keep) / stretch)


# ----------------------------------------------------------- the plain forms


def _turn(x, cos, sin, interleaved):
    half = cos.shape[-1]
    y = x.float()
    part = y[..., :2 * half]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :half],
                                                                   part[..., half:])
    c, d = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((c, d), -1).flatten(-2) if interleaved else torch.cat((c, d), -1)
    return torch.cat((turned, y[..., 2 * half:]), -1).to(x.dtype)


def _plain_rope(s):
    c = s["case"]
    angle = s["positions"].double()[:, None, None] * s["freqs"]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    out = {n: _turn(s[n].detach(), cos, sin, c["interleaved"]) for n in ("q", "k")}
    if c["train"]:
        out |= {n: _turn(s[n], cos, -sin, c["interleaved"]) for n in ("gq", "gk")}
    return out


def _plain_attend(s):
    c = s["case"]
    hq, hkv, dim = c["heads"], c["kv_heads"], c["dim"]
    group, nb, n = hq // hkv, c["batch"], s["max_len"]
    starts = s["starts"].long()
    lens = starts.diff()
    i = torch.arange(n, device="cuda")
    rows = (starts[:-1, None] + i).clamp(max=int(s["q"].shape[0]) - 1)
    live = i < lens[:, None]  # [batch, place]

    def padded(x, heads):  # [batch, kv head, member of the group, place, dim]
        x = x.detach().float()[rows] * live[..., None, None]
        return x.view(nb, n, hkv, heads // hkv, dim).permute(0, 2, 3, 1, 4).contiguous()

    def packed(x, heads):  # the reverse
        x = x.permute(0, 3, 1, 2, 4).reshape(nb, n, heads, dim)
        return x[live].to(s["q"].dtype)

    q, k, v = padded(s["q"], hq), padded(s["k"], hkv), padded(s["v"], hkv)
    flat = (nb, hkv, group * n, dim)
    kt = k[:, :, 0].transpose(-2, -1).contiguous()
    back = i[:, None] - i[None, :]
    hidden = back < 0
    if c["window"]:
        hidden = hidden | (back >= c["window"])
    hidden = hidden | ~live[:, None, :]
    p = torch.matmul(q.view(flat), kt).mul_(dim**-0.5).view(nb, hkv, group, n, n)
    p.masked_fill_(hidden[:, None, None], float("-inf"))
    top = p.amax(-1, keepdim=True)
    p = p.sub_(top.masked_fill_(top == float("-inf"), 0.0)).exp_()
    p /= p.sum(-1, keepdim=True).clamp_(min=1e-30)
    p2 = p.view(nb, hkv, group * n, n)
    o = torch.matmul(p2, v[:, :, 0])
    out = {"o": packed(o.view(q.shape), hq)}
    if c["train"]:
        go = padded(s["go"], hq).view(flat)
        dv = torch.matmul(p2.transpose(-2, -1), go)
        ds = torch.matmul(go, v[:, :, 0].transpose(-2, -1).contiguous())
        ds.sub_((go * o).sum(-1, keepdim=True)).mul_(p2).mul_(dim**-0.5)
        dq = torch.matmul(ds, k[:, :, 0])
        dk = torch.matmul(ds.transpose(-2, -1), q.view(flat))
        out |= {"dq": packed(dq.view(q.shape), hq), "dk": packed(dk.unsqueeze(2), hkv),
                "dv": packed(dv.unsqueeze(2), hkv)}
    return out


def _plain_loss(s):
    h, w, target = s["h"].detach().float(), s["w"].detach().float(), s["targets"]
    kept = target != _IGNORE
    at = target.clamp(min=0)[:, None]
    z = torch.matmul(h, w.t())
    top = z.amax(-1, keepdim=True)
    picked = z.gather(1, at) - top
    p = z.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    each = (total.log() - picked)[:, 0] * kept
    if not s["case"]["train"]:
        return {"losses": each}
    count = kept.sum()
    loss = (each.double().sum() / count).float()
    p /= total
    p.scatter_add_(1, at, torch.full_like(picked, -1.0))
    p *= (kept / count.float())[:, None]
    return {"loss": loss, "dh": torch.matmul(p, w).to(s["h"].dtype),
            "dw": torch.matmul(p.t(), h).to(s["w"].dtype)}


_PLAIN = {"rope": _plain_rope, "attend": _plain_attend, "loss": _plain_loss}


# ------------------------------------------------------ the framework's calls


def _own(s):
    from tcfp_amd import attention, loss, rotary

    c = s["case"]
    if c["kind"] == "rope":
        q, k = rotary.rotary_embedding(s["q"], s["k"], s["positions"], s["freqs"],
                                       interleaved=c["interleaved"])
        if not c["train"]:
            return {"q": q, "k": k}
        gq, gk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["gq"], s["gk"]))
        return {"q": q.detach(), "k": k.detach(), "gq": gq, "gk": gk}
    if c["kind"] == "attend":
        o = attention.packed_attention(s["q"], s["k"], s["v"], s["starts"], max_len=s["max_len"],
                                       window=c["window"])
        if not c["train"]:
            return {"o": o}
        dq, dk, dv = torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["go"])
        return {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv}
    if not c["train"]:
        return {"losses": loss.linear_cross_entropy(s["h"], s["w"], s["targets"],
                                                    ignore_index=_IGNORE, reduction="none")}
    mean = loss.linear_cross_entropy(s["h"], s["w"], s["targets"], ignore_index=_IGNORE)
    dh, dw = torch.autograd.grad(mean, (s["h"], s["w"]))
    return {"loss": mean.detach(), "dh": dh, "dw": dw}


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["kind"]](state)


def work(case):
    if case["kind"] == "rope":
        b = _BYTES[case["dtype"]]
        heads = case["heads"] + case["kv_heads"]
        passes = 2 if case["train"] else 1
        return {"bytes": case["tokens"] * (2 * passes * heads * case["dim"] * b + 8),
                "flops": passes * 3 * case["tokens"] * heads * case["rotary"]}
    if case["kind"] == "attend":
        hq, hkv, dim, w = case["heads"], case["kv_heads"], case["dim"], case["window"]
        lens = _lengths(case)
        pairs = 0
        for n in lens:
            m = min(n, w) if w else n
            pairs += m * (m + 1) // 2 + (n - m) * m
        tokens = sum(lens)
        # q and o; k and v; with them their gradients
        once = tokens * dim * 2 * (2 * hq + 2 * hkv)
        return {"bytes": once * (2 if case["train"] else 1),
                "flops": pairs * hq * dim * (14 if case["train"] else 4)}
    t, d, v = case["tokens"], case["d"], case["vocab"]
    if not case["train"]:
        return {"bytes": 2 * d * (t + v) + 12 * t, "flops": 2 * t * d * v}
    return {"bytes": 4 * d * (t + v) + 8 * t, "flops": 6 * t * d * v}


# ------------------------------------------------------- the same in 64 bits


def _exact_rope(s):
    c = s["case"]
    half = c["rotary"] // 2
    # a pair as a complex number, turned by multiplying it with e^(i angle)
    angle = s["positions"].double()[:, None] * s["freqs"][None, :]
    unit = torch.complex(torch.cos(angle), torch.sin(angle))[:, None, :]

    def turned(x, unit):
        x = x.detach().double().clone()
        if c["interleaved"]:
            first, second = slice(0, 2 * half, 2), slice(1, 2 * half, 2)
        else:
            first, second = slice(0, half), slice(half, 2 * half)
        z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * unit
        x[..., first], x[..., second] = z.real, z.imag
        return x

    out = {"q": turned(s["q"], unit), "k": turned(s["k"], unit)}
    if c["train"]:
        out |= {"gq": turned(s["gq"], unit.conj()), "gk": turned(s["gk"], unit.conj())}
    return out


def _exact_attend(s):
    # one sequence and one query head at a time
    c = s["case"]
    group, w, train = c["heads"] // c["kv_heads"], c["window"], c["train"]
    names = ("q", "k", "v", "go") if train else ("q", "k", "v")
    x = {n: s[n].detach() for n in names}
    out = {"o": torch.zeros(x["q"].shape, dtype=torch.float64, device="cuda")}
    if train:
        out |= {"d" + n: torch.zeros(x[n].shape, dtype=torch.float64, device="cuda")
                for n in ("q", "k", "v")}
    starts = s["starts"].tolist()
    c0 = 1.0 / math.sqrt(c["dim"])
    for lo, hi in zip(starts, starts[1:]):
        n = hi - lo
        seen = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
        if w:
            seen = seen.triu(1 - w)
        for h in range(c["heads"]):
            g = h // group
            q, k, v = (x[a][lo:hi, b].double() for a, b in (("q", h), ("k", g), ("v", g)))
            z = torch.mm(q, k.t().contiguous()) * c0
            p = torch.softmax(z.masked_fill_(~seen, -math.inf), 1)
            o = torch.mm(p, v)
            out["o"][lo:hi, h] = o
            if train:
                go = x["go"][lo:hi, h].double()
                out["dv"][lo:hi, g] += torch.mm(p.t().contiguous(), go)
                dp = torch.mm(go, v.t().contiguous())
                ds = p * (dp - (p * dp).sum(1, keepdim=True)) * c0
                out["dq"][lo:hi, h] = torch.mm(ds, k)
                out["dk"][lo:hi, g] += torch.mm(ds.t().contiguous(), q)
    return out


def _exact_loss(s):
    # 1024 tokens at a time
    h, w, target = s["h"].detach().double(), s["w"].detach().double(), s["targets"]
    wt = w.t().contiguous()
    kept = (target != _IGNORE).double()
    losses, dh, dw = [], [], torch.zeros_like(w)
    for lo in range(0, h.shape[0], 1024):
        x, t, live = h[lo:lo + 1024], target[lo:lo + 1024].clamp(min=0), kept[lo:lo + 1024]
        logp = torch.log_softmax(torch.mm(x, wt), 1)
        r = torch.arange(x.shape[0], device="cuda")
        losses.append(-logp[r, t] * live)
        if s["case"]["train"]:
            g = torch.exp(logp)
            g[r, t] -= 1.0
            g *= (live / kept.sum())[:, None]
            dh.append(torch.mm(g, w))
            dw += torch.mm(g.t().contiguous(), x)
    losses = torch.cat(losses)
    if not s["case"]["train"]:
        return {"losses": losses}
    return {"loss": losses.sum() / kept.sum(), "dh": torch.cat(dh), "dw": dw}


_EXACT = {"rope": _exact_rope, "attend": _exact_attend, "loss": _exact_loss}


def exact(case, seed):
    return _EXACT[case["kind"]](prepare(case, seed))
