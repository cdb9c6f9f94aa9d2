"""Train a small decoder on TCFP-12 layers, then generate from it through the
8-bit paged K/V cache.

    python examples/generate.py [--steps 600] [--tokens 64] [--rotary] [--fp32]

The model is the repository's small transformer (d_model 256, 4 layers, 4 heads,
FFN 1024, vocab 256) with root-mean-square norms: every norm stands in front of
a linear layer that reads FP8 codes, so ``TCFPNormLinear`` quantises where it
normalises.  Positions are a learned table, or with ``--rotary`` turns of the
queries and keys.  Training attends a batch's sequences packed one after another
and takes the loss from the hidden states, without the logits, both from bf16; with
``--fp32`` both are plain products in fp32.  Serving lays the
weight codes out once; a step of a batch -- whole prompts or one token each -- is,
per layer,

    rms_norm_quantize -> QKV GEMM -> cache write -> paged attention
    -> block_quantize -> output GEMM
    rms_norm_quantize -> FFN GEMM -> GELU -> block_quantize -> FFN GEMM

The training text are sequences that go on by a rule (arithmetic runs and
repeated motifs), so what is generated can be checked.
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch
import torch.nn as nn
import torch.nn.functional as F

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from tcfp_amd import kernels as K  # noqa: E402
from tcfp_amd import norm  # noqa: E402
from tcfp_amd.attention import PagedKVCache, packed_attention  # noqa: E402
from tcfp_amd.loss import linear_cross_entropy  # noqa: E402
from tcfp_amd.rotary import rotary_embedding, rotary_frequencies  # noqa: E402
from tcfp_amd.nn import TCFPLinear, TCFPNormLinear, TCFPRMSNorm  # noqa: E402

VOCAB, BLOCK = 256, 64


class Layer(nn.Module):
    def __init__(self, d: int, heads: int, ffn: int, fp32: bool = False) -> None:
        super().__init__()
        self.heads = heads
        self.plain = fp32 or d // heads not in (64, 128, 256)  # (what the kernel has)
        self.qkv = TCFPNormLinear(d, 3 * d, scale_block_size=BLOCK)
        self.proj = TCFPLinear(d, d, use_tensor_cores=True, scale_block_size=BLOCK)
        self.fc1 = TCFPNormLinear(d, ffn, scale_block_size=BLOCK)
        self.fc2 = TCFPLinear(ffn, d, use_tensor_cores=True, scale_block_size=BLOCK)

    def attend(self, qkv, starts, turn):
        """Every token on itself and those before it in its sequence."""
        b, t, c = qkv.shape[0], qkv.shape[1], qkv.shape[2] // 3
        dtype = torch.float32 if self.plain else torch.bfloat16
        q, k, v = qkv.to(dtype).reshape(b * t, 3, self.heads, -1).unbind(1)
        if turn is not None:
            q, k = rotary_embedding(q, k, *turn)
        if not self.plain:
            return packed_attention(q, k, v, starts, max_len=t).reshape(b, t, c)
        q, k, v = (z.reshape(b, t, self.heads, -1).transpose(1, 2).contiguous() for z in (q, k, v))
        att = torch.matmul(q, k.transpose(-2, -1).contiguous()) / q.shape[-1] ** 0.5
        mask = torch.triu(torch.ones(t, t, dtype=torch.bool, device=q.device), 1)
        att = F.softmax(att.masked_fill(mask, float("-inf")), dim=-1)
        return torch.matmul(att, v).transpose(1, 2).reshape(b, t, c)

    def forward(self, x, h, starts, turn):
        """``x``: what the layer before adds to the residual stream ``h``; ``starts``:
        where the batch's sequences begin; ``turn``: positions and frequencies."""
        qkv, h = self.qkv(x, h)
        y = self.attend(qkv, starts, turn)
        z, h = self.fc1(self.proj(y.to(h.dtype)), h)
        return self.fc2(F.gelu(z)), h


class Decoder(nn.Module):
    def __init__(self, d: int = 256, layers: int = 4, heads: int = 4, ffn: int = 1024,
                 positions: int = 256, rotary: bool = False, fp32: bool = False) -> None:
        super().__init__()
        self.tok, self.positions, self.fp32 = nn.Embedding(VOCAB, d), positions, fp32
        self.pos = None if rotary else nn.Embedding(positions, d)
        self.register_buffer("freqs", rotary_frequencies(d // heads) if rotary else None,
                             persistent=False)
        self.layers = nn.ModuleList(Layer(d, heads, ffn, fp32) for _ in range(layers))
        self.norm = TCFPRMSNorm(d)
        for m in self.modules():
            if isinstance(m, (nn.Embedding, TCFPLinear)):
                nn.init.normal_(m.weight, std=0.02)

    def embed(self, idx, pos):
        """What the first layer adds to the residual stream, and the stream."""
        h = self.tok(idx)
        return (torch.zeros_like(h) if self.pos is None else self.pos(pos).expand_as(h)), h

    def hidden(self, idx):
        """The hidden states in front of the head."""
        b, t = idx.shape
        if t > self.positions:
            raise ValueError(f"{t} tokens, the model has {self.positions} positions")
        pos = torch.arange(t, device=idx.device)
        x, h = self.embed(idx, pos)
        starts = torch.arange(0, b * t + 1, t, dtype=torch.int32, device=idx.device)
        turn = None if self.freqs is None else (pos.repeat(b), self.freqs)
        for layer in self.layers:
            x, h = layer(x, h, starts, turn)
        return self.norm(x, h)[0]

    def forward(self, idx):
        return self.hidden(idx).float() @ self.tok.weight.t()

    def loss(self, idx, targets):
        """Mean cross entropy, with the head in bf16 and its logits nowhere (or in fp32)."""
        if self.fp32:
            return F.cross_entropy(self(idx).reshape(-1, VOCAB), targets.reshape(-1))
        return linear_cross_entropy(self.hidden(idx).bfloat16(), self.tok.weight.bfloat16(),
                                    targets)


class Server:
    """A trained :class:`Decoder` served from weight codes and a paged cache."""

    def __init__(self, model: Decoder, pages: int = 256, page_size: int = 16) -> None:
        self.model = model
        self.codes = {m: K.fused_dual_quantize_fp8(m.weight.detach().contiguous(), BLOCK)
                      for m in model.modules() if isinstance(m, TCFPLinear)}
        d = model.tok.embedding_dim
        heads = model.layers[0].heads
        self.heads, self.dim = heads, d // heads
        self.cache = PagedKVCache(len(model.layers), pages, heads, self.dim, page_size=page_size,
                                  device=model.tok.weight.device)

    def _linear(self, m, codes, exps, out_dtype=torch.float32):
        hi, lo, e_hi, e_lo = self.codes[m]
        return K.fused_block_scaled_dual_gemm_forward(codes, hi, lo, exps, e_hi, e_lo, BLOCK,
                                                      bias=m.bias, out_dtype=out_dtype)

    @torch.no_grad()
    def step(self, seqs: list[int], tokens: list[list[int]]) -> torch.Tensor:
        """Append ``tokens[i]`` to sequence ``seqs[i]``; the logits of every new
        token, one sequence after another."""
        model, dev = self.model, self.model.tok.weight.device
        starts = [self.cache.length(s) for s in seqs]
        # (an index that a table does not have would end the process on the GPU)
        room = model.positions
        if any(a + len(t) > room for a, t in zip(starts, tokens)):
            raise ValueError(f"a sequence would pass the model's {room} positions")
        if any(not 0 <= t < model.tok.num_embeddings for ts in tokens for t in ts):
            raise ValueError(f"tokens must lie in [0, {model.tok.num_embeddings})")
        batch = self.cache.extend(seqs, [len(t) for t in tokens])
        idx = torch.tensor([t for ts in tokens for t in ts], device=dev)
        pos = torch.tensor([a + i for a, t in zip(starts, tokens) for i in range(len(t))],
                           device=dev)
        x, h = model.embed(idx, pos)
        for i, layer in enumerate(model.layers):
            q8, e, h, _ = norm.rms_norm_quantize(x, layer.qkv.norm_weight, h, eps=layer.qkv.eps,
                                                 block_size=BLOCK)
            qkv = self._linear(layer.qkv, q8, e, torch.bfloat16)
            q, k, v = (z.unflatten(1, (self.heads, self.dim)) for z in qkv.chunk(3, 1))
            if model.freqs is not None:
                q, k = rotary_embedding(q, k, pos, model.freqs)
            self.cache.write(i, k, v, batch)
            y = self.cache.attend(i, q, batch)
            x = self._linear(layer.proj, *K.block_quantize_fp8(y.flatten(1), BLOCK))
            q8, e, h, _ = norm.rms_norm_quantize(x, layer.fc1.norm_weight, h, eps=layer.fc1.eps,
                                                 block_size=BLOCK)
            z = F.gelu(self._linear(layer.fc1, q8, e))
            x = self._linear(layer.fc2, *K.block_quantize_fp8(z, BLOCK))
        y, _, _ = norm.rms_norm(x, model.norm.weight, h, eps=model.norm.eps)
        return y.float() @ model.tok.weight.t()

    def generate(self, prompts: list[list[int]], count: int) -> list[list[int]]:
        """The likeliest ``count`` tokens after each prompt (of a token or more)."""
        if not all(prompts):
            raise ValueError("a prompt needs a token")
        if count < 1:
            return [[] for _ in prompts]
        seqs = [self.cache.open() for _ in prompts]
        try:
            logits = self.step(seqs, prompts)
            ends = torch.tensor([len(p) for p in prompts]).cumsum(0) - 1
            new = logits[ends.to(logits.device)].argmax(-1).tolist()
            out = [[t] for t in new]
            for _ in range(count - 1):
                new = self.step(seqs, [[t] for t in new]).argmax(-1).tolist()
                for o, t in zip(out, new):
                    o.append(t)
            return out
        finally:
            for s in seqs:
                self.cache.close(s)


def patterns(n: int, length: int, gen: torch.Generator) -> torch.Tensor:
    """Token sequences that go on by a rule: steps of 1 to 3, motifs of 4 to 8."""
    t = torch.arange(length)
    rows = []
    for i in range(n):
        if i % 2:
            start, step = (int(torch.randint(lo, hi, (), generator=gen)) for lo, hi in
                           ((0, VOCAB), (1, 4)))
            rows.append((start + step * t) % VOCAB)
        else:
            size = int(torch.randint(4, 9, (), generator=gen))
            rows.append(torch.randint(0, VOCAB, (size,), generator=gen)[t % size])
    return torch.stack(rows)


def train(model: Decoder, steps: int, seq: int = 128, batch: int = 32, seed: int = 0) -> list[float]:
    dev = model.tok.weight.device
    gen = torch.Generator().manual_seed(seed)
    opt = torch.optim.AdamW(model.parameters(), lr=1e-3, weight_decay=0.01)
    losses = []
    for step in range(steps):
        for g in opt.param_groups:
            g["lr"] = 1e-3 * min(1.0, (step + 1) / 20)
        data = patterns(batch, seq + 1, gen).to(dev)
        loss = model.loss(data[:, :-1], data[:, 1:])
        opt.zero_grad(set_to_none=True)
        loss.backward()
        nn.utils.clip_grad_norm_(model.parameters(), 1.0)
        opt.step()
        losses.append(loss.detach())
    return [float(x) for x in losses]


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=600)
    ap.add_argument("--tokens", type=int, default=64)
    ap.add_argument("--rotary", action="store_true", help="rotary instead of learned positions")
    ap.add_argument("--fp32", action="store_true", help="train attention and head in fp32")
    a = ap.parse_args()
    torch.manual_seed(0)
    model = Decoder(rotary=a.rotary, fp32=a.fp32).cuda()
    losses = train(model, a.steps)
    print(f"loss {losses[0]:.3f} -> {losses[-1]:.3f} in {a.steps} steps", flush=True)
    server = Server(model)
    rows = patterns(8, 40 + a.tokens, torch.Generator().manual_seed(1))
    prompts = [r[:40 - i].tolist() for i, r in enumerate(rows)]
    got = server.generate(prompts, a.tokens)
    right = sum(g == int(r[len(p) + j]) for r, p, o in zip(rows, prompts, got)
                for j, g in enumerate(o))
    print(f"{right} of {len(rows) * a.tokens} generated tokens follow the rule")
    for p, o in zip(prompts[:4], got):
        print("  ...", p[-6:], "->", o[:12])


if __name__ == "__main__":
    main()
