"""Train a small decoder on TCFP-12 layers, then generate from it through the
8-bit paged K/V cache.

    python examples/generate.py [--steps 600] [--tokens 64]

The model is the repository's small transformer (d_model 256, 4 layers, 4 heads,
FFN 1024, vocab 256) with root-mean-square norms: every norm stands in front of
a linear layer that reads FP8 codes, so ``TCFPNormLinear`` quantises where it
normalises.  Serving lays the weight codes out once; a step of a batch -- whole
prompts or one token each -- is, per layer,

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
from tcfp_amd.attention import PagedKVCache  # noqa: E402
from tcfp_amd.nn import TCFPLinear, TCFPNormLinear, TCFPRMSNorm  # noqa: E402

VOCAB, BLOCK = 256, 64


class Layer(nn.Module):
    def __init__(self, d: int, heads: int, ffn: int) -> None:
        super().__init__()
        self.heads = heads
        self.qkv = TCFPNormLinear(d, 3 * d, scale_block_size=BLOCK)
        self.proj = TCFPLinear(d, d, use_tensor_cores=True, scale_block_size=BLOCK)
        self.fc1 = TCFPNormLinear(d, ffn, scale_block_size=BLOCK)
        self.fc2 = TCFPLinear(ffn, d, use_tensor_cores=True, scale_block_size=BLOCK)

    def forward(self, x, h):
        """``x``: what the layer before adds to the residual stream ``h``."""
        qkv, h = self.qkv(x, h)
        b, t, c = h.shape
        q, k, v = (z.contiguous() for z in
                   qkv.float().reshape(b, t, 3, self.heads, -1).permute(2, 0, 3, 1, 4))
        att = torch.matmul(q, k.transpose(-2, -1).contiguous()) / q.shape[-1] ** 0.5
        mask = torch.triu(torch.ones(t, t, dtype=torch.bool, device=x.device), 1)
        att = F.softmax(att.masked_fill(mask, float("-inf")), dim=-1)
        y = torch.matmul(att, v).transpose(1, 2).reshape(b, t, c)
        z, h = self.fc1(self.proj(y), h)
        return self.fc2(F.gelu(z)), h


class Decoder(nn.Module):
    def __init__(self, d: int = 256, layers: int = 4, heads: int = 4, ffn: int = 1024,
                 positions: int = 256) -> None:
        super().__init__()
        self.tok, self.pos = nn.Embedding(VOCAB, d), nn.Embedding(positions, d)
        self.layers = nn.ModuleList(Layer(d, heads, ffn) for _ in range(layers))
        self.norm = TCFPRMSNorm(d)
        for m in self.modules():
            if isinstance(m, (nn.Embedding, TCFPLinear)):
                nn.init.normal_(m.weight, std=0.02)

    def forward(self, idx):
        if idx.shape[1] > self.pos.num_embeddings:
            raise ValueError(f"{idx.shape[1]} tokens, the model has {self.pos.num_embeddings} "
                             "positions")
        h = self.tok(idx)
        x = self.pos(torch.arange(idx.shape[1], device=idx.device)).expand_as(h)
        for layer in self.layers:
            x, h = layer(x, h)
        y, _ = self.norm(x, h)
        return y.float() @ self.tok.weight.t()


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
        room = model.pos.num_embeddings
        if any(a + len(t) > room for a, t in zip(starts, tokens)):
            raise ValueError(f"a sequence would pass the model's {room} positions")
        if any(not 0 <= t < model.tok.num_embeddings for ts in tokens for t in ts):
            raise ValueError(f"tokens must lie in [0, {model.tok.num_embeddings})")
        batch = self.cache.extend(seqs, [len(t) for t in tokens])
        idx = torch.tensor([t for ts in tokens for t in ts], device=dev)
        pos = torch.tensor([a + i for a, t in zip(starts, tokens) for i in range(len(t))],
                           device=dev)
        h, x = model.tok(idx), model.pos(pos)
        for i, layer in enumerate(model.layers):
            q8, e, h, _ = norm.rms_norm_quantize(x, layer.qkv.norm_weight, h, eps=layer.qkv.eps,
                                                 block_size=BLOCK)
            qkv = self._linear(layer.qkv, q8, e, torch.bfloat16)
            q, k, v = (z.unflatten(1, (self.heads, self.dim)) for z in qkv.chunk(3, 1))
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
        loss = F.cross_entropy(model(data[:, :-1]).reshape(-1, VOCAB), data[:, 1:].reshape(-1))
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
    a = ap.parse_args()
    torch.manual_seed(0)
    model = Decoder().cuda()
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
