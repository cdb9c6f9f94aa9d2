"""The norm modules, and a decoder trained on them and served through the paged
cache (examples/generate.py)."""
import copy
import importlib.util
from pathlib import Path

import pytest
import torch
import torch.nn.functional as F

from oracle import gemm as og
from tcfp_amd import norm
from tcfp_amd.attention import PagedKVCache
from tcfp_amd.nn import (TCFPLinear, TCFPNormLinear, TCFPRMSNorm, _TCFP12BlockScaledFunction,
                         set_block_dgrad, set_block_wgrad)

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _example():
    path = Path(__file__).resolve().parent.parent / "examples" / "generate.py"
    spec = importlib.util.spec_from_file_location("generate_example", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def _rel(a, b):
    return og.rel_fro(a.detach().double().cpu().numpy(), b.detach().double().cpu().numpy())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("residual", [False, True])
def test_rms_norm_module_gradients(dev, dtype, residual):
    """Against autograd in 64 bits; fp32: sums of 512 terms to some 1e-6, bf16:
    gradients rounded once."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(3, 50, 512, generator=g).to(dtype).to(dev).requires_grad_(True)
    r = torch.randn(3, 50, 512, generator=g).to(dtype).to(dev).requires_grad_(True)
    gy, gh = (torch.randn(3, 50, 512, generator=g).to(dtype).to(dev) for _ in range(2))
    m = TCFPRMSNorm(512).to(dev)
    torch.nn.init.normal_(m.weight, 1.0, 0.1)
    xd, rd, wd = (t.detach().double().requires_grad_(True) for t in (x, r, m.weight))
    s = xd + rd if residual else xd
    # (the kernels' backward starts from the stored sum)
    stored = (x.float() + r.float()).to(dtype).double() if residual else s
    y = s * torch.rsqrt((s * s).mean(-1, keepdim=True) + m.eps) * wd
    loss = (y * gy.double()).sum() + ((s * gh.double()).sum() if residual else 0)
    loss.backward()
    assert torch.allclose(stored.detach(), s.detach(), rtol=2**-8 if dtype == BF16 else 2**-23,
                          atol=0)
    if residual:
        out, h = m(x, r)
        torch.autograd.backward([out, h], [gy, gh])
    else:
        out = m(x)
        out.backward(gy)
    tol = 1e-2 if dtype == BF16 else 2e-6
    assert out.dtype == dtype and x.grad.dtype == dtype
    assert _rel(out, y) < tol and _rel(x.grad, xd.grad) < tol
    assert _rel(m.weight.grad, wd.grad) < tol
    if residual:
        assert torch.equal(x.grad, r.grad)
    with torch.no_grad():
        again = m(x, r)[0] if residual else m(x)
    assert torch.equal(again, out)


def test_rms_norm_module_unused_outputs(dev):
    x = torch.randn(4, 64, device=dev, requires_grad=True)
    r = torch.randn(4, 64, device=dev, requires_grad=True)
    m = TCFPRMSNorm(64).to(dev)
    y, h = m(x, r)
    h.sum().backward()
    assert torch.equal(x.grad, torch.ones_like(x)) and torch.equal(r.grad, x.grad)
    assert (m.weight.grad == 0).all()
    m.weight.requires_grad_(False)
    y, h = m(x.detach(), r)
    y.sum().backward()


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("opt", ["plain", "srr", "abd", "fp8_dgrad", "bf16_wgrad", "hp"])
def test_norm_linear_is_the_layer_on_the_norm(dev, residual, dtype, opt):
    """The fused node against the norm in fp32 and the block-scaled layer's
    Function, forward and every gradient: the same kernels on the same codes,
    fp32 GEMMs summed in another order at most."""
    torch.manual_seed(1)
    x = (torch.randn(2, 96, 256, device=dev) * 2).to(dtype).requires_grad_(True)
    r = torch.randn(2, 96, 256, device=dev).to(dtype).requires_grad_(True)
    kw = {"srr": {"srr": True}, "abd": {"abd": True}, "hp": {"hp_grad_weight": True}}.get(opt, {})
    layer = TCFPNormLinear(256, 640, **kw).to(dev)
    torch.nn.init.normal_(layer.norm_weight, 1.0, 0.1)
    g = torch.randn(2, 96, 640, device=dev)
    gh = torch.randn(2, 96, 256, device=dev).to(dtype)
    try:
        set_block_dgrad("fp8" if opt == "fp8_dgrad" else "exact")
        set_block_wgrad("bf16" if opt == "bf16_wgrad" else "split")
        torch.manual_seed(5)  # (the SRR seed)
        out = layer(x, r) if residual else layer(x)
        out, h = out if residual else (out, None)
        torch.autograd.backward([out, h] if residual else [out], [g, gh] if residual else [g])
        x2, r2 = (t.detach().clone().requires_grad_(True) for t in (x, r))
        w2, b2 = (t.detach().clone().requires_grad_(True) for t in (layer.weight, layer.bias))
        y, h2, rstd = norm.rms_norm(x2.detach(), layer.norm_weight.detach(),
                                    r2.detach() if residual else None, eps=layer.eps,
                                    out_dtype=F32)
        y.requires_grad_(True)
        torch.manual_seed(5)
        ref = _TCFP12BlockScaledFunction.apply(y, w2, b2, 64, opt == "hp", None, "", opt == "abd",
                                               opt == "srr", False)
        ref.backward(g)
    finally:
        set_block_dgrad("exact")
        set_block_wgrad("split")
    gy = y.grad if dtype == F32 or opt == "hp" else y.grad.to(BF16)
    dx, dn = norm.rms_norm_backward(gy, h2.detach(), rstd, layer.norm_weight.detach(),
                                    gh if residual else None)
    tol = 1e-6 if dtype == F32 else 5e-3
    assert _rel(out, ref) < 1e-6
    assert _rel(layer.weight.grad, w2.grad) < 1e-6 and _rel(layer.bias.grad, b2.grad) < 1e-6
    assert _rel(x.grad, dx) < tol and _rel(layer.norm_weight.grad, dn) < tol
    if residual:
        assert torch.equal(h, h2) and _rel(r.grad, dx) < tol


def test_norm_linear_error_feedback_fallback_and_evaluation(dev):
    torch.manual_seed(2)
    layer = TCFPNormLinear(128, 128).to(dev)
    x = torch.randn(40, 128, device=dev)
    with torch.no_grad():
        a = layer(x)
    assert "" not in layer._error_state._buffers or (
        layer._error_state._buffers[""] == 0).all()
    b = layer(x)
    assert torch.equal(a, b)  # the first call's EF buffer was empty
    assert (layer._error_state._buffers[""] != 0).any()
    layer.fallback_to_bf16()
    y, _, _ = norm.rms_norm(x, layer.norm_weight.detach())
    assert _rel(layer(x), F.linear(y, layer.weight, layer.bias)) < 1e-6
    layer.restore_tcfp()
    with pytest.raises(ValueError, match="block scales"):
        TCFPNormLinear(128, 128, scale_block_size=None)
    s = copy.deepcopy(layer).state_dict()
    assert "norm_weight" in s


def test_cache_class_writes_reads_and_attends(dev):
    c = PagedKVCache(2, 64, 2, 64, page_size=16, device=dev)
    seqs = [c.open(), c.open()]
    g = torch.Generator().manual_seed(3)
    kept = {s: [] for s in seqs}
    for counts in ([20, 3], [1, 1], [0, 30], [5, 1]):
        batch = c.extend(seqs, counts)
        k, v = (torch.randn(sum(counts), 2, 64, generator=g).to(dev) for _ in range(2))
        c.write(1, k, v, batch)
        at = 0
        for s, n in zip(seqs, counts):
            kept[s].append((k[at:at + n], v[at:at + n]))
            at += n
        q = torch.randn(sum(counts), 4, 64, generator=g).bfloat16().to(dev)
        out = c.attend(1, q, batch)
        at = 0
        for s, n in zip(seqs, counts):
            rk, rv = c.read(1, s, out_dtype=F32)
            wk, wv = (torch.cat([p[i] for p in kept[s]]) for i in (0, 1))
            amax = wk.abs().amax(-1, keepdim=True)
            assert ((rk - wk).abs() <= 2**-4 * wk.abs() + 2**-16 * amax).all()
            total = rk.shape[0]
            mask = torch.arange(total, device=dev)[None] > torch.arange(
                total - n, total, device=dev)[:, None]
            for h in range(4):
                kh, vh = rk[:, h // 2].double(), rv[:, h // 2].double()
                s_ = (q[at:at + n, h].double() @ kh.t()) / 8
                want = torch.softmax(s_.masked_fill(mask, float("-inf")), 1) @ vh
                assert ((out[at:at + n, h].double() - want).abs()
                        <= 2**-7 * (want.abs() + vh.abs().max())).all()
            at += n
    assert (c.k_codes[0].view(torch.uint8) == 0).all()  # the other layer


def test_decoder_trains_and_generates(dev):
    """600 steps on sequences that go on by a rule (loss from ln 256 = 5.5 to
    under 1: the first tokens of a motif cannot be known), then served: prompts
    whole, in chunks and token by token give the same logits but for codes that
    another order of summation flips, close to the unserved model's, and the
    rules are continued."""
    ex = _example()
    torch.manual_seed(0)
    model = ex.Decoder().to(dev)
    losses = ex.train(model, 600)
    print(f"[decoder] loss {losses[0]:.3f} -> {losses[-1]:.3f}", flush=True)
    assert losses[0] > 5.0 and losses[-1] < 1.0
    rows = ex.patterns(4, 96, torch.Generator().manual_seed(1))
    server = ex.Server(model)
    whole = [server.cache.open() for _ in rows]
    a = server.step(whole, [r.tolist() for r in rows]).reshape(4, 96, -1)
    parts = [server.cache.open() for _ in rows]
    b, at = [], 0
    for n in (30, 1, 1, 40, 17, 1, 6):
        b.append(server.step(parts, [r[at:at + n].tolist() for r in rows]).reshape(4, n, -1))
        at += n
    assert at == 96
    b = torch.cat(b, 1)
    with torch.no_grad():
        full = model(rows.to(dev))
    print(f"[decoder] chunks against whole {_rel(b, a):.2e}, served against model "
          f"{_rel(a, full):.2e}", flush=True)
    # the model's attention is fp32 on unquantised keys and values; E4M3 has
    # 2^-4 half a step, some 2.5e-2 of a vector's norm, averaged over the keys
    assert _rel(b, a) < 0.05 and _rel(a, full) < 0.1
    for s in (*whole, *parts):
        server.cache.close(s)
    prompts = [r[:40 - i].tolist() for i, r in enumerate(rows)]
    got = server.generate(prompts, 40)
    right = sum(t == int(r[len(p) + j]) for r, p, o in zip(rows, prompts, got)
                for j, t in enumerate(o))
    print(f"[decoder] {right} of 160 tokens follow the rule", flush=True)
    assert right >= 144
    assert server.cache.free_pages == 256
