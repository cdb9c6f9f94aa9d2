"""The gradients that TCFPNormLinear and TCFPRMSNorm hand back, with the kernels
replaced by plain arithmetic (no GPU needed): tensors that the caller may change
in place, whatever else holds them."""
import pytest
import torch

from tcfp_amd import nn as tn
from tcfp_amd.nn import TCFPNormLinear, TCFPRMSNorm


def _norm(x, weight, residual=None, *, eps=1e-6, out_dtype=None):
    s = x.float() if residual is None else x.float() + residual.float()
    rstd = torch.rsqrt(s.square().mean(-1) + eps)
    h = x if residual is None else s.to(residual.dtype)
    return (s * rstd[..., None] * weight).to(out_dtype or x.dtype), h, rstd


def _norm_backward(grad_y, h, rstd, weight, grad_h=None, *, need_weight_grad=True):
    xh = h.float() * rstd[..., None]
    g = grad_y.float() * weight
    dx = rstd[..., None] * (g - xh * (g * xh).mean(-1, keepdim=True))
    if grad_h is not None:
        dx = dx + grad_h.float()
    dw = (grad_y.float() * xh).reshape(-1, xh.shape[-1]).sum(0)
    return dx.to(h.dtype), dw if need_weight_grad else None


@pytest.fixture
def plain(monkeypatch):
    """The ops under the two modules in plain arithmetic, nothing quantised."""
    one = torch.ones(1)
    monkeypatch.setattr(tn.N, "rms_norm", _norm)
    monkeypatch.setattr(tn.N, "rms_norm_backward", _norm_backward)

    def quantize(x, weight, residual=None, *, eps, block_size):
        y, h, rstd = _norm(x, weight, residual, eps=eps, out_dtype=torch.float32)
        return y, one, h, rstd

    monkeypatch.setattr(tn.N, "rms_norm_quantize", quantize)
    monkeypatch.setattr(tn.K, "fused_dual_quantize_fp8",
                        lambda w, *a, **k: (w.detach().clone(), one, one, one))
    monkeypatch.setattr(
        tn.K, "fused_block_scaled_dual_gemm_forward",
        lambda q, hi, lo, e, sh, sl, bs, bias=None: torch.nn.functional.linear(q, hi, bias))

    def layer_backward(ctx, grad):
        q, _, w_hi, *_ = ctx.saved_tensors
        g = grad.reshape(-1, grad.shape[-1])
        need_dx, need_dw, need_db = ctx.needs_input_grad
        return (g @ w_hi if need_dx else None, g.t() @ q if need_dw else None,
                g.sum(0) if need_db else None)

    monkeypatch.setattr(tn._TCFP12BlockScaledFunction, "backward", staticmethod(layer_backward))


def _storage(t):
    return t.untyped_storage().data_ptr()


def _module(kind):
    torch.manual_seed(0)
    return TCFPNormLinear(64, 64) if kind == "linear" else TCFPRMSNorm(64)


@pytest.mark.parametrize("kind", ["linear", "norm"])
@pytest.mark.parametrize("shape", [(6, 64), (2, 3, 64)])
@pytest.mark.parametrize("use", ["both", "out", "sum"])
def test_gradients_of_input_and_residual_are_apart(plain, kind, shape, use):
    """Leaves x and residual of one dtype: gradients in storages of their own,
    not the caller's either, and twice one pass after two."""
    m = _module(kind)
    x, r = (torch.randn(shape, requires_grad=True) for _ in range(2))
    gy, gh = torch.randn(shape), torch.randn(shape)
    kept = gy.clone(), gh.clone()

    def backward():
        out, h = m(x, r)
        pairs = {"both": ([out, h], [gy, gh]), "out": ([out], [gy]), "sum": ([h], [gh])}
        torch.autograd.backward(*pairs[use])

    backward()
    assert _storage(x.grad) != _storage(r.grad)
    assert not {_storage(x.grad), _storage(r.grad)} & {_storage(gy), _storage(gh)}
    once = x.grad.clone()
    assert torch.equal(r.grad, once)
    backward()
    assert torch.equal(x.grad, 2 * once) and torch.equal(r.grad, 2 * once)
    x.grad.zero_()
    assert torch.equal(r.grad, 2 * once)
    assert torch.equal(gy, kept[0]) and torch.equal(gh, kept[1])


@pytest.mark.parametrize("kind", ["linear", "norm"])
@pytest.mark.parametrize("shape", [(6, 64), (2, 3, 64)])
@pytest.mark.parametrize("residual", [False, True])
def test_gradients_under_other_dtypes_and_uses(plain, kind, shape, residual):
    """Another dtype of the input, one leaf only, and one tensor as both."""
    m = _module(kind)
    base, rest = torch.randn(shape), torch.randn(shape)
    got = {}
    for name, x in (("fp32", base), ("bf16", base.bfloat16())):
        x = x.detach().clone().requires_grad_(True)
        r = rest.clone() if residual else None
        out = m(x, r) if residual else (m(x),)
        out[0].float().sum().backward()
        got[name] = x.grad
        assert x.grad.dtype == x.dtype and x.grad.shape == x.shape
    far = (got["fp32"] - got["bf16"].float()).abs().max()
    assert far <= 0.05 * got["fp32"].abs().max() + 1e-3
    if residual:
        x = base.clone().requires_grad_(True)
        out, h = m(x, x)
        (out.sum() + h.sum()).backward()
        y, z = (base.clone().requires_grad_(True) for _ in range(2))
        out, h = m(y, z)
        (out.sum() + h.sum()).backward()
        assert torch.equal(x.grad, y.grad + z.grad)
