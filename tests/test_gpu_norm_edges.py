"""The norm at the edges of its shapes."""
import pytest
import torch

from tcfp_amd import norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(0,), (1, 0), (5, 0), (2, 3, 0), (1500, 0), (0, 0)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("residual", [False, True])
def test_rows_without_columns(dev, shape, dtype, residual):
    """1 / sqrt(mean + eps) of no values is NaN, as torch's mean of nothing is,
    in every row; the other outputs are empty."""
    x, w = torch.empty(shape, dtype=dtype, device=dev), torch.empty(0, device=dev)
    r = torch.empty_like(x) if residual else None
    want = torch.rsqrt(x.float().square().mean(-1) + 1e-6)
    assert want.isnan().all()
    for call in (lambda: norm.rms_norm(x, w, r), lambda: norm.rms_norm_quantize(x, w, r)):
        # (finite values where the outputs may be allocated)
        old = [torch.full((max(want.numel(), 1),), 7.0, device=dev) for _ in range(8)]
        del old
        *out, rstd = call()
        assert rstd.shape == want.shape and rstd.isnan().all()
        assert out[0].shape == x.shape and out[-1].shape == x.shape
    dx, dw = norm.rms_norm_backward(x, x, rstd, w, r)
    assert dx.shape == x.shape and dw.shape == (0,)
    with pytest.raises(ValueError, match="rstd must hold"):
        norm.rms_norm_backward(x, x, torch.ones(4000, device=dev), w)
