"""Residual + RMS norm (plain and FP8 output) and its backward against the
formulas in 64 bits.

Tolerances: an fp32 sum of D <= 32768 squares in partial sums of at most 512
terms is within 512 * 2^-24 = 3e-5 of the exact one in the worst case and some
1e-6 of it for values of random size, and rstd has half of that; y adds three
roundings of 2^-24.  2e-6 (relative, per element) is asked of y and rstd, 2^-8
more of what is rounded to bf16.  Sums over rows: chains of at most 512
additions, 512 * 2^-24 of the sum of magnitudes."""
import pytest
import torch

from tcfp_amd import kernels as K
from tcfp_amd import norm

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2
EPS = 1e-6


def _bits(t):
    return t.contiguous().view(torch.uint8)


def _inputs(dev, m, d, xt, rt, seed=0):
    g = torch.Generator().manual_seed(seed)
    chan = torch.exp(0.5 * torch.randn(d, generator=g))
    x = (torch.randn(m, d, generator=g) * chan).to(xt).to(dev)
    r = None if rt is None else (torch.randn(m, d, generator=g) * chan).to(rt).to(dev)
    w = (1 + 0.1 * torch.randn(d, generator=g)).to(dev)
    return x, r, w


def _exact(x, r, w):
    s = x.double() if r is None else x.double() + r.double()
    rstd = 1 / torch.sqrt((s * s).mean(-1, keepdim=True) + EPS)
    return s, rstd[..., 0], s * rstd * w.double()


SIZES = [(1, 32), (1, 4096), (3, 1), (2, 7), (5, 96), (7, 257), (33, 1056), (64, 256), (130, 512),
         (16, 1000), (17, 2080), (40, 4096), (9, 5120), (3, 8192), (2, 16384), (2, 20000),
         (2, 32768)]


@pytest.mark.parametrize("m,d", SIZES)
@pytest.mark.parametrize("xt,rt", [(F32, None), (BF16, None), (F32, F32), (BF16, BF16),
                                   (F32, BF16), (BF16, F32)])
def test_plain_output(dev, m, d, xt, rt):
    print(f"[norm] {m} x {d} {xt} {rt}", flush=True)
    x, r, w = _inputs(dev, m, d, xt, rt)
    s, rstd, y = _exact(x, r, w)
    for out, wt in ((F32, F32), (BF16, BF16)):
        wo = w.to(wt)
        yo = y if wt == F32 else s * rstd[:, None] * wo.double()
        got, h, rs = norm.rms_norm(x, wo, r, eps=EPS, out_dtype=out)
        assert got.dtype == out and rs.dtype == F32 and rs.shape == (m,)
        tol = 2e-6 if out == F32 else 2e-6 + 2**-8
        assert ((got.double() - yo).abs() <= tol * yo.abs() + 1e-37).all()
        assert ((rs.double() - rstd).abs() <= 2e-6 * rstd).all()
        if r is None:
            assert h is x
        else:
            assert h.dtype == rt
            assert torch.equal(h, (x.float() + r.float()).to(rt))


@pytest.mark.parametrize("m,d", [s for s in SIZES if s[1] % 32 == 0])
@pytest.mark.parametrize("xt,rt", [(F32, None), (BF16, BF16), (F32, BF16)])
def test_codes_are_the_block_quantisation_of_the_norm(dev, m, d, xt, rt):
    print(f"[norm] codes {m} x {d} {xt} {rt}", flush=True)
    x, r, w = _inputs(dev, m, d, xt, rt, seed=1)
    y, h0, rs0 = norm.rms_norm(x, w, r, eps=EPS, out_dtype=F32)
    _, _, exact = _exact(x, r, w)
    for bs in (32, 64, 128):
        if d % bs:
            continue
        for fmt in (E4M3, E5M2):
            for sf in ("exponent", "fp32"):
                q, sc, h, rs = norm.rms_norm_quantize(x, w, r, eps=EPS, block_size=bs,
                                                      fp8_dtype=fmt, scale_format=sf)
                q0, sc0 = K.block_quantize_fp8(y, bs, fmt, scale_format=sf)
                assert torch.equal(_bits(q), _bits(q0)) and torch.equal(sc, sc0)
                assert torch.equal(rs, rs0) and torch.equal(h, h0)
                mul = torch.exp2(sc.double()) if sf == "exponent" else sc.double()
                mul = mul.t().repeat_interleave(bs, 1)
                # half a step of the format: 2^-4 (E4M3) / 2^-3 (E5M2) of a
                # normal value, half the smallest subnormal else
                half, tiny = (2**-4, 2**-10) if fmt == E4M3 else (2**-3, 2**-17)
                err = (q.double() * mul - exact).abs()
                assert (err <= half * exact.abs() * (1 + 1e-5) + tiny * mul).all()


def test_rows_apart_and_misaligned(dev):
    """Slices of a wider matrix, at an address that no vector load takes."""
    g = torch.Generator().manual_seed(2)
    wide = torch.randn(20, 1400, generator=g).to(dev)
    w = torch.randn(1024, generator=g).to(dev)
    for dt in (F32, BF16):
        for at in (0, 1, 64):
            x, r = wide.to(dt)[:, at:at + 1024], wide.to(dt)[:, 300 + at:1324 + at]
            a = norm.rms_norm_quantize(x, w, r)
            b = norm.rms_norm_quantize(x.contiguous(), w, r.contiguous())
            for u, v in zip(a, b):
                assert torch.equal(_bits(u), _bits(v))
    ws = torch.cat([w[:1], w])[1:]  # a weight off its alignment
    x = wide[:, :1024]
    assert torch.equal(norm.rms_norm(x, w)[0], norm.rms_norm(x, ws)[0])


def test_leading_dimensions_and_empty(dev):
    x = torch.randn(2, 3, 64, device=dev)
    w = torch.ones(64, device=dev)
    q, s, h, rs = norm.rms_norm_quantize(x, w, x)
    assert q.shape == (2, 3, 64) and s.shape == (1, 6) and rs.shape == (2, 3)
    assert h.shape == x.shape
    xt = x.transpose(0, 1)
    assert torch.equal(norm.rms_norm(xt, w)[0], norm.rms_norm(xt.contiguous(), w)[0])
    e = x[:0]
    q, s, h, rs = norm.rms_norm_quantize(e, w, e)
    assert q.shape == (0, 3, 64) and s.shape == (1, 0) and rs.shape == (0, 3)
    dx, dw = norm.rms_norm_backward(e, h, rs, w)
    assert dx.shape == e.shape and torch.equal(dw, torch.zeros(64, device=dev))


def test_zeros_and_values_that_are_not_finite(dev):
    x = torch.zeros(4, 128, device=dev)
    x[1, 3], x[2, 5] = float("nan"), float("inf")
    x[3] = 1e-30
    w = torch.ones(128, device=dev)
    y, _, rs = norm.rms_norm(x, w)
    assert torch.equal(y[0], torch.zeros(128, device=dev)) and y[1].isnan().all()
    assert y[2, 5].isnan() and (y[2, :5] == 0).all()
    assert torch.isfinite(y[3]).all() and float(rs[0]) == pytest.approx(1e3, rel=1e-5)
    for sf in ("exponent", "fp32"):
        q, s, _, _ = norm.rms_norm_quantize(x, w, scale_format=sf)
        q0, s0 = K.block_quantize_fp8(y, 64, scale_format=sf)
        assert torch.equal(q.float().isnan(), q0.float().isnan())
        assert torch.equal(q.float().nan_to_num(), q0.float().nan_to_num())
        assert torch.equal(s.float().nan_to_num(7.0), s0.float().nan_to_num(7.0))


@pytest.mark.parametrize("m,d", [*SIZES, (1000, 1056), (3000, 256), (700, 4096)])
@pytest.mark.parametrize("ht,gt,add", [(F32, F32, True), (BF16, BF16, True), (F32, BF16, False),
                                       (BF16, F32, False), (BF16, BF16, False)])
def test_backward(dev, m, d, ht, gt, add):
    print(f"[norm] backward {m} x {d} {ht} {gt}", flush=True)
    g = torch.Generator().manual_seed(3)
    h, _, w = _inputs(dev, m, d, ht, None, seed=3)
    _, _, rs = norm.rms_norm(h, w, eps=EPS)
    gy = torch.randn(m, d, generator=g).to(gt).to(dev)
    gh = torch.randn(m, d, generator=g).to(ht).to(dev) if add else None
    for wt in (F32, BF16):
        dx, dw = norm.rms_norm_backward(gy, h, rs, w.to(wt), gh)
        hd, gd, rd, wd = h.double(), gy.double(), rs.double()[:, None], w.to(wt).double()
        xh, gg = hd * rd, gd * wd
        mean = (gg * xh).mean(1, keepdim=True)
        exact = rd * (gg - xh * mean)
        size = rd * (gg.abs() + xh.abs() * (gg * xh).abs().mean(1, keepdim=True))
        if add:
            exact, size = exact + gh.double(), size + gh.double().abs()
        tol = 4e-6 * size + (2**-8 * exact.abs() if ht == BF16 else 0)
        assert dx.dtype == ht and ((dx.double() - exact).abs() <= tol + 1e-37).all()
        dwe, mag = (gd * xh).sum(0), (gd * xh).abs().sum(0)
        assert dw.dtype == F32 and ((dw.double() - dwe).abs() <= 512 * 2**-24 * mag + 1e-37).all()
        again = norm.rms_norm_backward(gy, h, rs, w.to(wt), gh)
        assert torch.equal(dx, again[0]) and torch.equal(dw, again[1])
    dx2, none = norm.rms_norm_backward(gy, h, rs, w.to(wt), gh, need_weight_grad=False)
    assert none is None and torch.equal(dx2, dx)


# Widths of every number of threads a row may have, two vectors a thread (one at
# 512), in more than 1024 rows: so few that the input may be cached, and so many
# that it is read past the caches.
WIDE = [512, 1024, 1056, 2080, 4096, 8192, 16384]


def _large(dev, d, many, bytes_each, seed):
    m = (100 << 20) // (d * bytes_each) + 7 if many else 1100
    g = torch.Generator(dev).manual_seed(seed)
    return m, lambda dt: torch.randn(m, d, generator=g, device=dev).to(dt)


@pytest.mark.parametrize("d", WIDE)
@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("xt,rt", [(F32, None), (BF16, None), (F32, F32), (BF16, BF16),
                                   (F32, BF16), (BF16, F32)])
def test_many_rows(dev, d, many, xt, rt):
    each = sum({F32: 4, BF16: 2}[t] for t in (xt, rt) if t is not None)
    m, rand = _large(dev, d, many, each, 7)
    print(f"[norm] {m} x {d} {xt} {rt}", flush=True)
    x, r = rand(xt), None if rt is None else rand(rt)
    w = 1 + 0.1 * torch.randn(d, device=dev)
    y, h, rs = norm.rms_norm(x, w, r, eps=EPS, out_dtype=F32)
    _, rstd, exact = _exact(x, r, w)
    assert ((rs.double() - rstd).abs() <= 2e-6 * rstd).all()
    assert ((y.double() - exact).abs() <= 2e-6 * exact.abs() + 1e-37).all()
    if r is not None:
        assert torch.equal(h, (x.float() + r.float()).to(rt))
    del exact
    for bs, sf in ((32, "exponent"), (32, "fp32")):
        q, sc, hq, rq = norm.rms_norm_quantize(x, w, r, eps=EPS, block_size=bs, scale_format=sf)
        q0, sc0 = K.block_quantize_fp8(y, bs, E4M3, scale_format=sf)
        assert torch.equal(_bits(q), _bits(q0)) and torch.equal(sc, sc0)
        assert torch.equal(rq, rs) and torch.equal(hq, h)


@pytest.mark.parametrize("m,d", [*(s for s in SIZES if s[1] % 32 == 0), (40, 1024)])
@pytest.mark.parametrize("xt,rt", [(BF16, F32), (F32, F32), (BF16, None), (F32, BF16)])
def test_codes_of_other_types(dev, m, d, xt, rt):
    test_codes_are_the_block_quantisation_of_the_norm(dev, m, d, xt, rt)


@pytest.mark.parametrize("d", WIDE)
@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("ht,gt", [(F32, F32), (BF16, BF16), (F32, BF16), (BF16, F32)])
def test_backward_of_many_rows(dev, d, many, ht, gt):
    size = {F32: 4, BF16: 2}
    m, rand = _large(dev, d, many, size[gt] + 2 * size[ht], 8)
    print(f"[norm] backward {m} x {d} {ht} {gt}", flush=True)
    h, gy, gh = rand(ht), rand(gt), rand(ht)
    w = 1 + 0.1 * torch.randn(d, device=dev)
    _, _, rs = norm.rms_norm(h, w, eps=EPS)
    dx, dw = norm.rms_norm_backward(gy, h, rs, w, gh)
    rd = rs.double()[:, None]
    gd, xh = gy.double(), h.double() * rd
    dwe, mag = (gd * xh).sum(0), (gd * xh).abs().sum(0)
    # chains of at most 512 additions on the way to a sum of m rows
    assert ((dw.double() - dwe).abs() <= 512 * 2**-24 * mag + 1e-37).all()
    gg = gd * w.double()
    exact = rd * (gg - xh * (gg * xh).mean(1, keepdim=True)) + gh.double()
    far = rd * (gg.abs() + xh.abs() * (gg * xh).abs().mean(1, keepdim=True)) + gh.double().abs()
    tol = 4e-6 * far + (2**-8 * exact.abs() if ht == BF16 else 0)
    assert ((dx.double() - exact).abs() <= tol + 1e-37).all()
    again = norm.rms_norm_backward(gy, h, rs, w, gh)
    assert torch.equal(dx, again[0]) and torch.equal(dw, again[1])


def test_backward_of_1030_rows(dev):
    """Two vectors a thread of 512, from inputs that may be cached."""
    test_backward(dev, 1030, 5120, F32, F32, True)


def test_backward_against_differences(dev):
    """Central differences of the formula in 64 bits, step 1e-5: exact to some
    1e-9; the fp32 gradient to 1e-5 of its largest value."""
    g = torch.Generator().manual_seed(4)
    m, d = 3, 40
    x = torch.randn(m, d, generator=g, dtype=torch.float64)
    w = 1 + 0.1 * torch.randn(d, generator=g, dtype=torch.float64)
    gy = torch.randn(m, d, generator=g, dtype=torch.float64)
    x, w, gy = (t.float().double() for t in (x, w, gy))

    def loss(x, w):
        return (gy * x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w).sum()

    num_x, num_w = torch.zeros_like(x), torch.zeros_like(w)
    for t, out in ((x, num_x), (w, num_w)):
        flat, res = t.view(-1), out.view(-1)
        for i in range(flat.numel()):
            old = float(flat[i])
            flat[i] = old + 1e-5
            up = float(loss(x, w))
            flat[i] = old - 1e-5
            res[i] = (up - float(loss(x, w))) / 2e-5
            flat[i] = old
    xd, wd = x.float().to(dev), w.float().to(dev)
    _, h, rs = norm.rms_norm(xd, wd, eps=EPS)
    dx, dw = norm.rms_norm_backward(gy.float().to(dev), h, rs, wd)
    assert (dx.cpu().double() - num_x).abs().max() <= 1e-5 * num_x.abs().max()
    assert (dw.cpu().double() - num_w).abs().max() <= 1e-5 * num_w.abs().max()


def test_on_another_stream_and_in_a_graph(dev):
    x, r, w = _inputs(dev, 64, 1024, BF16, BF16, seed=5)
    gy = torch.randn(64, 1024, device=dev).bfloat16()
    want = norm.rms_norm_quantize(x, w, r)
    back = norm.rms_norm_backward(gy, want[2], want[3], w, gy)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = norm.rms_norm_quantize(x, w, r)
        gback = norm.rms_norm_backward(gy, got[2], got[3], w, gy)
    torch.cuda.synchronize()
    for u, v in zip((*want, *back), (*got, *gback)):
        assert torch.equal(_bits(u), _bits(v))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = norm.rms_norm_quantize(x, w, r)
        gback = norm.rms_norm_backward(gy, got[2], got[3], w, gy)
    for i in range(3):
        x.mul_(1.5)
        want = norm.rms_norm_quantize(x, w, r)
        back = norm.rms_norm_backward(gy, want[2], want[3], w, gy)
        graph.replay()
        torch.cuda.synchronize()
        for u, v in zip((*want, *back), (*got, *gback)):
            assert torch.equal(_bits(u), _bits(v)), i


def test_refusals(dev):
    x, w = torch.zeros(2, 64, device=dev), torch.ones(64, device=dev)
    with pytest.raises(RuntimeError, match="only on the GPU"):
        norm.rms_norm(x.cpu(), w.cpu())
    with pytest.raises(RuntimeError, match="only on the GPU"):
        norm.rms_norm(x, w.cpu())
    with pytest.raises(TypeError, match="unsupported input dtype"):
        norm.rms_norm(x.half(), w)
    with pytest.raises(TypeError, match="unsupported output dtype"):
        norm.rms_norm(x, w, out_dtype=torch.float16)
    with pytest.raises(ValueError, match="weight must have shape"):
        norm.rms_norm(x, w[:32])
    with pytest.raises(ValueError, match="residual shape"):
        norm.rms_norm(x, w, x[:1])
    with pytest.raises(ValueError, match="at least one dimension"):
        norm.rms_norm(x[0, 0], w)
    with pytest.raises(ValueError, match="block_size must be"):
        norm.rms_norm_quantize(x, w, block_size=48)
    with pytest.raises(ValueError, match="must be divisible by block_size"):
        norm.rms_norm_quantize(x, w, block_size=128)
    with pytest.raises(ValueError, match="scale_format"):
        norm.rms_norm_quantize(x, w, scale_format="int")
    with pytest.raises(TypeError, match="unsupported fp8 dtype"):
        norm.rms_norm_quantize(x, w, fp8_dtype=torch.float16)
    rs = torch.ones(2, device=dev)
    with pytest.raises(ValueError, match="grad_y shape"):
        norm.rms_norm_backward(x[:1], x, rs, w)
    with pytest.raises(ValueError, match="rstd must hold"):
        norm.rms_norm_backward(x, x, rs[:1], w)
    with pytest.raises(ValueError, match="grad_h shape"):
        norm.rms_norm_backward(x, x, rs, w, x[:1])
    with pytest.raises(TypeError, match="grad_h must have"):
        norm.rms_norm_backward(x, x, rs, w, x.bfloat16())
