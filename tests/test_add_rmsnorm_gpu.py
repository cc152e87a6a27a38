"""kiln_add_rmsnorm and the MXFP8 rows against 64 bits: types, widths about a chunk's and a wave's, strides, in place, values out of fp32's
squares, and MXFP8 codes bit by bit."""

import math

import pytest
import torch

import kiln_amd as ka

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
EPS = 1e-6


def window(rows, cols, dt, extra=0, off=0):
    """[rows, cols] inside rows of cols + extra elements, off elements in; the rest holds 5."""
    buf = torch.full((rows, cols + extra), 5.0, dtype=dt, device=DEV)
    return buf, buf[:, off:off + cols]


def reference(x, res, w, eps=EPS):
    h = x.double() + (res.double() if res is not None else 0)
    return h, h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * (w.double() if w is not None else 1)


def u(dt):
    return torch.finfo(dt).eps / 2


def close(got, ref, dt, rel, what):
    tol = (u(dt) * (1 + rel) + rel) * ref.abs() + torch.finfo(dt).smallest_normal * u(dt)
    err = (got.double() - ref).abs()
    assert torch.isfinite(got).all(), what
    assert (err <= tol).all(), (what, (err / tol).max().item())


def norm_rel(dim):
    """Relative error of the fp32 arithmetic: h 2^-24; its square, chains of 32 to 64 sums a lane, 6 across lanes and 16 across waves, all of
    positive terms, half of it in the root; root, division, two products: 2^-24 each (and the weight's product)."""
    return (1 + (2 + 64 + 6 + 16) / 2 + 8) * 2.0 ** -24


DIMS = [1, 7, 8, 31, 32, 64, 500, 512, 520, 1000, 1024, 1032, 2048, 2080, 4096, 5120, 8192, 9000, 16384, 20000, 32768]


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("x,r,y", [(F16, F32, F16), (BF16, F32, BF16), (F32, F32, F32), (F16, None, F16), (F32, None, BF16), (BF16, BF16, BF16),
                                   (F32, F16, F32), (F16, BF16, F32), (BF16, None, F32), (BF16, F16, F16)])
def test_types_and_widths(gpu, dim, x, r, y):
    g = torch.Generator(device=DEV).manual_seed(dim)
    for rows, extra, off in ((1, 0, 0), (5, 0, 0), (9, 8, 0), (6, 5, 3)):
        def randn(dt):
            buf, t = window(rows, dim, dt, extra, off)
            t.copy_(torch.randn(rows, dim, generator=g, device=DEV) * torch.exp(torch.randn(dim, generator=g, device=DEV)))
            return t
        X, R = randn(x), None if r is None else randn(r)
        w = (1 + torch.randn(dim, generator=g, device=DEV) / 4).to(BF16) if rows != 5 else None
        hb, H = window(rows, dim, r or F32, extra, off)
        yb, Y = window(rows, dim, y, extra, off)
        ka.add_rmsnorm(Y, X, R, w, h=H if r else None)
        h, ref = reference(X, R, w)
        close(Y, ref, y, norm_rel(dim), f"y {rows}x{dim} {x} {r} {y}")
        if r is not None:
            close(H, h, r, 2.0 ** -24, "h")
        for buf in (yb, hb):
            rest = torch.ones(dim + extra, dtype=torch.bool, device=DEV)
            rest[off:off + dim] = False
            assert (buf[:, rest] == 5).all()


def test_in_place(gpu):
    for dt in (F32, F16, BF16):
        x, r = torch.randn(33, 2048, device=DEV).to(dt), torch.randn(33, 2048, device=DEV)
        w = torch.randn(2048, device=DEV).to(BF16)
        y, h = torch.empty_like(x), torch.empty_like(r)
        ka.add_rmsnorm(y, x, r, w, h=h)
        x2, r2 = x.clone(), r.clone()
        ka.add_rmsnorm(x2, x2, r2, w)
        assert torch.equal(x2, y) and torch.equal(r2, h)


@pytest.mark.parametrize("dim", [64, 2048, 4096, 20000])
def test_large_and_small_values(gpu, dim):
    """Squares beyond fp32's range; rows of zeros and of values whose squares vanish; eps that counts."""
    x = torch.randn(6, dim, device=DEV)
    x[0] *= 1e25
    x[1] *= 1e37
    x[2] = 0
    x[3] *= 1e-30
    x[4] *= 1e-3
    y = torch.empty_like(x)
    ka.add_rmsnorm(y, x)
    _, ref = reference(x, None, None)
    tol = 2 * norm_rel(dim) * ref.abs() + 2.0 ** -149
    assert ((y.double() - ref).abs() <= tol).all()
    assert (y[2] == 0).all()


def test_infinities_and_nans_stay_in_their_row(gpu):
    x = torch.randn(4, 512, device=DEV)
    x[1, 7], x[2, 9] = math.inf, math.nan
    y = torch.empty_like(x)
    ka.add_rmsnorm(y, x)
    assert torch.isfinite(y[0]).all() and torch.isfinite(y[3]).all()
    assert torch.isnan(y[2]).all() and torch.isnan(y[1, 7]) and (y[1, :7] == 0).all()


# ---- MXFP8 ----

def mx8(x):
    """Codes and scales by the definition, in 64 bits: the smallest power of two (not below 2^-127) with the largest magnitude at most 448
    times it; the nearest of the 127 magnitudes, ties to the even code."""
    b = x.double().reshape(x.shape[0], -1, 32)
    top = b.abs().amax(-1, keepdim=True)
    ok = torch.isfinite(top)
    e = torch.ceil(torch.log2(torch.where(ok & (top > 0), top, 1.0) / 448))
    for _ in range(2):  # log2's own rounding
        e = torch.where(torch.where(ok, top, 0.0) > 448 * torch.exp2(e), e + 1, e)
        e = torch.where((top <= 224 * torch.exp2(e)) & ok, e - 1, e)
    e = torch.where(top == 0, -127.0, e).clamp(min=-127)
    grid = torch.arange(127, dtype=torch.uint8, device=x.device).view(torch.float8_e4m3fn).double()
    mid = (grid[1:] + grid[:-1]) / 2
    a = (b.abs() / torch.exp2(e)).contiguous()
    i = torch.bucketize(a, mid)
    i = i + ((i < 126) & (a == mid[i.clamp(max=125)]) & (i % 2 == 1))
    codes = i + 128 * torch.signbit(b)
    codes = torch.where(ok, codes, 0).to(torch.uint8).view(x.shape)
    return codes, torch.where(ok, e + 127, 255.0).to(torch.uint8).view(x.shape[0], -1)


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("rows,cols,extra", [(1, 32, 0), (3, 64, 3), (77, 1024, 0), (50, 2080, 8), (1000, 96, 0), (1, 8192, 0)])
def test_mxfp8_codes(gpu, dt, rows, cols, extra):
    g = torch.Generator(device=DEV).manual_seed(rows)
    _, x = window(rows, cols, dt, extra)
    x.copy_(torch.randn(rows, cols, generator=g, device=DEV) * torch.exp(3 * torch.randn(cols, generator=g, device=DEV)))
    codes, scales = ka.mxfp8_quantize(x)
    want_c, want_s = mx8(x)
    assert torch.equal(scales, want_s) and torch.equal(codes, want_c)
    for out in (F32, F16, BF16):
        yb, y = window(rows, cols, out, extra)
        ka.mxfp8_dequantize(y, codes, scales)
        ref = want_c.view(torch.float8_e4m3fn).double() * torch.exp2(want_s.double() - 127).repeat_interleave(32, 1)
        ref = torch.where((want_s == 255).repeat_interleave(32, 1), math.nan, ref)  # (some fp16 inputs are infinite)
        assert torch.allclose(y.double(), ref.to(out).double(), rtol=0, atol=0, equal_nan=True)
        assert (yb[:, cols:] == 5).all()


def test_mxfp8_borders(gpu):
    """Every border between neighbouring codes and its two neighbours in fp32; largest magnitudes about 448 times a power of two; the ends
    of fp32's range; zeros of both signs; infinities and NaNs."""
    grid = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    mid = (grid[1:] + grid[:-1]) / 2
    vals = torch.cat([grid, mid, torch.nextafter(mid, torch.tensor(0.0)), torch.nextafter(mid, torch.tensor(1e9))])
    vals = torch.cat([vals, -vals])
    n = (len(vals) + 30) // 31
    x = torch.zeros(n, 32)
    x[:, 31] = 448.0  # fixes the scale at 1
    flat = torch.zeros(n * 31)
    flat[:len(vals)] = vals
    x[:, :31] = flat.view(n, 31)
    tops = []
    for e in (-149, -140, -133, -127, -126, -119, -118, -60, -1, 0, 1, 60, 118, 119):
        for m in (1.0, 1.5, 1.75, 1.7500001, 1.99):
            tops.append(torch.full((32,), m * 2.0 ** e, dtype=torch.float64).float() * torch.linspace(0, 1, 32))
    y = torch.cat([x, torch.stack(tops), torch.tensor([[-0.0] * 16 + [0.0] * 16]), torch.full((1, 32), math.inf), torch.full((1, 32), math.nan)])
    y[-2, 1:], y[-1, 3:] = 1.0, 2.0
    y = y.to(DEV)
    codes, scales = ka.mxfp8_quantize(y)
    want_c, want_s = mx8(y)
    bad = (codes != want_c).any(1) | (scales != want_s).any(1)
    assert not bad.any(), (y[bad][:3], codes[bad][:3], want_c[bad][:3], scales[bad][:3], want_s[bad][:3])
    out = torch.empty_like(y)
    ka.mxfp8_dequantize(out, codes, scales)
    assert torch.isnan(out[-2:]).all()
    ref = want_c[:-2].view(torch.float8_e4m3fn).double() * torch.exp2(want_s[:-2].double() - 127)
    assert torch.equal(out[:-2].double(), ref)


@pytest.mark.parametrize("dim", [32, 64, 992, 1024, 2048, 2080, 5120, 8192, 32768])
@pytest.mark.parametrize("x,r", [(F16, F32), (BF16, None), (F32, F16)])
def test_norm_to_mxfp8(gpu, dim, x, r):
    """The codes of the fp32 norm are within half a step of the 64-bit norm, its scales those of it (a value within the norm's own error
    of a border may go either way)."""
    g = torch.Generator(device=DEV).manual_seed(dim)
    X = torch.randn(21, dim, generator=g, device=DEV).to(x)
    R = None if r is None else (3 * torch.randn(21, dim, generator=g, device=DEV)).to(r)
    w = (1 + torch.randn(dim, generator=g, device=DEV) / 4).to(BF16)
    codes = torch.empty(21, dim, dtype=torch.uint8, device=DEV)
    scales = torch.empty(21, dim // 32, dtype=torch.uint8, device=DEV)
    H = None if R is None else torch.empty_like(R)
    ka.add_rmsnorm(codes, X, R, w, h=H, scales=scales)
    h, ref = reference(X, R, w)
    if R is not None:
        close(H, h, r, 2.0 ** -24, "h")
    rel = norm_rel(dim)
    lo, hi = mx8((ref * (1 - rel)))[1], mx8((ref * (1 + rel)))[1]
    assert ((scales == lo) | (scales == hi)).all()
    sc = torch.exp2(scales.double() - 127).repeat_interleave(32, 1)
    got = codes.view(torch.float8_e4m3fn).double() * sc
    # half a step: 2^-4 of the value's power of two, at least half of 2^-9 scales
    step = torch.exp2(torch.floor(torch.log2((ref.abs() / sc).clamp(min=2.0 ** -6))) - 3) * sc
    assert ((got - ref).abs() <= step / 2 * (1 + 1e-6) + 2 * rel * ref.abs()).all()


def test_norm_to_mxfp8_is_the_norm_and_its_codes(gpu):
    """The fused codes equal those of the fp32 output, value by value."""
    x, r = torch.randn(300, 2048, device=DEV).half(), torch.randn(300, 2048, device=DEV)
    w = torch.randn(2048, device=DEV).to(BF16)
    y, h = torch.empty(300, 2048, device=DEV), torch.empty_like(r)
    ka.add_rmsnorm(y, x, r, w, h=h)
    codes, scales = torch.empty(300, 2048, dtype=torch.uint8, device=DEV), torch.empty(300, 64, dtype=torch.uint8, device=DEV)
    ka.add_rmsnorm(codes, x, r, w, h=h, scales=scales)
    c, s = ka.mxfp8_quantize(y)
    assert torch.equal(c, codes) and torch.equal(s, scales)


def test_capture(gpu):
    x, r = torch.randn(40, 1024, device=DEV).half(), torch.randn(40, 1024, device=DEV)
    y, h = torch.empty_like(x), torch.empty_like(r)
    ka.add_rmsnorm(y, x, r, h=h)
    eager = y.clone(), h.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ka.add_rmsnorm(y, x, r, h=h)
    for _ in range(3):
        y.zero_()
        h.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, eager[0]) and torch.equal(h, eager[1])


@pytest.mark.parametrize("dim", [96, 2048, 32768])
def test_rows_of_the_largest_values(gpu, dim):
    """Sums of squares beyond fp32, up to full rows of fp32's largest values: h / rms(h) is then 1, off by the roundings of a sum, a division, a root
    and two products."""
    top = torch.finfo(torch.float32).max
    x = torch.full((3, dim), top, device=DEV)
    x[1] *= -1
    x[2, 1:] = 2.0 ** 60
    y = torch.empty_like(x)
    ka.add_rmsnorm(y, x)
    want = torch.ones_like(x, dtype=torch.float64)
    want[1] = -1
    want[2] = 2.0 ** 60 / (top / dim ** 0.5)
    want[2, 0] = dim ** 0.5
    # a sum of dim terms over 64 lanes at least: dim / 64 + 10 roundings and as many of the squares
    tol = (dim / 64 + 20) * 2.0 ** -24
    assert ((y.double() - want).abs() <= tol * want.abs()).all()
