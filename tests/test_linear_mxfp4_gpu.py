"""kiln_linear_mxfp4 against the 64-bit product of the MXFP4 values: sizes, types, epilogues, strides, few rows and tiles."""
import math

import pytest
import torch

import kiln_amd as ka
from tests import mxfp4_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPI = dict(f32=ka.KILN_EPI_F32, f16=ka.KILN_EPI_F16, gelu=ka.KILN_EPI_GELU16, resid=ka.KILN_EPI_RESID)


def mx(t):
    return torch.from_numpy(ref.values(*ref.quantize(t))).to(DEV)


def make(T, N, K, dt, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + 31 * T + N)
    x = (torch.randn(T, K, device=DEV, generator=g) * torch.exp(torch.randn(K, device=DEV, generator=g))).to(dt)
    w = (torch.randn(N, K, device=DEV, generator=g) / K ** 0.5).bfloat16()
    return x, w


def check(y, x, w, epi, what, y0=None, gate=None, beta=0.0):
    xq, wq = mx(x), mx(w)
    acc, mag = xq @ wq.t(), xq.abs() @ wq.abs().t()
    # every product is exact; each of the K / 128 matrix instructions and of the joins of up to eight partial sums rounds
    # within 2^-23 of the magnitudes summed so far
    tol = (math.ceil(x.shape[1] / 128) + 8) * 2.0 ** -23 * mag
    if epi == "gelu":
        out = acc * torch.special.ndtr(acc)
        # |GELU'| < 1.13; its own evaluation: v - v Phi(-v) for v > 0 and v Phi(v) otherwise, with Phi(-z) = 2^P(z) within
        # 2^-17 (test_gelu_polynomial); the exponential's 2^-22 and the fma's 2^-24 are in the bound's slack
        tol = 1.13 * tol + 2.0 ** -17 * out.abs() + 2.0 ** -24 * 1e-3
    elif epi == "resid":
        gt = torch.ones_like(acc[0]) if gate is None else gate.double()
        out = y0.double() + gt * acc
        tol = tol * gt.abs() + 2.0 ** -23 * (gt * acc).abs() + 2.0 ** -24 * out.abs()
    else:
        out = acc + (beta * y0.double() if beta else 0)
        if beta:
            tol = tol + 2.0 ** -23 * (beta * y0.double()).abs() + 2.0 ** -24 * out.abs()
    if y.dtype == torch.float16:
        tol = tol + 2.0 ** -11 * (out.abs() + tol) + 2.0 ** -25
    err = (y.double() - out).abs()
    print(f"[linear_mxfp4] {what}: worst error / tolerance {(err / tol.clamp(min=1e-300)).max():.3f}", flush=True)
    assert torch.isfinite(y).all()
    assert (err <= tol).all(), what


def out_of(epi, T, N):
    return torch.full((T, N), float("nan"), device=DEV, dtype=torch.float32 if epi in ("f32", "resid") else torch.float16)


SIZES = [(1, 16, 32), (1, 1, 32), (1, 2048, 2048), (2, 33, 64), (16, 128, 160), (17, 100, 96), (32, 2048, 8192), (33, 65, 1024),
                                   (64, 257, 128), (65, 257, 128), (65, 1, 32), (128, 128, 2048), (129, 130, 288), (300, 2048, 1024), (1537, 256, 512),
                                   (2048, 2048, 256), (257, 8192, 2048), (4100, 4100, 96), (2047, 8190, 640), (2048, 8192, 96)]
EPI_SIZES = [(1, 48, 64), (20, 130, 96), (50, 1024, 1024), (64, 2048, 1024), (70, 2048, 4096), (200, 129, 2048), (1000, 2048, 1024), (4352, 4352, 64),
             (300, 2048, 1024), (2047, 8190, 640)]


@pytest.mark.parametrize("sizes", [SIZES, EPI_SIZES])
def test_sizes_reach_every_tile(gpu, sizes):
    assert {ka.linear_mxfp4_tile(*s) for s in sizes} == {(16, 16), (16, 32), (16, 64), (32, 32), (64, 64), (128, 128), (256, 256)}


@pytest.mark.parametrize("T,N,K", SIZES)
@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16])
def test_sizes(gpu, T, N, K, dt):
    x, w = make(T, N, K, dt)
    W = ka.linear_mxfp4_weight(w)
    y = ka.linear_mxfp4(out_of("f32", T, N), x, W)
    check(y, x, w, "f32", f"{T} x {N} x {K} {dt}")
    assert torch.equal(y, ka.linear_mxfp4(out_of("f32", T, N), x, W))


@pytest.mark.parametrize("T,N,K", EPI_SIZES)
@pytest.mark.parametrize("epi", list(EPI))
def test_epilogues(gpu, T, N, K, epi):
    x, w = make(T, N, K, torch.float16, 5)
    W = ka.linear_mxfp4_weight(w)
    gate = torch.randn(N, device=DEV)
    y0 = torch.randn(T, N, device=DEV)
    if epi == "resid":
        check(ka.linear_mxfp4(y0.clone(), x, W, epi=EPI[epi], gate=gate), x, w, epi, f"{T} x {N} x {K} gated", y0, gate)
        check(ka.linear_mxfp4(y0.clone(), x, W, epi=EPI[epi]), x, w, epi, f"{T} x {N} x {K} residual", y0)
    else:
        check(ka.linear_mxfp4(out_of(epi, T, N), x, W, epi=EPI[epi]), x, w, epi, f"{T} x {N} x {K} {epi}")
    if epi == "f32":
        check(ka.linear_mxfp4(y0.clone(), x, W, beta=0.5), x, w, epi, f"{T} x {N} x {K} beta", y0, beta=0.5)


@pytest.mark.parametrize("T", [3, 150])
@pytest.mark.parametrize("epi", list(EPI))
@pytest.mark.parametrize("off,ldy,ldx", [(0, 72, 136), (1, 71, 129), (4, 68, 133), (2, 70, 131)])
def test_strides(gpu, T, epi, off, ldy, ldx):
    """Rows of x and y of every alignment; columns beside y's and rows around it keep what they held."""
    N, K = 66, 128
    xb = torch.randn(T * ldx + off, device=DEV).half()
    x = xb[off:off + T * ldx].view(T, ldx)[:, :K]
    _, w = make(T, N, K, torch.float16)
    dt = torch.float32 if epi in ("f32", "resid") else torch.float16
    yb = torch.full((T * ldy + off + 64,), 2.0, device=DEV, dtype=dt)
    y = yb[off:off + T * ldy].view(T, ldy)[:, :N]
    y0 = y.clone()
    ka.linear_mxfp4(y, x, ka.linear_mxfp4_weight(w), epi=EPI[epi])
    check(y, x, w, epi, f"off {off} ldy {ldy} ldx {ldx} {epi}", y0)
    rest = torch.ones_like(yb, dtype=torch.bool)
    rest[off:off + T * ldy].view(T, ldy)[:, :N] = False
    assert (yb[rest] == 2).all()


@pytest.mark.parametrize("T", [5, 100])
def test_nonfinite_rows(gpu, T):
    """A NaN or an infinity in a row of x makes that row NaN and no other; one in a weight row its column."""
    x, w = make(T, 80, 256, torch.float16)
    x[1, 200], x[3, 7] = float("nan"), float("inf")
    w[17, 0] = float("inf")
    y = ka.linear_mxfp4(out_of("f32", T, 80), x, ka.linear_mxfp4_weight(w))
    want = torch.zeros(T, 80, dtype=torch.bool, device=DEV)
    want[1] = want[3] = True
    want[:, 17] = True
    assert torch.equal(torch.isnan(y), want)
    keep = [r for r in range(T) if r not in (1, 3)]
    cols = [c for c in range(80) if c != 17]
    check(y[keep][:, cols], x[keep], w[cols], "f32", "finite rows")


def test_scales_far_apart(gpu):
    """Blocks from 2^-120 to 2^60 next to each other, and subnormal ones: what is small against the sum is lost, nothing else."""
    T, N, K = 70, 64, 512
    x, w = make(T, N, K, torch.bfloat16)
    x = (x.float() * torch.exp2(torch.linspace(-120, 60, T, device=DEV))[:, None]).bfloat16()
    check(ka.linear_mxfp4(out_of("f32", T, N), x, ka.linear_mxfp4_weight(w)), x, w, "f32", "row scales")
    x2 = make(T, N, K, torch.bfloat16)[0].float()
    x2[:, :256] *= 2.0 ** -40
    x2[:, 256:288] = 2.0 ** -130
    x2 = x2.bfloat16()
    check(ka.linear_mxfp4(out_of("f32", T, N), x2, ka.linear_mxfp4_weight(w)), x2, w, "f32", "block scales")


def test_weight_from_codes(gpu):
    """Plain codes and scales, as a checkpoint holds them, and the weight quantised here are the same layer."""
    x, w = make(90, 200, 320, torch.float16)
    codes, scales = ka.mxfp4_quantize(w)
    a = ka.linear_mxfp4(out_of("f32", 90, 200), x, ka.linear_mxfp4_weight(w))
    b = ka.linear_mxfp4(out_of("f32", 90, 200), x, ka.linear_mxfp4_weight(codes, scales))
    assert torch.equal(a, b)


def test_lora_by_linear16(gpu):
    """A LoRA pair beside the 4-bit weight: linear16 on the same y, beta = 1."""
    T, N, K, r = 130, 256, 512, 32
    x, w = make(T, N, K, torch.float16)
    a2, w2 = torch.randn(T, r, device=DEV).half(), (0.1 * torch.randn(N, r, device=DEV)).half()
    y = ka.linear_mxfp4(out_of("f32", T, N), x, ka.linear_mxfp4_weight(w))
    base = y.clone()
    ka.linear16(y, a2, w2, epi=ka.KILN_EPI_F32, beta=1.0)
    want = base.double() + a2.double() @ w2.double().t()
    assert ((y.double() - want).abs() <= 2.0 ** -22 * (base.double().abs() + a2.double().abs() @ w2.double().abs().t())).all()


def test_python_checks(gpu):
    x, w = make(100, 64, 64, torch.float16)
    W = ka.linear_mxfp4_weight(w)
    y = out_of("f32", 100, 64)
    for bad in (lambda: ka.linear_mxfp4(y.half(), x, W), lambda: ka.linear_mxfp4(y[:50], x, W), lambda: ka.linear_mxfp4(y, x[:, :32], W),
                lambda: ka.linear_mxfp4(y, x, W, epi=ka.KILN_EPI_RESID, gate=torch.ones(63, device=DEV)),
                lambda: ka.linear_mxfp4(y.t(), x, W)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(ka.KilnError) as e:
        ka.linear_mxfp4(y, x, W, workspace=torch.empty(16, dtype=torch.uint8, device=DEV))
    assert e.value.status == ka.KILN_ENOMEM


@pytest.mark.parametrize("T,N,bits,tile", [(20, 256, 27, 16), (100, 256, 25, 32), (1000, 1024, 22, 64), (1537, 2048, 21, 128), (4352, 8192, 19, 256)])
@pytest.mark.parametrize("dt", [torch.float16, torch.float32])
def test_rows_past_32_bits(gpu, T, N, bits, tile, dt):
    """Rows of x and y so far apart that elements pass 2^31 and bytes 2^32: the results of dense rows, bit for bit."""
    x, w = make(T, N, 128, dt)
    W = ka.linear_mxfp4_weight(w)
    assert ka.linear_mxfp4_tile(T, N, 128)[0] == tile
    epi = EPI["f16" if dt == torch.float16 else "f32"]
    far = torch.empty(T, (1 << bits) + 8, dtype=dt, device=DEV)
    far[:, :128] = x
    ka.linear_mxfp4(far[:, 128:128 + N], far[:, :128], W, epi=epi)
    assert torch.equal(far[:, 128:128 + N], ka.linear_mxfp4(torch.empty(T, N, dtype=dt, device=DEV), x, W, epi=epi))
