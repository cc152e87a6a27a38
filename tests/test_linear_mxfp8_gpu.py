"""kiln_linear_mxfp8 against the product of the dequantised operands in 64 bits: every tile, odd sizes, part blocks of columns, strides and
alignment of y, epilogues, and NaN blocks."""

import math

import pytest
import torch

import kiln_amd as ka

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16 = torch.float32, torch.float16
EPIS = [ka.KILN_EPI_F32, ka.KILN_EPI_F16, ka.KILN_EPI_GELU16, ka.KILN_EPI_RESID]


def make(T, N, K, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + T * 7 + N + K)
    x = torch.randn(T, K, generator=g, device=DEV) * torch.exp(torch.randn(K, generator=g, device=DEV) / 2)
    w = (torch.rand(N, K, generator=g, device=DEV) * 2 - 1) / K ** 0.5
    codes, scales = ka.mxfp8_quantize(x)
    wc, wsc = ka.mxfp4_quantize(w)
    xv, wv = torch.empty(T, K, device=DEV), torch.empty(N, K, device=DEV)
    ka.mxfp8_dequantize(xv, codes, scales)
    ka.mxfp4_dequantize(wv, wc, wsc)
    return codes, scales, ka.linear_mxfp4_weight(wc, wsc), xv.double(), wv.double()


def check(y, before, xv, wv, epi, gate, beta, what):
    acc = xv @ wv.t()
    mag = xv.abs() @ wv.abs().t()
    # products exact, sums in fp32 in an unknown order: K terms at most. The smaller of X's two parts may lose, of eight products, seven times
    # 2^-13 of the largest, which is below 2^2 6 in units of a block's scale; the block's largest value is at least 224 of them
    block = xv.abs().view(xv.shape[0], -1, 32).amax(-1) @ wv.abs().view(wv.shape[0], -1, 32).amax(-1).t()
    tol = xv.shape[1] * 2.0 ** -24 * mag + 4 * 7 * 2.0 ** -13 * 4 / 224 * block
    if epi == ka.KILN_EPI_F32:
        ref = acc + beta * before.double()
        tol = tol + 2 * 2.0 ** -24 * (ref.abs() + (beta * before.double()).abs())
    elif epi == ka.KILN_EPI_RESID:
        gd = gate.double() if gate is not None else 1.0
        ref = before.double() + gd * acc
        tol = tol * (abs(gd) if gate is None else gd.abs()) + 2 * 2.0 ** -24 * (ref.abs() + (gd * acc).abs())
    else:
        ref = acc * torch.special.ndtr(acc) if epi == ka.KILN_EPI_GELU16 else acc
        # fp16 outputs: of eight neighbours' products, seven lose less than 2^-13 of the largest one's power of two.
        # GELU's slope is at most 1.13; its polynomial 2^-17 of min(|v|, v Phi)
        tol = tol + 7 * 2.0 ** -13 * mag
        tol = 1.13 * tol + (2.0 ** -17 * acc.abs() if epi == ka.KILN_EPI_GELU16 else 0)
        tol = tol + 2.0 ** -11 * (ref.abs() + tol) + 2.0 ** -25
    err = (y.double() - ref).abs()
    assert torch.isfinite(y).all(), what
    assert (err <= tol).all(), (what, (err / tol).max().item())
    print(f"[linear_mxfp8] {what}: worst error / tolerance {(err / tol).max():.3f}", flush=True)


SIZES = [(1, 1, 32), (1, 2048, 2048), (3, 33, 96), (16, 100, 1024), (17, 64, 160), (33, 47, 2080), (64, 2048, 8192), (65, 130, 64), (120, 2048, 2048),
         (200, 2048, 1056), (129, 255, 128), (500, 1024, 2048), (1537, 2048, 2048), (1000, 1500, 224), (2000, 4096, 1024), (2049, 4111, 992), (3, 70000, 64),
         (100000, 7, 64), (300, 300, 20000), (1500, 8190, 2048), (6700, 2040, 2080)]


def test_sizes_reach_every_tile(gpu):
    tiles = {ka.linear_mxfp8_tile(*s, epi) for s in SIZES for epi in EPIS}
    more = [(T, N, K) for T in (1, 17, 33, 64, 65, 100, 200, 400, 800, 1500, 3000, 7000) for N in (1024, 2048, 8192) for K in (1024, 2048, 8192)]
    assert tiles >= {ka.linear_mxfp8_tile(*s, epi) for s in more for epi in EPIS}


@pytest.mark.parametrize("T,N,K", SIZES)
def test_sizes(gpu, T, N, K):
    codes, scales, w, xv, wv = make(T, N, K)
    for epi in EPIS:
        y = torch.randn(T, N, device=DEV).to(F32 if epi in (0, 3) else F16)
        before, gate = y.clone(), torch.randn(N, device=DEV) if T % 2 else None
        ka.linear_mxfp8(y, codes, scales, w, epi=epi, gate=gate if epi == 3 else None, beta=0.5 if epi == 0 else 0.0)
        check(y, before, xv, wv, epi, gate, 0.5, f"{T}x{N}x{K} epilogue {epi} tile {ka.linear_mxfp8_tile(T, N, K, epi)}")


@pytest.mark.parametrize("T,N,K", [(5, 70, 96), (40, 200, 128), (130, 300, 256), (700, 1030, 160), (2100, 2052, 128), (1530, 8190, 2080)])
@pytest.mark.parametrize("extra,off", [(3, 1), (4, 0), (8, 4)])
def test_strides(gpu, T, N, K, extra, off):
    """Rows of y of any stride and alignment; what lies between them stays."""
    codes, scales, w, xv, wv = make(T, N, K, seed=1)
    for epi in (ka.KILN_EPI_F32, ka.KILN_EPI_F16):
        buf = torch.full((T, N + extra + off), 5.0, dtype=F32 if epi == 0 else F16, device=DEV)
        y = buf[:, off:off + N]
        ka.linear_mxfp8(y, codes, scales, w, epi=epi)
        check(y, y, xv, wv, epi, None, 0.0, f"stride {N + extra + off} from {off}")
        rest = torch.ones(N + extra + off, dtype=torch.bool, device=DEV)
        rest[off:off + N] = False
        assert (buf[:, rest] == 5).all()


@pytest.mark.parametrize("T", [1, 40, 300, 2100])
def test_unaligned_scales(gpu, T):
    """Scales at any address; columns past the last read as nothing, whatever lies behind a row (NaN codes and scales here)."""
    codes, scales, w, xv, wv = make(T, 260, 416, seed=2)
    for off in (0, 1, 2, 3):
        buf = torch.full((scales.numel() + 8,), 255, dtype=torch.uint8, device=DEV)
        s = buf[off:off + scales.numel()].view(scales.shape)
        s.copy_(scales)
        c = torch.full((codes.numel() + 512,), 0x7f, dtype=torch.uint8, device=DEV)[:codes.numel()].view(codes.shape)
        c.copy_(codes)
        y = torch.empty(T, 260, device=DEV)
        ka.linear_mxfp8(y, c, s, w)
        check(y, y, xv, wv, 0, None, 0.0, f"scales from byte {off}, T {T}")


@pytest.mark.parametrize("T,N,K", [(4, 64, 128), (40, 64, 256), (300, 600, 416), (2100, 2100, 512), (1530, 8190, 2080)])
def test_nan_blocks(gpu, T, N, K):
    """A NaN block of X makes its row NaN, one of W its column, and nothing else."""
    codes, scales, w, xv, wv = make(T, N, K, seed=3)
    clean = torch.empty(T, N, device=DEV)
    ka.linear_mxfp8(clean, codes, scales, w)
    scales[T // 2, K // 64] = 255
    codes[T // 3, 5] = 0x7f
    y = torch.empty(T, N, device=DEV)
    ka.linear_mxfp8(y, codes, scales, w)
    rows = torch.zeros(T, dtype=torch.bool, device=DEV)
    rows[[T // 2, T // 3]] = True
    assert torch.isnan(y[rows]).all() and torch.equal(y[~rows], clean[~rows])


def test_equals_mxfp4_rows_that_both_hold(gpu):
    """Rows whose values are 4-bit codes times powers of two are the same in MXFP8: both layers' results agree to the sums' order."""
    T, N, K = 200, 256, 512
    x = torch.randn(T, K, device=DEV)
    c4, s4 = ka.mxfp4_quantize(x)
    xv = torch.empty(T, K, device=DEV)
    ka.mxfp4_dequantize(xv, c4, s4)
    codes, scales = ka.mxfp8_quantize(xv)
    back = torch.empty_like(xv)
    ka.mxfp8_dequantize(back, codes, scales)
    assert torch.equal(back, xv)
    w = ka.linear_mxfp4_weight(torch.randn(N, K, device=DEV) / K ** 0.5)
    a, b = torch.empty(T, N, device=DEV), torch.empty(T, N, device=DEV)
    ka.linear_mxfp8(a, codes, scales, w)
    ka.linear_mxfp4(b, xv, w)
    assert ((a - b).abs() <= 2 * K * 2.0 ** -24 * (xv.abs().sum(1, keepdim=True) * 6)).all()


def test_capture_and_repeat(gpu):
    for T in (1, 100, 600):
        codes, scales, w, xv, wv = make(T, 512, 1024, seed=4)
        y = torch.empty(T, 512, device=DEV)
        ka.linear_mxfp8(y, codes, scales, w)
        eager = y.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ka.linear_mxfp8(y, codes, scales, w)
        for _ in range(3):
            y.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, eager)
