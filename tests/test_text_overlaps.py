"""The norm's buffers that share bytes are refused before anything reaches the GPU: its scales and weight as well as its rows; windows that lie in
each other's gaps are not."""

import pytest
import torch

import kiln_amd as ka

EINVAL = ka.KILN_EINVAL
F32, F16 = ka.KILN_F32, ka.KILN_F16
A = [(1 << 30) + (i << 28) for i in range(10)]  # addresses 2^28 apart
OUT, SCALES, H, X, RES, W = A[:6]
# 40 rows of 256: codes 10240 bytes, scales 320, fp16 rows 20480, fp32 rows 40960, w 512


def fused(L, codes=OUT, scales=SCALES, h=H, ldh=256, x=X, ldx=256, res=RES, ldr=256, w=W, rows=40, dim=256):
    return L.kiln_add_rmsnorm_mxfp8(codes, scales, h, ldh, x, F16, ldx, res, F32, ldr, w, rows, dim, 1e-6, None)


def plain(L, y=OUT, ldy=256, h=H, ldh=256, x=X, ldx=256, res=RES, ldr=256, w=W, rows=40, dim=256):
    return L.kiln_add_rmsnorm(y, F16, ldy, h, ldh, x, F16, ldx, res, F32, ldr, w, rows, dim, 1e-6, None)


@pytest.mark.parametrize("kw", [
    dict(scales=X), dict(scales=X + 20479), dict(scales=X - 319), dict(scales=RES + 5), dict(scales=RES + 40959), dict(scales=H + 100), dict(scales=OUT), dict(scales=OUT + 10239),
    dict(scales=OUT - 319), dict(scales=W), dict(scales=W + 511), dict(scales=W - 319), dict(w=OUT + 10238), dict(w=OUT - 510), dict(w=H), dict(w=H + 40958),
    dict(h=RES, w=RES + 64), dict(scales=X + 512, ldx=300), dict(scales=X + 200, ldx=1024)])
def test_mxfp8(kw):
    assert fused(ka.lib(), **kw) == EINVAL, kw
    assert b"overlap" in ka.lib().kiln_attn_last_error()


@pytest.mark.parametrize("kw", [dict(w=OUT), dict(w=OUT + 20478), dict(w=OUT - 510), dict(w=H + 2), dict(h=RES, w=RES + 40958), dict(y=X, w=X + 2), dict(w=OUT + 100, ldy=400)])
def test_rows(kw):
    assert plain(ka.lib(), **kw) == EINVAL, kw
    assert b"overlap" in ka.lib().kiln_attn_last_error()


@pytest.mark.gpu
def test_windows_in_gaps(gpu):
    """Scales, weight and one row in the gaps of other buffers' rows, or right beside them, run."""
    rows, dim = 40, 256
    x = torch.randn(rows, dim, device="cuda").half()
    w = torch.randn(dim, device="cuda").to(torch.bfloat16)
    want_c, want_s = torch.empty(rows, dim, dtype=torch.uint8, device="cuda"), torch.empty(rows, dim // 32, dtype=torch.uint8, device="cuda")
    ka.add_rmsnorm(want_c, x, w=w, scales=want_s)
    buf = torch.zeros(rows, 2 * dim, dtype=torch.float16, device="cuda")  # x in the left half; w, then the scales, in the gaps at the right
    xx = buf[:, :dim]
    xx.copy_(x)
    ww = buf[3, dim:].view(torch.bfloat16)
    ww.copy_(w)
    ss = buf[5, dim:].view(torch.uint8)[192:192 + rows * dim // 32].view(rows, dim // 32)
    codes = torch.empty_like(want_c)
    ka.add_rmsnorm(codes, xx, w=ww, scales=ss)
    assert torch.equal(codes, want_c) and torch.equal(ss, want_s) and torch.equal(xx, x)
    # an output with the weight in its gap, against rows of their own
    y, want = torch.zeros(rows, 3 * dim, dtype=torch.float16, device="cuda"), torch.empty(rows, dim, dtype=torch.float16, device="cuda")
    ka.add_rmsnorm(want, x, w=w)
    gap = y[rows - 2, dim:2 * dim].view(torch.bfloat16)
    gap.copy_(w)
    ka.add_rmsnorm(y[:, :dim], x, w=gap)
    assert torch.equal(y[:, :dim], want) and torch.equal(gap, w)


@pytest.mark.gpu
def test_one_byte_too_far(gpu):
    """The same places a byte or a row further are refused."""
    rows, dim = 40, 256
    buf = torch.zeros(rows + 1, 2 * dim, dtype=torch.float16, device="cuda")
    x, flat = buf[:rows, :dim], buf.view(torch.uint8).view(-1)
    codes = torch.empty(rows, dim, dtype=torch.uint8, device="cuda")
    n = rows * dim // 32
    for first in (1024 * 5 + 1024 - n + 1, 1024 * 5 + 511, 1024 * 5 + 512 - n, 1024 * (rows - 1) + 500):
        with pytest.raises(ka.KilnError, match="overlap"):
            ka.add_rmsnorm(codes, x, scales=flat[first:first + n].view(rows, dim // 32))
    ka.add_rmsnorm(codes, x, scales=flat[1024 * 5 + 1024 - n:1024 * 6].view(rows, dim // 32))
    ka.add_rmsnorm(codes, x, scales=flat[1024 * (rows - 1) + 512:1024 * (rows - 1) + 512 + n].view(rows, dim // 32))
