"""kiln_mxfp4_quantize and kiln_mxfp4_dequantize, equal to the definition's codes, scales and values to the bit."""
import numpy as np
import pytest
import torch

import kiln_amd as ka
from tests import mxfp4_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def check(x, what):
    """x as given (strides and all) on the GPU against the definition."""
    codes, scales = ka.mxfp4_quantize(x)
    want_c, want_s = ref.quantize(x)
    np.testing.assert_array_equal(scales.cpu().numpy(), want_s, err_msg=what)
    got = codes.cpu().numpy()
    np.testing.assert_array_equal(got, want_c, err_msg=what)
    v = torch.from_numpy(ref.values(codes, scales))
    for dt in DTYPES:
        y = ka.mxfp4_dequantize(torch.empty(x.shape, dtype=dt, device=DEV), codes, scales)
        assert torch.equal(torch.nan_to_num(y.cpu(), nan=7.0), torch.nan_to_num(v.to(dt), nan=7.0)), (what, dt)


@pytest.mark.parametrize("rows,cols", [(1, 32), (1, 8192), (3, 96), (77, 1024), (129, 160), (1000, 64), (4097, 32)])
@pytest.mark.parametrize("dt", DTYPES)
def test_values(gpu, rows, cols, dt):
    g = torch.Generator(device=DEV).manual_seed(rows)
    x = torch.randn(rows, cols, device=DEV, generator=g) * torch.exp(2 * torch.randn(cols, device=DEV, generator=g))
    check(x.to(dt), f"{rows} x {cols} {dt}")


@pytest.mark.parametrize("dt", DTYPES)
def test_borders(gpu, dt):
    """Every border between neighbouring codes and the values next to it, both signs, beside largest values that set the scale
    at both ends of its octave; powers of two over the type's whole range, subnormals among them."""
    mids = torch.tensor([0.0, 0.25, 0.5, 0.75, 1.0, 1.25, 1.5, 1.75, 2.0, 2.5, 3.0, 3.5, 4.0, 5.0, 6.0])
    rows = []
    lo, hi = {torch.float32: (-149, 127), torch.float16: (-24, 15), torch.bfloat16: (-133, 127)}[dt]
    for e in range(lo, hi + 1, 1 if dt == torch.float16 else 3):
        for top in (4.0, 5.0, 7.0, 7.96875):
            v = mids.double().clone()
            s = torch.cat([v, -v, torch.tensor([top, -top]).double()])
            rows.append(torch.ldexp(s, torch.tensor(e - 2)))
    x = torch.stack(rows).to(dt)
    x = x[torch.isfinite(x).all(-1)].to(DEV)
    check(x, f"borders {dt}")
    # the neighbours of the borders in the type itself
    i = torch.int32 if dt == torch.float32 else torch.int16
    for step in (-1, 1):
        y = x.clone().view(i)
        y[:, :30] += step
        y = y.view(dt)
        check(torch.where(torch.isfinite(y), y, torch.zeros_like(y)), f"beside the borders {dt} {step}")


@pytest.mark.parametrize("dt", DTYPES)
def test_nonfinite_and_zero_blocks(gpu, dt):
    x = torch.randn(6, 128, device=DEV).to(dt)
    x[0] = 0
    x[1] = -0.0
    x[2, 5], x[3, 40], x[4, 127] = float("nan"), float("inf"), float("-inf")
    check(x, f"{dt}")
    _, s = ka.mxfp4_quantize(x)
    s = s.cpu()
    assert (s[0] == 0).all() and s[2, 0] == 255 and s[3, 1] == 255 and s[4, 3] == 255 and int((s == 255).sum()) == 3


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("off,ld", [(0, 104), (1, 97), (4, 100), (2, 99)])
def test_strides(gpu, dt, off, ld):
    buf = torch.randn(50 * ld + off, device=DEV).to(dt)
    x = buf[off:off + 50 * ld].view(50, ld)[:, :96]
    check(x, f"off {off} ld {ld} {dt}")
    codes, scales = ka.mxfp4_quantize(x)
    y = torch.full((50 * ld + off,), 3.0, dtype=dt, device=DEV)
    rows = y[off:off + 50 * ld].view(50, ld)
    ka.mxfp4_dequantize(rows[:, :96], codes, scales)
    assert torch.equal(rows[:, :96].cpu(), torch.from_numpy(ref.values(codes, scales)).to(dt))
    assert (rows[:, 96:] == 3).all() and (y[:off] == 3).all()


def test_idempotent(gpu):
    """Values of the format are kept as they are, unless the block's largest moved to another octave."""
    x = torch.randn(64, 256, device=DEV)
    c, s = ka.mxfp4_quantize(x)
    y = ka.mxfp4_dequantize(torch.empty_like(x), c, s)
    z = ka.mxfp4_dequantize(torch.empty_like(x), *ka.mxfp4_quantize(y))
    assert torch.equal(y, z)


def test_python_checks(gpu):
    x = torch.randn(4, 64, device=DEV)
    c, s = ka.mxfp4_quantize(x)
    with pytest.raises(ValueError):
        ka.mxfp4_quantize(x, c, None)
    with pytest.raises(ValueError):
        ka.mxfp4_quantize(x, c[:, :16], s)
    with pytest.raises(ValueError):
        ka.mxfp4_quantize(x.t(), c, s)
    with pytest.raises(TypeError):
        ka.mxfp4_quantize(x.double(), c, s)
    with pytest.raises(ValueError):
        ka.mxfp4_dequantize(x, c, s.cpu()[:2])
    with pytest.raises(ka.KilnError):
        ka.mxfp4_quantize(torch.randn(4, 40, device=DEV), torch.empty(4, 20, dtype=torch.uint8, device=DEV),
                          torch.empty(4, 1, dtype=torch.uint8, device=DEV))


def test_rows_past_32_bits(gpu):
    """Rows so far apart that elements pass 2^31 and bytes 2^32."""
    x = torch.randn(40, 96, device=DEV).half()
    far = torch.empty(40, (1 << 26) + 8, dtype=torch.float16, device=DEV)
    far[:, :96] = x
    c, s = ka.mxfp4_quantize(far[:, :96])
    c0, s0 = ka.mxfp4_quantize(x)
    assert torch.equal(c, c0) and torch.equal(s, s0)
    ka.mxfp4_dequantize(far[:, 96:192], c, s)
    assert torch.equal(far[:, 96:192], ka.mxfp4_dequantize(torch.empty_like(x), c, s))


def test_many_blocks(gpu):
    """2^32 + 4096 values in one call, each pass of a thread through the loop: the last rows as by themselves."""
    x = torch.empty((1 << 20) + 1, 4096, dtype=torch.float16, device=DEV)
    x[:-5] = 1
    x[-5:] = torch.randn(5, 4096, device=DEV)
    c, s = ka.mxfp4_quantize(x)
    c5, s5 = ka.mxfp4_quantize(x[-5:])
    assert torch.equal(c[-5:], c5) and torch.equal(s[-5:], s5) and (s[:-5] == 125).all() and (c[:-5] == 0x66).all()
    assert torch.equal(ka.mxfp4_dequantize(x.clone(), c, s)[-5:], ka.mxfp4_dequantize(torch.empty_like(x[-5:]), c5, s5))
