"""Calls of the attention section over an encoder's states that are refused before anything reaches the GPU."""
import pytest

import kiln_amd as ka

EINVAL, EUNSUP, ENOMEM = ka.KILN_EINVAL, ka.KILN_EUNSUPPORTED, ka.KILN_ENOMEM
F32, F16, BF16 = ka.KILN_F32, ka.KILN_F16, ka.KILN_BF16
P, Q, R, S = (1 << 20) * 16, (1 << 21) * 16, (1 << 22) * 16, (1 << 23) * 16  # addresses that no call below touches


@pytest.fixture(scope="module")
def L():
    return ka.lib()


@pytest.mark.parametrize("scale", [2.4e38, 3.4e38])
def test_cross_attn_scale(L, scale):
    """A scale that is finite but not in the units of log2 that the kernel works in: 0 times it would be a NaN."""
    assert L.kiln_cross_attn(P, 256, 1024, Q, 256, 1024, R, 256, 2048, S, 256, 2048, F16, 2, 4, 8, 2, 2, 128, scale, None, None, 8, None, 0,
                             None) == EINVAL


def linear(L, y=P, ldy=128, x=Q, dt=F16, ldx=128, T=200, wp=R, rows=128, cols=128, epi=ka.KILN_EPI_F16, ws=None, wsb=0):
    return L.kiln_linear_mxfp4(y, ldy, x, dt, ldx, T, wp, rows, cols, epi, None, 0.0, ws, wsb, None)


@pytest.mark.parametrize("T", [1, 4, 16, 40, 200, 5000])
def test_linear_mxfp4_overlap(L, T):
    """y over x: few rows are quantised by workgroups that others' outputs would overtake, many before the first output; refused alike.
    One and the same window, of either size of element, and windows that share some of their bytes."""
    ws = dict(ws=S, wsb=1 << 30)
    assert linear(L, T=T, y=Q, **ws) == EINVAL
    assert linear(L, T=T, y=Q, dt=F32, epi=ka.KILN_EPI_RESID, **ws) == EINVAL
    assert linear(L, T=T, y=Q, epi=ka.KILN_EPI_F32, **ws) == EINVAL              # fp32 over fp16
    assert linear(L, T=T, y=Q + 254, **ws) == EINVAL                             # from x's last column
    assert linear(L, T=T, y=Q - 254, **ws) == EINVAL                             # up to x's first
    assert linear(L, T=T, y=Q + (T - 1) * 256 + 128, **ws) == EINVAL             # over x's last row
    if T > 1:
        assert linear(L, T=T, y=Q + 256, ldx=256, ldy=320, **ws) == EINVAL       # rows of other strides run into x's
        assert linear(L, T=T, y=Q + 254, ldx=256, ldy=256, **ws) == EINVAL
        assert linear(L, T=T, y=Q + 258, ldx=256, ldy=256, **ws) == EINVAL       # y's end is x's next row
        assert linear(L, T=T, y=Q + 256, ldx=256, ldy=256, epi=ka.KILN_EPI_F32, **ws) == EINVAL


def test_linear_mxfp4_side_by_side(L):
    """Windows that share no byte pass on to the check of the workspace: columns side by side in rows of one stride in bytes, rows
    one block behind the other."""
    for kw in (dict(y=Q + 256, ldx=256, ldy=256), dict(y=Q - 256, ldx=256, ldy=256), dict(y=Q + 256, ldx=384, ldy=192, epi=ka.KILN_EPI_F32),
               dict(y=Q + 512, dt=F32, ldx=192, ldy=384), dict(y=Q + 200 * 256), dict(y=Q - 200 * 256), dict(y=Q + 199 * 256 + 256, ldy=999)):
        assert linear(L, **kw) == ENOMEM, kw
