"""Rotary positions, cross-attention and MXFP4 layers on the CPU: the host frequencies against their formulas, buffer sizes, and
the calls that are refused before anything reaches the GPU."""
import ctypes
import math

import numpy as np
import pytest

import kiln_amd as ka

EINVAL, EUNSUP, ENOMEM = ka.KILN_EINVAL, ka.KILN_EUNSUPPORTED, ka.KILN_ENOMEM
F32, F16, BF16 = ka.KILN_F32, ka.KILN_F16, ka.KILN_BF16
P, Q, R, S = (1 << 20) * 16, (1 << 21) * 16, (1 << 22) * 16, (1 << 23) * 16  # addresses that no call below touches


@pytest.fixture(scope="module")
def L():
    return ka.lib()


@pytest.mark.parametrize("rot,theta,factor,trained", [(2, 1e4, 1.0, 2048), (32, 1e4, 4.0, 4096), (64, 5e5, 8.0, 8192), (128, 1e6, 40.0, 32768)])
def test_rope_freqs(L, rot, theta, factor, trained):
    # 64-bit arithmetic on both sides: a few roundings of pow, which the libraries give to within an ulp or two
    def close(got, want):
        np.testing.assert_allclose(got.numpy(), np.array(want), rtol=8 * 2.0 ** -52, atol=0)
    n = rot // 2
    f = [theta ** (-2 * i / rot) for i in range(n)]
    got, m = ka.rope_freqs(rot, theta)
    close(got, f)
    assert m == 1.0
    close(ka.rope_freqs(rot, theta, "linear", factor)[0], [x / factor for x in f])
    if rot > 2:
        close(ka.rope_freqs(rot, theta, "ntk", factor)[0], [(theta * factor ** (rot / (rot - 2))) ** (-2 * i / rot) for i in range(n)])
    # the ramp: pairs below lo keep their frequency, pairs above hi are stretched, linear between
    pair = lambda turns: rot * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
    lo, hi = max(math.floor(pair(32)), 0), min(math.ceil(pair(1)), rot - 1)
    w = [min(max((i - lo) / max(hi - lo, 0.001), 0), 1) for i in range(n)]
    got, m = ka.rope_freqs(rot, theta, "ramp", factor, trained)
    close(got, [x / factor * a + x * (1 - a) for x, a in zip(f, w)])
    assert m == np.float32(0.1 * math.log(factor) + 1)
    # bands: by the turns over the trained length, 4 and more keep, 1 and fewer are stretched
    got, m = ka.rope_freqs(rot, theta, "bands", factor, trained)
    keep = [min(max((trained * x / (2 * math.pi) - 1) / 3, 0), 1) for x in f]
    close(got, [x * a + x / factor * (1 - a) for x, a in zip(f, keep)])
    assert m == 1.0


def test_rope_freqs_refusals(L):
    for kw in (dict(rot=3), dict(rot=0), dict(rot=2, scaling="ntk", factor=2.0), dict(rot=8, theta=0.0), dict(rot=8, theta=math.inf),
               dict(rot=8, scaling="linear", factor=0.5), dict(rot=8, scaling="linear", factor=math.nan), dict(rot=8, scaling="ramp", factor=2.0),
               dict(rot=8, scaling="bands", factor=2.0, trained=100, slow=4.0, fast=4.0), dict(rot=8, theta=1.0, scaling="ramp", factor=2.0, trained=100)):
        with pytest.raises(ka.KilnError) as e:
            ka.rope_freqs(**kw)
        assert e.value.status == EINVAL
    with pytest.raises(ValueError):
        ka.rope_freqs(8, scaling="other")
    assert L.kiln_rope_freqs(None, None, 8, 1e4, 0, 1.0, 0.0, 1.0, 32.0) == EINVAL


def rope(L, y=P, ldy=256, x=Q, ldx=256, dt=F16, T=4, H=2, Dh=128, rot=128, pos=None, freqs=R):
    return L.kiln_rope(y, ldy, x, ldx, dt, T, H, Dh, rot, 0, pos, 0, freqs, 1.0, None)


def test_rope_refusals(L):
    for kw in (dict(dt=3), dict(dt=-1), dict(T=-1), dict(H=0), dict(Dh=0), dict(rot=0), dict(rot=3), dict(rot=130), dict(y=None), dict(x=None),
               dict(freqs=None), dict(ldx=255), dict(ldy=255)):
        assert rope(L, **kw) == EINVAL, kw
    for kw in (dict(Dh=2048, ldx=4096, ldy=4096), dict(H=65536, Dh=2, rot=2, ldx=1 << 18, ldy=1 << 18), dict(T=(1 << 30) + 1), dict(x=Q + 1), dict(dt=F32, y=P + 2),
               dict(freqs=R + 4), dict(pos=S + 2)):
        assert rope(L, **kw) == EUNSUP, kw
    # overlaps: shifted by a row, by some columns, with another stride; columns side by side are fine as far as the checks go
    assert rope(L, x=P + 256 * 2) == EINVAL
    assert rope(L, x=P + 16, ldx=512, ldy=512) == EINVAL
    assert rope(L, x=P, ldx=512) == EINVAL
    assert rope(L, T=0) == 0


def cross(L, out=P, ldo=256, bso=1024, q=Q, ldq=256, bsq=1024, k=R, ldk=256, bsk=2048, v=S, ldv=256, bsv=2048, dt=F16, B=2, Tq=4, Tk=8, Hq=2,
          Hkv=2, Dh=128, scale=0.1, klen=None, kmask=None, ws=None, wsb=0):
    return L.kiln_cross_attn(out, ldo, bso, q, ldq, bsq, k, ldk, bsk, v, ldv, bsv, dt, B, Tq, Tk, Hq, Hkv, Dh, scale, klen, kmask, 8, ws, wsb, None)


def test_cross_attn_refusals(L):
    for kw in (dict(dt=F32), dict(dt=7), dict(B=-1), dict(Tq=-1), dict(Tk=-1), dict(Hq=0), dict(Hkv=0), dict(Hq=3), dict(scale=0.0),
               dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(out=None), dict(q=None), dict(k=None), dict(v=None),
               dict(ldo=248), dict(ldq=0), dict(ldk=-256), dict(ldv=128), dict(bso=0), dict(bso=128), dict(bso=256), dict(bso=768), dict(bso=-768),
               dict(bso=256, ldo=504), dict(bso=128, Hq=1, Hkv=1, B=3, ldo=256)):
        assert cross(L, **kw) == EINVAL, kw
    for kw in (dict(Dh=96), dict(Dh=32), dict(out=P + 8), dict(q=Q + 2), dict(k=R + 8), dict(v=S + 4), dict(ldo=260), dict(ldk=257), dict(bsq=1028),
               dict(bsv=2049), dict(ldk=1 << 25), dict(klen=S + 2), dict(ws=S + 8, wsb=1 << 30), dict(Tk=(1 << 30) + 1), dict(Tq=1 << 30, Hq=4, ldo=512, ldq=512)):
        assert cross(L, **kw) == EUNSUP, kw
    assert cross(L, B=0) == 0 and cross(L, Tq=0) == 0


def test_cross_attn_workspace(L):
    w = ka.cross_attn_workspace_bytes
    assert w(0, 1, 8, 2, 2, 128) == 0 and w(1, 1, 8, 3, 2, 128) == 0 and w(1, 1, 8, 2, 2, 96) == 0
    # one token against few states needs none; against long ones, partial rows of Dh + 2 floats
    assert w(1, 1, 64, 16, 16, 128) == 0
    assert w(1, 1, 8192, 16, 4, 128) % ((128 + 2) * 4 * 16) == 0 and w(1, 1, 8192, 16, 4, 128) > 0
    assert w(2, 4096, 512, 16, 16, 128) == 0


def test_mxfp4_refusals(L):
    qz = lambda codes=P, scales=Q, x=R, dt=F16, ldx=64, rows=4, cols=64: L.kiln_mxfp4_quantize(codes, scales, x, dt, ldx, rows, cols, None)  # noqa: E731
    dq = lambda y=R, dt=F16, ldy=64, codes=P, scales=Q, rows=4, cols=64: L.kiln_mxfp4_dequantize(y, dt, ldy, codes, scales, rows, cols, None)  # noqa: E731
    for kw in (dict(codes=None), dict(scales=None), dict(dt=5), dict(rows=-1), dict(cols=0), dict(cols=-32)):
        assert qz(**kw) == EINVAL and dq(**kw) == EINVAL, kw
    assert qz(x=None) == EINVAL and dq(y=None) == EINVAL and qz(ldx=63) == EINVAL and dq(ldy=32) == EINVAL
    for kw in (dict(cols=40), dict(codes=P + 4), dict(rows=(1 << 30) + 1)):
        assert qz(**kw) == EUNSUP and dq(**kw) == EUNSUP, kw
    assert qz(x=R + 1) == EUNSUP and dq(y=R + 2, dt=F32) == EUNSUP
    assert qz(rows=0) == 0 and dq(rows=0) == 0


def test_linear_mxfp4_refusals(L):
    def lin(y=P, ldy=128, x=Q, dt=F16, ldx=64, T=100, wp=R, rows=128, cols=64, epi=0, gate=None, beta=0.0, ws=S, wsb=1 << 20):
        return L.kiln_linear_mxfp4(y, ldy, x, dt, ldx, T, wp, rows, cols, epi, gate, beta, ws, wsb, None)
    for kw in (dict(dt=3), dict(epi=4), dict(epi=-1), dict(T=-1), dict(rows=0), dict(rows=-4), dict(cols=0), dict(y=None), dict(x=None), dict(wp=None),
               dict(ldx=63), dict(ldy=127)):
        assert lin(**kw) == EINVAL, kw
    for kw in (dict(cols=48), dict(x=Q + 1), dict(y=P + 2), dict(epi=1, y=P + 1), dict(wp=R + 8), dict(gate=Q + 2), dict(ws=S + 4)):
        assert lin(**kw) == EUNSUP, kw
    assert lin(ws=None) == ENOMEM and lin(wsb=100) == ENOMEM
    assert lin(T=0) == 0
    pw = lambda wp=P, codes=Q, scales=R, rows=64, cols=64: L.kiln_linear_mxfp4_prepare_weight(wp, codes, scales, rows, cols, None)  # noqa: E731
    for kw in (dict(wp=None), dict(codes=None), dict(scales=None), dict(rows=0), dict(cols=0)):
        assert pw(**kw) == EINVAL, kw
    for kw in (dict(wp=P + 8), dict(codes=Q + 2), dict(cols=33)):
        assert pw(**kw) == EUNSUP, kw


def test_mxfp4_sizes(L):
    # 64-row groups x 128-column blocks: half a byte per code and a byte per 32
    per = 64 * 64 + 64 * 4
    assert L.kiln_linear_mxfp4_weight_bytes(1, 32) == per
    assert L.kiln_linear_mxfp4_weight_bytes(65, 160) == 4 * per
    assert L.kiln_linear_mxfp4_weight_bytes(2048, 2048) == 32 * 16 * per
    assert L.kiln_linear_mxfp4_weight_bytes(64, 33) == 0 and L.kiln_linear_mxfp4_weight_bytes(0, 32) == 0
    assert ka.linear_mxfp4_workspace_bytes(1, 2048, 2048) == 0
    assert ka.linear_mxfp4_workspace_bytes(1000, 2048, 2048) == 16 * 16 * per
    assert ka.linear_mxfp4_workspace_bytes(0, 2048, 2048) == 0


def test_gelu_polynomial():
    """The coefficients in gemm_mxfp4.hip: 2^P(z) is Phi(-z) within 2^-17 on [0, 6], in fp32 Horner steps, and decreases beyond: the
    polynomial itself is off by 2^-18.2, and the last steps round values of up to 30 by 2^-20 each (log2 units; 0.7 2^-20 of Phi)."""
    import os
    import re
    from scipy.special import log_ndtr
    src = open(os.path.join(os.path.dirname(ka.__file__), "csrc", "gemm_mxfp4.hip")).read()
    body = src[src.index("float mx_gelu(float v)"):]
    c = [np.float32(x) for x in re.findall(r"(-?\d[\d.]*(?:e-?\d+)?)f", body[:body.index("return")])]
    assert len(c) == 8
    z = np.linspace(0, 6, 400001).astype(np.float32)
    q = np.full_like(z, c[0])
    for k in c[1:]:
        q = (q.astype(np.float64) * z + k).astype(np.float32)  # one rounding, as an fma
    err = np.abs(np.expm1((q.astype(np.float64) * np.log(2)) - log_ndtr(-z.astype(np.float64))))
    assert err.max() <= 2.0 ** -17
    far = np.geomspace(6, 1e30, 10000)
    v = np.polynomial.polynomial.polyval(far, [float(x) for x in c[::-1]])
    assert (np.diff(v) < 0).all() and v[0] < -29


def test_python_checks():
    import torch
    x = torch.zeros(4, 256, dtype=torch.float16)
    with pytest.raises(ValueError, match="GPU"):
        ka.rope(x, x, 2, 128, torch.zeros(64, dtype=torch.float64))
    with pytest.raises(ValueError, match="GPU"):
        ka.cross_attn(x[None], x[None], x[None], x[None], 2)
    with pytest.raises(ValueError, match="GPU"):
        ka.mxfp4_quantize(x)
    assert ctypes.sizeof(ctypes.c_double) == 8


def test_forms_of_refused_sizes(L):
    assert L.kiln_cross_attn_form(0, 1, 1, 1, 1, 64) == 0 and L.kiln_cross_attn_form(1, 1, 1, 3, 2, 64) == 0
    assert L.kiln_cross_attn_form(1, 1, 1, 1, 1, 96) == 0 and L.kiln_cross_attn_form(1, 1, (1 << 30) + 1, 1, 1, 64) == 0
    assert L.kiln_linear_mxfp4_tile(0, 64, 64) == 0 and L.kiln_linear_mxfp4_tile(64, 64, 40) == 0
    assert ka.linear_mxfp4_tile(1, 64, 64) == (16, 16)
