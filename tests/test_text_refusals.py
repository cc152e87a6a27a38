"""Calls of a text encoder's layer that are refused before anything reaches the GPU, and what its sizes say without one."""
import math

import pytest

import kiln_amd as ka

EINVAL, EUNSUP, OK = ka.KILN_EINVAL, ka.KILN_EUNSUPPORTED, ka.KILN_OK
F32, F16, BF16 = ka.KILN_F32, ka.KILN_F16, ka.KILN_BF16
A = [(1 << 30) + (i << 28) for i in range(10)]  # addresses 2^28 apart that no call below touches


@pytest.fixture(scope="module")
def L():
    return ka.lib()


def attn(L, out=A[0], ldo=512, q=A[1], ldq=512, k=A[2], ldk=256, v=A[3], ldv=256, dt=F16, Tq=8, Tk=8, Hq=4, Hkv=2, Dh=128, scale=0.1, B=2, qs=A[4],
         ks=None, kl=None, pk=None, ldpk=0, pv=None, ldpv=0, P=0, ws=None, wsb=0):
    return L.kiln_prompt_attn(out, ldo, q, ldq, k, ldk, v, ldv, dt, Tq, Tk, Hq, Hkv, Dh, scale, B, qs, ks, kl, pk, ldpk, pv, ldpv, P, ws, wsb, None)


@pytest.mark.parametrize("want,kw", [
    (EINVAL, dict(dt=F32)), (EINVAL, dict(dt=7)), (EINVAL, dict(B=-1)), (EINVAL, dict(Tq=-1)), (EINVAL, dict(Tk=-1)), (EINVAL, dict(P=-1)), (EINVAL, dict(Hq=0)),
    (EINVAL, dict(Hkv=0)), (EINVAL, dict(Hkv=3)), (EUNSUP, dict(Dh=96)), (EUNSUP, dict(Dh=256)), (EINVAL, dict(scale=0.0)), (EINVAL, dict(scale=-1.0)),
    (EINVAL, dict(scale=math.nan)), (EINVAL, dict(scale=math.inf)), (EINVAL, dict(scale=3e38)), (EINVAL, dict(ks=A[5])), (EINVAL, dict(kl=A[5])),
    (EINVAL, dict(qs=None)), (EINVAL, dict(Tk=9)), (EINVAL, dict(Tk=7)), (EINVAL, dict(out=None)), (EINVAL, dict(q=None)), (EINVAL, dict(k=None)),
    (EINVAL, dict(v=None)), (EINVAL, dict(P=4)), (EINVAL, dict(P=4, pk=A[6])), (EINVAL, dict(ldo=511)), (EINVAL, dict(ldk=255)), (EINVAL, dict(ldv=128)),
    (EUNSUP, dict(ldq=516)), (EUNSUP, dict(ldk=260)), (EUNSUP, dict(q=A[1] + 8)), (EUNSUP, dict(out=A[0] + 2)), (EUNSUP, dict(k=A[2] + 4)), (EUNSUP, dict(ldq=(1 << 24) + 8)),
    (EINVAL, dict(P=4, pk=A[6], pv=A[7], ldpk=255, ldpv=256)), (EUNSUP, dict(P=4, pk=A[6] + 8, pv=A[7], ldpk=256, ldpv=256)),
    (EUNSUP, dict(qs=A[4] + 2)), (EUNSUP, dict(ks=A[5] + 1, kl=A[6])), (EUNSUP, dict(ws=A[8] + 8, wsb=1 << 20)),
    (EINVAL, dict(out=A[1])), (EINVAL, dict(out=A[1] + 1024)), (EINVAL, dict(out=A[2] + 16)), (EINVAL, dict(out=A[3])),
    (EINVAL, dict(P=4, pk=A[0] + 64, pv=A[7], ldpk=256, ldpv=256)), (EINVAL, dict(P=4, pk=A[6], pv=A[0], ldpk=256, ldpv=256)),
    (EUNSUP, dict(B=1 << 24)), (EUNSUP, dict(B=(1 << 14) + 1)), (EUNSUP, dict(Tq=1 << 30, Tk=1 << 30, q=1 << 50, k=1 << 52, v=1 << 53, out=1 << 54)),
])
def test_prompt_attn(L, want, kw):
    assert attn(L, **kw) == want, ka.lib().kiln_attn_last_error()


def test_prompt_attn_nothing_to_do(L):
    assert attn(L, B=0, qs=None, Tk=0) == OK
    assert attn(L, Tq=0, Tk=0, out=None, q=None) == OK


def test_prompt_attn_workspace_sizes():
    w = ka.prompt_attn_workspace_bytes
    assert w(0, 8, 8, 0, 4, 2, 128) == 0 and w(1, 0, 8, 0, 4, 2, 128) == 0 and w(1, 8, 8, 0, 4, 3, 128) == 0 and w(1, 8, 8, 0, 4, 2, 96) == 0
    assert w(1, 8192, 8192, 0, 16, 8, 128) == 0  # many rows: no need to split the keys
    with pytest.raises(ValueError):
        w(1 << 40, 8, 8, 0, 4, 2, 128)


def norm(L, y=A[0], ydt=F16, ldy=64, h=A[1], ldh=64, x=A[2], xdt=F16, ldx=64, res=A[3], rdt=F32, ldr=64, w=A[4], rows=4, dim=64, eps=1e-6):
    return L.kiln_add_rmsnorm(y, ydt, ldy, h, ldh, x, xdt, ldx, res, rdt, ldr, w, rows, dim, eps, None)


@pytest.mark.parametrize("want,kw", [
    (EINVAL, dict(ydt=3)), (EINVAL, dict(xdt=-1)), (EINVAL, dict(rdt=9)), (EINVAL, dict(rows=-1)), (EINVAL, dict(dim=0)), (EUNSUP, dict(dim=32769, ldy=1 << 20, ldx=1 << 20, ldh=1 << 20, ldr=1 << 20)),
    (EUNSUP, dict(rows=(1 << 30) + 1)), (EINVAL, dict(eps=0.0)), (EINVAL, dict(eps=-1.0)), (EINVAL, dict(eps=math.nan)), (EINVAL, dict(eps=math.inf)),
    (EINVAL, dict(h=None)), (EINVAL, dict(res=None)), (EINVAL, dict(y=None)), (EINVAL, dict(x=None)), (EINVAL, dict(ldx=63)), (EINVAL, dict(ldy=63)),
    (EINVAL, dict(ldr=63)), (EINVAL, dict(ldh=63)), (EUNSUP, dict(x=A[2] + 1)), (EUNSUP, dict(y=A[0] + 1)), (EUNSUP, dict(res=A[3] + 2)), (EUNSUP, dict(h=A[1] + 2)),
    (EUNSUP, dict(w=A[4] + 1)), (EINVAL, dict(y=A[2], ldy=72)), (EINVAL, dict(y=A[2], ydt=BF16)), (EINVAL, dict(y=A[2] + 2)), (EINVAL, dict(h=A[3], ldh=72)),
    (EINVAL, dict(h=A[3] + 4)), (EINVAL, dict(h=A[2], rdt=F16)), (EINVAL, dict(y=A[1])), (EINVAL, dict(y=A[3])),
])
def test_add_rmsnorm(L, want, kw):
    assert norm(L, **kw) == want, ka.lib().kiln_attn_last_error()


def test_add_rmsnorm_mxfp8(L):
    def call(codes=A[0], scales=A[1], rows=4, dim=64, x=A[2], ldx=64, res=None, h=None):
        return L.kiln_add_rmsnorm_mxfp8(codes, scales, h, 64, x, F16, ldx, res, F32, 64, None, rows, dim, 1e-6, None)
    assert call(dim=48, ldx=48) == EUNSUP
    assert call(codes=None) == EINVAL and call(scales=None) == EINVAL and call(x=None) == EINVAL
    assert call(codes=A[0] + 8) == EUNSUP
    assert call(codes=A[2]) == EINVAL and call(codes=A[2] + 128) == EINVAL
    assert call(res=A[3]) == EINVAL and call(rows=-1) == EINVAL and call(dim=0) == EINVAL
    assert call(rows=0, codes=None, scales=None, x=None) == OK


def test_mxfp8_rows(L):
    def quant(codes=A[0], scales=A[1], x=A[2], dt=F16, ldx=64, rows=4, cols=64):
        return L.kiln_mxfp8_quantize(codes, scales, x, dt, ldx, rows, cols, None)

    def back(y=A[2], dt=F16, ldy=64, codes=A[0], scales=A[1], rows=4, cols=64):
        return L.kiln_mxfp8_dequantize(y, dt, ldy, codes, scales, rows, cols, None)
    for f in (quant, back):
        assert f(dt=5) == EINVAL and f(cols=40) == EUNSUP and f(cols=0) == EINVAL and f(rows=-1) == EINVAL and f(rows=(1 << 30) + 1) == EUNSUP
        assert f(codes=None) == EINVAL and f(scales=None) == EINVAL and f(codes=A[0] + 4) == EUNSUP and f(rows=0, codes=None, scales=None) == OK
    assert quant(x=None) == EINVAL and quant(ldx=63) == EINVAL and quant(x=A[2] + 1) == EUNSUP
    assert back(y=None) == EINVAL and back(ldy=63) == EINVAL and back(y=A[2] + 1) == EUNSUP


def test_linear_mxfp8(L):
    def call(y=A[0], ldy=128, codes=A[1], scales=A[2], T=40, wp=A[3], rows=128, cols=64, epi=0, gate=None):
        return L.kiln_linear_mxfp8(y, ldy, codes, scales, T, wp, rows, cols, epi, gate, 0.0, None)
    assert call(epi=4) == EINVAL and call(epi=-1) == EINVAL and call(cols=48) == EUNSUP and call(cols=0) == EINVAL and call(rows=0) == EINVAL and call(T=-1) == EINVAL
    assert call(cols=(1 << 22) + 32) == EUNSUP and call(T=1 << 30, rows=1 << 20) == EUNSUP
    assert call(y=None) == EINVAL and call(codes=None) == EINVAL and call(scales=None) == EINVAL and call(wp=None) == EINVAL and call(ldy=127) == EINVAL
    assert call(wp=A[3] + 8) == EUNSUP and call(codes=A[1] + 8) == EUNSUP and call(y=A[0] + 2) == EUNSUP and call(gate=A[4] + 2, epi=3) == EUNSUP
    assert call(y=A[1]) == EINVAL and call(y=A[1] + 16) == EINVAL and call(y=A[2]) == EINVAL and call(y=A[1] - 128, epi=1) == EINVAL
    assert call(T=0, y=None, codes=None, scales=None, wp=None) == OK


def test_linear_mxfp8_tiles():
    for epi in range(4):
        assert ka.linear_mxfp8_tile(1, 2048, 2048, epi) == (16, 16)
        assert ka.linear_mxfp8_tile(0, 2048, 2048, epi) == (0, 0) and ka.linear_mxfp8_tile(5, 2048, 2000, epi) == (0, 0)
    assert ka.linear_mxfp8_tile(5, 2048, 2048, 9) == (0, 0)
    assert ka.linear_mxfp8_tile(6912, 8192, 2048, ka.KILN_EPI_GELU16) == (256, 128)
    with pytest.raises(ValueError):
        ka.linear_mxfp8_tile(1 << 33, 2048, 2048)
