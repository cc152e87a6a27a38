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


def far_views(monkeypatch):
    """The wrappers up to the launch, on tensors without memory: views whose strides and sizes pass 32 bits cost nothing."""
    import torch
    monkeypatch.setattr(ka, "_gpu", lambda *t: 0)

    def launched(*a):
        raise AssertionError("reached the launch")
    monkeypatch.setattr(ka, "_launch", launched)
    monkeypatch.setattr(ka, "_scratch", lambda n, dev, stream: torch.empty(n, dtype=torch.uint8, device="meta"))

    def view(*shape, stride=None, dt=torch.float16):
        t = torch.empty(1, dtype=dt, device="meta")
        return torch.empty(shape, dtype=dt, device="meta") if stride is None else t.as_strided(shape, stride)
    return torch, view


BIG = 1 << 32


def test_python_strides_past_32_bits(monkeypatch):
    """A stride of 2^32 + W would arrive in the C ABI as W. (Of a single row it means nothing and passes.)"""
    torch, view = far_views(monkeypatch)
    f64 = view(64, dt=torch.float64)
    for big in (BIG + 256, 1 << 31):
        far, x = view(2, 256, stride=(big, 1)), view(2, 256)
        w = ka.Mxfp4Weight(view(1 << 16, dt=torch.uint8), 256, 256)
        codes, scales = view(2, 128, dt=torch.uint8), view(2, 8, dt=torch.uint8)
        x3, far3 = view(2, 2, 256), view(2, 2, 256, stride=(512, big, 1))
        calls = [lambda: ka.rope(far, x, 2, 128, f64), lambda: ka.rope(x, far, 2, 128, f64), lambda: ka.linear_mxfp4(far, x, w, epi=1),
                 lambda: ka.linear_mxfp4(x, far, w, epi=1), lambda: ka.mxfp4_quantize(far, codes, scales), lambda: ka.mxfp4_dequantize(far, codes, scales)]
        calls += [lambda i=i: ka.cross_attn(*[far3 if i == j else x3 for j in range(4)], 2) for i in range(4)]
        for i, call in enumerate(calls):
            with pytest.raises(ValueError, match="32 bits"):
                call()
    one, one3 = view(1, 256, stride=(BIG + 3, 1)), view(2, 1, 256, stride=(256, BIG + 8, 1))
    for call in (lambda: ka.rope(one, one, 2, 128, f64), lambda: ka.cross_attn(one3, one3, one3, one3, 2)):
        with pytest.raises(AssertionError, match="reached"):
            call()


def test_python_sizes_past_32_bits(monkeypatch):
    torch, view = far_views(monkeypatch)
    f64, u8, x = view(64, dt=torch.float64), torch.uint8, view(2, 256)
    tall, wide = view(BIG + 2, 256), view(2, BIG + 256)
    for call in (lambda: ka.rope(tall, tall, 2, 128, f64), lambda: ka.rope(x, x, 2, 128, f64, pos0=1 << 31), lambda: ka.rope(x, x, 2, 128, f64, pos0=-BIG),
                 lambda: ka.rope(x, x, 2, 128, view((BIG + 64) // 2, dt=torch.float64)),
                 lambda: ka.cross_attn(*[view(1, BIG + 2, 256)] * 2, *[view(1, 2, 256)] * 2, 2),
                 lambda: ka.cross_attn(*[view(1, 2, 256)] * 2, *[view(1, BIG + 2, 256)] * 2, 2), lambda: ka.cross_attn(*[view(BIG + 2, 1, 256)] * 4, 2),
                 lambda: ka.mxfp4_quantize(tall, view(BIG + 2, 128, dt=u8), view(BIG + 2, 8, dt=u8)),
                 lambda: ka.mxfp4_dequantize(wide, view(2, BIG // 2 + 128, dt=u8), view(2, BIG // 32 + 8, dt=u8)),
                 lambda: ka.linear_mxfp4_weight(view(BIG + 2, 128, dt=u8), view(BIG + 2, 8, dt=u8)), lambda: ka.rope_freqs(BIG + 64),
                 lambda: ka.linear_mxfp4(x, x, ka.Mxfp4Weight(view(9, dt=u8), 256, 256), epi=BIG + 1),
                 lambda: ka.cross_attn_workspace_bytes(1, 1, BIG + 8192, 16, 4, 128), lambda: ka.cross_attn_form(1, BIG + 1, 8, 1, 1, 64),
                 lambda: ka.linear_mxfp4_workspace_bytes(BIG + 1000, 2048, 2048), lambda: ka.linear_mxfp4_tile(1, 64, BIG + 64)):
        with pytest.raises(ValueError, match="32 bits"):
            call()
