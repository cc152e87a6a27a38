"""kiln_cross_attn at the ends of its types' ranges: values up to the largest finite number, in every form."""
import pytest
import torch

import kiln_amd as ka
from tests.test_cross_attn_gpu import SHAPES, check, make

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def both(q, k, v, Hq, Hkv, **kw):
    """The call with its workspace and with one too small to split the keys."""
    for ws in (None, torch.empty(16, dtype=torch.uint8, device=DEV)):
        yield ka.cross_attn(torch.full_like(q, float("nan")), q, k, v, Hq, Hkv, workspace=ws, **kw)


@pytest.mark.parametrize("B,Tq,Tk,Hq,Hkv,Dh", SHAPES)
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_largest_values(gpu, B, Tq, Tk, Hq, Hkv, Dh, dt):
    """Every key holds the type's largest number, or its negative: so does the output, whatever the weights, which are a convex
    combination. Exactly so: the sums' and the division's relative error, (Tk / 4 + 64) 2^-24 + 2^-21 < 2^-12, is less than half
    the step below the largest number (2^-9 of it in bf16, 2^-12 in fp16), and beyond it nothing rounds up to infinity
    (from half a step above on). Scores that rise by up to 7 in log2 keep the first maximum, so that weights pass 1."""
    assert (Tk / 4 + 64) * 2.0 ** -24 + 2.0 ** -21 < 2.0 ** -12
    q, k, _ = make(B, Tq, Tk, Hq, Hkv, Dh, dt)
    top = torch.finfo(dt).max
    v = torch.full_like(k, top)
    v[..., ::3] = -top
    want = v[:, :1, :Dh].repeat(1, Tq, Hq)
    want.view(B, Tq, Hq, Dh)[:] = v[:, :1].view(B, 1, Hkv, 1, Dh).expand(B, 1, Hkv, Hq // Hkv, Dh).reshape(B, 1, Hq, Dh)
    for out in both(q, k, v, Hq, Hkv):
        assert torch.equal(out, want)
    q, k = torch.zeros_like(q), torch.zeros_like(k)
    q.view(B, Tq, Hq, Dh)[..., 0] = 1
    k.view(B, Tk, Hkv, Dh)[..., 0] = (torch.arange(Tk, device=DEV) * (4.85 / Tk))[None, :, None].to(dt)  # 4.85 / ln 2 < 7
    klen = torch.full((B,), Tk, dtype=torch.int32, device=DEV)
    klen[-1] = max(1, Tk // 2)
    for out in both(q, k, v, Hq, Hkv, scale=1.0, klen=klen):
        assert torch.equal(out, want)


@pytest.mark.parametrize("B,Tq,Tk,Hq,Hkv,Dh", SHAPES)
@pytest.mark.parametrize("e", [126, -80])
def test_bf16_far_from_one(gpu, B, Tq, Tk, Hq, Hkv, Dh, e):
    """bf16 values about 2^126 and 2^-80, of either sign, within the tolerance of those about 1."""
    q, k, v = make(B, Tq, Tk, Hq, Hkv, Dh, torch.bfloat16)
    v = (v.double().clamp(-3.9, 3.9) * 2.0 ** e).bfloat16()
    for out in both(q, k, v, Hq, Hkv):
        check(out, q, k, v, Hq, Hkv, what=f"{B} {Tq} {Tk} {Hq} {Hkv} {Dh} 2^{e}")


def test_one_bf16_key(gpu):
    q, k, _ = make(1, 90, 1, 4, 4, 128, torch.bfloat16)
    v = torch.full_like(k, 3e36)
    out = ka.cross_attn(torch.empty_like(q), q, k, v, 4)
    assert torch.equal(out, v.expand_as(out))
