"""kiln_cross_attn at the ends of its types' ranges: values up to the largest finite number, scores far from zero, in every form."""
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


@pytest.mark.parametrize("B,Tq,Tk,Hq,Hkv,Dh", SHAPES)
@pytest.mark.parametrize("dt,e,sign", [(torch.float16, e, s) for e, s in ((10, 1), (17, 1), (20, -1), (26, 1), (26, -1), (30, 1), (30, -1))] +
                         [(torch.bfloat16, e, s) for e, s in ((10, -1), (17, 1), (20, 1), (26, -1), (30, 1), (36, -1), (60, 1), (100, -1))])
def test_scores_far_from_zero(gpu, B, Tq, Tk, Hq, Hkv, Dh, dt, e, sign):
    """Scores of +-2^e and twelve steps beside it, which rise along the keys for even heads and fall for odd ones: steps of 1 up to
    e = 20, where every key counts, of 2^(e - 22) from e = 26 on, where the keys of the largest score share the output."""
    near = e <= 20
    a = 0 if near else (e - 22) // 2
    b = 0 if near else e - 22 - a
    q, k, v = make(B, Tq, Tk, Hq, Hkv, Dh, dt)
    q, k = torch.zeros_like(q), torch.zeros_like(k)
    qv, kv = q.view(B, Tq, Hq, Dh), k.view(B, Tk, Hkv, Dh)
    qv[..., 0], kv[..., 0] = 2.0 ** (e // 2), sign * 2.0 ** (e - e // 2)
    qv[:, :, 0::2, 1], qv[:, :, 1::2, 1] = 2.0 ** a, -(2.0 ** a)
    j = torch.arange(Tk, device=DEV) * 12 // Tk
    kv[..., 1] = (j * 2.0 ** b)[None, :, None].to(dt)
    step = 2.0 ** (a + b)
    p = torch.softmax(torch.stack([j * step, -j * step]).double(), -1)[torch.arange(Hq, device=DEV) % 2]  # [Hq, Tk]
    vv = v.double().view(B, Tk, Hkv, Dh).repeat_interleave(Hq // Hkv, 2)
    over = lambda x: (p.t()[None, :, :, None] * x).sum(1).reshape(B, 1, Hq * Dh)  # noqa: E731
    ref, mag = over(vv), over(vv.abs())
    u = torch.finfo(dt).eps / 2
    # P rounded to the type; sums; exp2, the rescales and the division. The scores are exact in fp32; times log2 e they are off by
    # half a unit of 2^e's last place, d = 2^(e - 24), the key's and the maximum's: weights within 2^(2 d), their share within 2^(4 d).
    # From e = 26 on a key of the next score has at most 2^(-1.44 2^(e - 22) + 2 d) <= 2^-15 of the weight of one of the largest,
    # and there are at most as many of each score as one more than of another: twice 11 in all, and what they hold
    rel = u + (Tk / 4 + 64) * 2.0 ** -24 + 2.0 ** -21
    tol = (rel + (2.0 ** (4 * 2.0 ** (e - 24)) - 1 if near else 0)) * mag
    if not near:
        tol = tol + 44 * 2.0 ** -15 * vv.abs().amax(1).reshape(B, 1, Hq * Dh)
    if dt == torch.float16:
        tol = tol + 2.0 ** -32 * vv.abs().sum(1).reshape(B, 1, Hq * Dh)
    tol = tol + u * (ref.abs() + tol) + torch.finfo(dt).smallest_normal * u
    for out in both(q, k, v, Hq, Hkv, scale=1.0):
        err = (out.double() - ref).abs()
        print(f"[cross_attn] {B} {Tq} {Tk} {Hq} {Hkv} {Dh} {dt} 2^{e}: worst error / tolerance {(err / tol).max():.3f}", flush=True)
        assert torch.isfinite(out).all()
        assert (err <= tol).all()
