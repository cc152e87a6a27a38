"""kiln_cross_attn against 64-bit attention: every form (rows per workgroup, keys split over waves and workgroups), shared key
heads, lengths, masks, strides, values that move the maximum, and what masked states may hold."""

import math

import pytest
import torch

import kiln_amd as ka

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def reference(q, k, v, Hq, Hkv, scale, keep):
    """Output, and per element the weighted magnitude sum p |v|, the plain sum |v| over the row's keys, and the score errors'
    scale, all in 64 bits. keep [B, Tk]."""
    B, Tq, W = q.shape
    Dh = W // Hq
    out, wmag, vsum, smag = (torch.zeros(B, Tq, W, dtype=torch.float64, device=DEV) for _ in range(4))
    for b in range(B):
        rows = keep[b].nonzero()[:, 0]
        if not len(rows):
            continue
        for h in range(Hq):
            kv = slice(h * Hkv // Hq * Dh, (h * Hkv // Hq + 1) * Dh)
            hs = slice(h * Dh, (h + 1) * Dh)
            qq, kk, vv = q[b, :, hs].double(), k[b, rows, kv].double(), v[b, rows, kv].double()
            s = scale * qq @ kk.t()
            p = torch.softmax(s, -1)
            out[b, :, hs], wmag[b, :, hs] = p @ vv, p @ vv.abs()
            vsum[b, :, hs] = vv.abs().sum(0)
            # the scores' magnitude: sum |q k| bounds the product's rounding, the score range the exponent's
            smag[b, :, hs] = (scale * (qq.abs() @ kk.abs().t()).amax(-1) + (s.amax(-1) - s.amin(-1)))[:, None]
    return out, wmag, vsum, smag


def check(out, q, k, v, Hq, Hkv, keep=None, scale=None, what=""):
    B, Tq, W = q.shape
    Dh, Tk = W // Hq, k.shape[1]
    keep = torch.ones(B, Tk, dtype=torch.bool, device=DEV) if keep is None else keep
    ref, wmag, vsum, smag = reference(q, k, v, Hq, Hkv, Dh ** -0.5 if scale is None else scale, keep)
    u = torch.finfo(q.dtype).eps / 2
    # relative to the weights: P rounded to the type (u); scores within (Dh / 32 + 2) 2^-23 of sum |q k| and their exponents'
    # arguments within 2^-23 of the score range; sums of up to Tk / 4 + 64 terms; 2^-21 for exp2, the rescales and the division
    rel = u + (Dh / 32 + 2) * 2.0 ** -22 * smag + (Tk / 4 + 64) * 2.0 ** -24 + 2.0 ** -21
    tol = rel * wmag
    if q.dtype == torch.float16:
        tol = tol + 2.0 ** -32 * vsum  # weights below fp16's normal range (2^-25), against a largest of 2^7 at least
    tol = tol + u * (ref.abs() + tol) + torch.finfo(q.dtype).smallest_normal * u
    err = (out.double() - ref).abs()
    print(f"[cross_attn] {what}: worst error / tolerance {(err / tol).max():.3f}", flush=True)
    assert torch.isfinite(out).all(), what
    assert (err <= tol).all(), what
    none = ~keep.any(1)
    assert (out[none] == 0).all()


def make(B, Tq, Tk, Hq, Hkv, Dh, dt, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + Tq * 131 + Tk)
    q, k, v = (torch.randn(B, t, h * Dh, device=DEV, generator=g) for t, h in ((Tq, Hq), (Tk, Hkv), (Tk, Hkv)))
    k = k * (1 + torch.randn(B, Tk, 1, device=DEV, generator=g).abs())
    return q.to(dt), k.to(dt), v.to(dt)


SHAPES = [  # B, Tq, Tk, Hq, Hkv, Dh
    (1, 1, 1, 1, 1, 64), (1, 1, 33, 16, 16, 128), (3, 1, 300, 16, 4, 64), (2, 3, 65, 20, 4, 128), (8, 1, 5000, 16, 4, 128), (1, 1, 9001, 2, 1, 64),
    (1, 20, 2500, 2, 2, 64),
    (1, 16, 2049, 4, 4, 128), (1, 17, 31, 2, 2, 64), (1, 17, 4000, 2, 2, 128), (2, 65, 96, 10, 10, 64), (1, 200, 1111, 8, 8, 64), (1, 512, 120, 16, 16, 64),
    (1, 130, 1000, 12, 1, 128), (2, 700, 77, 10, 10, 64), (2, 2048, 77, 10, 10, 128), (2, 1025, 130, 32, 8, 64), (1, 4097, 40, 16, 16, 128),
    (2, 4097, 300, 16, 16, 64), (64, 1, 70, 16, 16, 64), (40, 2, 200, 16, 16, 128)]


def test_shapes_reach_every_form(gpu):
    """16 rows: one wave alone, on a range of the keys or on all of them, or four waves that split them; 64, 128 and (heads of 64) 256
    rows, 64 also on ranges of the keys."""
    forms = {(d, ka.cross_attn_form(*s)) for s in SHAPES for d in (s[5],)}
    want = {(16, 1, False), (16, 1, True), (16, 4, False), (64, 1, False), (64, 1, True), (128, 1, False)}
    assert forms == {(d, f) for d in (64, 128) for f in want} | {(64, (256, 1, False))}


@pytest.mark.parametrize("B,Tq,Tk,Hq,Hkv,Dh", SHAPES)
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_shapes(gpu, B, Tq, Tk, Hq, Hkv, Dh, dt):
    q, k, v = make(B, Tq, Tk, Hq, Hkv, Dh, dt)
    out = ka.cross_attn(torch.full_like(q, float("nan")), q, k, v, Hq, Hkv)
    check(out, q, k, v, Hq, Hkv, what=f"{B} {Tq} {Tk} {Hq} {Hkv} {Dh} {dt}")
    assert torch.equal(out, ka.cross_attn(torch.full_like(q, float("nan")), q, k, v, Hq, Hkv))
    # a workspace too small to split the keys over workgroups
    one = ka.cross_attn(torch.full_like(q, float("nan")), q, k, v, Hq, Hkv, workspace=torch.empty(16, dtype=torch.uint8, device=DEV))
    check(one, q, k, v, Hq, Hkv, what="unsplit")


@pytest.mark.parametrize("B,Tq,Tk,Hq,Hkv,Dh", [s for s in SHAPES if s[2] > 1])
@pytest.mark.parametrize("kind", ["len", "mask", "both"])
def test_lengths_and_masks(gpu, B, Tq, Tk, Hq, Hkv, Dh, kind):
    """Lengths from none to all, sparse masks, items without a key; what is left out holds NaN and infinities."""
    dt = torch.bfloat16 if kind == "mask" else torch.float16
    B = B + 3
    q, k, v = make(B, Tq, Tk, Hq, Hkv, Dh, dt)
    g = torch.Generator(device=DEV).manual_seed(Tk)
    keep = torch.ones(B, Tk, dtype=torch.bool, device=DEV)
    klen = kmask = None
    if kind != "mask":
        klen = torch.randint(0, Tk + 1, (B,), device=DEV, generator=g, dtype=torch.int32)
        klen[0], klen[1] = Tk + 5, 0
        klen[2] = -3
        keep &= torch.arange(Tk, device=DEV) < klen[:, None]
    if kind != "len":
        kmask = torch.rand(B, Tk, device=DEV, generator=g) < torch.rand(B, 1, device=DEV, generator=g)
        kmask[2] = False
        kmask[0, :-1] = False  # the last key alone
        kmask[0, -1] = True
        keep &= kmask
    bad = torch.tensor([float("nan"), float("inf"), float("-inf"), 3e4], device=DEV).to(dt)
    fill = bad[torch.randint(0, 4, k.shape, device=DEV, generator=g)]
    k2, v2 = torch.where(keep[..., None], k, fill), torch.where(keep[..., None], v, fill)
    out = ka.cross_attn(torch.full_like(q, float("nan")), q, k2, v2, Hq, Hkv, klen=klen, kmask=kmask)
    check(out, q, k, v, Hq, Hkv, keep, what=f"{kind} {B} {Tq} {Tk} {Hq} {Hkv} {Dh}")


@pytest.mark.parametrize("Tq", [1, 40, 600])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_moving_maximum(gpu, Tq, dt):
    """Scores up to several hundred that rise along the keys for some rows and fall for others: rescales at many tiles."""
    Tk, H, Dh = 700, 4, 64
    q, k, v = make(1, Tq, Tk, H, H, Dh, dt, 3)
    k = (k.float() * torch.linspace(0.1, 12, Tk, device=DEV)[None, :, None]).to(dt)
    check(ka.cross_attn(torch.empty_like(q), q, k, v, H), q, k, v, H, H, what=f"rising {dt}")
    k = k.flip(1).contiguous()
    check(ka.cross_attn(torch.empty_like(q), q, k, v, H), q, k, v, H, H, what=f"falling {dt}")
    check(ka.cross_attn(torch.empty_like(q), q, k, v, H, scale=1e-3), q, k, v, H, H, scale=1e-3, what="flat")


@pytest.mark.parametrize("Tq,Tk", [(1, 3000), (5, 40), (300, 200)])
def test_strides(gpu, Tq, Tk):
    """Queries, keys and values as columns of stacked projections, states shared by the batch (item stride 0), a strided mask, and
    an output among other columns that keep what they held."""
    B, Hq, Hkv, Dh = 3, 8, 2, 64
    g = torch.Generator(device=DEV).manual_seed(1)
    qb = torch.randn(B, Tq, Hq * Dh + 24, device=DEV, generator=g).half()
    kvb = torch.randn(1, Tk, 2 * Hkv * Dh + 8, device=DEV, generator=g).half()
    q, k, v = qb[..., 16:16 + Hq * Dh], kvb[..., :Hkv * Dh].expand(B, -1, -1), kvb[..., Hkv * Dh:2 * Hkv * Dh].expand(B, -1, -1)
    ob = torch.full((B, Tq + 2, Hq * Dh + 16), 5.0, device=DEV, dtype=torch.float16)
    out = ob[:, 1:-1, 8:8 + Hq * Dh]
    mb = (torch.rand(B, Tk + 3, device=DEV, generator=g) < 0.5).to(torch.uint8) * 200
    km = mb[:, 1:1 + Tk]
    ka.cross_attn(out, q, k, v, Hq, Hkv, kmask=km)
    check(out, q, k, v, Hq, Hkv, km != 0, what="strides")
    rest = torch.ones_like(ob, dtype=torch.bool)
    rest[:, 1:-1, 8:8 + Hq * Dh] = False
    assert (ob[rest] == 5).all()


@pytest.mark.parametrize("Tq", [1, 80])
def test_offsets_past_32_bits(gpu, Tq):
    """States 2^17 elements apart, 5 GB of them: byte offsets pass 2^32."""
    Tk, H, Dh, ld = 20000, 1, 128, 1 << 17
    kb = torch.zeros(Tk, ld, dtype=torch.float16, device=DEV)
    q, k, v = make(1, Tq, Tk, H, H, Dh, torch.float16)
    kb[:, :Dh], kb[:, Dh:2 * Dh] = k[0], v[0]
    out = ka.cross_attn(torch.empty_like(q), q, kb[None, :, :Dh], kb[None, :, Dh:2 * Dh], H)
    check(out, q, k, v, H, H, what=f"far rows Tq={Tq}")


def test_nonfinite_states_propagate(gpu):
    """A NaN among the kept states reaches its item's rows of that head and no other."""
    q, k, v = make(2, 20, 100, 4, 2, 64, torch.float16)
    k[0, 50, 3] = float("nan")
    v[1, 99, 64 + 7] = float("nan")
    out = ka.cross_attn(torch.empty_like(q), q, k, v, 4, 2)
    want = torch.zeros_like(out, dtype=torch.bool)
    want[0, :, :2 * 64] = True
    want[1, :, 2 * 64 + 7] = want[1, :, 3 * 64 + 7] = True
    assert torch.equal(torch.isnan(out), want)


@pytest.mark.parametrize("Tq", [1, 17])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_many_small_weights(gpu, dt, Tq):
    """One state of weight 1 and value 0 ahead of 2^17 of weight 2^-25.5 and value 1: together 2^-8.5 of the output, though each
    is less than fp16's least number. Without a workspace, so that they share a maximum."""
    Tk, Dh = (1 << 17) + 1, 64
    q, k, v = torch.zeros(1, Tq, Dh, device=DEV, dtype=dt), torch.zeros(1, Tk, Dh, device=DEV, dtype=dt), torch.ones(1, Tk, Dh, device=DEV, dtype=dt)
    q[:, :, 0], k[:, 1:, 0], v[:, 0] = 1, -25.5, 0  # a score in log2 each
    out = ka.cross_attn(torch.empty_like(q), q, k, v, 1, scale=math.log(2), workspace=torch.empty(16, dtype=torch.uint8, device=DEV))
    tail = 2.0 ** (17 - 25.5)
    # each weight 2^7 2^-25.5 to fp16's step of 2^-24, half of it (bf16: 2^-8 of it); 2^17 fp32 additions; the exponent's argument
    # within 2^-21; the output's rounding
    u = torch.finfo(dt).eps / 2
    rel = (2.0 ** -25 / 2.0 ** -18.5 if dt == torch.float16 else u) + 2.0 ** -24 * (Tk / 4 + 64) + 2.0 ** -21 + u
    assert ((out.double() - tail / (1 + tail)).abs() <= rel * tail).all()


def test_strides_of_single_rows(gpu):
    """One query and one state: their row strides mean nothing, however large or odd."""
    q, k, v = make(2, 1, 1, 2, 2, 64, torch.float16)
    odd = lambda t: t.as_strided(t.shape, (t.stride(0), (1 << 30) + 3, 1))  # noqa: E731
    assert torch.equal(ka.cross_attn(torch.empty_like(q), odd(q), odd(k), odd(v), 2), v)


def test_no_keys_at_all(gpu):
    q = torch.randn(2, 3, 128, device=DEV).half()
    k = torch.empty(2, 0, 128, device=DEV, dtype=torch.float16)
    out = ka.cross_attn(torch.full_like(q, 4.0), q, k, k, 1)
    assert (out == 0).all()


def test_one_key_returns_its_value(gpu):
    q, k, v = make(1, 90, 1, 4, 4, 128, torch.bfloat16)
    out = ka.cross_attn(torch.empty_like(q), q, k, v, 4)
    assert torch.equal(out, v.expand_as(out))


def test_python_checks(gpu):
    q, k, v = make(2, 4, 8, 4, 2, 64, torch.float16)
    o = torch.empty_like(q)
    i32 = dict(dtype=torch.int32, device=DEV)
    for bad in (lambda: ka.cross_attn(o, q, k, v, 4, 3), lambda: ka.cross_attn(o, q, k, v, 4, 4), lambda: ka.cross_attn(o, q, k, v[:, :7], 4, 2),
                lambda: ka.cross_attn(o.float(), q, k, v, 4, 2), lambda: ka.cross_attn(o, q, k.bfloat16(), v, 4, 2),
                lambda: ka.cross_attn(o, q, k, v, 4, 2, klen=torch.ones(3, **i32)), lambda: ka.cross_attn(o, q, k, v, 4, 2, klen=torch.ones(2, device=DEV)),
                lambda: ka.cross_attn(o, q, k, v, 4, 2, kmask=torch.ones(2, 7, dtype=torch.bool, device=DEV)),
                lambda: ka.cross_attn(o, q, k, v, 4, 2, kmask=torch.ones(2, 8, device=DEV)), lambda: ka.cross_attn(o[0], q[0], k[0], v[0], 4, 2)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(ka.KilnError):
        ka.cross_attn(o[:1].expand(2, -1, -1), q, k, v, 4, 2)
    with pytest.raises(ka.KilnError):
        ka.cross_attn(torch.empty(2, 4, 96, device=DEV).half(), torch.zeros(2, 4, 96, device=DEV).half(), *[torch.zeros(2, 8, 96, device=DEV).half()] * 2, 1)


@pytest.mark.parametrize("B,Tq,Tk,Hq,Hkv,Dh", [(3, 40, 100, 4, 2, 64), (2, 1, 2000, 8, 2, 128), (2, 3, 50, 2, 2, 128), (2, 1500, 90, 16, 16, 128)])
def test_items_side_by_side(gpu, B, Tq, Tk, Hq, Hkv, Dh):
    """Tokens first, items second: the results of items one behind the other, bit for bit. A stride at which the items' outputs meet is refused."""
    q, k, v = make(B, Tq, Tk, Hq, Hkv, Dh, torch.bfloat16)
    klen = torch.arange(B, device=DEV, dtype=torch.int32) * 7 + 33
    want = ka.cross_attn(torch.empty_like(q), q, k, v, Hq, Hkv, klen=klen)
    tb = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    out = tb(torch.empty_like(q))
    ka.cross_attn(out, tb(q), tb(k), tb(v), Hq, Hkv, klen=klen)
    assert torch.equal(out, want)
    W = Hq * Dh
    flat = torch.empty(B * Tq * W + W, device=DEV, dtype=q.dtype)
    if Tq > 1:
        with pytest.raises(ka.KilnError):
            ka.cross_attn(flat.as_strided((B, Tq, W), (W, W, 1)), q, k, v, Hq, Hkv, klen=klen)
