"""kiln_rope against 64-bit rotations: layouts, partial heads, types, strides, in place, far and negative positions."""
import math

import pytest
import torch

import kiln_amd as ka

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def reference(x, H, Dh, f, pos, inter, m):
    """The rotated rows in 64 bits, and per element |u| + |v| of its pair (0 where it does not turn)."""
    T, rot = x.shape[0], 2 * f.numel()
    a = pos.double()[:, None] * f
    c, s = m * torch.cos(a)[:, None], m * torch.sin(a)[:, None]
    x = x.double().reshape(T, H, Dh)
    y, mag = x.clone(), torch.zeros_like(x)
    i0, i1 = (slice(0, rot, 2), slice(1, rot, 2)) if inter else (slice(0, rot // 2), slice(rot // 2, rot))
    u, v = x[..., i0], x[..., i1]
    y[..., i0], y[..., i1] = u * c - v * s, v * c + u * s
    mag[..., i0] = mag[..., i1] = u.abs() + v.abs()
    return y.reshape(T, H * Dh), mag.reshape(T, H * Dh)


def check(y, x, H, Dh, f, pos, inter, m, what):
    ref, mag = reference(x, H, Dh, f, pos, inter, m)
    # per product: cos or sin off by 2^-23 (its function) + pi 2^-24 (the fraction of a turn in fp32), their scaling, the product
    # and the sum by 2^-24 each: (2 + 3.2 + 3) 2^-24 of |u| + |v|; then the output's rounding, or its subnormals' step
    u = torch.finfo(x.dtype).eps / 2
    tol = 9 * 2.0 ** -24 * m * mag
    tol = tol + u * (ref.abs() + tol) * (mag > 0) + torch.finfo(x.dtype).smallest_normal * u
    err = (y.double() - ref).abs()
    print(f"[rope] {what}: worst error / tolerance {(err / tol).max():.3f}", flush=True)
    assert (err <= tol).all()
    assert torch.equal(y.double()[mag == 0], ref[mag == 0])


@pytest.mark.parametrize("T,H,Dh,rot", [(1, 1, 2, 2), (1, 16, 128, 128), (3, 5, 80, 32), (77, 16, 64, 64), (130, 2, 96, 48), (33, 3, 20, 14),
                                        (5, 1, 1024, 1024), (700, 20, 128, 64), (2, 300, 256, 256), (1500, 1, 64, 64)])
@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("inter", [False, True])
def test_rope(gpu, T, H, Dh, rot, dt, inter):
    g = torch.Generator(device=DEV).manual_seed(T * 7 + H)
    x = torch.randn(T, H * Dh, device=DEV, generator=g).to(dt)
    f, m = ka.rope_freqs(rot, 1e4, "ramp", 4.0, 4096, device=DEV)
    pos = torch.randint(-5, 1000000, (T,), device=DEV, generator=g, dtype=torch.int32)
    y = ka.rope(torch.full_like(x, float("nan")), x, H, Dh, f, pos=pos, interleaved=inter, mscale=m)
    check(y, x, H, Dh, f, pos, inter, m, f"{T}x{H}x{Dh} rot {rot} {dt} inter {inter}")
    assert torch.equal(ka.rope(x.clone(), x, H, Dh, f, pos=pos, interleaved=inter, mscale=m), y)
    z = x.clone()
    ka.rope(z, z, H, Dh, f, pos=pos, interleaved=inter, mscale=m)  # in place
    assert torch.equal(z, y)


@pytest.mark.parametrize("off,ld", [(0, 400), (8, 408), (1, 401), (3, 390), (4, 388)])
@pytest.mark.parametrize("dt", [torch.float32, torch.float16])
def test_strides(gpu, off, ld, dt):
    """Row strides and bases of every alignment; nothing beside the heads is touched."""
    T, H, Dh, rot = 19, 3, 128, 96
    f, m = ka.rope_freqs(rot, device=DEV)
    buf = torch.randn(T * ld + off + 16, device=DEV).to(dt)
    x = buf[off:off + T * ld].view(T, ld)[:, :H * Dh]
    out = torch.full((T * 416 + 16,), 7.0, device=DEV, dtype=dt)
    y = out[2:2 + T * 416].view(T, 416)[:, :H * Dh]
    for inter in (False, True):
        ka.rope(y, x, H, Dh, f, pos0=11, interleaved=inter)
        check(y, x, H, Dh, f, torch.arange(11, 11 + T, device=DEV), inter, m, f"off {off} ld {ld} {dt}")
    assert (out[2:2 + T * 416].view(T, 416)[:, H * Dh:] == 7).all() and (out[:2] == 7).all() and (out[2 + T * 416:] == 7).all()
    before = buf.clone()
    z = x.clone()
    ka.rope(x, x, H, Dh, f, pos0=11)  # in place on the strided rows
    want = ka.rope(torch.empty_like(z), z, H, Dh, f, pos0=11)
    assert torch.equal(x, want)
    rest = torch.ones_like(buf, dtype=torch.bool)
    rest[off:off + T * ld].view(T, ld)[:, :H * Dh] = False
    assert torch.equal(buf[rest], before[rest])


def test_side_by_side(gpu):
    """Queries and keys of one stacked projection: a call on both (neighbouring heads), and out of one part into another."""
    T, Dh = 40, 64
    f, _ = ka.rope_freqs(Dh, device=DEV)
    x = torch.randn(T, 6 * Dh, device=DEV).half()
    want = ka.rope(torch.empty(T, 6 * Dh, device=DEV).half(), x, 6, Dh, f)
    part = x.clone()
    ka.rope(part[:, :4 * Dh], part[:, :4 * Dh], 4, Dh, f)
    assert torch.equal(part[:, :4 * Dh], want[:, :4 * Dh]) and torch.equal(part[:, 4 * Dh:], x[:, 4 * Dh:])
    ka.rope(part[:, 4 * Dh:], x[:, :2 * Dh], 2, Dh, f)
    assert torch.equal(part[:, 4 * Dh:], want[:, :2 * Dh])
    ka.rope(part[:, :2 * Dh], part[:, 4 * Dh:], 2, Dh, f)  # same buffer, other columns
    assert torch.equal(part[:, 4 * Dh:], want[:, :2 * Dh])
    with pytest.raises(ka.KilnError):
        ka.rope(part[:, Dh:3 * Dh], part[:, :2 * Dh], 2, Dh, f)


@pytest.mark.parametrize("at", [0, 2 ** 31 - 8, -2 ** 31])
def test_far_positions(gpu, at):
    """pos0 + t past 32 bits' fp32 precision and up to the ends of int32, with positions given and counted."""
    T, H, Dh = 7, 2, 64
    f, m = ka.rope_freqs(Dh, 1e4, device=DEV)
    x = torch.randn(T, H * Dh, device=DEV)
    p = torch.arange(T, device=DEV, dtype=torch.int64) + at
    y = ka.rope(torch.empty_like(x), x, H, Dh, f, pos0=at)
    assert torch.equal(y, ka.rope(torch.empty_like(x), x, H, Dh, f, pos=p.to(torch.int32)))
    # the angle itself is rounded in 64 bits on both sides: |p f| 2^-52, up to 2^-21 rad here
    ref, mag = reference(x, H, Dh, f, p, False, m)
    tol = (10 * 2.0 ** -24 + abs(at) * 2.0 ** -51) * mag + 2.0 ** -24 * ref.abs()
    assert ((y.double() - ref).abs() <= tol).all()


def test_inverse_is_the_gradient(gpu):
    """<r, rope(x)> has the gradient rope with -pos of r: against the formula's and against differences."""
    T, H, Dh, rot = 6, 2, 32, 24
    f, m = ka.rope_freqs(rot, 1e4, "ramp", 2.0, 100, device=DEV)
    pos = torch.randint(0, 5000, (T,), device=DEV, dtype=torch.int32)
    x, r = torch.randn(T, H * Dh, device=DEV), torch.randn(T, H * Dh, device=DEV)
    for inter in (False, True):
        grad = ka.rope(torch.empty_like(r), r, H, Dh, f, pos=-pos, interleaved=inter, mscale=m)
        xd = x.double().requires_grad_()
        a = pos.double()[:, None] * f
        c, s = m * torch.cos(a)[:, None], m * torch.sin(a)[:, None]
        h = xd.view(T, H, Dh)
        i0, i1 = (slice(0, rot, 2), slice(1, rot, 2)) if inter else (slice(0, rot // 2), slice(rot // 2, rot))
        rr = r.double().view(T, H, Dh)
        loss = ((h[..., i0] * c - h[..., i1] * s) * rr[..., i0]).sum() + ((h[..., i1] * c + h[..., i0] * s) * rr[..., i1]).sum() + \
            (h[..., rot:] * rr[..., rot:]).sum()
        loss.backward()
        mag = reference(r, H, Dh, f, -pos, inter, m)[1]
        assert ((grad.double() - xd.grad).abs() <= 10 * 2.0 ** -24 * m * mag + 2.0 ** -24 * xd.grad.abs()).all()
        # the map is linear: a difference of step 1 along d is exact but for the two results' rounding
        d = torch.randn_like(x)
        up, dn = (ka.rope(torch.empty_like(x), v, H, Dh, f, pos=pos, interleaved=inter, mscale=m).double() for v in (x + d, x))
        moved = ((x + d).double() - x.double())
        lhs, rhs = ((up - dn) * r.double()).sum(), (moved * grad.double()).sum()
        scale = (r.double().abs() * (x.abs() + d.abs()).double()).sum() * 4 * m
        assert (lhs - rhs).abs() <= 20 * 2.0 ** -24 * scale


def test_nonfinite_stay_in_their_pair(gpu):
    T, H, Dh = 4, 1, 16
    f, _ = ka.rope_freqs(8, device=DEV)
    x = torch.ones(T, Dh, device=DEV)
    x[1, 2], x[2, 12] = math.nan, math.inf
    y = ka.rope(torch.empty_like(x), x, H, Dh, f)
    bad = ~torch.isfinite(y)
    want = torch.zeros_like(bad)
    want[1, 2] = want[1, 6] = want[2, 12] = True
    assert torch.equal(bad, want)


def test_batch_of_rows_is_each_row(gpu):
    """A row's result does not depend on the call it is in, nor on how tokens and heads are spread."""
    T, H, Dh = 2500, 4, 64
    f, m = ka.rope_freqs(Dh, device=DEV)
    x = torch.randn(T, H * Dh, device=DEV).bfloat16()
    y = ka.rope(torch.empty_like(x), x, H, Dh, f)
    for t in (0, 1, 1249, 2499):
        assert torch.equal(ka.rope(torch.empty_like(x[:1]), x[t:t + 1], H, Dh, f, pos0=t), y[t:t + 1])


@pytest.mark.parametrize("inter", [False, True])
def test_rows_past_32_bits(gpu, inter):
    """Rows so far apart that elements pass 2^31 and bytes 2^32, into another part of themselves and in place."""
    T, H, Dh = 40, 2, 64
    f, _ = ka.rope_freqs(Dh, device=DEV)
    x = torch.randn(T, H * Dh, device=DEV).half()
    want = ka.rope(torch.empty_like(x), x, H, Dh, f, interleaved=inter)
    far = torch.empty(T, (1 << 26) + 8, dtype=torch.float16, device=DEV)
    far[:, :H * Dh] = x
    ka.rope(far[:, H * Dh:2 * H * Dh], far[:, :H * Dh], H, Dh, f, interleaved=inter)
    ka.rope(far[:, :H * Dh], far[:, :H * Dh], H, Dh, f, interleaved=inter)
    assert torch.equal(far[:, H * Dh:2 * H * Dh], want) and torch.equal(far[:, :H * Dh], want)
