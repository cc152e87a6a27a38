"""A text encoder's layer past 32 bits: caches, rows and strides whose bytes lie beyond 2^32, and millions of keys of one token."""

import pytest
import torch

import kiln_amd as ka
from test_linear_mxfp8_gpu import make
from test_prompt_attn_gpu import DEV, check

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def run(q, k, v, Hq, Hkv, starts, places, prefix=None, out=None):
    out = torch.empty_like(q) if out is None else out
    ka.prompt_attn(out, q, k, v, Hq, Hkv, q_start=ints(*starts), k_start=ints(*[a for a, _ in places]), k_len=ints(*[n for _, n in places]), prefix=prefix)
    check(out, q, k, v, Hq, Hkv, [(a, b - a, *p) for a, b, p in zip(starts, starts[1:], places)], prefix, what=f"{places}")


@pytest.mark.parametrize("nq", [1, 50])
def test_places_far_into_a_cache(gpu, nq):
    """K and V of 4.5 GiB each; sequences at their beginning, across 2^32 bytes and at their end."""
    n, W = 2_300_000, 8 * 128
    k, v = (torch.empty(n, W, dtype=F16, device=DEV) for _ in range(2))
    places = [(0, 100), ((1 << 21) - 60, 300), (n - 777, 777)]
    for a, m in places:
        k[a:a + m], v[a:a + m] = torch.randn(m, W, device=DEV), torch.randn(m, W, device=DEV)
    run(torch.randn(3 * nq, 16 * 128, device=DEV).half(), k, v, 16, 8, [0, nq, 2 * nq, 3 * nq], places)


def test_rows_far_apart(gpu):
    """Rows 2^24 elements apart, the most there may be, in every tensor."""
    def rows(n, w):
        t = torch.empty(n, 1 << 24, dtype=BF16, device=DEV)[:, (1 << 24) - w:]
        t.copy_(torch.randn(n, w, device=DEV))
        return t
    q, k, v, out, pk, pv = rows(150, 256), rows(200, 128), rows(200, 128), rows(150, 256), rows(70, 128), rows(70, 128)
    run(q, k, v, 4, 2, [0, 140, 150], [(3, 180), (185, 12)], (pk, pv), out)


@pytest.mark.parametrize("dt", [F16, BF16])
def test_millions_of_keys(gpu, dt):
    """A token, and three behind each other, after two million keys."""
    n = 2_100_003
    k, v = (torch.randn(n, 64, device=DEV).to(dt) for _ in range(2))
    run(torch.randn(4, 128, device=DEV).to(dt), k, v, 2, 1, [0, 1, 4], [(0, n), (5, n - 5)])
    pre = (k[:1_000_001], v[:1_000_001])
    run(torch.randn(4, 128, device=DEV).to(dt), k[:500], v[:500], 2, 1, [0, 1, 4], [(0, 300), (300, 200)], pre)


def test_norm_of_far_rows(gpu):
    """Windows in rows 2^16 elements apart, 8.6 GiB to the last, and dense rows of more than 2^32 values: as near ones."""
    rows, dim = 70_000, 64
    w = torch.randn(dim, device=DEV).to(BF16)
    x, r = torch.randn(rows, dim, device=DEV).half(), torch.randn(rows, dim, device=DEV).half()
    y, h = torch.empty_like(x), torch.empty_like(r)
    ka.add_rmsnorm(y, x, r, w, h=h)
    big = [torch.empty(rows, 1 << 16, dtype=F16, device=DEV) for _ in range(2)]
    bx, br = big[0][:, -dim:], big[1][:, 8:8 + dim]
    bx.copy_(x)
    br.copy_(r)
    ka.add_rmsnorm(bx, bx, br, w)
    assert torch.equal(bx, y) and torch.equal(br, h)
    del big, bx, br
    rows, dim = (1 << 21) + 37, 2048
    x = torch.empty(rows, dim, dtype=F16, device=DEV)
    x[:1000], x[-1000:] = torch.randn(1000, dim, device=DEV), torch.randn(1000, dim, device=DEV)
    x[1000:-1000] = 1
    codes, scales = torch.empty(rows, dim, dtype=torch.uint8, device=DEV), torch.empty(rows, dim // 32, dtype=torch.uint8, device=DEV)
    for make_codes in (lambda c, s, t: ka.add_rmsnorm(c, t, scales=s), lambda c, s, t: ka.mxfp8_quantize(t, c, s)):
        codes.fill_(1)
        make_codes(codes, scales, x)
        for at in (slice(0, 1000), slice(rows // 2, rows // 2 + 8), slice(rows - 1000, rows)):
            c, s = torch.empty_like(codes[at]), torch.empty_like(scales[at])
            make_codes(c, s, x[at])
            assert torch.equal(c, codes[at]) and torch.equal(s, scales[at])
    ka.mxfp8_dequantize(x, codes, scales)
    back = torch.empty(1000, dim, dtype=F16, device=DEV)
    ka.mxfp8_dequantize(back, codes[-1000:].contiguous(), scales[-1000:].contiguous())
    assert torch.equal(back, x[-1000:])


@pytest.mark.parametrize("N", [48, 300])
def test_linear_of_many_rows(gpu, N):
    """Codes of 4.4 GiB: 1000 rows over and over, each time the same result; y's rows far apart for the last of them."""
    T, K, n = 1000, 8192, 570
    codes, scales, w, xv, wv = make(T, N, K, seed=6)
    many, many_s = codes.repeat(n, 1), scales.repeat(n, 1)
    for dt, epi in ((torch.float32, ka.KILN_EPI_F32), (F16, ka.KILN_EPI_F16)):
        y = torch.empty(n * T, N, dtype=dt, device=DEV)
        ka.linear_mxfp8(y, many, many_s, w, epi=epi)
        assert torch.equal(y.view(n, T, N), y[:T].expand(n, T, N))
        ref = xv @ wv.t()
        assert (y[:T].double() - ref).abs().max() <= 2.0 ** -9 * ref.abs().max()
    apart = torch.empty(T, 1 << 23, dtype=torch.float16, device=DEV)[:, -N:]
    ka.linear_mxfp8(apart, codes, scales, w, epi=ka.KILN_EPI_F16)
    near = torch.empty(T, N, dtype=F16, device=DEV)
    ka.linear_mxfp8(near, codes, scales, w, epi=ka.KILN_EPI_F16)
    assert torch.equal(apart, near)
