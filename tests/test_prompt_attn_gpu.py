"""kiln_prompt_attn against 64-bit causal attention: packed sequences of every length about a tile's, cached keys, shared prefixes, shared
key heads, strides, lengths on the device that are wrong, values that move the maximum, and what hidden keys may hold."""

import math

import pytest
import torch

import kiln_amd as ka

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
NAN = float("nan")


def visible(nq, nk, P):
    """[nq, P + nk]: the keys that each query sees."""
    own = torch.arange(nk, device=DEV) <= torch.arange(nk - nq, nk, device=DEV)[:, None]
    return torch.cat((torch.ones(nq, P, dtype=torch.bool, device=DEV), own), 1)


def check(out, q, k, v, Hq, Hkv, seqs, prefix=None, scale=None, what=""):
    """out against softmax attention in 64 bits; seqs: (first query, queries, first key, keys) of each sequence. Hidden keys do not enter the
    reference at all. Rows of no sequence are not looked at."""
    Dh = q.shape[1] // Hq
    scale = Dh ** -0.5 if scale is None else scale
    u, P, worst = torch.finfo(q.dtype).eps / 2, 0 if prefix is None else prefix[0].shape[0], 0.0
    for q0, nq, k0, nk in seqs:
        if not nq:
            continue
        see = visible(nq, nk, P)
        n = see.sum(1, keepdim=True).double()
        for h in range(Hq):
            hs, kv = slice(h * Dh, (h + 1) * Dh), slice(h * Hkv // Hq * Dh, (h * Hkv // Hq + 1) * Dh)
            qq, kk, vv = q[q0:q0 + nq, hs].double(), k[k0:k0 + nk, kv].double(), v[k0:k0 + nk, kv].double()
            if P:
                kk, vv = torch.cat((prefix[0][:, kv].double(), kk)), torch.cat((prefix[1][:, kv].double(), vv))
            s = (scale * qq @ kk.t()).masked_fill(~see, -math.inf)
            p = torch.softmax(s, -1).masked_fill(~see, 0)  # (a row without keys: zeros)
            ref, wmag = p @ vv, p @ vv.abs()
            # the scores' magnitude: sum |q k| bounds the product's rounding, the score range the exponent's
            mag = (scale * (qq.abs() @ kk.abs().t())).masked_fill(~see, 0)
            smag = (mag.amax(-1) + (s.amax(-1) - s.masked_fill(~see, math.inf).amin(-1)).clamp(min=0).nan_to_num(0, 0, 0))[:, None] if mag.shape[1] else mag.new_zeros(nq, 1)
            # relative to the weights: P rounded to the type (u); scores within (Dh / 32 + 2) 2^-23 of sum |q k| and their exponents'
            # arguments within 2^-23 of the score range; sums of up to n / 4 + 64 terms; 2^-21 for exp2, the rescales and the division
            tol = (u + (Dh / 32 + 2) * 2.0 ** -22 * smag + (n / 4 + 64) * 2.0 ** -24 + 2.0 ** -21) * wmag
            if q.dtype == torch.float16:  # weights below fp16's normal range (2^-25), against a largest of 2^7 at least
                tol = tol + 2.0 ** -32 * (see.double() @ vv.abs())
            tol = tol + u * (ref.abs() + tol) + torch.finfo(q.dtype).smallest_normal * u
            got = out[q0:q0 + nq, hs].double()
            assert torch.isfinite(got).all(), (what, q0, h)
            err = (got - ref).abs()
            assert (err <= tol).all(), (what, q0, nq, nk, h, (err / tol).max().item())
            worst = max(worst, (err / tol).max().item())
    print(f"[prompt_attn] {what}: worst error / tolerance {worst:.3f}", flush=True)


class Case:
    """Packed sequences of lens (queries, keys), keys packed apart from the queries with gaps between them where cached (gap rows NaN)."""

    def __init__(self, lens, Hq, Hkv, Dh, dt, P=0, seed=0, pad=0, lead=0, cached=None, extra=0):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.Hq, self.Hkv, self.Dh = Hq, Hkv, Dh
        own = all(nq == nk for nq, nk in lens) if cached is None else not cached
        q0, self.seqs, starts = lead, [], [lead]
        k0 = lead if own else 2
        for nq, nk in lens:
            self.seqs.append((q0, nq, q0 if own else k0, nk))
            q0 += nq
            k0 += nk + 3
            starts.append(q0)
        Tq = q0 + pad
        Tk = Tq if own else k0

        def rows(n, w, size=1):
            t = torch.full((n, w + extra), NAN, dtype=dt, device=DEV)[:, :w]
            t.copy_(torch.randn(n, w, device=DEV, generator=g) * size)
            return t

        grow = 1 + torch.randn(Tk, 1, device=DEV, generator=g).abs()
        self.q, self.k, self.v = rows(Tq, Hq * Dh), rows(Tk, Hkv * Dh, grow), rows(Tk, Hkv * Dh)
        used = torch.zeros(Tk, dtype=torch.bool, device=DEV)
        for _, _, a, n in self.seqs:
            used[a:a + n] = True
        self.k[~used], self.v[~used] = NAN, NAN
        self.prefix = (rows(P, Hkv * Dh, 1.5), rows(P, Hkv * Dh)) if P else None
        self.q_start = torch.tensor(starts, dtype=torch.int32, device=DEV)
        self.k_start = self.k_len = None
        if not own:
            self.k_start = torch.tensor([s[2] for s in self.seqs], dtype=torch.int32, device=DEV)
            self.k_len = torch.tensor([s[3] for s in self.seqs], dtype=torch.int32, device=DEV)
        self.out = rows(Tq, Hq * Dh)
        self.out.fill_(7.0)

    def run(self, **kw):
        return ka.prompt_attn(self.out, self.q, self.k, self.v, self.Hq, self.Hkv, q_start=self.q_start, k_start=self.k_start, k_len=self.k_len,
                              prefix=self.prefix, **kw)

    def check(self, what, **kw):
        check(self.out, self.q, self.k, self.v, self.Hq, self.Hkv, self.seqs, self.prefix, what=what, **kw)
        free = torch.ones(self.out.shape[0], dtype=torch.bool, device=DEV)
        for q0, nq, _, _ in self.seqs:
            free[q0:q0 + nq] = False
        assert (self.out[free] == 7).all(), what


WHOLE = [(1, 1), (0, 0), (31, 31), (32, 32), (33, 33), (0, 0), (64, 64), (65, 65), (130, 130)]
CACHED = [(1, 1), (1, 31), (0, 9), (1, 33), (3, 700), (64, 64), (17, 1000), (2, 65), (100, 164)]
LATE = [(10, 4), (3, 0), (1, 0), (70, 66)]  # queries ahead of the first key
TOKENS = [(1, n) for n in (1, 2, 31, 32, 33, 64, 100, 500, 1300, 2049, 3, 77)]
HEADS = [(1, 1, 64), (4, 2, 128), (16, 8, 128), (7, 1, 64), (32, 4, 64), (12, 4, 128)]


@pytest.mark.parametrize("Hq,Hkv,Dh", HEADS)
@pytest.mark.parametrize("P", [0, 1, 31, 32, 33, 200])
@pytest.mark.parametrize("name", ["whole", "cached", "late", "tokens"])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_sequences(gpu, name, P, Hq, Hkv, Dh, dt):
    lens = dict(whole=WHOLE, cached=CACHED, late=LATE, tokens=TOKENS)[name]
    c = Case(lens, Hq, Hkv, Dh, dt, P=P, seed=P + Hq, pad=5, lead=2)
    c.run()
    c.check(f"{name} P={P} {Hq}/{Hkv} of {Dh} {dt}")


MANY = [
    ([(1500, 1500)], 4, 2, 128, 0), ([(2049, 2049)], 2, 2, 64, 0), ([(700, 700), (1, 1), (1200, 1200), (5, 5)], 16, 8, 128, 0), ([(900, 3000)], 2, 1, 128, 0),
    ([(1, 20000)], 2, 1, 128, 0), ([(1, 9001), (1, 4)], 16, 2, 64, 0), ([(40, 6000), (7, 100)], 8, 8, 128, 0), ([(1, 300)] * 40, 16, 8, 128, 2500),
    ([(1, 1)] * 70, 4, 1, 64, 5000), ([(300, 300)] * 3, 16, 8, 128, 1000), ([(2, 2)], 1, 1, 128, 9000), ([(1, 12)] * 300, 4, 2, 128, 70),
    ([(i % 7, i % 7 + i % 41) for i in range(600)], 2, 1, 64, 0), ([(200, 200)] * 40, 16, 8, 128, 0), ([(150, 150)] * 90, 8, 8, 64, 33),
    ([(70, 70)] * 5, 4, 4, 64, 0), ([(20, 220)] * 6, 8, 8, 64, 3001), ([(30, 30), (25, 400)] * 4, 2, 2, 128, 4000), ([(33, 9000)], 4, 4, 64, 0)]


def form_of(lens, Hq, Hkv, Dh, P):
    Tq, own = sum(nq for nq, _ in lens) + 1, all(nq == nk for nq, nk in lens)
    return Dh, ka.prompt_attn_form(len(lens), Tq, Tq if own else sum(nk + 3 for _, nk in lens) + 2, P, Hq, Hkv, Dh)


def test_cases_reach_every_form(gpu):
    """A workgroup per row tile of 64 or 128 rows; keys shared out over single waves of 16 rows and workgroups of 64; a prefix once for all rows."""
    forms = {form_of(*c) for c in MANY}
    assert forms == {(d, f) for d in (64, 128) for f in ((64, 0), (128, 0), (16, 1), (64, 1), (16, 2), (64, 2))}


@pytest.mark.parametrize("lens,Hq,Hkv,Dh,P", MANY)
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_long_and_many(gpu, lens, Hq, Hkv, Dh, P, dt):
    c = Case(lens, Hq, Hkv, Dh, dt, P=P, seed=len(lens), pad=1)
    c.run()
    c.check(f"{len(lens)} sequences from {lens[0]} P={P} {Hq}/{Hkv} of {Dh} {dt}")
    split = c.out.clone()
    c.run(workspace=torch.empty(0, dtype=torch.uint8, device=DEV))
    c.check("the same without a workspace")
    c.run()
    assert torch.equal(c.out, split)  # the same bits again


@pytest.mark.parametrize("Hq,Hkv,Dh,P", [(32, 4, 64, 4001), (4, 2, 128, 12000)])
def test_many_tokens_behind_a_long_prefix(gpu, Hq, Hkv, Dh, P):
    """Single tokens whose prefix is taken by workgroups of 64 rows, each sequence's own keys too."""
    lens = [(1, 1 + 13 * i % 90) for i in range(150)]
    assert form_of(lens, Hq, Hkv, Dh, P) == (Dh, (64, 2))
    c = Case(lens, Hq, Hkv, Dh, torch.float16, P=P, seed=9, pad=1)
    c.run()
    c.check(f"150 tokens behind {P}")


def test_one_sequence_without_starts(gpu):
    c = Case([(77, 77)], 4, 2, 64, torch.float16)
    ka.prompt_attn(c.out, c.q, c.k, c.v, 4, 2)
    c.check("no starts")


def test_stacked_projection(gpu):
    """q, k and v as columns of one projection's rows, out with a stride of its own; the rest stays."""
    c = Case([(40, 40), (3, 3)], 4, 2, 128, torch.bfloat16)
    T, Wq, Wk = 43, 512, 256
    qkv = torch.randn(T, Wq + 2 * Wk, device=DEV).to(torch.bfloat16)
    q, k, v = qkv[:, :Wq], qkv[:, Wq:Wq + Wk], qkv[:, Wq + Wk:]
    buf = torch.full((T, Wq + 24), 5.0, dtype=torch.bfloat16, device=DEV)
    out = buf[:, 8:8 + Wq]
    ka.prompt_attn(out, q, k, v, 4, 2, q_start=c.q_start)
    check(out, q, k, v, 4, 2, c.seqs, what="stacked")
    assert (buf[:, :8] == 5).all() and (buf[:, 8 + Wq:] == 5).all()


@pytest.mark.parametrize("bad", [math.inf, -math.inf, NAN])
@pytest.mark.parametrize("Hq,Hkv,Dh", [(4, 2, 128), (7, 1, 64)])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("P", [0, 40])
def test_hidden_keys_hold_anything(gpu, bad, Hq, Hkv, Dh, dt, P):
    """One token's K and V, or a single value of V, are not finite: earlier tokens' rows are as without it, later ones' as in 64 bits:
    a row that sees an infinity of V has that infinity in its column."""
    n, at = 200, 70
    c = Case([(n, n), (30, 30)], Hq, Hkv, Dh, dt, P=P, seed=3)
    c.run()
    clean = c.out.clone()
    rows = torch.arange(n + 30, device=DEV)
    later = (rows >= at) & (rows < n)
    # a whole token
    k, v = c.k.clone(), c.v.clone()
    c.k[at], c.v[at] = bad, bad
    c.run()
    assert torch.equal(c.out[~later], clean[~later])
    assert not torch.isfinite(c.out[later]).any()
    # single values of V in several places of a tile
    c.k, c.v = k, v.clone()
    places = [(at, 0), (at + 5, Dh - 1), (at + 23, Dh // 2 + 1), (at + 100, 3)]
    for t, d in places:
        c.v[t, d] = bad
    c.run()
    want = torch.zeros(n + 30, Hkv * Dh, dtype=torch.bool, device=DEV)
    for t, d in places:
        want[t:n, d] = True
    want = want.view(-1, Hkv, 1, Dh).expand(-1, Hkv, Hq // Hkv, Dh).reshape(n + 30, Hq * Dh)
    assert torch.equal(c.out[~want], clean[~want])
    got = c.out[want]
    assert (torch.isnan(got) if math.isnan(bad) else got == bad).all()


def test_far_scores_and_moving_maxima(gpu):
    """Scores of up to 2^22 in log2, rising and falling along the keys."""
    for falling in (False, True):
        c = Case([(150, 150)], 2, 1, 64, torch.bfloat16, seed=9)
        grow = torch.linspace(1, 3e3, 150, device=DEV)[:, None].to(torch.bfloat16)
        c.k *= grow.flip(0) if falling else grow
        c.q *= 30
        # the exponent's argument is rounded in units of the scores' last place: far rows are checked against weights that are 0 or 1 by
        # a wide margin only
        c.run()
        assert torch.isfinite(c.out).all()
        s = (c.q[:, :64].double() @ c.k.double().t() / 8).masked_fill(~visible(150, 150, 0), -math.inf)
        top = s.topk(2, -1).values
        clear = top[:, 0] - top[:, 1] > 100
        assert clear.sum() > 50
        ref = c.v.double()[s.argmax(-1)]
        assert torch.equal(c.out[:, :64].double()[clear], ref[clear])


def test_large_values(gpu):
    """bf16 values near the type's largest survive any number of keys."""
    c = Case([(300, 300), (1, 1)], 2, 2, 128, torch.bfloat16, seed=4, P=64)
    big = torch.finfo(torch.bfloat16).max
    c.v.fill_(big)
    c.prefix[1].fill_(big)
    c.run()
    assert (c.out >= big * (1 - 2.0 ** -7)).all()


def test_masked_scores_of_the_lowest_value(gpu):
    """Keys whose every score is -inf: zeros, as for no key at all."""
    c = Case([(5, 5)], 2, 1, 64, torch.float16)
    c.q.fill_(1.0)
    c.k.fill_(-math.inf)
    c.run()
    assert (c.out == 0).all()


def test_starts_that_are_wrong(gpu):
    """Starts and lengths are clamped to the tensors: nothing outside is read or written, whatever they say."""
    c = Case([(20, 20), (30, 30), (10, 10)], 4, 2, 64, torch.float16, pad=4, cached=True)
    n = c.q.shape[0]
    for starts, ks, kl in (([-5, 20, 1 << 30, 7], [-3, 1 << 30, 5], [1 << 30, 4, -7]), ([50, 10, 60, 0], [0, 0, 0], [10, 1 << 31 - 1, 20]),
                           ([0, 0, 0, 0], [0, 0, 0], [0, 0, 0]), ([n, n + 1, n + 2, n + 3], [0, 0, 0], [5, 5, 5])):
        c.q_start.copy_(torch.tensor(starts))
        c.k_start.copy_(torch.tensor(ks))
        c.k_len.copy_(torch.tensor(kl).clamp(max=(1 << 31) - 1))
        c.k.nan_to_num_(0)
        c.v.nan_to_num_(0)
        c.out.fill_(7.0)
        c.run()
        assert torch.isfinite(c.out).all()
        cl = [min(max(s, 0), n) for s in starts]
        free = torch.ones(n, dtype=torch.bool, device=DEV)
        for a, b in zip(cl, cl[1:]):
            free[a:b] = False
        assert (c.out[free] == 7).all()


def test_many_sequences(gpu):
    """The most sequences there may be, single tokens with a key each (out = v), and all of them claiming all rows (nothing else
    is touched)."""
    B, H, Dh = 1 << 14, 2, 64
    q, k, v = (torch.randn(B, H * Dh, device=DEV).half() for _ in range(3))
    out, starts = torch.empty_like(q), torch.arange(B + 1, dtype=torch.int32, device=DEV)
    ka.prompt_attn(out, q, k, v, H, H, q_start=starts)
    assert torch.equal(out, v)
    with pytest.raises(ka.KilnError):
        ka.prompt_attn(out, q, k, v, H, H, q_start=torch.arange(B + 2, dtype=torch.int32, device=DEV))
    for rows in (40, 2000):
        starts = (torch.arange(B + 1, device=DEV) % 2 * rows).to(torch.int32)
        for P in (0, 100):
            out.fill_(7.0)
            pre = (k[:P], v[:P]) if P else None
            ka.prompt_attn(out[:rows], q[:rows], k[:rows], v[:rows], H, H, q_start=starts, prefix=pre)
            assert (out[rows:] == 7).all()


def test_shared_cache_places(gpu):
    """Sequences may read the same keys: three streams that continue one prompt."""
    c = Case([(1, 90)] * 3, 4, 2, 128, torch.float16, cached=True)
    c.k_start.fill_(2)
    c.k_len.copy_(torch.tensor([90, 60, 90]))
    c.seqs = [(0, 1, 2, 90), (1, 1, 2, 60), (2, 1, 2, 90)]
    c.run()
    c.check("shared places")


@pytest.mark.parametrize("lens,P", [(WHOLE, 0), (TOKENS, 0), (TOKENS, 300), ([(1, 9000)] * 2, 0)])
def test_capture_stream_and_replay(gpu, lens, P):
    """A captured call follows the lengths on the device; replays with eager work between them; another stream."""
    c = Case(lens, 16, 8, 128, torch.float16, P=P, cached=True)
    n = ka.prompt_attn_workspace_bytes(len(lens), c.q.shape[0], c.k.shape[0], P, 16, 8, 128)
    ws = torch.empty(n, dtype=torch.uint8, device=DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    c.run(workspace=ws, stream=s)
    s.synchronize()
    c.check("another stream")
    eager = c.out.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.run(workspace=ws)
    for i in range(3):
        c.out.fill_(7.0)
        ws.fill_(255)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(c.out, eager), i
        torch.randn(1000, device=DEV).sum().item()
    c.k_len.copy_((c.k_len * 2 // 3).clamp(min=1))
    c.seqs = [(a, nq, k0, int(m)) for (a, nq, k0, _), m in zip(c.seqs, c.k_len.tolist())]
    c.out.fill_(7.0)
    g.replay()
    torch.cuda.synchronize()
    c.check("replay with other lengths")


def test_no_rows(gpu):
    q = torch.empty(0, 256, dtype=torch.float16, device=DEV)
    kv = torch.empty(0, 128, dtype=torch.float16, device=DEV)
    ka.prompt_attn(q, q, kv, kv, 4, 2)
    c = Case([], 4, 2, 64, torch.float16, pad=3)
    c.run()
    assert (c.out == 7).all()
