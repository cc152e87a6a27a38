"""A text encoder's layer as it is used: residual + RMS norm to MXFP8, the stacked projection, rotary positions, causal attention over packed prompts
(whole, behind a prefix, or single tokens on caches), the output projection, the MLP; stage by stage against 64 bits, captured and replayed, on
other streams, through the profiler's categories and through the C++ mirror."""
import os
import subprocess

import pytest
import torch

import kiln_amd as ka
from tests.test_prompt_attn_gpu import check as check_attention

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HERE = os.path.dirname(os.path.abspath(__file__))


class Layer:
    """A layer of D = H * Dh columns over packed sequences lens (new tokens, cached keys ahead of them) behind P prefix keys."""

    def __init__(self, lens, H, Hkv, Dh, mlp, P=0, seed=0):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.lens, self.H, self.Hkv, self.Dh, self.P, self.mlp = lens, H, Hkv, Dh, P, mlp
        self.D, self.KV = H * Dh, Hkv * Dh
        self.T = sum(n for n, _ in lens)

        def w(r, c):
            return ka.linear_mxfp4_weight((torch.randn(r, c, device=DEV, generator=g) / c ** 0.5).bfloat16())

        self.Wqkv, self.Wo, self.Wup, self.Wdown = w(self.D + 2 * self.KV, self.D), w(self.D, self.D), w(mlp, self.D), w(self.D, mlp)
        self.n1, self.n2 = ((1 + torch.randn(self.D, device=DEV, generator=g) / 4).bfloat16() for _ in range(2))
        starts = [0]
        for n, _ in lens:
            starts.append(starts[-1] + n)
        self.starts = starts
        self.q_start = torch.tensor(starts, dtype=torch.int32, device=DEV)
        # caches: places of the longest sequence's size, the new keys written behind the cached ones
        self.cap = max(n + c for n, c in lens)
        self.cached = any(c for _, c in lens)
        B = len(lens)
        self.k_start = torch.arange(B, dtype=torch.int32, device=DEV) * self.cap
        self.k_len = torch.tensor([n + c for n, c in lens], dtype=torch.int32, device=DEV)
        self.place = torch.cat([torch.arange(c, c + n, device=DEV) + s * self.cap for s, (n, c) in enumerate(lens)])
        self.cache = torch.randn(B * self.cap, 2 * self.KV, device=DEV, generator=g).half()
        self.prefix = tuple(torch.randn(P, self.KV, device=DEV, generator=g).half() for _ in range(2)) if P else None
        self.freqs, _ = ka.rope_freqs(Dh, 1e6, device=DEV)
        self.pos = torch.cat([torch.arange(P + c, P + c + n, device=DEV) for n, c in lens]).to(torch.int32)
        T, D = self.T, self.D
        u8 = dict(dtype=torch.uint8, device=DEV)
        self.c, self.s = torch.empty(T, D, **u8), torch.empty(T, D // 32, **u8)
        self.cm, self.sm = torch.empty(T, mlp, **u8), torch.empty(T, mlp // 32, **u8)
        f16 = dict(dtype=torch.float16, device=DEV)
        self.qkv, self.at, self.up, self.o = torch.empty(T, D + 2 * self.KV, **f16), torch.empty(T, D, **f16), torch.empty(T, mlp, **f16), torch.empty(T, D, **f16)
        Tk = self.cache.shape[0] if self.cached else T
        self.ws = torch.empty(ka.prompt_attn_workspace_bytes(B, T, Tk, P, H, Hkv, Dh), **u8)

    def inputs(self, seed):
        g = torch.Generator(device=DEV).manual_seed(100 + seed)
        return torch.randn(self.T, self.D, device=DEV, generator=g).half(), torch.randn(self.T, self.D, device=DEV, generator=g)

    def keys(self):
        """(k, v) rows that the attention reads: the projection's own, or the caches'."""
        t = self.cache if self.cached else self.qkv[:, self.D:]
        return t[:, :self.KV], t[:, self.KV:]

    def run(self, x, r, ws="own", stream=None, after=lambda name: None):
        """x: the last layer's output, added to the residual stream r in place; r leaves with this layer's MLP added."""
        k = dict(stream=stream)
        D, KV = self.D, self.KV
        ka.add_rmsnorm(self.c, x, r, self.n1, scales=self.s, **k)
        after("norm")
        ka.linear_mxfp8(self.qkv, self.c, self.s, self.Wqkv, epi=ka.KILN_EPI_F16, **k)
        after("projected")
        q, kk = self.qkv[:, :D], self.qkv[:, D:D + KV]
        ka.rope(q, q, self.H, self.Dh, self.freqs, pos=self.pos, **k)
        ka.rope(kk, kk, self.Hkv, self.Dh, self.freqs, pos=self.pos, **k)
        if self.cached:
            with torch.cuda.stream(stream):
                self.cache[self.place] = self.qkv[:, D:]
        kk, vv = self.keys()
        kw = dict(k_start=self.k_start, k_len=self.k_len) if self.cached else {}
        ka.prompt_attn(self.at, q, kk, vv, self.H, self.Hkv, q_start=self.q_start, prefix=self.prefix, workspace=self.ws if ws == "own" else ws, **kw, **k)
        after("attended")
        ka.mxfp8_quantize(self.at, self.c, self.s, **k)
        ka.linear_mxfp8(self.o, self.c, self.s, self.Wo, epi=ka.KILN_EPI_F16, **k)
        after("out")
        ka.add_rmsnorm(self.c, self.o, r, self.n2, scales=self.s, **k)
        ka.linear_mxfp8(self.up, self.c, self.s, self.Wup, epi=ka.KILN_EPI_GELU16, **k)
        after("up")
        ka.mxfp8_quantize(self.up, self.cm, self.sm, **k)
        ka.linear_mxfp8(r, self.cm, self.sm, self.Wdown, epi=ka.KILN_EPI_RESID, **k)
        return r


LAYERS = [([(120, 0), (33, 0), (1, 0), (77, 0)], 16, 8, 128, 1024, 0), ([(1, 700), (1, 0), (1, 3000), (1, 64)], 8, 2, 64, 256, 0),
          ([(20, 0), (5, 0), (64, 0)], 4, 4, 64, 512, 300), ([(1, 30)] * 9, 4, 2, 128, 96, 3000), ([(300, 500)], 4, 1, 128, 160, 50)]


def weight_values(W):
    """A prepared weight's values, from the product with unit rows (exact: one term each)."""
    rows, cols = W.shape
    eye = torch.eye(cols, device=DEV)
    c, s = ka.mxfp8_quantize(eye)
    y = torch.empty(cols, rows, device=DEV)
    ka.linear_mxfp8(y, c, s, W)
    return y.t().double()


def values8(c, s):
    return c.view(torch.float8_e4m3fn).double() * torch.exp2(s.double() - 127).repeat_interleave(32, 1)


@pytest.mark.parametrize("args", LAYERS)
def test_stages(gpu, args):
    a = Layer(*args)
    x, r = a.inputs(1)
    r0, seen = r.clone(), {}
    names = ("c", "s", "qkv", "at", "o", "up", "cache")
    a.run(x, r, after=lambda n: seen.update({n: {k: getattr(a, k).clone() for k in names} | {"r": r.clone()}}))
    u = 2.0 ** -11

    def product(c, s, W):
        xv, wv = values8(c, s), weight_values(W)
        mag = xv.abs() @ wv.abs().t()
        block = xv.abs().view(xv.shape[0], -1, 32).amax(-1) @ wv.abs().view(wv.shape[0], -1, 32).amax(-1).t()
        return xv @ wv.t(), xv.shape[1] * 2.0 ** -24 * mag, 7 * 2.0 ** -13 * mag, 4 * 7 * 2.0 ** -13 * 4 / 224 * block

    def close(got, ref, tol, what):
        worst = ((got.double() - ref).abs() / tol).max().item()
        print(f"[text layer] {what}: worst error / tolerance {worst:.3f}", flush=True)
        assert worst <= 1, what

    def half(ref, tol):
        return tol + u * (ref.abs() + tol) + 2.0 ** -25

    def norm(xx, rr, w, c, s, after, what):
        h = xx.double() + rr.double()
        close(after, h, 2.0 ** -24 * h.abs() + 1e-30, what + " sum")
        y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-6) * w.double()
        sc = torch.exp2(s.double() - 127).repeat_interleave(32, 1)
        step = torch.exp2(torch.floor(torch.log2((y.abs() / sc).clamp(min=2.0 ** -6))) - 3) * sc
        close(values8(c, s), y, step / 2 * (1 + 1e-6) + 2.0 ** -17 * y.abs(), what)

    n = seen["norm"]
    norm(x, r0, a.n1, n["c"], n["s"], n["r"], "first norm")
    ref, t32, t16, _ = product(n["c"], n["s"], a.Wqkv)
    close(seen["projected"]["qkv"], ref, half(ref, t32 + t16), "projection")
    e = seen["attended"]
    kv = e["cache"] if a.cached else e["qkv"][:, a.D:]
    seqs = [(q0, nq, s * a.cap if a.cached else q0, nq + nc) for s, (q0, (nq, nc)) in enumerate(zip(a.starts, a.lens))]
    check_attention(e["at"], e["qkv"][:, :a.D], kv[:, :a.KV], kv[:, a.KV:], a.H, a.Hkv, seqs, a.prefix, what=f"layer of {len(a.lens)} sequences")
    o = seen["out"]
    ref, t32, t16, _ = product(o["c"], o["s"], a.Wo)
    close(o["o"], ref, half(ref, t32 + t16), "output projection")
    m = seen["up"]
    norm(o["o"], o["r"], a.n2, m["c"], m["s"], m["r"], "second norm")
    ref, t32, t16, _ = product(m["c"], m["s"], a.Wup)
    g = ref * torch.special.ndtr(ref)
    close(m["up"], g, half(g, 1.13 * (t32 + t16) + 2.0 ** -17 * ref.abs()), "MLP up")
    ref, t32, _, part = product(a.cm, a.sm, a.Wdown)
    close(r, m["r"].double() + ref, t32 + part + 2.0 ** -23 * ((m["r"].double() + ref).abs() + ref.abs()) + 1e-30, "MLP down")


@pytest.mark.parametrize("args", LAYERS)
def test_captured(gpu, args):
    """One capture, replayed on new inputs with eager runs and synchronizations between: every replay equals the eager result."""
    a = Layer(*args)
    x, r = a.inputs(0)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        a.run(x, r.clone())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.run(x, r)
    for seed in range(4):
        nx, nr = a.inputs(seed)
        eager = a.run(nx, nr.clone())
        x.copy_(nx)
        r.copy_(nr)
        if seed % 2:
            torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(r, eager), f"replay {seed}"


def test_two_graphs_share_a_workspace(gpu):
    """Graphs that share a workspace and are replayed in order on one stream."""
    layers = [Layer(*LAYERS[1], seed=1), Layer(*LAYERS[3], seed=2)]
    ws = torch.empty(max(a.ws.numel() for a in layers), dtype=torch.uint8, device=DEV)
    ins, graphs, want = [a.inputs(5 + i) for i, a in enumerate(layers)], [], []
    for a, (x, r) in zip(layers, ins):
        want.append(a.run(x, r.clone()))
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            a.run(x, r, ws=ws)
        graphs.append(g)
    first = [r.clone() for _, r in ins]
    for _ in range(3):
        for (_, r), f in zip(ins, first):
            r.copy_(f)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for (_, r), w in zip(ins, want):
            assert torch.equal(r, w)


def test_streams_at_once(gpu):
    """Two layers at once on two streams, each call taking its scratch from its own stream (no workspace given)."""
    layers = [Layer(*LAYERS[3], seed=i) for i in range(2)]
    ins = [a.inputs(7 + i) for i, a in enumerate(layers)]
    want = [a.run(x, r.clone()) for a, (x, r) in zip(layers, ins)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in layers]
    for turn in range(8):
        got = []
        for a, (x, r), st in zip(layers, ins, streams):
            with torch.cuda.stream(st):
                y = r.clone()
            got.append(a.run(x, y, ws=None, stream=st))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert torch.equal(g, w), f"turn {turn}"


def test_profiled(gpu):
    a = Layer(*LAYERS[2])
    x, r = a.inputs(3)
    ka.prof_enable(True)
    a.run(x, r)
    cats, _ = ka.prof_report()
    ka.prof_enable(False)
    assert {k: v[1] for k, v in cats.items()} == {"norm": 2, "gemm_mxfp8": 4, "rope": 2, "attention": 1, "mxfp8": 2}


def test_cpp_mirror(gpu):
    exe, src = (os.path.join(HERE, "cpp", "text_layer_test" + x) for x in ("", ".cpp"))
    if not os.path.exists(exe) or os.path.getmtime(exe) < os.path.getmtime(src):
        subprocess.run(["bash", os.path.join(HERE, "cpp", "build.sh")], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=100)
    print(r.stdout, r.stderr, flush=True)
    assert r.returncode == 0, r.stdout + r.stderr
