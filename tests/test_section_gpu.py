"""The attention section over an encoder's states as it is used: MXFP4 projections, rotary positions on queries and keys,
cross-attention with lengths, the gated MXFP4 output projection; eagerly, on other streams, captured and replayed, through the
profiler's categories and through the C++ mirror."""
import os
import subprocess

import numpy as np
import pytest
import torch

import kiln_amd as ka
from tests import mxfp4_ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HERE = os.path.dirname(os.path.abspath(__file__))


class Section:
    """One block's section: T target tokens of B items against S states of the encoder, D = H * 64."""

    def __init__(self, B, T, S, H, Hkv, text, seed=0):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.B, self.T, self.S, self.H, self.Hkv, self.text, self.D, self.KV = B, T, S, H, Hkv, text, H * 64, Hkv * 64
        w = lambda r, c: (torch.randn(r, c, device=DEV, generator=g) / c ** 0.5).bfloat16()  # noqa: E731
        self.wq, self.wkv, self.wo = w(self.D, self.D), w(2 * self.KV, text), w(self.D, self.D)
        self.Wq, self.Wkv, self.Wo = (ka.linear_mxfp4_weight(t) for t in (self.wq, self.wkv, self.wo))
        self.freqs, self.m = ka.rope_freqs(64, 1e4, "ramp", 2.0, 256, device=DEV)
        self.pos_q = (torch.arange(B * T, device=DEV) % T).to(torch.int32) + 100
        self.pos_k = (torch.arange(B * S, device=DEV) % S).to(torch.int32)
        self.gate = torch.randn(self.D, device=DEV, generator=g)
        self.q = torch.empty(B * T, self.D, device=DEV, dtype=torch.float16)
        self.kv = torch.empty(B * S, 2 * self.KV, device=DEV, dtype=torch.float16)
        self.at = torch.empty_like(self.q)
        n = max(ka.linear_mxfp4_workspace_bytes(B * T, self.D, self.D), ka.linear_mxfp4_workspace_bytes(B * S, 2 * self.KV, text),
                ka.cross_attn_workspace_bytes(B, T, S, H, Hkv, 64), 16)
        self.ws = torch.empty(n, dtype=torch.uint8, device=DEV)

    def inputs(self, seed):
        g = torch.Generator(device=DEV).manual_seed(1000 + seed)
        x = torch.randn(self.B * self.T, self.D, device=DEV, generator=g).half()
        e = torch.randn(self.B * self.S, self.text, device=DEV, generator=g).half()
        y = torch.randn(self.B * self.T, self.D, device=DEV, generator=g)
        klen = torch.randint(1, self.S + 1, (self.B,), device=DEV, generator=g, dtype=torch.int32)
        return x, e, y, klen

    def run(self, x, e, y, klen, ws="own", stream=None, after=lambda name: None):
        """y += gate * Wo attention(rope(Wq x), rope(Wk e), Wv e), in place on y."""
        k = dict(workspace=self.ws if ws == "own" else ws, stream=stream)
        ka.linear_mxfp4(self.q, x, self.Wq, epi=ka.KILN_EPI_F16, **k)
        ka.linear_mxfp4(self.kv, e, self.Wkv, epi=ka.KILN_EPI_F16, **k)
        after("projected")
        keys = self.kv[:, :self.KV]
        ka.rope(self.q, self.q, self.H, 64, self.freqs, pos=self.pos_q, mscale=self.m, stream=stream)
        ka.rope(keys, keys, self.Hkv, 64, self.freqs, pos=self.pos_k, mscale=self.m, stream=stream)
        after("turned")
        kv3 = self.kv.view(self.B, self.S, -1)
        ka.cross_attn(self.at.view(self.B, self.T, -1), self.q.view(self.B, self.T, -1), kv3[..., :self.KV], kv3[..., self.KV:], self.H,
                      self.Hkv, klen=klen, **k)
        after("attended")
        ka.linear_mxfp4(y, self.at, self.Wo, epi=ka.KILN_EPI_RESID, gate=self.gate, **k)
        return y


SIZES = [(1, 512, 120, 16, 16, 1024), (2, 1, 300, 8, 2, 256), (3, 77, 45, 4, 4, 96), (2, 130, 2100, 4, 1, 128)]


def mx(t):
    return torch.from_numpy(mxfp4_ref.values(*mxfp4_ref.quantize(t))).to(DEV)


@pytest.mark.parametrize("size", SIZES)
def test_stages(gpu, size):
    """Every stage against 64 bits from the stage before it, as it was computed."""
    s = Section(*size)
    x, e, y, klen = s.inputs(1)
    y0, seen = y.clone(), {}
    s.run(x, e, y, klen, after=lambda name: seen.update({name: (s.q.clone(), s.kv.clone(), s.at.clone())}))
    u, tiny = 2.0 ** -11, 2.0 ** -25

    def close(got, ref, tol, what):
        tol = tol + (u * (ref.abs() + tol) + tiny if got.dtype == torch.float16 else 2.0 ** -24 * ref.abs())
        worst = ((got.double() - ref).abs() / tol).max().item()
        print(f"[section] {size} {what}: worst error / tolerance {worst:.3f}", flush=True)
        assert worst <= 1

    def product(xin, w):  # K / 128 instructions and up to eight joins round by 2^-23 of the magnitudes
        a, b = mx(xin), mx(w)
        return a @ b.t(), (-(-xin.shape[1] // 128) + 8) * 2.0 ** -23 * (a.abs() @ b.abs().t())

    q, kv, _ = seen["projected"]
    close(q, *product(x, s.wq), "queries")
    close(kv, *product(e, s.wkv), "keys and values")
    tq, tkv, _ = seen["turned"]
    for before, after, H, pos in ((q, tq, s.H, s.pos_q), (kv[:, :s.KV], tkv[:, :s.KV], s.Hkv, s.pos_k)):
        a = pos.double()[:, None] * s.freqs
        c, sn = s.m * torch.cos(a)[:, None], s.m * torch.sin(a)[:, None]
        h = before.double().reshape(-1, H, 2, 32)
        p, r = h[:, :, 0], h[:, :, 1]
        mag = 9 * 2.0 ** -24 * s.m * (p.abs() + r.abs())
        close(after, torch.cat([p * c - r * sn, r * c + p * sn], -1).reshape(before.shape), torch.cat([mag, mag], -1).reshape(before.shape), "positions")
    assert torch.equal(kv[:, s.KV:], tkv[:, s.KV:])
    at = seen["attended"][2]
    G = s.H // s.Hkv
    for b in range(s.B):
        n = int(klen[b])
        rows = slice(b * s.S, b * s.S + n)
        for h in range(s.H):
            qq = tq[b * s.T:(b + 1) * s.T, h * 64:(h + 1) * 64].double()
            kk, vv = (tkv[rows, o + h // G * 64:o + (h // G + 1) * 64].double() for o in (0, s.KV))
            sc = qq @ kk.t() / 8
            p = torch.softmax(sc, -1)
            smag = ((qq.abs() @ kk.abs().t()).amax(-1) / 8 + sc.amax(-1) - sc.amin(-1))[:, None]
            tol = (u + 4 * 2.0 ** -22 * smag + (n / 4 + 64) * 2.0 ** -24 + 2.0 ** -21) * (p @ vv.abs()) + 2.0 ** -25 * vv.abs().sum(0)
            close(at[b * s.T:(b + 1) * s.T, h * 64:(h + 1) * 64], p @ vv, tol, f"attention {b} {h}")
    acc, tol = product(at, s.wo)
    g = s.gate.double()
    close(y, y0.double() + g * acc, tol * g.abs() + 2.0 ** -23 * (g * acc).abs(), "output")


@pytest.mark.parametrize("size", SIZES)
def test_captured(gpu, size):
    """One capture, replayed on new inputs with eager runs and synchronizations between: every replay equals the eager result."""
    s = Section(*size)
    x, e, y, klen = s.inputs(0)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        s.run(x, e, y.clone(), klen)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.run(x, e, y, klen)
    for seed in range(4):
        new = s.inputs(seed)
        eager = s.run(new[0], new[1], new[2].clone(), new[3])
        for dst, src in zip((x, e, y, klen), new):
            dst.copy_(src)
        if seed % 2:
            torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, eager), f"replay {seed}"


def test_two_graphs_share_a_workspace(gpu):
    """Graphs that share a workspace and are replayed in order on one stream."""
    a, b = Section(1, 150, 1100, 4, 4, 128, 1), Section(2, 200, 130, 4, 2, 96, 2)
    ws = torch.empty(max(a.ws.numel(), b.ws.numel()), dtype=torch.uint8, device=DEV)
    ins, graphs, want = [a.inputs(5), b.inputs(6)], [], []
    for s, i in zip((a, b), ins):
        want.append(s.run(i[0], i[1], i[2].clone(), i[3]))
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s.run(*i, ws=ws)
        graphs.append(g)
    y0 = [i[2].clone() for i in ins]
    for _ in range(3):
        for i, y in zip(ins, y0):
            i[2].copy_(y)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for i, y in zip(ins, want):
            assert torch.equal(i[2], y)


def test_streams_at_once(gpu):
    """Two sections at once on two streams, each call taking its scratch from its own stream (no workspace given)."""
    secs = [Section(2, 300, 900, 4, 4, 256, i) for i in range(2)]
    ins = [s.inputs(7 + i) for i, s in enumerate(secs)]
    want = [s.run(i[0], i[1], i[2].clone(), i[3]) for s, i in zip(secs, ins)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in secs]
    for turn in range(10):
        ys = [i[2].clone() for i in ins]
        torch.cuda.synchronize()
        for _ in range(3):
            got = []
            for s, i, y, st in zip(secs, ins, ys, streams):
                with torch.cuda.stream(st):
                    y.copy_(i[2])
                got.append(s.run(i[0], i[1], y, i[3], ws=None, stream=st))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert torch.equal(g, w), f"turn {turn}"


def test_profiled(gpu):
    s = Section(1, 100, 60, 4, 4, 96)
    x, e, y, klen = s.inputs(3)
    ka.prof_enable(True)
    s.run(x, e, y, klen)
    ka.mxfp4_quantize(x)
    cats, _ = ka.prof_report()
    ka.prof_enable(False)
    assert {k: v[1] for k, v in cats.items()} == {"gemm_mxfp4": 3, "rope": 2, "attention": 1, "mxfp4": 1}


def test_cpp_mirror(gpu):
    exe, src = (os.path.join(HERE, "cpp", "encoder_section_test" + x) for x in ("", ".cpp"))
    if not os.path.exists(exe) or os.path.getmtime(exe) < os.path.getmtime(src):
        subprocess.run(["bash", os.path.join(HERE, "cpp", "build.sh")], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=100)
    print(r.stdout, r.stderr, flush=True)
    assert r.returncode == 0, r.stdout + r.stderr


def test_numpy_oracle_agrees_with_torch(gpu):
    """The oracle's quantiser against a second statement of it: distances to the grid."""
    x = torch.randn(8, 64, dtype=torch.float64)
    c, s = mxfp4_ref.quantize(x)
    v = mxfp4_ref.values(c, s)
    sc = np.repeat(np.exp2(s.astype(np.float64) - 127), 32, axis=1)
    grid = np.concatenate([mxfp4_ref.GRID, -mxfp4_ref.GRID])
    nearest = np.abs(x.numpy()[..., None] / sc[..., None] - grid).min(-1)
    np.testing.assert_allclose(np.abs(x.numpy() - v) / sc, nearest, rtol=0, atol=1e-12)
