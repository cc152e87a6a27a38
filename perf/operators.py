"""The attention section over an encoder's states, as timed cases: rotary positions, cross-attention to the encoder's keys and
values, and linear layers whose weights and activations are held in microscaled 4-bit floating point (MXFP4).

Kinds of case:

  rope    rotary positions of a projection's heads, angles from positions and frequencies: half and interleaved pairs, all of
          a head or its first dimensions, frequencies scaled for long contexts
  cross   attention of B x Tq queries to Tk states of another length: shared key heads, a length or a key mask per item
  quant   a matrix to MXFP4 (32 values share a power-of-two scale) and back to the values it stands for
  linear  a linear layer with an MXFP4 weight: the rows of x quantised, the product, the epilogue

Widths are the engine's: D = 2048 (16 heads of 128), MLP 8192, text 1024 (16 heads of 64), pictures of 64 x 64 and 48 x 72 tokens,
text contexts of 77 to 512 tokens. Drawn cases spread the sizes over their whole ranges, on a log scale.
"""
import math

import numpy as np
import torch

own = False
DEV = "cuda"
DT = dict(f32=torch.float32, f16=torch.float16, bf16=torch.bfloat16)
BYTES = dict(f32=4, f16=2, bf16=2)


def listed():
    return [
        # one new token of each of four streams: queries and four key heads of a stacked projection, latency
        dict(name="rope 4 tokens", kind="rope", T=4, H=20, Dh=128, rot=128, inter=False, dt="f16", scaling="none", factor=1.0, far=30000),
        # a prompt's tokens, interleaved pairs, the first 32 of 80 dimensions turn, several prompts packed
        dict(name="rope 1000 partial", kind="rope", T=1000, H=32, Dh=80, rot=32, inter=True, dt="bf16", scaling="linear", factor=4.0, far=8000),
        # a long text at once, positions past the trained length
        dict(name="rope 32768 long", kind="rope", T=32768, H=20, Dh=128, rot=128, inter=False, dt="f16", scaling="ramp", factor=16.0, far=131072),
        # the text adapter's block: 512 target tokens against the encoder's states of an ordinary prompt
        dict(name="cross adapter", kind="cross", B=1, Tq=512, Tk=120, Hq=16, Hkv=16, Dh=64, dt="f16", lens="full"),
        # a CFG pair of 1024x1024 pictures against contexts of different lengths in one buffer
        dict(name="cross picture", kind="cross", B=2, Tq=4096, Tk=512, Hq=16, Hkv=16, Dh=128, dt="f16", lens="ragged"),
        # heads of 64 over 77 text states, some masked
        dict(name="cross 77 masked", kind="cross", B=2, Tq=4096, Tk=77, Hq=10, Hkv=10, Dh=64, dt="bf16", lens="mask"),
        # one query token per stream against long states, four query heads to a key head
        dict(name="cross one token", kind="cross", B=8, Tq=1, Tk=8192, Hq=16, Hkv=4, Dh=128, dt="bf16", lens="ragged"),
        # a text context's rows: few and odd in number
        dict(name="quant 77x1024", kind="quant", rows=77, cols=1024, dt="f32"),
        # a weight at load
        dict(name="quant 8192x2048", kind="quant", rows=8192, cols=2048, dt="bf16"),
        # a single row through the MLP's first layer: the weight's bytes
        dict(name="linear 1 row gelu", kind="linear", T=1, N=8192, K=2048, dt="f16", epi="gelu"),
        # a projection of a middle-sized picture's tokens and one more
        dict(name="linear 1537", kind="linear", T=1537, N=2048, K=2048, dt="bf16", epi="f32"),
        # the MLP's first layer for a CFG pair of 768x1152 pictures
        dict(name="linear 6912 gelu", kind="linear", T=6912, N=8192, K=2048, dt="f16", epi="gelu"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "rope", "cross", "cross", "cross", "quant", "linear", "linear", "linear"])
    dt = rng.choice(["f16", "bf16"])
    if kind == "rope":
        Dh = rng.choice([64, 80, 96, 128, 256])
        H = rng.choice([1, 4, 8, 16, 20, 32])
        rot = rng.choice([Dh, Dh, Dh // 2, 2 * rng.randint(2, Dh // 2)])
        T = min(_log(rng, 1, 32768), 32768 * 2560 // (2 * H * Dh))
        return dict(kind=kind, T=T, H=H, Dh=Dh, rot=rot, inter=rng.choice([False, True]), dt=rng.choice(["f32", "f16", "bf16"]),
                    scaling=rng.choice(["none", "linear", "ntk", "ramp", "bands"]), factor=rng.choice([2.0, 4.0, 8.0, 16.0]),
                    far=_log(rng, 1000, 1000000))
    if kind == "cross":
        Dh = rng.choice([64, 128])
        Hq, Hkv = rng.choice([(16, 16), (16, 16), (10, 10), (20, 20), (16, 4), (16, 8), (32, 4), (12, 1)])
        B, lens = rng.randint(1, 8), rng.choice(["full", "ragged", "mask"])
        form = rng.choice(["token", "few", "picture", "picture", "long"])
        Tq = {"token": 1, "few": _log(rng, 2, 64), "picture": _log(rng, 64, 4096), "long": _log(rng, 64, 1024)}[form]
        Tk = _log(rng, 1, 512) if form == "picture" else _log(rng, 1, 8192)
        while B * Hq * Tq * Tk * Dh > 2 * 16 * 4096 * 512 * 128 or B * Hkv * Tk * Dh > 8 * 4 * 8192 * 128:
            B, Tk = max(1, B // 2), max(1, Tk * 2 // 3)
        return dict(kind=kind, B=B, Tq=Tq, Tk=Tk, Hq=Hq, Hkv=Hkv, Dh=Dh, dt=dt, lens=lens)
    if kind == "quant":
        cols = 32 * _log(rng, 1, 256)
        return dict(kind=kind, rows=min(_log(rng, 1, 8192), 8192 * 2048 // (2 * cols)), cols=cols, dt=rng.choice(["f32", "f16", "bf16"]))
    N, K = rng.choice([(2048, 2048), (8192, 2048), (2048, 8192), (2048, 1024), (1024, 1024), (32 * rng.randint(1, 64) + 1, 32 * rng.randint(1, 64))])
    T = min(rng.choice([rng.randint(1, 64), _log(rng, 1, 6912)]), 6912 * 8192 * 2048 // (N * K))
    return dict(kind=kind, T=T, N=N, K=K, dt=rng.choice(["f32", "f16", "bf16"]), epi=rng.choice(["f32", "f16", "gelu"]))


# ---- inputs, from the seed alone ----

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed((seed * 1000003 + 12345) % (1 << 62))


def _inputs(case, seed):
    g, k = _gen(seed), case["kind"]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    if k == "rope":
        # sequences packed one after the other: positions count up from several starts
        T, far = case["T"], case["far"]
        t = torch.arange(T, device=DEV)
        starts = torch.randint(0, far, (4,), generator=g, device=DEV)
        pos = (starts[(4 * t // T)] + t) % far
        return dict(x=randn(T, case["H"] * case["Dh"]).to(DT[case["dt"]]), pos=pos.to(torch.int32))
    if k == "cross":
        B, Tq, Tk, Dh, dt = case["B"], case["Tq"], case["Tk"], case["Dh"], DT[case["dt"]]
        # queries and keys after their norm: unit variance, and a few directions that the heads share, so that some keys win
        q, kk, v = randn(B, Tq, case["Hq"] * Dh), randn(B, Tk, case["Hkv"] * Dh), randn(B, Tk, case["Hkv"] * Dh)
        kk = kk * (1 + randn(B, Tk, 1).abs() / 2)
        r = dict(q=q.to(dt), k=kk.to(dt), v=v.to(dt), klen=None, kmask=None)
        if case["lens"] == "ragged":
            klen = (Tk * torch.rand(B, generator=g, device=DEV).sqrt()).to(torch.int32) + 1
            klen[0] = Tk
            r["klen"] = klen.clamp(max=Tk)
        elif case["lens"] == "mask":
            keep = torch.rand(B, Tk, generator=g, device=DEV) < 0.8
            keep[:, 0] = True
            r["kmask"] = keep
        return r
    if k == "quant":
        # a weight's or an activation's spread: columns of different size
        return dict(x=(randn(case["rows"], case["cols"]) * torch.exp(randn(case["cols"]))).to(DT[case["dt"]]))
    w = (torch.rand(case["N"], case["K"], generator=g, device=DEV) * 2 - 1) / case["K"] ** 0.5
    return dict(x=randn(case["T"], case["K"]).to(DT[case["dt"]]), w=w.to(torch.bfloat16))


THETA, TRAINED = 10000.0, 8192  # the base of the frequencies, and the length that a scaled model was trained at


def _freqs(case):
    """Frequencies (radians per position, 64 bits) and the factor on the rotated values."""
    rot, s, kind = case["rot"], case["factor"], case["scaling"]
    i = np.arange(rot // 2, dtype=np.float64)
    theta = THETA * s ** (rot / (rot - 2)) if kind == "ntk" else THETA
    f = theta ** (-2.0 * i / rot)
    if kind == "linear":
        return f / s, 1.0
    if kind == "ramp":
        lo, hi = (rot * math.log(TRAINED / (2 * math.pi * turns)) / (2 * math.log(THETA)) for turns in (32.0, 1.0))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), rot - 1)
        slow = np.clip((i - lo) / max(hi - lo, 0.001), 0, 1)
        return f / s * slow + f * (1 - slow), 0.1 * math.log(s) + 1
    if kind == "bands":
        turns = TRAINED * f / (2 * math.pi)
        keep = np.clip((turns - 1) / (4 - 1), 0, 1)
        return f / s * (1 - keep) + f * keep, 1.0
    return f, 1.0


def _plain_fp4(x):
    """The MXFP4 values of x [rows, cols]: 32 neighbours share the scale 2^(floor(log2 of their largest) - 2); each is rounded to
    the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 times it (ties to the even code), larger ones to 6."""
    b = x.float().view(x.shape[0], -1, 32)
    _, e = torch.frexp(b.abs().amax(-1, keepdim=True))
    scale = torch.ldexp(torch.ones_like(b[..., :1]), (e - 3).clamp(min=-120))
    a = (b / scale).abs().clamp(max=6)
    # the grid's step is 0.5 below 2, 1 below 4 and 2 above; torch.round takes ties to the even multiple, as the codes do
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return (torch.sign(b) * torch.round(a / step) * step * scale).view(x.shape)


def prepare(case, seed):
    s, k = dict(_inputs(case, seed), case=case), case["kind"]
    if own:
        import kiln_amd
    if k == "rope":
        if own:
            s["freqs"], s["mscale"] = kiln_amd.rope_freqs(case["rot"], THETA, case["scaling"], case["factor"], TRAINED, device=DEV)
        else:
            f, s["mscale"] = _freqs(case)
            s["freqs"] = torch.from_numpy(f).to(DEV)
        s["y"] = torch.empty_like(s["x"])
    elif k == "cross":
        s["out"] = torch.empty_like(s["q"])
        if own:
            n = kiln_amd.cross_attn_workspace_bytes(case["B"], case["Tq"], case["Tk"], case["Hq"], case["Hkv"], case["Dh"])
            s["ws"] = torch.empty(n, dtype=torch.uint8, device=DEV)
    elif k == "quant":
        if own:
            s["codes"] = torch.empty(case["rows"], case["cols"] // 2, dtype=torch.uint8, device=DEV)
            s["scales"] = torch.empty(case["rows"], case["cols"] // 32, dtype=torch.uint8, device=DEV)
        s["y"] = torch.empty_like(s["x"])
    else:
        s["y"] = torch.empty(case["T"], case["N"], dtype=torch.float32 if case["epi"] == "f32" else torch.float16, device=DEV)
        w = s.pop("w")
        if own:
            s["w"] = kiln_amd.linear_mxfp4_weight(w)
            s["ws"] = torch.empty(kiln_amd.linear_mxfp4_workspace_bytes(case["T"], case["N"], case["K"]), dtype=torch.uint8, device=DEV)
        else:
            s["w"] = _plain_fp4(w)
    return s


def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    import kiln_amd
    case = s["case"]
    k = case["kind"]
    if k == "rope":
        return kiln_amd.rope(s["y"], s["x"], case["H"], case["Dh"], s["freqs"], pos=s["pos"], interleaved=case["inter"], mscale=s["mscale"])
    if k == "cross":
        return kiln_amd.cross_attn(s["out"], s["q"], s["k"], s["v"], case["Hq"], case["Hkv"], klen=s["klen"], kmask=s["kmask"],
                                   workspace=s["ws"])
    if k == "quant":
        kiln_amd.mxfp4_quantize(s["x"], s["codes"], s["scales"])
        return kiln_amd.mxfp4_dequantize(s["y"], s["codes"], s["scales"])
    epi = dict(f32=kiln_amd.KILN_EPI_F32, f16=kiln_amd.KILN_EPI_F16, gelu=kiln_amd.KILN_EPI_GELU16)[case["epi"]]
    return kiln_amd.linear_mxfp4(s["y"], s["x"], s["w"], epi=epi, workspace=s["ws"])


def _plain(s):
    case = s["case"]
    k = case["kind"]
    if k == "rope":
        T, H, Dh, rot = case["T"], case["H"], case["Dh"], case["rot"]
        a = s["pos"].double()[:, None] * s["freqs"]
        c, sn = (torch.cos(a) * s["mscale"]).float()[:, None], (torch.sin(a) * s["mscale"]).float()[:, None]
        x = s["x"].view(T, H, Dh)
        y = s["y"].view(T, H, Dh)
        if case["inter"]:
            x0, x1, i0, i1 = x[..., 0:rot:2].float(), x[..., 1:rot:2].float(), slice(0, rot, 2), slice(1, rot, 2)
        else:
            x0, x1, i0, i1 = x[..., :rot // 2].float(), x[..., rot // 2:rot].float(), slice(0, rot // 2), slice(rot // 2, rot)
        y[..., i0] = (x0 * c - x1 * sn).to(y.dtype)
        y[..., i1] = (x1 * c + x0 * sn).to(y.dtype)
        y[..., rot:] = x[..., rot:]
        return s["y"]
    if k == "cross":
        B, Tq, Tk, Hq, Hkv, Dh = (case[n] for n in ("B", "Tq", "Tk", "Hq", "Hkv", "Dh"))
        # the query heads of a key head are rows of one product
        q = s["q"].float().view(B, Tq, Hkv, Hq // Hkv, Dh).permute(0, 2, 3, 1, 4).reshape(B * Hkv, Hq // Hkv * Tq, Dh)
        kt = s["k"].float().view(B, Tk, Hkv, Dh).permute(0, 2, 3, 1).reshape(B * Hkv, Dh, Tk)
        v = s["v"].float().view(B, Tk, Hkv, Dh).permute(0, 2, 1, 3).reshape(B * Hkv, Tk, Dh)
        p = torch.matmul(q, kt) * Dh ** -0.5
        keep = s["kmask"]
        if s["klen"] is not None:
            keep = torch.arange(Tk, device=DEV) < s["klen"][:, None]
        if keep is not None:
            p = p.view(B, Hkv, -1, Tk).masked_fill(~keep[:, None, None], -math.inf).view(B * Hkv, -1, Tk)
        p = torch.exp(p - p.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        o = torch.matmul(p, v).view(B, Hkv, Hq // Hkv, Tq, Dh).permute(0, 3, 1, 2, 4)
        s["out"].copy_(o.reshape(B, Tq, Hq * Dh))
        return s["out"]
    if k == "quant":
        s["y"].copy_(_plain_fp4(s["x"]))
        return s["y"]
    acc = torch.matmul(_plain_fp4(s["x"]), s["w"].t())
    if case["epi"] == "gelu":
        acc = acc * 0.5 * (1 + torch.erf(acc * 0.5 ** 0.5))
    s["y"].copy_(acc)
    return s["y"]


# ---- the definitions in 64 bits ----

_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _exact_fp4(x):
    """MXFP4 values by comparison with the borders between neighbours of the grid; a value on a border goes to the even code."""
    b = x.double().reshape(x.shape[0], -1, 32)
    top = b.abs().amax(-1, keepdim=True)
    scale = torch.where(top > 0, torch.exp2(torch.floor(torch.log2(torch.where(top > 0, top, 1.0))) - 2), 1.0)
    scale = torch.where(top < 4 * scale, scale / 2, torch.where(top >= 8 * scale, scale * 2, scale))  # log2's own rounding
    a = b.abs() / scale
    r = torch.zeros_like(a)
    for i in range(7):
        border = (_GRID[i] + _GRID[i + 1]) / 2
        up = a >= border if i % 2 else a > border
        r = torch.where(up, _GRID[i + 1], r)
    return (torch.where(b < 0, -r, r) * scale).reshape(x.shape)


def exact(case, seed):
    s, k = _inputs(case, seed), case["kind"]
    if k == "rope":
        T, H, Dh, rot = case["T"], case["H"], case["Dh"], case["rot"]
        f, m = _freqs(case)
        turn = torch.polar(torch.full((T, rot // 2), m, dtype=torch.float64, device=DEV), s["pos"].double()[:, None] * torch.from_numpy(f).to(DEV))
        x = s["x"].double().view(T, H, Dh)
        pairs = x[..., :rot].reshape(T, H, rot // 2, 2) if case["inter"] else x[..., :rot].reshape(T, H, 2, rot // 2).transpose(2, 3)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn[:, None])
        z = z.reshape(T, H, rot) if case["inter"] else z.transpose(2, 3).reshape(T, H, rot)
        return torch.cat([z, x[..., rot:]], -1).view(T, H * Dh)
    if k == "cross":
        B, Tq, Hq, Hkv, Dh = (case[n] for n in ("B", "Tq", "Hq", "Hkv", "Dh"))
        out = torch.zeros(B, Tq, Hq * Dh, dtype=torch.float64, device=DEV)
        for b in range(B):
            rows = torch.arange(case["Tk"], device=DEV)
            if s["klen"] is not None:
                rows = rows[:int(s["klen"][b])]
            elif s["kmask"] is not None:
                rows = rows[s["kmask"][b]]
            for h in range(Hq):
                kv = slice(h * Hkv // Hq * Dh, (h * Hkv // Hq + 1) * Dh)
                w = torch.softmax(s["q"][b, :, h * Dh:(h + 1) * Dh].double() @ s["k"][b, rows, kv].double().t() / math.sqrt(Dh), -1)
                out[b, :, h * Dh:(h + 1) * Dh] = w @ s["v"][b, rows, kv].double()
        return out
    if k == "quant":
        return _exact_fp4(s["x"])
    acc = _exact_fp4(s["x"]) @ _exact_fp4(s["w"]).t()
    return torch.special.ndtr(acc) * acc if case["epi"] == "gelu" else acc


# ---- the least a pass can do ----

def work(case):
    k = case["kind"]
    if k == "rope":
        T, n, e = case["T"], case["T"] * case["H"] * case["Dh"], BYTES[case["dt"]]
        return dict(bytes=2.0 * n * e + 4 * T + 4 * case["rot"], flops=3.0 * T * case["H"] * case["rot"])
    if k == "cross":
        B, Tq, Tk, Hq, Hkv, Dh = (case[n] for n in ("B", "Tq", "Tk", "Hq", "Hkv", "Dh"))
        # ragged lengths are the square root of a uniform number of the whole: two thirds, the first item all of it; a mask keeps 0.8
        keys = B * Tk * dict(full=1.0, mask=0.8, ragged=(1 + (B - 1) * 2 / 3) / B)[case["lens"]]
        return dict(bytes=2.0 * Dh * (2 * B * Tq * Hq + 2 * keys * Hkv), flops=4.0 * keys * Tq * Hq * Dh)
    if k == "quant":
        n = case["rows"] * case["cols"]
        # the matrix, its codes and scales, and the values they stand for
        return dict(bytes=n * (2.0 * BYTES[case["dt"]] + 2 * (0.5 + 1 / 32)), flops=3.0 * n)
    T, N, K = case["T"], case["N"], case["K"]
    return dict(bytes=1.0 * T * K * BYTES[case["dt"]] + N * K * (0.5 + 1 / 32) + T * N * (4 if case["epi"] == "f32" else 2), flops=2.0 * T * N * K)
