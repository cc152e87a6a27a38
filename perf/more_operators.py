"""A text encoder's layer, as timed cases: causal attention over packed prompts and over the caches of running ones, a long prefix
that a batch shares, the RMS norm with the residual's addition, and linear layers that take 8-bit rows (MXFP8) against 4-bit
weights (MXFP4).

Kinds of case:

  prompt  causal attention of B packed sequences of different lengths, key heads shared by query heads; with C > 0 each sequence
          has up to C cached keys ahead of its new rows (one new row each: single tokens); with P > 0 all of them also see the P
          keys of a prefix that they share
  norm    the sum of a layer's output and the residual stream, and its RMS norm in the stream's or a 16-bit type, or as MXFP8 (e4m3
          codes, 32 values share a power-of-two scale) and back to the values it stands for
  linear  a linear layer of MXFP8 rows with an MXFP4 weight, and its epilogue

Widths are the engine's: the text encoder's 16 query heads on 8 key heads of 128, the text adapter's 1024 (heads of 64), D = 2048, MLP
8192; prompts of 77 to 8192 tokens. Drawn cases spread the sizes over their whole ranges, on a log scale.
"""
import math
import random

import torch

own = False
DEV = "cuda"
DT = dict(f32=torch.float32, f16=torch.float16, bf16=torch.bfloat16)
BYTES = dict(f32=4, f16=2, bf16=2)


def listed():
    return [
        # the prompts and negative prompts of two pictures, as they come: latency
        dict(name="prompt 4x120", kind="prompt", B=4, L=120, C=0, P=0, ragged=True, mix=1, Hq=16, Hkv=8, Dh=128, dt="f16", pad=0),
        # a data set's captions, packed into one batch with a padded end
        dict(name="prompt pack of 24", kind="prompt", B=24, L=2000, C=0, P=0, ragged=True, mix=2, Hq=16, Hkv=8, Dh=128, dt="bf16", pad=37),
        # one long document
        dict(name="prompt 8192", kind="prompt", B=1, L=8192, C=0, P=0, ragged=False, mix=3, Hq=16, Hkv=8, Dh=128, dt="f16", pad=0),
        # a few new rows of each of three prompts whose beginnings are cached, heads of 64
        dict(name="prompt 3x100 after 4000", kind="prompt", B=3, L=100, C=4000, P=0, ragged=True, mix=4, Hq=32, Hkv=4, Dh=64, dt="bf16", pad=0),
        # one new token of each of 16 streams
        dict(name="prompt tokens after 8191", kind="prompt", B=16, L=1, C=8191, P=0, ragged=True, mix=5, Hq=16, Hkv=8, Dh=128, dt="f16", pad=0),
        # variations of a prompt behind the template that they share
        dict(name="prefix 8 prompts", kind="prompt", B=8, L=200, C=0, P=1000, ragged=True, mix=6, Hq=16, Hkv=8, Dh=128, dt="bf16", pad=0),
        # one new token of each of 32 streams behind a long prefix
        dict(name="prefix 32 tokens", kind="prompt", B=32, L=1, C=300, P=4096, ragged=True, mix=7, Hq=16, Hkv=8, Dh=128, dt="f16", pad=0),
        # a single row between two layers: latency
        dict(name="norm 1 row", kind="norm", rows=1, dim=2048, x="f16", res="f32", y="f16"),
        # the tokens of a CFG pair of 768x1152 pictures, to the 8 bits of the next linear layer
        dict(name="norm 6912 rows 8 bits", kind="norm", rows=6912, dim=2048, x="bf16", res="f32", y="bf16", bits8=True),
        # a single row through the MLP's first layer: the weight's bytes
        dict(name="linear 1 row gelu", kind="linear", T=1, N=8192, K=2048, epi="gelu"),
        # a projection of one prompt's tokens
        dict(name="linear 120 rows", kind="linear", T=120, N=2048, K=2048, epi="f32"),
        # the MLP's first layer for a CFG pair of 768x1152 pictures
        dict(name="linear 6912 gelu", kind="linear", T=6912, N=8192, K=2048, epi="gelu"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "prompt", "prefix", "prefix", "norm", "linear", "linear"])
    if kind in ("prompt", "prefix"):
        Dh = rng.choice([64, 128])
        Hq, Hkv = rng.choice([(16, 8), (16, 8), (16, 16), (32, 4), (16, 2), (12, 4), (7, 1)])
        form = rng.choice(["tokens", "chunk", "whole", "whole"])
        B = _log(rng, 1, 64)
        P = _log(rng, 1, 8192) if kind == "prefix" else 0
        L = 1 if form == "tokens" else _log(rng, 2, 300) if form == "chunk" else _log(rng, 2, 8192)
        C = 0 if form == "whole" else _log(rng, 1, 8191)
        case = dict(kind="prompt", B=B, L=L, C=C, P=P, ragged=rng.choice([True, True, False]), mix=rng.randrange(1 << 20), Hq=Hq, Hkv=Hkv, Dh=Dh,
                    dt=rng.choice(["f16", "bf16"]), pad=rng.choice([0, 0, rng.randint(1, 100)]))
        while work(case)["flops"] > 4.0 * 8192 * 8193 / 2 * 16 * 128 or case["B"] * (case["L"] + case["C"]) * Hkv * Dh > 16 * 8192 * 8 * 128:
            case["B"] = max(1, case["B"] // 2)
            if case["B"] == 1:
                case["L"], case["P"] = max(1, case["L"] * 2 // 3), case["P"] * 2 // 3
        return case
    if kind == "norm":
        dim = rng.choice([1024, 2048, 2048, 5120, 8192, 32 * _log(rng, 1, 256), 32 * _log(rng, 1, 256)])
        y = rng.choice(["f16", "bf16"])
        bits8 = rng.choice([True, False])
        if not bits8 and rng.random() < 0.3:
            dim += rng.randint(1, 31)
        return dict(kind="norm", rows=max(1, min(_log(rng, 1, 8192), 6912 * 2048 // dim)), dim=dim, x=rng.choice(["f16", "bf16", "f32"]),
                    res=rng.choice(["f32", "f32", "f16", "bf16", "none"]), y=y, bits8=bits8)
    N, K = rng.choice([(2048, 2048), (8192, 2048), (2048, 8192), (2048, 1024), (1024, 1024), (32 * rng.randint(1, 64) + 1, 32 * rng.randint(1, 64))])
    T = min(rng.choice([rng.randint(1, 64), _log(rng, 1, 6912)]), 6912 * 8192 * 2048 // (N * K))
    return dict(kind="linear", T=T, N=N, K=K, epi=rng.choice(["f32", "f16", "gelu"]))


def _lens(case):
    """(new rows, keys) of each sequence: the first is the longest, the others' lengths the square root of a uniform number of it."""
    rng = random.Random(case["mix"])
    lens = []
    for s in range(case["B"]):
        full = s == 0 or not case["ragged"]
        nq = case["L"] if full or case["L"] == 1 else int(case["L"] * rng.random() ** 0.5)
        lens.append((nq, nq + (case["C"] if full else int(case["C"] * rng.random() ** 0.5))))
    return lens


# ---- inputs, from the seed alone ----

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed((seed * 1000003 + 54321) % (1 << 62))


def _mx(x, bits):
    """x [rows, cols] to microscaled codes and scales: e4m3 (8) with the smallest scale that holds the block's largest magnitude, or
    E2M1 (4) with the scale 2^(floor(log2 largest) - 2)."""
    b = x.float().view(x.shape[0], -1, 32)
    m, e = torch.frexp(b.abs().amax(-1, keepdim=True))
    e = (e - 9 + (m > 0.875).int() if bits == 8 else e - 3).clamp(min=-120)
    a = torch.ldexp(b, -e)
    scales = (e + 127).to(torch.uint8).view(x.shape[0], -1)
    if bits == 8:
        return a.to(torch.float8_e4m3fn).view(torch.uint8).view(x.shape), scales
    a, grid = a.abs().clamp(max=6), torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=x.device)
    i = torch.bucketize(a, (grid[1:] + grid[:-1]) / 2)
    c = (i + 8 * (b < 0)).to(torch.uint8).view(x.shape)
    return c[:, ::2] | c[:, 1::2] << 4, scales


def _inputs(case, seed):
    g, k = _gen(seed), case["kind"]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    if k == "prompt":
        lens, dt = _lens(case), DT[case["dt"]]
        qs = [0]
        for nq, _ in lens:
            qs.append(qs[-1] + nq)
        # keys: a prompt's own rows, or the beginning of its place in a cache of equal places
        cap = case["L"] + case["C"]
        ks = qs[:-1] if not case["C"] else [s * cap for s in range(case["B"])]
        Tq = qs[-1] + case["pad"]
        Tk = Tq if not case["C"] else cap * case["B"]
        wq, wk = case["Hq"] * case["Dh"], case["Hkv"] * case["Dh"]

        def states(n, w):
            # after their norm: unit variance; keys of different size, so that some win
            return (randn(n, w) * (1 + randn(n, 1).abs() / 2)).to(dt)

        r = dict(q=randn(Tq, wq).to(dt), k=states(Tk, wk), v=randn(Tk, wk).to(dt), lens=lens, qs=qs, ks=ks, prefix=None)
        if case["P"]:
            r["prefix"] = (states(case["P"], wk), randn(case["P"], wk).to(dt))
        return r
    if k == "norm":
        # a residual stream's spread: channels of different size
        spread = torch.exp(randn(case["dim"]) / 2)
        r = dict(x=(randn(case["rows"], case["dim"]) * spread).to(DT[case["x"]]), res=None, w=(1 + randn(case["dim"]) / 4).to(torch.bfloat16))
        if case["res"] != "none":
            r["res"] = (2 * randn(case["rows"], case["dim"]) * spread).to(DT[case["res"]])
        return r
    x, w = randn(case["T"], case["K"]) * torch.exp(randn(case["K"]) / 2), (torch.rand(case["N"], case["K"], generator=g, device=DEV) * 2 - 1) / case["K"] ** 0.5
    return dict(x=_mx(x, 8), w=_mx(w, 4))


def prepare(case, seed):
    s, k = dict(_inputs(case, seed), case=case), case["kind"]
    if own:
        import kiln_amd
    if k == "prompt":
        s["out"] = torch.zeros_like(s["q"])
        if own:
            s["q_start"] = torch.tensor(s["qs"], dtype=torch.int32, device=DEV)
            s["k_start"] = s["k_len"] = None
            if case["C"]:
                s["k_start"] = torch.tensor(s["ks"], dtype=torch.int32, device=DEV)
                s["k_len"] = torch.tensor([nk for _, nk in s["lens"]], dtype=torch.int32, device=DEV)
            n = kiln_amd.prompt_attn_workspace_bytes(case["B"], s["q"].shape[0], s["k"].shape[0], case["P"], case["Hq"], case["Hkv"], case["Dh"])
            s["ws"] = torch.empty(n, dtype=torch.uint8, device=DEV)
    elif k == "norm":
        s["y"] = torch.empty(case["rows"], case["dim"], dtype=DT[case["y"]], device=DEV)
        s["h"] = torch.empty_like(s["res"]) if s["res"] is not None else None
        if own and case.get("bits8"):
            s["codes"] = torch.empty(case["rows"], case["dim"], dtype=torch.uint8, device=DEV)
            s["scales"] = torch.empty(case["rows"], case["dim"] // 32, dtype=torch.uint8, device=DEV)
    else:
        s["y"] = torch.empty(case["T"], case["N"], dtype=torch.float32 if case["epi"] == "f32" else torch.float16, device=DEV)
        s["w"] = kiln_amd.linear_mxfp4_weight(*s["w"]) if own else _values4(*s["w"])
    return s


def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    import kiln_amd
    case = s["case"]
    k = case["kind"]
    if k == "prompt":
        return kiln_amd.prompt_attn(s["out"], s["q"], s["k"], s["v"], case["Hq"], case["Hkv"], q_start=s["q_start"], k_start=s["k_start"],
                                    k_len=s["k_len"], prefix=s["prefix"], workspace=s["ws"])
    if k == "norm":
        if case.get("bits8"):
            kiln_amd.add_rmsnorm(s["codes"], s["x"], s["res"], s["w"], h=s["h"], scales=s["scales"])
            y = kiln_amd.mxfp8_dequantize(s["y"], s["codes"], s["scales"])
        else:
            y = kiln_amd.add_rmsnorm(s["y"], s["x"], s["res"], s["w"], h=s["h"])
        return (y, s["h"]) if s["h"] is not None else y
    epi = dict(f32=kiln_amd.KILN_EPI_F32, f16=kiln_amd.KILN_EPI_F16, gelu=kiln_amd.KILN_EPI_GELU16)[case["epi"]]
    return kiln_amd.linear_mxfp8(s["y"], *s["x"], s["w"], epi=epi)


# ---- plain forms ----

EPS = 1e-6


def _values4(codes, scales):
    """The values that MXFP4 codes and scales stand for."""
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    v = grid[torch.stack((codes & 15, codes >> 4), -1).int()].view(codes.shape[0], -1, 32)
    return torch.ldexp(v, scales.int()[..., None] - 127).view(codes.shape[0], -1)


def _values8(codes, scales):
    """The values that MXFP8 codes and scales stand for: e4m3, exponents from -6, three bits of mantissa."""
    c = codes.int()
    e, m = c >> 3 & 15, c & 7
    v = torch.ldexp((m + 8 * (e > 0).int()).float(), e.clamp(min=1) - 10)
    v = torch.where(c >= 128, -v, v).view(codes.shape[0], -1, 32)
    return torch.ldexp(v, scales.int()[..., None] - 127).view(codes.shape)


def _plain_fp8(y):
    """The MXFP8 values of y [rows, cols]: steps of an eighth of the value's power of two, of 2^-9 below 2^-6, times the block's scale."""
    b = y.view(y.shape[0], -1, 32)
    m, e = torch.frexp(b.abs().amax(-1, keepdim=True))
    e = (e - 9 + (m > 0.875).int()).clamp(min=-120)
    a = torch.ldexp(b, -e)
    _, ea = torch.frexp(a)
    step = (ea - 4).clamp(min=-9)
    return torch.ldexp(torch.round(torch.ldexp(a, -step)), step + e).view(y.shape)


def _plain(s):
    case = s["case"]
    k = case["kind"]
    if k == "prompt":
        Hq, Hkv, Dh, P = case["Hq"], case["Hkv"], case["Dh"], case["P"]
        G = Hq // Hkv
        for (nq, nk), q0, k0 in zip(s["lens"], s["qs"], s["ks"]):
            if not nq:
                continue
            # the query heads of a key head are rows of one product
            q = s["q"][q0:q0 + nq].float().view(nq, Hkv, G, Dh).permute(1, 2, 0, 3).reshape(Hkv, G * nq, Dh)
            kk, v = s["k"][k0:k0 + nk], s["v"][k0:k0 + nk]
            if P:
                kk, v = torch.cat((s["prefix"][0], kk)), torch.cat((s["prefix"][1], v))
            n = P + nk
            kt = kk.float().view(n, Hkv, Dh).permute(1, 2, 0).contiguous()
            v = v.float().view(n, Hkv, Dh).permute(1, 0, 2).contiguous()
            hidden = torch.arange(n, device=DEV) > torch.arange(n - nq, n, device=DEV)[:, None]
            o = torch.empty_like(q)
            step = max(1, (1 << 29) // (G * nq * n))  # heads at a time
            for h in range(0, Hkv, step):
                p = torch.matmul(q[h:h + step], kt[h:h + step]) * Dh ** -0.5
                p.view(-1, G, nq, n).masked_fill_(hidden, -math.inf)
                p = torch.exp(p - p.amax(-1, keepdim=True))
                p = p / p.sum(-1, keepdim=True)
                o[h:h + step] = torch.matmul(p, v[h:h + step])
            s["out"][q0:q0 + nq] = o.view(Hkv, G, nq, Dh).permute(2, 0, 1, 3).reshape(nq, Hq * Dh).to(s["out"].dtype)
        return s["out"]
    if k == "norm":
        h = s["x"].float()
        if s["res"] is not None:
            h = h + s["res"].float()
            s["h"].copy_(h)
        y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * s["w"].float()
        s["y"].copy_(_plain_fp8(y) if case.get("bits8") else y)
        return (s["y"], s["h"]) if s["h"] is not None else s["y"]
    acc = torch.matmul(_values8(*s["x"]), s["w"].t())
    if case["epi"] == "gelu":
        acc = acc * 0.5 * (1 + torch.erf(acc * 0.5 ** 0.5))
    s["y"].copy_(acc)
    return s["y"]


# ---- the definitions in 64 bits ----

def _exact_values8(codes, scales):
    return codes.view(torch.float8_e4m3fn).double() * torch.exp2(scales.double() - 127).repeat_interleave(32, 1)


def _exact_values4(codes, scales):
    c = torch.stack((codes & 15, codes >> 4), -1).view(codes.shape[0], -1).long()
    mag = torch.where(c % 8 < 2, (c % 8) / 2.0, (2.0 + c % 2) / 2 * torch.exp2((c % 8 // 2 - 1).double()))
    return torch.where(c > 7, -mag, mag) * torch.exp2(scales.double() - 127).repeat_interleave(32, 1)


def _exact_fp8(y):
    """MXFP8 values by comparison with the borders between neighbours of the grid; a value on a border goes to the even code."""
    b = y.reshape(y.shape[0], -1, 32)
    top = b.abs().amax(-1, keepdim=True)
    scale = torch.exp2(torch.floor(torch.log2(torch.where(top > 0, top, 1.0))) - 8)
    scale = torch.where(top > 448 * scale, 2 * scale, scale)
    scale = torch.where(top <= 224 * scale, scale / 2, scale)  # log2's own rounding
    grid = torch.arange(127, dtype=torch.uint8, device=y.device).view(torch.float8_e4m3fn).double()
    borders = (grid[1:] + grid[:-1]) / 2
    a = (b.abs() / scale).contiguous()
    i = torch.bucketize(a, borders)
    on = (i < 126) & (a == borders[i.clamp(max=125)]) & (i % 2 == 1)
    r = grid[i + on.long()]
    return (torch.where(b < 0, -r, r) * scale).reshape(y.shape)


def exact(case, seed):
    s, k = _inputs(case, seed), case["kind"]
    if k == "prompt":
        Dh, G = case["Dh"], case["Hq"] // case["Hkv"]
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        for (nq, nk), q0, k0 in zip(s["lens"], s["qs"], s["ks"]):
            for h in range(case["Hq"] if nq else 0):
                a, b = h * Dh, h // G * Dh
                kk, v = s["k"][k0:k0 + nk, b:b + Dh].double(), s["v"][k0:k0 + nk, b:b + Dh].double()
                w = s["q"][q0:q0 + nq, a:a + Dh].double() @ kk.t() / math.sqrt(Dh)
                ahead = torch.ones(nq, nk, dtype=torch.bool, device=DEV).triu(nk - nq + 1)
                w = w.masked_fill(ahead, -math.inf)
                if s["prefix"]:
                    pk, pv = (t[:, b:b + Dh].double() for t in s["prefix"])
                    w = torch.cat((s["q"][q0:q0 + nq, a:a + Dh].double() @ pk.t() / math.sqrt(Dh), w), 1)
                    v = torch.cat((pv, v))
                out[q0:q0 + nq, a:a + Dh] = torch.softmax(w, -1) @ v
        return out
    if k == "norm":
        h = s["x"].double() if s["res"] is None else s["x"].double() + s["res"].double()
        y = h / torch.sqrt(h.square().sum(-1, keepdim=True) / case["dim"] + EPS) * s["w"].double()
        if case.get("bits8"):
            y = _exact_fp8(y)
        return (y, h) if s["res"] is not None else y
    acc = _exact_values8(*s["x"]) @ _exact_values4(*s["w"]).t()
    return torch.special.ndtr(acc) * acc if case["epi"] == "gelu" else acc


# ---- the least a pass can do ----

def work(case):
    k = case["kind"]
    if k == "prompt":
        lens, P, W = _lens(case), case["P"], 2.0 * case["Dh"]
        rows, keys = sum(nq for nq, _ in lens), P + sum(nk for nq, nk in lens if nq)
        pairs = sum(nq * (P + nk - nq) + nq * (nq + 1) // 2 for nq, nk in lens)
        return dict(bytes=W * (2 * rows * case["Hq"] + 2 * keys * case["Hkv"]), flops=4.0 * pairs * case["Hq"] * case["Dh"])
    if k == "norm":
        n = float(case["rows"] * case["dim"])
        each = BYTES[case["x"]] + BYTES[case["y"]]
        if case["res"] != "none":
            each += 2 * BYTES[case["res"]]
        if case.get("bits8"):  # codes and scales written, and read for the values they stand for
            each += 2 * (1 + 1 / 32)
        return dict(bytes=n * each + 2 * case["dim"], flops=5.0 * n)
    T, N, K = case["T"], case["N"], case["K"]
    return dict(bytes=T * K * (1 + 1 / 32) + N * K * (0.5 + 1 / 32) + T * N * (4 if case["epi"] == "f32" else 2), flops=2.0 * T * N * K)
