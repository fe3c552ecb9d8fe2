"""Cases that measure the 4-bit linears and the rotated keys of a decoder layer: the quantizer to e2m1 codes with block
scales (`quantize`), the product of two such operands (`product`), the per-head RMSNorm with the position rotation (`rotate`),
and the write into the paged cache with both on the way (`append`).

`run` computes a pass in plain torch operations in 32 bits (angles in 64), or, with `own`, by the calls a user makes. `exact`
computes the same from the definitions in 64 bits.

Formats. A code is one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign, two to a byte, the even element in the low half. "mxfp4": a
scale 2^(byte - 127) per 32 elements. "nvfp4": an e4m3 scale per 16 elements, and one fp32 scale per row. Scale bytes lie in
tiles of 128 rows x 4 groups, 512 bytes each: [row blocks, group blocks, 32, 4, 4] for row 32 i + r of the block, group j: [r, i, j].
"""
import math
import os
import sys

import numpy as np
import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_PKG = os.path.join(_ROOT, "comfyui-hy-nomas_b200")
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = {"nvfp4": 16, "mxfp4": 32}
YARN = {"type": "yarn", "factor": 16.0, "original": 4096}


# --------------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # one token in front of a linear: the latency of a decoding step
        {"name": "quantize 1x4096 nvfp4", "op": "quantize", "rows": 1, "k": 4096, "kind": "nvfp4", "dtype": "bf16"},
        # a ragged batch of prompts in half precision, a width that is not a multiple of the scale tiles
        {"name": "quantize 333x2080 mxfp4 fp16", "op": "quantize", "rows": 333, "k": 2080, "kind": "mxfp4", "dtype": "fp16"},
        # a whole denoising segment with its history: 23 x 22 x 40 tokens of 4096 channels
        {"name": "quantize 20240x4096 nvfp4", "op": "quantize", "rows": 20240, "k": 4096, "kind": "nvfp4", "dtype": "bf16"},
        # one token through the second MLP linear: the weights' bytes
        {"name": "product 1x4096x16384 nvfp4", "op": "product", "m": 1, "n": 4096, "k": 16384, "kind": "nvfp4", "bias": False,
         "out": "bf16"},
        # one token each of 48 branches through the stacked q|k linear
        {"name": "product 48x8192x4096 mxfp4", "op": "product", "m": 48, "n": 8192, "k": 4096, "kind": "mxfp4", "bias": False,
         "out": "bf16"},
        # ragged prompts, an odd number of channels, with a bias, fp32 out
        {"name": "product 777x5001x2080 nvfp4", "op": "product", "m": 777, "n": 5001, "k": 2080, "kind": "nvfp4", "bias": True,
         "out": "fp32"},
        # the second MLP linear of a whole segment
        {"name": "product 20240x4096x16384 nvfp4", "op": "product", "m": 20240, "n": 4096, "k": 16384, "kind": "nvfp4",
         "bias": False, "out": "bf16"},
        # one token's queries: latency
        {"name": "rotate 1x1 half", "op": "rotate", "batch": 1, "tokens": 1, "heads": 32, "dim": 128, "rot": 128,
         "layout": "half", "scaling": None, "norm": True, "dtype": "bf16", "first": 777},
        # a part of a head of 96, fp32, far positions of a scaled context
        {"name": "rotate 5x777 part of 96 fp32", "op": "rotate", "batch": 5, "tokens": 777, "heads": 12, "dim": 96, "rot": 48,
         "layout": "interleaved", "scaling": "yarn", "norm": False, "dtype": "fp32", "first": 60000},
        # the queries of a whole segment
        {"name": "rotate 20240 interleaved", "op": "rotate", "batch": 1, "tokens": 20240, "heads": 32, "dim": 128, "rot": 128,
         "layout": "interleaved", "scaling": None, "norm": True, "dtype": "bf16", "first": 0},
        # one token for each of 48 branches
        {"name": "append 48x1 bf16", "op": "append", "batch": 48, "tokens": 1, "heads": 32, "kv": 8, "page": 64, "start": 300,
         "kind": "bf16", "rot": 128, "layout": "half", "scaling": None, "norm": True},
        # the cache pass of a generated segment: 5 frames of 880 tokens, two branches, half of the head rotated, int8 history
        {"name": "append 2x4400 int8", "op": "append", "batch": 2, "tokens": 4400, "heads": 16, "kv": 16, "page": 32,
         "start": 15840, "kind": "int8", "rot": 64, "layout": "half", "scaling": "yarn", "norm": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "quantize", "product", "product", "product", "product", "rotate", "rotate", "append", "append"])
    kind = rng.choice(["nvfp4", "mxfp4"])
    if op == "quantize":
        k = _log(rng, 16, 16384)
        if rng.random() < 0.6:
            k = max(32, k // 32 * 32)
        return {"op": op, "rows": _log(rng, 1, max(1, 20240 * 4096 // k)), "k": k, "kind": kind,
                "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    if op == "product":
        m = rng.choice([1, 2, _log(rng, 1, 20240), _log(rng, 1, 20240)])
        n, k = _log(rng, 8, 16384), 32 * _log(rng, 1, 512)
        while m * n * k > 20240 * 4096 * 16384:
            m //= 2
        return {"op": op, "m": m, "n": n, "k": k, "kind": kind, "bias": rng.random() < 0.4,
                "out": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    layout, scaling = rng.choice(["half", "interleaved"]), rng.choice([None, "linear", "ntk", "yarn"])
    tokens = 1 if rng.random() < 0.4 else _log(rng, 2, 20240 if op == "rotate" else 4400)
    if op == "rotate":
        dim = 8 * rng.randint(2, 32)
        heads = rng.choice([1, 2, 5, 8, 12, 16, 32])
        batch = _log(rng, 1, max(1, min(64, 20240 * 32 * 128 // (tokens * heads * dim))))
        while batch * tokens * heads * dim > 20240 * 32 * 128:
            tokens //= 2
        return {"op": op, "batch": batch, "tokens": tokens, "heads": heads, "dim": dim,
                "rot": dim if rng.random() < 0.5 else 8 * rng.randint(1, dim // 8), "layout": layout, "scaling": scaling,
                "norm": rng.random() < 0.6, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "first": _log(rng, 1, 10 ** 6) - 1}
    kv = rng.choice([1, 2, 4, 8, 16])
    heads = kv * rng.choice([1, 2, 4, 7, 8])
    most = max(1, min(64, 2 * 4400 * 48 // (tokens * (heads + 2 * kv))))
    while tokens * (heads + 2 * kv) > 2 * 4400 * 48:
        tokens //= 2
    return {"op": op, "batch": _log(rng, 1, most), "tokens": tokens, "heads": heads, "kv": kv,
            "page": rng.choice([16, 32, 48, 64, 128]), "start": _log(rng, 1, 900) - 1, "kind": rng.choice(["bf16", "int8"]),
            "rot": rng.choice([128, 128, 64, 96, 32, 8]), "layout": layout, "scaling": scaling, "norm": rng.random() < 0.6}


def work(c):
    if c["op"] == "quantize":
        n = c["rows"] * c["k"]
        scales = n // BLOCK[c["kind"]] + (4 * c["rows"] if c["kind"] == "nvfp4" else 0)
        return {"bytes": n * DTYPES[c["dtype"]].itemsize + n // 2 + scales, "flops": 6 * n}
    if c["op"] == "product":
        m, n, k = c["m"], c["n"], c["k"]
        scales = (m + n) * k // BLOCK[c["kind"]] + (4 * (m + n) if c["kind"] == "nvfp4" else 0)
        return {"bytes": (m + n) * k // 2 + scales + m * n * DTYPES[c["out"]].itemsize + (2 * n if c["bias"] else 0),
                "flops": 2 * m * n * k}
    if c["op"] == "rotate":
        n = c["batch"] * c["tokens"] * c["heads"] * c["dim"]
        return {"bytes": 2 * n * DTYPES[c["dtype"]].itemsize, "flops": 8 * n}
    rows, q = c["batch"] * c["tokens"] * c["kv"], c["batch"] * c["tokens"] * c["heads"]
    return {"bytes": 4 * 128 * q + rows * (2 * 256 + 2 * (256 if c["kind"] == "bf16" else 132)), "flops": 8 * 128 * (q + 2 * rows)}


# --------------------------------------------------------------------------------------------------- inputs

def _framework():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)


def _randn(shape, gen, dtype=torch.bfloat16, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _scaling(c):
    return {None: None, "linear": {"type": "linear", "factor": 4.0}, "ntk": {"type": "ntk", "factor": 8.0}, "yarn": YARN}[c["scaling"]]


def _frequencies(rot, scaling, theta=10000.0):
    """Radians a position in 64 bits, and the factor on cos and sin."""
    i = np.arange(rot // 2)
    kind = scaling["type"] if scaling else None
    if kind == "ntk" and rot > 2:
        theta = theta * scaling["factor"] ** (rot / (rot - 2))
    f = theta ** (-2.0 * i / rot)
    if kind == "linear":
        return f / scaling["factor"], 1.0
    if kind != "yarn":
        return f, 1.0
    # the dimension whose angle makes `turns` turns over the original context
    at = lambda turns: rot * math.log(scaling["original"] / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
    low, high = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
    ramp = np.clip((i - low) / max(high - low, 0.001), 0.0, 1.0)
    return f * (1 - ramp) + f / scaling["factor"] * ramp, 0.1 * math.log(scaling["factor"]) + 1.0


def _weights_like(rows, k, kind, gen):
    """Codes, tiled scales and row scales as a quantizer leaves them: normal numbers with a few loud channels."""
    loud = torch.where(torch.rand(k, generator=gen, device="cuda") < 0.01, 8.0, 1.0)
    out = [torch.empty((rows, k // 2), dtype=torch.uint8, device="cuda"),
           torch.empty((rows, k // BLOCK[kind]), dtype=torch.uint8, device="cuda"),
           torch.empty(rows, dtype=torch.float32, device="cuda") if kind == "nvfp4" else None]
    step = max(1, (1 << 26) // k)
    for r in range(0, rows, step):
        n = min(step, rows - r)
        idx, sb, sr = _quantize(torch.randn((n, k), generator=gen, device="cuda") * loud, kind)
        out[0][r:r + n] = idx[:, 0::2] | idx[:, 1::2] << 4
        out[1][r:r + n] = _scale_bytes(sb, kind)
        if sr is not None:
            out[2][r:r + n] = sr
    return out[0], _tile(out[1]), out[2]


def _tile(plain):
    """[rows, groups] bytes -> tiles of 128 rows x 4 groups."""
    rows, groups = plain.shape
    full = plain.new_zeros((-(-rows // 128) * 128, -(-groups // 4) * 4))
    full[:rows, :groups] = plain
    return full.view(full.shape[0] // 128, 4, 32, full.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).reshape(
        full.shape[0] // 128, full.shape[1] // 4, 512).contiguous()


def _untile(tiled, rows, groups):
    a, b, _ = tiled.shape
    return tiled.view(a, b, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(a * 128, b * 4)[:rows, :groups]


def prepare(c, seed):
    gen, rnd = torch.Generator(device="cuda").manual_seed(seed), np.random.default_rng(seed)
    s = {"case": c}
    if own:
        _framework()
        from hy_nomas_b200 import kernels, paged, rotary
        s["kernels"], s["rotary"] = kernels, rotary
    if c["op"] == "quantize":
        loud = torch.where(torch.rand(c["k"], generator=gen, device="cuda") < 0.01, 12.0, 1.0)
        s["x"] = (torch.randn((c["rows"], c["k"]), generator=gen, device="cuda") * loud).to(DTYPES[c["dtype"]])
        return s
    if c["op"] == "product":
        s["a"] = _weights_like(c["m"], c["k"], c["kind"], gen)
        s["w"] = _weights_like(c["n"], c["k"], c["kind"], gen)
        s["bias"] = _randn((c["n"],), gen) if c["bias"] else None
        return s
    rot = c["rot"]
    s["freq"], s["factor"] = _frequencies(rot, _scaling(c))
    s["freq"] = torch.from_numpy(s["freq"]).cuda()
    if own:
        s["rot"] = rotary.Rotary(rot, 10000.0, c["layout"], _scaling(c))
    if c["op"] == "rotate":
        b, n, h, d = c["batch"], c["tokens"], c["heads"], c["dim"]
        s["x"] = _randn((b, n, h, d), gen, DTYPES[c["dtype"]], 2.0)
        s["w"] = (1 + 0.2 * torch.randn(d, generator=gen, device="cuda")).to(torch.bfloat16) if c["norm"] else None
        starts = torch.tensor([max(0, c["first"] - 131 * i) for i in range(b)], device="cuda")
        s["pos"] = (starts[:, None] + torch.arange(n, device="cuda")).int()
        return s
    b, n, h, kv, page = c["batch"], c["tokens"], c["heads"], c["kv"], c["page"]
    lens = [max(n, c["start"] + n - (i * 13) % (c["start"] + 1)) for i in range(b)]
    # the cache holds the pages from the first that is written on; those before stand in one table entry that is not touched
    width = max(-(-x // page) for x in lens)
    firsts = [(x - n) // page for x in lens]
    need = [-(-x // page) - f for x, f in zip(lens, firsts)]
    pages = sum(need) + 3
    ids = iter(rnd.permutation(np.arange(1, pages)).tolist())
    table = np.full((b, width), -1, np.int32)
    for i in range(b):
        table[i, :firsts[i]] = 0
        table[i, firsts[i]:firsts[i] + need[i]] = [next(ids) for _ in range(need[i])]
    refs = np.bincount(table[table >= 0], minlength=pages).astype(np.int32)
    s["meta"] = torch.from_numpy(np.concatenate([table.reshape(-1), np.array(lens, np.int32), refs])).cuda()
    s["table"], s["lengths"] = s["meta"][:b * width].view(b, width), s["meta"][b * width:b * width + b]
    shape = (1, pages, kv, page, 128)
    if c["kind"] == "bf16":
        s["k"], s["v"] = (torch.zeros(shape, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        s["ks"] = s["vs"] = None
    else:
        s["k"], s["v"] = (torch.zeros(shape, dtype=torch.int8, device="cuda") for _ in range(2))
        s["ks"], s["vs"] = (torch.ones(shape[:4], device="cuda") for _ in range(2))
    packed = _randn((b, n, h + 2 * kv, 128), gen, scale=2.0)           # the projection's q | k | v
    s.update(q=packed[:, :, :h], nk=packed[:, :, h:h + kv], nv=packed[:, :, h + kv:])
    s["wq"], s["wk"] = ((1 + 0.2 * torch.randn(128, generator=gen, device="cuda")).to(torch.bfloat16) if c["norm"] else None
                        for _ in range(2))
    s["rows"] = torch.arange(b, dtype=torch.int32, device="cuda")
    if own:
        s["cache"] = paged.KVCache.over(s["k"], s["v"], s["ks"], s["vs"], s["meta"], b, width)
    return s


# --------------------------------------------------------------------------------------------------- passes

def run(s):
    c = s["case"]
    if own:
        return _run_own(s, c)
    return {"quantize": _plain_quantize, "product": _plain_product, "rotate": _plain_rotate, "append": _plain_append}[c["op"]](s, c)


def _run_own(s, c):
    if c["op"] == "quantize":
        codes, scales, rows = s["kernels"].quantize_fp4(s["x"], c["kind"])
        out = {"values": s["kernels"].dequantize_fp4(codes, scales, rows, c["kind"], columns=c["k"])}
        return {**out, "rows": rows} if rows is not None else out
    if c["op"] == "product":
        return s["kernels"].fp4_gemm(*s["a"], *s["w"], bias=s["bias"], kind=c["kind"], out_dtype=DTYPES[c["out"]])
    if c["op"] == "rotate":
        return s["rotary"].rotate(s["x"], s["pos"], s["rot"], s["w"], EPS)
    cache = s["cache"]
    q = cache.append_rotated(0, s["q"], s["nk"], s["nv"], s["rows"], s["rot"], s["wq"], s["wk"], EPS)
    return _written(s, c, q)


def _written(s, c, q):
    """The queries and the pages, int8 codes as the values they stand for."""
    if c["kind"] == "bf16":
        return {"q": q, "k": s["k"], "v": s["v"]}
    if own:
        from hy_nomas_b200.world import dequantize_kv
        return {"q": q, "k": dequantize_kv(s["k"], s["ks"]), "v": dequantize_kv(s["v"], s["vs"]), "ks": s["ks"], "vs": s["vs"]}
    return {"q": q, "k": (s["k"].float() * s["ks"][..., None]).to(torch.bfloat16),
            "v": (s["v"].float() * s["vs"][..., None]).to(torch.bfloat16), "ks": s["ks"], "vs": s["vs"]}


def _e2m1(y):
    """Values -> 4-bit codes: to the nearest, ties to the even code, what lies beyond 6 to 6."""
    a = y.abs()
    n = (a > 0.25).to(torch.uint8)
    for edge, closed in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        n += (a >= edge) if closed else (a > edge)
    return n | torch.signbit(y).to(torch.uint8) << 3


def _value(codes):
    """4-bit codes -> values."""
    table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    return table[codes.long()]


def _quantize(x, kind):
    """fp32 [M, K], K a multiple of the block -> 4-bit codes [M, K] one to a byte, block scales [M, K / block] (values), row
    scales [M] or None."""
    m, k = x.shape
    blocks = x.view(m, -1, BLOCK[kind])
    peak = blocks.abs().amax(-1)
    if kind == "mxfp4":
        exponent = torch.frexp(peak)[1] - 3                     # floor(log2 peak) - 2
        sb = torch.exp2(exponent.clamp(-127, 127).double()).float()
        sb = torch.where(peak > 0, sb, torch.ones_like(sb))
        return _e2m1((blocks / sb[..., None]).view(m, k)), sb, None
    # products with short constants first: one rounding, at the division, so that what is half-way between two codes is so here
    top = peak.amax(-1)
    live = top >= 2.0 ** -100
    top = torch.where(live, top, torch.ones_like(top))
    sr = torch.where(live, top / 2688.0, torch.ones_like(top))
    sb = (0.875 * peak / (top * 2.0 ** -9)[:, None] * live[:, None]).to(torch.float8_e4m3fn).float()
    den = sb * (top * 2.0 ** -12)[:, None]
    y = torch.where(sb[..., None] > 0, 0.65625 * blocks / den[..., None], torch.zeros_like(blocks))
    return _e2m1(y.view(m, k)), sb, sr


def _scale_bytes(sb, kind):
    if kind == "nvfp4":
        return sb.to(torch.float8_e4m3fn).view(torch.uint8)
    return (torch.frexp(sb)[1] + 126).to(torch.uint8)


def _scale_values(b, kind):
    if kind == "nvfp4":
        return b.contiguous().view(torch.float8_e4m3fn).float()
    return torch.exp2(b.double() - 127).float()


def _plain_quantize(s, c):
    x, k, block = s["x"].float(), c["k"], BLOCK[c["kind"]]
    if k % block:
        x = torch.nn.functional.pad(x, (0, block - k % block))
    codes, sb, sr = _quantize(x, c["kind"])
    d = sb if sr is None else sb * sr[:, None]
    values = (_value(codes).view(*d.shape, block) * d[..., None]).view(codes.shape)[:, :k].to(torch.bfloat16)
    return {"values": values} if sr is None else {"values": values, "rows": sr}


def _operand(codes, tiled, kind):
    """fp32 values without the row scales."""
    m, k = codes.shape[0], codes.shape[1] * 2
    both = torch.stack([codes & 15, codes >> 4], -1).view(m, k)
    sb = _scale_values(_untile(tiled, m, k // BLOCK[kind]), kind)
    return (_value(both).view(m, -1, BLOCK[kind]) * sb[..., None]).view(m, k)


def _plain_product(s, c):
    (qa, sa, ra), (qw, sw, rw) = s["a"], s["w"]
    y = _operand(qa, sa, c["kind"]) @ _operand(qw, sw, c["kind"]).t()
    if ra is not None:
        y = y * ra[:, None] * rw
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(DTYPES[c["out"]])


def _plain_turn(x, pos, s, c, w):
    """x [B, n, H, D] fp32 normed and rotated."""
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()
    angle = pos.double()[..., None] * s["freq"]
    cos, sin = (f(angle).mul(s["factor"]).float()[:, :, None] for f in (torch.cos, torch.sin))
    rot = c["rot"]
    if c["layout"] == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned, x[..., rot:]], -1)


def _plain_rotate(s, c):
    return _plain_turn(s["x"].float(), s["pos"], s, c, s["w"]).to(DTYPES[c["dtype"]])


def _int8(x):
    """The cache's int8 format: absmax / 127 per (token, head), codes rounded half away from zero."""
    peak = x.abs().amax(-1, keepdim=True)
    sc = torch.where(peak > 0, peak / 127, torch.ones_like(peak))
    y = x / sc
    return torch.trunc(y + torch.copysign(torch.full_like(y, 0.5), y)).clamp(-127, 127).to(torch.int8), sc[..., 0]


def _plain_append(s, c):
    n, page = c["tokens"], c["page"]
    pos = s["lengths"].long()[:, None] - n + torch.arange(n, device="cuda")
    q = _plain_turn(s["q"].float(), pos, s, c, s["wq"]).to(torch.bfloat16)
    k = _plain_turn(s["nk"].float(), pos, s, c, s["wk"])
    ids, place = s["table"].long().gather(1, pos // page), pos % page
    for name, x in (("k", k), ("v", s["nv"].float())):
        if c["kind"] == "bf16":
            s[name][0, ids, :, place] = x.to(torch.bfloat16)
        else:
            codes, sc = _int8(x)
            s[name][0, ids, :, place] = codes
            s[name + "s"][0, ids, :, place] = sc
    return _written(s, c, q)


# --------------------------------------------------------------------------------------------------- 64 bits

def exact(c, seed):
    """The same outputs from the definitions in 64 bits: the scales before their rounding to 32 bits, the codes those of
    64-bit quotients."""
    global own
    was, own = own, False
    try:
        s = prepare(c, seed)
    finally:
        own = was
    return {"quantize": _exact_quantize, "product": _exact_product, "rotate": _exact_rotate, "append": _exact_append}[c["op"]](s, c)


def _exact_quantize(s, c):
    k, block = c["k"], BLOCK[c["kind"]]
    x = torch.nn.functional.pad(s["x"].double(), (0, -k % block)).reshape(c["rows"], -1, block)
    peak = x.abs().max(2).values
    if c["kind"] == "mxfp4":
        scale = torch.where(peak > 0, peak / torch.frexp(peak)[0] / 8, 1.0)     # a power of two, by exact divisions
        return {"values": _exact_codes(x, scale).flatten(1)[:, :k]}
    top = peak.max(1).values
    rows = torch.where(top > 0, top / 2688.0, 1.0)
    t = peak * 448.0 / top.clamp(min=1e-300).unsqueeze(1)
    normal = t.clamp(min=2.0 ** -6)
    step = normal / torch.frexp(normal)[0] / 16                                 # of e4m3 at t
    scale = torch.round(t / step) * step
    values = _exact_codes(x * 2688.0, scale * top.unsqueeze(1)) / 2688.0
    return {"values": values.flatten(1)[:, :k], "rows": rows}


def _exact_codes(x, scale):
    """What the nearest multiple of the scale in the list of codes is worth (ties to the even code)."""
    y = torch.where(scale.unsqueeze(2) > 0, x / scale.unsqueeze(2), 0.0)
    size = y.abs().clamp(max=6.0)
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    return torch.copysign(torch.round(size / step) * step, y) * scale.unsqueeze(2)


def _exact_operand(codes, tiled, rows, kind):
    """Row by row of the scale tiles: byte (r % 32) 16 + (r // 32 % 4) 4 + g % 4 of tile (r // 128, g // 4)."""
    m, k = codes.shape[0], codes.shape[1] * 2
    out = torch.empty((m, k), dtype=torch.float64, device=codes.device)
    for half, nibble in ((0, codes % 16), (1, codes // 16)):
        magnitude, sign = nibble % 8, 1.0 - 2.0 * (nibble // 8).double()
        e, f = (magnitude // 2).double(), (magnitude % 2).double()
        out[:, half::2] = sign * torch.where(e > 0, (1 + f / 2) * 2.0 ** (e - 1), f / 2)
    r = torch.arange(m, device=codes.device)[:, None]
    g = torch.arange(k // BLOCK[kind], device=codes.device)[None]
    byte = tiled[r // 128, g // 4, r % 32 * 16 + r // 32 % 4 * 4 + g % 4].double()
    if kind == "nvfp4":
        e, f = torch.div(byte, 8, rounding_mode="floor"), byte % 8      # e4m3 without a sign
        scale = torch.where(e > 0, (1 + f / 8) * 2.0 ** (e - 7), f / 8 * 2.0 ** -6)
    else:
        scale = 2.0 ** (byte - 127)
    out.view(m, -1, BLOCK[kind]).mul_(scale.unsqueeze(2))
    return out if rows is None else out.mul_(rows.double().unsqueeze(1))


def _exact_product(s, c):
    w = _exact_operand(*s["w"], c["kind"])
    y = _exact_operand(*s["a"], c["kind"]) @ w.t()
    return y if s["bias"] is None else y + s["bias"].double()


def _exact_turn(x, pos, c, w):
    x = x.double()
    if w is not None:
        x = x / (x.pow(2).mean(3, keepdim=True) + EPS).sqrt() * w.double()
    freq, factor = _frequencies(c["rot"], _scaling(c))
    out = x.clone()
    half = c["rot"] // 2
    for i in range(half):
        j, l = (i, i + half) if c["layout"] == "half" else (2 * i, 2 * i + 1)
        turn = torch.polar(torch.full(pos.shape, factor, dtype=torch.float64, device=pos.device), pos.double() * float(freq[i]))
        z = torch.complex(x[..., j], x[..., l]) * turn.unsqueeze(2)
        out[..., j], out[..., l] = z.real, z.imag
    return out


def _exact_rotate(s, c):
    return _exact_turn(s["x"], s["pos"], c, s["w"])


def _exact_append(s, c):
    n, page = c["tokens"], c["page"]
    at = s["lengths"].tolist()
    pos = torch.tensor([list(range(x - n, x)) for x in at], device="cuda")
    out = {"q": _exact_turn(s["q"], pos, c, s["wq"])}
    new = {"k": _exact_turn(s["nk"], pos, c, s["wk"]), "v": s["nv"].double()}
    table = s["table"].tolist()
    for name, x in new.items():
        pool = torch.zeros(s[name].shape, dtype=torch.float64, device="cuda")
        scales = torch.ones(pool.shape[:4], dtype=torch.float64, device="cuda")
        peak = x.abs().max(3).values
        for b, length in enumerate(at):
            for block in range((length - n) // page, (length - 1) // page + 1):
                lo, hi = max(length - n, block * page), min(length, (block + 1) * page)
                take, put = slice(lo - length + n, hi - length + n), slice(lo - block * page, hi - block * page)
                pool[0, table[b][block], :, put] = x[b, take].transpose(0, 1)
                scales[0, table[b][block], :, put] = torch.where(peak > 0, peak / 127.0, 1.0)[b, take].t()
        out[name] = pool
        if c["kind"] == "int8":
            y = pool / scales.unsqueeze(4)
            out[name] = torch.copysign(torch.floor(y.abs() + 0.5), y) * scales.unsqueeze(4)
            out[name + "s"] = scales
    return out
