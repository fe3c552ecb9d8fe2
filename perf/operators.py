"""Cases that measure the serving operators of a forked K/V cache: the write into its pages (`append`), the page
operations (`fork`, `free`, `compact`), the attention that reads the shared history once (`attention`), and the
residual + RMSNorm + 8-bit quantizer that closes a decoder layer (`norm`).

`run` computes a pass in plain torch operations in 32 bits, or, with `own`, by the calls a user makes. `exact` computes
the same from the definitions in 64 bits. Head dim 128 throughout. The K/V formats are the framework's: bf16, or int8
codes with one fp32 scale per (token, head).
"""
import math
import os
import sys

import numpy as np
import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_PKG = os.path.join(_ROOT, "comfyui-hy-nomas_b200")
D = 128
EPS = 1e-6


# --------------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # one token's residual and norm: the latency of a decoding step
        {"name": "norm 1x4096 fp8", "op": "norm", "rows": 1, "dim": 4096, "kind": "fp8", "per_token": False},
        # a ragged batch, int8 per token (the usual W8A8 activation format), the hidden size of the released model
        {"name": "norm 333x2048 int8 token", "op": "norm", "rows": 333, "dim": 2048, "kind": "int8", "per_token": True},
        # a whole denoising segment with its history: 23 x 22 x 40 tokens of 4096 channels
        {"name": "norm 20240x4096 fp8", "op": "norm", "rows": 20240, "dim": 4096, "kind": "fp8", "per_token": False},
        # one token for each of 48 branches
        {"name": "append 48x1 bf16", "op": "append", "batch": 48, "tokens": 1, "heads": 8, "page": 64, "start": 300,
         "kind": "bf16"},
        # the cache pass of a generated segment: 5 frames of 880 tokens, two branches, into the int8 history
        {"name": "append 2x4400 int8", "op": "append", "batch": 2, "tokens": 4400, "heads": 16, "page": 32, "start": 0,
         "kind": "int8"},
        # three branches from one short sequence
        {"name": "fork 1 to 3", "op": "fork", "layers": 2, "heads": 8, "page": 16, "parents": 1, "each": 3,
         "length": 203, "kind": "bf16"},
        # a beam step: 8 parents, 8 new branches each, through 36 layers
        {"name": "fork 8 to 64", "op": "fork", "layers": 36, "heads": 8, "page": 64, "parents": 8, "each": 8,
         "length": 929, "kind": "int8"},
        # half the sequences have ended: their holes are filled from the top of the pool
        {"name": "compact 1024 pages", "op": "compact", "layers": 16, "heads": 8, "page": 32, "pages": 1024, "live": 640,
         "moves": 240, "rows": 40, "kind": "bf16"},
        # one sequence, one token: latency
        {"name": "attend 1x1 over 777", "op": "attention", "batch": 1, "lq": 1, "heads": 32, "kv": 8, "page": 64,
         "shared": 0, "own": 777, "ragged": 1, "kind": "bf16", "causal": True},
        # 32 branches of one 18-frame history decode one token each
        {"name": "attend 32x1 over 15840", "op": "attention", "batch": 32, "lq": 1, "heads": 32, "kv": 8, "page": 32,
         "shared": 15840, "own": 512, "ragged": 300, "kind": "int8", "causal": True},
        # a few drafted tokens per branch, causal, small pages
        {"name": "attend 16x5 over 4096", "op": "attention", "batch": 16, "lq": 5, "heads": 16, "kv": 16, "page": 16,
         "shared": 4096, "own": 1101, "ragged": 700, "kind": "bf16", "causal": True},
        # two branches denoise a segment of 5 frames over the 18-frame int8 history
        {"name": "attend 2x4400 over 15840", "op": "attention", "batch": 2, "lq": 4400, "heads": 16, "kv": 16, "page": 32,
         "shared": 15840, "own": 4400, "ragged": 1, "kind": "int8", "causal": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        case = _drawn(rng)
        if 3072 not in case.values():
            return case


def _drawn(rng):
    op = rng.choice(["norm", "norm", "append", "append", "fork", "compact", "attention", "attention", "attention",
                     "attention"])
    kind = rng.choice(["bf16", "int8"])
    page = rng.choice([16, 32, 48, 64, 128])
    heads = rng.choice([1, 2, 5, 8, 16, 32])
    if op == "norm":
        dim = 128 * _log(rng, 1, 96)
        return {"op": op, "rows": _log(rng, 1, max(1, 20240 * 4096 // dim)), "dim": dim, "kind": rng.choice(["fp8", "int8"]),
                "per_token": rng.random() < 0.4}
    if op == "append":
        tokens = _log(rng, 1, 4400)
        most = max(1, min(64, 2 * 4400 * 16 // (tokens * heads)))
        return {"op": op, "batch": _log(rng, 1, most), "tokens": tokens, "heads": heads, "page": page,
                "start": _log(rng, 1, 900) - 1, "kind": kind}
    if op == "fork":
        parents, each = _log(rng, 1, 8), _log(rng, 1, 8)
        layers = _log(rng, 1, max(1, 36 * 8 // heads))
        return {"op": op, "layers": min(layers, 40), "heads": heads, "page": min(page, 64), "parents": parents,
                "each": each, "length": _log(rng, 1, 930), "kind": kind}
    if op == "compact":
        pages = _log(rng, 24, 1024)
        live = rng.randint(pages // 4, pages - 4)
        layers = _log(rng, 1, max(1, 16 * 8 * 32 // (heads * page)))
        return {"op": op, "layers": layers, "heads": heads, "page": page, "pages": pages, "live": live,
                "moves": rng.randint(0, min(live, pages - live, 240)), "rows": rng.randint(1, 40), "kind": kind}
    kv = rng.choice([1, 2, 4, 8, 16])
    heads = kv * rng.choice([1, 2, 4, 7, 8])
    lq = 1 if rng.random() < 0.4 else _log(rng, 2, 4400)
    batch = _log(rng, 1, 64)
    shared = 0 if rng.random() < 0.25 else _log(rng, page, 15840) // page * page
    mine = _log(rng, 1, 4400)
    causal = rng.random() < 0.6
    if causal and rng.random() < 0.85:
        mine = max(mine, lq)      # the queries' own tokens are in the cache; else the first of them see nothing
    case = {"op": op, "batch": batch, "lq": lq, "heads": heads, "kv": kv, "page": page, "shared": shared, "own": mine,
            "ragged": rng.randint(1, mine), "kind": kind, "causal": causal}
    # no more pairs of a query and a key than the largest listed case has, nor more keys in all
    for name, least in (("batch", 1), ("lq", 1), ("shared", 0), ("own", 1)):
        while _pairs(case) > 2 * 4400 * 16 * 20240 or (shared + batch * mine) * kv > 2 * 20240 * 16:
            if case[name] // 2 < least:
                break
            case[name] //= 2
            if name == "shared":
                case[name] = case[name] // page * page
            batch, mine, shared = case["batch"], case["own"], case["shared"]
    case["ragged"] = min(case["ragged"], case["own"])
    return case


def _pairs(c):
    return c["batch"] * c["lq"] * c["heads"] * (c["shared"] + c["own"])


def _lengths(c):
    """The whole length of each sequence: the shared tokens and its own, which differ by up to `ragged` - 1."""
    return [c["shared"] + c["own"] - (b * 37) % c["ragged"] for b in range(c["batch"])]


def _fork_lengths(c):
    return [max(1, c["length"] - 7 * p) for p in range(c["parents"])]


def _token_bytes(c):
    """K and V of one token and head in the cache."""
    return 2 * (D * 2 if c["kind"] == "bf16" else D + 4)


def work(c):
    if c["op"] == "norm":
        n = c["rows"] * c["dim"]
        scales = c["rows"] * (1 if c["per_token"] else c["dim"] // 128)
        return {"bytes": n * 7 + c["dim"] * 2 + scales * 4, "flops": 8 * n}
    if c["op"] == "append":
        n = c["batch"] * c["tokens"] * c["heads"]
        return {"bytes": n * (2 * D * 2 + _token_bytes(c)), "flops": 0 if c["kind"] == "bf16" else 6 * n * D}
    if c["op"] == "fork":
        tails = sum(n % c["page"] for n in _fork_lengths(c)) * c["each"]
        full = sum(-(-n // c["page"]) for n in _fork_lengths(c)) * c["each"]
        return {"bytes": 2 * tails * c["layers"] * c["heads"] * _token_bytes(c) + 16 * full, "flops": 0}
    if c["op"] == "compact":
        moved = c["moves"] * c["layers"] * c["heads"] * c["page"] * _token_bytes(c)
        return {"bytes": 2 * moved + 8 * (c["pages"] + c["live"]), "flops": 0}
    keys = c["shared"] + sum(n - c["shared"] for n in _lengths(c))
    if c["causal"]:
        pairs = sum(max(0, min(n, n - c["lq"] + i + 1)) for n in _lengths(c) for i in range(c["lq"]))
    else:
        pairs = sum(n * c["lq"] for n in _lengths(c))
    return {"bytes": 4 * c["batch"] * c["lq"] * c["heads"] * D + keys * c["kv"] * _token_bytes(c),
            "flops": 4 * D * c["heads"] * pairs}


# --------------------------------------------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(shape, gen, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(torch.bfloat16)


def _quantize(x):
    """The framework's K/V format: absmax / 127 per (token, head), codes rounded half away from zero."""
    x = x.float()
    peak = x.abs().amax(-1, keepdim=True)
    s = torch.where(peak > 0, peak / 127, torch.ones_like(peak))
    y = x / s
    return torch.trunc(y + torch.copysign(torch.full_like(y, 0.5), y)).clamp(-127, 127).to(torch.int8), s[..., 0]


def _pool(layers, pages, heads, page, kind, gen):
    """A pool that has been in use: every page holds K and V of some sequence. K is RMS-normed as QK-norm leaves it."""
    pools = []
    for which in range(2):
        x = torch.randn((layers, pages, heads, page, D), generator=gen, device="cuda")
        if which == 0:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True))
        pools.append((x.to(torch.bfloat16), None) if kind == "bf16" else _quantize(x.to(torch.bfloat16)))
        del x
    (k, ks), (v, vs) = pools
    return {"k": k, "v": v, "ks": ks, "vs": vs, "page": page}


def _meta(rows, width, pages, table, lengths):
    """Page table [rows, width] (-1: none), lengths [rows] and reference counts [pages], one int32 buffer."""
    flat = torch.full((rows * width + rows + pages,), -1, dtype=torch.int32)
    view = flat[:rows * width].view(rows, width)
    view.copy_(torch.as_tensor(np.ascontiguousarray(table), dtype=torch.int32))
    flat[rows * width:rows * width + rows] = torch.as_tensor(np.asarray(lengths), dtype=torch.int32)
    used = view[view >= 0].long()
    flat[rows * width + rows:] = torch.bincount(used, minlength=pages).int()
    return flat.cuda()


def _handle(s, rows, width, pages):
    """Views of the metadata, a copy of it to go back to, and the cache's handle a serving program keeps."""
    flat = s["meta"]
    s["table"] = flat[:rows * width].view(rows, width)
    s["lengths"] = flat[rows * width:rows * width + rows]
    s["refs"] = flat[rows * width + rows:]
    s["saved"] = flat.clone()
    if own:
        if _PKG not in sys.path:
            sys.path.insert(0, _PKG)
        from hy_nomas_b200 import paged
        s["cache"] = paged.KVCache.over(s["k"], s["v"], s["ks"], s["vs"], s["meta"], rows, width)
    return s


def prepare(c, seed):
    gen, rnd = _gen(seed), np.random.default_rng(seed)
    op = c["op"]
    if op == "norm":
        # a residual stream of a few units with a few large channels, and a sublayer's smaller output
        loud = torch.where(torch.rand(c["dim"], generator=gen, device="cuda") < 0.01, 12.0, 1.0)
        s = {"x": _randn((c["rows"], c["dim"]), gen, 0.5), "r": (torch.randn((c["rows"], c["dim"]), generator=gen,
             device="cuda") * loud).to(torch.bfloat16), "w": (1 + 0.2 * torch.randn(c["dim"], generator=gen,
             device="cuda")).to(torch.bfloat16)}
        if own:
            if _PKG not in sys.path:
                sys.path.insert(0, _PKG)
            from hy_nomas_b200 import fused
            s["call"] = fused.add_rmsnorm_quant
        return {**s, "case": c}
    if op == "append":
        b, n, h, page = c["batch"], c["tokens"], c["heads"], c["page"]
        lens = [max(n, c["start"] + n - (i * 13) % (c["start"] + 1)) for i in range(b)]
        width = max(-(-x // page) for x in lens)
        pages = b * width + 2
        ids = rnd.permutation(pages)[:b * width].reshape(b, width)
        table = np.where(np.arange(width)[None] * page < np.array(lens)[:, None], ids, -1)
        s = _pool(1, pages, h, page, c["kind"], gen)
        s["meta"] = _meta(b, width, pages, table, lens)
        packed = _randn((b, n, 3 * h, D), gen)        # the projection's q | k | v
        s.update(nk=packed[:, :, h:2 * h], nv=packed[:, :, 2 * h:], rows=torch.arange(b, dtype=torch.int32, device="cuda"))
        return {**_handle(s, b, width, pages), "case": c}
    if op == "fork":
        lens, page, each = _fork_lengths(c), c["page"], c["each"]
        width = -(-max(lens) // page) + 1
        rows = len(lens) * (each + 1)
        held = sum(-(-x // page) for x in lens)
        pages = held + len(lens) * each + 3
        ids = iter(rnd.permutation(pages))
        table, order = np.full((rows, width), -1), rnd.permutation(rows)
        length = np.zeros(rows, int)
        parent, child = order[:len(lens)], order[len(lens):]
        for r, x in zip(parent, lens):
            table[r, :-(-x // page)] = [next(ids) for _ in range(-(-x // page))]
            length[r] = x
        # the children still hold the branches of the step before: all but the tails of another parent's pages
        for i, r in enumerate(child):
            p = (i // each + 1) % len(lens)
            full = lens[p] // page
            table[r, :full] = table[parent[p], :full]
            length[r] = full * page
        s = _pool(c["layers"], pages, c["heads"], page, c["kind"], gen)
        s["meta"] = _meta(rows, width, pages, table, length)
        s.update(parents=torch.tensor(np.repeat(parent, each), dtype=torch.int32, device="cuda"),
                 children=torch.tensor(child, dtype=torch.int32, device="cuda"))
        return {**_handle(s, rows, width, pages), "case": c}
    if op == "compact":
        pages, live, moves, rows, page = c["pages"], c["live"], c["moves"], c["rows"], c["page"]
        low = rnd.permutation(live)[:live - moves]
        high = live + rnd.permutation(pages - live)[:moves]
        used = rnd.permutation(np.concatenate([low, high]))
        share = used[:max(1, live // 8)]              # pages that every sequence starts with
        rest = np.array_split(used[len(share):], rows)
        width = len(share) + max(len(r) for r in rest)
        table, length = np.full((rows, width), -1), np.zeros(rows, int)
        for i, r in enumerate(rest):
            mine = np.concatenate([share, r])
            table[i, :len(mine)] = mine
            length[i] = len(mine) * page - i % page
        s = _pool(c["layers"], pages, c["heads"], page, c["kind"], gen)
        s["meta"] = _meta(rows, width, pages, table, length)
        return {**_handle(s, rows, width, pages), "case": c}
    b, page, shared, lens = c["batch"], c["page"], c["shared"], _lengths(c)
    first = shared // page
    width = first + max(-(-(x - shared) // page) for x in lens)
    pages = first + sum(-(-(x - shared) // page) for x in lens) + 2
    ids = rnd.permutation(pages)
    table = np.full((b, width), -1)
    table[:, :first] = ids[:first]
    at = first
    for i, x in enumerate(lens):
        mine = -(-(x - shared) // page)
        table[i, first:first + mine] = ids[at:at + mine]
        at += mine
    s = _pool(1, pages, c["kv"], page, c["kind"], gen)
    s["meta"] = _meta(b, width, pages, table, lens)
    q = torch.randn((b, c["lq"], c["heads"], D), generator=gen, device="cuda")
    s["q"] = (q * torch.rsqrt(q.square().mean(-1, keepdim=True)) * 1.5).to(torch.bfloat16)
    s["rows"] = torch.arange(b, dtype=torch.int32, device="cuda")
    return {**_handle(s, b, width, pages), "case": c}


# --------------------------------------------------------------------------------------------------- passes

def run(s):
    c = s["case"]
    if own:
        return _run_own(s, c)
    return {"norm": _norm, "append": _append, "fork": _fork, "compact": _compact, "attention": _attention}[c["op"]](s, c)


def _run_own(s, c):
    op = c["op"]
    if op == "norm":
        total, codes, scales = s["call"](s["x"], s["r"], s["w"], eps=EPS, kind=c["kind"], per_token=c["per_token"])
        return {"sum": total, "codes": _values(codes, scales), "scales": scales}
    cache = s["cache"]
    if op == "append":
        cache.append(0, s["nk"], s["nv"], s["rows"])
        if c["kind"] == "int8":
            from hy_nomas_b200.world import dequantize_kv
            return {"k": dequantize_kv(cache.k, cache.k_scale), "v": dequantize_kv(cache.v, cache.v_scale),
                    "ks": cache.k_scale, "vs": cache.v_scale}
        return {"k": cache.k, "v": cache.v}
    if op == "fork":
        cache.restore(s["saved"])
        cache.free(s["children"])
        cache.fork(s["parents"], s["children"])
        return _whole(s)
    if op == "compact":
        cache.restore(s["saved"])
        cache.compact()
        return _whole(s)
    from hy_nomas_b200 import paged
    return paged.attention(s["q"], cache, 0, s["rows"], shared=c["shared"], causal=c["causal"])


def _values(codes, scales):
    """int8 codes as the values they stand for; e4m3 codes are numbers of their own."""
    if codes.dtype != torch.int8:
        return codes
    n, d = codes.shape
    out = torch.empty((n, scales.shape[1], d // scales.shape[1]), device="cuda", dtype=torch.bfloat16)
    return torch.mul(codes.view(out.shape), scales[..., None], out=out).view(n, d)


def _whole(s):
    out = {m: s[m] for m in ("k", "v", "table", "lengths", "refs")}
    if s["ks"] is not None:
        out.update(ks=s["ks"], vs=s["vs"])
    return out


def _norm(s, c):
    n, d = c["rows"], c["dim"]
    h = s["x"].float() + s["r"].float()
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * s["w"].float()
    y = y.view(n, 1 if c["per_token"] else d // 128, -1)
    peak = y.abs().amax(-1)
    if c["kind"] == "fp8":
        scales = peak.clamp_min(1e-12) / 448
        codes = (y / scales[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(n, d)
    else:
        scales = torch.where(peak > 0, peak / 127, torch.ones_like(peak))
        q = y / scales[..., None]
        codes = torch.trunc(q + torch.copysign(torch.full_like(q, 0.5), q)).clamp(-127, 127).to(torch.int8).view(n, d)
    return {"sum": h.to(torch.bfloat16), "codes": _values(codes, scales), "scales": scales}


def _slots(s, n):
    """(page id, place in the page) of the last n tokens of every listed row."""
    rows = s["rows"].long()
    at = s["lengths"][rows].long()[:, None] - n + torch.arange(n, device="cuda")
    return s["table"][rows[:, None], at // s["page"]].long(), at % s["page"]


def _append(s, c):
    ids, place = _slots(s, c["tokens"])
    if c["kind"] == "bf16":
        s["k"][0, ids, :, place] = s["nk"]
        s["v"][0, ids, :, place] = s["nv"]
        return {"k": s["k"], "v": s["v"]}
    for pool, scale, new in (("k", "ks", "nk"), ("v", "vs", "nv")):
        codes, sc = _quantize(s[new])
        s[pool][0, ids, :, place] = codes
        s[scale][0, ids, :, place] = sc
    return {"k": (s["k"].float() * s["ks"][..., None]).to(torch.bfloat16),
            "v": (s["v"].float() * s["vs"][..., None]).to(torch.bfloat16), "ks": s["ks"], "vs": s["vs"]}


def _count(s, ids, valid, step):
    s["refs"].index_add_(0, torch.where(valid, ids, 0).reshape(-1).long(), (valid.int() * step).reshape(-1))


def _fork(s, c):
    s["meta"].copy_(s["saved"])
    table, lengths, refs, page = s["table"], s["lengths"], s["refs"], s["page"]
    parents, children = s["parents"].long(), s["children"].long()
    old = table[children]
    _count(s, old, old >= 0, -1)
    table[children] = -1
    lengths[children] = 0
    length, rows = lengths[parents].long(), table[parents]
    full, rest = length // page, length % page
    need = rest > 0
    free = torch.argsort((refs != 0).int(), stable=True)
    new = free[torch.cumsum(need, 0) - need.long()].int()
    col = torch.arange(rows.shape[1], device="cuda")
    kept = col < full[:, None]
    table[children] = torch.where(kept, rows, torch.where((col == full[:, None]) & need[:, None], new[:, None], -1))
    lengths[children] = length.int()
    _count(s, rows, kept, 1)
    _count(s, new, need, 1)
    tail = rows.gather(1, full.clamp(max=rows.shape[1] - 1)[:, None])[:, 0].long()
    src, dst, rest = tail[need], new.long()[need], rest[need]
    valid = torch.arange(page, device="cuda") < rest[:, None]
    wide = valid[None, :, None, :]
    s["k"][:, dst] = torch.where(wide[..., None], s["k"][:, src], s["k"][:, dst])
    s["v"][:, dst] = torch.where(wide[..., None], s["v"][:, src], s["v"][:, dst])
    if s["ks"] is not None:
        s["ks"][:, dst] = torch.where(wide, s["ks"][:, src], s["ks"][:, dst])
        s["vs"][:, dst] = torch.where(wide, s["vs"][:, src], s["vs"][:, dst])
    return _whole(s)


def _compact(s, c):
    s["meta"].copy_(s["saved"])
    table, refs = s["table"], s["refs"]
    live = refs > 0
    ids = torch.arange(refs.numel(), device="cuda")
    n = live.sum()
    src = ids[live & (ids >= n)]
    dst = ids[~live & (ids < n)]
    where = ids.clone()
    where[src] = dst
    table.copy_(torch.where(table >= 0, where[table.clamp(min=0).long()].int(), -1))
    refs[dst] = refs[src]
    refs[src] = 0
    s["k"][:, dst] = s["k"][:, src]
    s["v"][:, dst] = s["v"][:, src]
    if s["ks"] is not None:
        s["ks"][:, dst] = s["ks"][:, src]
        s["vs"][:, dst] = s["vs"][:, src]
    return _whole(s)


def _gather(pool, scale, ids):
    """Pages `ids` [..., n] of one layer as fp32 [..., heads, n * page, 128]; page ids below 0 give page 0."""
    at = ids.clamp(min=0).long()
    x = pool[0][at].float()
    if scale is not None:
        x = x * scale[0][at][..., None]
    x = x.transpose(-4, -3)
    return x.reshape(*x.shape[:-3], -1, D)


def _attention(s, c):
    b, lq, heads, kv, shared = c["batch"], c["lq"], c["heads"], c["kv"], c["shared"]
    first, rows = shared // s["page"], s["rows"].long()
    table, length = s["table"][rows], s["lengths"][rows].long()
    q = s["q"].float().view(b, lq, kv, heads // kv, D).permute(2, 0, 3, 1, 4).reshape(kv, b, -1, D)
    q = q * (1 / math.sqrt(D))
    own_k = _gather(s["k"], s["ks"], table[:, first:])
    logits = torch.matmul(q, own_k.transpose(0, 1).transpose(-1, -2))
    if shared:
        shared_k = _gather(s["k"], s["ks"], table[0, :first])
        front = torch.matmul(q.reshape(kv, -1, D), shared_k.transpose(-1, -2))
        logits = torch.cat([front.view(kv, b, -1, shared), logits], -1)
    limit = length[:, None].expand(b, lq)
    if c["causal"]:
        limit = limit - lq + torch.arange(1, lq + 1, device="cuda")
    limit = limit[:, None].expand(b, heads // kv, lq).reshape(b, -1, 1)
    logits.masked_fill_(torch.arange(logits.shape[-1], device="cuda") >= limit, -math.inf)
    top = logits.amax(-1, keepdim=True)
    p = logits.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    own_v = _gather(s["v"], s["vs"], table[:, first:])
    o = torch.matmul(p[..., shared:], own_v.transpose(0, 1))
    if shared:
        shared_v = _gather(s["v"], s["vs"], table[0, :first])
        o = o + torch.matmul(p[..., :shared].reshape(kv, -1, shared), shared_v).view(o.shape)
    o = torch.where(total > 0, o / total, 0.0)
    return o.view(kv, b, heads // kv, lq, D).permute(1, 3, 0, 2, 4).reshape(b, lq, heads, D).to(torch.bfloat16)


# --------------------------------------------------------------------------------------------------- 64 bits

def exact(c, seed):
    """The same outputs from the definitions in 64 bits. What a code stands for is given as the value before its
    rounding to 8 bits, so the distance of a code from it is that rounding's."""
    global own
    was, own = own, False
    try:
        s = prepare(c, seed)
    finally:
        own = was
    return {"norm": _exact_norm, "append": _exact_append, "fork": _exact_pages, "compact": _exact_pages,
            "attention": _exact_attention}[c["op"]](s, c)


def _exact_norm(s, c):
    h = s["x"].double() + s["r"].double()
    y = h / (h.pow(2).mean(1, keepdim=True) + EPS).sqrt() * s["w"].double()
    width = c["dim"] if c["per_token"] else 128
    groups = y.reshape(c["rows"], -1, width)
    peak = groups.abs().max(2).values
    if c["kind"] == "int8":
        scales = torch.where(peak > 0, peak / 127.0, 1.0)
        return {"sum": h, "codes": y, "scales": scales}
    scales = peak.clamp(min=1e-12) / 448.0
    return {"sum": h, "codes": (groups / scales.unsqueeze(2)).reshape(y.shape), "scales": scales}


def _stored(pool, scale):
    return pool.double() if scale is None else pool.double() * scale.double().unsqueeze(-1)


def _exact_append(s, c):
    out = {"k": _stored(s["k"], s["ks"]), "v": _stored(s["v"], s["vs"])}
    if s["ks"] is not None:
        out.update(ks=s["ks"].double(), vs=s["vs"].double())
    table, lengths, n, page = s["table"].cpu().numpy(), s["lengths"].cpu().numpy(), c["tokens"], c["page"]
    for b in range(c["batch"]):
        for block in range((lengths[b] - n) // page, (lengths[b] - 1) // page + 1):
            lo, hi = max(lengths[b] - n, block * page), min(lengths[b], (block + 1) * page)
            take = slice(int(lo - lengths[b] + n), int(hi - lengths[b] + n))
            put = slice(int(lo - block * page), int(hi - block * page))
            for name, new in (("k", s["nk"]), ("v", s["nv"])):
                x = new[b, take].double().transpose(0, 1)
                out[name][0, int(table[b, block]), :, put] = x
                if s["ks"] is not None:
                    peak = x.abs().max(2).values
                    out[name + "s"][0, int(table[b, block]), :, put] = torch.where(peak > 0, peak / 127.0, 1.0)
    return out


def _exact_pages(s, c):
    table, lengths, refs = (s[m].cpu().numpy().copy() for m in ("table", "lengths", "refs"))
    page, copies = c["page"], []
    if c["op"] == "fork":
        parents, children = s["parents"].tolist(), s["children"].tolist()
        for r in children:
            for p in table[r][table[r] >= 0]:
                refs[p] -= 1
            table[r], lengths[r] = -1, 0
        free = iter([p for p in range(len(refs)) if refs[p] == 0])
        for a, r in zip(parents, children):
            full, rest = divmod(int(lengths[a]), page)
            for j in range(full):
                table[r, j] = table[a, j]
                refs[table[a, j]] += 1
            if rest:
                new = next(free)
                copies.append((int(table[a, full]), new, rest))
                table[r, full] = new
                refs[new] = 1
            lengths[r] = lengths[a]
    else:
        live = int((refs > 0).sum())
        holes = [p for p in range(live) if refs[p] == 0]
        for a, to in zip([p for p in range(live, len(refs)) if refs[p] > 0], holes):
            table[table == a] = to
            refs[to], refs[a] = refs[a], 0
            copies.append((a, to, page))
    out = {m: s[m].double() for m in ("k", "v", "ks", "vs") if s[m] is not None and s[m].is_floating_point()}
    for m in ("k", "v"):
        if s["ks"] is not None:
            out[m] = s[m].clone()
    for a, to, n in copies:
        for m in out.values():
            m[:, to, :, :n] = m[:, a, :, :n]
    return {**out, "table": table, "lengths": lengths, "refs": refs}


def _exact_attention(s, c):
    out = torch.zeros((c["batch"], c["lq"], c["heads"], D), dtype=torch.float64, device="cuda")
    group = c["heads"] // c["kv"]
    for b, n in enumerate(_lengths(c)):
        if n == 0:
            continue
        ids = s["table"][b, :-(-n // c["page"])].long()
        for h in range(c["kv"]):
            k, v = (_stored(s[m][0, ids, h], None if s[m + "s"] is None else s[m + "s"][0, ids, h]).reshape(-1, D)[:n]
                    for m in ("k", "v"))
            q = s["q"][b, :, h * group:(h + 1) * group].double()
            logits = torch.einsum("qgd,kd->gqk", q, k) / math.sqrt(D)
            if c["causal"]:
                last = n - c["lq"] + torch.arange(c["lq"], device="cuda")
                hidden = torch.arange(n, device="cuda")[None] > last[:, None]
                logits = logits.masked_fill(hidden, -math.inf)
                weight = torch.softmax(logits, -1).nan_to_num(0.0)
            else:
                weight = torch.softmax(logits, -1)
            out[b, :, h * group:(h + 1) * group] = torch.einsum("gqk,kd->qgd", weight, v)
    return out
