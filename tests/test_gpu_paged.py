"""The paged K/V cache and the attention that reads it, against plain models: page operations against a Python
simulation (equal everywhere), attention against the definition in 64 bits.

Attention's bound per output element: the output is rounded once to bf16 (2^-8 |o|); P is rounded once before the P V
product, to bf16 (2^-8 of each term) for a bf16 cache and to fp16 (2^-11) for an int8 one, so its part is that times
A = sum p |v| / sum p; everything else is fp32 (products and sums of 128 terms, logits of at most a few hundred in
base 2: 2^-12 A covers it). For an int8 cache fp16 has a smallest step, 2^-24, and P' = p sv is scaled to at most 2^14:
2^-39 of the largest p sv, for each of n codes of at most 127.
"""
import ctypes
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
D = 128


@pytest.fixture()
def paged(hn):
    from hy_nomas_b200 import paged
    return paged


def bits(t):
    return t.contiguous().view(torch.int16 if t.element_size() == 2 else torch.int8 if t.element_size() == 1
                               else torch.int32)


def quantize(x):
    """world.quantize_kv's arithmetic in torch."""
    x = x.float()
    peak = x.abs().amax(-1, keepdim=True)
    s = torch.where(peak > 0, peak / 127, torch.ones_like(peak))
    y = x / s
    return torch.trunc(y + torch.copysign(torch.full_like(y, 0.5), y)).clamp(-127, 127).to(torch.int8), s[..., 0]


def filled(paged, layers, pages, heads, page, slots, width, kind, seed, device="cuda"):
    """A cache whose every page holds random numbers (int8: with random scales)."""
    g = torch.Generator(device=device).manual_seed(seed)
    c = paged.KVCache(layers, pages, heads, page, slots, width, kind)
    for pool, scale in ((c.k, c.k_scale), (c.v, c.v_scale)):
        x = torch.randn(pool.shape, generator=g, device=device)
        if kind == "bf16":
            pool.copy_(x)
        else:
            q, s = quantize(x * (0.5 + torch.rand(pool.shape[:4], generator=g, device=device))[..., None])
            pool.copy_(q)
            scale.copy_(s)
    return c


def place(c, lengths, seed, shared=0):
    """Give the rows 0.. their pages, at random ids; the first `shared` tokens of all on the same pages."""
    rnd = np.random.default_rng(seed)
    ids = iter(rnd.permutation(c.pages).tolist())
    table = np.full((c.slots, c.width), -1, np.int32)
    first = [next(ids) for _ in range(shared // c.page)]
    for r, n in enumerate(lengths):
        need = -(-n // c.page)
        mine = first[:need]
        table[r, :need] = mine + [next(ids) for _ in range(need - len(mine))]
    length = np.zeros(c.slots, np.int32)
    length[:len(lengths)] = lengths
    c.table.copy_(torch.from_numpy(table))
    c.lengths.copy_(torch.from_numpy(length))
    c.refs.copy_(torch.from_numpy(np.bincount(table[table >= 0], minlength=c.pages).astype(np.int32)))


def keys_of(c, layer, row, n, h):
    """K, V of one row and K/V head in 64 bits."""
    ids = c.table[row, :-(-n // c.page)].long()
    out = []
    for pool, scale in ((c.k, c.k_scale), (c.v, c.v_scale)):
        x = pool[layer, ids, h].double()
        if scale is not None:
            x = x * scale[layer, ids, h].double()[..., None]
        out.append(x.reshape(-1, D)[:n])
    return out


def check_attention(c, layer, q, rows, out, lse, causal, scale):
    b, lq, heads, _ = q.shape
    group = heads // c.heads
    lens = c.lengths.tolist()
    half_p = 2.0 ** -8 if c.kind == "bf16" else 2.0 ** -11
    for i, row in enumerate(rows):
        n = lens[row]
        limit = torch.full((lq,), n, device="cuda") if not causal else n - lq + torch.arange(1, lq + 1, device="cuda")
        for h in range(c.heads):
            hs = slice(h * group, (h + 1) * group)
            got, got_lse = out[i, :, hs].double(), lse[i, hs].double().T          # [lq, g]
            seen = limit > 0
            assert torch.equal(got[~seen], torch.zeros_like(got[~seen]))
            assert (got_lse[~seen] == -math.inf).all()
            if n == 0 or not seen.any():
                continue
            k, v = keys_of(c, layer, row, n, h)
            s = torch.einsum("qgd,kd->qgk", q[i, :, hs].double(), k) * scale
            s = s.masked_fill(torch.arange(n, device="cuda") >= limit[:, None, None], -math.inf)
            want_lse = torch.logsumexp(s, -1)
            p = torch.exp(s[seen] - want_lse[seen][..., None])
            want, a = p @ v, p @ v.abs()
            err = (got[seen] - want).abs()
            bound = 2.0 ** -8 * want.abs() + (half_p + 2.0 ** -12) * a + 1e-30
            if c.kind == "int8":
                sv = c.v_scale[layer, c.table[row, :-(-n // c.page)].long(), h].reshape(-1)[:n].double()
                bound = bound + 2.0 ** -39 * 127 * n * (p * sv).amax(-1, keepdim=True)
            assert (err <= bound).all(), (i, h, float((err / bound).max()))
            assert (got_lse[seen] - want_lse[seen]).abs().max() < 1e-3
    # (a lse error of 1e-3 is far above what fp32 logits of a few hundred leave, and far below any mistake in the mask)


CASES = [
    # lq, heads, kv, page, shared, own lengths, causal
    (1, 8, 8, 16, 0, [1], True),
    (1, 8, 2, 16, 0, [0, 5, 16, 17, 64, 65, 200], True),
    (1, 32, 8, 32, 320, [0, 1, 31, 32, 33, 100], True),
    (1, 7, 1, 64, 640, [3, 700], False),
    (3, 4, 4, 48, 96, [3, 50, 2], True),                     # a sequence shorter than its queries past the shared part
    (5, 16, 2, 16, 16, [5, 6, 1000], True),
    (4, 4, 2, 16, 0, [2, 4, 0], True),                       # queries before the first token: empty rows
    (17, 3, 3, 128, 256, [17, 130], False),
    (70, 6, 2, 32, 64, [70, 300], True),
    (130, 2, 1, 16, 0, [130, 131, 64], True),
    (200, 4, 4, 64, 192, [200, 257], False),
    (333, 2, 2, 16, 16, [40, 333], True),                    # more queries than tokens
    (1, 32, 8, 32, 1600, [9] * 20 + [0, 33, 200], True),     # 92 rows of all sequences on the shared part
    (2, 16, 2, 16, 112, [2, 30, 65, 9, 2, 100, 7], True),    # ... 112, and one block
    (1, 8, 1, 16, 0, [300] * 3, False),
    (16, 64, 8, 16, 0, [16, 77, 900], True),                 # 128 rows of one sequence
    (3, 32, 1, 48, 48 * 40, [3, 500], True),                 # 192 rows on the shared part, one head
]


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_attention_against_64_bits(paged, cuda, kind, case):
    lq, heads, kv, page, shared, own, causal = case
    lens = [shared + n for n in own]
    width = -(-max(lens + [1]) // page) + 2
    pages = shared // page + sum(-(-n // page) for n in own) + 3
    c = filled(paged, 2, pages, kv, page, len(lens) + 1, width, kind, seed=lq)
    place(c, lens, seed=lq + 1, shared=shared)
    g = torch.Generator(device=cuda).manual_seed(lq + 2)
    q = (torch.randn((len(lens), lq, heads, D), generator=g, device=cuda) * 1.5).to(torch.bfloat16)
    rows = list(range(len(lens)))[::-1]
    for scale in (None, 0.3):
        for use in sorted({0, shared}):
            out, lse = paged.attention(q, c, 1, rows, shared=use, causal=causal, scale=scale, return_lse=True)
            check_attention(c, 1, q, rows, out, lse, causal, 1 / math.sqrt(D) if scale is None else scale)
    again = paged.attention(q, c, 1, rows, shared=shared, causal=causal, scale=0.3)
    assert torch.equal(bits(again), bits(out)) if use == shared else True
    c.check()


@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_attention_many_sequences(paged, cuda, kind):
    """300 sequences of lengths 0 to 299 past a shared part of two pages: more sequences than a scan step holds."""
    n = 300
    c = filled(paged, 1, n * 19 + 2, 1, 16, n, 24, kind, seed=1)
    lens = [32 + i for i in range(n)]
    place(c, lens, seed=2, shared=32)
    q = torch.randn((n, 1, 2, D), device=cuda).to(torch.bfloat16)
    rows = list(range(n))
    out, lse = paged.attention(q, c, 0, rows, shared=32, return_lse=True)
    check_attention(c, 0, q, rows, out, lse, True, 1 / math.sqrt(D))


@pytest.mark.parametrize("heads", [4, 64])
@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_attention_with_freed_and_short_rows(paged, cuda, kind, heads):
    """Rows that were freed or hold less than the shared part, the first one listed too: the others are not touched by it (64
    heads on one K/V head: the shared part's rows fill a tensor-core tile)."""
    c = filled(paged, 1, 40, 1, 16, 6, 12, kind, seed=11)
    c.extend([0], 130)
    c.fork([0, 0, 0], [1, 2, 3])
    c.extend([1, 2, 3], 7)
    c.free([0])
    c.extend([0], 20)
    c.fork([0], [4])                                     # holds less than the shared part, on pages of its own
    c.free([0])
    c.table[4, :2] = c.table[1, :2]                      # ... or rather on the first of the shared ones
    q = torch.randn((6, 1, heads, D), device=cuda).to(torch.bfloat16)
    for rows in ([5, 0, 1, 2, 3, 4], [0, 5, 4, 3, 2, 1]):
        out, lse = paged.attention(q, c, 0, rows, shared=128, return_lse=True)
        check_attention(c, 0, q, rows, out, lse, True, 1 / math.sqrt(D))
    out, lse = paged.attention(q[:3], c, 0, [5, 4, 0], shared=128, return_lse=True)      # none holds it all
    check_attention(c, 0, q[:3], [5, 4, 0], out, lse, True, 1 / math.sqrt(D))


@pytest.mark.parametrize("lq", [1, 300])
@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_attention_ignores_what_no_query_may_see(paged, cuda, kind, lq):
    """NaN and infinity in the tokens past a sequence's end, in pages that no row names and in the rows not listed
    leave the result's bits as they are."""
    lens = [331, 320, 333]
    c = filled(paged, 1, 40, 2, 32, 4, 12, kind, seed=3)
    place(c, lens + [100], seed=4)
    q = torch.randn((3, lq, 4, D), device=cuda).to(torch.bfloat16)
    clean = paged.attention(q, c, 0, [0, 1, 2])
    seen = torch.zeros(c.pages, c.page, dtype=torch.bool, device=cuda)
    for r, n in enumerate(lens):
        pos = torch.arange(n, device=cuda)
        seen[c.table[r][pos // 32].long(), pos % 32] = True
    hidden = (~seen)[None, :, None, :].expand(1, c.pages, 2, 32)
    for pool, scale, bad in ((c.k, c.k_scale, math.nan), (c.v, c.v_scale, math.inf)):
        (pool if kind == "bf16" else scale)[hidden] = bad
    assert torch.equal(bits(paged.attention(q, c, 0, [0, 1, 2])), bits(clean))


@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_attention_sharp_and_extreme_logits(paged, cuda, kind):
    """Large q and k (the maximum moves by hundreds), tiny and huge scales, zero rows."""
    c = filled(paged, 1, 60, 1, 16, 2, 40, kind, seed=5)
    place(c, [500, 333], seed=6, shared=160)
    ramp = torch.linspace(0.01, 3, c.pages, device=cuda).view(1, -1, 1, 1)
    if kind == "bf16":
        c.k.mul_(ramp[..., None])
        c.v[:, 3:6] = 0
    else:
        c.k_scale.mul_(ramp)
        c.v_scale.mul_(10 ** (6 * (ramp - 1.5)))
        c.v[:, 3:6] = 0
        c.v_scale[:, 3:6] = 1
    q = (torch.randn((2, 3, 4, D), device=cuda) * 4).to(torch.bfloat16)
    out, lse = paged.attention(q, c, 0, [0, 1], shared=160, return_lse=True)
    check_attention(c, 0, q, [0, 1], out, lse, True, 1 / math.sqrt(D))
    q.mul_(1e-6)
    q[:, :, 1] = 0
    out, lse = paged.attention(q, c, 0, [0, 1], return_lse=True)
    check_attention(c, 0, q, [0, 1], out, lse, True, 1 / math.sqrt(D))


def test_attention_strided_views_and_streams(paged, cuda):
    """q inside a packed projection, out inside a wider buffer, and a call on another stream."""
    c = filled(paged, 1, 20, 2, 16, 2, 10, "bf16", seed=7)
    place(c, [100, 77], seed=8)
    packed = torch.randn((2, 9, 8, D), device=cuda).to(torch.bfloat16)
    q, wide = packed[:, :, 2:6], torch.full((2, 9, 6, D), 7.0, dtype=torch.bfloat16, device=cuda)
    want = paged.attention(q.contiguous(), c, 0, [0, 1])
    got = paged.attention(q, c, 0, [0, 1], out=wide[:, :, 1:5])
    assert torch.equal(bits(got), bits(want))
    assert (wide[:, :, 0] == 7).all() and (wide[:, :, 5] == 7).all()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = paged.attention(q, c, 0, torch.tensor([0, 1], device=cuda))
    s.synchronize()
    assert torch.equal(bits(other), bits(want))


def test_attention_offsets_past_32_bits(paged, cuda):
    """Pages whose byte offsets in the pool pass 2^32."""
    pages = 2 ** 32 // (32 * 64 * D * 2) * 2 + 8
    c = paged.KVCache(1, pages, 32, 64, 1, 4, "bf16")
    c.table[0, :3] = torch.tensor([pages - 1, 0, pages - 2], device=cuda)
    c.lengths[0] = 150
    for p in (pages - 1, 0, pages - 2):
        c.k[:, p] = torch.randn(c.k[:, p].shape, device=cuda)
        c.v[:, p] = torch.randn(c.v[:, p].shape, device=cuda)
    for lq in (1, 130):
        q = torch.randn((1, lq, 32, D), device=cuda).to(torch.bfloat16)
        out, lse = paged.attention(q, c, 0, [0], return_lse=True)
        check_attention(c, 0, q, [0], out, lse, True, 1 / math.sqrt(D))
    k, v = (torch.randn((1, 9, 32, D), device=cuda).to(torch.bfloat16) for _ in range(2))
    c.append(0, k, v, [0])
    at = torch.arange(141, 150, device=cuda)
    assert torch.equal(c.k[0, pages - 2, :, at % 64].transpose(0, 1), k[0])
    c.free([0])
    c.check()


def test_attention_takes_nothing(paged, cuda):
    c = filled(paged, 1, 4, 1, 16, 2, 2, "bf16", seed=1)
    assert paged.attention(torch.zeros((0, 1, 2, D), dtype=torch.bfloat16, device=cuda), c, 0, []).shape == (0, 1, 2, D)
    assert paged.attention(torch.zeros((2, 0, 2, D), dtype=torch.bfloat16, device=cuda), c, 0, [0, 1]).shape == (2, 0, 2, D)


# ------------------------------------------------------------------------------------------------ page operations

class Model:
    """The page operations on Python lists, ids lowest first."""

    def __init__(self, c):
        self.page, self.width, self.pages, self.slots = c.page, c.width, c.pages, c.slots
        self.table = c.table.cpu().numpy().copy()
        self.lengths = c.lengths.cpu().numpy().copy()
        self.refs = c.refs.cpu().numpy().copy()
        self.pools = [None if t is None else t.cpu().clone() for t in (c.k, c.v, c.k_scale, c.v_scale)]
        self.failed = 0

    def copy(self, src, dst, n):
        for t in self.pools:
            if t is not None:
                t[:, dst, :, :n] = t[:, src, :, :n]

    def extend(self, rows, tokens):
        free = [p for p in range(self.pages) if self.refs[p] == 0]
        at = 0
        for i, r in enumerate(rows):
            if not 0 <= r < self.slots or r in rows[:i]:
                self.failed += 1
                continue
            have, want = -(-self.lengths[r] // self.page), -(-(self.lengths[r] + tokens) // self.page)
            if want > self.width:
                self.failed += 1
                continue
            at += want - have
            if at > len(free):
                self.failed += 1
                continue
            for j, p in enumerate(free[at - (want - have):at]):
                self.table[r, have + j] = p
                self.refs[p] = 1
            self.lengths[r] += tokens

    def free(self, rows):
        for r in rows:
            if not 0 <= r < self.slots:
                self.failed += 1
                continue
            for p in self.table[r][self.table[r] >= 0]:
                self.refs[p] -= 1
            self.table[r], self.lengths[r] = -1, 0

    def fork(self, parents, children):
        free = [p for p in range(self.pages) if self.refs[p] == 0]
        at, was = 0, self.lengths.copy()
        for i, (a, r) in enumerate(zip(parents, children)):
            bad = not (0 <= a < self.slots and 0 <= r < self.slots) or r in children[:i] or a in children
            if bad or was[r] != 0:
                self.failed += 1
                continue
            full, rest = divmod(int(was[a]), self.page)
            if rest:
                at += 1
                if at > len(free):
                    self.failed += 1
                    continue
                self.copy(self.table[a, full], free[at - 1], rest)
                self.table[r, full] = free[at - 1]
                self.refs[free[at - 1]] = 1
            self.table[r, :full] = self.table[a, :full]
            for p in self.table[a, :full]:
                self.refs[p] += 1
            self.lengths[r] = was[a]

    def compact(self):
        live = int((self.refs > 0).sum())
        holes = [p for p in range(live) if self.refs[p] == 0]
        for s, d in zip([p for p in range(live, self.pages) if self.refs[p] > 0], holes):
            self.copy(s, d, self.page)
            self.table[self.table == s] = d
            self.refs[d], self.refs[s] = self.refs[s], 0

    def same_as(self, c):
        assert np.array_equal(self.table, c.table.cpu().numpy())
        assert np.array_equal(self.lengths, c.lengths.cpu().numpy())
        assert np.array_equal(self.refs, c.refs.cpu().numpy())
        assert self.failed == int(c.failed)
        for t, m in zip((c.k, c.v, c.k_scale, c.v_scale), self.pools):
            assert t is None or torch.equal(bits(t.cpu()), bits(m))
        used = self.table[self.table >= 0]
        assert np.array_equal(np.bincount(used, minlength=self.pages), self.refs)


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("pages,slots,width,page,heads", [(40, 9, 6, 16, 3), (3000, 1500, 4, 16, 1), (20, 6, 8, 48, 2)])
def test_page_operations_against_the_model(paged, cuda, kind, pages, slots, width, page, heads):
    """Random sequences of operations, with requests that cannot be met among them, equal the model's after each."""
    rnd = np.random.default_rng(pages)
    c = filled(paged, 2, pages, heads, page, slots, width, kind, seed=pages)
    m = Model(c)
    most = 1200 if slots > 1000 else slots
    for step in range(40):
        op = rnd.choice(["extend", "extend", "fork", "fork", "free", "compact"])
        n = int(rnd.integers(1, most + 1))
        if op == "extend":
            rows = rnd.integers(-1, slots + 1, n).tolist()
            tokens = int(rnd.integers(0, 2 * page + 2))
            c.extend(rows, tokens)
            m.extend(rows, tokens)
        elif op == "fork":
            order = rnd.permutation(slots)
            held, empty = order[m.lengths[order] > 0], order[m.lengths[order] == 0]
            if len(held) == 0 or len(empty) == 0:
                continue
            children = rnd.choice(empty, min(n, len(empty)), replace=step % 5 == 0).tolist()
            parents = rnd.choice(held, len(children)).tolist()
            if step % 7 == 0:
                children[-1], parents[0] = int(held[0]), slots
            c.fork(torch.tensor(parents, device=cuda), torch.tensor(children, device=cuda))
            m.fork(parents, children)
        elif op == "free":
            rows = rnd.integers(0, slots, max(1, n // 4)).tolist() + [-3] * (step % 3 == 0)
            c.free(rows)
            m.free(rows)
        else:
            c.compact()
            m.compact()
        m.same_as(c)
    if m.failed:
        with pytest.raises(RuntimeError, match="could not be met"):
            c.check()
    c.check()


def test_save_and_restore(paged, cuda):
    c = filled(paged, 1, 16, 1, 16, 4, 4, "bf16", seed=1)
    c.extend([0, 1], 20)
    saved = c.save()
    c.fork([0], [2])
    c.free([1])
    c.restore(saved)
    assert c.lengths.tolist() == [20, 20, 0, 0]
    with pytest.raises(ValueError):
        c.restore(saved[1:])


def test_copy_pages(paged, cuda):
    c = filled(paged, 3, 12, 2, 32, 1, 1, "int8", seed=2)
    m = Model(c)
    c.copy_pages([1, 5, 40], [0, 7, 2])                  # a page out of range is left out
    m.copy(1, 0, 32)
    m.copy(5, 7, 32)
    m.same_as(c)


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("n,heads,page", [(1, 1, 16), (1, 8, 64), (37, 5, 48), (500, 2, 16)])
def test_append_equals_the_framework_quantizer(paged, hn, cuda, kind, n, heads, page):
    """New tokens land in their places, equal to what they were (bf16) or to world.quantize_kv's codes and scales, from
    strided views; nothing else changes."""
    slots, width = 5, -(-(700 + n) // page)
    c = filled(paged, 2, slots * width, heads, page, slots, width, kind, seed=n)
    for r, start in enumerate([0, 3, page, page - 1, 2 * page + 5]):
        c.extend([r], start)
    rows = [4, 0, 2, 1]
    c.extend(rows, n)
    m = Model(c)
    packed = torch.randn((4, n, 3 * heads, D), device=cuda).to(torch.bfloat16)
    packed[0, 0, heads] = 0
    packed[-1, -1, -1, 0] = 1e4
    k, v = packed[:, :, heads:2 * heads], packed[:, :, 2 * heads:]
    c.append(1, k, v, rows)
    for i, r in enumerate(rows):
        pos = m.lengths[r] - n + np.arange(n)
        ids = torch.from_numpy(m.table[r][pos // page]).long()
        for x, pool, scale in ((k, 0, 2), (v, 1, 3)):
            if kind == "bf16":
                m.pools[pool][1, ids, :, torch.from_numpy(pos % page)] = x[i].cpu()
            else:
                q, s = hn.world.quantize_kv(x[i])
                m.pools[pool][1, ids, :, torch.from_numpy(pos % page)] = q.cpu()
                m.pools[scale][1, ids, :, torch.from_numpy(pos % page)] = s[..., 0].cpu()
    m.same_as(c)


def test_append_without_room_is_counted(paged, cuda):
    c = filled(paged, 1, 4, 1, 16, 2, 2, "bf16", seed=3)
    m = Model(c)
    x = torch.zeros((2, 3, 1, D), dtype=torch.bfloat16, device=cuda)
    c.append(0, x, x, [0, 9])                            # row 0 is empty, row 9 does not exist
    m.failed = 6
    m.same_as(c)


def test_branches_attend_like_copies(paged, cuda):
    """A parent forked to five branches that go their own ways: attention with the shared part read once equals, within
    the bound, attention over what each branch holds."""
    c = filled(paged, 1, 60, 2, 16, 8, 16, "int8", seed=9)
    c.extend([0], 100)
    k, v = (torch.randn((1, 100, 2, D), device=cuda).to(torch.bfloat16) for _ in range(2))
    c.append(0, k, v, [0])
    rows = [1, 2, 3, 4, 5]
    c.fork([0] * 5, rows)
    for step in range(20):
        c.extend(rows, 1)
        k, v = (torch.randn((5, 1, 2, D), device=cuda).to(torch.bfloat16) for _ in range(2))
        c.append(0, k, v, rows)
    q = torch.randn((5, 1, 8, D), device=cuda).to(torch.bfloat16)
    out, lse = paged.attention(q, c, 0, rows, shared=96, return_lse=True)
    check_attention(c, 0, q, rows, out, lse, True, 1 / math.sqrt(D))
    assert int((c.refs > 0).sum()) == 6 + 1 + 5 * 2
    c.free(rows)
    c.compact()
    assert c.refs.tolist()[:8] == [1] * 7 + [0]
    c.check()


def test_refusals(paged, cuda):
    with pytest.raises(ValueError):
        paged.KVCache(1, 4, 1, 24, 2, 2)
    with pytest.raises(ValueError):
        paged.KVCache(1, 4, 1, 16, 2, 2, kind="fp8")
    c = filled(paged, 1, 4, 2, 16, 2, 2, "bf16", seed=1)
    q = torch.zeros((1, 1, 4, D), dtype=torch.bfloat16, device=cuda)
    bad = [dict(q=q.half()), dict(q=q[..., :64]), dict(q=q[:, :, :3]), dict(rows=[0, 1]), dict(shared=8), dict(shared=48),
           dict(layer=1), dict(out=torch.empty(4, device=cuda)), dict(rows=torch.zeros(1, device=cuda)),
           dict(rows=torch.zeros(1, dtype=torch.int32)), dict(q=q.cpu())]
    for change in bad:
        a = dict(q=q, layer=0, rows=[0], shared=0)
        a.update(change)
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            paged.attention(a["q"], c, a["layer"], a["rows"], shared=a["shared"], out=a.get("out"))
    x = torch.zeros((1, 1, 2, D), dtype=torch.bfloat16, device=cuda)
    for args in ((0, x.half(), x, [0]), (0, x[:, :, :1], x[:, :, :1], [0]), (2, x, x, [0]), (0, x, x, [0, 1]), (0, x.cpu(), x, [0])):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            c.append(*args)
    with pytest.raises(ValueError):
        c.fork([0], [1, 1])
    with pytest.raises(ValueError):
        c.extend([0], -1)
    with pytest.raises(ValueError):
        c.copy_pages([0], [1, 1])
    with pytest.raises(TypeError):
        c.free(torch.zeros(1, device=cuda))
    c.check()
    from hy_nomas_b200 import _lib
    L = _lib.lib
    one = torch.zeros(1, dtype=torch.int32, device=cuda)
    st = _lib.stream_of(q)

    def attend(**kw):
        a = dict(layer=0, q=q.data_ptr(), qb=512, ql=512, qh=128, rows=one.data_ptr(), b=1, lq=1, h=4, d=128, shared=0,
                 causal=1, scale=0.1, out=q.data_ptr(), ob=512, ol=512, oh=128, lse=None, ws=q.data_ptr(), size=0)
        a.update(kw)
        return L.hn_paged_attention(c._ref, *a.values(), st)
    assert attend(d=64) == 7 and attend(layer=-1) == 1 and attend(q=None) == 5 and attend(ql=100) == 2
    assert attend(h=3) == 1 and attend(b=5000) == 1 and attend(causal=2) == 5 and attend() == 5    # no workspace
    assert b"workspace" in L.hn_last_error()
    n = ctypes.c_int64()
    assert L.hn_cache_workspace(c._ref, 5, ctypes.byref(n)) == 0 and n.value == max(2 + 4 + 20, 4 + 12)
    assert L.hn_cache_workspace(c._ref, -1, ctypes.byref(n)) == 5
