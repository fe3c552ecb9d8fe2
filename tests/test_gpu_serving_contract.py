"""What the paged cache and its attention promise where a call meets a limit: rows without room, rows listed twice, shared parts
that nobody holds, numbers that are not finite, views that overlap. The bounds of attention are test_gpu_paged's."""
import ctypes
import math

import pytest
import torch

from test_gpu_paged import D, Model, bits, check_attention, filled, place

pytestmark = pytest.mark.gpu


@pytest.fixture()
def paged(hn):
    from hy_nomas_b200 import paged
    return paged


def tokens(b, n, heads, device, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)
    return [torch.randn((b, n, heads, D), generator=g, device=device).to(torch.bfloat16) for _ in range(2)]


# ------------------------------------------------------------------------------------- append without room

@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_append_after_a_refused_extend_writes_nothing(paged, hn, cuda, kind):
    """No page is left: two branches of a whole-page history, and a row on pages of its own, keep every byte."""
    c = filled(paged, 2, 6, 2, 16, 4, 8, kind, seed=1)
    c.extend([0], 32)
    c.fork([0, 0], [1, 2])
    c.extend([3], 64)
    m = Model(c)
    c.extend([1, 2], 1)
    m.extend([1, 2], 1)
    k, v = tokens(2, 1, 2, cuda)
    for layer in range(2):
        c.append(layer, k, v, [1, 2])
    c.extend([3], 16)
    m.extend([3], 16)
    k, v = tokens(1, 16, 2, cuda)
    c.append(0, k, v, [3])
    m.failed += 2 * 2 * 2 + 16 * 2
    assert m.failed == 3 + 40
    m.same_as(c)
    with pytest.raises(RuntimeError, match="could not be met"):
        c.check()
    # room again: the row that is extended is written, the other still is not
    c.free([3])
    c.extend([1], 1)
    page, before = int(c.table[1, 2]), c.k.clone()
    k, v = tokens(2, 1, 2, cuda, 1)
    c.append(1, k, v, [1, 2])
    assert int(c.failed) == 2
    if kind == "bf16":
        before[1, page, :, 0] = k[0, 0]
    else:
        before[1, page, :, 0] = hn.world.quantize_kv(k[0])[0][0]
    assert torch.equal(bits(c.k), bits(before))


def test_append_goes_on_after_free_fork_and_restore(paged, cuda):
    """A refusal ends with the row's next extend, free or fork, and with a table that is put back."""
    c = filled(paged, 1, 3, 1, 16, 3, 4, "bf16", seed=2)
    c.extend([0], 20)
    saved = c.save()
    k, v = tokens(1, 1, 1, cuda)

    def refuse():
        c.extend([0], 40)
        c.append(0, k, v, [0])
        with pytest.raises(RuntimeError, match="could not be met"):
            c.check()
    refuse()
    c.extend([0], 0)
    c.append(0, k, v, [0])
    c.check()
    refuse()
    c.restore(saved)
    c.append(0, k, v, [0])
    c.check()
    refuse()
    c.fork([0], [1])
    c.append(0, k, v, [1])
    c.check()
    c.free([0, 1])
    c.extend([2], 40)
    c.extend([1], 16)                                    # refused: row 1 is empty, the pool is not
    assert int(c.failed) == 1
    c.failed.zero_()
    c.free([2])
    c.extend([0], 5)
    c.fork([0], [1])                                     # a child that was refused while it was empty
    c.append(0, k, v, [1])
    c.check()


def test_append_leaves_shared_pages_alone(paged, cuda):
    """Without an extend the last tokens of a branch of whole pages are its parent's as well."""
    c = filled(paged, 1, 4, 2, 16, 3, 4, "bf16", seed=3)
    c.extend([0], 32)
    c.fork([0], [1])
    m = Model(c)
    k, v = tokens(1, 3, 2, cuda)
    c.append(0, k, v, [1])
    m.failed = 6
    m.same_as(c)
    c.free([1])
    c.append(0, k, v, [0])                               # its own again
    assert torch.equal(c.k[0, int(c.table[0, 1]), :, 13:].transpose(0, 1), k[0])


@pytest.mark.parametrize("n,b", [(1, 3), (40, 70)])
def test_append_takes_a_row_once(paged, cuda, n, b):
    """A row listed again: the first listing is written, the others are counted."""
    c = filled(paged, 1, 2 * b * -(-n // 16) + 2, 2, 16, b, -(-n // 16) + 1, "bf16", seed=4)
    rows = list(range(b))
    c.extend(rows, n)
    listed = rows + [b - 1, 0]
    k, v = tokens(b + 2, n, 2, cuda)
    c.append(0, k, v, listed)
    assert int(c.failed) == 2 * n * 2
    c.failed.zero_()
    for r in rows:
        pos = torch.arange(n, device=cuda)
        assert torch.equal(c.v[0, c.table[r][pos // 16].long(), :, pos % 16], v[r])


# ------------------------------------------------------------------------------------------- what extend and fork hand out

def test_extend_serves_in_order_up_to_the_first_shortage(paged, cuda):
    """A request that does not find its pages ends the call for those after it, whatever they need; listed first, they are met."""
    c = filled(paged, 1, 4, 1, 16, 4, 8, "bf16", seed=5)
    for row, n in ((1, 15), (2, 1), (3, 16)):
        c.extend([row], n)

    def state(failed, lengths):
        assert int(c.failed) == failed and c.lengths.tolist() == lengths
        c.failed.zero_()
    c.extend([0, 1], 17)                                 # two pages and one, of one
    state(2, [0, 15, 1, 16])
    c.extend([1, 0], 17)
    state(1, [0, 32, 1, 16])
    c.extend([3, 2], 15)                                 # one page and none, of none
    state(2, [0, 32, 1, 16])
    c.extend([2, 3], 15)
    state(1, [0, 32, 16, 16])


def test_extend_counts_pages_past_31_bits(paged, cuda):
    """1024 rows that want 2^22 pages each, of a pool of four."""
    c = paged.KVCache(1, 4, 1, 16, 1024, 1 << 22)
    c.extend(torch.arange(1024, dtype=torch.int32, device=cuda), 1 << 26)
    assert int(c.failed) == 1024 and int(c.refs.sum()) == 0 and int(c.lengths.abs().sum()) == 0
    assert int(c.table[:, :4].max()) == -1


def test_fork_of_a_broken_parent_takes_no_page(paged, cuda):
    """A parent whose last page is not there is refused; the page it would have taken goes to the next request."""
    c = filled(paged, 1, 3, 1, 16, 4, 2, "bf16", seed=6)
    c.extend([0], 5)
    c.extend([1], 5)
    c.table[0, 0] = -1
    c.fork([0, 1], [2, 3])
    assert int(c.failed) == 1 and c.lengths.tolist() == [5, 5, 0, 5]
    assert int(c.table[3, 0]) == 2


def test_ids_past_32_bits_are_out_of_range(paged, cuda):
    """64-bit ids are not taken modulo 2^32: row 2^32 is not row 0."""
    c = filled(paged, 1, 4, 1, 16, 2, 2, "bf16", seed=7)
    c.extend([0], 20)
    m = Model(c)
    c.free(torch.tensor([1 << 32, -(1 << 32), (1 << 40) + 1], device=cuda))
    m.failed = 3
    m.same_as(c)


# ------------------------------------------------------------------------------------------- shared parts

@pytest.mark.parametrize("heads", [4, 64])
@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_shared_part_that_nobody_holds_in_full(paged, cuda, kind, heads):
    """Three rows of 0, 20 and 37 tokens with 128 declared as shared: NaN past their ends, in every free page and in what an
    earlier call left in shared memory reaches nobody (64 heads on one: three tiles of 64 rows)."""
    c = filled(paged, 1, 40, 1, 16, 6, 12, kind, seed=8)
    q = torch.randn((3, 1, heads, D), device=cuda).to(torch.bfloat16)
    pools = [c.k, c.v] if kind == "bf16" else [c.k_scale, c.v_scale]
    kept = [t.clone() for t in pools]
    c.extend([0], 160)
    for t in pools:
        t.fill_(math.nan)
    paged.attention(q, c, 0, [0, 0, 0], shared=128)
    for t, was in zip(pools, kept):
        t.copy_(was)
    c.free([0])
    c.extend([1], 37)
    c.table[2, :2] = c.table[1, :2]
    c.lengths[2] = 20
    hidden = torch.ones(c.pages, c.page, dtype=torch.bool, device=cuda)
    pos = torch.arange(37, device=cuda)
    hidden[c.table[1][pos // 16].long(), pos % 16] = False
    for t in pools:
        t[hidden[None, :, None, :].expand(1, c.pages, 1, 16)] = math.nan
    for rows in ([1, 2, 3], [3, 2, 1]):
        for causal in (True, False):
            out, lse = paged.attention(q, c, 0, rows, shared=128, causal=causal, return_lse=True)
            check_attention(c, 0, q, rows, out, lse, causal, 1 / math.sqrt(D))


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("rows,shared,own", [(72, 8192, [5, 0, 40]), (100, 8256, [64, 1, 130, 0]), (128, 8704, [9] * 4)])
def test_long_shared_part_of_half_a_tile(paged, cuda, kind, rows, shared, own):
    """65 to 128 rows over 8192 shared tokens and more."""
    b = len(own)
    heads, kv = rows // b, 1
    lens = [shared + n for n in own]
    c = filled(paged, 1, shared // 64 + sum(-(-n // 64) for n in own) + 2, kv, 64, b, -(-max(lens) // 64) + 1, kind, seed=9)
    place(c, lens, seed=10, shared=shared)
    q = torch.randn((b, 1, heads, D), device=cuda).to(torch.bfloat16)
    out, lse = paged.attention(q, c, 0, list(range(b)), shared=shared, return_lse=True)
    check_attention(c, 0, q, list(range(b)), out, lse, True, 1 / math.sqrt(D))


@pytest.mark.parametrize("heads", [4, 64])
@pytest.mark.parametrize("shared", [0, 64])
@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_tokens_without_a_page_are_zeros(paged, cuda, kind, heads, shared):
    """Ids out of range in a table: as if the page held zeros, whatever shared memory held before."""
    c = filled(paged, 1, 40, 1, 16, 3, 12, kind, seed=31)
    place(c, [150, 131], seed=32, shared=shared)
    q = torch.randn((2, 1, heads, D), device=cuda).to(torch.bfloat16)
    pools = [c.k, c.v] if kind == "bf16" else [c.k_scale, c.v_scale]
    kept = [t.clone() for t in pools]
    for t in pools:
        t.fill_(math.nan)
    paged.attention(q, c, 0, [0, 1], shared=shared)
    for t, was in zip(pools, kept):
        t.copy_(was)
    zero = next(p for p in range(c.pages) if int(c.refs[p]) == 0)
    c.k[:, zero], c.v[:, zero] = 0, 0
    if kind == "int8":
        c.k_scale[:, zero], c.v_scale[:, zero] = 0, 0
    gone = ((0, 1, -1), (0, 6, 1 << 30), (1, 1, -1), (1, 8, c.pages))
    for r, j, bad in gone:
        c.table[r, j] = zero
    want = paged.attention(q, c, 0, [0, 1], shared=shared)
    for r, j, bad in gone:
        c.table[r, j] = bad
    got = paged.attention(q, c, 0, [0, 1], shared=shared)
    assert torch.equal(bits(got), bits(want))


# ... and on the tensor cores, which a shared part reaches by K/V heads x tokens x tiles of 64 rows

def on_tensor_cores(hn, c, b, lq, heads, shared):
    """By the call's workspace: a partial result of 256 rows for every SM and tile of the shared part."""
    n = ctypes.c_int64()
    assert hn.lib.lib.hn_paged_attention_workspace(c._ref, b, lq, heads, shared, 1, ctypes.byref(n)) == 0
    return n.value >= (hn.lib.lib.hn_num_sms() + c.heads * -(-b * lq * heads // c.heads // 256)) * 256 * 130 * 4


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("kv,group,lq,shared,page,own", [
    (16, 24, 1, 6144, 64, [5, 0, 40]),                   # 72 rows: a tile a quarter full
    (16, 32, 1, 6144, 128, [64, 1, 130, 7]),             # 128
    (8, 32, 2, 2048, 16, [2, 0, 1, 77] * 3 + [130]),     # 832 rows in four tiles
    (4, 7, 9, 4096, 32, [9, 500, 3, 31] * 3),            # 756, not whole groups
])
def test_shared_part_on_the_tensor_cores(paged, hn, cuda, kind, kv, group, lq, shared, page, own):
    b, lens = len(own), [shared + n for n in own]
    c = filled(paged, 1, shared // page + sum(-(-n // page) for n in own) + 2, kv, page, b, -(-max(lens) // page) + 1, kind, seed=22)
    place(c, lens, seed=23, shared=shared)
    assert on_tensor_cores(hn, c, b, lq, kv * group, shared)
    q = torch.randn((b, lq, kv * group, D), device=cuda).to(torch.bfloat16)
    rows = list(range(b))[::-1]
    for causal in (True, False):
        out, lse = paged.attention(q, c, 0, rows, shared=shared, causal=causal, return_lse=True)
        check_attention(c, 0, q, rows, out, lse, causal, 1 / math.sqrt(D))


@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_shared_part_on_the_tensor_cores_that_nobody_holds(paged, hn, cuda, kind):
    """As above: 13 sequences of 0 to 333 tokens with 2048 declared as shared, NaN wherever no row has a token."""
    b, kv, group, shared = 13, 8, 64, 2048
    c = filled(paged, 1, 150, kv, 16, b + 1, 130, kind, seed=24)
    assert on_tensor_cores(hn, c, b, 1, kv * group, shared)
    q = torch.randn((b, 1, kv * group, D), device=cuda).to(torch.bfloat16)
    pools = [c.k, c.v] if kind == "bf16" else [c.k_scale, c.v_scale]
    kept = [t.clone() for t in pools]
    c.extend([0], 2048)
    for t in pools:
        t.fill_(math.nan)
    paged.attention(q, c, 0, [0] * b, shared=shared)     # what is left in shared memory
    for t, was in zip(pools, kept):
        t.copy_(was)
    c.free([0])
    c.extend([4], 333)
    for i in range(1, b):
        if i != 4:
            c.table[i] = c.table[4]
            c.lengths[i] = 27 * (i - 1)
    hidden = torch.ones(c.pages, c.page, dtype=torch.bool, device=cuda)
    pos = torch.arange(333, device=cuda)
    hidden[c.table[4][pos // 16].long(), pos % 16] = False
    for t in pools:
        t[hidden[None, :, None, :].expand(1, c.pages, kv, 16)] = math.nan
    for rows in (list(range(b)), list(range(b))[::-1]):
        out, lse = paged.attention(q, c, 0, rows, shared=shared, return_lse=True)
        check_attention(c, 0, q, rows, out, lse, True, 1 / math.sqrt(D))
    c.table[4, 3], c.table[4, 18] = -1, 1 << 30          # ids out of range: zeros
    got = paged.attention(q, c, 0, [4] * b, shared=shared)
    zero = int((c.refs == 0).nonzero()[0])
    for t in (c.k, c.v, c.k_scale, c.v_scale):
        if t is not None:
            t[:, zero] = 0
    c.table[4, 3], c.table[4, 18] = zero, zero
    assert torch.equal(bits(got), bits(paged.attention(q, c, 0, [4] * b, shared=shared)))


# ------------------------------------------------------------------------------------------- scales, NaN, infinity

@pytest.mark.parametrize("lq", [1, 130])
@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_negative_scale(paged, cuda, kind, lq):
    c = filled(paged, 1, 40, 2, 16, 2, 12, kind, seed=11)
    place(c, [150, 131], seed=12)
    q = torch.randn((2, lq, 4, D), device=cuda).to(torch.bfloat16)
    for scale in (-0.2, -1e-3, 0.0):
        out, lse = paged.attention(q, c, 0, [0, 1], scale=scale, return_lse=True)
        check_attention(c, 0, q, [0, 1], out, lse, True, scale)


@pytest.mark.parametrize("scale", [math.nan, math.inf, -math.inf])
def test_a_scale_that_is_no_number_is_refused(paged, cuda, scale):
    c = filled(paged, 1, 4, 1, 16, 1, 2, "bf16", seed=13)
    c.extend([0], 5)
    q = torch.zeros((1, 1, 2, D), dtype=torch.bfloat16, device=cuda)
    with pytest.raises((ValueError, RuntimeError), match="scale"):
        paged.attention(q, c, 0, [0], scale=scale)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_appended_nan_and_infinity_are_seen(paged, cuda, kind, bad):
    """One such number among a token's K or V: the queries that see the token give NaN, those of other sequences do not."""
    for which in (0, 1):
        c = filled(paged, 1, 8, 1, 16, 2, 4, kind, seed=14)
        c.extend([0, 1], 20)
        kv = tokens(2, 20, 1, cuda)
        kv[which][0, 7, 0, 33] = bad
        c.append(0, *kv, [0, 1])
        if kind == "int8":
            scale = (c.k_scale, c.v_scale)[which][0, int(c.table[0, 0]), 0, 7]
            assert not torch.isfinite(scale)
        for lq in (1, 3, 70):
            q = torch.ones((2, lq, 1, D), dtype=torch.bfloat16, device=cuda)
            out = paged.attention(q, c, 0, [0, 1], causal=False)
            if which == 0 and not (kind == "int8" or math.isnan(bad)):
                # an infinite logit: the softmax is that token's (+) or leaves it out (-)
                assert torch.isnan(out[0]).all() if bad > 0 else torch.isfinite(out[0]).all()
            else:
                assert torch.isnan(out[0]).any(-1).all() or (torch.isinf(out[0]).any(-1).all() and which == 1)
            assert torch.isfinite(out[1]).all()


@pytest.mark.parametrize("spread", [20, 40])
@pytest.mark.parametrize("lq", [3, 70, 300])
def test_v_scales_far_apart(paged, cuda, lq, spread):
    """int8 V scales 2^20 and 2^40 apart: large ones under keys of no weight, and in tokens that only the last query sees, take
    nothing from the other tokens' precision."""
    c = filled(paged, 1, 60, 1, 16, 1, 60, "int8", seed=15)
    n = 500
    place(c, [n], seed=16)
    q = torch.randn((1, lq, 2, D), device=cuda).to(torch.bfloat16)
    q[..., 0] = 20
    at = torch.tensor([3, 200, 201, 333, n - lq // 2, n - 1], device=cuda)
    ids = c.table[0][at // 16].long()
    c.k[0, ids, 0, at % 16, 0] = -127
    c.k_scale[0, ids, 0, at % 16] = 0.5
    c.v_scale[0, ids, 0, at % 16] *= 2.0 ** spread
    out, lse = paged.attention(q, c, 0, [0], return_lse=True)
    check_attention(c, 0, q, [0], out, lse, True, 1 / math.sqrt(D))


@pytest.mark.parametrize("lq", [3, 20, 60, 70, 300])
@pytest.mark.parametrize("kind,which", [("bf16", "k"), ("int8", "k"), ("int8", "v")])
def test_nan_stays_with_the_queries_that_see_it(paged, cuda, kind, which, lq):
    """NaN in a token's K, or in its int8 V scale, that only the last queries see: theirs is NaN, the earlier ones' bits are as without."""
    c = filled(paged, 1, 60, 1, 16, 1, 60, kind, seed=19)
    place(c, [500], seed=20)
    q = torch.randn((1, lq, 1, D), device=cuda).to(torch.bfloat16)
    clean = paged.attention(q, c, 0, [0])
    at = 500 - 1 - lq // 3
    pool = getattr(c, which) if kind == "bf16" else getattr(c, which + "_scale")
    pool[0, int(c.table[0, at // 16]), 0, at % 16] = math.nan
    out = paged.attention(q, c, 0, [0])
    first = lq - 1 - lq // 3
    assert torch.equal(bits(out[:, :first]), bits(clean[:, :first]))
    assert torch.isnan(out[:, first:]).all()


# ------------------------------------------------------------------------------------------- outputs, errors

def test_an_output_that_overlaps_itself_is_refused(paged, cuda):
    c = filled(paged, 1, 4, 2, 16, 2, 2, "bf16", seed=17)
    c.extend([0, 1], 20)
    q = torch.randn((2, 3, 2, D), device=cuda).to(torch.bfloat16)
    store = torch.zeros(4096, dtype=torch.bfloat16, device=cuda)
    for shape, stride in (((2, 3, 2, D), (0, 256, 128)), ((2, 3, 2, D), (768, 128, 128)), ((2, 3, 2, D), (128, 256, 128)),
                          ((2, 3, 2, D), (768, 256, 8))):
        with pytest.raises(RuntimeError, match="out"):
            paged.attention(q, c, 0, [0, 1], out=store.as_strided(shape, stride + (1,)))
    want = paged.attention(q, c, 0, [0, 1])
    for stride in ((128, 512, 256), (128, 256, 1536)):
        got = paged.attention(q, c, 0, [0, 1], out=store.as_strided((2, 3, 2, D), stride + (1,)))
        assert torch.equal(bits(got), bits(want))
    one = paged.attention(q[:1, 2:], c, 0, [0], out=store.as_strided((1, 1, 2, D), (0, 0, 128, 1)))
    assert torch.equal(bits(one), bits(want[:1, 2:]))


def test_check_reports_a_wait_that_ran_out(paged, hn, cuda):
    """The bounded waits of the tensor-core line record where they gave up; check() tells."""
    c = filled(paged, 1, 4, 1, 16, 1, 2, "bf16", seed=18)
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        with torch.cuda.stream(stream):
            assert hn.lib.lib.hn_selftest_wait_timeout(1000, hn.lib.stream_of(c.k)) == 0
            with pytest.raises(RuntimeError, match="wait"):
                c.check()
            c.check()
