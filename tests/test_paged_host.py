"""Host checks of the paged cache, its attention and the residual + RMSNorm + quantizer, through the C ABI: bad arguments are
refused before a GPU is touched (CPU only; no pointer is ever followed)."""
import ctypes

import pytest
import torch

FAKE = 0x10000


def struct(paged, **kw):
    a = dict(k=FAKE, v=FAKE, k_scale=None, v_scale=None, table=FAKE, lengths=FAKE, refs=FAKE, failed=FAKE, layers=2, pages=100,
             heads=4, page=16, slots=8, width=10)
    a.update(kw)
    return paged._Struct(*a.values())


@pytest.fixture()
def paged(hn):
    from hy_nomas_b200 import paged
    return paged


def ref(s):
    return ctypes.addressof(s)


def test_cache_checks(hn, paged):
    L = hn.lib.lib
    n = ctypes.c_int64()
    ok = struct(paged)
    assert L.hn_cache_workspace(ref(ok), 3, ctypes.byref(n)) == 0 and n.value == 4 + 3 * 100
    assert L.hn_cache_workspace(ref(ok), 1000, ctypes.byref(n)) == 0 and n.value == 8 + 100 + 4000
    assert L.hn_cache_workspace(None, 3, ctypes.byref(n)) == 5
    assert L.hn_cache_workspace(ref(ok), -1, ctypes.byref(n)) == 5
    for change, code in ((dict(k=None), 5), (dict(refs=None), 5), (dict(k_scale=FAKE), 5), (dict(page=24), 1), (dict(page=0), 1),
                         (dict(pages=0), 1), (dict(width=1 << 40), 1), (dict(pages=1 << 30, heads=1 << 10), 1),
                         (dict(k=FAKE + 8), 2), (dict(slots=-1), 1)):
        bad = struct(paged, **change)
        assert L.hn_cache_workspace(ref(bad), 1, ctypes.byref(n)) == code, change
        assert b"hn_cache_workspace" in L.hn_last_error()
    assert L.hn_cache_extend(ref(ok), FAKE, -1, 1, FAKE, None) == 1
    assert L.hn_cache_extend(ref(ok), FAKE, 1, -1, FAKE, None) == 1
    assert L.hn_cache_extend(ref(ok), None, 1, 1, FAKE, None) == 5
    assert L.hn_cache_extend(ref(ok), None, 0, 1, None, None) == 0          # nothing to do
    assert L.hn_cache_free(ref(ok), None, 2, None) == 5
    assert L.hn_cache_fork(ref(ok), FAKE, None, 2, FAKE, None) == 5
    assert L.hn_cache_compact(ref(ok), None, None) == 5
    assert L.hn_cache_copy(ref(ok), FAKE, None, 2, None) == 5
    st = (512, 128, 128)
    assert L.hn_cache_append(ref(ok), 2, FAKE, *st, FAKE, *st, FAKE, 1, 1, None) == 1      # layer
    assert L.hn_cache_append(ref(ok), 0, FAKE, 512, 100, 128, FAKE, *st, FAKE, 1, 1, None) == 2
    assert L.hn_cache_append(ref(ok), 0, FAKE + 2, *st, FAKE, *st, FAKE, 1, 1, None) == 2
    assert L.hn_cache_append(ref(ok), 0, None, *st, FAKE, *st, FAKE, 1, 1, None) == 5
    assert L.hn_cache_append(ref(ok), 0, None, *st, None, *st, None, 0, 1, None) == 0


def test_attention_checks(hn, paged):
    L = hn.lib.lib
    ok = struct(paged)
    n = ctypes.c_int64()
    sizes = {}
    for b, lq, shared in ((1, 1, 0), (4, 1, 64), (4, 200, 64), (100, 1, 64), (4096, 1, 0)):
        assert L.hn_paged_attention_workspace(ref(ok), b, lq, 8, shared, 1, ctypes.byref(n)) == 0
        sizes[b, lq, shared] = n.value
        assert n.value >= 2 * 4 * (b + 1)
    assert sizes[4, 200, 64] > sizes[4, 1, 64]
    for args, code in (((4097, 1, 8, 0, 1), 1), ((1, 1, 6, 0, 1), 1), ((1, 1, 8, 8, 1), 1), ((1, 1, 8, 176, 1), 1), ((1, 1, 8, 0, 2), 5),
                       ((-1, 1, 8, 0, 1), 1), ((1, 1, 0, 0, 1), 1), ((4096, 1 << 20, 8, 0, 1), 1)):
        assert L.hn_paged_attention_workspace(ref(ok), *args, ctypes.byref(n)) == code, args

    def attend(**kw):
        a = dict(layer=0, q=FAKE, qb=1024, ql=1024, qh=128, rows=FAKE, b=1, lq=1, h=8, d=128, shared=0, causal=1, scale=0.1, out=FAKE,
                 ob=1024, ol=1024, oh=128, lse=None, ws=FAKE, size=1 << 40)
        a.update(kw)
        return L.hn_paged_attention(ref(ok), *a.values(), None)
    assert attend(d=64) == 7 and attend(layer=2) == 1 and attend(layer=-1) == 1 and attend(rows=None) == 5
    assert attend(qh=100) == 2 and attend(out=FAKE + 2) == 2 and attend(ws=FAKE + 4) == 2
    assert attend(b=0) == 0 and attend(lq=0) == 0


def test_workspace_of_calls_without_a_shared_part(hn, paged):
    """What is left in the workspace are the tiles that the cuts between CTAs fall into: it does not grow with the queries."""
    L = hn.lib.lib
    n = ctypes.c_int64()
    big = struct(paged, pages=1 << 16, page=64, width=1 << 13, slots=4096, heads=8)
    for b, lq, h in ((2, 4400, 16), (1, 1 << 15, 64), (64, 8192, 8), (1, 1 << 16, 1 << 13), (3, 64, 8), (1000, 1, 64)):
        assert L.hn_paged_attention_workspace(ref(big), b, lq, h, 0, 1, ctypes.byref(n)) == 0
        assert n.value <= 2 * 148 * 256 * 130 * 4 + 2 * 4 * (b + 1), (b, lq, h, n.value)


def test_norm_checks(hn):
    L = hn.lib.lib

    def call(**kw):
        a = dict(x=FAKE, ldx=256, r=FAKE, ldr=256, w=FAKE, rows=4, d=256, eps=1e-6, kind=0, flags=0, out=FAKE, ldo=256, q=FAKE,
                 ldq=256, s=FAKE, rs=2, gs=1)
        a.update(kw)
        return L.hn_add_rmsnorm_quant(*a.values(), None)
    assert call(r=None) == 5 and call(kind=3) == 5 and call(flags=2) == 5 and call(flags=4) == 5
    assert call(d=0) == 1 and call(d=192) == 1 and call(d=16512) == 1 and call(rows=-1) == 1 and call(ldo=128) == 1
    assert call(rs=1, gs=2) == 1 and call(ldx=260) == 2 and call(w=FAKE + 2) == 2 and call(ldq=264) == 2
    assert call(rows=0, x=None, r=None, out=None, q=None, s=None) == 0


def test_no_cpu_path(hn, paged):
    x = torch.zeros((2, 128), dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        hn.fused.add_rmsnorm_quant(x, x, x[0])
    pool = torch.zeros((1, 2, 1, 16, 128), dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        paged.KVCache.over(pool, pool, None, None, torch.zeros(7, dtype=torch.int32), 1, 4)
