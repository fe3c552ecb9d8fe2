"""A paged K/V cache for sequences that branch from one another, and the attention that reads it.

The reference keeps one int8 history per run (hy_nomas/world.py:80-204). Here many sequences live in one pool of
pages, in the framework's two formats - bf16, or `world.quantize_kv`'s int8 codes with one fp32 scale per (token, head) -
and a branch of a sequence shares its parent's full pages instead of copying them:

    cache = KVCache(layers, pages, heads, page, slots, width, kind="int8")
    cache.extend(rows, n)                        # room for n more tokens of each row
    cache.append(layer, k, v, rows)              # k, v [B, n, heads, 128]: those tokens, layer by layer
    q = cache.append_rotated(layer, q, k, v, rows, rot, q_norm, k_norm)   # ... or with norm and rotation on the way
    cache.fork(parents, children)                # children become branches: only a partial last page is copied
    out = attention(q, cache, layer, rows, shared=tokens)     # the shared tokens are read once for all rows
    cache.free(rows)
    cache.compact()                              # used pages move to the front of the pool

`rows`, `parents`, `children`, `src` and `dst` are int32 CUDA tensors (or sequences of ints, copied to the device). The
page table, lengths and reference counts live on the device and every call is asynchronous: a request that cannot be
met - no free page, a full table row, a row listed twice, a child that is not empty - leaves its row as it was and is counted,
and `check()` raises if any was. `append` leaves out a row whose last `extend` was not met, so a step that found no room
changes no token; the row goes on with its next `extend`. Head dim 128.
"""
import ctypes
import math

import torch

from . import _lib, rotary

HEAD_DIM = 128


class _Struct(ctypes.Structure):
    """hn_kv_cache of include/hynomas_b200.h."""
    _fields_ = [(n, ctypes.c_void_p) for n in ("k", "v", "k_scale", "v_scale", "table", "lengths", "refs", "failed")] + \
        [(n, ctypes.c_int64) for n in ("layers", "pages", "heads", "page", "slots", "width")] + \
        [("refused", ctypes.c_void_p), ("epoch", ctypes.c_int32)]


class KVCache:
    """The pools k, v [layers, pages, heads, page, 128] (and k_scale, v_scale [layers, pages, heads, page] for
    kind="int8"), and the metadata `table` [slots, width] (-1: no page), `lengths` [slots], `refs` [pages]: how many
    table entries name a page. `page` is a multiple of 16 tokens; a row holds at most width * page."""

    def __init__(self, layers, pages, heads, page, slots, width, kind="bf16", device="cuda"):
        if kind not in ("bf16", "int8"):
            raise ValueError(f"KVCache: kind {kind!r} (bf16 or int8)")
        if min(layers, pages, heads, slots, width) < 1 or page < 16 or page % 16:
            raise ValueError("KVCache: positive sizes and a page of a multiple of 16 tokens are needed")
        shape = (layers, pages, heads, page)
        dtype = torch.bfloat16 if kind == "bf16" else torch.int8
        k, v = (torch.zeros(shape + (HEAD_DIM,), dtype=dtype, device=device) for _ in range(2))
        ks, vs = (torch.ones(shape, dtype=torch.float32, device=device) for _ in range(2)) if kind == "int8" else (None, None)
        meta = torch.zeros(slots * width + slots + pages, dtype=torch.int32, device=device)
        meta[:slots * width] = -1
        self._set(k, v, ks, vs, meta, slots, width)

    @classmethod
    def over(cls, k, v, k_scale, v_scale, meta, slots, width):
        """A cache over tensors that are there already: contiguous pools, and `meta` = table, lengths, refs in one
        int32 tensor of slots * width + slots + pages."""
        self = cls.__new__(cls)
        self._set(k, v, k_scale, v_scale, meta, slots, width)
        return self

    def _set(self, k, v, ks, vs, meta, slots, width):
        _lib.require_cuda(k, v, ks, vs, meta)
        want = torch.bfloat16 if ks is None else torch.int8
        if k.dim() != 5 or k.shape != v.shape or k.shape[4] != HEAD_DIM or k.dtype != want or v.dtype != want:
            raise ValueError(f"KVCache: k and v must be {want} [layers, pages, heads, page, 128]")
        layers, pages, heads, page, _ = k.shape
        if (ks is None) != (vs is None) or (ks is not None and any(
                t.shape != k.shape[:4] or t.dtype != torch.float32 for t in (ks, vs))):
            raise ValueError("KVCache: k_scale and v_scale must be fp32 [layers, pages, heads, page], or both None")
        if meta.dtype != torch.int32 or meta.dim() != 1 or meta.numel() != slots * width + slots + pages:
            raise ValueError("KVCache: meta must be int32 of slots * width + slots + pages")
        if any(t is not None and (not t.is_contiguous() or t.device != k.device) for t in (k, v, ks, vs, meta)):
            raise ValueError("KVCache: contiguous tensors of one device are needed")
        self.k, self.v, self.k_scale, self.v_scale, self.meta = k, v, ks, vs, meta
        self.kind = "bf16" if ks is None else "int8"
        self.layers, self.pages, self.heads, self.page, self.slots, self.width = layers, pages, heads, page, slots, width
        self.device = k.device
        n = slots * width
        self.table, self.lengths, self.refs = meta[:n].view(slots, width), meta[n:n + slots], meta[n + slots:]
        self.failed, self._refused = torch.zeros(1 + slots, dtype=torch.int32, device=k.device).split([1, slots])
        p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        self._struct = _Struct(p(k), p(v), p(ks), p(vs), p(self.table), p(self.lengths), p(self.refs), p(self.failed),
                               layers, pages, heads, page, slots, width, p(self._refused), 1)
        self._ref = ctypes.addressof(self._struct)
        self._ws_bytes = {}

    def _ids(self, x, what):
        """A list of row or page ids as a contiguous int32 tensor on the cache's device."""
        if not isinstance(x, torch.Tensor):
            x = torch.tensor(x, dtype=torch.int32, device=self.device)
        elif x.dtype != torch.int32:
            if x.is_floating_point() or x.is_complex() or x.dtype == torch.bool:
                raise TypeError(f"{what}: ids must be integers, got {x.dtype}")
            if x.element_size() >= 4:               # not modulo 2^32: what does not fit stays out of range
                x = x.to(torch.int64).clamp(-1, 0x7fffffff)
            x = x.to(torch.int32)
        if x.device != self.device:
            raise RuntimeError(f"{what}: ids on {x.device}, the cache is on {self.device}")
        if x.dim() != 1:
            raise ValueError(f"{what}: ids must be a list, got {tuple(x.shape)}")
        return x if x.is_contiguous() else x.contiguous()

    def _scratch(self, n):
        words = max(self.slots + self.pages + 4 * n, 4 + 3 * self.pages)      # hn_cache_workspace
        return torch.empty(words, dtype=torch.int32, device=self.device)

    def extend(self, rows, tokens):
        """Every listed row grows by `tokens` tokens, on new pages (lowest free ids first, in the order listed). The first row
        that there are not enough pages for is refused, and so is every row listed after it."""
        rows = self._ids(rows, "extend")
        if tokens < 0:
            raise ValueError(f"extend: {tokens} tokens")
        ws = self._scratch(rows.numel())
        _lib.check(_lib.launch("hn_cache_extend", self.device, self._ref, rows.data_ptr(), rows.numel(), tokens,
                               ws.data_ptr()), "cache.extend")

    def append(self, layer, k, v, rows):
        """k, v [B, n, heads, 128] bf16 (any strides in whole 16-byte steps, the last dimension contiguous) into the last n
        tokens of the listed rows, which `extend` has made room for; once per layer. Rows whose last `extend` was not met,
        pages that other rows hold too and a row's listings after its first are left out and counted."""
        _lib.require_cuda(k, v)
        rows = self._ids(rows, "append")
        if k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16:
            raise TypeError(f"append: bf16 expected, got {k.dtype} and {v.dtype}")
        if k.dim() != 4 or k.shape != v.shape or k.shape[2] != self.heads or k.shape[3] != HEAD_DIM or \
                k.shape[0] != rows.numel():
            raise ValueError(f"append: k {tuple(k.shape)} and v {tuple(v.shape)} must be "
                             f"[{rows.numel()}, n, {self.heads}, {HEAD_DIM}]")
        if not 0 <= layer < self.layers:
            raise ValueError(f"append: layer {layer} of {self.layers}")
        k, v = _operand(k), _operand(v)
        if k.device != self.device or v.device != self.device:
            raise RuntimeError(f"append: k on {k.device} and v on {v.device}, the cache is on {self.device}")
        kb, kt, kh, _ = k.stride()
        vb, vt, vh, _ = v.stride()
        _lib.check(_lib.launch("hn_cache_append", self.device, self._ref, layer, k.data_ptr(), kb, kt, kh, v.data_ptr(), vb, vt,
                               vh, rows.data_ptr(), k.shape[0], k.shape[1]), "cache.append")

    def append_rotated(self, layer, q, k, v, rows, rot, q_norm=None, k_norm=None, eps=1e-6, positions=None):
        """`append` of k with its per-head RMSNorm (`k_norm` [128], None: none) and rotation (`rotary.Rotary`), and of v as it is, in
        one pass with the norm and rotation of q [B, n, H, 128] -> q' [B, n, H, 128] bf16, for `attention`. Positions are the
        tokens' places in their rows, or `positions` [B, n] or [n]. All in fp32, the weights in their own types (bf16, fp16, fp32); K is
        rounded once, to the cache's format.
        Rows that `append` leaves out are left out and counted in the same way; their q' means nothing."""
        what = "append_rotated"
        if not (q.is_cuda and k.is_cuda and v.is_cuda):
            _lib.require_cuda(q, k, v)
        rows, device, bf16 = self._ids(rows, what), self.device, torch.bfloat16
        if q.dtype != bf16 or k.dtype != bf16 or v.dtype != bf16:
            raise TypeError(f"{what}: bf16 expected, got {q.dtype}, {k.dtype} and {v.dtype}")
        b, qshape, shape = rows.shape[0], q.shape, k.shape
        if len(shape) != 4 or shape != v.shape or shape[2] != self.heads or shape[3] != HEAD_DIM or shape[0] != b or \
                len(qshape) != 4 or qshape[:2] != shape[:2] or qshape[3] != HEAD_DIM or qshape[2] == 0:
            raise ValueError(f"{what}: q {tuple(qshape)}, k {tuple(shape)} and v {tuple(v.shape)} must be "
                             f"[{b}, n, H, {HEAD_DIM}] and [{b}, n, {self.heads}, {HEAD_DIM}]")
        if not 0 <= layer < self.layers:
            raise ValueError(f"{what}: layer {layer} of {self.layers}")
        if q.device != device or k.device != device or v.device != device:
            raise RuntimeError(f"{what}: q on {q.device}, k on {k.device} and v on {v.device}, the cache is on {device}")
        rotary.check_rotary(rot, HEAD_DIM, device, what)
        n, h = shape[1], qshape[2]
        ptr, pb, pt, wide, positions = (None, 0, 0, 0, None) if positions is None else \
            rotary.positions_of(positions, b, n, device, what)
        (wq, wk), w_wide = rotary.norm_weights((q_norm, k_norm), HEAD_DIM, device, what)
        q, k, v = _operand(q), _operand(k), _operand(v)
        out = torch.empty((b, n, h, HEAD_DIM), dtype=torch.bfloat16, device=device)
        dim, layout, factor = rot._args
        qs, ks, vs = q.stride(), k.stride(), v.stride()
        _lib.check(_lib.launch(
            "hn_cache_append_rotated", device, self._ref, layer, q.data_ptr(), qs[0], qs[1], qs[2], h, k.data_ptr(), ks[0], ks[1],
            ks[2], v.data_ptr(), vs[0], vs[1], vs[2], rows.data_ptr(), b, n, ptr, pb, pt, wide, rot.freq.data_ptr(), dim,
            layout | w_wide, factor, None if wq is None else wq.data_ptr(), None if wk is None else wk.data_ptr(), eps, out.data_ptr()),
            "cache.append_rotated")
        return out

    def free(self, rows):
        """The listed rows drop their pages and become empty (a row listed twice, once). A page is free again when its last row
        drops it."""
        rows = self._ids(rows, "free")
        _lib.check(_lib.launch("hn_cache_free", self.device, self._ref, rows.data_ptr(), rows.numel()), "cache.free")

    def fork(self, parents, children):
        """children[i], an empty row, becomes a branch of parents[i]: it shares the full pages, and the tokens of a
        partial last page are copied to a page of its own in every layer."""
        parents, children = self._ids(parents, "fork"), self._ids(children, "fork")
        n = parents.numel()
        if children.numel() != n:
            raise ValueError(f"fork: {n} parents for {children.numel()} children")
        ws = self._scratch(n)
        _lib.check(_lib.launch("hn_cache_fork", self.device, self._ref, parents.data_ptr(), children.data_ptr(), n,
                               ws.data_ptr()), "cache.fork", 2)

    def compact(self):
        """The pages in use move to the lowest ids: the k-th used page above the number in use goes to the k-th free
        id below it, in every layer, and the table follows."""
        ws = self._scratch(0)
        _lib.check(_lib.launch("hn_cache_compact", self.device, self._ref, ws.data_ptr()), "cache.compact", 2)

    def copy_pages(self, src, dst):
        """Page src[i] to page dst[i] in every layer. No page may be both a source and a target, or twice a target."""
        src, dst = self._ids(src, "copy_pages"), self._ids(dst, "copy_pages")
        if src.numel() != dst.numel():
            raise ValueError(f"copy_pages: {src.numel()} sources for {dst.numel()} targets")
        _lib.check(_lib.launch("hn_cache_copy", self.device, self._ref, src.data_ptr(), dst.data_ptr(), src.numel()),
                   "cache.copy_pages")

    def save(self):
        """A copy of the table, lengths and reference counts, for `restore`."""
        return self.meta.clone()

    def restore(self, saved):
        """Back to a saved table. The pools are not touched: pages written since then keep what they hold."""
        if saved.shape != self.meta.shape or saved.dtype != torch.int32:
            raise ValueError("restore: not a saved table of this cache")
        self.meta.copy_(saved)
        self._struct.epoch = self._struct.epoch % 0x7fffffff + 1        # what extend refused since is past

    def check(self):
        """Waits for the calls so far on the current stream; raises if a request could not be met, and clears the count, or if
        a kernel on this stream gave up a bounded wait (`attention` then left rows unwritten)."""
        rc, code = _lib.device_error(torch.cuda.current_stream(self.device))
        if rc != _lib.HN_OK or code:
            raise RuntimeError(f"KVCache: {_lib.STATUS.get(rc, rc)}, device error word {code:#x}: {_lib.last_error()}")
        n = int(self.failed.item())
        if n:
            self.failed.zero_()
            raise RuntimeError(f"KVCache: {n} request(s) could not be met (no free page, a full row, a row listed twice or "
                               "out of range, a child that is not empty, or a token without a page of its row's own)")


def _operand(t):
    """t itself when its rows of 128 start on 16-byte boundaries, else a dense copy."""
    s = t.stride()
    if s[3] == 1 and not (s[0] | s[1] | s[2]) % 8 and t.data_ptr() % 16 == 0:
        return t
    return _lib.dense(t)


def attention(q, cache, layer, rows, shared=0, causal=True, scale=None, out=None, return_lse=False):
    """q [B, Lq, H, 128] bf16 over the tokens that `layer` of the cache holds for the B listed rows -> [B, Lq, H, 128]
    bf16 (and, `return_lse`, the natural log-sum-exp [B, H, Lq] fp32). H is a multiple of the cache's heads; query head
    h reads K/V head h * heads // H. `causal`: the queries are each sequence's last Lq tokens (already appended), and
    each sees the tokens up to itself; otherwise all of them. A query that sees no token gives 0 (lse -inf).

    `shared`: the rows' first `shared` tokens, a multiple of the page, are on the same pages, as `fork` leaves them;
    those are read together for all rows, where each has up to 64 queries times query heads per K/V head (with more, each walks
    all of its keys itself). The result is the same as with shared=0 up to rounding. A row may hold fewer: it sees what it holds."""
    device = cache.device
    if not q.is_cuda:
        _lib.require_cuda(q)
    if q.device != device:
        raise RuntimeError(f"attention: q on {q.device}, the cache is on {device}")
    if q.dtype != torch.bfloat16:
        raise TypeError(f"attention: q must be bf16, got {q.dtype}")
    if q.dim() != 4 or q.shape[3] != HEAD_DIM:
        raise ValueError(f"attention: q must be [B, Lq, H, {HEAD_DIM}], got {tuple(q.shape)}")
    rows = cache._ids(rows, "attention")
    b, lq, h, d = q.shape
    if rows.numel() != b:
        raise ValueError(f"attention: {rows.numel()} rows for {b} sequences")
    q = _operand(q)
    if out is None:
        out = torch.empty((b, lq, h, d), dtype=torch.bfloat16, device=device)
    elif out.shape != q.shape or out.dtype != torch.bfloat16 or out.device != device or _operand(out) is not out:
        raise ValueError(f"attention: out must be bf16 {tuple(q.shape)} with contiguous, 16-byte aligned rows of {d}")
    lse = torch.empty((b, h, lq), dtype=torch.float32, device=device) if return_lse else None
    causal = 1 if causal else 0
    plan = (b, lq, h, shared, causal)
    size = cache._ws_bytes.get(plan)            # the workspace's size goes by these numbers alone
    if size is None:
        n = ctypes.c_int64()
        _lib.check(_lib.lib.hn_paged_attention_workspace(cache._ref, b, lq, h, shared, causal, ctypes.byref(n)),
                   "paged.attention", 0)
        size = cache._ws_bytes[plan] = max(n.value, 16)
    ws = torch.empty(size, dtype=torch.uint8, device=device)
    qb, ql, qh, _ = q.stride()
    ob, ol, oh, _ = out.stride()
    _lib.check(_lib.launch(
        "hn_paged_attention", device, cache._ref, layer, q.data_ptr(), qb, ql, qh, rows.data_ptr(), b, lq, h, d, shared, causal,
        1.0 / math.sqrt(d) if scale is None else float(scale), out.data_ptr(), ob, ol, oh,
        None if lse is None else lse.data_ptr(), ws.data_ptr(), size), "paged.attention", 2)
    return (out, lse) if return_lse else out
