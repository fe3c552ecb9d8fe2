"""Rotary positions computed on the way: heads of any width up to 256, both pair layouts, a part of the head, scaled contexts.

`fused.qk_norm_rope` and `fused.pixelumm_qk` take tables of cos and sin [tokens, 128], as the reference makes them
(hy_nomas/fused.py:65-186). Here a call takes the tokens' positions, so that no table is made or read, and a token far into
a long context is turned as exactly as the first (up to position 2^39; a frequency is held to 2^-65 of a turn):

    rot = Rotary(128, theta=10000.0, layout="half")                          # once
    q = rotate(q, positions, rot, q_norm)                                    # RMSNorm per head, then the rotation
    q = cache.append_rotated(layer, q, k, v, rows, rot, q_norm, k_norm)      # paged.KVCache: k and v into the pages, too

Inference only, as the rest of the framework.
"""
import math
from decimal import Context, Decimal, localcontext

import torch

from . import _lib

LAYOUTS = {"half": 0, "interleaved": 1}
NORM_FP32 = 16
_FLOATS = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_SCALINGS = {"linear": {"factor"}, "ntk": {"factor"}, "yarn": {"factor", "original", "beta_fast", "beta_slow", "attention_factor"}}


# enough digits for 64 bits of a turn of frequencies up to 1e20 radians a position
_EXACT = Context(prec=60)
_UNITS = _EXACT.divide(2 ** 63, Decimal("3.14159265358979323846264338327950288419716939937510582097494459"))    # of a radian: 2^64 a turn


def _radians(dim, theta, scaling):
    """`frequencies` with the radians as Decimals: a double's 53 bits would leave the fixed-point ones some 2^-56 of a turn a
    position off."""
    if dim < 8 or dim > 256 or dim % 8:
        raise ValueError(f"rotary: {dim} rotated columns (a multiple of 8 up to 256)")
    if not (math.isfinite(theta) and theta > 1):
        raise ValueError(f"rotary: theta {theta}")
    scaling = dict(scaling or {})
    kind = scaling.pop("type", None)
    if kind not in _SCALINGS and (kind is not None or scaling):
        raise ValueError(f"rotary: scaling type {kind!r} (linear, ntk or yarn)")
    if kind is not None and (set(scaling) - _SCALINGS[kind] or "factor" not in scaling or (kind == "yarn" and "original" not in scaling)):
        raise ValueError(f"rotary: scaling {kind} with {sorted(scaling)}")
    if any(not (math.isfinite(v) and v > 0) for v in scaling.values()):
        raise ValueError(f"rotary: scaling {scaling} must be positive numbers")
    theta, factor = float(theta), float(scaling.get("factor", 1.0))
    with localcontext(_EXACT):
        base, by = Decimal(theta).ln(), Decimal(factor)
        if kind == "ntk":
            base += by.ln() * dim / (dim - 2)
            if base <= 0:
                raise ValueError(f"rotary: ntk factor {factor} leaves theta {float(base.exp())}")
        # powers of one ratio: 127 more roundings of 60 digits, and an exponential each would be most of a Rotary's time (2 ms)
        step, freq = (-2 * base / dim).exp(), [Decimal(1)]
        for _ in range(dim // 2 - 1):
            freq.append(freq[-1] * step)
        if kind == "linear":
            freq = [f / by for f in freq]
        if kind != "yarn":
            return freq, 1.0

        def column(turns):      # the (fractional) pair that turns so many times over the original context, in columns / 2
            return dim * math.log(scaling["original"] / (turns * 2 * math.pi)) / (2 * math.log(theta))
        low = max(math.floor(column(scaling.get("beta_fast", 32.0))), 0)
        high = min(math.ceil(column(scaling.get("beta_slow", 1.0))), dim - 1)
        ramp = [min(max((i - low) / Decimal(max(high - low, 0.001)), Decimal(0)), Decimal(1)) for i in range(dim // 2)]
        return [f * (1 - r) + f / by * r for f, r in zip(freq, ramp)], scaling.get("attention_factor", 0.1 * math.log(factor) + 1.0)


def frequencies(dim, theta=10000.0, scaling=None):
    """(radians per position of the dim / 2 pairs in 64 bits, on the CPU; the factor on cos and sin). `scaling`: None, or a dict
    {"type": ..., "factor": f}:
      "linear"  positions divided by f
      "ntk"     theta * f^(dim / (dim - 2)): the slowest pair is slowed f times, the fastest kept
      "yarn"    (Peng et al., arXiv 2309.00071) pairs that turn more than `beta_fast` (32) times over `original` positions are kept,
                those that turn less than `beta_slow` (1) times are slowed f times, a ramp between; cos and sin times
                `attention_factor` (0.1 ln f + 1)"""
    freq, factor = _radians(dim, theta, scaling)
    return torch.tensor([float(f) for f in freq], dtype=torch.float64), factor


class Rotary:
    """What turns the first `dim` columns of a head by position. `layout` "half": column i pairs with i + dim / 2; "interleaved": 2 i
    with 2 i + 1. `scaling`: see `frequencies`; or give `freq`, radians per position [dim / 2], and `factor` yourself."""

    def __init__(self, dim, theta=10000.0, layout="half", scaling=None, device="cuda", freq=None, factor=1.0):
        if layout not in LAYOUTS:
            raise ValueError(f"Rotary: layout {layout!r} (half or interleaved)")
        if freq is None:
            radians, factor = _radians(dim, theta, scaling)
            freq = torch.tensor([float(f) for f in radians], dtype=torch.float64)
        else:
            if scaling is not None:
                raise ValueError("Rotary: freq and scaling")
            _radians(dim, 10000.0, None)                        # the checks of dim
            freq = torch.as_tensor(freq, dtype=torch.float64).cpu()
            if freq.shape != (dim // 2,) or not bool(torch.isfinite(freq).all()):
                raise ValueError(f"Rotary: freq must be {dim // 2} finite numbers")
            radians = [Decimal(f) for f in freq.tolist()]
        if not math.isfinite(factor):
            raise ValueError(f"Rotary: factor {factor}")
        self.dim, self.layout, self.factor, self.radians = dim, layout, float(factor), freq
        # fractions of a turn times 2^64, to the nearest, as signed 64-bit integers: what is past a whole turn does not matter
        with localcontext(_EXACT):
            turns = [int((f * _UNITS).to_integral_value()) for f in radians]
        self.freq = torch.tensor([(t + 2 ** 63) % 2 ** 64 - 2 ** 63 for t in turns], dtype=torch.int64, device=device)
        self._args = (dim, LAYOUTS[layout], self.factor)


_WIDE = {torch.int32: 0, torch.int64: 1}


def positions_of(p, batch, tokens, device, what):
    """(pointer, batch stride, token stride, 1 if int64, the tensor) of positions [batch, tokens] or [tokens]."""
    wide = _WIDE.get(p.dtype) if isinstance(p, torch.Tensor) else None
    if wide is None:
        if not isinstance(p, torch.Tensor) or p.is_floating_point() or p.is_complex() or p.dtype == torch.bool:
            raise TypeError(f"{what}: positions must be a tensor of integers")
        p, wide = p.to(torch.int64), 1
    if p.device != device:
        raise RuntimeError(f"{what}: positions on {p.device}, the heads on {device}")
    shape = p.shape
    if shape == (tokens,):
        return p.data_ptr(), 0, p.stride(0), wide, p
    if shape != (batch, tokens):
        raise ValueError(f"{what}: positions {tuple(shape)} must be [{batch}, {tokens}] or [{tokens}]")
    pb, pt = p.stride()
    return p.data_ptr(), pb, pt, wide, p


def norm_weights(ws, dim, device, what):
    """Per-head norm weights (each a tensor [dim], or None) as the kernels take them, all bf16 or all fp32 and aligned -> (the tensors,
    what the layout is told). fp32 where any is not bf16: no weight loses bits (but those beyond fp32)."""
    wide = 0
    for w in ws:
        if w is None:
            continue
        if w.shape != (dim,):
            raise ValueError(f"{what}: norm weight {tuple(w.shape)} must be [{dim}]")
        if w.device != device:
            raise RuntimeError(f"{what}: norm weight on {w.device}, the heads on {device}")
        if w.dtype != torch.bfloat16:
            wide = NORM_FP32
    dtype, out = torch.float32 if wide else torch.bfloat16, []
    for w in ws:
        if w is not None:
            if w.dtype != dtype:
                w = w.to(dtype)
            if not w.is_contiguous() or w.data_ptr() % 16:
                w = _lib.dense(w)
        out.append(w)
    return out, wide


def check_rotary(rot, dim, device, what):
    if not isinstance(rot, Rotary):
        raise TypeError(f"{what}: a Rotary is needed, got {type(rot).__name__}")
    if rot.dim > dim:
        raise ValueError(f"{what}: {rot.dim} rotated columns of a head of {dim}")
    if rot.freq.device != device:
        raise RuntimeError(f"{what}: the Rotary is on {rot.freq.device}, the heads on {device}")


def _steps8(t):
    a, b, c, d = t.stride()
    return d == 1 and not (a | b | c) % 8 and t.data_ptr() % 16 == 0


def _span(t):
    """First byte and the byte after the last of a tensor that is not empty."""
    at = t.data_ptr()
    lo = sum(min(0, s * (n - 1)) for s, n in zip(t.stride(), t.shape))
    hi = sum(max(0, s * (n - 1)) for s, n in zip(t.stride(), t.shape))
    return at + lo * t.element_size(), at + (hi + 1) * t.element_size()


def _apart(t):
    """The heads of a tensor that is not empty do not overlap: each stride is past what the smaller ones reach."""
    reach = t.shape[3]
    for s, n in sorted((abs(s), n) for s, n in zip(t.stride()[:3], t.shape[:3]) if n > 1):
        if s < reach:
            return False
        reach += s * (n - 1)
    return True


def rotate(x, positions, rot, weight=None, eps=1e-6, out=None):
    """x [B, L, H, D] (bf16, fp16 or fp32; D a multiple of 8 up to 256; any strides in steps of 8 elements, the last dimension
    contiguous) at integer positions [B, L] or [L] -> [B, L, H, D] of x's dtype: RMSNorm over each head times `weight` [D] (bf16, fp16
    or fp32, taken as it is; None: no norm), then the rotation of its first rot.dim columns, in fp32 with one rounding. `out`: a
    caller-owned tensor like x, or x."""
    what = "rotate"
    if not x.is_cuda:
        _lib.require_cuda(x)
    device = x.device
    dtype = _FLOATS.get(x.dtype)
    if dtype is None:
        raise TypeError(f"rotate: x must be bf16, fp16 or fp32, got {x.dtype}")
    shape = x.shape
    if len(shape) != 4 or shape[3] % 8 or not 8 <= shape[3] <= 256:
        raise ValueError(f"rotate: x must be [B, L, H, D] with D a multiple of 8 up to 256, got {tuple(shape)}")
    b, l, h, d = shape
    check_rotary(rot, d, device, what)
    ptr, pb, pl, wide, keep = positions_of(positions, b, l, device, what)
    (w,), w_wide = norm_weights((weight,), d, device, what)
    src = x if _steps8(x) else _lib.dense(x)
    if out is None:
        out = torch.empty((b, l, h, d), dtype=x.dtype, device=device)
    else:
        if out.shape != x.shape or out.dtype != x.dtype or out.device != device or not _steps8(out):
            raise ValueError(f"rotate: out must be {x.dtype} {tuple(x.shape)} on {device} in steps of 8 elements, 16-byte aligned")
        if out.numel():
            if not _apart(out):
                raise ValueError("rotate: the heads of out overlap")
            same = out.data_ptr() == src.data_ptr() and out.stride() == src.stride()
            (a0, a1), (b0, b1) = _span(src), _span(out)
            if not same and a0 < b1 and b0 < a1:
                raise ValueError("rotate: out must be x itself or lie apart from it")
    dim, layout, factor = rot._args
    xs, os = src.stride(), out.stride()
    _lib.check(_lib.launch("hn_rotate", device, src.data_ptr(), xs[0], xs[1], xs[2], dtype, ptr, pb, pl, wide,
                           rot.freq.data_ptr(), dim, layout | w_wide, factor, None if w is None else w.data_ptr(), eps, b, l, h, d,
                           out.data_ptr(), os[0], os[1], os[2]), what)
    return out
