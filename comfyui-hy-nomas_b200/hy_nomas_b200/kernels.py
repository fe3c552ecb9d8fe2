"""Block-scaled W8A8 / FP8 linears on the B200 tensor cores - the drop-in for hy_nomas/kernels.py.

Same functions, arguments, shapes and dtypes as the reference module (hy_nomas/kernels.py:19-226):

    y[m, n] = sum_g  a_scale[m, g] * w_scale[n, g] * sum_{k in g} qa[m, k] * qw[n, k]   (+ bias[n])

with one scale per token and 128 channels for the activations (absmax/127, round half away from zero for
int8; absmax/448 for e4m3) and the checkpoint's weight scales. The work runs in libhynomas_b200.so
(tcgen05 tensor-core GEMM with the scale promotion, bias, GELU and requantization fused into its
epilogue); this module only allocates outputs with torch and passes pointers.

Beyond the reference's layouts, `block_gemm` also takes per-row scales (a_scale [M] per token, w_scale [N]
per output channel) and 128x128 weight-block scales [N/128, K/128] (the FP8 decoder's stored layout), and
`quantize_activations(..., per_token=True)` quantizes with one scale per row.
"""
import torch

from . import _lib

GROUP = 128
EPILOGUES = {None: 0, "gelu": 1, "gelu_quant": 2}


def _aligned(t):
    return t.data_ptr() % 16 == 0 and (t.stride(0) * t.element_size()) % 16 == 0 and t.stride(-1) == 1


def quantize_activations(x, kind="int8", per_token=False, round_half_even=False):
    """x [M, K] (K % 128 == 0) -> codes [M, K] and fp32 scales [M, K / 128] (hy_nomas/kernels.py:45-54).
    `per_token=True`: one scale per row, scales [M, 1]. `round_half_even=True` (int8): codes rounded half to
    even instead of the reference's half away from zero (torch.round's convention)."""
    _lib.require_cuda(x)
    m, k = x.shape
    if x.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        x = x.float()
    if not _aligned(x):
        x = _lib.dense(x)
    dtype = torch.int8 if kind == "int8" else torch.float8_e4m3fn
    q = torch.empty((m, k), device=x.device, dtype=dtype)
    if per_token:
        s = torch.empty((m, 1), device=x.device, dtype=torch.float32)
        srs, sgs = 1, 1
    else:
        s, srs, sgs = _lib.group_scales(m, k // GROUP, x.device)
    flags = (1 if per_token else 0) | (2 if round_half_even else 0)
    rc = _lib.lib.hn_quant_act(_lib.ptr(x), x.stride(0), _lib.DTYPE[x.dtype], m, k, _lib.KIND[kind], flags,
                               _lib.ptr(q), q.stride(0), _lib.ptr(s), srs, sgs, _lib.stream_of(x))
    _lib.check(rc, "quantize_activations")
    return q, s


def _scale_mode(s, rows, k, weight):
    """Classify a scale tensor: 'group' [rows, K/128], 'row' [rows] or [rows, 1], 'block' [rows/128, K/128]."""
    g = k // GROUP
    if s.dim() == 1 or (s.dim() == 2 and s.shape[1] == 1 and g != 1):
        if s.shape[0] != rows:
            raise ValueError(f"scale shape {tuple(s.shape)} does not match {rows} rows")
        return "row"
    if s.shape == (rows, g):
        return "group"
    if weight and s.shape == ((rows + 127) // 128, g):
        return "block"
    raise ValueError(f"scale shape {tuple(s.shape)} is none of [{rows}, {g}], [{rows}], [{(rows + 127) // 128}, {g}]")


def block_gemm(qa, sa, qw, sw, bias=None, out_dtype=torch.bfloat16, kind="int8", epilogue=None, out=None):
    """Block-scaled GEMM on quantized activations (hy_nomas/kernels.py:152-170). With epilogue "gelu_quant"
    returns (int8 [M, N], scales [M, N / 128]) ready for the next int8 linear; otherwise [M, N] in
    `out_dtype` (bf16, fp16, fp32; torch.int32 gives the raw int32 accumulator when both scales are per
    row and there is no bias).

    `out` (not in the reference): a caller-owned [M, N] destination with unit column stride (rows may be
    strided, e.g. a slice of a larger buffer), written instead of a fresh tensor; epilogues None and "gelu"."""
    _lib.require_cuda(qa, sa, qw, sw, bias)
    m, k = qa.shape
    n = qw.shape[0]
    mode = EPILOGUES[epilogue]
    sa_mode = _scale_mode(sa, m, k, weight=False)
    sw_mode = _scale_mode(sw, n, k, weight=True)
    if sa.dtype != torch.float32:
        sa = sa.float()
    if sw.dtype != torch.float32:
        sw = sw.float()
    if not _aligned(qa):
        qa = _lib.dense(qa)
    if not _aligned(qw):
        qw = _lib.dense(qw)
    if bias is not None and (bias.stride(0) != 1 or bias.data_ptr() % 16):
        bias = _lib.dense(bias)
    if mode == 2:
        if out is not None:
            raise ValueError("block_gemm: `out` is not supported with epilogue 'gelu_quant'")
        out = torch.empty((m, n), device=qa.device, dtype=torch.int8)
        qs, qrs, qgs = _lib.group_scales(m, n // GROUP, qa.device)
    else:
        want = out_dtype if mode == 0 else torch.bfloat16
        if out is None:
            out = torch.empty((m, n), device=qa.device, dtype=want)
        elif out.shape != (m, n) or out.dtype != want or out.stride(1) != 1 or out.device != qa.device:
            raise ValueError(f"block_gemm: out must be a {want} [{m}, {n}] tensor with unit column stride on "
                             f"{qa.device}")
        qs, qrs, qgs = None, 0, 0
    sa_rs, sa_gs = _lib.scale_strides(sa)
    sw_rs, sw_gs = _lib.scale_strides(sw)
    rc = _lib.lib.hn_block_gemm(
        _lib.ptr(qa), qa.stride(0), _lib.ptr(sa), sa_rs, sa_gs, _lib.SCALE_MODE[sa_mode],
        _lib.ptr(qw), qw.stride(0), _lib.ptr(sw), sw_rs, sw_gs, _lib.SCALE_MODE[sw_mode],
        _lib.ptr(bias), _lib.DTYPE[bias.dtype] if bias is not None else 0,
        _lib.ptr(out), out.stride(0), _lib.DTYPE[out.dtype] if mode != 2 else 0,
        _lib.ptr(qs), qrs, qgs,
        m, n, k, _lib.KIND[kind], mode, _lib.stream_of(qa))
    _lib.check(rc, "block_gemm")
    return (out, qs) if mode == 2 else out


def adaln_quant(x, shift, scale, eps=1e-6):
    """x [B, L, D] bf16, shift/scale [B, D] -> int8 codes [B * L, D] and scales [B * L, D / 128] of the modulated
    LayerNorm, for the q/k/v linears (hy_nomas/kernels.py:198-207)."""
    _lib.require_cuda(x, shift, scale)
    b, l, d = x.shape
    if x.dtype != torch.bfloat16 or shift.dtype != torch.bfloat16 or scale.dtype != torch.bfloat16:
        raise TypeError("adaln_quant: x, shift and scale must be bf16")
    x, shift, scale = _lib.dense(x), _lib.dense(shift), _lib.dense(scale)
    q = torch.empty((b * l, d), device=x.device, dtype=torch.int8)
    s, srs, sgs = _lib.group_scales(b * l, d // GROUP, x.device)
    rc = _lib.lib.hn_adaln_quant(_lib.ptr(x), _lib.ptr(shift), _lib.ptr(scale), b, l, d, eps, _lib.ptr(q),
                                 _lib.ptr(s), srs, sgs, _lib.stream_of(x))
    _lib.check(rc, "adaln_quant")
    return q, s


def block_linear(x, qw, sw, bias=None, kind="int8"):
    """F.linear with block-scaled 8-bit weights: x [..., K] -> [..., N] in x's dtype (hy_nomas/kernels.py:210-222).
    As in the reference, K % 128 != 0 or an empty input takes the dequantized bf16 linear."""
    _lib.require_cuda(x)
    shape = x.shape
    x2 = x.reshape(-1, shape[-1])
    if shape[-1] % GROUP or x2.shape[0] == 0:
        from .ops import dequantize_g128
        return torch.nn.functional.linear(x, dequantize_g128(qw, sw, x.dtype), bias)
    with torch.cuda.device(x.device):
        qa, sa = quantize_activations(x2, kind)
        out = block_gemm(qa, sa, qw, sw.float(), bias, x.dtype, kind)
    return out.reshape(*shape[:-1], qw.shape[0])


def int8_g128_linear(x, qw, sw, bias=None):
    """hy_nomas/kernels.py:225-226."""
    return block_linear(x, qw, sw, bias, kind="int8")


# ----------------------------------------------------------------------------------------------- 4-bit codes with block scales

FP4_SPAN = {"mxfp4": 128, "nvfp4": 64}      # columns of a scale tile
_FLOATS = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _fp4_kind(kind, what):
    code = _lib.FP4_KIND.get(kind)
    if code is None:
        raise ValueError(f"{what}: kind {kind!r} (mxfp4 or nvfp4)")
    return code


def _fp4_operand(q, s, r, kind, device, what, name):
    """The checks of one operand -> (codes whose rows start on 16 bytes, their row pitch, scales, row scales, rows, K)."""
    shape = q.shape
    if len(shape) != 2 or shape[1] % 16 or not shape[1] or q.dtype != torch.uint8:
        raise ValueError(f"{what}: the codes of {name} must be uint8 [rows, K / 2] with K a multiple of 32, got {q.dtype} "
                         f"{tuple(shape)}")
    rows, half = shape
    span = FP4_SPAN[kind] // 2
    want = ((rows + 127) // 128, (half + span - 1) // span, 512)
    if s.shape != want or s.dtype != torch.uint8:
        raise ValueError(f"{what}: the scales of {name} must be uint8 {want} for {kind}, got {s.dtype} {tuple(s.shape)}")
    if s.device != device:
        raise RuntimeError(f"{what}: scales of {name} on {s.device}, the codes on {device}")
    if r is not None:
        if kind == "mxfp4":
            raise ValueError(f"{what}: mxfp4 has no row scales")
        if r.dtype != torch.float32 or r.shape != (rows,):
            raise ValueError(f"{what}: the row scales of {name} must be fp32 [{rows}], got {r.dtype} {tuple(r.shape)}")
        if r.device != device:
            raise RuntimeError(f"{what}: row scales of {name} on {r.device}, the codes on {device}")
        if not r.is_contiguous():
            r = r.contiguous()
    pitch = half
    if not q.is_contiguous():
        pitch = q.stride(0)
        if q.stride(1) != 1 or pitch % 16 or pitch < half:
            q, pitch = _lib.dense(q), half
    if q.data_ptr() % 16:
        q, pitch = _lib.dense(q), half
    if not s.is_contiguous() or s.data_ptr() % 16:
        s = _lib.dense(s)
    return q, pitch, s, r, rows, 2 * half


def quantize_fp4(x, kind="nvfp4"):
    """x [M, K] -> (codes, scales, row scales): e2m1 codes uint8 [M, Kp / 2], two to a byte (the even column in the low half), Kp =
    K rounded up to 32; scale bytes uint8 [M / 128, tiles, 512] (rounded up) in the tensor cores' order (`ops.untile_fp4_scales`).

    "nvfp4": an e4m3 scale per 16 columns and an fp32 scale per row, max|row| / 2688 (fp32 [M]), so no scale has to be known
    beforehand. "mxfp4": a scale 2^e per 32 columns, e = floor(log2 max|x|) - 2; the row scales are None. A NaN or an infinity
    makes its row (nvfp4) or its 32 columns (mxfp4) NaN; nvfp4 rows below 2^-100 count as zeros."""
    code = _fp4_kind(kind, "quantize_fp4")
    if not x.is_cuda:
        _lib.require_cuda(x)
    shape = x.shape
    if len(shape) != 2 or shape[1] == 0:
        raise ValueError(f"quantize_fp4: x must be [M, K], got {tuple(shape)}")
    dtype = _FLOATS.get(x.dtype)
    if dtype is None:
        x, dtype = x.float(), 2
    m, k = shape
    pitch = k
    if not x.is_contiguous():
        if x.stride(1) == 1 and x.stride(0) >= k:
            pitch = x.stride(0)
        else:
            x = x.contiguous()
    kp, device, span = (k + 31) // 32 * 32, x.device, FP4_SPAN[kind]
    q = torch.empty((m, kp // 2), dtype=torch.uint8, device=device)
    s = torch.empty(((m + 127) // 128, (kp + span - 1) // span, 512), dtype=torch.uint8, device=device)
    r = torch.empty(m, dtype=torch.float32, device=device) if code == 3 else None
    _lib.check(_lib.launch("hn_quantize_fp4", device, x.data_ptr(), pitch, dtype, m, k, code, q.data_ptr(), kp // 2, s.data_ptr(),
                           None if r is None else r.data_ptr()), "quantize_fp4")
    return q, s, r


def dequantize_fp4(q, s, r=None, kind="nvfp4", dtype=torch.bfloat16, columns=None):
    """What codes, scales and row scales (None: all 1) stand for: code * (scale * row scale), rounded once to `dtype` (bf16, fp16,
    fp32) [M, columns]. `columns`: the K that was quantized, where it was no multiple of 32."""
    code = _fp4_kind(kind, "dequantize_fp4")
    if not q.is_cuda:
        _lib.require_cuda(q)
    device = q.device
    q, pitch, s, r, m, kp = _fp4_operand(q, s, r, kind, device, "dequantize_fp4", "q")
    k = kp if columns is None else columns
    if not kp - 32 < k <= kp:
        raise ValueError(f"dequantize_fp4: {k} columns of {kp}")
    if dtype not in _FLOATS:
        raise TypeError(f"dequantize_fp4: dtype {dtype} (bf16, fp16 or fp32)")
    if r is None and kind == "nvfp4":
        r = torch.ones(m, dtype=torch.float32, device=device)
    out = torch.empty((m, k), dtype=dtype, device=device)
    _lib.check(_lib.launch("hn_dequantize_fp4", device, q.data_ptr(), pitch, s.data_ptr(), None if r is None else r.data_ptr(), m, k,
                           kp, code, out.data_ptr(), k, _FLOATS[dtype]), "dequantize_fp4")
    return out


def fp4_gemm(qa, sa, ra, qw, sw, rw, bias=None, out_dtype=torch.bfloat16, kind="nvfp4", out=None):
    """The product of two operands of `quantize_fp4`: (qa, sa, ra) [M, K] activations, (qw, sw, rw) [N, K] weights -> [M, N] in
    `out_dtype` (bf16, fp16, fp32), a . w^T (+ bias [N] in one of these types), summed in fp32 on the tensor cores with the block
    scales, rounded once. `ra`, `rw` None: row scales of 1.

    `out`: a caller-owned [M, N] destination of `out_dtype` with unit column stride (rows may be strided)."""
    code = _fp4_kind(kind, "fp4_gemm")
    if not (qa.is_cuda and qw.is_cuda):
        _lib.require_cuda(qa, qw)
    device = qa.device
    if qw.device != device:
        raise RuntimeError(f"fp4_gemm: a on {device}, w on {qw.device}")
    qa, lda, sa, ra, m, k = _fp4_operand(qa, sa, ra, kind, device, "fp4_gemm", "a")
    qw, ldw, sw, rw, n, kw = _fp4_operand(qw, sw, rw, kind, device, "fp4_gemm", "w")
    if kw != k:
        raise ValueError(f"fp4_gemm: a has {k} columns, w {kw}")
    if n == 0:
        raise ValueError("fp4_gemm: w has no rows")
    dtype = _FLOATS.get(out_dtype)
    if dtype is None:
        raise TypeError(f"fp4_gemm: out_dtype {out_dtype} (bf16, fp16 or fp32)")
    if bias is not None:
        if bias.shape != (n,) or bias.dtype not in _FLOATS:
            raise ValueError(f"fp4_gemm: bias must be bf16, fp16 or fp32 [{n}], got {bias.dtype} {tuple(bias.shape)}")
        if bias.device != device:
            raise RuntimeError(f"fp4_gemm: a on {device}, bias on {bias.device}")
        if not bias.is_contiguous():
            bias = bias.contiguous()
    ldo = n
    if out is None:
        out = torch.empty((m, n), dtype=out_dtype, device=device)
    else:
        if out.shape != (m, n) or out.dtype != out_dtype or out.device != device or (n > 1 and out.stride(1) != 1) or \
                (m > 1 and out.stride(0) < n):
            raise ValueError(f"fp4_gemm: out must be a {out_dtype} [{m}, {n}] tensor with unit column stride on {device}")
        if m > 1:
            ldo = out.stride(0)
    _lib.check(_lib.launch("hn_fp4_gemm", device, qa.data_ptr(), lda, sa.data_ptr(), None if ra is None else ra.data_ptr(),
                           qw.data_ptr(), ldw, sw.data_ptr(), None if rw is None else rw.data_ptr(),
                           None if bias is None else bias.data_ptr(), 0 if bias is None else _FLOATS[bias.dtype], out.data_ptr(),
                           ldo, dtype, m, n, k, code), "fp4_gemm")
    return out


def fp4_linear(x, qw, sw, rw=None, bias=None, kind="nvfp4"):
    """F.linear with 4-bit weights, as `block_linear` has it for 8-bit ones: x [..., K] -> [..., N] in x's dtype (bf16, fp16 or
    fp32), the activations quantized on the way."""
    if x.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise TypeError(f"fp4_linear: x must be bf16, fp16 or fp32, got {x.dtype}")
    shape = x.shape
    x2 = x.reshape(-1, shape[-1])
    if qw.dim() != 2 or (shape[-1] + 31) // 32 * 16 != qw.shape[1]:
        raise ValueError(f"fp4_linear: x {tuple(shape)} does not fit codes {tuple(qw.shape)}")
    return fp4_gemm(*quantize_fp4(x2, kind), qw, sw, rw, bias, x.dtype, kind).reshape(*shape[:-1], qw.shape[0])
