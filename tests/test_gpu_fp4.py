"""The 4-bit linears: quantizer and dequantizer against their definition evaluated operation by operation in fp32 (equal bits),
the product against 64 bits.

The product's bound per output: the sum of Kp / 16 partial sums of 16 products (each exact in fp32) is rounded, or cut, to fp32 at
every addition: 2^-23 of A = sum |a w| with all scales, Kp / 16 times; three fp32 operations behind it (row scales, bias), 2^-24
of what they give each; half a step of the output's type.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
BLOCK = {"nvfp4": 16, "mxfp4": 32}
VALUES = np.array([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], np.float64)
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


# ------------------------------------------------------------------------------------------------- definitions

def e2m1(y):
    """Nearest code, ties to the even code, in numpy."""
    a = np.abs(y)
    n = np.zeros(y.shape, np.uint8)
    for edge, closed in ((.25, False), (.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        n += (a >= edge) if closed else (a > edge)
    return n | (np.signbit(y).astype(np.uint8) << 3)


def e4m3(t):
    """fp32 -> (byte, value), nearest even, all within 448."""
    f = torch.from_numpy(np.ascontiguousarray(t)).to(torch.float8_e4m3fn)
    return f.view(torch.uint8).numpy(), f.float().numpy()


def define(x, kind):
    """x [M, K] -> codes [M, Kp] (one to a byte), scale bytes [M, Kp / block], row scales, by the definition in fp32."""
    x = x.float().cpu().numpy()
    m, k = x.shape
    x = np.pad(x, ((0, 0), (0, -k % 32)))
    b = x.reshape(m, -1, BLOCK[kind])
    with np.errstate(all="ignore"):
        peak = np.abs(b).max(-1)                      # a NaN stays
        if kind == "mxfp4":
            bad = ~np.isfinite(peak)
            e = np.where(peak > 0, np.floor(np.log2(np.where(bad | (peak == 0), 1, peak).astype(np.float64))) - 2, 0).clip(-127, 127)
            byte = np.where(bad, 255, e + 127).astype(np.uint8)
            y = b * np.exp2(-e)[..., None]
            codes = np.where(bad[..., None], 0, e2m1(np.where(bad[..., None], 0, y)))
            return codes.reshape(m, -1), byte, None
        top = peak.max(-1)
        live = np.isfinite(top) & (top >= np.float32(2.0 ** -100))
        r = np.where(live, top / np.float32(2688), np.where(top < np.float32(2.0 ** -100), np.float32(1), np.float32(np.nan)))
        safe = np.where(live, top, np.float32(1))
        t = np.where(live[:, None], np.float32(0.875) * peak / (safe * np.float32(2.0 ** -9))[:, None], np.float32(0))
        byte, sb = e4m3(t.astype(np.float32))
        den = sb * (safe * np.float32(2.0 ** -12))[:, None]
        y = np.where(sb[..., None] > 0, np.float32(0.65625) * b / np.where(den > 0, den, 1)[..., None], np.float32(0))
        assert y.dtype == np.float32 and den.dtype == np.float32
        return np.where(sb[..., None] > 0, e2m1(y), 0).reshape(m, -1), byte, r.astype(np.float32)


def unpack(q):
    q = q.cpu().numpy()
    return np.stack([q & 15, q >> 4], -1).reshape(q.shape[0], -1)


def scale_values(byte, kind):
    if kind == "nvfp4":
        return torch.from_numpy(np.ascontiguousarray(byte)).view(torch.float8_e4m3fn).double().numpy()
    return np.where(byte == 255, np.nan, np.exp2(byte.astype(np.float64) - 127))


def values64(hn, q, s, r, kind):
    """What an operand stands for, in 64 bits."""
    c = unpack(q)
    byte = hn.ops.untile_fp4_scales(s, c.shape[0], c.shape[1] // BLOCK[kind]).cpu().numpy()
    v = VALUES[c].reshape(c.shape[0], -1, BLOCK[kind]) * scale_values(byte, kind)[..., None]
    v = v.reshape(c.shape)
    return v if r is None else v * r.double().cpu().numpy()[:, None]


def check_quantized(hn, x, kind, got):
    q, s, r = got
    codes, byte, rows = define(x, kind)
    assert np.array_equal(unpack(q), codes)
    m = x.shape[0]
    plain = hn.ops.untile_fp4_scales(s, m, byte.shape[1]).cpu().numpy()
    assert np.array_equal(plain, byte)
    # whole tiles: zeros behind the rows and behind the groups
    assert torch.equal(s.cpu(), hn.ops.tile_fp4_scales(torch.from_numpy(byte)))
    if kind == "nvfp4":
        assert np.array_equal(r.cpu().numpy(), rows, equal_nan=True)
    else:
        assert r is None


def randn(shape, seed, dtype=torch.bfloat16, loud=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(shape, generator=g, device="cuda")
    if loud:
        x = x * torch.where(torch.rand(shape[-1], generator=g, device="cuda") < 0.02, 12.0, 1.0)
    return x.to(dtype)


# ------------------------------------------------------------------------------------------------- quantizer

@pytest.mark.parametrize("kind", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("m,k", [(1, 1), (1, 16), (3, 22), (5, 32), (130, 33), (129, 100), (40, 128), (33, 250), (2, 256), (70, 500),
                                 (333, 1040), (9, 2080), (3, 4096), (2, 8190), (2, 16384), (3, 16400), (1, 40001), (1000, 64), (5, 1500), (6, 2040),
                                 (3, 6001), (2, 12000)])
def test_quantize_equals_its_definition(hn, cuda, kind, m, k):
    for dtype in DTYPES:
        x = randn((m, k), m * 7 + k, dtype)
        check_quantized(hn, x, kind, hn.kernels.quantize_fp4(x, kind))


@pytest.mark.parametrize("kind", ["nvfp4", "mxfp4"])
def test_quantize_special_numbers(hn, cuda, kind):
    """Zeros, signed zeros, ties, the largest and smallest numbers, NaN and infinities, each in rows of its own."""
    for dtype, big, small in ((torch.bfloat16, 3.38e38, 1e-40), (torch.float16, 65504.0, 6e-8), (torch.float32, 3.4e38, 1e-45)):
        x = randn((16, 200), 3, dtype, loud=False).float()
        x[0] = 0
        x[1] = -0.0
        x[2, 5] = float("nan")
        x[3, 199] = float("inf")
        x[4, 64] = -float("inf")
        x[5] = big * x[5].clamp(-1, 1)
        x[6] = small
        x[7] *= 1e-31 if dtype != torch.float16 else 1e-7
        x[8, 32:64] = 0
        x[9] = torch.arange(200, device="cuda") * 0.25 % 8          # ties of MX, and of NV with a top of 6
        x[9, 0] = 6.0
        x[10] = -x[9]
        x[11, :] = 1.0
        x[12, 1:] *= 1e-6
        x[13] = 2.0 ** -100 * (1 if dtype != torch.float16 else 0)
        x = x.to(dtype)
        check_quantized(hn, x, kind, hn.kernels.quantize_fp4(x, kind))


@pytest.mark.parametrize("kind", ["nvfp4", "mxfp4"])
def test_quantize_views(hn, cuda, kind):
    """Rows at odd offsets and strides, columns that are not contiguous, an expanded row."""
    base = randn((40, 1000), 1)
    for x in (base[:, 3:500], base[1::3, 8:648], base.t()[:100], base[:1].expand(5, 1000), base[:, :77].float().half(),
              base[:, 2:502], base[:, 2:99].float(), base[:, 998:]):
        check_quantized(hn, x, kind, hn.kernels.quantize_fp4(x, kind))


@pytest.mark.parametrize("kind", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k", [(1, 32), (3, 77), (130, 1000), (5, 4096), (2, 33)])
def test_dequantize(hn, cuda, kind, dtype, m, k):
    """code * RN(scale * row scale), rounded once."""
    q, s, r = hn.kernels.quantize_fp4(randn((m, k), k, torch.float32), kind)
    out = hn.kernels.dequantize_fp4(q, s, r, kind, dtype, columns=k)
    c = unpack(q)
    byte = hn.ops.untile_fp4_scales(s, m, c.shape[1] // BLOCK[kind]).cpu().numpy()
    d = scale_values(byte, kind).astype(np.float32)
    if r is not None:
        d = d * r.cpu().numpy()[:, None]
    v = VALUES[c].astype(np.float32).reshape(m, -1, BLOCK[kind]) * d[..., None]
    want = torch.from_numpy(v.reshape(m, -1)[:, :k].copy()).to(dtype)
    assert out.dtype == dtype and torch.equal(out.cpu(), want)


def test_dequantize_without_row_scales(hn, cuda):
    q, s, r = hn.kernels.quantize_fp4(randn((3, 64), 5), "nvfp4")
    one = torch.ones_like(r)
    assert torch.equal(hn.kernels.dequantize_fp4(q, s), hn.kernels.dequantize_fp4(q, s, one))


def test_values_are_near(hn, cuda):
    """Largest error against the input: half the widest step (2 of 6 + what the scale's rounding adds) of the block's scale."""
    x = randn((64, 4096), 9)
    for kind in ("nvfp4", "mxfp4"):
        v = hn.kernels.dequantize_fp4(*hn.kernels.quantize_fp4(x, kind), kind, torch.float32).double()
        peak = x.double().view(64, -1, BLOCK[kind]).abs().amax(-1, keepdim=True)
        err = (v - x.double()).view(64, -1, BLOCK[kind]).abs()
        top = x.double().abs().amax(-1).view(-1, 1, 1)
        # MX: up to a quarter of the peak (what lies in (6, 8) of the scale goes to 6); NV: 1 / 6 (1 + 2^-4), or, where the scale is
        # an e4m3 below 2^-6, half a step 2^-10 of it times 6 more
        bound = peak / 4 if kind == "mxfp4" else peak / 6 * (1 + 2.0 ** -4) + 6 * 2.0 ** -10 * top / 2688
        assert bool((err <= bound * (1 + 2.0 ** -20)).all())


# ------------------------------------------------------------------------------------------------- product

def operands(hn, m, n, k, kind, seed):
    a = hn.kernels.quantize_fp4(randn((m, k), seed), kind)
    w = hn.kernels.quantize_fp4(randn((n, k), seed + 1), kind)
    return a, w


def check_product(hn, out, a, w, kind, bias=None):
    va, vw = (torch.from_numpy(values64(hn, *t, kind)).cuda() for t in (a, w))
    want, mass = va @ vw.t(), va.abs() @ vw.abs().t()
    bound = mass * (va.shape[1] // 16 * 2.0 ** -23) + (want.abs() + mass * 2.0 ** -20) * 3 * 2.0 ** -24
    if bias is not None:
        want = want + bias.double()
        bound = bound + want.abs() * 2.0 ** -24
    bound = bound + (want.abs() + bound) * (torch.finfo(out.dtype).eps / 2) + torch.finfo(out.dtype).smallest_normal * 2.0 ** -10
    err = (out.double() - want).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


@pytest.mark.parametrize("kind", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 130, 32), (1, 257, 4096), (2, 8, 96), (3, 1000, 2080), (4, 300, 16416), (1, 4096, 1000)])
def test_few_rows(hn, cuda, kind, m, n, k):
    a, w = operands(hn, m, n, k, kind, 11)
    for dtype in DTYPES:
        check_product(hn, hn.kernels.fp4_gemm(*a, *w, kind=kind, out_dtype=dtype), a, w, kind)


@pytest.mark.parametrize("kind", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("m,n,k", [(5, 1, 32), (5, 128, 64), (16, 128, 256), (17, 130, 96), (48, 257, 512), (128, 128, 1024),
                                   (129, 100, 160), (130, 1001, 2080), (300, 5001, 320), (48, 256, 16384), (7, 8, 40000),
                                   (700, 700, 700), (257, 512, 4096), (9, 19000, 256), (777, 5001, 352), (1300, 1700, 2400)])
def test_product(hn, cuda, kind, m, n, k):
    a, w = operands(hn, m, n, k, kind, 12)
    for dtype in DTYPES:
        check_product(hn, hn.kernels.fp4_gemm(*a, *w, kind=kind, out_dtype=dtype), a, w, kind)


@pytest.mark.parametrize("kind", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("m,n,k", [(2304, 2304, 256), (2100, 2300, 160), (20000, 130, 64), (257, 9500, 2080), (4700, 1101, 4128),
                                   (9472, 512, 96)])
def test_product_many_rows(hn, cuda, kind, m, n, k):
    a, w = operands(hn, m, n, k, kind, 13)
    for dtype in DTYPES:
        check_product(hn, hn.kernels.fp4_gemm(*a, *w, kind=kind, out_dtype=dtype), a, w, kind)


@pytest.mark.parametrize("kind", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("n", [2064, 2068, 2066, 2065])
@pytest.mark.parametrize("m,k", [(1793, 2080), (2600, 96), (1200, 1312)])
def test_product_rows_of_any_alignment(hn, cuda, kind, n, m, k):
    """Pairs of CTAs, a tile each and several: outputs stored 16, 8, 4 and 2 bytes at a time."""
    a, w = operands(hn, m, n, k, kind, 14)
    for dtype in DTYPES:
        for pad in (0, 16):
            base = torch.full((m, n + pad), 7.0, dtype=dtype, device="cuda")
            out = base[:, :n]
            hn.kernels.fp4_gemm(*a, *w, None, dtype, kind, out)
            check_product(hn, out, a, w, kind)
            assert bool((base[:, n:] == 7).all())


@pytest.mark.parametrize("kind", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("m,n,k", [(1, 40, 96), (2, 300, 2080), (20, 300, 512), (130, 200, 4096), (2500, 2400, 128)])
def test_product_nan_stays_in_its_row_and_column(hn, cuda, kind, m, n, k):
    """A NaN or an infinity in a row of either operand: its outputs are NaN, all others as without it."""
    x, y = randn((m, k), 1), randn((n, k), 2)
    clean = hn.kernels.fp4_gemm(*hn.kernels.quantize_fp4(x, kind), *hn.kernels.quantize_fp4(y, kind), kind=kind, out_dtype=torch.float32)
    x[m - 1, k - 1], y[n // 2, 0], y[n - 1, k // 2] = float("nan"), float("inf"), float("nan")
    out = hn.kernels.fp4_gemm(*hn.kernels.quantize_fp4(x, kind), *hn.kernels.quantize_fp4(y, kind), kind=kind, out_dtype=torch.float32)
    bad = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    bad[m - 1], bad[:, n // 2], bad[:, n - 1] = True, True, True
    assert bool(out[bad].isnan().all()) and torch.equal(out[~bad], clean[~bad])


@pytest.mark.parametrize("kind", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("m,n,k", [(1, 300, 512), (60, 301, 512), (600, 301, 96), (2500, 2401, 96), (2500, 2400, 96)])
def test_product_bias_out_and_views(hn, cuda, kind, m, n, k):
    """Biases of all types at odd addresses, outputs with strided rows at odd addresses, codes with strided rows."""
    a, w = operands(hn, m, n, k, kind, 21)
    wide = torch.zeros((m, k), dtype=torch.uint8, device="cuda")
    wide[:, :k // 2] = a[0]
    av = (wide[:, :k // 2], a[1], a[2])
    for bias_dtype in DTYPES:
        for out_dtype in DTYPES:
            bias = randn((n + 1,), 3, bias_dtype, loud=False)[1:]
            base = torch.full((m, n + 6), 7.0, dtype=out_dtype, device="cuda")
            out = base[:, 3:n + 3]
            assert hn.kernels.fp4_gemm(*av, *w, bias, out_dtype, kind, out) is out
            check_product(hn, out, a, w, kind, bias)
            assert bool((base[:, :3] == 7).all()) and bool((base[:, n + 3:] == 7).all())


def test_product_without_row_scales(hn, cuda):
    a, w = operands(hn, 70, 50, 320, "nvfp4", 5)
    one = lambda t: (t[0], t[1], torch.ones_like(t[2]))  # noqa: E731
    for m in (1, 70):
        q, s, r = hn.kernels.quantize_fp4(randn((m, 320), 9), "nvfp4")
        assert torch.equal(hn.kernels.fp4_gemm(q, s, None, w[0], w[1], None), hn.kernels.fp4_gemm(*one((q, s, r)), *one(w)))
        assert torch.equal(hn.kernels.fp4_gemm(q, s, r, w[0], w[1], None), hn.kernels.fp4_gemm(q, s, r, *one(w)))


def test_product_largest_scales(hn, cuda):
    """MX scales from 2^-127 to 2^120. With s = 2^(ea + ew - 254) every partial sum is a multiple of s / 4 up to 2^14 s: exact in fp32
    from ea + ew = 130 on (s / 4 = 2^-126) while 2^14 s stays finite (ea + ew < 366); below, each of 16 partial sums may lose what
    lies under the smallest normal number; above, what is infinite is not finite (infinities of both signs may meet)."""
    a, w = operands(hn, 5, 130, 256, "mxfp4", 6)
    va, vw = (torch.from_numpy(VALUES[unpack(t[0])]).cuda() for t in (a, w))
    sums = va @ vw.t()                                    # exact: small integers times 0.25
    for ea, ew in ((1, 100), (0, 140), (127, 127), (200, 60), (247, 127), (247, 200), (0, 0)):
        sa, sw = torch.full_like(a[1], ea), torch.full_like(w[1], ew)
        want = (sums * 2.0 ** (ea + ew - 254)).float()
        for m in (1, 5):
            out = hn.kernels.fp4_gemm(a[0][:m].contiguous(), sa, None, w[0], sw, None, kind="mxfp4", out_dtype=torch.float32)
            if 130 <= ea + ew < 366:
                assert torch.equal(out, want[:m]), (ea, ew, m)
            elif ea + ew < 130:
                assert bool(((out - want[:m]).abs() <= 16 * 2.0 ** -126).all()), (ea, ew, m)
            else:
                assert not bool(out[want[:m].isinf()].isfinite().any()), (ea, ew, m)


def test_linear(hn, cuda):
    x = randn((3, 5, 100), 7)
    w = hn.kernels.quantize_fp4(randn((40, 100), 8), "nvfp4")
    bias = randn((40,), 9, loud=False)
    y = hn.kernels.fp4_linear(x, *w, bias)
    assert y.shape == (3, 5, 40) and y.dtype == torch.bfloat16
    assert torch.equal(y.view(15, 40), hn.kernels.fp4_gemm(*hn.kernels.quantize_fp4(x.view(15, 100)), *w, bias))
    assert hn.kernels.fp4_linear(x[:0], *w).shape == (0, 5, 40) and hn.kernels.fp4_linear(x[0, 0], *w).shape == (40,)
    assert hn.kernels.fp4_linear(x.float(), *w).dtype == torch.float32
    for bad, error in ((lambda: hn.kernels.fp4_linear(x[..., :60], *w), ValueError), (lambda: hn.kernels.fp4_linear(x.long(), *w), TypeError)):
        with pytest.raises(error):
            bad()


def test_stacked(hn, cuda):
    """Linears stacked along N give their outputs side by side, for every kernel."""
    for m in (1, 30, 3000):
        x = hn.kernels.quantize_fp4(randn((m, 288), m))
        parts = [hn.kernels.quantize_fp4(randn((n, 288), n)) for n in (128, 1280, 1000)]
        both = hn.kernels.fp4_gemm(*x, *hn.ops.stack_fp4_linears(*parts))
        assert torch.equal(both, torch.cat([hn.kernels.fp4_gemm(*x, *p) for p in parts], 1))


def test_refusals(hn, cuda):
    K = hn.kernels
    a, w = operands(hn, 5, 40, 96, "nvfp4", 3)
    x = randn((5, 96), 1)
    for bad, error in ((lambda: K.quantize_fp4(x, "fp4"), ValueError), (lambda: K.quantize_fp4(x[0]), ValueError),
                       (lambda: K.quantize_fp4(x[:, :0]), ValueError), (lambda: K.dequantize_fp4(*a, columns=64), ValueError),
                       (lambda: K.dequantize_fp4(*a, columns=97), ValueError), (lambda: K.dequantize_fp4(*a, dtype=torch.int8), TypeError),
                       (lambda: K.dequantize_fp4(*a, "mxfp4"), ValueError), (lambda: K.dequantize_fp4(a[0], a[1], a[2][:4]), ValueError),
                       (lambda: K.dequantize_fp4(a[0], a[1].cpu(), a[2]), RuntimeError),
                       (lambda: K.fp4_gemm(*a, *w, kind="mxfp4"), ValueError), (lambda: K.fp4_gemm(*a, w[0][:, :32], w[1][:, :1], w[2]), ValueError),
                       (lambda: K.fp4_gemm(*a, w[0][:0], w[1][:0], w[2][:0]), ValueError), (lambda: K.fp4_gemm(a[0].int(), *a[1:], *w), ValueError),
                       (lambda: K.fp4_gemm(a[0], a[1][:, :1], a[2], *w), ValueError), (lambda: K.fp4_gemm(a[0], a[1], a[2].double(), *w), ValueError),
                       (lambda: K.fp4_gemm(*a, *w, out_dtype=torch.int32), TypeError), (lambda: K.fp4_gemm(*a, *w, bias=x[0]), ValueError),
                       (lambda: K.fp4_gemm(*a, *w, bias=x[0, :40].cpu()), RuntimeError), (lambda: K.fp4_gemm(*a, w[0].cpu(), *w[1:]), RuntimeError),
                       (lambda: K.fp4_gemm(*a, *w, out=x), ValueError), (lambda: K.fp4_gemm(*a, *w, out=x[:1, :40].expand(5, 40)), ValueError)):
        with pytest.raises(error):
            bad()
    assert K.fp4_gemm(*(t[:0] for t in a), *w).shape == (0, 40)
    assert K.dequantize_fp4(*(t[:0] for t in a)).shape == (0, 96)
    q = K.quantize_fp4(x[:0])
    assert q[0].shape == (0, 48) and q[1].shape == (0, 2, 512) and q[2].shape == (0,)


def test_product_leaves_reserved_sms(hn, cuda):
    """The GEMMs' SM reserve holds for the persistent kernel, too; its results do not depend on it."""
    a, w = operands(hn, 2500, 2400, 96, "nvfp4", 30)
    want = hn.kernels.fp4_gemm(*a, *w)
    L, was = hn.lib.lib, hn.lib.lib.hn_get_gemm_sm_reserve()
    try:
        for n in (1, 20, 64):
            assert L.hn_set_gemm_sm_reserve(n) == 0
            assert torch.equal(hn.kernels.fp4_gemm(*a, *w), want)
    finally:
        L.hn_set_gemm_sm_reserve(was)
