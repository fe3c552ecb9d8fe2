"""The 4-bit product at the ends of its scales: powers of two far apart, every e4m3 block scale, NaN scales, row scales whose product
with a sum leaves fp32 though the output does not. By each of its kernels: one and two rows, some rows, many."""
import numpy as np
import pytest
import torch

from test_gpu_fp4 import VALUES, check_product, operands, randn, unpack

pytestmark = pytest.mark.gpu
SIZES = [(1, 130, 256), (2, 130, 256), (5, 130, 256), (300, 257, 96), (2500, 2400, 96)]
PARTS = [(48, 300, 1024), (48, 300, 2048), (48, 300, 4096)]         # K over two, four and eight CTAs


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("ea,ew", [(252, 100), (100, 252), (254, 0), (0, 254), (254, 3), (252, 113), (130, 1), (1, 130), (180, 180)])
def test_powers_far_apart(hn, cuda, m, n, k, ea, ew):
    """Scales 2^(ea - 127) and 2^(ew - 127). Partial sums are multiples of 2^(ea + ew - 256) below 2^14 2^(ea + ew - 254): exact in fp32
    for the sums ea + ew here (from 130 to 365), whatever each of the two is alone."""
    assert 130 <= ea + ew < 366
    a, w = operands(hn, m, n, k, "mxfp4", 40)
    va, vw = (torch.from_numpy(VALUES[unpack(t[0])]).cuda() for t in (a, w))
    want = (va @ vw.t() * 2.0 ** (ea + ew - 254)).float()               # the sums are exact: small integers times 0.25
    assert bool(want.isfinite().all())
    sa, sw = torch.full_like(a[1], ea), torch.full_like(w[1], ew)
    out = hn.kernels.fp4_gemm(a[0], sa, None, w[0], sw, None, kind="mxfp4", out_dtype=torch.float32)
    assert torch.equal(out, want)


@pytest.mark.parametrize("m,n,k", SIZES)
def test_powers_far_apart_block_by_block(hn, cuda, m, n, k):
    """Blocks whose two scales are far apart in turn, one way and the other: their products are all 2^98, and the sums exact."""
    a, w = operands(hn, m, n, k, "mxfp4", 41)
    va, vw = (torch.from_numpy(VALUES[unpack(t[0])]).cuda() for t in (a, w))
    groups = k // 32
    turn = torch.arange(groups, device="cuda") % 2 == 0
    pa, pw = torch.where(turn, 252, 100).to(torch.uint8), torch.where(turn, 100, 252).to(torch.uint8)
    sa, sw = (hn.ops.tile_fp4_scales(p.expand(rows, groups)) for p, rows in ((pa, m), (pw, n)))
    out = hn.kernels.fp4_gemm(a[0], sa, None, w[0], sw, None, kind="mxfp4", out_dtype=torch.float32)
    assert torch.equal(out, (va @ vw.t() * 2.0 ** 98).float())


@pytest.mark.parametrize("m,n,k", SIZES + PARTS)
def test_large_activations_small_weights(hn, cuda, m, n, k):
    """From the quantizer on: rows near 2^126 against weights near 2^-30, mxfp4."""
    x, y = randn((m, k), 1, loud=False).float() * 2.0 ** 124, randn((n, k), 2, loud=False).float() * 2.0 ** -30
    a, w = hn.kernels.quantize_fp4(x, "mxfp4"), hn.kernels.quantize_fp4(y, "mxfp4")
    for dtype in (torch.bfloat16, torch.float32):
        check_product(hn, hn.kernels.fp4_gemm(*a, *w, kind="mxfp4", out_dtype=dtype), a, w, "mxfp4")


@pytest.mark.parametrize("m,n,k", SIZES + PARTS)
def test_every_e4m3_scale(hn, cuda, m, n, k):
    """Block scales from all bytes 0 to 126: zero, the subnormals, 448."""
    a, w = operands(hn, m, n, k, "nvfp4", 42)
    gen = torch.Generator(device="cuda").manual_seed(7)
    sa, sw = (hn.ops.tile_fp4_scales(torch.randint(0, 127, (rows, k // 16), device="cuda", dtype=torch.uint8, generator=gen))
              for rows in (m, n))
    a, w = (a[0], sa, a[2]), (w[0], sw, w[2])
    for dtype in (torch.bfloat16, torch.float32):
        check_product(hn, hn.kernels.fp4_gemm(*a, *w, kind="nvfp4", out_dtype=dtype), a, w, "nvfp4")
    # subnormal scales alone: the sums are multiples of 2^-20
    low = tuple(hn.ops.tile_fp4_scales(torch.randint(0, 8, (rows, k // 16), device="cuda", dtype=torch.uint8, generator=gen))
                for rows in (m, n))
    out = hn.kernels.fp4_gemm(a[0], low[0], None, w[0], low[1], None, out_dtype=torch.float32)
    check_product(hn, out, (a[0], low[0], None), (w[0], low[1], None), "nvfp4")


@pytest.mark.parametrize("kind,nan", [("nvfp4", 127), ("mxfp4", 255)])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_nan_scale(hn, cuda, kind, nan, m, n, k):
    """A NaN block scale of either operand: the outputs of its row or column are NaN, all others as without it."""
    a, w = operands(hn, m, n, k, kind, 43)
    clean = hn.kernels.fp4_gemm(*a, *w, kind=kind, out_dtype=torch.float32)
    groups = k // (16 if kind == "nvfp4" else 32)
    sa, sw = hn.ops.untile_fp4_scales(a[1], m, groups), hn.ops.untile_fp4_scales(w[1], n, groups)
    sa[m - 1, groups - 1], sw[n // 2, 0] = nan, nan
    out = hn.kernels.fp4_gemm(a[0], hn.ops.tile_fp4_scales(sa), a[2], w[0], hn.ops.tile_fp4_scales(sw), w[2], kind=kind,
                              out_dtype=torch.float32)
    bad = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    bad[m - 1], bad[:, n // 2] = True, True
    assert bool(out[bad].isnan().all()) and torch.equal(out[~bad], clean[~bad])


@pytest.mark.parametrize("m,n,k", SIZES + PARTS)
def test_row_scales_far_apart(hn, cuda, m, n, k):
    """nvfp4 rows of activations near 2^120 against weights near 2^-60, and the other way: the sum times the larger row scale alone
    leaves fp32, the output does not."""
    for big, small in ((2.0 ** 118, 2.0 ** -60), (2.0 ** -60, 2.0 ** 118)):
        x, y = randn((m, k), 1, loud=False).float() * big, randn((n, k), 2, loud=False).float() * small
        if m > 2:
            x[1::2] = randn((x[1::2].shape[0], k), 3, loud=False).float() * min(big, 1.0)      # rows of both sorts side by side
        a, w = hn.kernels.quantize_fp4(x), hn.kernels.quantize_fp4(y)
        for dtype in (torch.bfloat16, torch.float32):
            out = hn.kernels.fp4_gemm(*a, *w, out_dtype=dtype)
            assert bool(out.isfinite().all())
            check_product(hn, out, a, w, "nvfp4")
