"""The residual's addition + RMSNorm + quantizer (fused.add_rmsnorm_quant) against the definition in 64 bits.

The sum is the fp32 sum rounded once to bf16: equal bits. In fp32, y carries the error of the mean of squares (a sum of at
most 16384 positive terms in a tree: below 2^-18) and of a few roundings, so a scale is within 1e-5 of the exact one, and a
code is within half a step of y / scale, plus 2e-5 of the largest code.
"""
import ctypes
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

CASES = [(1, 128), (1, 4096), (3, 256), (5, 384), (129, 640), (64, 1024), (7, 1152), (33, 2048), (2, 2944), (17, 4096),
         (9, 4224), (5, 8192), (3, 12288), (2, 16384), (1000, 128)]


def data(rows, d, device, seed):
    g = torch.Generator(device=device).manual_seed(seed)
    x = torch.randn((rows, d), generator=g, device=device).to(torch.bfloat16)
    r = (torch.randn((rows, d), generator=g, device=device) * 3).to(torch.bfloat16)
    w = (1 + 0.3 * torch.randn(d, generator=g, device=device)).to(torch.bfloat16)
    return x, r, w


def check(x, r, w, eps, kind, per_token, total, q, s):
    rows, d = x.shape
    h32 = x.float() + r.float()
    assert torch.equal(total.view(torch.int16), h32.to(torch.bfloat16).view(torch.int16))
    h = x.double() + r.double()
    y = h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps) * w.double()
    y = y.view(rows, 1 if per_token else d // 128, -1)
    peak = y.abs().amax(-1)
    want = torch.where(peak > 0, peak / 127, 1.0) if kind == "int8" else peak.clamp_min(1e-12) / 448
    assert s.shape == want.shape and s.dtype == torch.float32
    assert ((s.double() - want).abs() <= 1e-5 * want).all()
    t = y / s.double()[..., None]
    codes = q.float().double().view(t.shape)
    err = (codes - t).abs()
    if kind == "int8":
        assert q.dtype == torch.int8 and (err <= 0.5 + 127 * 2e-5).all()
    else:
        # e4m3: 3 bits after the leading one, steps of 2^-9 below 2^-6
        step = torch.exp2(torch.floor(torch.log2(t.abs().clamp_min(2.0 ** -6))) - 3)
        assert q.dtype == torch.float8_e4m3fn and (err <= step / 2 + 448 * 2e-5).all()


@pytest.mark.parametrize("per_token", [False, True])
@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("rows,d", CASES)
def test_against_64_bits(hn, cuda, rows, d, kind, per_token):
    x, r, w = data(rows, d, cuda, rows + d)
    got = hn.fused.add_rmsnorm_quant(x, r, w, 1e-6, kind, per_token)
    check(x, r, w, 1e-6, kind, per_token, *got)
    again = hn.fused.add_rmsnorm_quant(x, r, w, 1e-6, kind, per_token)
    assert all(a.cpu().numpy().tobytes() == b.cpu().numpy().tobytes() if a.dtype == torch.float32 else
               torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, again))


def test_views_and_in_place(hn, cuda):
    """Strided rows, a misaligned view, leading dimensions, an expanded residual; the stream updated in place."""
    x, r, w = data(12, 512, cuda, 1)
    wide = torch.zeros((12, 1024), dtype=torch.bfloat16, device=cuda)
    wide[:, 256:768] = x
    want = hn.fused.add_rmsnorm_quant(x, r, w)
    odd = torch.zeros(12 * 512 + 1, dtype=torch.bfloat16, device=cuda)[1:].view(12, 512)
    odd.copy_(r)
    for a, b in ((wide[:, 256:768], r), (x, odd), (x.view(3, 4, 512), r.view(3, 4, 512))):
        got = hn.fused.add_rmsnorm_quant(a, b, w)
        assert got[0].shape == a.shape
        assert torch.equal(got[0].reshape(12, 512), want[0]) and torch.equal(got[1].view(torch.uint8), want[1].view(torch.uint8))
        assert torch.equal(got[2], want[2])
    row = r[:1].expand(12, 512)
    a, b = hn.fused.add_rmsnorm_quant(x, row, w), hn.fused.add_rmsnorm_quant(x, row.contiguous(), w)
    assert torch.equal(a[0], b[0]) and torch.equal(a[2], b[2])
    stream = x.clone()
    total, q, s = hn.fused.add_rmsnorm_quant(stream, r, w, out=stream)
    assert total is stream and torch.equal(stream, want[0]) and torch.equal(s, want[2])
    assert hn.fused.add_rmsnorm_quant(x[:0], r[:0], w)[1].shape == (0, 512)


@pytest.mark.parametrize("kind,per_token", [("fp8", False), ("int8", False), ("int8", True)])
def test_permuted_inputs(hn, cuda, kind, per_token):
    """Dense tensors whose dimensions are stored in another order (tokens first): the sum's rows are the inputs' rows."""
    x, r, w = data(30, 256, cuda, 7)
    x, r = x.view(5, 3, 2, 256), r.view(5, 3, 2, 256)
    for order in ((1, 0, 2, 3), (2, 1, 0, 3), (1, 2, 0, 3)):
        a, b = x.permute(order), r.permute(order)
        want = hn.fused.add_rmsnorm_quant(a.contiguous(), b.contiguous(), w, kind=kind, per_token=per_token)
        for u, v in ((a, b), (a.contiguous(), b), (a, b.contiguous())):
            got = hn.fused.add_rmsnorm_quant(u, v, w, kind=kind, per_token=per_token)
            assert got[0].shape == a.shape and torch.equal(got[0], want[0])
            assert torch.equal(got[1].view(torch.uint8), want[1].view(torch.uint8)) and torch.equal(got[2], want[2])
            check(a.reshape(-1, 256), b.reshape(-1, 256), w, 1e-6, kind, per_token, got[0].reshape(-1, 256), *got[1:])


def test_zeros_nan_and_infinity(hn, cuda):
    x, r, w = data(4, 256, cuda, 2)
    x[0], r[0] = 0, 0
    x[1, 5] = math.nan
    x[2, 200], r[3, 3] = math.inf, -math.inf
    for kind in ("int8", "fp8"):
        for per_token in (False, True):
            total, q, s = hn.fused.add_rmsnorm_quant(x, r, w, kind=kind, per_token=per_token)
            assert (total[0] == 0).all() and (q[0].float() == 0).all()
            assert torch.allclose(s[0], torch.full_like(s[0], 1.0 if kind == "int8" else 1e-12 / 448))
            assert torch.isnan(s[1]).all() and torch.isnan(total[1, 5])
            assert torch.isnan(s[2]).any() and torch.isnan(s[3]).any()      # inf / inf: the group that holds it


def test_linear_reads_its_output(hn, cuda):
    """Codes and scales go to the GEMM as the activation quantizer's do."""
    x, r, w = data(40, 512, cuda, 3)
    weight = torch.randn((256, 512), device=cuda) * 0.05
    for kind, per_token in (("int8", False), ("int8", True), ("fp8", False)):
        total, q, s = hn.fused.add_rmsnorm_quant(x, r, w, kind=kind, per_token=per_token)
        if kind == "fp8":
            qw, sw = hn.ops.quantize_fp8_block(weight)
            dense = hn.ops.dequantize_fp8_block(qw, sw, torch.float64)
        else:
            qw, sw = hn.ops.quantize_g128(weight)
            dense = hn.ops.dequantize_g128(qw, sw, torch.float64)
            if per_token:
                sw = weight.abs().amax(1) / 127
                qw = (weight / sw[:, None]).round().to(torch.int8)
                dense = qw.double() * sw.double()[:, None]
        y = hn.kernels.block_gemm(q, s, qw, sw, kind=kind)
        h = x.double() + r.double()
        n = h / torch.sqrt(h.square().mean(-1, keepdim=True) + 1e-6) * w.double()
        want = n @ dense.T
        assert float((y.double() - want).norm() / want.norm()) < (0.04 if kind == "fp8" else 0.02)


def test_refusals(hn, cuda):
    x, r, w = data(4, 256, cuda, 4)
    f = hn.fused.add_rmsnorm_quant
    for args, kw in (((x.float(), r, w), {}), ((x, r[:3], w), {}), ((x, r, w[:128]), {}), ((x.cpu(), r, w), {}),
                     ((x, r, w), dict(out=r[:2])), ((x, r, w), dict(kind="fp4")), ((x[:, :200], r[:, :200], w[:200]), {})):
        with pytest.raises((ValueError, TypeError, RuntimeError, KeyError)):
            f(*args, **kw)
    L = hn.lib.lib
    st = hn.lib.stream_of(x)
    s = torch.empty((4, 2), device=cuda)
    q = torch.empty((4, 256), dtype=torch.int8, device=cuda)

    def call(**kw):
        a = dict(x=x.data_ptr(), ldx=256, r=r.data_ptr(), ldr=256, w=w.data_ptr(), rows=4, d=256, eps=1e-6, kind=0, flags=0,
                 out=x.data_ptr(), ldo=256, q=q.data_ptr(), ldq=256, s=s.data_ptr(), rs=2, gs=1)
        a.update(kw)
        return L.hn_add_rmsnorm_quant(*a.values(), st)
    assert call(x=None) == 5 and call(kind=2) == 5 and call(flags=2) == 5 and call(d=200) == 1 and call(d=16512) == 1
    assert call(ldx=128) == 1 and call(ldr=260) == 2 and call(q=q.data_ptr() + 4) == 2 and call(gs=2) == 1
    assert call() == 0
    assert ctypes.c_void_p(x.data_ptr()).value
    torch.cuda.synchronize()
