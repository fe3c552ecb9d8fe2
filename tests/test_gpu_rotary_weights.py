"""Norm weights in their own type: fp32 and fp16 weights reach the norm without a rounding, in `rotate` and in the append. The bounds are
those of test_gpu_rotary.py (a weight rounded to bf16 would be 2^-9 off)."""
import pytest
import torch

from test_gpu_rotary import check, check_int8, filled, randn, turned

pytestmark = pytest.mark.gpu
WEIGHTS = [torch.float32, torch.float16, torch.float64]


@pytest.fixture()
def rotary(hn):
    from hy_nomas_b200 import rotary
    return rotary


@pytest.fixture()
def paged(hn):
    from hy_nomas_b200 import paged
    return paged


def weight(d, seed, dtype):
    w = 1 + 0.3 * torch.randn(d, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")
    return w.to(dtype)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("wdtype", WEIGHTS)
@pytest.mark.parametrize("d,r", [(16, 16), (24, 8), (40, 32), (64, 48), (96, 96), (128, 120), (128, 128), (136, 128), (200, 16), (256, 256)])
def test_rotate(rotary, cuda, layout, wdtype, d, r):
    rot, w = rotary.Rotary(r, 10000.0, layout), weight(d, d, wdtype)
    pos = torch.arange(7, device="cuda") + 90
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        x = randn((2, 7, 5, d), r, dtype)
        check(rotary.rotate(x, pos, rot, w), x, pos, rot, w.float())
        odd = torch.empty(d + 1, dtype=wdtype, device="cuda")[1:].copy_(w)          # at no 16-byte boundary
        assert torch.equal(rotary.rotate(x, pos, rot, odd), rotary.rotate(x, pos, rot, w))
        bf16 = w.to(torch.bfloat16)
        assert torch.equal(rotary.rotate(x, pos, rot, bf16), rotary.rotate(x, pos, rot, bf16.to(wdtype)))


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("layout,r", [("half", 128), ("half", 120), ("interleaved", 64), ("interleaved", 8)])
@pytest.mark.parametrize("wq,wk", [(torch.float32, torch.float32), (torch.float32, None), (None, torch.float16),
                                   (torch.bfloat16, torch.float32), (torch.float16, torch.bfloat16)])
def test_append(paged, rotary, cuda, kind, layout, r, wq, wk):
    """q' and K against 64 bits, and q' as `rotate` gives it, whatever types the two weights have."""
    c = filled(paged, 20, 2, 16, 2, 8, kind, 1)
    c.extend([0], 9)
    c.extend([1, 0], 21)
    q, k, v = (randn((2, 21, n, 128), n) for n in (5, 2, 2))
    rot = rotary.Rotary(r, 10000.0, layout)
    wq, wk = (None if t is None else weight(128, i, t) for i, t in enumerate((wq, wk)))
    out = c.append_rotated(1, q, k, v, [1, 0], rot, wq, wk)
    pos = torch.arange(21, device="cuda") + torch.tensor([[0], [9]], device="cuda")
    check(out, q, pos, rot, None if wq is None else wq.float())
    assert torch.equal(out, rotary.rotate(q, pos, rot, wq))
    k64, mass = turned(k, pos, rot, None if wk is None else wk.float())
    if kind == "int8":
        check_int8(c, 1, [1, 0], 21, k64, mass, v)
    else:
        for i, row in enumerate((1, 0)):
            page, place = c.table[row].long()[pos[i] // 16], pos[i] % 16
            got = c.k[1][page, :, place].double()
            assert bool(((got - k64[i]).abs() <= mass[i] * 2.0 ** -20 + (k64[i].abs() + mass[i] * 2.0 ** -20) * 2.0 ** -8).all())
    c.check()
