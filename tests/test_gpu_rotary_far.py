"""Far positions against the angles themselves, worked out with 60 digits: a frequency is held to 2^-65 of a turn, so at position p an
angle is off by 2 pi p 2^-65 more than the kernel's own 2^-20 (test_gpu_rotary.py)."""
import math
from decimal import Context, Decimal, localcontext

import pytest
import torch

from test_gpu_rotary import randn

pytestmark = pytest.mark.gpu
PI = Decimal("3.14159265358979323846264338327950288419716939937510582097494459")


def angles(p, dim, theta):
    """p theta^(-2 i / dim) modulo 2 pi, within (-pi, pi)."""
    with localcontext(Context(prec=60)):
        turns = [p * (Decimal(theta) ** (Decimal(-2 * i) / dim)) / (2 * PI) for i in range(dim // 2)]
        return [float((t - t.to_integral_value()) * 2 * PI) for t in turns]


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,theta", [(128, 10000), (64, 1000000), (24, 500000)])
def test_far_positions(hn, cuda, layout, dim, theta):
    from hy_nomas_b200 import rotary
    rot = rotary.Rotary(dim, theta, layout)
    for p in (3, 100000, 2 ** 31 - 1, -2 ** 31, -2 ** 36 - 17, 2 ** 40 + 12345, 2 ** 44 + 1):
        x = randn((1, 1, 3, dim), 5, torch.float32)
        out = rotary.rotate(x, torch.tensor([p], device="cuda"), rot)
        a = torch.tensor(angles(p, dim, theta), dtype=torch.float64, device="cuda")
        c, s = torch.cos(a), torch.sin(a)
        i = torch.arange(dim // 2, device="cuda")
        j, l = (i, i + dim // 2) if layout == "half" else (2 * i, 2 * i + 1)
        u, v = x.double()[..., j], x.double()[..., l]
        bound = (u.abs() + v.abs()) * (2.0 ** -20 + 2 * math.pi * abs(p) * 2.0 ** -65)
        assert bool(((out.double()[..., j] - (u * c - v * s)).abs() <= bound).all()), p
        assert bool(((out.double()[..., l] - (v * c + u * s)).abs() <= bound).all()), p


def test_out_whose_heads_overlap_is_refused(hn, cuda):
    from hy_nomas_b200 import rotary
    rot, pos = rotary.Rotary(64), torch.arange(3, device="cuda")
    base = randn((4096,), 1)
    kept = base.clone()
    x = randn((2, 3, 4, 64), 2)
    for strides in ((768, 256, 56), (768, 192, 64), (256, 256, 64), (8, 1024, 64)):
        out = base.as_strided((2, 3, 4, 64), strides + (1,))
        for src in (x, out):                                    # another tensor, and in place
            with pytest.raises(ValueError, match="overlap"):
                rotary.rotate(src, pos, rot, out=out)
    assert torch.equal(base, kept)
    out = base.as_strided((2, 3, 4, 64), (64, 512, 128, 1))     # batches between heads: apart
    assert torch.equal(rotary.rotate(x, pos, rot, out=out), rotary.rotate(x, pos, rot))
