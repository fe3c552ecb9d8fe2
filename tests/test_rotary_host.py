"""Host checks of the rotations beside those of test_more_host.py, through the C ABI (CPU only; no pointer is ever followed)."""
import math
from fractions import Fraction

import pytest
import torch

from test_more_host import refused, rotation
from test_paged_host import FAKE, ref, struct


@pytest.fixture()
def paged(hn):
    from hy_nomas_b200 import paged
    return paged


def rotate_args(**kw):
    return dict(dict(x=FAKE, xb=1536, xl=512, xh=128, dt=0), **rotation(), w=FAKE, eps=1e-6, B=2, L=3, H=4, D=128, out=FAKE, ob=1536,
                ol=512, oh=128, stream=None, **kw)


def append_args(cache):
    good = dict(cache=ref(cache), layer=0)
    for name in "qkv":
        good.update({name: FAKE, name + "b": 512, name + "t": 128, name + "h": 128})
        if name == "q":
            good["H"] = 8
    return dict(good, rows=FAKE, B=2, n=3, **rotation(), wq=FAKE, wk=None, eps=1e-6, out=FAKE, stream=None)


def test_layout_tells_the_weights_type(hn, paged):
    """The layout with HN_ROPE_NORM_FP32 (16) is taken, any other bit is not."""
    cache = struct(paged, refused=FAKE, epoch=1)
    for name, good, empty in (("hn_rotate", rotate_args(), dict(B=0, x=None)),
                              ("hn_cache_append_rotated", append_args(cache), dict(B=0, q=None, rows=None))):
        for layout in (0, 1, 16, 17):
            assert getattr(hn.lib.lib, name)(*dict(good, layout=layout, **empty).values()) == 0
        refused(hn, name, good, [(dict(layout=n), 5) for n in (2, 8, 18, 32, 33, -1, -16)])
        refused(hn, name, good, [(dict(layout=16, **{"w" if name == "hn_rotate" else "wq": FAKE + 8}), 2)])


@pytest.mark.parametrize("strides,apart", [
    ((1536, 512, 128), True), ((512, 1024, 128), True), ((128, 1024, 256), True), ((1536, 128, 384), True), ((-1536, -512, -128), True),
    ((1536, 512, 64), False), ((1536, 512, 0), False), ((512, 512, 128), False), ((1024, 512, 128), False), ((0, 512, 128), False),
    ((1536, 384, 128), False), ((120, 1024, 256), False), ((-1536, -504, 128), False)])
def test_rotate_refuses_heads_of_out_that_overlap(hn, strides, apart):
    """B = 2, L = 3, H = 4 heads of 128: refused in the library and seen in the Python layer."""
    from hy_nomas_b200 import rotary
    if not apart:
        good = rotate_args()
        refused(hn, "hn_rotate", good, [(dict(zip(("ob", "ol", "oh"), strides)), 1)])
    low = -sum(min(0, s * (n - 1)) for s, n in zip(strides, (2, 3, 4)))
    if low == 0:
        assert rotary._apart(torch.empty(8192).as_strided((2, 3, 4, 128), strides + (1,))) == apart
    assert rotary._apart(torch.empty(8192).as_strided((1, 1, 1, 128), (0, 8, 0, 1)))


PI = Fraction(3141592653589793238462643383279502884197, 10 ** 39)           # cut, so pi is less than 10^-39 above


@pytest.mark.parametrize("dim,theta", [(8, 10000.0), (64, 10000.0), (128, 500000.0), (256, 1e6), (96, 1.5)])
@pytest.mark.parametrize("factor", [None, 4.0])
def test_fixed_point_frequencies_are_the_nearest(hn, dim, theta, factor):
    """freq / 2^64 turns a position is theta^(-2 i / dim) / (2 pi) (over the factor) to the nearest: half a unit more or less, times 2 pi
    and to the power `dim`, lies on either side of theta^(-2 i), in exact rational numbers."""
    from hy_nomas_b200 import rotary
    rot = rotary.Rotary(dim, theta, device="cpu", scaling=None if factor is None else {"type": "linear", "factor": factor})
    for i, f in enumerate(rot.freq.tolist()):
        f %= 2 ** 64
        want = Fraction(theta) ** (-2 * i)
        below, above = (Fraction(2 * f + d, 2 ** 65) * Fraction(factor or 1) for d in (-1, 1))
        assert (2 * PI * below) ** dim < want < (2 * (PI + Fraction(1, 10 ** 39)) * above) ** dim, i
    r64 = torch.tensor([f % 2 ** 64 for f in rot.freq.tolist()], dtype=torch.float64) / 2.0 ** 64 * 2 * math.pi
    # half a unit of 2 pi 2^-64, and the doubles' own roundings (up to three here, one there, 2^-53 each)
    assert torch.allclose(r64, rot.radians, rtol=2.0 ** -50, atol=math.pi * 2.0 ** -64)


def test_fixed_point_of_given_frequencies(hn):
    """Given radians are taken as the numbers they are, whole turns dropped."""
    from hy_nomas_b200 import rotary
    freq = [1.0, 0.1, -3.0, 1e9 + 0.125]
    got = rotary.Rotary(8, freq=freq, device="cpu").freq.tolist()
    for g, f in zip(got, freq):
        turns = Fraction(f) / (2 * PI) * 2 ** 64
        assert abs((turns - g + 2 ** 63) % 2 ** 64 - 2 ** 63) <= Fraction(1, 2) + abs(turns) / 10 ** 38
