"""Host checks of the rotations beside those of test_more_host.py, through the C ABI (CPU only; no pointer is ever followed)."""
import pytest

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
