"""Host checks of the 4-bit linears and the rotations, through the C ABI and the Python layer: bad arguments are refused before a
GPU is touched (CPU only; no pointer is ever followed), scale tiles and frequencies against their definitions."""
import math

import pytest
import torch

from test_paged_host import FAKE, ref, struct


@pytest.fixture()
def paged(hn):
    from hy_nomas_b200 import paged
    return paged


@pytest.fixture()
def rotary(hn):
    from hy_nomas_b200 import rotary
    return rotary


def refused(hn, name, good, changes):
    """`good` as a dict in argument order; each change is refused with its code, and names the entry."""
    fn = getattr(hn.lib.lib, name)
    for change, code in changes:
        args = dict(good, **change)
        assert fn(*args.values()) == code, change
        assert name.encode() in hn.lib.lib.hn_last_error(), change


def test_quantize_fp4_checks(hn):
    good = dict(x=FAKE, ldx=100, dt=0, M=3, K=100, kind=3, q=FAKE, ldq=64, s=FAKE, r=FAKE, stream=None)
    refused(hn, "hn_quantize_fp4", good, [
        (dict(kind=0), 5), (dict(kind=4), 5), (dict(dt=3), 5), (dict(M=-1), 1), (dict(K=0), 1), (dict(K=1 << 31), 1), (dict(M=1 << 31), 1),
        (dict(x=None), 5), (dict(q=None), 5), (dict(s=None), 5), (dict(r=None), 5), (dict(ldx=99), 1), (dict(ldq=48), 1),
        (dict(ldq=72), 2), (dict(q=FAKE + 8), 2), (dict(s=FAKE + 4), 2), (dict(x=FAKE + 1), 2), (dict(r=FAKE + 2), 2)])
    assert hn.lib.lib.hn_quantize_fp4(*dict(good, M=0, x=None, q=None, s=None, r=None).values()) == 0


def test_dequantize_fp4_checks(hn):
    good = dict(q=FAKE, ldq=64, s=FAKE, r=FAKE, M=3, K=100, Kp=128, kind=3, out=FAKE, ldo=100, dt=0, stream=None)
    refused(hn, "hn_dequantize_fp4", good, [
        (dict(kind=1), 5), (dict(dt=3), 5), (dict(K=129), 1), (dict(Kp=120), 1), (dict(K=0), 1), (dict(r=None), 5), (dict(out=None), 5),
        (dict(ldo=99), 1), (dict(ldq=48), 1), (dict(ldq=72), 2), (dict(out=FAKE + 1), 2)])


def test_fp4_gemm_checks(hn):
    good = dict(qa=FAKE, lda=64, sa=FAKE, ra=FAKE, qw=FAKE, ldw=64, sw=FAKE, rw=FAKE, bias=FAKE, bdt=0, out=FAKE, ldo=10, dt=0, M=4,
                N=10, K=128, kind=3, stream=None)
    refused(hn, "hn_fp4_gemm", good, [
        (dict(kind=0), 5), (dict(kind=2), 5), (dict(dt=3), 5), (dict(bdt=3), 5), (dict(K=100), 1), (dict(K=0), 1), (dict(N=0), 1),
        (dict(M=-1), 1), (dict(M=1 << 31), 1), (dict(M=1 << 30, N=1 << 30), 1), (dict(qa=None), 5), (dict(sw=None), 5), (dict(out=None), 5),
        (dict(lda=48), 1), (dict(ldw=48), 1), (dict(ldo=9), 1), (dict(lda=72), 2), (dict(qw=FAKE + 8), 2), (dict(sa=FAKE + 8), 2),
        (dict(ra=FAKE + 1), 2), (dict(out=FAKE + 1), 2), (dict(bias=FAKE + 1), 2)])
    assert hn.lib.lib.hn_fp4_gemm(*dict(good, M=0, qa=None).values()) == 0


def rotation():
    return dict(pos=FAKE, pb=3, pl=1, wide=0, freq=FAKE, rot=64, layout=0, factor=1.0)


ROTATION_CHANGES = [(dict(rot=4), 1), (dict(rot=12), 1), (dict(rot=136), 1), (dict(layout=2), 5), (dict(wide=2), 5), (dict(freq=None), 5),
                    (dict(factor=float("nan")), 5), (dict(eps=float("inf")), 5), (dict(eps=-1e-6), 5), (dict(freq=FAKE + 4), 2),
                    (dict(pos=FAKE + 4, wide=1), 2), (dict(pos=FAKE + 2), 2)]


def test_rotate_checks(hn):
    st = dict(x=FAKE, xb=512, xl=512, xh=128, dt=0)
    good = dict(st, **rotation(), w=FAKE, eps=1e-6, B=2, L=3, H=4, D=128, out=FAKE, ob=512, ol=512, oh=128, stream=None)
    refused(hn, "hn_rotate", good, ROTATION_CHANGES + [
        (dict(dt=3), 5), (dict(D=264, rot=64), 1), (dict(D=60), 1), (dict(B=-1), 1), (dict(H=65537), 1), (dict(x=None), 5),
        (dict(pos=None), 5), (dict(out=None), 5), (dict(xh=100), 2), (dict(ol=4), 2), (dict(x=FAKE + 8), 2), (dict(w=FAKE + 8), 2)])
    assert hn.lib.lib.hn_rotate(*dict(good, B=0, x=None).values()) == 0


def test_append_rotated_checks(hn, paged):
    c = struct(paged, refused=FAKE, epoch=1)
    st = [("q", 512), ("k", 512), ("v", 512)]
    good = dict(cache=ref(c), layer=0)
    for name, s in st:
        good.update({name: FAKE, name + "b": s, name + "t": 128, name + "h": 128})
        if name == "q":
            good["H"] = 8
    good.update(rows=FAKE, B=2, n=3, **rotation(), wq=FAKE, wk=None, eps=1e-6, out=FAKE, stream=None)
    refused(hn, "hn_cache_append_rotated", good, ROTATION_CHANGES + [
        (dict(cache=None), 5), (dict(layer=2), 1), (dict(H=0), 1), (dict(B=-1), 1), (dict(q=None), 5), (dict(rows=None), 5),
        (dict(out=None), 5), (dict(kt=100), 2), (dict(qh=4), 2), (dict(v=FAKE + 2), 2), (dict(wk=FAKE + 2), 2),
        (dict(cache=ref(struct(paged, refused=FAKE, epoch=0))), 5), (dict(cache=ref(struct(paged, refused=None, epoch=1))), 5)])
    assert hn.lib.lib.hn_cache_append_rotated(*dict(good, B=0, q=None, rows=None).values()) == 0


def test_python_layer_wants_cuda(hn, rotary):
    x = torch.zeros(3, 64)
    q, s = torch.zeros(3, 32, dtype=torch.uint8), torch.zeros(1, 1, 512, dtype=torch.uint8)
    for call in (lambda: hn.kernels.quantize_fp4(x), lambda: hn.kernels.dequantize_fp4(q, s), lambda: hn.kernels.fp4_gemm(q, s, None, q, s, None),
                 lambda: rotary.rotate(x.view(1, 1, 3, 64), torch.zeros(1, dtype=torch.int32), rotary.Rotary(64, device="cpu"))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(ValueError, match="kind"):
        hn.kernels.quantize_fp4(x, "int8")


@pytest.mark.parametrize("rows,groups", [(1, 1), (128, 4), (129, 5), (300, 10), (33, 7)])
def test_scale_tiles(hn, rows, groups):
    s = torch.randint(0, 256, (rows, groups), dtype=torch.uint8, generator=torch.Generator().manual_seed(rows))
    t = hn.ops.tile_fp4_scales(s)
    assert t.shape == (-(-rows // 128), -(-groups // 4), 512)
    seen = torch.zeros_like(t)
    for r in range(rows):
        for g in range(groups):
            at = 16 * (r % 32) + 4 * (r // 32 % 4) + g % 4
            assert t[r // 128, g // 4, at] == s[r, g]
            seen[r // 128, g // 4, at] = 1
    assert not bool(t[seen == 0].any())
    assert torch.equal(hn.ops.untile_fp4_scales(t, rows, groups), s)
    e = (s & 0x77).view(torch.float8_e4m3fn)
    assert torch.equal(hn.ops.untile_fp4_scales(hn.ops.tile_fp4_scales(e), rows, groups).view(torch.float8_e4m3fn).view(torch.uint8),
                       e.view(torch.uint8))
    for bad in (lambda: hn.ops.tile_fp4_scales(s.float()), lambda: hn.ops.tile_fp4_scales(s[0]),
                lambda: hn.ops.untile_fp4_scales(t, 128 * t.shape[0] + 1, 1), lambda: hn.ops.untile_fp4_scales(t[0], 1, 1)):
        with pytest.raises(ValueError):
            bad()


def test_stacked_linears(hn):
    def linear(n, r=True):
        return (torch.full((n, 32), n % 251, dtype=torch.uint8), torch.full((-(-n // 128), 1, 512), n % 250, dtype=torch.uint8),
                torch.full((n,), float(n)) if r else None)
    q, s, r = hn.ops.stack_fp4_linears(linear(128), linear(256), linear(40))
    assert q.shape == (424, 32) and s.shape == (4, 1, 512) and r.tolist() == [128.0] * 128 + [256.0] * 256 + [40.0] * 40
    assert hn.ops.stack_fp4_linears(linear(128, False), linear(5, False))[2] is None
    with pytest.raises(ValueError, match="128"):
        hn.ops.stack_fp4_linears(linear(40), linear(128))
    with pytest.raises(ValueError, match="row scales"):
        hn.ops.stack_fp4_linears(linear(128), linear(128, False))


def test_frequencies(rotary):
    f, m = rotary.frequencies(128, 10000.0)
    assert m == 1.0 and f[0] == 1.0 and abs(float(f[63]) - 10000.0 ** (-126 / 128)) < 1e-18
    f2, _ = rotary.frequencies(128, 10000.0, {"type": "linear", "factor": 4.0})
    assert torch.equal(f2, f / 4)
    f3, _ = rotary.frequencies(128, 10000.0, {"type": "ntk", "factor": 8.0})
    assert f3[0] == 1.0 and abs(float(f3[63] * 8 / f[63]) - 1) < 1e-12
    f4, m4 = rotary.frequencies(128, 10000.0, {"type": "yarn", "factor": 16.0, "original": 4096})
    turns = f * 4096 / (2 * math.pi)
    assert torch.equal(f4[turns > 40], f[turns > 40]) and torch.allclose(f4[turns < 0.9], f[turns < 0.9] / 16, rtol=1e-12)
    assert bool((f4 <= f).all()) and bool((f4 >= f / 16 * (1 - 1e-12)).all()) and abs(m4 - (0.1 * math.log(16) + 1)) < 1e-15
    for bad in (dict(dim=4), dict(dim=260), dict(dim=12), dict(dim=64, theta=1.0), dict(dim=64, theta=float("nan")),
                dict(dim=64, scaling={"type": "other", "factor": 2.0}), dict(dim=64, scaling={"factor": 2.0}),
                dict(dim=64, scaling={"type": "linear"}), dict(dim=64, scaling={"type": "linear", "factor": 0.0}),
                dict(dim=64, scaling={"type": "linear", "factor": 2.0, "original": 5}), dict(dim=64, scaling={"type": "yarn", "factor": 2.0})):
        with pytest.raises(ValueError):
            rotary.frequencies(**bad)


def test_rotary_turns(rotary):
    """The fixed-point frequencies are the radians as parts of a turn; given frequencies, negative and beyond a turn ones too."""
    r = rotary.Rotary(64, device="cpu")
    got = torch.tensor([f / 2 ** 64 for f in r.freq.tolist()], dtype=torch.float64)
    assert torch.allclose(got * 2 * math.pi, r.radians, rtol=1e-15)
    freq = [0.1, -0.2, 5.0, 7.0]
    r = rotary.Rotary(8, freq=freq, factor=0.5, device="cpu")
    for a, b in zip(r.freq.tolist(), freq):
        assert abs(math.cos(a / 2 ** 64 * 2 * math.pi) - math.cos(b)) < 1e-15 and abs(math.sin(a / 2 ** 64 * 2 * math.pi) - math.sin(b)) < 1e-15
    assert r.factor == 0.5
    for bad in (dict(dim=8, freq=[1.0]), dict(dim=8, freq=[1.0, 2.0, 3.0, float("inf")]), dict(dim=64, layout="pairs"),
                dict(dim=8, freq=freq, scaling={"type": "linear", "factor": 2.0}), dict(dim=8, freq=freq, factor=float("nan"))):
        with pytest.raises(ValueError):
            rotary.Rotary(device="cpu", **bad)
