"""Rotation by position and the append that rotates, against the definition in 64 bits.

Bound per output, before its rounding (half a step of its type): the angle's part of a turn is cut to 32 bits and rounded to fp32
(2^-24 of at most half a turn: 2^-22.3 rad), sincospi is off by 2 units at most (2^-23): together below 2^-21 of |x| + |partner|.
Products and sum: 3 x 2^-24. The norm: squares and sums of a head (eight in a lane, then a tree: below 16 x 2^-24, halved by the
square root), mean, eps, root, reciprocal, two products: below 2^-20 in all with the former.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
YARN = {"type": "yarn", "factor": 16.0, "original": 4096}


@pytest.fixture()
def rotary(hn):
    from hy_nomas_b200 import rotary
    return rotary


@pytest.fixture()
def paged(hn):
    from hy_nomas_b200 import paged
    return paged


def turned(x, pos, rot, w, eps=1e-6):
    """-> (y, |x| + |partner|) in 64 bits; pos [B, L]."""
    x = x.double()
    if w is not None:
        x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double()
    r = rot.dim
    angle = pos.double()[..., None] * rot.radians.to(x.device)
    c, s = (f(angle)[:, :, None] * rot.factor for f in (torch.cos, torch.sin))
    i = torch.arange(r // 2, device=x.device)
    a, b = (i, i + r // 2) if rot.layout == "half" else (2 * i, 2 * i + 1)
    y, mass = x.clone(), x.abs()
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    both = (x[..., a].abs() + x[..., b].abs()) * rot.factor
    mass[..., a], mass[..., b] = both, both
    return y, mass


def check(out, x, pos, rot, w, eps=1e-6):
    want, mass = turned(x, pos.expand(x.shape[:2]), rot, w, eps)
    bound = mass * 2.0 ** -20
    info = torch.finfo(out.dtype)
    bound = bound + (want.abs() + bound) * info.eps / 2 + info.smallest_normal * info.eps
    err = (out.double() - want).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


def randn(shape, seed, dtype=torch.bfloat16, scale=2.0):
    return (torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda") * scale).to(dtype)


def weight(d, seed):
    return (1 + 0.3 * torch.randn(d, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")).to(torch.bfloat16)


# ------------------------------------------------------------------------------------------------- rotate

@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("b,l,h,d,r", [(1, 1, 1, 8, 8), (1, 1, 32, 128, 128), (2, 3, 5, 16, 8), (3, 7, 9, 24, 24), (2, 5, 12, 96, 48),
                                       (1, 40, 3, 40, 32), (2, 33, 7, 64, 64), (1, 300, 16, 128, 64), (1, 9, 31, 80, 80),
                                       (2, 17, 4, 136, 120), (1, 5, 2, 256, 256), (1, 3000, 2, 128, 128), (2, 2, 33, 200, 16)])
def test_rotate(rotary, cuda, layout, norm, b, l, h, d, r):
    rot = rotary.Rotary(r, 10000.0, layout)
    w = weight(d, d) if norm else None
    pos = torch.randint(-50, 100000, (b, l), device="cuda", dtype=torch.int32, generator=torch.Generator("cuda").manual_seed(l))
    for dtype in DTYPES:
        x = randn((b, l, h, d), r + h, dtype)
        check(rotary.rotate(x, pos, rot, w), x, pos, rot, w)
        assert torch.equal(rotary.rotate(x, pos.long(), rot, w), rotary.rotate(x, pos, rot, w))


@pytest.mark.parametrize("scaling", [{"type": "linear", "factor": 4.0}, {"type": "ntk", "factor": 8.0}, YARN,
                                     {"type": "yarn", "factor": 4.0, "original": 32768, "beta_fast": 16, "attention_factor": 1.0}])
def test_scaled_contexts(rotary, cuda, scaling):
    rot = rotary.Rotary(96, 500000.0, "half", scaling)
    x, pos = randn((2, 50, 3, 128), 1, torch.float32), torch.arange(50, device="cuda") + 1000000
    check(rotary.rotate(x, pos, rot), x, pos, rot, None)


def test_far_positions(rotary, cuda):
    """Up to the largest positions of both integer types. 2^62 x f / 2 pi as the 64-bit frequency has it (its own rounding, 2^-65
    of a turn a position, is what it is): held against integers, not against a product of floats."""
    rot = rotary.Rotary(32, 10000.0, "interleaved")
    for p in (2 ** 31 - 1, -2 ** 31, 2 ** 40 + 12345, 2 ** 62 + 987654321, -2 ** 63):
        x = randn((1, 1, 2, 32), 3, torch.float32)
        pos = torch.tensor([p], device="cuda", dtype=torch.int64)
        out = rotary.rotate(x, pos, rot)
        turns = [(p * f) % 2 ** 64 / 2 ** 64 for f in rot.freq.tolist()]
        c = torch.tensor([math.cos(2 * math.pi * t) for t in turns], dtype=torch.float64, device="cuda")
        s = torch.tensor([math.sin(2 * math.pi * t) for t in turns], dtype=torch.float64, device="cuda")
        a, b = x.double()[..., 0::2], x.double()[..., 1::2]
        want = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
        bound = (a.abs() + b.abs()).repeat_interleave(2, -1) * 2.0 ** -20
        assert bool(((out.double() - want).abs() <= bound).all())
        if abs(p) < 2 ** 32:
            assert p == -2 ** 31 or torch.equal(out, rotary.rotate(x, pos.int(), rot))


def test_position_zero_and_unrotated_columns(rotary, cuda):
    x = randn((1, 3, 2, 64), 4)
    x[0, 1, 0, 40] = float("nan")
    x[0, 2, 1, 50] = -0.0
    rot = rotary.Rotary(32, layout="half")
    out = rotary.rotate(x, torch.tensor([0, 5, 9], device="cuda"), rot)
    assert torch.equal(out[0, 0], x[0, 0])
    a, b = (torch.where(z.isnan(), 7.0, z).contiguous().view(torch.int16) for z in (out[..., 32:], x[..., 32:]))
    assert torch.equal(a, b) and bool(out[0, 1, 0, 40].isnan())
    assert not bool(out[..., :32].isnan().any())


def test_rotate_views_and_out(rotary, cuda):
    packed = randn((3, 40, 24, 128), 5)
    rot = rotary.Rotary(128)
    pos = torch.arange(40, device="cuda", dtype=torch.int32)
    w = weight(128, 1)
    q = packed[:, :, 4:20]
    want = rotary.rotate(q.contiguous(), pos, rot, w)
    check(want, q, pos, rot, w)
    assert torch.equal(rotary.rotate(q, pos, rot, w), want)
    assert torch.equal(rotary.rotate(q.transpose(0, 1).contiguous().transpose(0, 1), pos[None].expand(3, 40), rot, w), want)
    strided = torch.stack([pos, pos + 1], -1)[:, 0]
    assert torch.equal(rotary.rotate(q, strided, rot, w), want)
    odd = randn((1, 3, 2, 136), 6)[..., 3:131]                       # rows that do not start on 16 bytes
    check(rotary.rotate(odd, pos[:3], rot, w), odd, pos[:3], rot, w)
    wide = torch.zeros((3, 40, 20, 128), dtype=torch.bfloat16, device="cuda")
    assert rotary.rotate(q, pos, rot, w, out=wide[:, :, 2:18]).data_ptr() == wide[:, :, 2:18].data_ptr()
    assert torch.equal(wide[:, :, 2:18], want) and not bool(wide[:, :, :2].any()) and not bool(wide[:, :, 18:].any())
    for layout in ("half", "interleaved"):
        r2 = rotary.Rotary(96, layout=layout)
        again, want2 = packed.clone(), rotary.rotate(q, pos, r2, w)
        rotary.rotate(again[:, :, 4:20], pos, r2, w, out=again[:, :, 4:20])
        assert torch.equal(again[:, :, 4:20], want2)
        assert torch.equal(again[:, :, :4], packed[:, :, :4]) and torch.equal(again[:, :, 20:], packed[:, :, 20:])


def test_rotate_norm_edges(rotary, cuda):
    """Heads of zeros stay zeros, large eps, a NaN stays in its head."""
    rot = rotary.Rotary(64)
    x = randn((1, 4, 3, 64), 7)
    x[0, 0] = 0
    x[0, 1, 1, 3] = float("nan")
    pos = torch.arange(4, device="cuda")
    out = rotary.rotate(x, pos, rot, weight(64, 2), eps=0.5)
    assert not bool(out[0, 0].any())
    assert bool(out[0, 1, 1].isnan().all()) and not bool(out[0, 1, 0].isnan().any()) and not bool(out[0, 1, 2].isnan().any())
    check(out[:, 2:], x[:, 2:], pos[2:], rot, weight(64, 2), 0.5)


def test_rotate_refusals(rotary, cuda):
    rot, x, pos = rotary.Rotary(64), randn((2, 3, 4, 64), 8), torch.arange(3, device="cuda")
    for bad, error in ((lambda: rotary.rotate(x.double(), pos, rot), TypeError), (lambda: rotary.rotate(x[0], pos, rot), ValueError),
                       (lambda: rotary.rotate(x[..., :60], pos, rot), ValueError), (lambda: rotary.rotate(x[..., :32], pos, rot), ValueError),
                       (lambda: rotary.rotate(x, pos.float(), rot), TypeError), (lambda: rotary.rotate(x, pos[:2], rot), ValueError),
                       (lambda: rotary.rotate(x, [0, 1, 2], rot), TypeError), (lambda: rotary.rotate(x, pos.cpu(), rot), RuntimeError),
                       (lambda: rotary.rotate(x, pos, "half"), TypeError), (lambda: rotary.rotate(x.cpu(), pos, rot), RuntimeError),
                       (lambda: rotary.rotate(x, pos, rotary.Rotary(64, device="cpu")), RuntimeError),
                       (lambda: rotary.rotate(x, pos, rot, weight(32, 1)), ValueError),
                       (lambda: rotary.rotate(x, pos, rot, weight(64, 1).cpu()), RuntimeError),
                       (lambda: rotary.rotate(x, pos, rot, weight(64, 1), eps=float("nan")), RuntimeError),
                       (lambda: rotary.rotate(x, pos, rot, weight(64, 1), eps=-1.0), RuntimeError),
                       (lambda: rotary.rotate(x, pos, rot, out=x[:, :2]), ValueError),
                       (lambda: rotary.rotate(x, pos, rot, out=x.float()), ValueError),
                       (lambda: rotary.rotate(x, pos, rot, out=x[:1].expand(2, 3, 4, 64)), ValueError)):
        with pytest.raises(error):
            bad()
    big = randn((3, 3, 4, 64), 8)
    with pytest.raises(ValueError, match="apart"):
        rotary.rotate(big[:2], pos, rot, out=big[1:])
    assert rotary.rotate(x[:0], pos, rot).shape == (0, 3, 4, 64)
    assert rotary.rotate(x[:, :0], pos[:0], rot).shape == (2, 0, 4, 64)


# ------------------------------------------------------------------------------------------------- append

def filled(paged, pages, heads, page, slots, width, kind, seed, layers=2):
    c = paged.KVCache(layers, pages, heads, page, slots, width, kind)
    g = torch.Generator(device="cuda").manual_seed(seed)
    for t in (c.k, c.v):
        t.copy_(torch.randn(t.shape, generator=g, device="cuda") * (1 if kind == "bf16" else 40))
    return c


def twin(paged, c):
    copy = lambda t: None if t is None else t.clone()  # noqa: E731
    t = paged.KVCache.over(copy(c.k), copy(c.v), copy(c.k_scale), copy(c.v_scale), c.meta.clone(), c.slots, c.width)
    t._refused.copy_(c._refused)
    return t


def check_int8(c, layer, rows, n, k64, mass, v):
    """Codes within half a step of the 64-bit value over its scale, and what the value itself may be off by."""
    lengths = c.lengths.tolist()
    for i, r in enumerate(rows):
        at = torch.arange(lengths[r] - n, lengths[r], device="cuda")
        page, place = c.table[r].long()[at // c.page], at % c.page
        for pool, scale, x, m in ((c.k, c.k_scale, k64[i], mass[i]), (c.v, c.v_scale, v[i].double(), 0 * v[i].double())):
            got = pool[layer][page, :, place].double() * scale[layer][page, :, place].double()[..., None]
            peak = x.abs().amax(-1, keepdim=True)
            assert torch.allclose(scale[layer][page, :, place].double()[..., None], peak / 127, rtol=2.0 ** -18, atol=1e-30)
            assert bool(((got - x).abs() <= peak / 127 * (0.5 + 2.0 ** -15) + m * 2.0 ** -19).all())


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("b,n,h,kv,page,r,layout,norm,scaling", [
    (1, 1, 1, 1, 16, 128, "half", True, None), (3, 1, 8, 2, 16, 64, "interleaved", True, None), (2, 5, 7, 1, 32, 8, "half", False, None),
    (5, 1, 32, 8, 64, 128, "half", True, YARN), (2, 70, 4, 4, 48, 96, "half", True, None), (1, 300, 3, 3, 16, 128, "interleaved", False, None),
    (2, 700, 16, 16, 32, 64, "half", True, YARN), (4, 3, 5, 5, 16, 120, "half", True, {"type": "ntk", "factor": 2.0})])
def test_append_rotated(paged, rotary, cuda, kind, b, n, h, kv, page, r, layout, norm, scaling):
    """q as `rotate` gives it; K and V as `append` writes rotate's K (bf16: the same bits; int8: one rounding less)."""
    width = 40 + n // page
    c = filled(paged, b * width + 3, kv, page, b + 1, width, kind, 1)
    for i in range(b):
        c.extend([i], 7 * i + 3)
    rows = list(range(b))[::-1]
    c.extend(rows, n)
    plain = twin(paged, c)
    packed = randn((b, n, h + 2 * kv, 128), n + h)
    q, k, v = packed[:, :, :h], packed[:, :, h:h + kv], packed[:, :, h + kv:]
    rot = rotary.Rotary(r, 10000.0, layout, scaling)
    wq, wk = (weight(128, 1), weight(128, 2)) if norm else (None, None)
    out = c.append_rotated(1, q, k, v, rows, rot, wq, wk)
    pos = (c.lengths[torch.tensor(rows, device="cuda")] - n)[:, None] + torch.arange(n, device="cuda", dtype=torch.int32)
    assert torch.equal(out, rotary.rotate(q, pos, rot, wq))
    plain.append(1, rotary.rotate(k, pos, rot, wk), v, rows)
    assert torch.equal(c.v, plain.v) and torch.equal(c.meta, plain.meta)
    assert torch.equal(c.k[0], plain.k[0])                              # the other layer
    if kind == "bf16":
        assert torch.equal(c.k.view(torch.int16), plain.k.view(torch.int16))
    else:
        assert torch.equal(c.v_scale, plain.v_scale)
        k64, mass = turned(k, pos, rot, wk)
        check_int8(c, 1, rows, n, k64, mass, v)
        assert int((c.k != plain.k).any(-1).sum()) <= b * n * kv         # nothing but the new tokens
    c.check()


def test_append_rotated_weights_apart_and_positions(paged, rotary, cuda):
    """A norm on one of the two only; positions given, of both types and shapes."""
    c = filled(paged, 20, 2, 16, 3, 6, "bf16", 2)
    c.extend([0, 1], 20)
    q, k, v = (randn((2, 20, n, 128), n) for n in (5, 2, 2))
    rot = rotary.Rotary(128, layout="interleaved")
    pos = torch.randint(-9, 70000, (2, 20), device="cuda")
    for wq, wk in ((weight(128, 3), None), (None, weight(128, 4))):
        for p in (pos, pos.int(), pos[0], torch.stack([pos, pos], -1)[..., 1].int()):
            plain = twin(paged, c)
            out = c.append_rotated(0, q, k, v, [0, 1], rot, wq, wk, positions=p)
            full = p.expand(2, 20)
            assert torch.equal(out, rotary.rotate(q, full, rot, wq))
            plain.append(0, rotary.rotate(k, full, rot, wk), v, [0, 1])
            assert torch.equal(c.k.view(torch.int16), plain.k.view(torch.int16)) and torch.equal(c.v, plain.v)
    c.check()


@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_append_rotated_leaves_out_what_append_does(paged, rotary, cuda, kind):
    """Refused rows, shared pages, rows listed twice or out of range: as `append`, counted alike."""
    c = filled(paged, 6, 2, 16, 5, 8, kind, 3)
    c.extend([0], 32)
    c.fork([0], [1])                       # shares both pages
    c.extend([2], 50)                      # the four that are left
    c.extend([1], 1)                       # refused
    q, k, v = (randn((6, 1, n, 128), n) for n in (4, 2, 2))
    rows = [2, 1, 0, 2, 77, -1]
    plain = twin(paged, c)
    before = int(c.failed)
    out = c.append_rotated(1, q, k, v, rows, rotary.Rotary(128), weight(128, 1), weight(128, 2))
    pos = torch.tensor([[49], [31], [31], [49], [-1], [-1]], device="cuda")
    kk = rotary.rotate(k, pos, rotary.Rotary(128), weight(128, 2))
    plain.append(1, kk, v, rows)
    assert int(c.failed) - before == int(plain.failed) == 5 * 2
    assert torch.equal(c.v, plain.v) and torch.equal(c.meta, plain.meta)
    if kind == "bf16":
        assert torch.equal(c.k, plain.k)
    else:
        assert int((c.k != plain.k).any(-1).sum()) <= 2 and torch.equal(c.v_scale, plain.v_scale)
    assert torch.equal(out[0], rotary.rotate(q[:1], pos[:1], rotary.Rotary(128), weight(128, 1))[0])
    with pytest.raises(RuntimeError, match="could not be met"):
        c.check()


def test_append_rotated_nan(paged, rotary, cuda):
    """A NaN or an infinity in a head's K or V: a NaN scale for that token and head, and for no other."""
    c = filled(paged, 4, 2, 16, 1, 4, "int8", 4)
    c.extend([0], 4)
    q, k, v = (randn((1, 4, 2, 128), n) for n in (1, 2, 3))
    k[0, 1, 0, 7], v[0, 2, 1, 100], k[0, 3, 1, 127] = float("nan"), float("inf"), -float("inf")
    c.append_rotated(0, q, k, v, [0], rotary.Rotary(64))
    page = int(c.table[0, 0])
    bad_k, bad_v = c.k_scale[0, page, :, :4].isnan().cpu(), c.v_scale[0, page, :, :4].isnan().cpu()
    assert bad_k.nonzero().tolist() == [[0, 1], [1, 3]] and bad_v.nonzero().tolist() == [[1, 2]]


def test_append_rotated_refusals(paged, rotary, cuda):
    c = filled(paged, 4, 2, 16, 2, 4, "bf16", 5)
    c.extend([0], 3)
    q, k, v = (randn((1, 3, n, 128), n) for n in (4, 2, 2))
    rot = rotary.Rotary(128)
    saved = c.k.clone(), c.v.clone()
    for bad, error in ((lambda: c.append_rotated(2, q, k, v, [0], rot), ValueError), (lambda: c.append_rotated(0, q[:, :2], k, v, [0], rot), ValueError),
                       (lambda: c.append_rotated(0, q, k[:, :, :1], v[:, :, :1], [0], rot), ValueError),
                       (lambda: c.append_rotated(0, q[:, :, :0], k, v, [0], rot), ValueError),
                       (lambda: c.append_rotated(0, q, k, v, [0, 1], rot), ValueError), (lambda: c.append_rotated(0, q.half(), k, v, [0], rot), TypeError),
                       (lambda: c.append_rotated(0, q, k, v.cpu(), [0], rot), RuntimeError), (lambda: c.append_rotated(0, q, k, v, [0], None), TypeError),
                       (lambda: c.append_rotated(0, q, k, v, [0], rotary.Rotary(136)), ValueError),
                       (lambda: c.append_rotated(0, q, k, v, [0], rot, weight(64, 1)), ValueError),
                       (lambda: c.append_rotated(0, q, k, v, [0], rot, positions=torch.zeros(4, device="cuda", dtype=torch.int64)), ValueError),
                       (lambda: c.append_rotated(0, q, k, v, [0], rot, eps=float("inf")), RuntimeError)):
        with pytest.raises(error):
            bad()
    assert torch.equal(c.k, saved[0]) and torch.equal(c.v, saved[1])
    assert c.append_rotated(0, q[:0], k[:0], v[:0], [], rot).shape == (0, 3, 4, 128)
    assert c.append_rotated(0, q[:, :0], k[:, :0], v[:, :0], [0], rot).shape == (1, 0, 4, 128)
    c.check()
