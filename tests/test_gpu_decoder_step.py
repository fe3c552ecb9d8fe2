"""The decoder step over forked sequences (decoder.Decoder): a history, branches forked from it and decoded together, against
the same layers in 64 bits on the dequantized weights, each branch on its own.

Each of a layer's four linears quantizes its input to e4m3 (2.6% rms of what it gives); a branch's stream is the sum of the
sublayers' outputs, which are no larger than the stream here: eight linears give sqrt(8) * 2.6% = 7.4% at most; held to 10%.
Branches that share pages and branches that were written out one by one run the same kernels on the same tokens, but
attention cuts its sums elsewhere: a bf16 step (2^-8) of attention's output can move e4m3 codes: held to 4%.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
HEADS, KV, HIDDEN, INTER, D = 4, 2, 512, 768, 128


def build(hn, device, layers=2, seed=0):
    from hy_nomas_b200.decoder import Decoder, DecoderLayer
    g = torch.Generator(device=device).manual_seed(seed)

    def linear(n, k):
        w = torch.randn((n, k), generator=g, device=device) * (k ** -0.5)
        return hn.ops.quantize_fp8_block(w)

    def norm(n):
        return (1 + 0.1 * torch.randn(n, generator=g, device=device)).to(torch.bfloat16)
    made = []
    for _ in range(layers):
        qkv = hn.ops.stack_fp8_linears(linear(HEADS * D, HIDDEN), linear(KV * D, HIDDEN), linear(KV * D, HIDDEN))
        gate_up = hn.ops.stack_fp8_linears(linear(INTER, HIDDEN), linear(INTER, HIDDEN))
        made.append(DecoderLayer(norm(HIDDEN), norm(HIDDEN), (norm(64), norm(64)), (norm(64), norm(64)), qkv,
                                 linear(HIDDEN, HEADS * D), gate_up, linear(HIDDEN, INTER)))
    return Decoder(made, HEADS, KV, norm(HIDDEN))


def tables(pos, device):
    f = 1.0 / 10000 ** (torch.arange(64, device=device) / 64)
    a = torch.cat([pos.reshape(-1, 1).float() * f] * 2, -1)
    return a.cos(), a.sin()


def plain(hn, dec, x, pos):
    """All tokens of one sequence at once, 64 bits: x [n, hidden]."""
    deq = lambda w: hn.ops.dequantize_fp8_block(*w, dtype=torch.float64)  # noqa: E731
    rms = lambda t, w: t / torch.sqrt(t.square().mean(-1, keepdim=True) + dec.eps) * w.double()  # noqa: E731
    n = x.shape[0]
    cos, sin = (t.double() for t in tables(pos, x.device))

    def qk(t, heads, weights):
        # split RMSNorm (halves), then rotate-half on each of the sections [0, 64), [64, 96), [96, 128)
        t = t.view(n, heads, D)
        t = torch.cat([rms(t[..., :64], weights[0]), rms(t[..., 64:], weights[1])], -1)
        parts, at = [], 0
        for size in (64, 32, 32):
            u, c, s = t[..., at:at + size], cos[:, None, at:at + size], sin[:, None, at:at + size]
            rot = torch.cat([-u[..., size // 2:], u[..., :size // 2]], -1)
            parts.append(u * c + rot * s)
            at += size
        return torch.cat(parts, -1)
    h = x.double()
    mask = torch.full((n, n), -math.inf, device=x.device, dtype=torch.float64).triu(1)
    for w in dec.layers:
        q, k, v = (rms(h, w.input_norm) @ deq(w.qkv).T).split([HEADS * D, KV * D, KV * D], -1)
        q, k = qk(q, HEADS, w.q_norm), qk(k, KV, w.k_norm)
        k, v = (t.reshape(n, KV, D).repeat_interleave(HEADS // KV, 1) for t in (k, v))
        p = torch.softmax(torch.einsum("qhd,khd->hqk", q, k) / math.sqrt(D) + mask, -1)
        o = torch.einsum("hqk,khd->qhd", p, v).reshape(n, -1)
        h = h + o @ deq(w.out).T
        g, u = (rms(h, w.post_norm) @ deq(w.gate_up).T).chunk(2, -1)
        h = h + (torch.nn.functional.silu(g) * u) @ deq(w.down).T
    return h


@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_branches_of_one_history(hn, cuda, kind):
    from hy_nomas_b200 import paged
    dec = build(hn, cuda)
    past, branches, steps = 53, 5, 3
    history = torch.randn((1, past, HIDDEN), device=cuda).to(torch.bfloat16)
    tokens = torch.randn((steps, branches, 1, HIDDEN), device=cuda).to(torch.bfloat16)

    def run(fork):
        cache = paged.KVCache(len(dec.layers), 64, KV, 16, 8, 8, kind)
        pos = torch.arange(past, device=cuda)
        rows = list(range(1, branches + 1))
        if fork:
            first, _, _ = dec.step(history, *tables(pos, cuda), cache, [0])
            cache.fork([0] * branches, rows)
            cache.free([0])
        else:
            first, _, _ = dec.step(history.expand(branches, -1, -1).contiguous(), *tables(pos.repeat(branches), cuda), cache, rows)
        out = []
        for i in range(steps):
            p = torch.full((branches,), past + i, device=cuda)
            h, codes, scales = dec.step(tokens[i], *tables(p, cuda), cache, rows, shared=past // 16 * 16 if fork else 0)
            out.append(h[:, 0])
        used = int((cache.refs > 0).sum())
        cache.check()
        assert codes.shape == (branches, HIDDEN) and scales.shape == (branches, HIDDEN // 128)
        return first[0].float(), torch.stack(out, 1).float(), used
    first, got, used = run(True)
    first2, apart, used_apart = run(False)
    assert used == past // 16 + branches and used_apart == branches * 4
    assert float((got - apart).norm() / apart.norm()) < 0.04
    for b in range(branches):
        x = torch.cat([history[0], tokens[:, b, 0]])
        want = plain(hn, dec, x, torch.arange(past + steps, device=cuda))
        assert float((first.double() - want[:past]).norm() / want[:past].norm()) < 0.1
        assert float((got[b].double() - want[past:]).norm() / want[past:].norm()) < 0.1


@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_step_without_room_keeps_the_history(hn, cuda, kind):
    """Two branches of a whole-page history and a pool with one free page: the second branch's step is counted, and the shared
    pages hold what they held. With room it goes on where it was."""
    from hy_nomas_b200 import paged
    from test_gpu_paged import bits
    dec = build(hn, cuda)
    cache = paged.KVCache(len(dec.layers), 4, KV, 16, 4, 4, kind)
    history = torch.randn((1, 48, HIDDEN), device=cuda).to(torch.bfloat16)
    dec.step(history, *tables(torch.arange(48, device=cuda), cuda), cache, [0])
    cache.fork([0, 0], [1, 2])
    pools = [t for t in (cache.k, cache.v, cache.k_scale, cache.v_scale) if t is not None]
    before = [t[:, :3].clone() for t in pools]
    x = torch.randn((2, 1, HIDDEN), device=cuda).to(torch.bfloat16)
    at = tables(torch.full((2,), 48, device=cuda), cuda)
    dec.step(x, *at, cache, [1, 2], shared=48)
    with pytest.raises(RuntimeError, match="could not be met"):
        cache.check()
    assert cache.lengths.tolist() == [48, 49, 48, 0]
    assert all(torch.equal(bits(t[:, :3]), bits(was)) for t, was in zip(pools, before))
    cache.free([1])
    got, _, _ = dec.step(x[1:], *(t[1:] for t in at), cache, [2])
    cache.check()
    fresh = paged.KVCache(len(dec.layers), 4, KV, 16, 4, 4, kind)
    dec.step(history, *tables(torch.arange(48, device=cuda), cuda), fresh, [0])
    want, _, _ = dec.step(x[1:], *(t[1:] for t in at), fresh, [0])
    assert torch.equal(got, want)


def test_step_refuses_before_it_touches_the_cache(hn, cuda):
    """A cache or inputs of another shape than the layers': an error, and the rows are as they were."""
    from hy_nomas_b200 import paged
    dec = build(hn, cuda)
    x = torch.randn((2, 3, HIDDEN), device=cuda).to(torch.bfloat16)
    cos, sin = tables(torch.arange(3, device=cuda).repeat(2), cuda)
    for kw in (dict(layers=1), dict(heads=KV + 1)):
        a = dict(layers=2, heads=KV)
        a.update(kw)
        cache = paged.KVCache(a["layers"], 8, a["heads"], 16, 4, 4)
        with pytest.raises(ValueError):
            dec.step(x, cos, sin, cache, [0, 1])
        assert cache.lengths.tolist() == [0] * 4
    cache = paged.KVCache(2, 8, KV, 16, 4, 4)
    for args in ((x[:, :, :128], cos, sin), (x[0], cos, sin), (x.float(), cos, sin), (x, cos[:5], sin), (x, cos, sin[:, :64]),
                 (x[:1], cos[:3], sin[:3])):
        with pytest.raises((ValueError, TypeError)):
            dec.step(*args, cache, [0, 1])
    with pytest.raises(ValueError):
        dec.step(x, cos, sin, cache, [0, 1], shared=8)
    assert cache.lengths.tolist() == [0] * 4
    cache.check()
