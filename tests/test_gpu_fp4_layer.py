"""The 4-bit linears, the rotating append and the paged attention as a decoder layer runs them together; captured into a graph and
replayed on new inputs; on streams other than the default one, two at a time."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
D = 128


@pytest.fixture()
def mods(hn):
    from hy_nomas_b200 import paged, rotary
    return hn, paged, rotary


def randn(shape, seed, scale=1.0, dtype=torch.bfloat16):
    return (torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda") * scale).to(dtype)


class Layer:
    """q|k|v, norm + rotation + append, attention, output linear."""

    def __init__(self, mods, kind, cache_kind, hidden=512, heads=8, kv=2, rows=3):
        hn, paged, rotary = mods
        self.k, self.paged, self.kind, self.heads, self.kv = hn.kernels, paged, kind, heads, kv
        self.qkv = self.k.quantize_fp4(randn(((heads + 2 * kv) * D, hidden), 1, 0.05), kind)
        self.out = self.k.quantize_fp4(randn((hidden, heads * D), 2, 0.05), kind)
        self.qn, self.kn = (1 + 0.2 * randn((D,), s, dtype=torch.float32) for s in (3, 4))
        self.qn, self.kn = self.qn.to(torch.bfloat16), self.kn.to(torch.bfloat16)
        self.rot = rotary.Rotary(96, 10000.0, "half", {"type": "yarn", "factor": 4.0, "original": 64})
        self.cache = paged.KVCache(1, 60, kv, 16, rows, 20, cache_kind)
        self.rows = torch.arange(rows, dtype=torch.int32, device="cuda")

    def step(self, x):
        b, n, hidden = x.shape
        self.cache.extend(self.rows, n)
        qkv = self.k.fp4_linear(x, *self.qkv, kind=self.kind).view(b, n, -1, D)
        h, kv = self.heads, self.kv
        q = self.cache.append_rotated(0, qkv[:, :, :h], qkv[:, :, h:h + kv], qkv[:, :, h + kv:], self.rows, self.rot, self.qn, self.kn)
        o = self.paged.attention(q, self.cache, 0, self.rows)
        return self.k.fp4_linear(o.view(b, n, -1), *self.out, kind=self.kind)


def exact_layer(mods, layer, xs):
    """All tokens at once in 64 bits, but for the two quantizers of activations: theirs is the format's rounding, taken as it is."""
    hn = mods[0]
    value = lambda t: hn.kernels.dequantize_fp4(*t, layer.kind, torch.float32).double()  # noqa: E731
    quant = lambda t: value(hn.kernels.quantize_fp4(t, layer.kind))  # noqa: E731
    x = torch.cat(xs, 1)
    b, n, hidden = x.shape
    h, kv, rot = layer.heads, layer.kv, layer.rot
    qkv = (quant(x.view(-1, hidden)) @ value(layer.qkv).t()).view(b, n, -1, D)

    def turn(t, w):
        t = t / (t.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
        angle = torch.arange(n, device="cuda").double()[:, None] * rot.radians.cuda()
        c, s = torch.cos(angle)[:, None] * rot.factor, torch.sin(angle)[:, None] * rot.factor
        i = torch.arange(rot.dim // 2, device="cuda")
        y, j = t.clone(), i + rot.dim // 2
        y[..., i], y[..., j] = t[..., i] * c - t[..., j] * s, t[..., j] * c + t[..., i] * s
        return y
    q, k, v = turn(qkv[:, :, :h], layer.qn), turn(qkv[:, :, h:h + kv], layer.kn), qkv[:, :, h + kv:]
    k, v = (t.repeat_interleave(h // kv, 2) for t in (k, v))
    logits = torch.einsum("bqhd,bkhd->bhqk", q, k) / math.sqrt(D)
    logits.masked_fill_(torch.ones(n, n, device="cuda").triu(1).bool(), -math.inf)
    o = torch.einsum("bhqk,bkhd->bqhd", logits.softmax(-1), v)
    return o, value(layer.out)


@pytest.mark.parametrize("kind", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("cache_kind", ["bf16", "int8"])
def test_layer_prompt_then_tokens(mods, cuda, kind, cache_kind):
    """A prompt of 37 tokens, a chunk of 5, then single tokens: attention's output against 64 bits. Each of q, k, v, o is rounded to
    bf16 (2^-8 once each, and once more where a norm or rotation writes it), K and V of the int8 cache to 1 / 254 of their
    peak; logits of up to ~30 turn 2^-8 of q and k into weights a few per cent off: the relative L2 stays below 2^-5."""
    layer = Layer(mods, kind, cache_kind)
    xs = [randn((3, n, 512), 10 + i) for i, n in enumerate((37, 5, 1, 1, 1))]
    seen = []
    real = layer.paged.attention

    class Spy:
        def attention(self, *a, **kw):
            seen.append(real(*a, **kw))
            return seen[-1]
    layer.paged = Spy()
    ys = [layer.step(x) for x in xs]
    layer.cache.check()
    o, w = exact_layer(mods, layer, xs)
    got = torch.cat(seen, 1).double()
    assert float((got - o).norm() / o.norm()) < 2.0 ** -5
    # the output linear, of what it was given
    q = mods[0].kernels.quantize_fp4(torch.cat(seen, 1).reshape(-1, 8 * D), kind)
    want = mods[0].kernels.dequantize_fp4(*q, kind, torch.float32).double() @ w.t()
    y = torch.cat(ys, 1).reshape(-1, 512).double()
    assert float((y - want).norm() / want.norm()) < 2.0 ** -8


@pytest.mark.parametrize("kind", ["nvfp4", "mxfp4"])
def test_layer_captured_and_replayed(mods, cuda, kind):
    """One decoding step captured: every replay takes the next token, as the eager steps do, bit for bit."""
    layers = [Layer(mods, kind, "bf16") for _ in range(2)]
    prompt, tokens = randn((3, 20, 512), 5), [randn((3, 1, 512), 20 + i) for i in range(4)]
    for layer in layers:
        layer.step(prompt)
        layer.step(tokens[0])
    x = torch.empty_like(tokens[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layers[0].step(x)
    for t in tokens[1:]:
        x.copy_(t)
        graph.replay()
        assert torch.equal(y, layers[1].step(t))
    assert torch.equal(layers[0].cache.k, layers[1].cache.k) and torch.equal(layers[0].cache.meta, layers[1].cache.meta)


def test_operators_captured(mods, cuda):
    """Each operator alone, at sizes of all its kernels, replayed on inputs that change."""
    hn, paged, rotary = mods
    rot = rotary.Rotary(64)
    w = {(n, k): hn.kernels.quantize_fp4(randn((n, k), n), "nvfp4") for n, k in ((300, 1024), (2600, 320))}
    for m, n, k in ((1, 300, 1024), (48, 300, 1024), (2000, 2600, 320)):
        x = randn((m, k), 1)

        def call():
            q = hn.kernels.quantize_fp4(x)
            return (hn.kernels.fp4_gemm(*q, *w[n, k]), hn.kernels.dequantize_fp4(*q),
                    rotary.rotate(x.view(1, m, -1, 64), torch.arange(m, device="cuda"), rot))
        call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        for seed in (2, 3):
            x.copy_(randn((m, k), seed))
            graph.replay()
            assert all(torch.equal(a, b) for a, b in zip(out, call()))


def test_streams(mods, cuda):
    """Calls on two streams at once, the products of all three kernels among them, give what they give alone."""
    hn, paged, rotary = mods
    rot = rotary.Rotary(128, layout="interleaved")
    work = []
    for i, (m, n, k) in enumerate(((1, 512, 4096), (100, 512, 4096), (3000, 2048, 512), (2, 2048, 512), (700, 900, 2080), (2304, 2304, 64))):
        x, w = randn((m, k), i), hn.kernels.quantize_fp4(randn((n, k), 50 + i), "mxfp4")
        work.append((x, w))

    def call(x, w):
        y = hn.kernels.fp4_linear(x, *w, kind="mxfp4")
        z = rotary.rotate(y[:, :y.shape[1] // 128 * 128].reshape(1, x.shape[0], -1, 128), torch.arange(x.shape[0], device="cuda"), rot)
        return y, z
    want = [call(*t) for t in work]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for rounds in range(5):
        for i, t in enumerate(work):
            with torch.cuda.stream(streams[(i + rounds) % 2]):
                got.append((i, call(*t)))
    torch.cuda.synchronize()
    for i, (y, z) in got:
        assert torch.equal(y, want[i][0]) and torch.equal(z, want[i][1])
    for s in streams:
        assert hn.lib.device_error(s) == (0, 0)
