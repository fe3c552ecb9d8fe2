"""A decoder step over forked sequences: the layers of the PixelUMM decoder's shape (hy_nomas/pixelumm.py:246-337 - RMSNorm,
FP8 linears, split-norm MRoPE, grouped K/V heads, gated MLP) with their K/V in a `paged.KVCache`, so that many branches of
one history decode together and read its pages once. Inference only, as every weight here is 8-bit codes.

    dec = Decoder([DecoderLayer(...), ...], heads, kv_heads, final_norm)
    cache = paged.KVCache(len(dec.layers), pages, kv_heads, page, slots, width, kind="int8")
    h, codes, scales = dec.step(x, cos, sin, cache, [row])       # the history, a row of its own: x [1, n, hidden]
    cache.fork([row] * n_branches, branches)
    h, codes, scales = dec.step(x, cos, sin, cache, branches, shared=shared)     # a token or more per branch: x [B, n, hidden]

One step of a layer: the stacked q|k|v FP8 GEMM, `fused.pixelumm_qk` on q and k, `cache.append`, `paged.attention`, the output
projection, `fused.add_rmsnorm_quant`, gate|up, `fused.silu_mul_quant`, down, `fused.add_rmsnorm_quant` with the next layer's
norm: the residual stream is read and written once per sublayer and no normalized activations are stored.
"""
from dataclasses import dataclass

import torch

from . import fused, kernels, paged


@dataclass
class DecoderLayer:
    """FP8 linears as (codes [N, K], block scales [N/128, K/128]); bf16 norm weights. `qkv` = ops.stack_fp8_linears(q, k, v)
    and `gate_up` = ops.stack_fp8_linears(gate, up)."""
    input_norm: torch.Tensor
    post_norm: torch.Tensor
    q_norm: tuple           # (t, hw) weights [64] of pixelumm_qk
    k_norm: tuple
    qkv: tuple
    out: tuple
    gate_up: tuple
    down: tuple


class Decoder:
    def __init__(self, layers, heads, kv_heads, final_norm, eps=1e-6):
        if heads % kv_heads:
            raise ValueError(f"Decoder: {heads} heads on {kv_heads} K/V heads")
        self.layers, self.heads, self.kv_heads, self.final_norm, self.eps = list(layers), heads, kv_heads, final_norm, eps

    def step(self, x, cos, sin, cache, rows, shared=0):
        """x [B, n, hidden] bf16: the next n tokens of the cache's rows `rows` (room is made for them here), cos / sin
        [B * n, 128] fp32 their rotary tables. Causal within the step. `shared` as in paged.attention. Returns the final
        norm's input [B, n, hidden] and its FP8 codes and scales [B * n, ...] for the head that follows. A row that there is no
        room for keeps its tokens and is counted (`cache.check()`); what the step returns for it means nothing."""
        rows = cache._ids(rows, "Decoder.step")
        self._check(x, cos, sin, cache, rows, shared)           # before the rows grow
        b, n, hidden = x.shape
        tokens, h, hk = b * n, self.heads, self.kv_heads
        cache.extend(rows, n)
        stream = x.reshape(tokens, hidden)
        codes, scales = fused.rmsnorm_quant(stream, self.layers[0].input_norm, self.eps)
        for i, w in enumerate(self.layers):
            qkv = kernels.block_gemm(codes, scales, *w.qkv, kind="fp8").view(1, tokens, h + 2 * hk, paged.HEAD_DIM)
            q = fused.pixelumm_qk(qkv[:, :, :h], *w.q_norm, cos, sin, self.eps)
            k = fused.pixelumm_qk(qkv[:, :, h:h + hk], *w.k_norm, cos, sin, self.eps)
            cache.append(i, k.view(b, n, hk, -1), qkv[0, :, h + hk:].unflatten(0, (b, n)), rows)
            o = paged.attention(q.view(b, n, h, -1), cache, i, rows, shared=shared)
            codes, scales = kernels.quantize_activations(o.view(tokens, -1), "fp8")
            y = kernels.block_gemm(codes, scales, *w.out, kind="fp8")
            stream, codes, scales = fused.add_rmsnorm_quant(y, stream, w.post_norm, self.eps)
            gu = kernels.block_gemm(codes, scales, *w.gate_up, kind="fp8")
            inter = gu.shape[1] // 2
            codes, scales = fused.silu_mul_quant(gu[:, :inter], gu[:, inter:])
            y = kernels.block_gemm(codes, scales, *w.down, kind="fp8")
            norm = self.layers[i + 1].input_norm if i + 1 < len(self.layers) else self.final_norm
            stream, codes, scales = fused.add_rmsnorm_quant(y, stream, norm, self.eps)
        return stream.view(b, n, hidden), codes, scales

    def _check(self, x, cos, sin, cache, rows, shared):
        hidden = self.final_norm.shape[0]
        if x.dtype != torch.bfloat16:
            raise TypeError(f"Decoder.step: x must be bf16, got {x.dtype}")
        if x.dim() != 3 or x.shape[0] != rows.numel() or x.shape[2] != hidden:
            raise ValueError(f"Decoder.step: x {tuple(x.shape)} must be [{rows.numel()}, n, {hidden}]")
        tokens = x.shape[0] * x.shape[1]
        if any(t.shape[-1] != paged.HEAD_DIM or t.numel() != tokens * paged.HEAD_DIM for t in (cos, sin)):
            raise ValueError(f"Decoder.step: cos {tuple(cos.shape)} and sin {tuple(sin.shape)} must be "
                             f"{(tokens, paged.HEAD_DIM)}")
        if any(t.device != cache.device for t in (x, cos, sin)):
            raise ValueError(f"Decoder.step: x on {x.device}, cos on {cos.device}, sin on {sin.device}, the cache on {cache.device}")
        if cache.layers < len(self.layers) or cache.heads != self.kv_heads:
            raise ValueError(f"Decoder.step: a cache of {cache.layers} layers and {cache.heads} heads for {len(self.layers)} "
                             f"layers and {self.kv_heads} K/V heads")
        if not 0 <= shared <= cache.width * cache.page or shared % cache.page:
            raise ValueError(f"Decoder.step: shared must be whole pages of {cache.page} within the table, got {shared}")
