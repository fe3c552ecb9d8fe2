// rotary.cuh - positions to rotations: what the rotation kernel and the rotating append share.
//
// The angle of pair i at position t is t f_i, and only its part of a turn matters. f_i is held as a fraction of a turn in 64
// bits, so t f_i modulo one turn is the wrapped 64-bit product: exact for any position, where an fp32 product would be off by
// t 2^-25 turns. Its upper 32 bits, signed, go to sincospi in fp32 (2^-25 of half a turn).
#pragma once
#include "hn_common.cuh"

namespace hn {
namespace rotary {

constexpr int MAX_PAIRS = 128;      // rotated columns: at most 256
constexpr int INTERLEAVED = 1;      // pair i is columns 2 i, 2 i + 1; else columns i, i + rot / 2

struct Rotation {
    const int64_t *freq;            // [rot / 2] fractions of a turn a position, times 2^64
    int rot, layout;                // rotated columns, the first of the head; a multiple of 8
    float factor;                   // on cos and sin
};

// cos and sin of all pairs at position t into the warp's `table` ([2][MAX_PAIRS])
__device__ __forceinline__ void turn_table(const Rotation &r, int64_t t, float *table, int lane) {
    __syncwarp();                   // the table's readers of the token before
    for (int i = lane; i < r.rot >> 1; i += 32) {
        const uint64_t turns = (uint64_t)t * (uint64_t)r.freq[i];
        float s, c;
        sincospif((float)(int32_t)(turns >> 32) * 0x1p-31f, &s, &c);
        table[i] = c * r.factor;
        table[MAX_PAIRS + i] = s * r.factor;
    }
    __syncwarp();
}

// A lane's eight columns of a head, 8 sub to 8 sub + 7, in two runs of four. `off[j]`: where run j's partners stand (columns
// from the run's own), 0: the run is not rotated. Half layout only; pairs of the interleaved layout are a lane's own.
struct Turn {
    float c[8], s[8];               // half: per column, s with its sign; interleaved: c[0..3], s[0..3] per pair
    int off[2];
    bool own;                       // interleaved and rotated
};
__device__ __forceinline__ void partners(const Rotation &r, int sub, Turn &t) {
    const int half = r.rot >> 1;
    t.own = r.layout == INTERLEAVED && 8 * sub < r.rot;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int col = 8 * sub + 4 * j;
        t.off[j] = r.layout == INTERLEAVED || col >= r.rot ? 0 : col < half ? half : -half;
    }
}
__device__ __forceinline__ void turn_of(const Rotation &r, int sub, const float *table, Turn &t) {
    if (t.own) {
#pragma unroll
        for (int i = 0; i < 4; ++i) { t.c[i] = table[4 * sub + i]; t.s[i] = table[MAX_PAIRS + 4 * sub + i]; }
        return;
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        if (t.off[j] == 0) continue;
        const int pair = 8 * sub + 4 * j + (t.off[j] < 0 ? t.off[j] : 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            t.c[4 * j + i] = table[pair + i];
            t.s[4 * j + i] = t.off[j] > 0 ? -table[MAX_PAIRS + pair + i] : table[MAX_PAIRS + pair + i];
        }
    }
}
// v: the lane's columns, o: their partners (half layout)
__device__ __forceinline__ void turn(const Turn &t, float (&v)[8], const float (&o)[8]) {
    if (t.own) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a = v[2 * i], b = v[2 * i + 1];
            v[2 * i] = a * t.c[i] - b * t.s[i];
            v[2 * i + 1] = b * t.c[i] + a * t.s[i];
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        if (t.off[j] == 0) continue;
#pragma unroll
        for (int i = 4 * j; i < 4 * j + 4; ++i) v[i] = v[i] * t.c[i] + o[i] * t.s[i];
    }
}

// eight or four columns to fp32, and back with one rounding
__device__ __forceinline__ void load8(const __nv_bfloat16 *p, float (&v)[8]) { Elem<__nv_bfloat16>::load8(p, v); }
__device__ __forceinline__ void load8(const __half *p, float (&v)[8]) { Elem<__half>::load8(p, v); }
__device__ __forceinline__ void load8(const float *p, float (&v)[8]) { Elem<float>::load8(p, v); }
__device__ __forceinline__ void load4(const __nv_bfloat16 *p, float *v) {
    const uint2 w = *reinterpret_cast<const uint2 *>(p);
    v[0] = bf16_lo(w.x); v[1] = bf16_hi(w.x); v[2] = bf16_lo(w.y); v[3] = bf16_hi(w.y);
}
__device__ __forceinline__ void load4(const __half *p, float *v) {
    uint2 w = *reinterpret_cast<const uint2 *>(p);
    const float2 a = __half22float2(*reinterpret_cast<__half2 *>(&w.x)), b = __half22float2(*reinterpret_cast<__half2 *>(&w.y));
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
}
__device__ __forceinline__ void load4(const float *p, float *v) {
    const float4 w = *reinterpret_cast<const float4 *>(p);
    v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
}
__device__ __forceinline__ void store8(__nv_bfloat16 *p, const float (&v)[8]) {
    *reinterpret_cast<uint4 *>(p) = make_uint4(bf16x2_rn(v[0], v[1]), bf16x2_rn(v[2], v[3]), bf16x2_rn(v[4], v[5]), bf16x2_rn(v[6], v[7]));
}
__device__ __forceinline__ void store8(__half *p, const float (&v)[8]) {
    *reinterpret_cast<uint4 *>(p) = make_uint4(pack_f16_rn(v[0], v[1]), pack_f16_rn(v[2], v[3]), pack_f16_rn(v[4], v[5]), pack_f16_rn(v[6], v[7]));
}
__device__ __forceinline__ void store8(float *p, const float (&v)[8]) {
    *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4 *>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
// the partners of a lane's columns, `x` its first
template <typename E> __device__ __forceinline__ void load_partners(const E *x, const Turn &t, float (&o)[8]) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
        if (t.off[j] != 0) load4(x + 4 * j + t.off[j], o + 4 * j);
}

// Norm weights of a lane's columns and of their partners
struct Weights {
    float own[8], other[8];
};
__device__ __forceinline__ void load_weights(const __nv_bfloat16 *w, const Turn &t, Weights &out) {
    load8(w, out.own);
    load_partners(w, t, out.other);
}
// x / sqrt(mean x^2 + eps) * w over the P lanes of a head of D columns (v is 0 in lanes behind it)
template <int P>
__device__ __forceinline__ void head_norm(float (&v)[8], float (&o)[8], const Weights &w, const Turn &t, int D, float eps) {
    float ss = v[0] * v[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) ss = fmaf(v[i], v[i], ss);
#pragma unroll
    for (int i = 1; i < P; i <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, i);
    const float inv = rsqrt_cr(__fadd_rn(__fdiv_rn(ss, (float)D), eps));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = v[i] * inv * w.own[i];
#pragma unroll
    for (int j = 0; j < 2; ++j)
        if (t.off[j] != 0)
#pragma unroll
            for (int i = 4 * j; i < 4 * j + 4; ++i) o[i] = o[i] * inv * w.other[i];
}

} // namespace rotary
} // namespace hn
