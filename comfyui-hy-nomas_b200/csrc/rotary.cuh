// rotary.cuh - positions to rotations: what the rotation kernel and the rotating append share.
//
// The angle of pair i at position t is t f_i, and only its part of a turn matters. f_i is held as a fraction of a turn in 64
// bits, so t f_i modulo one turn is the wrapped 64-bit product, which rounds nothing: what f_i was rounded by counts t times, t 2^-65
// of a turn (an fp32 product would be off by t 2^-25). Its upper 32 bits, signed, go to sincospi in fp32 (2^-25 of half a
// turn, so that far positions are turned as well as the first ones up to 2^39).
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
template <bool INTER> __device__ __forceinline__ void turn(const Turn &t, float (&v)[8], const float (&o)[8]) {
    if constexpr (INTER) {
        if (!t.own) return;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a = v[2 * i], b = v[2 * i + 1];
            v[2 * i] = a * t.c[i] - b * t.s[i];
            v[2 * i + 1] = b * t.c[i] + a * t.s[i];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            if (t.off[j] == 0) continue;
#pragma unroll
            for (int i = 4 * j; i < 4 * j + 4; ++i) v[i] = v[i] * t.c[i] + o[i] * t.s[i];
        }
    }
}

// eight or four columns to fp32 (of heads bf16, of norm weights fp32, too), and back with one rounding
__device__ __forceinline__ void load8(const __nv_bfloat16 *p, float (&v)[8]) { Elem<__nv_bfloat16>::load8(p, v); }
__device__ __forceinline__ void load8(const float *p, float (&v)[8]) { Elem<float>::load8(p, v); }
__device__ __forceinline__ void load4(const __nv_bfloat16 *p, float *v) {
    const uint2 w = *reinterpret_cast<const uint2 *>(p);
    v[0] = bf16_lo(w.x); v[1] = bf16_hi(w.x); v[2] = bf16_lo(w.y); v[3] = bf16_hi(w.y);
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
// of columns from `first` on; w: bf16, or fp32 (`wide`), as the caller has them
template <typename E> __device__ __forceinline__ void load_weights(const E *w, const Turn &t, Weights &out) {
    load8(w, out.own);
    load_partners(w, t, out.other);
}
__device__ __forceinline__ void load_weights(const void *w, int wide, int first, const Turn &t, Weights &out) {
    if (wide) load_weights(static_cast<const float *>(w) + first, t, out);
    else load_weights(static_cast<const __nv_bfloat16 *>(w) + first, t, out);
}
// x / sqrt(mean x^2 + eps) * w over the P lanes of a head (v is 0 in lanes behind it); rd = 1 / D
template <int P>
__device__ __forceinline__ void head_norm(float (&v)[8], float (&o)[8], const Weights &w, const Turn &t, float rd, float eps) {
    float ss = v[0] * v[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) ss = fmaf(v[i], v[i], ss);
#pragma unroll
    for (int i = 1; i < P; i <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, i);
    const float inv = rsqrtf(fmaf(ss, rd, eps));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = v[i] * inv * w.own[i];
#pragma unroll
    for (int j = 0; j < 2; ++j)
        if (t.off[j] != 0)
#pragma unroll
            for (int i = 4 * j; i < 4 * j + 4; ++i) o[i] = o[i] * inv * w.other[i];
}

// ---------------------------------------------------------------------------------------------------
// Sixteen columns a lane: two runs of eight that hold eight whole pairs, so that no partner stands elsewhere. Heads whose width and
// rotated part are multiples of 16. In the half layout a rotated lane's runs are half the rotated part apart, in the interleaved
// one they follow each other, as they do in lanes that are not rotated.
struct Lane16 {
    int a, b;                       // first columns of the two runs
    bool on;                        // rotated
    int pair;                       // its first pair
};
template <bool INTER> __device__ __forceinline__ Lane16 lane16(const Rotation &r, int sub) {
    Lane16 l;
    l.on = 16 * sub < r.rot;
    l.a = INTER || !l.on ? 16 * sub : 8 * sub;
    l.b = INTER || !l.on ? l.a + 8 : l.a + (r.rot >> 1);
    l.pair = 8 * sub;
    return l;
}
// A lane's columns as eight f32x2: x[i] the first columns of pairs 2 i and 2 i + 1, y[i] their partners. Products and fused
// multiply-adds on them take one instruction for two columns.
struct Cols {
    uint64_t x[4], y[4];
};
struct Turn16 {
    uint64_t c[4], s[4], ns[4];
};
__device__ __forceinline__ void turn16_of(const Lane16 &l, const float *table, Turn16 &t) {
    if (!l.on) return;
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        const ulonglong2 c = *reinterpret_cast<const ulonglong2 *>(table + l.pair + 2 * i);
        const ulonglong2 s = *reinterpret_cast<const ulonglong2 *>(table + MAX_PAIRS + l.pair + 2 * i);
        t.c[i] = c.x; t.c[i + 1] = c.y;
        t.s[i] = s.x; t.s[i + 1] = s.y;
        t.ns[i] = s.x ^ 0x8000000080000000ull; t.ns[i + 1] = s.y ^ 0x8000000080000000ull;
    }
}
__device__ __forceinline__ void turn16(const Lane16 &l, const Turn16 &t, Cols &v) {
    if (!l.on) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint64_t u = x2_fma(v.y[i], t.ns[i], x2_mul(v.x[i], t.c[i]));
        v.y[i] = x2_fma(v.x[i], t.s[i], x2_mul(v.y[i], t.c[i]));
        v.x[i] = u;
    }
}
// x / sqrt(mean x^2 + eps) * w over the P lanes of a head; v is 0 in lanes behind it. rd = 1 / D
template <int P> __device__ __forceinline__ void norm16(Cols &v, const Cols &w, float rd, float eps) {
    uint64_t a = x2_mul(v.x[0], v.x[0]), b = x2_mul(v.y[0], v.y[0]);
#pragma unroll
    for (int i = 1; i < 4; ++i) {
        a = x2_fma(v.x[i], v.x[i], a);
        b = x2_fma(v.y[i], v.y[i], b);
    }
    float a0, a1, b0, b1;
    x2_split(a, a0, a1);
    x2_split(b, b0, b1);
    float ss = (a0 + a1) + (b0 + b1);
#pragma unroll
    for (int i = 1; i < P; i <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, i);
    const uint64_t inv = x2_splat(rsqrtf(fmaf(ss, rd, eps)));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v.x[i] = x2_mul(x2_mul(v.x[i], inv), w.x[i]);
        v.y[i] = x2_mul(x2_mul(v.y[i], inv), w.y[i]);
    }
}
// eight columns in order <-> half of a lane's: run `r` (0 or 1)
template <bool INTER> __device__ __forceinline__ void put_run(Cols &c, int r, const float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (!INTER) (r ? c.y : c.x)[i] = x2(v[2 * i], v[2 * i + 1]);
        else if (i < 2) c.x[2 * r + i] = x2(v[4 * i], v[4 * i + 2]);
        else c.y[2 * r + i - 2] = x2(v[4 * i - 7], v[4 * i - 5]);
    }
}
template <bool INTER> __device__ __forceinline__ void take_run(const Cols &c, int r, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (!INTER) x2_split((r ? c.y : c.x)[i], v[2 * i], v[2 * i + 1]);
        else if (i < 2) x2_split(c.x[2 * r + i], v[4 * i], v[4 * i + 2]);
        else x2_split(c.y[2 * r + i - 2], v[4 * i - 7], v[4 * i - 5]);
    }
}
// eight columns as loaded, to be widened later
template <typename E> struct Raw8 {
    uint4 w;
    __device__ __forceinline__ void load(const E *p) { w = *reinterpret_cast<const uint4 *>(p); }
    __device__ __forceinline__ void clear() { w = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void widen(float (&v)[8]) const;
};
template <> __device__ __forceinline__ void Raw8<__nv_bfloat16>::widen(float (&v)[8]) const {
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[2 * i] = bf16_lo(x[i]); v[2 * i + 1] = bf16_hi(x[i]); }
}
template <> __device__ __forceinline__ void Raw8<__half>::widen(float (&v)[8]) const {
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&x[i]));
        v[2 * i] = f.x; v[2 * i + 1] = f.y;
    }
}
template <> struct Raw8<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float *p) {
        a = *reinterpret_cast<const float4 *>(p);
        b = *reinterpret_cast<const float4 *>(p + 4);
    }
    __device__ __forceinline__ void clear() { a = b = make_float4(0.0f, 0.0f, 0.0f, 0.0f); }
    __device__ __forceinline__ void widen(float (&v)[8]) const {
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
};
// four columns as loaded
template <typename E> struct Raw4 {
    uint2 w;
    __device__ __forceinline__ void load(const E *p) { w = *reinterpret_cast<const uint2 *>(p); }
    __device__ __forceinline__ void widen(float *v) const;
};
template <> __device__ __forceinline__ void Raw4<__nv_bfloat16>::widen(float *v) const {
    v[0] = bf16_lo(w.x); v[1] = bf16_hi(w.x); v[2] = bf16_lo(w.y); v[3] = bf16_hi(w.y);
}
template <> __device__ __forceinline__ void Raw4<__half>::widen(float *v) const {
    const uint32_t x[2] = {w.x, w.y};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&x[i]));
        v[2 * i] = f.x; v[2 * i + 1] = f.y;
    }
}
template <> struct Raw4<float> {
    float4 w;
    __device__ __forceinline__ void load(const float *p) { w = *reinterpret_cast<const float4 *>(p); }
    __device__ __forceinline__ void widen(float *v) const { v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w; }
};
template <bool INTER, typename E> __device__ __forceinline__ void widen16(const Raw8<E> (&raw)[2], Cols &c) {
    float v[8];
    raw[0].widen(v);
    put_run<INTER>(c, 0, v);
    raw[1].widen(v);
    put_run<INTER>(c, 1, v);
}
template <bool INTER, typename E> __device__ __forceinline__ void store_runs(E *p, const Lane16 &l, const Cols &c) {
    float v[8];
    take_run<INTER>(c, 0, v);
    store8(p + l.a, v);
    take_run<INTER>(c, 1, v);
    store8(p + l.b, v);
}
template <bool INTER, typename E> __device__ __forceinline__ void load_weights16(const E *w, const Lane16 &l, Cols &c) {
    Raw8<E> raw[2];
    raw[0].load(w + l.a);
    raw[1].load(w + l.b);
    widen16<INTER>(raw, c);
}
template <bool INTER> __device__ __forceinline__ void load_weights16(const void *w, int wide, const Lane16 &l, Cols &c) {
    if (wide) load_weights16<INTER>(static_cast<const float *>(w), l, c);
    else load_weights16<INTER>(static_cast<const __nv_bfloat16 *>(w), l, c);
}

} // namespace rotary
} // namespace hn
