// fp4_quant.cu - the quantizer to 4-bit codes with block scales, and back.
//
//   MX   s = 2^(floor(log2 peak) - 2) per 32 columns (1 where all are 0), code = e2m1(x / s): the power of two is exact
//   NV   per row r = top / 2688 (448 x 6; 1 where top < 2^-100: such a row counts as zero), per 16 columns
//        s = e4m3((0.875 peak) / (top 2^-9)) = e4m3(448 peak / top), code = e2m1((0.65625 x) / (s top 2^-12)) = e2m1(x / (s r)).
//        In this order a 16-bit input is rounded once, at the division, so a value half-way between two codes is seen as such.
// A NaN or an infinity makes its block's scale NaN (MX) or its row's (NV), with zero codes, so that what reads it gives NaN.
//
// Bound by HBM: 2 B read (bf16) and 0.5 B + 1/16 B written per element. NV needs the row's top before its first code, so T
// threads hold a row in registers as it was loaded, NCH chunks of 16 columns each (chunk i T + t), and x is read once; rows of more
// than 16384 columns are read twice. A chunk is a block of NV and half a block of MX; the lanes of a scale tile's word (4 or
// 8) gather its bytes before the one store. Measured, 20240 x 4096 bf16: MX 32 us (6.5 TB/s), NV 41 us (5.2 TB/s: its twelve
// instructions a column, four of them the exact quotient, are what is left; a persistent loop over rows with the next one's loads
// ahead did not help). Rows that start on 4 or 8 bytes: 40000 x 1500 44 us (floor 23), 20240 x 4100 65; on odd elements 20240 x 4095 96, of
// fp32 163 (floor 58): one element a load. Back to bf16: 35 us (6.0 TB/s, 16 bytes out a thread and chunk, up to
// four chunks' loads under way). One row of 4096: 2.6 us, a launch.
#include "fp4.cuh"
#include "hn_kernels.h"

namespace hn {
namespace fp4q {

using namespace fp4;

struct Params {
    const void *x;
    int64_t ldx, M, rows;       // rows: M rounded up to whole scale tiles; those from M on get zero scales
    int K, nch, tiles;          // chunks of the padded row, group blocks
    uint8_t *q;
    int64_t ldq;
    uint8_t *s;
    float *r;
};

// sixteen columns as loaded, widened when they are used
template <typename E> struct Chunk {                // two to a word
    uint32_t w[8];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = 0;
    }
    __device__ __forceinline__ void load(const E *p) {
        const uint4 a = *reinterpret_cast<const uint4 *>(p), b = *reinterpret_cast<const uint4 *>(p + 8);
        w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w; w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
    }
    __device__ __forceinline__ void load4(const E *p) {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = reinterpret_cast<const uint32_t *>(p)[i];
    }
    __device__ __forceinline__ void put(int j, const E *p) { w[j >> 1] |= (uint32_t)*reinterpret_cast<const uint16_t *>(p) << (16 * (j & 1)); }
    __device__ __forceinline__ void widen(float (&v)[16]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 f = pair(w[i], E());
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
    static __device__ __forceinline__ float2 pair(uint32_t x, __nv_bfloat16) { return make_float2(bf16_lo(x), bf16_hi(x)); }
    static __device__ __forceinline__ float2 pair(uint32_t x, __half) { return __half22float2(*reinterpret_cast<const __half2 *>(&x)); }
};
template <> struct Chunk<float> {
    float w[16];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < 16; ++i) w[i] = 0.0f;
    }
    __device__ __forceinline__ void load(const float *p) {
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const float4 a = *reinterpret_cast<const float4 *>(p + i);
            w[i] = a.x; w[i + 1] = a.y; w[i + 2] = a.z; w[i + 3] = a.w;
        }
    }
    __device__ __forceinline__ void load4(const float *p) {
#pragma unroll
        for (int i = 0; i < 16; ++i) w[i] = p[i];
    }
    __device__ __forceinline__ void put(int j, const float *p) { w[j] = *p; }
    __device__ __forceinline__ void widen(float (&v)[16]) const {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = w[i];
    }
};

// columns 16 c to 16 c + 15 of a row, zeros behind its end. VEC: all rows start on 16 bytes (2), on 4 (1, 16-bit types), or
// anywhere (0)
template <typename E, int VEC> __device__ __forceinline__ void load_chunk(const E *row, int c, int K, Chunk<E> &v) {
    v.clear();
    if (VEC == 2 && 16 * c + 16 <= K) {
        v.load(row + 16 * c);
    } else if (VEC == 1 && 16 * c + 16 <= K) {
        v.load4(row + 16 * c);
    } else {
#pragma unroll
        for (int j = 0; j < 16; ++j)
            if (16 * c + j < K) v.put(j, row + 16 * c + j);
    }
}
// The largest magnitude of a chunk as a number that orders as magnitudes do, NaN above infinity: of 16-bit types the bits without
// the sign (two columns an instruction), of fp32 the value. `magnitude` makes it a float (a NaN or an infinity of its own).
__device__ __forceinline__ uint32_t peak_bits(const uint32_t (&w)[8]) {
    uint32_t m = __vimax3_u16x2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu, w[2] & 0x7fff7fffu);
    m = __vimax3_u16x2(m, w[3] & 0x7fff7fffu, w[4] & 0x7fff7fffu);
    m = __vimax3_u16x2(m, w[5] & 0x7fff7fffu, w[6] & 0x7fff7fffu);
    m = __vmaxu2(m, w[7] & 0x7fff7fffu);
    return max(m & 0xffffu, m >> 16);
}
template <typename E> __device__ __forceinline__ uint32_t peak16(const Chunk<E> &c) { return peak_bits(c.w); }
template <> __device__ __forceinline__ uint32_t peak16(const Chunk<float> &c) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 16; j += 2) m = __vimax3_u32(m, __float_as_uint(c.w[j]) & 0x7fffffffu, __float_as_uint(c.w[j + 1]) & 0x7fffffffu);
    return m;
}
template <typename E> __device__ __forceinline__ float magnitude(uint32_t bits);
template <> __device__ __forceinline__ float magnitude<__nv_bfloat16>(uint32_t bits) { return __uint_as_float(bits << 16); }
template <> __device__ __forceinline__ float magnitude<__half>(uint32_t bits) { return __half2float(__ushort_as_half((unsigned short)bits)); }
template <> __device__ __forceinline__ float magnitude<float>(uint32_t bits) { return __uint_as_float(bits); }
template <int W> __device__ __forceinline__ uint32_t lanes_most(uint32_t v) {
#pragma unroll
    for (int o = 1; o < W; o <<= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ uint2 pack16(const float (&v)[16]) {
    return make_uint2(pack8_e2m1(*reinterpret_cast<const float(*)[8]>(v)), pack8_e2m1(*reinterpret_cast<const float(*)[8]>(v + 8)));
}

// MX: codes and scale byte of a chunk whose block's largest magnitude is `peak`
template <typename E> __device__ __forceinline__ uint2 chunk_mx(const Chunk<E> &c, float peak, uint32_t &byte) {
    const uint32_t be = __float_as_uint(peak) >> 23;
    if (be == 255) { byte = 255; return make_uint2(0, 0); }
    byte = peak == 0.0f ? 127 : be < 2 ? 0 : be - 2;
    const uint64_t inv = x2_splat(__uint_as_float((254 - byte) << 23));     // 2^(127 - byte): byte <= 252
    float v[16];
    c.widen(v);
#pragma unroll
    for (int j = 0; j < 16; j += 2) x2_split(x2_mul(x2(v[j], v[j + 1]), inv), v[j], v[j + 1]);
    return pack16(v);
}

// what a row's top fixes
struct RowNV {
    float ndiv, rdiv, den;      // -top 2^-9, its reciprocal, top 2^-12
    bool live;
};
__device__ __forceinline__ RowNV row_nv(float top, float *r) {
    RowNV n;
    n.live = top >= 0x1p-100f && top < INFINITY;
    n.ndiv = top * -0x1p-9f;
    n.rdiv = __frcp_rn(top * 0x1p-9f);
    n.den = top * 0x1p-12f;
    *r = n.live ? __fdiv_rn(top, 2688.0f) : top < 0x1p-100f ? 1.0f : __int_as_float(0x7fffffff);
    return n;
}
template <typename E> __device__ __forceinline__ uint2 chunk_nv(const Chunk<E> &c, float peak, const RowNV &n, uint32_t &byte) {
    byte = 0;
    if (!n.live) return make_uint2(0, 0);
    // RN(0.875 peak / (top 2^-9)): the quotient corrected once, as in x2_quot (what a remainder loses below 2^-126 is far below
    // the smallest scale)
    const float a = 0.875f * peak, q0 = a * n.rdiv;
    byte = e4m3_byte(fmaf(fmaf(q0, n.ndiv, a), n.rdiv, q0));
    if (byte == 0) return make_uint2(0, 0);
    const float den = scale_value<NV>(byte) * n.den;
    float v[16];
    c.widen(v);
    if (den >= 0x1p-90f) {
        // x2_quot with the remainder's and the reciprocal's signs turned: a zero keeps its sign
        const uint64_t d = x2_splat(den), nr = x2_splat(-__frcp_rn(den));
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
            const uint64_t np = x2_mul(x2(v[j], v[j + 1]), x2_splat(-0.65625f)), q0 = x2_mul(np, nr);
            x2_split(x2_fma(x2_fma(q0, d, np), nr, q0), v[j], v[j + 1]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = __fdiv_rn(0.65625f * v[j], den);
    }
    return pack16(v);
}

// the bytes of W neighbouring lanes' blocks (B lanes each) -> one word in every lane
template <int W, int B> __device__ __forceinline__ uint32_t gather_word(uint32_t byte) {
    uint32_t w = byte << (8 * ((threadIdx.x % W) / B));
#pragma unroll
    for (int o = B; o < W; o <<= 1) w |= __shfl_xor_sync(0xffffffffu, w, o);
    return w;
}

// T threads a row (below 32: so many lanes of a warp), the row in registers
template <typename E, int KIND, int VEC, int T, int NCH>
__global__ void __launch_bounds__(T < 128 ? 128 : T) k_quant_fp4(Params p) {
    constexpr int BLK = GROUP<KIND> / 16, LANES = SPAN<KIND> / 16, W = LANES < T ? LANES : T;
    __shared__ uint32_t red[T < 128 ? 128 / T : 1][T < 32 ? 1 : T / 32];
    const int t = threadIdx.x % T, lane = threadIdx.x & 31, warp = (threadIdx.x % T) >> 5;
    const int64_t m = T < 128 ? (int64_t)blockIdx.x * (128 / T) + threadIdx.x / T : (int64_t)blockIdx.x;
    const bool row = m < p.M;                   // p.rows is whole blocks of threads, so no thread leaves before a shuffle
    Chunk<E> v[NCH];
    uint32_t peak[NCH];
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        const int c = i * T + t;
        load_chunk<E, VEC>(static_cast<const E *>(p.x) + m * p.ldx, c, row ? p.K : 0, v[i]);
    }
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        peak[i] = lanes_most<BLK>(peak16(v[i]));
        top = max(top, peak[i]);
    }
    RowNV n;
    if (KIND == NV) {
#pragma unroll
        for (int o = 1; o < (T < 32 ? T : 32); o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (T > 32) {
            uint32_t *mine = red[T < 128 ? threadIdx.x / T : 0];
            if (lane == 0) mine[warp] = top;
            __syncthreads();
            top = mine[0];
#pragma unroll
            for (int i = 1; i < T / 32; ++i) top = max(top, mine[i]);
        }
        float r;
        n = row_nv(magnitude<E>(top), &r);
        if (row && t == 0) p.r[m] = r;
    }
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        const int c = i * T + t;
        uint32_t byte = 0;
        if (row && c < p.nch)
            *reinterpret_cast<uint2 *>(p.q + m * p.ldq + 8 * c) = KIND == MX ? chunk_mx(v[i], magnitude<E>(peak[i]), byte) : chunk_nv(v[i], magnitude<E>(peak[i]), n, byte);
        const uint32_t word = gather_word<W, BLK>(byte);
        if (t % W == 0 && c / LANES < p.tiles) *reinterpret_cast<uint32_t *>(p.s + scale_word(m, c / LANES, p.tiles)) = word;
    }
}

// any row length: the row's top in a pass of its own (NV)
template <typename E, int KIND, int VEC> __global__ void __launch_bounds__(256) k_quant_fp4_long(Params p) {
    constexpr int BLK = GROUP<KIND> / 16, LANES = SPAN<KIND> / 16, T = 256;
    __shared__ uint32_t red[T / 32];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int64_t m = blockIdx.x;
    const bool row = m < p.M;
    const E *x = static_cast<const E *>(p.x) + m * p.ldx;
    RowNV n;
    if (KIND == NV) {
        uint32_t top = 0;
#pragma unroll 4
        for (int c = t; c < (row ? p.nch : 0); c += T) {
            Chunk<E> v;
            load_chunk<E, VEC>(x, c, p.K, v);
            top = max(top, peak16(v));
        }
        top = lanes_most<32>(top);
        if (lane == 0) red[warp] = top;
        __syncthreads();
        top = red[0];
#pragma unroll
        for (int i = 1; i < T / 32; ++i) top = max(top, red[i]);
        float r;
        n = row_nv(magnitude<E>(top), &r);
        if (row && t == 0) p.r[m] = r;
    }
    for (int c0 = 0; c0 < p.tiles * LANES; c0 += T) {           // whole warps: the words' lanes stay together
        const int c = c0 + t;
        Chunk<E> v;
        load_chunk<E, VEC>(x, c, row ? p.K : 0, v);
        const float peak = magnitude<E>(lanes_most<BLK>(peak16(v)));
        uint32_t byte = 0;
        if (row && c < p.nch)
            *reinterpret_cast<uint2 *>(p.q + m * p.ldq + 8 * c) = KIND == MX ? chunk_mx(v, peak, byte) : chunk_nv(v, peak, n, byte);
        const uint32_t word = gather_word<LANES, BLK>(byte);
        if (t % LANES == 0 && c / LANES < p.tiles) *reinterpret_cast<uint32_t *>(p.s + scale_word(m, c / LANES, p.tiles)) = word;
    }
}

template <typename E, int KIND, int VEC, int T, int NCH> cudaError_t go(const Params &p, cudaStream_t st) {
    constexpr int per = T < 128 ? 128 / T : 1;
    k_quant_fp4<E, KIND, VEC, T, NCH><<<(unsigned)cdiv(p.rows, per), T < 128 ? 128 : T, 0, st>>>(p);
    return cudaGetLastError();
}

// T and NCH by the row's length alone: the fewest chunks that hold it. Measured, bf16, NV (MX), us: fewer than 32 threads a row against
// 32 for all: 400000 x 32 9 (7) / 130 (93), 400000 x 128 32 (24) / 132 (95), 300000 x 256 46 (34) / 100 (73). Three chunks against the
// next power of two: 60000 x 1040 47 (35) / 60 (42), 30000 x 3008 47 (38) / 59 (42), 12000 x 6000 41 (31) / 48 (35),
// 6000 x 12000 45 (30) / 67 (34)
template <typename E, int KIND, int VEC> cudaError_t pick(const Params &p, cudaStream_t st) {
    if (p.nch <= 2) return go<E, KIND, VEC, 2, 1>(p, st);
    if (p.nch <= 4) return go<E, KIND, VEC, 4, 1>(p, st);
    if (p.nch <= 8) return go<E, KIND, VEC, 8, 1>(p, st);
    if (p.nch <= 16) return go<E, KIND, VEC, 16, 1>(p, st);
    if (p.nch <= 32) return go<E, KIND, VEC, 32, 1>(p, st);
    if (p.nch <= 64) return go<E, KIND, VEC, 32, 2>(p, st);
    if (p.nch <= 96) return go<E, KIND, VEC, 32, 3>(p, st);
    if (p.nch <= 128) return go<E, KIND, VEC, 64, 2>(p, st);
    if (p.nch <= 192) return go<E, KIND, VEC, 64, 3>(p, st);
    if (p.nch <= 256) return go<E, KIND, VEC, 128, 2>(p, st);
    if (p.nch <= 384) return go<E, KIND, VEC, 128, 3>(p, st);
    if (p.nch <= 512) return go<E, KIND, VEC, 256, 2>(p, st);
    if (p.nch <= 768) return go<E, KIND, VEC, 256, 3>(p, st);
    if (p.nch <= 1024) return go<E, KIND, VEC, 512, 2>(p, st);
    k_quant_fp4_long<E, KIND, VEC><<<(unsigned)p.rows, 256, 0, st>>>(p);
    return cudaGetLastError();
}
template <typename E> cudaError_t pick_kind(const Params &p, int kind, cudaStream_t st) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p.x) | (uintptr_t)(p.ldx * (int64_t)sizeof(E));
    if (at % 16 == 0) return kind == MX ? pick<E, MX, 2>(p, st) : pick<E, NV, 2>(p, st);
    if constexpr (sizeof(E) == 2)
        if (at % 4 == 0) return kind == MX ? pick<E, MX, 1>(p, st) : pick<E, NV, 1>(p, st);
    return kind == MX ? pick<E, MX, 0>(p, st) : pick<E, NV, 0>(p, st);
}

struct BackParams {
    const uint8_t *q;
    int64_t ldq, M;
    int K, nch, tiles;          // chunks of 8 columns
    const uint8_t *s;
    const float *r;
    void *out;
    int64_t ldo;
};

template <typename E> __device__ __forceinline__ void store1(E *p, float v);
template <> __device__ __forceinline__ void store1(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ void store1(__half *p, float v) { *p = __float2half_rn(v); }
template <> __device__ __forceinline__ void store1(float *p, float v) { *p = v; }
__device__ __forceinline__ void store8(__nv_bfloat16 *o, const float (&v)[8]) {
    *reinterpret_cast<uint4 *>(o) = make_uint4(pack_bf16_rn(v[0], v[1]), pack_bf16_rn(v[2], v[3]), pack_bf16_rn(v[4], v[5]), pack_bf16_rn(v[6], v[7]));
}
__device__ __forceinline__ void store8(__half *o, const float (&v)[8]) {
    *reinterpret_cast<uint4 *>(o) = make_uint4(pack_f16_rn(v[0], v[1]), pack_f16_rn(v[2], v[3]), pack_f16_rn(v[4], v[5]), pack_f16_rn(v[6], v[7]));
}
__device__ __forceinline__ void store8(float *o, const float (&v)[8]) {
    *reinterpret_cast<float4 *>(o) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4 *>(o + 4) = make_float4(v[4], v[5], v[6], v[7]);
}

// code * RN(scale * row scale), one rounding to the output type. T threads a row, which take its chunks of 8 columns in turn (16
// bytes out, neighbouring lanes write on), so that a row's address and scale are worked out once. VEC: 16-byte stores
template <typename E, int KIND, bool VEC, int T, int U> __global__ void __launch_bounds__(256) k_dequant_fp4(BackParams p) {
    const int64_t m = (int64_t)blockIdx.x * (256 / T) + threadIdx.x / T;
    if (m >= p.M) return;
    const uint32_t *q = reinterpret_cast<const uint32_t *>(p.q + m * p.ldq);
    const uint8_t *s = p.s + scale_word(m, 0, p.tiles);
    const float r = KIND == NV ? p.r[m] : 1.0f;
    E *out = static_cast<E *>(p.out) + m * p.ldo;
    for (int c0 = threadIdx.x % T; c0 < p.nch; c0 += U * T) {
        uint32_t w[U];
        uint8_t sb[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int c = c0 + i * T, g = 8 * c / GROUP<KIND>;
            w[i] = c < p.nch ? q[c] : 0;
            sb[i] = c < p.nch ? s[(int64_t)(g >> 2) * TILE + (g & 3)] : 0;
        }
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int c = c0 + i * T;
            if (c >= p.nch) break;
            float d = scale_value<KIND>(sb[i]);
            if (KIND == NV) d = __fmul_rn(d, r);
            uint32_t h[4];
            unpack8_e2m1(w[i], h);
            float v[8];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h[k]));
                v[2 * k] = f.x * d;
                v[2 * k + 1] = f.y * d;
            }
            if (VEC && 8 * c + 8 <= p.K) {
                store8(out + 8 * c, v);
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (8 * c + k < p.K) store1(out + 8 * c + k, v[k]);
            }
        }
    }
}

template <typename E, int KIND, bool VEC> cudaError_t back_rows(const BackParams &p, cudaStream_t st) {
    auto go = [&](auto kernel, int per) {
        kernel<<<(unsigned)cdiv(p.M, per), 256, 0, st>>>(p);
        return cudaGetLastError();
    };
    // Two to eight chunks a thread where there are rows enough, all on their way together. Measured, bf16, against one to four, two at
    // a time (us): 20240 x 4096 NV 44.2 -> 35.3, 80960 x 1024 44.1 -> 35.6, 20240 x 2080 30.7 -> 21.0. Few rows: more threads a row
    // (1 x 4096: 2.2, as above 2.6)
    const bool few = p.M < 8 * num_sms();
    if (p.nch <= 4) return go(k_dequant_fp4<E, KIND, VEC, 4, 1>, 64);
    if (p.nch <= 8) return go(k_dequant_fp4<E, KIND, VEC, 4, 2>, 64);
    if (p.nch <= 32) return go(k_dequant_fp4<E, KIND, VEC, 16, 2>, 16);
    if (p.nch <= 128 && !few) return go(k_dequant_fp4<E, KIND, VEC, 16, 4>, 16);
    if (p.nch <= 256 || (p.nch <= 1024 && !few)) return go(k_dequant_fp4<E, KIND, VEC, 64, 4>, 4);
    return go(k_dequant_fp4<E, KIND, VEC, 256, 4>, 1);
}
template <typename E> cudaError_t back(const BackParams &p, int kind, cudaStream_t st) {
    const bool vec = reinterpret_cast<uintptr_t>(p.out) % 16 == 0 && p.ldo * (int64_t)sizeof(E) % 16 == 0;
    if (kind == MX) return vec ? back_rows<E, MX, true>(p, st) : back_rows<E, MX, false>(p, st);
    return vec ? back_rows<E, NV, true>(p, st) : back_rows<E, NV, false>(p, st);
}

} // namespace fp4q

cudaError_t launch_quant_fp4(const void *x, int64_t ldx, int x_dtype, int64_t M, int64_t K, int kind, void *q, int64_t ldq,
                             void *s, float *r, cudaStream_t st) {
    fp4q::Params p;
    p.x = x; p.ldx = ldx; p.M = M; p.rows = cdiv(M, 128) * 128; p.K = (int)K;
    p.nch = (int)(cdiv(K, 32) * 2);
    p.tiles = (int)cdiv(K, kind == fp4::MX ? 128 : 64);
    p.q = static_cast<uint8_t *>(q); p.ldq = ldq; p.s = static_cast<uint8_t *>(s); p.r = r;
    if (x_dtype == 0) return fp4q::pick_kind<__nv_bfloat16>(p, kind, st);
    if (x_dtype == 1) return fp4q::pick_kind<__half>(p, kind, st);
    return fp4q::pick_kind<float>(p, kind, st);
}

cudaError_t launch_dequant_fp4(const void *q, int64_t ldq, const void *s, const float *r, int64_t M, int64_t K, int64_t Kp,
                               int kind, void *out, int64_t ldo, int out_dtype, cudaStream_t st) {
    fp4q::BackParams p;
    p.q = static_cast<const uint8_t *>(q); p.ldq = ldq; p.M = M; p.K = (int)K; p.nch = (int)cdiv(K, 8);
    p.tiles = (int)cdiv(Kp, kind == fp4::MX ? 128 : 64);
    p.s = static_cast<const uint8_t *>(s); p.r = r; p.out = out; p.ldo = ldo;
    if (out_dtype == 0) return fp4q::back<__nv_bfloat16>(p, kind, st);
    if (out_dtype == 1) return fp4q::back<__half>(p, kind, st);
    return fp4q::back<float>(p, kind, st);
}

} // namespace hn
