// fp4_quant.cu - the quantizer to 4-bit codes with block scales, and back.
//
//   MX   s = 2^(floor(log2 peak) - 2) per 32 columns (1 where all are 0), code = e2m1(x / s): the power of two is exact
//   NV   per row r = top / 2688 (448 x 6; 1 where top < 2^-100: such a row counts as zero), per 16 columns
//        s = e4m3((0.875 peak) / (top 2^-9)) = e4m3(448 peak / top), code = e2m1((0.65625 x) / (s top 2^-12)) = e2m1(x / (s r)).
//        In this order a 16-bit input is rounded once, at the division, so a value half-way between two codes is seen as such.
// A NaN or an infinity makes its block's scale NaN (MX) or its row's (NV), with zero codes, so that what reads it gives NaN.
//
// Bound by HBM: 2 B read (bf16) and 0.5 B + 1/16 B written per element. NV needs the row's top before its first code, so T
// threads hold a row in registers, NCH chunks of 8 columns each (chunk i T + t), and x is read once; rows of more than 16384
// columns are read twice. A chunk's block is 2 (NV) or 4 (MX) neighbouring lanes, and the lanes of a scale tile's word (8 or
// 16) gather its bytes before the one store.
#include "fp4.cuh"
#include "hn_kernels.h"

namespace hn {
namespace fp4q {

using namespace fp4;

struct Params {
    const void *x;
    int64_t ldx, M, rows;       // rows: M rounded up to whole scale tiles; those from M on get zero scales
    int K, nch, tiles;          // chunks of the padded row, group blocks
    uint32_t *q;                // [M][nch] words of eight codes
    int64_t ldq;                // in words
    uint8_t *s;
    float *r;
};

// columns 8 c to 8 c + 7 of a row, zeros behind its end. VEC: the row starts on 16 bytes
template <typename E, bool VEC> __device__ __forceinline__ void load_chunk(const E *row, int c, int K, float (&v)[8]) {
    if (VEC && 8 * c + 8 <= K) {
        Elem<E>::load8(row + 8 * c, v);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 8 * c + j < K ? Elem<E>::load1(row + 8 * c + j) : 0.0f;
    }
}
__device__ __forceinline__ float peak8(const float (&v)[8]) {
    float p = nanmax_abs3(0.0f, v[0], v[1]);
    p = nanmax_abs3(p, v[2], v[3]);
    p = nanmax_abs3(p, v[4], v[5]);
    return nanmax_abs3(p, v[6], v[7]);
}

// MX: codes and scale byte of a chunk whose block's largest magnitude is `peak`
__device__ __forceinline__ uint32_t chunk_mx(float (&v)[8], float peak, uint32_t &byte) {
    const uint32_t be = __float_as_uint(peak) >> 23;
    if (be == 255) { byte = 255; return 0; }
    byte = peak == 0.0f ? 127 : be < 2 ? 0 : be - 2;
    const float inv = __uint_as_float((254 - byte) << 23);      // 2^(127 - byte): byte <= 252
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= inv;
    return pack8_e2m1(v);
}

// what a row's top fixes
struct RowNV {
    float div, den;      // top 2^-9 and top 2^-12
    bool live;
};
__device__ __forceinline__ RowNV row_nv(float top, float *r) {
    RowNV n;
    n.live = top >= 0x1p-100f && top < INFINITY;
    n.div = top * 0x1p-9f;
    n.den = top * 0x1p-12f;
    *r = n.live ? __fdiv_rn(top, 2688.0f) : top < 0x1p-100f ? 1.0f : __int_as_float(0x7fffffff);
    return n;
}
__device__ __forceinline__ uint32_t chunk_nv(float (&v)[8], float peak, const RowNV &n, uint32_t &byte) {
    byte = n.live ? e4m3_byte(__fdiv_rn(0.875f * peak, n.div)) : 0;
    if (byte == 0) return 0;
    const float den = scale_value<NV>(byte) * n.den;
    if (den >= 0x1p-90f) {
        const uint64_t ns = x2_splat(-den), rs = x2_splat(__frcp_rn(den));
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const uint64_t p = x2_mul(x2(v[j], v[j + 1]), x2_splat(0.65625f));
            float a, b;
            x2_split(x2_quot(p, ns, rs), a, b);
            v[j] = copysignf(a, v[j]);          // of a zero
            v[j + 1] = copysignf(b, v[j + 1]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = __fdiv_rn(0.65625f * v[j], den);
    }
    return pack8_e2m1(v);
}

// the bytes of W neighbouring lanes' blocks (B lanes each) -> one word in every lane
template <int W, int B> __device__ __forceinline__ uint32_t gather_word(uint32_t byte) {
    uint32_t w = byte << (8 * ((threadIdx.x % W) / B));
#pragma unroll
    for (int o = B; o < W; o <<= 1) w |= __shfl_xor_sync(0xffffffffu, w, o);
    return w;
}

// T threads a row (below 32: so many lanes of a warp), the row in registers
template <typename E, int KIND, bool VEC, int T, int NCH>
__global__ void __launch_bounds__(T < 128 ? 128 : T) k_quant_fp4(Params p) {
    constexpr int BLK = GROUP<KIND> / 8, LANES = SPAN<KIND> / 8, W = LANES < T ? LANES : T;
    __shared__ float red[T < 128 ? 1 : T / 32];
    const int t = threadIdx.x % T, lane = threadIdx.x & 31, warp = (threadIdx.x % T) >> 5;
    const int64_t m = T < 128 ? (int64_t)blockIdx.x * (128 / T) + threadIdx.x / T : (int64_t)blockIdx.x;
    const bool row = m < p.M;                   // p.rows is whole blocks of threads, so no thread leaves before a shuffle
    float v[NCH][8], peak[NCH];
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        const int c = i * T + t;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
        if (row && c < p.nch) load_chunk<E, VEC>(static_cast<const E *>(p.x) + m * p.ldx, c, p.K, v[i]);
    }
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        peak[i] = lanes_max<BLK>(peak8(v[i]));
        top = nanmax(top, peak[i]);
    }
    RowNV n;
    if (KIND == NV) {
#pragma unroll
        for (int o = BLK; o < (T < 32 ? T : 32); o <<= 1) top = nanmax(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (T >= 128) {
            if (lane == 0) red[warp] = top;
            __syncthreads();
            top = red[0];
#pragma unroll
            for (int i = 1; i < T / 32; ++i) top = nanmax(top, red[i]);
        }
        float r;
        n = row_nv(top, &r);
        if (row && t == 0) p.r[m] = r;
    }
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        const int c = i * T + t;
        uint32_t byte = 0;
        if (row && c < p.nch) p.q[m * p.ldq + c] = KIND == MX ? chunk_mx(v[i], peak[i], byte) : chunk_nv(v[i], peak[i], n, byte);
        const uint32_t word = gather_word<W, BLK>(byte);
        if (t % W == 0 && c / LANES < p.tiles) *reinterpret_cast<uint32_t *>(p.s + scale_word(m, c / LANES, p.tiles)) = word;
    }
}

// any row length: the row's top in a pass of its own (NV)
template <typename E, int KIND, bool VEC> __global__ void __launch_bounds__(256) k_quant_fp4_long(Params p) {
    constexpr int BLK = GROUP<KIND> / 8, LANES = SPAN<KIND> / 8, T = 256;
    __shared__ float red[T / 32];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int64_t m = blockIdx.x;
    const bool row = m < p.M;
    const E *x = static_cast<const E *>(p.x) + m * p.ldx;
    RowNV n;
    if (KIND == NV) {
        float top = 0.0f;
        for (int c = t; row && c < p.nch; c += T) {
            float v[8];
            load_chunk<E, VEC>(x, c, p.K, v);
            top = nanmax(top, peak8(v));
        }
        top = lanes_max<32>(top);
        if (lane == 0) red[warp] = top;
        __syncthreads();
        top = red[0];
#pragma unroll
        for (int i = 1; i < T / 32; ++i) top = nanmax(top, red[i]);
        float r;
        n = row_nv(top, &r);
        if (row && t == 0) p.r[m] = r;
    }
    for (int c0 = 0; c0 < p.tiles * LANES; c0 += T) {           // whole warps: the words' lanes stay together
        const int c = c0 + t;
        float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        if (row && c < p.nch) load_chunk<E, VEC>(x, c, p.K, v);
        const float peak = lanes_max<BLK>(peak8(v));
        uint32_t byte = 0;
        if (row && c < p.nch) p.q[m * p.ldq + c] = KIND == MX ? chunk_mx(v, peak, byte) : chunk_nv(v, peak, n, byte);
        const uint32_t word = gather_word<LANES, BLK>(byte);
        if (t % LANES == 0 && c / LANES < p.tiles) *reinterpret_cast<uint32_t *>(p.s + scale_word(m, c / LANES, p.tiles)) = word;
    }
}

template <typename E, int KIND, bool VEC, int T, int NCH> cudaError_t go(const Params &p, cudaStream_t st) {
    constexpr int per = T < 128 ? 128 / T : 1;
    k_quant_fp4<E, KIND, VEC, T, NCH><<<(unsigned)cdiv(p.rows, per), T < 128 ? 128 : T, 0, st>>>(p);
    return cudaGetLastError();
}

// T by the row's length alone, as the residual's norm and quantizer have it
template <typename E, int KIND, bool VEC> cudaError_t pick(const Params &p, cudaStream_t st) {
    if (p.nch <= 4) return go<E, KIND, VEC, 4, 1>(p, st);
    if (p.nch <= 16) return go<E, KIND, VEC, 16, 1>(p, st);
    if (p.nch <= 32) return go<E, KIND, VEC, 32, 1>(p, st);
    if (p.nch <= 64) return go<E, KIND, VEC, 32, 2>(p, st);
    if (p.nch <= 128) return go<E, KIND, VEC, 32, 4>(p, st);
    if (p.nch <= 256) return go<E, KIND, VEC, 128, 2>(p, st);
    if (p.nch <= 512) return go<E, KIND, VEC, 128, 4>(p, st);
    if (p.nch <= 1024) return go<E, KIND, VEC, 256, 4>(p, st);
    if (p.nch <= 2048) return go<E, KIND, VEC, 256, 8>(p, st);
    k_quant_fp4_long<E, KIND, VEC><<<(unsigned)p.rows, 256, 0, st>>>(p);
    return cudaGetLastError();
}
template <typename E> cudaError_t pick_kind(const Params &p, int kind, cudaStream_t st) {
    const bool vec = reinterpret_cast<uintptr_t>(p.x) % 16 == 0 && p.ldx * (int64_t)sizeof(E) % 16 == 0;
    if (kind == MX) return vec ? pick<E, MX, true>(p, st) : pick<E, MX, false>(p, st);
    return vec ? pick<E, NV, true>(p, st) : pick<E, NV, false>(p, st);
}

struct BackParams {
    const uint32_t *q;
    int64_t ldq, M;
    int K, nch, tiles;
    const uint8_t *s;
    const float *r;
    void *out;
    int64_t ldo;
};

// code * RN(scale * row scale), one rounding to the output type. A thread takes a chunk of 8 columns; VEC: 16-byte stores
template <typename E> __device__ __forceinline__ void store1(E *p, float v);
template <> __device__ __forceinline__ void store1(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ void store1(__half *p, float v) { *p = __float2half_rn(v); }
template <> __device__ __forceinline__ void store1(float *p, float v) { *p = v; }

template <typename E, int KIND, bool VEC> __global__ void __launch_bounds__(256) k_dequant_fp4(BackParams p) {
    const int64_t n = p.M * p.nch;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t m = div_nonneg(i, p.nch);
        const int c = (int)(i - m * p.nch), g = 8 * c / GROUP<KIND>;
        if (8 * c >= p.K) continue;
        const uint32_t w = p.q[m * p.ldq + c];
        float d = scale_value<KIND>(p.s[scale_word(m, g >> 2, p.tiles) + (g & 3)]);
        if (KIND == NV) d = __fmul_rn(d, p.r[m]);
        uint32_t h[4];
        unpack8_e2m1(w, h);
        float v[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h[j]));
            v[2 * j] = f.x * d;
            v[2 * j + 1] = f.y * d;
        }
        E *o = static_cast<E *>(p.out) + m * p.ldo + 8 * c;
        if (VEC && 8 * c + 8 <= p.K) {
            if (sizeof(E) == 4) {
                *reinterpret_cast<float4 *>(o) = make_float4(v[0], v[1], v[2], v[3]);
                *reinterpret_cast<float4 *>(reinterpret_cast<float *>(o) + 4) = make_float4(v[4], v[5], v[6], v[7]);
            } else {
                E e[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) store1(&e[j], v[j]);
                *reinterpret_cast<uint4 *>(o) = *reinterpret_cast<uint4 *>(e);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (8 * c + j < p.K) store1(o + j, v[j]);
        }
    }
}

template <typename E> cudaError_t back(const BackParams &p, int kind, cudaStream_t st) {
    const bool vec = reinterpret_cast<uintptr_t>(p.out) % 16 == 0 && p.ldo * (int64_t)sizeof(E) % 16 == 0;
    const int64_t want = cdiv(p.M * p.nch, 256), most = (int64_t)num_sms() * 8;
    const unsigned grid = (unsigned)(want < most ? want : most);
    if (kind == MX) {
        if (vec) k_dequant_fp4<E, MX, true><<<grid, 256, 0, st>>>(p);
        else k_dequant_fp4<E, MX, false><<<grid, 256, 0, st>>>(p);
    } else {
        if (vec) k_dequant_fp4<E, NV, true><<<grid, 256, 0, st>>>(p);
        else k_dequant_fp4<E, NV, false><<<grid, 256, 0, st>>>(p);
    }
    return cudaGetLastError();
}

} // namespace fp4q

cudaError_t launch_quant_fp4(const void *x, int64_t ldx, int x_dtype, int64_t M, int64_t K, int kind, void *q, int64_t ldq,
                             void *s, float *r, cudaStream_t st) {
    fp4q::Params p;
    p.x = x; p.ldx = ldx; p.M = M; p.rows = cdiv(M, 128) * 128; p.K = (int)K;
    p.nch = (int)(cdiv(K, 32) * 4);
    p.tiles = (int)cdiv(K, kind == fp4::MX ? 128 : 64);
    p.q = static_cast<uint32_t *>(q); p.ldq = ldq / 4; p.s = static_cast<uint8_t *>(s); p.r = r;
    if (x_dtype == 0) return fp4q::pick_kind<__nv_bfloat16>(p, kind, st);
    if (x_dtype == 1) return fp4q::pick_kind<__half>(p, kind, st);
    return fp4q::pick_kind<float>(p, kind, st);
}

cudaError_t launch_dequant_fp4(const void *q, int64_t ldq, const void *s, const float *r, int64_t M, int64_t K, int64_t Kp,
                               int kind, void *out, int64_t ldo, int out_dtype, cudaStream_t st) {
    fp4q::BackParams p;
    p.q = static_cast<const uint32_t *>(q); p.ldq = ldq / 4; p.M = M; p.K = (int)K; p.nch = (int)cdiv(K, 8);
    p.tiles = (int)cdiv(Kp, kind == fp4::MX ? 128 : 64);
    p.s = static_cast<const uint8_t *>(s); p.r = r; p.out = out; p.ldo = ldo;
    if (out_dtype == 0) return fp4q::back<__nv_bfloat16>(p, kind, st);
    if (out_dtype == 1) return fp4q::back<__half>(p, kind, st);
    return fp4q::back<float>(p, kind, st);
}

} // namespace hn
