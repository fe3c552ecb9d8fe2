// fp4_gemv.cu - the product of few rows of activations with 4-bit weights: a read of the weights, once.
//
// Bound by HBM: half a byte and 1/16 (1/32) byte of scales per weight. A CTA takes the eight weight rows r and r + 1 of each
// quarter of a scale tile's 128 (their scales are 32 neighbouring bytes), its warps the chunks of 1024 columns in turn, so a
// lane has 16 bytes of every row in flight. Codes become fp16 pairs, exactly; the products of a block of 16 are
// summed in fp16 pairs of eight products each, whose sum is exact too (at most 288 in steps of 0.25: 1152 of 2048), and leave
// as fp32, times both scales. MX: these are powers of two that may be far apart, whose product with a sum need not be (2^125 and
// 2^-27), so the activations' goes in two factors with exponents of one sign, half before the weights' and half after: no step
// leaves fp32 unless the result does. The order of the sums is fixed. Measured: one row over 4096 x 16384 NV: 9.7 us with its launch
// (3.9 TB/s; with weights from HBM, 12 sets in turn, 9.8), MX 10.7, two rows 14.2 (the tile kernel, three rows and more: 15). Four rows in flight and 64 registers, so that all CTAs of
// that case are resident: 10.8 -> 9.7.
#include "fp4.cuh"
#include "hn_kernels.h"

namespace hn {
namespace fp4v {

using namespace fp4;

constexpr int ROWS = 8, CHUNK = 1024, WARPS = 8;

struct Params {
    const uint8_t *qa, *sa, *qw, *sw;
    int64_t lda, ldw;
    int M, N, Kp, tiles;
    Result o;
};

__device__ __forceinline__ __half2 h2(uint32_t w) { return *reinterpret_cast<__half2 *>(&w); }

// 32 codes -> 16 pairs
__device__ __forceinline__ void unpack32(const uint4 &w, uint32_t (&h)[16]) {
    unpack8_e2m1(w.x, *reinterpret_cast<uint32_t(*)[4]>(h));
    unpack8_e2m1(w.y, *reinterpret_cast<uint32_t(*)[4]>(h + 4));
    unpack8_e2m1(w.z, *reinterpret_cast<uint32_t(*)[4]>(h + 8));
    unpack8_e2m1(w.w, *reinterpret_cast<uint32_t(*)[4]>(h + 12));
}
// sum of a block of 16 products
__device__ __forceinline__ float dot16(const uint32_t *a, const uint32_t *b) {
    __half2 s = __hmul2(h2(a[0]), h2(b[0]));
#pragma unroll
    for (int i = 1; i < 8; ++i) s = __hfma2(h2(a[i]), h2(b[i]), s);
    const float2 f = __half22float2(s);
    return f.x + f.y;
}

// the value of an MX scale byte (2^(byte - 127), 255: NaN) as two factors, their exponents of one sign and half of its each
__device__ __forceinline__ void halves(uint32_t byte, float (&f)[2]) {
    const int e = (int)byte - 127, h = e / 2;
    f[0] = byte == 255 ? __int_as_float(0x7fffffff) : __uint_as_float((uint32_t)(127 + h) << 23);
    f[1] = __uint_as_float((uint32_t)(127 + e - h) << 23);
}

template <int KIND, int MT> __global__ void __launch_bounds__(32 * WARPS, MT == 1 ? 4 : 2) k_fp4_gemv(Params p) {
    __shared__ float sums[WARPS][ROWS * MT];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int64_t block = blockIdx.x >> 4;                      // of 128 rows
    const int pair = 2 * (blockIdx.x & 15);                     // rows pair, pair + 1 of each 32
    float acc[MT][ROWS];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < ROWS; ++j) acc[i][j] = 0.0f;
    for (int c0 = warp * CHUNK; c0 < p.Kp; c0 += warps * CHUNK) {
        const int k = c0 + 32 * lane;
        const bool in = k < p.Kp;
        const int tile = k / SPAN<KIND>;                        // NV: a tile is two lanes' columns, MX: four lanes'
        const int g = KIND == NV ? 2 * (lane & 1) : lane & 3;   // the first of this lane's groups in it
        uint32_t x[MT][16];
        float xs[MT][2];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            uint4 a = make_uint4(0, 0, 0, 0);
            uint32_t word = 0;
            if (in && i < p.M) {
                a = __ldg(reinterpret_cast<const uint4 *>(p.qa + i * p.lda + (k >> 1)));
                word = __ldg(reinterpret_cast<const uint32_t *>(p.sa + scale_word(i, tile, p.tiles)));
            }
            unpack32(a, x[i]);
            if (KIND == MX) {
                halves(word >> (8 * g) & 255, xs[i]);
            } else {
                xs[i][0] = scale_value<KIND>(word >> (8 * g) & 255);
                xs[i][1] = scale_value<KIND>(word >> (8 * g + 8) & 255);
            }
        }
        const uint4 *scales = reinterpret_cast<const uint4 *>(p.sw + (block * p.tiles + tile) * TILE + 16 * pair);
#pragma unroll
        for (int half = 0; half < 2; ++half) {                  // row `pair`, then `pair` + 1, of each 32: four rows in flight
            uint4 w[4], s = make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t n = block * 128 + 32 * j + pair + half;
                w[j] = make_uint4(0, 0, 0, 0);
                if (in && n < p.N) w[j] = ldg_stream(p.qw + n * p.ldw + (k >> 1));
            }
            if (in) s = __ldg(scales + half);
            const uint32_t words[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float s0 = scale_value<KIND>(words[j] >> (8 * g) & 255);
                const float s1 = KIND == NV ? scale_value<KIND>(words[j] >> (8 * g + 8) & 255) : 0.0f;
                uint32_t h[16];
                unpack32(w[j], h);
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    const float d0 = dot16(h, x[i]), d1 = dot16(h + 8, x[i] + 8);
                    float &sum = acc[i][2 * j + half];
                    if (KIND == NV) sum = fmaf(d1, xs[i][1] * s1, fmaf(d0, xs[i][0] * s0, sum));
                    else sum = fmaf((d0 + d1) * xs[i][0] * s0, xs[i][1], sum);
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < ROWS; ++j) {
            const float v = warp_sum_tree(acc[i][j]);
            if (lane == 0) sums[warp][i * ROWS + j] = v;
        }
    __syncthreads();
    const int t = threadIdx.x;
    if (t >= ROWS * MT) return;
    const int i = t / ROWS, j = t % ROWS;
    const int64_t n = block * 128 + 32 * (j >> 1) + pair + (j & 1);
    if (i >= p.M || n >= p.N) return;
    float v = sums[0][t];
    for (int w = 1; w < warps; ++w) v += sums[w][t];
    store_result(p.o, i * p.o.ldo + n, finish(p.o, v, p.o.ra ? p.o.ra[i] : 1.0f, n));
}

template <int KIND> cudaError_t go(const Params &p, cudaStream_t st) {
    const int chunks = (int)cdiv(p.Kp, CHUNK), warps = chunks < WARPS ? chunks : WARPS;
    const unsigned grid = (unsigned)(cdiv(p.N, 128) * 16);
    if (p.M == 1) k_fp4_gemv<KIND, 1><<<grid, 32 * warps, 0, st>>>(p);
    else k_fp4_gemv<KIND, 2><<<grid, 32 * warps, 0, st>>>(p);
    return cudaGetLastError();
}

} // namespace fp4v

bool fp4_gemv_applies(const Fp4GemmArgs &a) { return a.M <= FP4_GEMV_MAX_M; }

cudaError_t launch_fp4_gemv(const Fp4GemmArgs &a, cudaStream_t st) {
    fp4v::Params p;
    p.qa = static_cast<const uint8_t *>(a.qa); p.sa = static_cast<const uint8_t *>(a.sa); p.lda = a.lda;
    p.qw = static_cast<const uint8_t *>(a.qw); p.sw = static_cast<const uint8_t *>(a.sw); p.ldw = a.ldw;
    p.M = (int)a.M; p.N = (int)a.N; p.Kp = (int)a.K;
    p.tiles = (int)cdiv(a.K, a.kind == fp4::MX ? 128 : 64);
    p.o = {a.ra, a.rw, a.bias, a.bias_dtype, a.out, a.ldo, a.out_dtype};
    return a.kind == fp4::MX ? fp4v::go<fp4::MX>(p, st) : fp4v::go<fp4::NV>(p, st);
}

} // namespace hn
