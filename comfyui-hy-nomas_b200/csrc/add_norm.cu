// add_norm.cu - the residual's addition, RMSNorm and the 8-bit quantizer of the linears that follow, in one pass:
//   h = x + r (fp32);  out = bf16(h);  y = h / sqrt(mean(h^2) + eps) * w;  codes and scales of y
// per row and 128 columns, or per row. The sum is rounded once, where it is stored: the norm reads the unrounded h, and y
// goes to the quantizer in fp32 (int8: absmax / 127, half away from zero; e4m3: max(absmax, 1e-12) / 448, nearest
// even), so each output carries one rounding. A NaN in a row gives NaN scales.
//
// Bound by HBM: 4 B read and 3 B written per element (+ scales). T threads hold a row in registers, NCH chunks of 8
// elements each (chunk i * T + t at elements [8c, 8c + 8)), so that x and r are read once; a 128-column group is 16
// neighbouring lanes of one i. Measured (kernel alone): 20240 x 4096, e4m3: 89 us, 6.5 TB/s; 1 x 4096: 4.2 us, a launch.
#include "hn_common.cuh"
#include "hn_kernels.h"

namespace hn {
namespace addnorm {

// absmax -> scale; a zero group has scale 1 (int8), a NaN stays a NaN
template <int KIND> __device__ __forceinline__ float scale_of(float peak) {
    if (KIND == 0) return peak == 0.0f ? 1.0f : __fdiv_rn(peak, 127.0f);
    return __fdiv_rn(peak < 1e-12f ? 1e-12f : peak, 448.0f);
}

struct Params {
    const __nv_bfloat16 *x, *r, *w;
    __nv_bfloat16 *out;
    uint8_t *q;
    float *s;
    int64_t ldx, ldr, ldo, ldq, s_rs, s_gs, rows;
    int D;
    float eps;
};

// ROW: one scale per row. Blocks of max(T, 128) threads; a warp per row (T = 32) needs no shared memory.
template <int KIND, bool ROW, int T, int NCH>
__global__ void __launch_bounds__(T < 128 ? 128 : T) k_add_rms_quant(Params p) {
    constexpr int WARPS = T / 32;
    __shared__ float red[2][WARPS];
    const int t = threadIdx.x % T, lane = threadIdx.x & 31, warp = (threadIdx.x % T) >> 5;
    const int64_t m = T < 128 ? (int64_t)blockIdx.x * (128 / T) + threadIdx.x / T : (int64_t)blockIdx.x;
    if (T < 128 && m >= p.rows) return;             // whole warps
    const int nch = p.D >> 3;
    float h[NCH][8];
    uint4 a[NCH], b[NCH];
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        const int c = i * T + t;
        a[i] = b[i] = make_uint4(0, 0, 0, 0);
        if (c < nch) {
            a[i] = ldg_stream(p.x + m * p.ldx + 8 * c);
            b[i] = ldg_stream(p.r + m * p.ldr + 8 * c);
        }
    }
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        const uint32_t aw[4] = {a[i].x, a[i].y, a[i].z, a[i].w}, bw[4] = {b[i].x, b[i].y, b[i].z, b[i].w};
        uint32_t o[4];
        float part = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            h[i][2 * j] = __fadd_rn(bf16_lo(aw[j]), bf16_lo(bw[j]));
            h[i][2 * j + 1] = __fadd_rn(bf16_hi(aw[j]), bf16_hi(bw[j]));
            o[j] = bf16x2_rn(h[i][2 * j], h[i][2 * j + 1]);
            part = fmaf(h[i][2 * j], h[i][2 * j], part);
            part = fmaf(h[i][2 * j + 1], h[i][2 * j + 1], part);
        }
        ss += part;
        const int c = i * T + t;
        if (c < nch) *reinterpret_cast<uint4 *>(p.out + m * p.ldo + 8 * c) = make_uint4(o[0], o[1], o[2], o[3]);
    }
    ss = warp_sum_tree(ss);
    if (T > 32) {
        if (lane == 0) red[0][warp] = ss;
        __syncthreads();
        ss = 0.0f;
#pragma unroll
        for (int i = 0; i < WARPS; ++i) ss += red[0][i];
    }
    const float inv = rsqrt_cr(__fadd_rn(__fdiv_rn(ss, (float)p.D), p.eps));
    float peak[NCH];
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        const int c = i * T + t;
        float wv[8];
        if (c < nch) Elem<__nv_bfloat16>::load8(p.w + 8 * c, wv);
        peak[i] = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            h[i][j] = c < nch ? h[i][j] * inv * wv[j] : 0.0f;
            h[i][j + 1] = c < nch ? h[i][j + 1] * inv * wv[j + 1] : 0.0f;
            peak[i] = nanmax_abs3(peak[i], h[i][j], h[i][j + 1]);
        }
    }
    if (ROW) {
        float all = peak[0];
#pragma unroll
        for (int i = 1; i < NCH; ++i) all = nanmax(all, peak[i]);
        all = lanes_max<32>(all);
        if (T > 32) {
            if (lane == 0) red[1][warp] = all;
            __syncthreads();
            all = red[1][0];
#pragma unroll
            for (int i = 1; i < WARPS; ++i) all = nanmax(all, red[1][i]);
        }
#pragma unroll
        for (int i = 0; i < NCH; ++i) peak[i] = all;
    } else {
#pragma unroll
        for (int i = 0; i < NCH; ++i) peak[i] = lanes_max<16>(peak[i]);
    }
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        const int c = i * T + t;
        const float sc = scale_of<KIND>(peak[i]);
        const bool fast = sc >= 0x1p-90f;
        if (c < nch) {
            *reinterpret_cast<uint2 *>(p.q + m * p.ldq + 8 * c) =
                quant_chunk8<KIND, false>(h[i], sc, fast, x2_splat(-sc), x2_splat(__frcp_rn(sc)));
            if (ROW ? c == 0 : (c & 15) == 0) p.s[m * p.s_rs + (ROW ? 0 : (c >> 4)) * p.s_gs] = sc;
        }
    }
}

template <int KIND, bool ROW, int T, int NCH> cudaError_t go(const Params &p, cudaStream_t st) {
    constexpr int per = T < 128 ? 128 / T : 1;
    k_add_rms_quant<KIND, ROW, T, NCH><<<(unsigned)cdiv(p.rows, per), T < 128 ? 128 : T, 0, st>>>(p);
    return cudaGetLastError();
}

// T by the row's length alone: a warp up to 1024 columns, 128 threads up to 4096, 256 up to 16384
template <int KIND, bool ROW> cudaError_t pick(const Params &p, cudaStream_t st) {
    const int nch = p.D >> 3;
    if (nch <= 32) return go<KIND, ROW, 32, 1>(p, st);
    if (nch <= 64) return go<KIND, ROW, 32, 2>(p, st);
    if (nch <= 128) return go<KIND, ROW, 32, 4>(p, st);
    if (nch <= 256) return go<KIND, ROW, 128, 2>(p, st);
    if (nch <= 384) return go<KIND, ROW, 128, 3>(p, st);
    if (nch <= 512) return go<KIND, ROW, 128, 4>(p, st);
    if (nch <= 768) return go<KIND, ROW, 256, 3>(p, st);
    if (nch <= 1024) return go<KIND, ROW, 256, 4>(p, st);
    if (nch <= 1536) return go<KIND, ROW, 256, 6>(p, st);
    return go<KIND, ROW, 256, 8>(p, st);
}

} // namespace addnorm

cudaError_t launch_add_rmsnorm_quant(const void *x, int64_t ldx, const void *r, int64_t ldr, const void *weight,
                                     int64_t rows, int64_t D, float eps, int kind, bool per_row, void *out, int64_t ldo,
                                     void *q, int64_t ldq, float *s, int64_t s_rs, int64_t s_gs, cudaStream_t st) {
    addnorm::Params p;
    p.x = static_cast<const __nv_bfloat16 *>(x); p.ldx = ldx;
    p.r = static_cast<const __nv_bfloat16 *>(r); p.ldr = ldr;
    p.w = static_cast<const __nv_bfloat16 *>(weight);
    p.out = static_cast<__nv_bfloat16 *>(out); p.ldo = ldo;
    p.q = static_cast<uint8_t *>(q); p.ldq = ldq;
    p.s = s; p.s_rs = s_rs; p.s_gs = s_gs;
    p.rows = rows; p.D = (int)D; p.eps = eps;
    if (kind == 0) return per_row ? addnorm::pick<0, true>(p, st) : addnorm::pick<0, false>(p, st);
    return per_row ? addnorm::pick<1, true>(p, st) : addnorm::pick<1, false>(p, st);
}

} // namespace hn
