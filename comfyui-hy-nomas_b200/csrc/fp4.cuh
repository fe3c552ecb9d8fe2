// fp4.cuh - the 4-bit operand formats of the FP4 linears.
//
// A code is e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign), two to a byte, the even column in the low half; a row of K columns is
// padded with zero codes to Kp = K rounded up to 32, so that it is whole 16-byte units.
//   MX  one scale 2^(byte - 127) per 32 columns (byte 255: NaN)
//   NV  one e4m3 scale per 16 columns, and one fp32 scale per row
// Scale bytes lie as the tensor cores read them: tiles of 128 rows x 4 groups, 512 bytes each, [row block][group block]; in a tile
// the four groups of row r are the word at 16 (r % 32) + 4 (r / 32). A group block is 128 columns (MX) or 64 (NV).
#pragma once
#include "hn_common.cuh"

namespace hn {
namespace fp4 {

constexpr int MX = 0, NV = 1;
constexpr int TILE = 512;                                        // bytes of a scale tile
template <int KIND> constexpr int GROUP = KIND == MX ? 32 : 16;  // columns of a scale
template <int KIND> constexpr int SPAN = 4 * GROUP<KIND>;        // columns of a scale tile

// byte offset of the word of row r and group block j, `tiles` group blocks in all
__device__ __forceinline__ int64_t scale_word(int64_t r, int64_t j, int64_t tiles) {
    const int in = (int)(r & 127);
    return ((r >> 7) * tiles + j) * TILE + (in & 31) * 16 + (in >> 5) * 4;
}

// eight fp32 values -> eight codes, nearest with ties to the even code, beyond 6 to 6; v[0] in the lowest four bits
__device__ __forceinline__ uint32_t pack8_e2m1(const float (&v)[8]) {
    uint32_t r;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}

// eight codes -> four half2 (exact), column order
__device__ __forceinline__ void unpack8_e2m1(uint32_t w, uint32_t (&h)[4]) {
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "mov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(w));
}

// fp32 -> e4m3 byte, nearest even, beyond 448 to 448
__device__ __forceinline__ uint32_t e4m3_byte(float v) { return (uint32_t)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3); }

// what a scale byte stands for
template <int KIND> __device__ __forceinline__ float scale_value(uint32_t byte) {
    if (KIND == MX) {
        if (byte == 255) return __int_as_float(0x7fffffff);
        return byte ? __uint_as_float(byte << 23) : 0x1p-127f;
    }
    const __half_raw h = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3);
    return __half2float(__half(h));
}

// the outputs of a product: y = RN(sum ra[m] rb[n] + bias[n]); the row scales and the bias may be absent (null)
struct Result {
    const float *ra, *rb;
    const void *bias;
    int bias_dtype;
    void *out;
    int64_t ldo;
    int out_dtype;
};
__device__ __forceinline__ float bias_at(const Result &o, int64_t n) {
    return o.bias_dtype == 2 ? static_cast<const float *>(o.bias)[n]
         : o.bias_dtype == 0 ? __bfloat162float(static_cast<const __nv_bfloat16 *>(o.bias)[n])
                             : __half2float(static_cast<const __half *>(o.bias)[n]);
}
// sum ra rb in an order that leaves fp32 only where the result does: the largest sum, 36 448^2 K, is below 2^53, so it bears a row
// scale up to 2^60 at once, and a larger one after the column's
__device__ __forceinline__ bool is_far(float ra) { return fabsf(ra) > 0x1p60f; }
__device__ __forceinline__ float scaled(float sum, float ra, float rb) {
    const bool far = is_far(ra);
    return __fmul_rn(__fmul_rn(sum, far ? rb : ra), far ? ra : rb);
}
// fp32 result of column n; ra: the row's scale, or 1
__device__ __forceinline__ float finish(const Result &o, float sum, float ra, int64_t n) {
    if (o.ra || o.rb) sum = scaled(sum, ra, o.rb ? o.rb[n] : 1.0f);
    return o.bias ? __fadd_rn(sum, bias_at(o, n)) : sum;
}
__device__ __forceinline__ void store_result(const Result &o, int64_t at, float v) {
    if (o.out_dtype == 0) static_cast<__nv_bfloat16 *>(o.out)[at] = __float2bfloat16_rn(v);
    else if (o.out_dtype == 1) static_cast<__half *>(o.out)[at] = __float2half_rn(v);
    else static_cast<float *>(o.out)[at] = v;
}

} // namespace fp4
} // namespace hn
