// paged_tc.cu - the tensor-core line of the paged attention: tiles of 65 rows and more (a segment's queries over its own
// and the shared tokens, or the rows of many sequences over the shared ones). tcgen05 kind::f16 products, S / P and O in
// tensor memory; the pieces, partial results and formulas are paged.cuh's and paged_attention.cu's.
//
// One CTA per SM, 128 keys per block, two softmax groups of 128 rows each. Two row tiles of one K/V head share each K and
// V block (a tile of 256 rows), or, for tiles of at most 128 rows (`halves` 2), the groups hold the same rows and take the even
// and the odd blocks. Either way one group's exponentials run beside the other's products:
//   warps 0-7    softmax: a thread per row (its TMEM lane). Loads q, writes it to shared memory; per block reads S, keeps the
//                running maximum and sum, writes P over S (S 0-127, 128-255; O 256-383, 384-511), rescales O only when the
//                maximum grew by more than 2^8.
//   warp 8       MMA issuer: S_g(i) = Q_g K^T, O_g += P_g(i) V, in the order S0 S1 | PV0 S0' | PV1 S1' | ... S_g(i + 1) overwrites
//                P_g(i), which the product before it in the pipe has read.
//   warps 12-15  producer: gathers the pages' rows of K and V into a ring of four 32 KB slots (K, V, K, V), in the
//                128-byte-swizzled layout of the products (K-major K, MN-major V); rows past the end are zeros. bf16 rows go by cp.async;
//                int8 codes go through registers and become fp16 integers (exact), with (sk scale log2 e, log2 sv, 1 / sv)
//                of each key in a second ring of four.
// The register file is split by setmaxnreg: 2 x 128 x 184 for the softmax, the rest of 512 x 128 for the other two warpgroups.
// Every mbarrier wait is bounded; on expiry the kernel records HN_DEVERR_TIMEOUT, the roles leave their loops, copies and MMAs in
// flight are drained (bounded) and TMEM is freed.
#include <cuda_fp16.h>

#include "hn_tc.cuh"
#include "paged.cuh"

namespace hn {
namespace paged {
using namespace tc;

constexpr int BKT = 128;                    // keys per block
constexpr int HALF = 128 * 128;             // [128 rows][128 B]: one half (64 elements) of the head dim
constexpr int TILE = 2 * HALF;
constexpr int NS = 4;                       // ring slots (K and V blocks in turn)
constexpr int NSC = 4;                      // scale ring
constexpr int TC_THREADS = 512;
constexpr int OFF_Q = 0;
constexpr int OFF_KV = 2 * TILE;
constexpr int OFF_SC = OFF_KV + NS * TILE;  // per block: [64 key pairs]{a0, a1, l0, l1}, then [128] 1 / sv
constexpr int SC_BYTES = BKT * 12;
constexpr int OFF_BAR = OFF_SC + NSC * SC_BYTES;
// full[NS], empty[NS], s[2], p[2], q[2], o[2], scales[NSC], end
constexpr int NBARS = 2 * NS + 8 + NSC + 1;
constexpr int OFF_MISC = OFF_BAR + NBARS * 8;
constexpr int OFF_PRE = OFF_MISC + 16 + 32 * 4;
constexpr uint32_t TMEM_COLS = 512;
constexpr uint64_t WAIT_NS = 2000000000ull;     // 2 s
// int8: P' <= 2^7 at the running maximum, so <= 2^15 at one stale by 2^8; the partial results are brought to the
// streaming kernel's 2^14
constexpr float TC_SHIFT = 7.0f, STREAM_SHIFT = 14.0f;

__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
// 32 lanes x 32 columns into registers, not waited for
__device__ __forceinline__ void ld32_async(uint32_t taddr, uint32_t *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
// orders the registers' uses after the loads: the first call waits for all of them
__device__ __forceinline__ void ld_fence32(uint32_t *r, bool wait) {
    if (wait) asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
    asm volatile(""
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                   "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]),
                   "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]),
                   "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}
// 32 lanes x 16 columns from registers, not waited for
__device__ __forceinline__ void st16_async(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
                 "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                   "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
// D (TMEM, fp32) (+)= A (TMEM, 16-bit pairs per column, one row per lane) x B (smem), K = 16
__device__ __forceinline__ void mma_pv(uint32_t d, uint32_t a, uint64_t bd, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(bd), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void sts16(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
// 16-byte chunk c (of 16) of row r of a [128][128 elements] operand tile
__device__ __forceinline__ uint32_t chunk_at(int r, int c) { return (c >> 3) * HALF + r * 128 + (((c & 7) ^ (r & 7)) << 4); }

template <bool I8> __global__ void __launch_bounds__(TC_THREADS, 1) k_paged_tc(const Params p) {
    extern __shared__ __align__(1024) uint8_t smem[];
    constexpr int R_SOFTMAX = 184, R_MMA = I8 ? 40 : 48, R_LOAD = I8 ? 104 : 96;
    static_assert(2 * R_SOFTMAX + R_MMA + R_LOAD == 512, "the registers that the block was launched with");
    const uint32_t sb = smem_u32(smem);
    const uint32_t b_full = sb + OFF_BAR, b_empty = b_full + 8 * NS, b_s = b_empty + 8 * NS, b_p = b_s + 16, b_q = b_p + 16,
                   b_o = b_q + 16, b_sc = b_o + 16, b_end = b_sc + 8 * NSC;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + OFF_MISC);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + OFF_MISC + 4);
    int *sums = reinterpret_cast<int *>(smem + OFF_MISC + 16), *pre = reinterpret_cast<int *>(smem + OFF_PRE);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (sb & 1023) {                            // the swizzled tiles need it; shared memory starts on such a boundary
        if (threadIdx.x == 0) atomicOr(p.err, HN_DEVERR_TIMEOUT);
        return;
    }

    if (threadIdx.x == 0) {
        for (int i = 0; i < NS; ++i) { mbar_init(b_full + 8 * i, 128); mbar_init(b_empty + 8 * i, 1); }
        for (int i = 0; i < 2; ++i) {
            mbar_init(b_s + 8 * i, 1);
            mbar_init(b_p + 8 * i, 4);
            mbar_init(b_q + 8 * i, 128);
            mbar_init(b_o + 8 * i, 1);
        }
        for (int i = 0; i < NSC; ++i) mbar_init(b_sc + 8 * i, 128);
        mbar_init(b_end, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async();
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(TMEM_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    prefix_blocks(p, pre, sums, TC_THREADS);
    if (blockIdx.x == 0)
        for (int b = threadIdx.x; b <= p.B; b += TC_THREADS) p.sched[b] = pre[b];
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const bool split = p.halves == 2;           // the groups share the rows and take every other block
    const int rows_all = p.nbA ? p.B * p.Lq * p.G : p.Lq * p.G;
    Walker walk(p, pre, blockIdx.x);
    Piece w;
    bool ok = true;

    if (warp < 8) {
        // ------------------------------------------------------------------ softmax and the results
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R_SOFTMAX));
        const int g = warp >> 2, wq = warp & 3, rr = 32 * wq + lane;
        const uint32_t tl = tmem + ((uint32_t)(32 * wq) << 16), ts = tl + 128 * g, to = tl + 256 + 128 * g;
        int n_s = 0, n_piece = 0, n_tile = 0;   // phases: blocks this group has seen, pieces, blocks of the CTA
        while (ok && walk.next(p, pre, blockIdx.x, w)) {
            const int r = w.row0 + (split ? 0 : 128 * g) + rr;
            const bool valid = r < rows_all;
            int b = 0, l = 0, gm = 0, lim = w.kend;       // a row past the tile's end: computed and dropped
            if (valid) {
                split_row(p, w, r, b, l, gm);
                lim = row_limit(p, seq_length(p, b), l);
                lim = lim > w.kend ? w.kend : lim;
            }
            // --- q to shared memory (a row past the tile's end: zeros)
            float rs = I8 ? 1.0f : p.sl2;       // int8: the keys' factors carry scale * log2 e
            {
                const __nv_bfloat16 *qp = p.q + b * p.q_bs + l * p.q_ls + (int64_t)(w.h * p.G + gm) * p.q_hs;
                uint32_t x[64];
#pragma unroll
                for (int c = 0; c < 16; ++c) {
                    uint4 y = make_uint4(0, 0, 0, 0);
                    if (valid) y = *reinterpret_cast<const uint4 *>(qp + 8 * c);
                    x[4 * c] = y.x ^ p.flip; x[4 * c + 1] = y.y ^ p.flip;
                    x[4 * c + 2] = y.z ^ p.flip; x[4 * c + 3] = y.w ^ p.flip;
                }
                if (I8) {
                    float top = 0.0f;
#pragma unroll
                    for (int i = 0; i < 64; ++i) top = fmaxf(top, fmaxf(fabsf(bf16_lo(x[i])), fabsf(bf16_hi(x[i]))));
                    const int e = row_exponent(top);
                    const float down = pow2i(-e);
                    rs = pow2i(e);
#pragma unroll
                    for (int i = 0; i < 64; ++i) x[i] = pack_f16_rn(bf16_lo(x[i]) * down, bf16_hi(x[i]) * down);
                }
#pragma unroll
                for (int c = 0; c < 16; ++c)
                    sts16(sb + OFF_Q + g * TILE + chunk_at(rr, c), x[4 * c], x[4 * c + 1], x[4 * c + 2], x[4 * c + 3]);
            }
            fence_async();
            mbar_arrive(b_q + 8 * g);

            float m = -INFINITY, sum = 0.0f;
            const int count = split ? (w.nblk + 1 - g) >> 1 : w.nblk;
            for (int i = 0; i < count; ++i) {
                const int j = split ? 2 * i + g : i;
                ok = warp_wait(lane, b_s + 8 * g, n_s & 1, abort_flag, WAIT_NS, p.err);
                ++n_s;
                if (!ok) break;
                tc_fence_after();
                uint32_t x[128];
#pragma unroll
                for (int c = 0; c < 4; ++c) ld32_async(ts + 32 * c, x + 32 * c);
                const float4 *al = nullptr, *iv = nullptr;
                if (I8) {
                    const int t = n_tile + j;
                    ok = warp_wait(lane, b_sc + 8 * (t % NSC), (t / NSC) & 1, abort_flag, WAIT_NS, p.err);
                    if (!ok) break;
                    __syncwarp();
                    al = reinterpret_cast<const float4 *>(smem + OFF_SC + (t % NSC) * SC_BYTES);
                    iv = al + 64;
                }
                ld_fence32(x, true);
                ld_fence32(x + 32, false);
                ld_fence32(x + 64, false);
                ld_fence32(x + 96, false);
                const uint64_t rs2 = x2_splat(rs);
                if (I8) {           // base-2 logits + log2 sv
#pragma unroll
                    for (int c = 0; c < 64; ++c) {
                        const float4 f = al[c];
                        float y0, y1;
                        x2_split(x2_fma(x2_mul(x2(__uint_as_float(x[2 * c]), __uint_as_float(x[2 * c + 1])), x2(f.x, f.y)), rs2,
                                        x2(f.z, f.w)), y0, y1);
                        x[2 * c] = __float_as_uint(y0);
                        x[2 * c + 1] = __float_as_uint(y1);
                    }
                }
                const int k0 = w.kbeg + (w.blk0 + j) * BKT;
                if (__any_sync(0xffffffffu, k0 + BKT > lim)) {
                    const int seen = lim - k0;
#pragma unroll
                    for (int c = 0; c < 128; ++c)
                        if (c >= seen) x[c] = __float_as_uint(-INFINITY);
                }
                float mx[8];
#pragma unroll
                for (int c = 0; c < 8; ++c) mx[c] = max3(__uint_as_float(x[c]), __uint_as_float(x[8 + c]), __uint_as_float(x[16 + c]));
#pragma unroll
                for (int c = 24; c < 120; c += 16)
#pragma unroll
                    for (int u = 0; u < 8; ++u)
                        mx[u] = max3(mx[u], __uint_as_float(x[c + u]), __uint_as_float(x[c + 8 + u]));
#pragma unroll
                for (int u = 0; u < 8; ++u) mx[u] = fmaxf(mx[u], __uint_as_float(x[120 + u]));
                float top = max3(max3(mx[0], mx[1], mx[2]), max3(mx[3], mx[4], mx[5]), fmaxf(mx[6], mx[7]));
                if (!I8) top *= rs;
                const float mn = fmaxf(m, top);
                if (i == 0) {
                    m = mn;
                } else {
                    const bool need = mn > m + 8.0f;
                    if (__any_sync(0xffffffffu, need)) {
                        // O holds this group's products up to the block before (S's commit came after them)
                        const float alpha = need ? ex2(m - mn) : 1.0f;
                        if (need) { sum *= alpha; m = mn; }
#pragma unroll 1
                        for (int c = 0; c < HD; c += 16) {
                            uint32_t o[16];
                            asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 "
                                         "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
                                         "tcgen05.wait::ld.sync.aligned;"
                                         : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3]), "=r"(o[4]), "=r"(o[5]),
                                           "=r"(o[6]), "=r"(o[7]), "=r"(o[8]), "=r"(o[9]), "=r"(o[10]), "=r"(o[11]),
                                           "=r"(o[12]), "=r"(o[13]), "=r"(o[14]), "=r"(o[15])
                                         : "r"(to + c)
                                         : "memory");
#pragma unroll
                            for (int u = 0; u < 16; ++u) o[u] = __float_as_uint(__uint_as_float(o[u]) * alpha);
                            st16_async(to + c, o);
                        }
                    }
                }
                const float ref = m == -INFINITY ? 0.0f : m;
                const uint64_t nref = x2_splat(I8 ? TC_SHIFT - ref : -ref);
                uint64_t acc = 0ull;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t pk[16];
#pragma unroll
                    for (int u = 0; u < 16; ++u) {
                        const int k = 32 * c + 2 * u;
                        const uint64_t s2 = x2(__uint_as_float(x[k]), __uint_as_float(x[k + 1]));
                        float a0, a1;
                        x2_split(I8 ? x2_add(s2, nref) : x2_fma(s2, rs2, nref), a0, a1);
                        const float e0 = ex2(a0), e1 = ex2(a1);
                        if (I8) {
                            const float2 v = reinterpret_cast<const float2 *>(iv)[16 * c + u];
                            acc = x2_fma(x2(e0, e1), x2(v.x, v.y), acc);
                            pk[u] = pack_f16_rn(e0, e1);
                        } else {
                            acc = x2_add(acc, x2(e0, e1));
                            pk[u] = bf16x2_rn(e0, e1);
                        }
                    }
                    st16_async(ts + 16 * c, pk);
                }
                float a0, a1;
                x2_split(acc, a0, a1);
                sum += a0 + a1;
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(b_p + 8 * g);
            }
            if (!ok) break;
            n_tile += w.nblk;
            // --- O: to the output, or to the piece's slot
            ok = warp_wait(lane, b_o + 8 * g, n_piece & 1, abort_flag, WAIT_NS, p.err);
            ++n_piece;
            if (!ok) break;
            tc_fence_after();
            const bool ends = w.slot < 0;
            const float inv = ends ? inverse(sum) : 1.0f;
            const int head = w.h * p.G + gm;
            const int64_t at = (int64_t)(ends ? 0 : w.slot) * p.part_rows + 128 * g + rr;
            __nv_bfloat16 *op = p.out + b * p.o_bs + l * p.o_ls + head * p.o_hs;
#pragma unroll 1
            for (int c = 0; c < HD; c += 32) {
                uint32_t o[32];
                if (count > 0) {
                    tmem_ld32(to + c, o);
                } else {
#pragma unroll
                    for (int u = 0; u < 32; ++u) o[u] = 0u;
                }
                if (valid && ends) {
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        uint4 y;
                        uint32_t *z = &y.x;
#pragma unroll
                        for (int v = 0; v < 4; ++v)
                            z[v] = bf16x2_rn(__uint_as_float(o[8 * u + 2 * v]) * inv, __uint_as_float(o[8 * u + 2 * v + 1]) * inv);
                        *reinterpret_cast<uint4 *>(op + c + 8 * u) = y;
                    }
                } else if (valid) {
#pragma unroll
                    for (int u = 0; u < 8; ++u)
                        *reinterpret_cast<uint4 *>(p.part_o + at * HD + c + 4 * u) =
                            make_uint4(o[4 * u], o[4 * u + 1], o[4 * u + 2], o[4 * u + 3]);
                }
                __syncwarp();
            }
            if (valid) {
                const float M = I8 ? m + (STREAM_SHIFT - TC_SHIFT) : m;
                if (!ends) *reinterpret_cast<float2 *>(p.part_ml + 2 * at) = make_float2(M, sum);
                else if (p.lse != nullptr) p.lse[((int64_t)b * p.H + head) * p.Lq + l] = row_lse(p, M, sum);
            }
            tc_fence_before();          // O is read before the next piece's products, which wait for this group's P
        }
    } else if (warp < 12) {
        // ------------------------------------------------------------------ MMA issuer (warp 8)
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R_MMA));
        if (warp == 8) {
            // kind::f16: fp32 D (bit 4), A and B bf16 (bits 7, 10) or f16 (0), N / 8 at bit 17, M / 16 at bit 24; V is MN-major (bit 16)
            const uint32_t types = (1u << 4) | (I8 ? 0u : (1u << 7) | (1u << 10)) | ((uint32_t)(BKT >> 3) << 17) | (8u << 24);
            const uint32_t idesc_s = types, idesc_o = types | (1u << 16);
            uint32_t half0 = 0;                 // ring index of the piece's first K block
            int n_p[2] = {0, 0}, n_piece = 0;
            while (ok && walk.next(p, pre, blockIdx.x, w)) {
                const int tasks = split ? w.nblk : 2 * w.nblk;
                for (int g = 0; g < 2 && ok; ++g)
                    ok = warp_wait(lane, b_q + 8 * g, n_piece & 1, abort_flag, WAIT_NS, p.err);
                ++n_piece;
                if (!ok) break;
                auto issue_s = [&](int t) -> bool {
                    const int g = t & 1, j = split ? t : t >> 1;
                    const uint32_t h = half0 + 2 * j, slot = h % NS;
                    if (!warp_wait(lane, b_full + 8 * slot, (h / NS) & 1, abort_flag, WAIT_NS, p.err)) return false;
                    tc_fence_after();
                    if (lane == 0) {
                        const uint32_t qa = sb + OFF_Q + g * TILE, ka = sb + OFF_KV + slot * TILE;
#pragma unroll
                        for (int i = 0; i < HD / 16; ++i)
                            mma_f16(tmem + 128 * g, sdesc(qa + (i >> 2) * HALF) + 2 * (i & 3), sdesc(ka + (i >> 2) * HALF) + 2 * (i & 3),
                                    idesc_s, (uint32_t)(i > 0));
                        mma_commit(b_s + 8 * g);
                        if (split || g == 1) mma_commit(b_empty + 8 * slot);
                    }
                    __syncwarp();
                    return true;
                };
                for (int t = 0; t < 2 && t < tasks && ok; ++t) ok = issue_s(t);
                for (int t = 0; t < tasks && ok; ++t) {
                    const int g = t & 1, j = split ? t : t >> 1, i = t >> 1;
                    const uint32_t h = half0 + 2 * j + 1, slot = h % NS;
                    ok = warp_wait(lane, b_full + 8 * slot, (h / NS) & 1, abort_flag, WAIT_NS, p.err);
                    if (ok) ok = warp_wait(lane, b_p + 8 * g, n_p[g] & 1, abort_flag, WAIT_NS, p.err);
                    if (!ok) break;
                    ++n_p[g];
                    tc_fence_after();
                    if (lane == 0) {
                        const uint32_t va = sb + OFF_KV + slot * TILE;
#pragma unroll
                        for (int u = 0; u < BKT / 16; ++u)      // 16 keys: 8 columns of P, two 8-row groups of V
                            mma_pv(tmem + 256 + 128 * g, tmem + 128 * g + 8 * u, sdesc_mn(va, HALF) + (uint64_t)(2048 >> 4) * u, idesc_o,
                                   (uint32_t)(i > 0 || u > 0));
                        if (split || g == 1) mma_commit(b_empty + 8 * slot);
                        if (t + 2 >= tasks) mma_commit(b_o + 8 * g);
                    }
                    __syncwarp();
                    if (t + 2 < tasks) ok = issue_s(t + 2);
                }
                // a group without a block has its phase completed all the same
                if (ok && tasks == 1 && lane == 0) mbar_arrive(b_o + 8);
                __syncwarp();
                half0 += 2 * w.nblk;
            }
            // every MMA issued has completed before TMEM is freed
            if (lane == 0) {
                mma_commit(b_end);
                volatile int never = 0;
                mbar_wait(b_end, 0, &never, 100000000ull, p.err);
            }
            __syncwarp();
        }
    } else {
        // ------------------------------------------------------------------ producer
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R_LOAD));
        const int tid = threadIdx.x - 384;
        constexpr int ROW = I8 ? HD : 2 * HD;
        uint32_t half = 0;                      // ring index
        int n_tile = 0;
        while (ok && walk.next(p, pre, blockIdx.x, w)) {
            const int seq = p.rows[w.own_b < 0 ? 0 : w.own_b];
            const int *tab = p.table + (int64_t)((unsigned)seq < (unsigned)p.slots ? seq : 0) * p.width;
            // lane s < 8: the token index of key 16 s of block j in the pool, or -1; the 16 keys are in one page
            auto place = [&](int j) -> int64_t {
                const int kk = w.kbeg + (w.blk0 + j) * BKT + 16 * (lane & 7), pg = kk / p.page;
                const int id = kk < w.kend && pg < p.width ? tab[pg] : -1;
                return (unsigned)id < (unsigned)p.pages ? ((int64_t)id * p.Hkv + w.h) * p.page + (kk - pg * p.page) : -1;
            };
            if (!I8) {
                const int c = tid & 15, r8 = tid >> 4;
                int64_t at = place(0);
                for (int j = 0; j < w.nblk && ok; ++j) {
                    const int64_t next = j + 1 < w.nblk ? place(j + 1) : -1;
                    const int k0 = w.kbeg + (w.blk0 + j) * BKT;
#pragma unroll
                    for (int kv = 0; kv < 2; ++kv) {
                        const uint32_t slot = half % NS;
                        ok = warp_wait(lane, b_empty + 8 * slot, ((half / NS) & 1) ^ 1, abort_flag, WAIT_NS, p.err);
                        if (!ok) break;
                        const uint8_t *pool = kv ? p.v : p.k;
                        const uint32_t dst = sb + OFF_KV + slot * TILE;
#pragma unroll
                        for (int it = 0; it < 16; ++it) {
                            const int64_t base = __shfl_sync(0xffffffffu, at, it >> 1);
                            const int row = 8 * it + r8;
                            const bool here = base >= 0 && k0 + row < w.kend;
                            const uint8_t *src = here ? pool + (base + (row & 15)) * ROW + 16 * c : pool;
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                                         ::"r"(dst + chunk_at(row, c)), "l"(src), "r"(here ? 16 : 0) : "memory");
                        }
                        asm volatile("cp.async.commit_group;" ::: "memory");
                        // the block two before has landed: hand it over
                        asm volatile("cp.async.wait_group 2;" ::: "memory");
                        fence_async();
                        if (half >= 2) mbar_arrive(b_full + 8 * ((half - 2) % NS));
                        ++half;
                    }
                    at = next;
                }
            } else {
                // a quarter of a warp holds 64 B of two neighbouring rows, so that its 16-byte stores use every bank once
                const int row16 = 2 * (tid >> 4) + ((tid >> 2) & 1), c = ((tid >> 3) & 1) * 4 + (tid & 3);
                uint4 kreg[8], vreg[8];
                float sk = 0.0f, sv = 1.0f;
                auto fetch = [&](uint4 (&reg)[8], const uint8_t *pool, int64_t at, int j) {
                    const int k0 = w.kbeg + (w.blk0 + j) * BKT;
#pragma unroll
                    for (int it = 0; it < 8; ++it) {
                        const int64_t base = __shfl_sync(0xffffffffu, at, it);
                        reg[it] = make_uint4(0, 0, 0, 0);
                        if (base >= 0 && k0 + 16 * it + row16 < w.kend)
                            reg[it] = ldg_stream(pool + (base + row16) * ROW + 16 * c);
                    }
                };
                auto fetch_scales = [&](int64_t at, int j) {
                    const int64_t base = __shfl_sync(0xffffffffu, at, tid >> 4);
                    sk = 0.0f; sv = 1.0f;
                    if (base >= 0 && w.kbeg + (w.blk0 + j) * BKT + tid < w.kend) {
                        sk = p.ks[base + (tid & 15)];
                        sv = p.vs[base + (tid & 15)];
                    }
                };
                auto store = [&](const uint4 (&reg)[8], uint32_t slot) {
                    const uint32_t dst = sb + OFF_KV + slot * TILE;
#pragma unroll
                    for (int it = 0; it < 8; ++it) {
                        const int row = 16 * it + row16;
                        const uint32_t x[4] = {reg[it].x ^ 0x80808080u, reg[it].y ^ 0x80808080u, reg[it].z ^ 0x80808080u,
                                               reg[it].w ^ 0x80808080u};
                        sts16(dst + chunk_at(row, 2 * c), codes_f16<0x4140>(x[0]), codes_f16<0x4342>(x[0]),
                              codes_f16<0x4140>(x[1]), codes_f16<0x4342>(x[1]));
                        sts16(dst + chunk_at(row, 2 * c + 1), codes_f16<0x4140>(x[2]), codes_f16<0x4342>(x[2]),
                              codes_f16<0x4140>(x[3]), codes_f16<0x4342>(x[3]));
                    }
                };
                int64_t at = place(0);
                fetch(kreg, p.k, at, 0);
                fetch_scales(at, 0);
                fetch(vreg, p.v, at, 0);
                at = w.nblk > 1 ? place(1) : -1;
                for (int j = 0; j < w.nblk && ok; ++j, ++n_tile) {
                    uint32_t slot = half % NS;
                    ok = warp_wait(lane, b_empty + 8 * slot, ((half / NS) & 1) ^ 1, abort_flag, WAIT_NS, p.err);
                    if (!ok) break;
                    store(kreg, slot);
                    {
                        float *sc = reinterpret_cast<float *>(smem + OFF_SC + (n_tile % NSC) * SC_BYTES);
                        // a scale below 2^-100 (an all but zero row) counts as 2^-100: its values then are below 2^-93
                        const float s1 = sv < 0x1p-100f ? 0x1p-100f : sv;
                        sc[4 * (tid >> 1) + (tid & 1)] = sk * p.sl2;
                        sc[4 * (tid >> 1) + 2 + (tid & 1)] = lg2(s1);
                        sc[2 * BKT + tid] = __frcp_rn(s1);
                        mbar_arrive(b_sc + 8 * (n_tile % NSC));
                    }
                    fence_async();
                    mbar_arrive(b_full + 8 * slot);
                    ++half;
                    const int64_t next = j + 2 < w.nblk ? place(j + 2) : -1;
                    if (j + 1 < w.nblk) { fetch(kreg, p.k, at, j + 1); fetch_scales(at, j + 1); }
                    slot = half % NS;
                    ok = warp_wait(lane, b_empty + 8 * slot, ((half / NS) & 1) ^ 1, abort_flag, WAIT_NS, p.err);
                    if (!ok) break;
                    store(vreg, slot);
                    fence_async();
                    mbar_arrive(b_full + 8 * slot);
                    ++half;
                    if (j + 1 < w.nblk) fetch(vreg, p.v, at, j + 1);
                    at = next;
                }
            }
        }
        if (!I8) {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            fence_async();
            for (uint32_t h = half >= 2 ? half - 2 : 0; h < half && ok; ++h) mbar_arrive(b_full + 8 * (h % NS));
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    }
}

cudaError_t launch_tc(const Params &p, cudaStream_t st) {
    const bool i8 = p.ks != nullptr;
    static bool configured[HN_MAX_DEV];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= HN_MAX_DEV) return cudaErrorInvalidDevice;
    if (!configured[dev]) {
        const int most = OFF_PRE + (MAX_B + 1) * 4;
        static_assert(OFF_PRE + (MAX_B + 1) * 4 <= 232448, "shared memory budget");
        e = cudaFuncSetAttribute(k_paged_tc<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(k_paged_tc<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
        if (e != cudaSuccess) return e;
        configured[dev] = true;
    }
    const int smem = OFF_PRE + (p.B + 1) * 4;
    if (i8) k_paged_tc<true><<<p.ctas, TC_THREADS, smem, st>>>(p);
    else k_paged_tc<false><<<p.ctas, TC_THREADS, smem, st>>>(p);
    return cudaGetLastError();
}

} // namespace paged
} // namespace hn
