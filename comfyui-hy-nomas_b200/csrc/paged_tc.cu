// paged_tc.cu - the tensor-core line of the paged attention: many rows (a segment's queries over its own and the shared
// tokens, or the rows of many sequences over the shared ones). tcgen05 kind::f16 products, S / P and O in
// tensor memory; the pieces, partial results and formulas are paged.cuh's and paged_attention.cu's.
//
// One CTA per SM, tiles of 256 rows: two softmax groups of 128 rows each share the K and V blocks of 128 keys.
// A block goes through a group in two steps of 64 keys, with S in one of two TMEM buffers: the products of step k + 1 run
// while step k is in the softmax (with one buffer of 128 keys the softmax waited for S 2250 of every 5100 clocks).
//   NW warps     softmax. q to shared memory (half a row a thread), then per step: S from TMEM in the fragment layout (a thread
//                holds a quarter of the columns of every eighth row), running maximum and sum, P over S; O is rescaled only when
//                the maximum grew by more than 2^STALE. TMEM: S / P of group g and step k at 128 g + 64 (k % 2), O at
//                256 + 128 g. int8: sixteen warps of 16 rows. A warp's chain of load, factors, maximum, exponentials and store is
//                latency, and with 32 rows its body, beside the producers', did not fit the instruction caches (2 stalls on
//                instructions an issue): 2.91 ms with eight warps, 2.45 with their rows in two turns of one body and the
//                producers' loop by a step, 2.17 with sixteen (2.21 since V's scales are in the exponent). bf16: eight of 32 rows, whose body is shorter and whose
//                handovers are what counts: causal 1.68-1.71 ms, sixteen 1.85 (2 x 4400 queries over 20240 keys, 16 heads).
//                Polynomials on the FMA pipe for 3 of 8 exponentials cost 8%.
//   2 warps      MMA issuers, one per group: O_g += P(k) V, and, when that is done, S(k + 2) = Q_g K^T over P(k). A wait on the
//                thread that issues blocks until its products have read their operands, so each group has a thread of its own:
//                the tensor pipe runs one's products while the other waits.
//   1 warp       walks the line: the CTA's pieces into a ring of four
//   1 warp       int8: looks the block's pages up, sends for their codes (to L2; from a cold L2 2.41 ms without, 2.26 with; now 2.31) and
//                gathers its keys' factors, into a second ring of four
//   4 warps      producers: the pages' rows of K and V into a ring of nine 16 KB slots (K and V of a step in turn: given
//                back a step at a time, blocks in slots of 32 KB came late by a third of a step), in the 128-byte-swizzled layout
//                of the products (K-major K, MN-major V; V rows past the end become zeros, K's are masked). bf16: TMA, one warp.
//                int8: four warps; codes go through registers, a step ahead, and become fp16 integers (exact).
//
// int8, as on the streaming line: x_j = (q . ck_j) sk_j scale log2 e 2^e + log2 sv_j (2^e: the row's power of two), m the running
// maximum of x over what the row sees, P'_j = 2^(x_j - m + 12), and the normaliser sums P'_j / sv_j: however far apart V's scales
// are, a P' is small only where p sv is. The factor warp takes the logarithm and the reciprocal, once per key.
// The register file is split by setmaxnreg: what each role needs without spills (with shared memory taking all of L1, a spilled
// register comes back from L2).
// Every mbarrier wait is bounded; on expiry the kernel records HN_DEVERR_TIMEOUT, the roles leave their loops, copies and MMAs in
// flight are drained (bounded) and TMEM is freed.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_fp16.h>
#include <string.h>

#include "hn_tc.cuh"
#include "paged.cuh"

namespace hn {
namespace paged {
using namespace tc;

constexpr int BKT = 128;                    // keys per block
constexpr int HALF = 128 * 128;             // q: [128 rows][128 B], one half (64 elements) of the head dim
constexpr int TILE = 2 * HALF;
constexpr int STEP = 64;                    // keys of a step
constexpr int KHALF = STEP * 128;           // K, V of a step: [64 rows][128 B] twice
constexpr int KTILE = 2 * KHALF;
constexpr int NS = 9;                       // ring slots (K and V of the steps in turn); int8 with 8: 2.99 ms, with 9: 2.80
constexpr int NSC = 4;                      // scale ring
// 16-row parts of a group that a softmax warp takes, and the softmax warps (of both groups); four issuers and helpers, four producers
template <bool I8> constexpr int PARTS = I8 ? 1 : 2;
template <bool I8> constexpr int SOFTMAX_WARPS = 16 / PARTS<I8>;
template <bool I8> constexpr int TC_THREADS = 32 * (SOFTMAX_WARPS<I8> + 8);
constexpr int OFF_Q = 0;
constexpr int OFF_KV = 2 * TILE;
constexpr int OFF_SC = OFF_KV + NS * KTILE;  // per block: sk scale log2 e, log2 sv, 1 / sv [128] each, in the fragments' order;
                                            // where the 8 groups of 16 keys are (32 B)
constexpr int SC_BYTES = BKT * 12 + 32;
constexpr int OFF_BAR = OFF_SC + NSC * SC_BYTES;
constexpr int NP = 4;                       // pieces
// full[NS], empty[NS], s[2][2], p[2][2], q[2], v[2][2] (of a group's steps in turn: two of them may be on their way, and a parity
// tells a phase from its neighbours only), scales full[NSC], scales empty[NSC], piece full[NP], piece empty[NP], end[2], tail
constexpr int NBARS = 2 * NS + 14 + 2 * NSC + 2 * NP + 3;
constexpr int OFF_PIECE = OFF_BAR + NBARS * 8;
constexpr int OFF_MISC = OFF_PIECE + NP * 32;
constexpr int OFF_PRE = OFF_MISC + 16 + 32 * 4;        // misc: TMEM address, abort flag, the leading sequence; 32 sums
constexpr int SMEM_MOST = 232448;
constexpr int TC_MAX_B = (SMEM_MOST - OFF_PRE) / 4 - 1;        // sequences whose prefix sums fit
constexpr uint32_t TMEM_COLS = 512;
constexpr uint64_t WAIT_NS = 2000000000ull;     // 2 s
// A row's reference m is the maximum it was set at plus AHEAD, and is moved (and O rescaled) when a logit passes it by STALE.
// int8: P' <= 2^12 at the reference, so <= 2^15 (fp16 ends at 65504); what is lost below fp16's smallest step is 2^-35 of the
// largest. AHEAD spares most of the moves that come as the maximum of more and more keys grows. Partial results are
// brought to the streaming kernel's 2^14.
constexpr float TC_SHIFT = 12.0f, STREAM_SHIFT = 14.0f;

__device__ __forceinline__ float nan_max3(float a, float b, float c) {
    float y;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
__device__ __forceinline__ float nan_max(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
// The fragment layout of 16 TMEM lanes: lane l of the warp holds row l / 4 (and, in the second pair of registers, row l / 4 + 8),
// columns 8 c + 2 (l % 4) and the next. 32 columns into registers, not waited for:
__device__ __forceinline__ void ld_frag(uint32_t taddr, uint32_t *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {"
        "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
// the registers' uses stay behind this (and a wait::ld before it)
template <int N> __device__ __forceinline__ void frag_fence(uint32_t (&r)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 8)
        asm volatile("" : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]),
                          "+r"(r[i + 6]), "+r"(r[i + 7]) :: "memory");
}
// 16-bit pairs of 32 columns (16 TMEM columns): lane l holds pair 4 c + l % 4 of rows l / 4 and l / 4 + 8
__device__ __forceinline__ void st_frag(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.16x128b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]));
}
// 32 columns of 16 lanes in the fragment layout, times f0 (rows l / 4) and f1 (rows l / 4 + 8)
__device__ __forceinline__ void scale_frag(uint32_t taddr, float f0, float f1) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {"
        "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * (i & 2 ? f1 : f0));
    asm volatile(
        "tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], {"
        "%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
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
// 16-byte chunk c (of 16) of row r of an operand tile whose halves are `half` bytes
template <int half> __device__ __forceinline__ uint32_t chunk_at(int r, int c) {
    return (c >> 3) * half + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

// box of 64 elements x rows at (0, token, half, page and head) of a bf16 pool
__device__ __forceinline__ void tma_rows(const CUtensorMap *map, uint32_t dst, uint32_t bar, int token, int half, int page) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
                 ::"r"(dst), "l"((uint64_t)map), "r"(bar), "r"(0), "r"(token), "r"(half), "r"(page) : "memory");
}

// `box`: tokens per TMA box (bf16), a divisor of the page and of 128
template <bool I8> __global__ void __launch_bounds__(TC_THREADS<I8>, 1)
    k_paged_tc(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const Params p, int box) {
    extern __shared__ __align__(1024) uint8_t smem[];
    constexpr float STALE = I8 ? 3.0f : 8.0f, AHEAD = I8 ? 2.0f : 0.0f;
    constexpr int H = PARTS<I8>, NW = SOFTMAX_WARPS<I8>;
    constexpr int R_SOFTMAX = I8 ? 88 : 192, R_MMA = I8 ? 48 : 56, R_LOAD = I8 ? 80 : 72;      // what each role needs without spills
    static_assert(NW / 4 * R_SOFTMAX + R_MMA + R_LOAD <= (I8 ? 6 * 80 : 4 * 128), "the registers that the block was launched with");
    const uint32_t sb = smem_u32(smem);
    const uint32_t b_full = sb + OFF_BAR, b_empty = b_full + 8 * NS, b_s = b_empty + 8 * NS, b_p = b_s + 32, b_q = b_p + 32,
                   b_v = b_q + 16, b_sc = b_v + 32, b_se = b_sc + 8 * NSC, b_pf = b_se + 8 * NSC, b_pe = b_pf + 8 * NP, b_end = b_pe + 8 * NP, b_tail = b_end + 16;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + OFF_MISC);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + OFF_MISC + 4);
    unsigned long long *lead = reinterpret_cast<unsigned long long *>(smem + OFF_MISC + 8);
    int *sums = reinterpret_cast<int *>(smem + OFF_MISC + 16), *pre = reinterpret_cast<int *>(smem + OFF_PRE);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (sb & 1023) {                            // the swizzled tiles need it; shared memory starts on such a boundary
        if (threadIdx.x == 0) atomicOr(p.err, HN_DEVERR_TIMEOUT);
        return;
    }

    if (threadIdx.x == 0) {
        // a block is given back by both groups' issuers
        for (int i = 0; i < NS; ++i) { mbar_init(b_full + 8 * i, I8 ? 128 : 1); mbar_init(b_empty + 8 * i, 2); }
        for (int i = 0; i < NP; ++i) { mbar_init(b_pf + 8 * i, 1); mbar_init(b_pe + 8 * i, NW + 2 + (I8 ? 5 : 1)); }   // softmax, issuers, producers
        for (int i = 0; i < 4; ++i) { mbar_init(b_s + 8 * i, 1); mbar_init(b_p + 8 * i, NW / 2); mbar_init(b_v + 8 * i, 1); }
        for (int i = 0; i < 2; ++i) mbar_init(b_q + 8 * i, 16 * NW);
        for (int i = 0; i < NSC; ++i) { mbar_init(b_sc + 8 * i, 1); mbar_init(b_se + 8 * i, NW + 4); }   // softmax, producers
        mbar_init(b_end, 1);
        mbar_init(b_end + 8, 1);
        mbar_init(b_tail, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async();
    }
    if (warp == NW) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(TMEM_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    dep_launch();
    prefix_blocks(p, pre, sums, lead, TC_THREADS<I8>);
    if (blockIdx.x == 0)
        for (int b = threadIdx.x; b <= p.B; b += TC_THREADS<I8>) p.sched[b] = pre[b];
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int rows_all = p.nbA ? p.B * p.Lq * p.G : p.Lq * p.G;
    bool ok = true;
    // the next piece of the ring, for every warp that reads pieces; nblk 0: there are no more
    const Piece *ring = reinterpret_cast<const Piece *>(smem + OFF_PIECE);
    int n_piece = 0;
    auto next_piece = [&]() -> const Piece * {
        ok = warp_wait(lane, b_pf + 8 * (n_piece % NP), (n_piece / NP) & 1, abort_flag, WAIT_NS, p.err);
        __syncwarp();
        const Piece *w = ring + n_piece % NP;
        return ok && w->nblk > 0 ? w : nullptr;
    };
    auto done_piece = [&]() {
        __syncwarp();
        if (lane == 0) mbar_arrive(b_pe + 8 * (n_piece % NP));
        ++n_piece;
    };

    if (warp < NW) {
        // ------------------------------------------------------------------ softmax and the results
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R_SOFTMAX));
        const int g = warp / (NW / 2), row0 = 32 * (warp & 3) + (H == 1 ? 16 * ((warp >> 2) & 1) : 0);       // of the group's 128 rows
        const uint32_t tl = tmem + ((uint32_t)row0 << 16), ts = tl + 128 * g, to = tl + 256 + 128 * g;
        int n_s = 0, n_tile = 0;                // steps of this group, blocks of the CTA
        while (const Piece *pc = next_piece()) {
            const Piece &w = *pc;
            int seen[2 * H];                    // keys, from the piece's first, that rows 8 u + lane / 4 see
            float m[2 * H], sum[2 * H], rsf[2 * H];
#pragma unroll
            for (int hf = 0; hf < H; ++hf) {
                // --- q to shared memory, half a row a thread (a row past the tile's end: zeros)
                const int rr = row0 + 16 * hf + (lane & 15), r = w.row0 + 128 * g + rr, c0 = 8 * (lane >> 4);
                int lim = w.kend;               // a row past the tile's end: computed and dropped
                float rs = I8 ? 1.0f : p.sl2;   // int8: the keys' factors carry scale * log2 e
                uint32_t x[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) x[i] = 0;
                if (r < rows_all) {
                    int b, l, gm;
                    split_row(p, w, r, b, l, gm);
                    const __nv_bfloat16 *qp = p.q + b * p.q_bs + l * p.q_ls + (int64_t)(w.h * p.G + gm) * p.q_hs + 8 * c0;
                    lim = row_limit(p, seq_length(p, b), l);
                    lim = lim > w.kend ? w.kend : lim;
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        const uint4 y = *reinterpret_cast<const uint4 *>(qp + 8 * c);
                        x[4 * c] = y.x ^ p.flip; x[4 * c + 1] = y.y ^ p.flip;
                        x[4 * c + 2] = y.z ^ p.flip; x[4 * c + 3] = y.w ^ p.flip;
                    }
                }
                if (I8) {
                    float top = 0.0f;
#pragma unroll
                    for (int i = 0; i < 32; ++i) top = fmaxf(top, fmaxf(fabsf(bf16_lo(x[i])), fabsf(bf16_hi(x[i]))));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                    const int e = row_exponent(top);
                    const float down = pow2i(-e);
                    rs = pow2i(e);
#pragma unroll
                    for (int i = 0; i < 32; ++i) x[i] = pack_f16_rn(bf16_lo(x[i]) * down, bf16_hi(x[i]) * down);
                }
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    sts16(sb + OFF_Q + g * TILE + chunk_at<HALF>(rr, c0 + c), x[4 * c], x[4 * c + 1], x[4 * c + 2], x[4 * c + 3]);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    seen[2 * hf + u] = __shfl_sync(0xffffffffu, lim, 8 * u + (lane >> 2)) - (w.kbeg + w.blk0 * BKT);
                    rsf[2 * hf + u] = I8 ? __shfl_sync(0xffffffffu, rs, 8 * u + (lane >> 2)) : rs;
                    m[2 * hf + u] = -INFINITY;
                    sum[2 * hf + u] = 0.0f;
                }
            }
            fence_async();
            mbar_arrive(b_q + 8 * g);
            const int nblk = w.nblk;
            for (int k = 0; k < 2 * nblk; ++k, ++n_s) {         // steps of 64 keys
                const int sub = k & 1, t = n_tile + (k >> 1);
                const uint32_t tsb = ts + 64 * sub;
                const ulonglong2 *factors = reinterpret_cast<const ulonglong2 *>(smem + OFF_SC + (t % NSC) * SC_BYTES) +
                                            16 * sub + (lane & 3);
                if (I8 && sub == 0) {
                    ok = warp_wait(lane, b_sc + 8 * (t % NSC), (t / NSC) & 1, abort_flag, WAIT_NS, p.err);
                    if (!ok) break;
                    __syncwarp();
                }
                ok = warp_wait(lane, b_s + 16 * g + 8 * sub, (n_s >> 1) & 1, abort_flag, WAIT_NS, p.err);
                if (!ok) break;
                tc_fence_after();
                uint32_t x[32 * H];             // [16-row part][8 column groups][row l / 4, l / 4 + 8][2 columns]
#pragma unroll
                for (int c = 0; c < 2 * H; ++c) ld_frag(tsb + ((uint32_t)(16 * (c >> 1)) << 16) + 32 * (c & 1), x + 16 * c);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                frag_fence(x);
                if (I8) {
#pragma unroll
                    for (int c = 0; c < 8; c += 2) {
                        const ulonglong2 kf = factors[2 * c], lv = factors[32 + 2 * c];
#pragma unroll
                        for (int v = 0; v < 4 * H; ++v) {       // 2 column groups x the rows
                            uint32_t *y = x + 32 * (v >> 2) + 4 * (c + (v & 1)) + (v & 2);
                            float y0, y1;
                            x2_split(x2_fma(x2_mul(x2(__uint_as_float(y[0]), __uint_as_float(y[1])), v & 1 ? kf.y : kf.x),
                                            x2_splat(rsf[2 * (v >> 2) + ((v >> 1) & 1)]), v & 1 ? lv.y : lv.x), y0, y1);
                            y[0] = __float_as_uint(y0);
                            y[1] = __float_as_uint(y1);
                        }
                    }
                }
                int least = seen[0];
#pragma unroll
                for (int u = 1; u < 2 * H; ++u) least = min(least, seen[u]);
                if (__any_sync(0xffffffffu, least < 64)) {
#pragma unroll
                    for (int c = 0; c < 32 * H; ++c)
                        if (8 * ((c & 31) >> 2) + 2 * (lane & 3) + (c & 1) >= seen[2 * (c >> 5) + ((c >> 1) & 1)])
                            x[c] = __float_as_uint(-INFINITY);
                }
                float mn[2 * H];
                bool need = false;
#pragma unroll
                for (int u = 0; u < 2 * H; ++u) {
                    const uint32_t *y = x + 32 * (u >> 1) + 2 * (u & 1);
                    float mx[4];
#pragma unroll
                    for (int c = 0; c < 4; ++c) mx[c] = nan_max(__uint_as_float(y[4 * c]), __uint_as_float(y[4 * c + 1]));
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        mx[c] = nan_max3(mx[c], __uint_as_float(y[16 + 4 * c]), __uint_as_float(y[16 + 4 * c + 1]));
                    mn[u] = nan_max(nan_max3(mx[0], mx[1], mx[2]), mx[3]);
                }
#pragma unroll
                for (int u = 0; u < 2 * H; ++u) mn[u] = nan_max(mn[u], __shfl_xor_sync(0xffffffffu, mn[u], 1));
#pragma unroll
                for (int u = 0; u < 2 * H; ++u) {
                    mn[u] = nan_max(mn[u], __shfl_xor_sync(0xffffffffu, mn[u], 2));
                    if (!I8) mn[u] *= rsf[u];
                    need |= !(mn[u] <= m[u] + STALE);           // or a NaN, which stays in the row
                }
                if (k == 0) {
#pragma unroll
                    for (int u = 0; u < 2 * H; ++u) m[u] = mn[u] + AHEAD;
                } else if (__any_sync(0xffffffffu, need)) {
#pragma unroll
                    for (int u = 0; u < 2 * H; ++u) {
                        const bool grow = !(mn[u] <= m[u] + STALE);
                        const float al = grow ? ex2(m[u] - (mn[u] + AHEAD)) : 1.0f;
                        m[u] = grow ? mn[u] + AHEAD : m[u];
                        mn[u] = al;
                        sum[u] *= al;
                    }
                    // the product before this step's is the last one given to the pipe
                    ok = warp_wait(lane, b_v + 16 * g + 8 * (sub ^ 1), ((n_s - 1) >> 1) & 1, abort_flag, WAIT_NS, p.err);
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < HD; c += 32) {
#pragma unroll
                        for (int hf = 0; hf < H; ++hf)
                            scale_frag(to + ((uint32_t)(16 * hf) << 16) + c, mn[2 * hf], mn[2 * hf + 1]);
                    }
                }
#pragma unroll
                for (int hf = 0; hf < H; ++hf) {
                    uint64_t nref[2], acc[2] = {0ull, 0ull};
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const float ref = m[2 * hf + u] == -INFINITY ? 0.0f : m[2 * hf + u];
                        nref[u] = x2_splat(fmaf(ref, 0.0f, I8 ? TC_SHIFT - ref : -ref));        // an infinite maximum: NaN
                    }
#pragma unroll
                    for (int c = 0; c < 8; c += 4) {                // 4 column groups: a store of 8 registers
                        uint64_t v[4];
                        if (I8) {
                            const ulonglong2 f0 = factors[64 + 2 * c], f1 = factors[64 + 2 * c + 4];
                            v[0] = f0.x; v[1] = f0.y; v[2] = f1.x; v[3] = f1.y;
                        }
                        uint32_t pk[8];
#pragma unroll
                        for (int q = 0; q < 8; ++q) {               // column group c + q / 2, row q % 2
                            const int u = q & 1;
                            const uint32_t *y = x + 32 * hf + 4 * c + 2 * q;
                            const uint64_t z = x2(__uint_as_float(y[0]), __uint_as_float(y[1]));
                            const uint64_t a = I8 ? x2_add(z, nref[u]) : x2_fma(z, x2_splat(rsf[2 * hf + u]), nref[u]);
                            float a0, a1;
                            x2_split(a, a0, a1);
                            const float e0 = ex2(a0), e1 = ex2(a1);
                            acc[u] = I8 ? x2_fma(x2(e0, e1), v[q >> 1], acc[u]) : x2_add(acc[u], x2(e0, e1));
                            pk[q] = I8 ? pack_f16_rn(e0, e1) : bf16x2_rn(e0, e1);
                        }
                        st_frag(tsb + ((uint32_t)(16 * hf) << 16) + 4 * c, pk);
                    }
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        float a0, a1;
                        x2_split(acc[u], a0, a1);
                        sum[2 * hf + u] += a0 + a1;
                    }
                }
#pragma unroll
                for (int u = 0; u < 2 * H; ++u) seen[u] -= 64;
                if (!ok) break;
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(b_p + 16 * g + 8 * sub);
                    if (I8 && sub == 1) mbar_arrive(b_se + 8 * (t % NSC));
                }
            }
            if (!ok) break;
            n_tile += nblk;
            // --- O: to the output, or to the piece's slot
            ok = warp_wait(lane, b_v + 16 * g + 8, ((n_s - 1) >> 1) & 1, abort_flag, WAIT_NS, p.err);
            if (!ok) break;
            tc_fence_after();
            const bool ends = w.slot < 0;
#pragma unroll
            for (int hf = 0; hf < H; ++hf) {
                float inv[2];
                bool valid[2];
                __nv_bfloat16 *op[2];
                float *part[2];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    sum[2 * hf + u] += __shfl_xor_sync(0xffffffffu, sum[2 * hf + u], 1);
                    sum[2 * hf + u] += __shfl_xor_sync(0xffffffffu, sum[2 * hf + u], 2);
                    const float ref = I8 ? m[2 * hf + u] + (STREAM_SHIFT - TC_SHIFT) : m[2 * hf + u];
                    const int rr = row0 + 16 * hf + 8 * u + (lane >> 2), r = w.row0 + 128 * g + rr;
                    valid[u] = r < rows_all;
                    int b = 0, l = 0, gm = 0;
                    if (valid[u]) split_row(p, w, r, b, l, gm);
                    const int head = w.h * p.G + gm;
                    const int64_t at = (int64_t)(ends ? 0 : w.slot) * p.part_rows + 128 * g + rr;
                    inv[u] = inverse(sum[2 * hf + u]);
                    op[u] = p.out + b * p.o_bs + l * p.o_ls + head * p.o_hs + 2 * (lane & 3);
                    part[u] = p.part_o + at * HD + 2 * (lane & 3);
                    if (valid[u] && (lane & 3) == 0) {
                        if (!ends) *reinterpret_cast<float2 *>(p.part_ml + 2 * at) = make_float2(ref, sum[2 * hf + u]);
                        else if (p.lse != nullptr) p.lse[((int64_t)b * p.H + head) * p.Lq + l] = row_lse(p, ref, sum[2 * hf + u]);
                    }
                }
#pragma unroll 1
                for (int c = 0; c < HD; c += 32) {
                    uint32_t o[16];                 // [4 column groups][2 rows][2 columns]
                    ld_frag(to + ((uint32_t)(16 * hf) << 16) + c, o);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    frag_fence(o);
#pragma unroll
                    for (int v = 0; v < 8; ++v) {
                        const int u = v & 1, at = c + 8 * (v >> 1);
                        if (!valid[u]) continue;
                        const float a0 = __uint_as_float(o[2 * v]), a1 = __uint_as_float(o[2 * v + 1]);
                        if (ends) *reinterpret_cast<uint32_t *>(op[u] + at) = bf16x2_rn(a0 * inv[u], a1 * inv[u]);
                        else *reinterpret_cast<float2 *>(part[u] + at) = make_float2(a0, a1);
                    }
                    __syncwarp();
                }
            }
            tc_fence_before();          // O is read before the next piece's products, which wait for this group's P
            done_piece();
        }
    } else if (warp < NW + 4) {
        // ------------------------------------------------------------------ MMA issuers, walker
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R_MMA));
        if (warp < NW + 2) {
            // kind::f16: fp32 D (bit 4), A and B bf16 (bits 7, 10) or f16 (0), N / 8 at bit 17, M / 16 at bit 24; V is MN-major (bit 16)
            constexpr uint32_t types = (1u << 4) | (I8 ? 0u : (1u << 7) | (1u << 10)) | (8u << 24);
            constexpr uint32_t idesc_s = types | (8u << 17), idesc_o = types | ((uint32_t)(HD >> 3) << 17) | (1u << 16);
            const int g = warp - NW;
            const uint32_t ds = tmem + 128 * g, dout = tmem + 256 + 128 * g;
            uint32_t h = 0;                         // ring index of the next step's K; V follows it
            uint32_t n_p = 0;
            while (const Piece *pc = next_piece()) {
                const int nblk = pc->nblk;
                ok = warp_wait(lane, b_q + 8 * g, n_piece & 1, abort_flag, WAIT_NS, p.err);
                auto wait_full = [&](uint32_t x) {
                    return warp_wait(lane, b_full + 8 * (x % NS), (x / NS) & 1, abort_flag, WAIT_NS, p.err);
                };
                // the step whose K is at ring index x
                auto issue_s = [&](uint32_t x, uint32_t sub) {
                    const uint64_t qd = sdesc(sb + OFF_Q + g * TILE), kd = sdesc(sb + OFF_KV + (x % NS) * KTILE);
#pragma unroll
                    for (int i = 0; i < HD / 16; ++i)
                        mma_f16(ds + 64 * sub, qd + (HALF >> 4) * (i >> 2) + 2 * (i & 3), kd + (KHALF >> 4) * (i >> 2) + 2 * (i & 3),
                                idesc_s, (uint32_t)(i > 0));
                    mma_commit(b_s + 16 * g + 8 * sub);
                    mma_commit(b_empty + 8 * (x % NS));
                };
                for (uint32_t k = 0; k < 2 && ok; ++k) {
                    ok = wait_full(h + 2 * k);
                    tc_fence_after();
                    if (ok && lane == 0) issue_s(h + 2 * k, k);
                    __syncwarp();
                }
                for (int k = 0; k < 2 * nblk && ok; ++k, ++n_p, h += 2) {
                    const uint32_t sub = k & 1;
                    ok = wait_full(h + 1);
                    if (ok) ok = warp_wait(lane, b_p + 16 * g + 8 * sub, (n_p >> 1) & 1, abort_flag, WAIT_NS, p.err);
                    if (!ok) break;
                    tc_fence_after();
                    if (lane == 0) {
                        const uint64_t vd = sdesc_mn(sb + OFF_KV + ((h + 1) % NS) * KTILE, KHALF);
#pragma unroll
                        for (int u = 0; u < STEP / 16; ++u)     // 16 keys: 8 columns of P, two 8-row groups of V
                            mma_pv(dout, ds + 64 * sub + 8 * u, vd + (uint64_t)(2048 >> 4) * u, idesc_o, (uint32_t)(k > 0 || u > 0));
                        mma_commit(b_v + 16 * g + 8 * sub);
                        mma_commit(b_empty + 8 * ((h + 1) % NS));
                    }
                    __syncwarp();
                    if (k + 2 < 2 * nblk) {
                        // S(k + 2) goes over P(k): products on different accumulators are not ordered, so P V has to be done
                        // (it is, long before the softmax of step k + 1 asks for S(k + 2))
                        ok = wait_full(h + 4);
                        if (ok) ok = warp_wait(lane, b_v + 16 * g + 8 * sub, (n_p >> 1) & 1, abort_flag, WAIT_NS, p.err);
                        tc_fence_after();
                        if (ok && lane == 0) issue_s(h + 4, sub);
                        __syncwarp();
                    }
                }
                if (!ok) break;
                done_piece();
            }
            // every MMA issued has completed before TMEM is freed
            if (lane == 0) {
                mma_commit(b_end + 8 * g);
                volatile int never = 0;
                mbar_wait(b_end + 8 * g, 0, &never, 100000000ull, p.err);
            }
            __syncwarp();
        } else if (warp == NW + 2 && lane == 0) {
            Walker walk(p, pre, (int)*lead, blockIdx.x);
            Piece w;
            for (bool more = true; more; ++n_piece) {
                if (!mbar_wait(b_pe + 8 * (n_piece % NP), ((n_piece / NP) & 1) ^ 1, abort_flag, WAIT_NS, p.err)) break;
                more = walk.next(p, pre, blockIdx.x, w);
                if (!more) w.nblk = 0;
                const_cast<Piece *>(ring)[n_piece % NP] = w;
                mbar_arrive(b_pf + 8 * (n_piece % NP));
            }
        } else if (I8 && warp == NW + 3) {
            int n_tile = 0;
            while (const Piece *pc = next_piece()) {
                const int own_b = pc->own_b, head = pc->h, kend = pc->kend, nblk = pc->nblk, key0 = pc->kbeg + pc->blk0 * BKT;
                const int seq = p.rows[own_b < 0 ? (int)*lead : own_b];
                const int *tab = p.table + (int64_t)((unsigned)seq < (unsigned)p.slots ? seq : 0) * p.width;
                auto page_of = [&](int j, int &off) -> int {        // lane s < 8 (and its copies): the page of key 16 s of block j
                    const int kk = key0 + j * BKT + 16 * (lane & 7), pg = kk / p.page;
                    off = kk - pg * p.page;
                    return j < nblk && kk < kend && pg < p.width ? tab[pg] : -1;
                };
                // in flight: the pages of block j + 2 and the factors of block j + 1, while block j is written
                int off, id = page_of(0, off), at, at_next;
                float sk[4], sv[4], sk_next[4], sv_next[4];
                auto gather = [&](int j, int &where, float (&k)[4], float (&v)[4]) {
                    // where key 16 s is in the pool, in units of 16 tokens (pages are multiples of 16), -1: not there
                    where = (unsigned)id < (unsigned)p.pages ? (id * p.Hkv + head) * (p.page >> 4) + (off >> 4) : -1;
                    int x[4];                                       // key 32 u + lane; the shuffles before any load: one behind
#pragma unroll                                                              // a load waits some 290 clocks (measured)
                    for (int u = 0; u < 4; ++u) x[u] = __shfl_sync(0xffffffffu, where, 2 * u + (lane >> 4));
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        k[u] = v[u] = 0.0f;
                        if (x[u] >= 0 && 32 * u + lane < kend - (key0 + j * BKT)) {
                            k[u] = p.ks[(int64_t)x[u] * 16 + (lane & 15)];
                            v[u] = p.vs[(int64_t)x[u] * 16 + (lane & 15)];
                        }
                    }
                    // the block's codes on their way to L2: the producers' loads are a step ahead, less than a trip to HBM takes
                    if (lane < 16 && where >= 0)
                        asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"((lane < 8 ? p.k : p.v) + (int64_t)where * (16 * HD)),
                                     "r"(16 * HD)
                                     : "memory");
                    id = page_of(j + 1, off);
                };
                gather(0, at_next, sk_next, sv_next);
                for (int j = 0; j < nblk && ok; ++j, ++n_tile) {
                    at = at_next;
#pragma unroll
                    for (int u = 0; u < 4; ++u) { sk[u] = sk_next[u]; sv[u] = sv_next[u]; }
                    if (j + 1 < nblk) gather(j + 1, at_next, sk_next, sv_next);
                    ok = warp_wait(lane, b_se + 8 * (n_tile % NSC), ((n_tile / NSC) & 1) ^ 1, abort_flag, WAIT_NS, p.err);
                    if (!ok) break;
                    float *sc = reinterpret_cast<float *>(smem + OFF_SC + (n_tile % NSC) * SC_BYTES);
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        // key 8 c + 2 q + e goes to the quad's lane q, place 2 c + e of 32; four places of the four lanes in turn, so
                        // that the lanes' 16-byte loads meet different banks
                        const int key = 32 * u + lane, place = 2 * (key >> 3) + (key & 1);
                        const int to = 16 * (place >> 2) + 4 * ((key >> 1) & 3) + (place & 3);
                        sc[to] = sk[u] * p.sl2;
                        // below 2^-100 as on the other line; the reciprocal of a NaN stays a number, for the rows that do not see it
                        sc[BKT + to] = lg2(sv[u] < 0x1p-100f ? 0x1p-100f : sv[u]);
                        sc[2 * BKT + to] = __frcp_rn(fmaxf(sv[u], 0x1p-100f));
                    }
                    if (lane < 8) reinterpret_cast<int *>(sc)[3 * BKT + lane] = at;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(b_sc + 8 * (n_tile % NSC));
                }
                done_piece();
            }
        }
    } else {
        // ------------------------------------------------------------------ producers
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R_LOAD));
        const int tid = threadIdx.x - 32 * (NW + 4);
        uint32_t half = 0;                      // ring index
        uint32_t tails = 0;
        int n_tile = 0;
        while (I8 || warp == NW + 4) {
            const Piece *pc = next_piece();
            if (pc == nullptr) break;
            const int kend = pc->kend, nblk = pc->nblk, key0 = pc->kbeg + pc->blk0 * BKT;
            if (!I8) {
                const int own_b = pc->own_b, head = pc->h, seq = p.rows[own_b < 0 ? (int)*lead : own_b];
                const int *tab = p.table + (int64_t)((unsigned)seq < (unsigned)p.slots ? seq : 0) * p.width;
                const int groups = STEP / box;                  // a lane each
                for (int k = 0; k < 2 * nblk && ok; ++k) {
                    const int k0 = key0 + k * STEP, kk = k0 + box * lane, pg = kk / p.page;
                    const int id = lane < groups && kk < kend && pg < p.width ? tab[pg] : -1;
                    const bool here = (unsigned)id < (unsigned)p.pages;
                    const uint32_t bytes = 256u * box * __popc(__ballot_sync(0xffffffffu, here));
                    // groups of the step before the end whose page id is none: zeros, as on the streaming line
                    const uint32_t gone = __ballot_sync(0xffffffffu, lane < groups && kk < kend && !here);
                    const int left = max(kend - k0, 0);         // rows of the step that are there
#pragma unroll 1
                    for (int kv = 0; kv < 2; ++kv, ++half) {
                        const uint32_t slot = half % NS;
                        ok = warp_wait(lane, b_empty + 8 * slot, ((half / NS) & 1) ^ 1, abort_flag, WAIT_NS, p.err);
                        if (!ok) break;
                        const bool tail = (kv == 1 && left < STEP) || gone;
                        const uint32_t bar = tail ? b_tail : b_full + 8 * slot, dst = sb + OFF_KV + slot * KTILE;
                        if (lane == 0) mbar_arrive_tx(bar, bytes);
                        __syncwarp();
                        if (here)
                            for (int u = 0; u < 2; ++u)
                                tma_rows(kv ? &tm_v : &tm_k, dst + u * KHALF + lane * box * 128, bar, kk - pg * p.page, u,
                                         id * p.Hkv + head);
                        __syncwarp();
                        if (tail) {                             // rows past the end: zeros, whatever the page holds there
                            ok = warp_wait(lane, b_tail, tails & 1, abort_flag, WAIT_NS, p.err);
                            ++tails;
                            if (!ok) break;
                            for (int r = gone ? 0 : left; r < STEP; ++r)
                                if (lane < 16 && ((kv == 1 && r >= left) || (gone >> (r / box) & 1)))
                                    sts16(dst + chunk_at<KHALF>(r, lane), 0, 0, 0, 0);
                            fence_async();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(b_full + 8 * slot);
                        }
                    }
                }
            } else {
                // a quarter of a warp holds 64 B of two neighbouring rows, so that its 16-byte stores use every bank once
                const int row16 = 2 * (tid >> 4) + ((tid >> 2) & 1), c = ((tid >> 3) & 1) * 4 + (tid & 3), mine = row16 * HD + 16 * c;
                // a step of K or V per thread: 4 chunks; the registers hold the step ahead
                uint4 kreg[4], vreg[4];
                auto fetch = [&](uint4 (&reg)[4], const uint8_t *pool, int k, int t) {
                    const int left = kend - (key0 + k * STEP) - row16;
                    const int4 a = reinterpret_cast<const int4 *>(smem + OFF_SC + (t % NSC) * SC_BYTES + 12 * BKT)[k & 1];
                    const int at[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
                    for (int it = 0; it < 4; ++it) {
                        reg[it] = make_uint4(0, 0, 0, 0);
                        if (at[it] >= 0 && 16 * it < left) reg[it] = ldg_stream(pool + (int64_t)at[it] * (16 * HD) + mine);
                    }
                };
                auto wait_index = [&](int t) {
                    const bool r = warp_wait(lane, b_sc + 8 * (t % NSC), (t / NSC) & 1, abort_flag, WAIT_NS, p.err);
                    __syncwarp();
                    return r;
                };
                auto hand_over = [&](const uint4 (&reg)[4]) {
                    const uint32_t slot = half % NS, dst = sb + OFF_KV + slot * KTILE;
                    if (!warp_wait(lane, b_empty + 8 * slot, ((half / NS) & 1) ^ 1, abort_flag, WAIT_NS, p.err)) return false;
#pragma unroll
                    for (int it = 0; it < 4; ++it) {
                        const int row = 16 * it + row16;
                        const uint32_t x[4] = {reg[it].x ^ 0x80808080u, reg[it].y ^ 0x80808080u, reg[it].z ^ 0x80808080u,
                                               reg[it].w ^ 0x80808080u};
                        sts16(dst + chunk_at<KHALF>(row, 2 * c), codes_f16<0x4140>(x[0]), codes_f16<0x4342>(x[0]),
                              codes_f16<0x4140>(x[1]), codes_f16<0x4342>(x[1]));
                        sts16(dst + chunk_at<KHALF>(row, 2 * c + 1), codes_f16<0x4140>(x[2]), codes_f16<0x4342>(x[2]),
                              codes_f16<0x4140>(x[3]), codes_f16<0x4342>(x[3]));
                    }
                    fence_async();
                    mbar_arrive(b_full + 8 * slot);
                    ++half;
                    return true;
                };
                ok = wait_index(n_tile);
                if (ok) {
                    fetch(kreg, p.k, 0, n_tile);
                    fetch(vreg, p.v, 0, n_tile);
                }
#pragma unroll 1
                for (int k = 0; k < 2 * nblk && ok; ++k) {
                    const bool more = k + 1 < 2 * nblk;
                    if (k & 1) {                                // the block's index has been read
                        __syncwarp();
                        if (lane == 0) mbar_arrive(b_se + 8 * (n_tile % NSC));
                        ++n_tile;
                        if (more) ok = wait_index(n_tile);
                    }
                    if (ok) ok = hand_over(kreg);
                    if (ok && more) fetch(kreg, p.k, k + 1, n_tile);
                    if (ok) ok = hand_over(vreg);
                    if (ok && more) fetch(vreg, p.v, k + 1, n_tile);
                }
            }
            if (ok) done_piece();
        }
        // every copy issued has landed before the CTA may exit (immediate on the normal path)
        if (!I8 && warp == NW + 4 && lane == 0) {
            volatile int never = 0;
            for (uint32_t h = half >= NS ? half - NS : 0; h < half; ++h)
                mbar_wait(b_full + 8 * (h % NS), (h / NS) & 1, &never, 100000000ull, p.err);
            if (!ok && tails) mbar_wait(b_tail, (tails - 1) & 1, &never, 100000000ull, p.err);
        }
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == NW) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    }
}

// 4-D map {64 elements, tokens of a page, 2 halves of the head dim, pages x heads} over one layer's bf16 pool
static bool make_map(CUtensorMap *map, const void *pool, const Params &p, int box) {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    if (fn == nullptr) {
        void *ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &ptr, 12000, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            return false;
        fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
    }
    cuuint64_t dims[4] = {64, (cuuint64_t)p.page, 2, (cuuint64_t)p.pages * p.Hkv};
    cuuint64_t strides[3] = {2 * HD, HD, (cuuint64_t)p.page * 2 * HD};
    cuuint32_t boxes[4] = {64, (cuuint32_t)box, 1, 1}, estr[4] = {1, 1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void *>(pool), dims, strides, boxes, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int tc_most_sequences() { return TC_MAX_B; }

cudaError_t launch_tc(const Params &p, cudaStream_t st) {
    const bool i8 = p.ks != nullptr;
    static bool configured[HN_MAX_DEV];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= HN_MAX_DEV) return cudaErrorInvalidDevice;
    if (!configured[dev]) {
        const int most = OFF_PRE + (TC_MAX_B + 1) * 4;
        static_assert(TC_MAX_B >= 1024, "shared memory budget");
        e = cudaFuncSetAttribute(k_paged_tc<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(k_paged_tc<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
        if (e != cudaSuccess) return e;
        configured[dev] = true;
    }
    const int smem = OFF_PRE + (p.B + 1) * 4;
    int box = STEP;                             // the largest power of two up to 64 that divides the page
    while (p.page % box) box >>= 1;
    CUtensorMap tk, tv;
    memset(&tk, 0, sizeof(tk));
    memset(&tv, 0, sizeof(tv));
    if (!i8 && !(make_map(&tk, p.k, p, box) && make_map(&tv, p.v, p, box))) return cudaErrorInvalidValue;
    if (i8) k_paged_tc<true><<<p.ctas, TC_THREADS<true>, smem, st>>>(tk, tv, p, box);
    else k_paged_tc<false><<<p.ctas, TC_THREADS<false>, smem, st>>>(tk, tv, p, box);
    return cudaGetLastError();
}

} // namespace paged
} // namespace hn
