// fp4_gemm.cu - the product of two operands of 4-bit codes with block scales, on the sm_100a tensor cores.
//
//   y[m, n] = ra[m] rb[n] sum_g sa[m, g] sb[n, g] sum_{k in g} a[m, k] b[n, k]  (+ bias[n])
//
// tcgen05.mma.kind::mxf4 (scales 2^e per 32) and kind::mxf4nvf4 (e4m3 per 16) multiply the block scales in, so the accumulator
// in tensor memory is the whole sum in fp32; the row scales, the bias and the one rounding are the epilogue's.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <type_traits>

#include "fp4.cuh"
#include "fp4_handoff.h"
#include "hn_kernels.h"
#include "hn_tc.cuh"

namespace hn {
namespace fp4g {

using namespace fp4;
using namespace tc;

constexpr uint64_t WAIT_NS = 2000000000ull;     // 2 s
constexpr int KB = 256;                         // columns of a stage: 128 bytes of codes a row

// Some rows: tiles of 128 x 128 outputs. A cluster of S CTAs shares one: each takes a part of K, leaves its fp32 sums in its shared
// memory, and CTA r of the cluster adds those of its share of the rows, in the CTAs' order, and writes them: no workspace, one
// launch, the same bits every time. Bound by latency: a stage's round trip is 1.8 us, so that a lone CTA has six of them (3 x 36 KB:
// 0.6 us a step of 256 columns), and what does not depend on K, launch to store, is 6 us. Measured (us): 48 x 8192 x 4096 MX 9.9,
// 777 x 5001 x 2080 NV fp32 out 17; the sums' reduction is 1 us of the former (its loads from the other CTAs go out together). Long K:
// 0.32 us a step of 36 KB, some 60 bytes a clock and SM, the most seen here. 48 x 8192 x 4096 from HBM (24 sets of operands in turn):
// 11.1 (NV 12.4, from L2 10.8). 128 x 256 outputs a CTA, one an SM, take a quarter less from L2, and the
// issuer's 12 copies of scales a step eat that up (2048 x 2048 x 4096 19.6 -> 21.7).
template <int KIND, int STAGES_> struct Cfg {
    static constexpr int BM = 128, BN = 128, STAGES = STAGES_;
    static constexpr int CTAS = STAGES > 3 ? 1 : 2;             // an SM
    static constexpr int TILES = KB / SPAN<KIND>;               // scale tiles of an operand in a stage
    static constexpr int OP = 128 * 128, SF = TILES * TILE;     // bytes of a stage: codes and scales of an operand
    static constexpr int STAGE = 2 * OP + 2 * SF;
    static constexpr int OFF_BAR = STAGES * STAGE;
    static constexpr int PITCH = BN + 4;                        // floats a row of the fp32 tile (in the stages' place)
    static_assert(BM * PITCH * 4 <= OFF_BAR, "the fp32 tile lies over the stages");
    static constexpr int OFF_MISC = OFF_BAR + 8 * (2 * STAGES + 1);
    static constexpr int SMEM = OFF_MISC + 16 + 1024;           // + alignment slack
    static constexpr int ACC = 0, SFC = BN;                     // tensor memory columns: sums, then 8 x TILES a stage
    static constexpr int COLS = CTAS == 1 ? 512 : 256;
    static constexpr int THREADS = 192;                         // producer, issuer, four warps that empty tensor memory
    static_assert(SFC + STAGES * 8 * TILES <= COLS, "tensor memory");
    static_assert(CTAS * (SMEM + 1024) <= 228 * 1024, "shared memory");
};

struct Params {
    Result o;
    int vec;                    // four outputs at a time
    int M, N, Kp;
    int m_tiles, parts;
    int *err;
};

// scale tiles: 32 rows of 16 bytes each, no swizzle, 128 bytes between groups of 8 rows
__device__ __forceinline__ uint64_t sdesc_scale(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)(128 >> 4) << 32) | ((uint64_t)1 << 46);
}
__device__ __forceinline__ void copy_scale(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
template <int KIND>
__device__ __forceinline__ void mma(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t acc) {
    if (KIND == NV)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
                     ::"r"(d), "l"(ad), "l"(bd), "r"(idesc), "r"(acc), "r"(sa), "r"(sb) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
                     ::"r"(d), "l"(ad), "l"(bd), "r"(idesc), "r"(acc), "r"(sa), "r"(sb) : "memory");
}
// e2m1 x e2m1 (type 1 of both); bit 23: scales 2^e; the scale's place in its word (MX: 0 or 2) goes into bits 4 and 29
template <int KIND, int M, int N> constexpr uint32_t instruction() {
    return (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | (KIND == MX ? 1u << 23 : 0u) | ((uint32_t)(M >> 4) << 24);
}

__device__ __forceinline__ void tma_load_2d(const CUtensorMap *map, uint32_t dst, uint32_t bar, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 ::"r"(dst), "l"((uint64_t)map), "r"(bar), "r"(x), "r"(y)
                 : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr, uint32_t rank) {
    float4 v;
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ float ld_cluster1(uint32_t addr, uint32_t rank) {
    float v;
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}

// Rows [r0, r1) of a tile's sums: P CTAs' partial sums added in their order, scales, bias, rounding. A warp takes every WARPS-th
// row, U of them at a time so that their loads overlap; a lane has the same four columns throughout (VEC: neighbours, one store).
// FAR: rows whose scales need an order of their own (`scaled`) may be among them
template <int P, bool VEC, bool FAR, int WARPS>
__device__ __forceinline__ void write_rows(const Params &p, const float *tile, int pitch, int m0, int n0, int r0, int r1) {
    constexpr int U = P == 8 ? 2 : 4;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float cs[4], cb[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int n = n0 + (VEC ? 4 * lane + j : lane + 32 * j);
        cs[j] = p.o.rb && n < p.N ? p.o.rb[n] : 1.0f;
        cb[j] = p.o.bias && n < p.N ? bias_at(p.o, n) : 0.0f;
    }
    for (int r = r0 + warp; r < r1; r += U * WARPS) {
        float v[U][P][4], ra[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int row = r + u * WARPS < r1 ? r + u * WARPS : r;
            ra[u] = p.o.ra ? p.o.ra[m0 + row] : 1.0f;
            const float *at = tile + row * pitch;
#pragma unroll
            for (int i = 0; i < P; ++i) {
                if (VEC) {
                    const float4 x = P == 1 ? *reinterpret_cast<const float4 *>(at + 4 * lane) : ld_cluster4(smem_u32(at + 4 * lane), i);
                    v[u][i][0] = x.x; v[u][i][1] = x.y; v[u][i][2] = x.z; v[u][i][3] = x.w;
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[u][i][j] = P == 1 ? at[lane + 32 * j] : ld_cluster1(smem_u32(at + lane + 32 * j), i);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int row = r + u * WARPS;
            if (row >= r1) break;
            float o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                o[j] = v[u][0][j];
#pragma unroll
                for (int i = 1; i < P; ++i) o[j] += v[u][i][j];
                o[j] = __fadd_rn(FAR ? scaled(o[j], ra[u], cs[j]) : __fmul_rn(__fmul_rn(o[j], ra[u]), cs[j]), cb[j]);
            }
            const int64_t off = (int64_t)(m0 + row) * p.o.ldo + n0;
            if (VEC) {
                if (n0 + 4 * lane >= p.N) continue;
                if (p.o.out_dtype == 2)
                    *reinterpret_cast<float4 *>(static_cast<float *>(p.o.out) + off + 4 * lane) = make_float4(o[0], o[1], o[2], o[3]);
                else
                    *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p.o.out) + off + 4 * lane) =
                        p.o.out_dtype == 0 ? make_uint2(pack_bf16_rn(o[0], o[1]), pack_bf16_rn(o[2], o[3]))
                                           : make_uint2(pack_f16_rn(o[0], o[1]), pack_f16_rn(o[2], o[3]));
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (n0 + lane + 32 * j < p.N) store_result(p.o, off + lane + 32 * j, o[j]);
            }
        }
    }
}

template <int KIND, int STAGES>
__global__ void __launch_bounds__(Cfg<KIND, STAGES>::THREADS, Cfg<KIND, STAGES>::CTAS)
    k_fp4_gemm(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
               const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSB, const Params p) {
    using C = Cfg<KIND, STAGES>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t sbase = smem_u32(smem);
    const uint32_t bar_full = sbase + C::OFF_BAR, bar_empty = bar_full + 8 * C::STAGES, bar_done = bar_empty + 8 * C::STAGES;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + C::OFF_MISC);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + C::OFF_MISC + 4);
    volatile int *far = reinterpret_cast<volatile int *>(smem + C::OFF_MISC + 8);       // a row's scale is_far
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tile = blockIdx.x / p.parts, part = blockIdx.x - tile * p.parts;
    const int m0 = tile % p.m_tiles * C::BM, n0 = tile / p.m_tiles * C::BN;
    const int kts = (p.Kp + KB - 1) / KB;
    const int kt0 = (int)((int64_t)kts * part / p.parts), kt1 = (int)((int64_t)kts * (part + 1) / p.parts);

    auto load = [&](int kt, int stage) {
        // boxes that run past the operand are zero-filled and count their full bytes
        const uint32_t at = sbase + stage * C::STAGE, fb = bar_full + 8 * stage;
        mbar_arrive_tx(fb, C::STAGE);
        tma_load_2d(&tmA, at, fb, kt * 128, m0);
        tma_load_2d(&tmB, at + C::OP, fb, kt * 128, n0);
        tma_load_3d(&tmSA, at + 2 * C::OP, fb, kt * C::TILES, m0 >> 7);
        tma_load_3d(&tmSB, at + 2 * C::OP + C::SF, fb, kt * C::TILES, n0 >> 7);
    };
    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; ++s) { mbar_init(bar_full + 8 * s, 1); mbar_init(bar_empty + 8 * s, 1); }
        mbar_init(bar_done, 1);
        *abort_flag = 0;
        *far = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        for (int s = 0; s < C::STAGES && kt0 + s < kt1; ++s) load(kt0 + s, s);      // the first stages, while the others prepare
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(C::COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    bool ok = true;
    if (warp == 0) {
        int stage = 0, issued = min(C::STAGES, kt1 - kt0);
        uint32_t phase = 1;
        if (issued < C::STAGES) { stage = issued; phase = 0; }
        for (int kt = kt0 + issued; kt < kt1; ++kt) {
            ok = warp_wait(lane, bar_empty + 8 * stage, phase ^ 1, abort_flag, WAIT_NS, p.err);
            if (!ok) break;
            if (lane == 0) load(kt, stage);
            ++issued;
            if (++stage == C::STAGES) { stage = 0; phase ^= 1; }
        }
        // the last copies land before the stages' place is used again
        for (int i = 0; i < C::STAGES && i < issued; ++i) {
            if (--stage < 0) { stage = C::STAGES - 1; phase ^= 1; }
            volatile int never = 0;
            if (lane == 0) mbar_wait(bar_full + 8 * stage, phase, &never, 100000000ull, p.err);
        }
        __syncwarp();
    } else if (warp == 1) {
        constexpr uint32_t idesc = instruction<KIND, C::BM, C::BN>();
        int stage = 0;
        uint32_t phase = 0;
        for (int kt = kt0; kt < kt1; ++kt) {
            ok = warp_wait(lane, bar_full + 8 * stage, phase, abort_flag, WAIT_NS, p.err);
            if (!ok) break;
            tc_fence_after();
            if (lane == 0) {
                const uint32_t at = sbase + stage * C::STAGE, sf = tmem + C::SFC + stage * 8 * C::TILES;
                // a stage's scale columns are its own: the MMAs that read them last are done when its operands are
#pragma unroll
                for (int j = 0; j < C::TILES; ++j) {
                    copy_scale(sf + 4 * j, sdesc_scale(at + 2 * C::OP + j * TILE));
                    copy_scale(sf + 4 * (C::TILES + j), sdesc_scale(at + 2 * C::OP + C::SF + j * TILE));
                }
                const uint64_t ad = sdesc(at), bd = sdesc(at + C::OP);
#pragma unroll
                for (int k = 0; k < KB / 64; ++k) {
                    const int j = KIND == NV ? k : k >> 1;
                    const uint32_t id = KIND == NV ? idesc : idesc | (k & 1) << 5 | (uint32_t)(k & 1) << 30;
                    mma<KIND>(tmem + C::ACC, ad + 2 * k, bd + 2 * k, id, sf + 4 * j, sf + 4 * (C::TILES + j),
                              (uint32_t)(kt > kt0 || k > 0));
                }
                mma_commit(bar_empty + 8 * stage);
            }
            __syncwarp();
            if (++stage == C::STAGES) { stage = 0; phase ^= 1; }
        }
        if (lane == 0) mma_commit(bar_done);        // also after a wait that gave up: what was issued is awaited
        __syncwarp();
    } else if (KIND == NV && p.o.ra) {              // beside the MMAs: the rows' loop below pays 1% for the test
        const int row = m0 + threadIdx.x - 64;
        if (row < p.M && is_far(p.o.ra[row])) *far = 1;
    }
    ok = warp_wait(lane, bar_done, 0, abort_flag, WAIT_NS + 1000000000ull, p.err) && ok;
    tc_fence_after();
    __syncthreads();                                // all copies and MMAs are done: the fp32 tile takes the stages' place
    float *tile_s = reinterpret_cast<float *>(smem);
    if (warp >= 2) {
        const int q = warp & 3, row = 32 * q + lane;
#pragma unroll
        for (int c = 0; c < C::BN / 32; ++c) {
            uint32_t r[32];
            tmem_ld32(tmem + C::ACC + 32 * c + ((uint32_t)(32 * q) << 16), r);
#pragma unroll
            for (int j = 0; j < 32; j += 4)
                *reinterpret_cast<uint4 *>(tile_s + row * C::PITCH + 32 * c + j) = make_uint4(r[j], r[j + 1], r[j + 2], r[j + 3]);
        }
    }
    tc_fence_before();
    cluster_arrive();                               // every CTA of the cluster comes by, a failed one too
    cluster_wait();
    if (ok) {
        const int rows = min(C::BM, p.M - m0), r0 = rows * part / p.parts, r1 = rows * (part + 1) / p.parts;
        auto write = [&](auto parts) {
            constexpr int P = decltype(parts)::value, W = C::THREADS / 32;
            if (KIND == NV && *far) write_rows<P, false, true, W>(p, tile_s, C::PITCH, m0, n0, r0, r1);
            else if (p.vec) write_rows<P, true, false, W>(p, tile_s, C::PITCH, m0, n0, r0, r1);
            else write_rows<P, false, false, W>(p, tile_s, C::PITCH, m0, n0, r0, r1);
        };
        if (p.parts == 1) write(std::integral_constant<int, 1>());
        else if (p.parts == 2) write(std::integral_constant<int, 2>());
        else if (p.parts == 4) write(std::integral_constant<int, 4>());
        else write(std::integral_constant<int, 8>());
    }
    __syncwarp();
    cluster_arrive();                               // nobody leaves while its sums are read
    cluster_wait();
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::COLS) : "memory");
}

// ---------------------------------------------------------------------------------------------------
// Many rows: tiles of 256 x 256 outputs, a pair of CTAs (cta_group::2) on each, one pair per two SMs, over the tiles in turn.
// Each CTA brings 128 rows of A and 128 of B into its shared memory, the pair's MMA reads both halves, so an operand byte from
// L2 serves twice the outputs of a tile that one SM holds alone. A step is 256 columns; the full barriers are the first CTA's, on
// which the copies of both complete. Scales of all 256 rows of B are brought to both CTAs.
//   warps 0, 1, 2   codes of A, codes of B, scales (each CTA its own; a request costs its thread some 35 ns and a wait 100 and
//                   more, so one warp for all three would be the bound: 412 ns a step)
//   warps 4 to 7    (first CTA) scales to tensor memory, every fourth step each: a tcgen05.cp of 512 bytes takes its thread some
//                   30 ns, 12 of them a step. A stage has scale columns of its own, so they run ahead of the MMAs
//   warp 3          (first CTA) the MMAs. It meets warps 4 to 7 at named barriers: its own look at a barrier in shared memory would
//                   wait until its MMAs have read their operands. Its four MMAs a step have no branch between them
//   warps 8 to 15   the sums: a thread holds 128 columns of a row in registers, hands tensor memory back, and only then scales,
//                   rounds and writes, beside the next tile's MMAs; 32 bytes of a row at a time go through shared memory, so that a
//                   row's outputs leave as whole sectors, 16 bytes a store or as many as N and the rows' starts allow
//                   (18944 rows, K = 4096: N = 4096 158 us, 4100 168, 4094 161, 4095 176; all but the first 217 - 229 one by one)
// Bound by the operands' way from L2, whether by its latency or by an SM's port is open. A step brings 38 KB to each SM (MX 35), 76
// (70) bytes a clock at the MMAs' rate of 512 clocks a step; 48 arrive (counters, NV, 9472 x 2048 x 16384: tensor pipe active
// 63%, L2 44%), NV and MX times are to one another as these bytes, and the port has been seen to give 60 (the tiles above). For
// latency: the 160 KB of codes under way over a round trip of 1.8 us are 48 bytes a clock, scales sent for further ahead were worth 8%,
// and codes released later cost 8%. Measured, 18944 x 4096 x 16384 (16 tiles a pair, 1024 steps): NV 498 us (5.1 PFLOP/s), MX 456;
// 15% more under the power limit of a long run. A tile's end costs 2 us (the wake of the epilogue, tensor memory's read 0.4, the
// issuer's wake). How far the scales' loads run ahead counts: 4 slots 536 us, 8 slots 491 (another GPU). All warps of the epilogue
// looking for the sums: 510; sleeps between the other looks change nothing. Groups of 8 column tiles (the rule below: 16 here): 520, of
// 4 543. Tried and slower (20240 x 4096 x 16384 NV, us, of 552 then): scale copies by the MMAs' thread 877, by one other warp 699,
// by two 593; a branch for the last columns between the MMAs 600; scales written to tensor memory from registers 1676; codes
// released every other step 8% more.
template <int KIND> struct Wide {
    static constexpr int BM = 256, BN = 256;
    static constexpr int TILES = KB / SPAN<KIND>;
    static constexpr int OP = 128 * 128, SFA = TILES * TILE, SFB = 2 * TILES * TILE;
    static constexpr int STAGES = Handoff::STAGES, STAGE = 2 * OP;      // codes of both operands
    static constexpr int CP = Handoff::CP;                      // warps that copy scales
    static constexpr int SLOTS = 2 * CP, SLOT = SFA + SFB;      // scales on their way to tensor memory
    static constexpr int ACC = 0, SFC = BN, SFW = 12 * TILES;   // tensor memory columns; SFW: a stage's scales
    static_assert(SFC + STAGES * SFW <= 512, "tensor memory");
    static constexpr int EPI = 8, PITCH = 48;                   // warps; bytes a row of their chunks of 32
    static constexpr int OFF_SF = STAGES * STAGE, OFF_EPI = OFF_SF + SLOTS * SLOT;
    static constexpr int OFF_COLS = OFF_EPI + EPI * 32 * PITCH;                             // column scales and bias: [2][2][256]
    static constexpr int OFF_ONES = OFF_COLS + 2 * 2 * 256 * 4;                            // 128 column scales of 1
    static constexpr int OFF_BAR = OFF_ONES + 128 * 4;
    static constexpr int OFF_MISC = OFF_BAR + 8 * (2 * STAGES + 2 * SLOTS + 3);
    static constexpr int SMEM = OFF_MISC + 16 + 1024;
    static_assert(SMEM <= 232448, "shared memory");
    static constexpr int THREADS = 256 + 32 * EPI;
    // registers a thread: launched with 128 (512 x 128 = 65536), the epilogue's warps take over what the others leave
    static constexpr int REGS = 56, EPI_REGS = 200;
    static_assert(THREADS == 512 && 256 * REGS + 32 * EPI * EPI_REGS <= THREADS * 128, "registers");
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
    return a;
}
// tile loads into this CTA's shared memory that complete on a barrier of either CTA of the pair
__device__ __forceinline__ void pair_load_2d(const CUtensorMap *map, uint32_t dst, uint32_t bar, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 ::"r"(dst), "l"((uint64_t)map), "r"(bar), "r"(x), "r"(y)
                 : "memory");
}
__device__ __forceinline__ void pair_load_3d(const CUtensorMap *map, uint32_t dst, uint32_t bar, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(dst), "l"((uint64_t)map), "r"(bar), "r"(0), "r"(y), "r"(z)
                 : "memory");
}
__device__ __forceinline__ void pair_copy_scale(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
template <int KIND>
__device__ __forceinline__ void pair_mma(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t acc) {
    if (KIND == NV)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
                     ::"r"(d), "l"(ad), "l"(bd), "r"(idesc), "r"(acc), "r"(sa), "r"(sb) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
                     ::"r"(d), "l"(ad), "l"(bd), "r"(idesc), "r"(acc), "r"(sa), "r"(sb) : "memory");
}
// arrives on the barrier at this offset in both CTAs when the MMAs so far are done
__device__ __forceinline__ void pair_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(bar), "h"((uint16_t)3) : "memory");
}
// ... in this CTA alone
__device__ __forceinline__ void pair_commit1(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void arrive_at(uint32_t cluster_bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}

// a wait of a step's chain: some looks before the clock of the bounded wait is read (504 -> 495 us at 18944 x 4096 x 16384)
__device__ __forceinline__ bool spin_wait(int lane, uint32_t bar, uint32_t parity, volatile int *abort_flag, int *err) {
    bool ok = true;
    if (lane == 0) {
        bool in = false;
#pragma unroll 1
        for (int i = 0; i < 200 && !in; ++i) in = mbar_try(bar, parity);
        if (!in) ok = mbar_wait(bar, parity, abort_flag, WAIT_NS, err);
    }
    return __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
}
// W warps meet at named barrier 1: whether `stop` holds in any of them
template <int W> __device__ __forceinline__ bool any_of(bool stop) {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(r) : "r"(stop ? 1u : 0u), "n"(32 * W) : "memory");
    return r != 0;
}
// after a wait that gave up: time for the copies in flight, of both CTAs, to land
__device__ __forceinline__ void land() {
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 10000000ull) { }
}

// tile t -> (row tile, column tile): groups of `gn` column tiles, whose weights stay in L2 while the rows pass
struct Raster {
    int m_tiles, n_tiles, gn;
};
__device__ __forceinline__ void tile_at(const Raster &r, int t, int &mt, int &nt) {
    const int g = t / (r.m_tiles * r.gn), in = t - g * r.m_tiles * r.gn;
    const int width = r.n_tiles - g * r.gn < r.gn ? r.n_tiles - g * r.gn : r.gn;
    mt = in / width;
    nt = g * r.gn + in - mt * width;
}

// a pair's steps: the stages of its tiles, tile by tile
struct Step {
    int tile, kt, mt, nt;
};
__device__ __forceinline__ Step first_step(const Raster &r, int tile) {
    Step s;
    s.tile = tile; s.kt = 0;
    tile_at(r, tile, s.mt, s.nt);
    return s;
}
__device__ __forceinline__ void next_step(const Raster &r, Step &s, int kts, int pairs) {
    if (++s.kt < kts) return;
    s.kt = 0;
    s.tile += pairs;
    if (s.tile < r.m_tiles * r.n_tiles) tile_at(r, s.tile, s.mt, s.nt);
}

struct WideParams {
    Result o;
    int unit;                   // bytes that are stored at a time: 16, 8, 4 or 2
    int M, N, Kp, tiles;
    Raster raster;
    int *err;
};

// EB: bytes of an output
template <int KIND, int EB>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Wide<KIND>::THREADS, 1)
    k_fp4_gemm_wide(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                    const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSB, const WideParams p) {
    using C = Wide<KIND>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t sbase = smem_u32(smem);
    const uint32_t bar_full = sbase + C::OFF_BAR, bar_empty = bar_full + 8 * C::STAGES;
    const uint32_t bar_sfull = bar_empty + 8 * C::STAGES, bar_sempty = bar_sfull + 8 * C::SLOTS;
    const uint32_t bar_tfull = bar_sempty + 8 * C::SLOTS, bar_tempty = bar_tfull + 8, bar_drain = bar_tempty + 8;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + C::OFF_MISC);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + C::OFF_MISC + 4);
    volatile int *taken = reinterpret_cast<volatile int *>(smem + C::OFF_MISC + 8);     // steps that the issuer has met
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_rank(), pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const int kts = (p.Kp + KB - 1) / KB;

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; ++s) {
            mbar_init(bar_full + 8 * s, 3);         // A, B, and their scales in tensor memory
            mbar_init(bar_empty + 8 * s, 1);
        }
        for (int s = 0; s < C::SLOTS; ++s) { mbar_init(bar_sfull + 8 * s, 1); mbar_init(bar_sempty + 8 * s, 1); }
        mbar_init(bar_tfull, 1);
        mbar_init(bar_tempty, 2 * C::EPI);
        mbar_init(bar_drain, 1);
        *abort_flag = 0;
        *taken = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp >= 8 && warp < 12) reinterpret_cast<float *>(smem + C::OFF_ONES)[threadIdx.x - 256] = 1.0f;
    if (warp == 4) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_arrive();                       // the other CTA's barriers are there before a copy completes on them
    cluster_wait();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    const int steps = (p.tiles - pair + pairs - 1) / pairs * kts;      // of this pair's tiles, one after the other
    if (warp < 8) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REGS));
    if (warp < 2) {
        int stage = 0;
        uint32_t phase = 0;
        Step s = first_step(p.raster, pair);
        bool ok = true;
        for (int i = 0; i < steps + C::STAGES; ++i) {       // the last only wait: this CTA stays until their arrivals have reached it
            ok = spin_wait(lane, bar_empty + 8 * stage, phase ^ 1, abort_flag, p.err);
            if (!ok) break;
            if (lane == 0 && i < steps) {
                const uint32_t at = sbase + stage * C::STAGE + warp * C::OP, fb = in_cta(bar_full + 8 * stage, 0);
                if (rank == 0) mbar_arrive_tx(bar_full + 8 * stage, 2 * C::OP);
                pair_load_2d(warp == 0 ? &tmA : &tmB, at, fb, s.kt * 128, (warp == 0 ? s.mt : s.nt) * 256 + rank * 128);
            }
            __syncwarp();
            if (i < steps) next_step(p.raster, s, kts, pairs);
            if (++stage == C::STAGES) { stage = 0; phase ^= 1; }
        }
        if (!ok) land();
    } else if (warp == 2) {
        int slot = 0;
        uint32_t phase = 0;
        Step s = first_step(p.raster, pair);
        bool ok = true;
        for (int i = 0; i < steps + C::SLOTS; ++i) {
            ok = spin_wait(lane, bar_sempty + 8 * slot, phase ^ 1, abort_flag, p.err);
            if (!ok) break;
            if (lane == 0 && i < steps) {
                const uint32_t at = sbase + C::OFF_SF + slot * C::SLOT, fb = in_cta(bar_sfull + 8 * slot, 0);
                if (rank == 0) mbar_arrive_tx(bar_sfull + 8 * slot, 2 * C::SLOT);
                pair_load_3d(&tmSA, at, fb, s.kt * C::TILES, 2 * s.mt + rank);
                pair_load_3d(&tmSB, at + C::SFA, fb, s.kt * C::TILES, 2 * s.nt);
            }
            __syncwarp();
            if (i < steps) next_step(p.raster, s, kts, pairs);
            if (++slot == C::SLOTS) { slot = 0; phase ^= 1; }
        }
        if (!ok) land();
    } else if (warp >= 4 && warp < 8 && rank == 0) {
        // step i, every C::CP-th: its scales into the columns of its stage, when the MMAs that read them last are done; then, when they
        // and the codes are in, the issuer's release. After a wait that gave up the steps that are left are only released, each not
        // before the issuer has met the step that had its barrier before (Handoff), so that the issuer comes to its end: it needs
        // steps i - CP to i - 1 for that, whose warps have released theirs or are themselves on the way, and its own wait is bounded.
        // A parity tells a phase from its neighbours only, and these warps skip steps. So each has two slots of its own, whose phases
        // it sees one after the other; that MMAs of step i - 2 STAGES are over, when those of i - STAGES are waited for, follows from
        // step i - CP, whose codes the warp has seen in (they came after the MMAs of step i - CP - STAGES); and that the full
        // barrier's phase before is over follows from the MMAs of step i - STAGES.
        static_assert(C::SLOTS == 2 * C::CP && C::CP <= C::STAGES, "phases that a warp may find");
        int stage = warp - 4, slot = warp - 4, last = -1;
        uint32_t phase = 0, sphase = 0, last_phase = 0;
        bool ok = true;
        for (int i = warp - 4; i < steps; i += C::CP) {
            ok = ok && spin_wait(lane, bar_sfull + 8 * slot, sphase, abort_flag, p.err);
            ok = ok && spin_wait(lane, bar_empty + 8 * stage, phase ^ 1, abort_flag, p.err);
            if (ok) {
                tc_fence_after();
                if (lane == 0) {
                    const uint32_t at = sbase + C::OFF_SF + slot * C::SLOT, sf = tmem + C::SFC + stage * C::SFW;
#pragma unroll
                    for (int j = 0; j < C::TILES; ++j) {        // of A 4 columns, of B 8 (its two blocks of 128 rows) a tile
                        pair_copy_scale(sf + 4 * j, sdesc_scale(at + j * TILE));
                        pair_copy_scale(sf + 4 * C::TILES + 8 * j, sdesc_scale(at + C::SFA + j * TILE));
                        pair_copy_scale(sf + 4 * C::TILES + 8 * j + 4, sdesc_scale(at + C::SFA + (C::TILES + j) * TILE));
                    }
                    pair_commit1(bar_full + 8 * stage);
                    pair_commit(bar_sempty + 8 * slot);
                }
                __syncwarp();
                last = slot;
                last_phase = sphase;
                ok = spin_wait(lane, bar_full + 8 * stage, phase, abort_flag, p.err);
            }
            if (!ok) {
                const uint64_t t0 = globaltimer_ns();
                while (*taken < Handoff::taken_before(i) && globaltimer_ns() - t0 < 4 * WAIT_NS) { }
                __syncwarp();
            }
            asm volatile("barrier.cta.arrive %0, 64;" ::"r"(2 + stage) : "memory");
            if ((stage += C::CP) >= C::STAGES) { stage -= C::STAGES; phase ^= 1; }
            if ((slot += C::CP) >= C::SLOTS) { slot -= C::SLOTS; sphase ^= 1; }
        }
        if (last >= 0 && lane == 0) {
            volatile int never = 0;
            mbar_wait(bar_sempty + 8 * last, last_phase, &never, 100000000ull, p.err);
        }
        __syncwarp();
    } else if (warp == 3 && rank == 0) {
        constexpr uint32_t idesc = instruction<KIND, C::BM, C::BN>();
        int stage = 0, kt = 0;
        uint32_t tphase = 0;
        bool ok = true;
        for (int i = 0; i < steps; ++i) {
            if (kt == 0 && ok) {
                ok = warp_wait(lane, bar_tempty, tphase ^ 1, abort_flag, WAIT_NS, p.err);
                tphase ^= 1;
            }
            asm volatile("barrier.cta.sync %0, 64;" ::"r"(2 + stage) : "memory");
            if (lane == 0) *taken = i + 1;
            if (ok) {
                tc_fence_after();
                if (lane == 0) {
                    const uint32_t at = sbase + stage * C::STAGE, sf = tmem + C::SFC + stage * C::SFW;
                    const uint64_t ad = sdesc(at), bd = sdesc(at + C::OP);
#pragma unroll
                    for (int k = 0; k < KB / 64; ++k) {
                        const int j = KIND == NV ? k : k >> 1;
                        const uint32_t id = KIND == NV ? idesc : idesc | (k & 1) << 5 | (uint32_t)(k & 1) << 30;
                        pair_mma<KIND>(tmem + C::ACC, ad + 2 * k, bd + 2 * k, id, sf + 4 * j, sf + 4 * C::TILES + 8 * j,
                                       (uint32_t)(kt > 0 || k > 0));
                    }
                    pair_commit(bar_empty + 8 * stage);
                    if (kt == kts - 1) pair_commit(bar_tfull);
                }
                __syncwarp();
            }
            if (++kt == kts) kt = 0;
            if (++stage == C::STAGES) stage = 0;
        }
        // what was issued finishes before tensor memory is released
        if (lane == 0) {
            volatile int never = 0;
            pair_commit1(bar_drain);
            mbar_wait(bar_drain, 0, &never, 100000000ull, p.err);
        }
        __syncwarp();
    } else if (warp >= 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::EPI_REGS));
        const int q = warp & 3, half = (warp - 8) >> 2, thread = threadIdx.x - 256;
        const uint32_t tcol = tmem + C::ACC + 128 * half + ((uint32_t)(32 * q) << 16);
        const uint32_t tempty = in_cta(bar_tempty, 0);
        uint8_t *chunk = smem + C::OFF_EPI + (warp - 8) * 32 * C::PITCH;
        uint32_t tphase = 0;
        int it = 0;
        bool ok = true;
        for (int tile = pair; tile < p.tiles; tile += pairs, ++it) {
            int mt, nt;
            tile_at(p.raster, tile, mt, nt);
            const int m0 = mt * 256 + rank * 128 + 32 * q, n0 = nt * 256 + 128 * half;
            // the tile's column scales and bias into shared memory (two tiles' places in turn) and the row's scale, beside its MMAs
            float *cols = reinterpret_cast<float *>(smem + C::OFF_COLS) + (it & 1) * 512;
            const int n = nt * 256 + thread;
            cols[thread] = p.o.rb && n < p.N ? p.o.rb[n] : 1.0f;
            cols[256 + thread] = p.o.bias && n < p.N ? bias_at(p.o, n) : 0.0f;
            float ra = p.o.ra && m0 + lane < p.M ? p.o.ra[m0 + lane] : 1.0f;
            // one warp looks at the barrier, the others wait for it asleep; all leave together
            if (warp == 8) ok = warp_wait(lane, bar_tfull, tphase, abort_flag, 2 * WAIT_NS, p.err);
            ok = !any_of<C::EPI>(!ok);
            if (!ok) break;
            tphase ^= 1;
            tc_fence_after();
            uint32_t r[4][32];
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_ld32(tcol + 32 * c, r[c]);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) arrive_at(tempty);
            const float *rb = cols + 128 * half, *bias = rb + 256;
            if (KIND == NV && __any_sync(0xffffffffu, is_far(ra))) {
                // rare, so apart: the scales in an order of their own here, and ones for them below (a test in the loop below:
                // 157 -> 165 us at 18944 x 4096 x 4096; a second loop: 178 -> 187 at 18944 x 4095 x 4096)
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int j = 0; j < 32; ++j) r[c][j] = __float_as_uint(scaled(__uint_as_float(r[c][j]), ra, rb[32 * c + j]));
                ra = 1.0f;
                rb = reinterpret_cast<const float *>(smem + C::OFF_ONES);
            }
            constexpr int COLS = 32 / EB;               // of a chunk: 32 bytes a row
#pragma unroll
            for (int c = 0; c < 128 / COLS; ++c) {
                uint32_t w[8];
#pragma unroll
                for (int j = 0; j < COLS; j += 4) {
                    const float4 s = *reinterpret_cast<const float4 *>(rb + COLS * c + j), b = *reinterpret_cast<const float4 *>(bias + COLS * c + j);
                    const uint32_t *x = &r[(COLS * c + j) >> 5][(COLS * c + j) & 31];
                    float v[4] = {__uint_as_float(x[0]), __uint_as_float(x[1]), __uint_as_float(x[2]), __uint_as_float(x[3])};
                    if (KIND == NV) {
                        v[0] = __fmul_rn(__fmul_rn(v[0], ra), s.x); v[1] = __fmul_rn(__fmul_rn(v[1], ra), s.y);
                        v[2] = __fmul_rn(__fmul_rn(v[2], ra), s.z); v[3] = __fmul_rn(__fmul_rn(v[3], ra), s.w);
                    }
                    v[0] = __fadd_rn(v[0], b.x); v[1] = __fadd_rn(v[1], b.y); v[2] = __fadd_rn(v[2], b.z); v[3] = __fadd_rn(v[3], b.w);
                    if (EB == 4) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) w[j + i] = __float_as_uint(v[i]);
                    } else if (p.o.out_dtype == 0) {
                        w[j >> 1] = pack_bf16_rn(v[0], v[1]);
                        w[(j >> 1) + 1] = pack_bf16_rn(v[2], v[3]);
                    } else {
                        w[j >> 1] = pack_f16_rn(v[0], v[1]);
                        w[(j >> 1) + 1] = pack_f16_rn(v[2], v[3]);
                    }
                }
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    *reinterpret_cast<uint4 *>(chunk + lane * C::PITCH + 16 * j) = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
                __syncwarp();
                const int nc = n0 + COLS * c;
                uint8_t *out = static_cast<uint8_t *>(p.o.out) + ((int64_t)m0 * p.o.ldo + nc) * EB;
                auto store = [&](auto zero) {           // units of U bytes: 32 / U lanes a row, U rows at a time
                    using T = decltype(zero);
                    constexpr int U = sizeof(T), G = U < 8 ? 8 : 32 / U;
                    const int at = U * (lane % (32 / U)), row0 = lane / (32 / U);
                    const bool in = nc + at / EB < p.N;
#pragma unroll
                    for (int g = 0; g < 32 / U; g += G) {
                        T y[G];
#pragma unroll
                        for (int i = 0; i < G; ++i) y[i] = *reinterpret_cast<const T *>(chunk + (U * (g + i) + row0) * C::PITCH + at);
#pragma unroll
                        for (int i = 0; i < G; ++i) {
                            const int row = U * (g + i) + row0;
                            if (in && m0 + row < p.M) *reinterpret_cast<T *>(out + (int64_t)row * p.o.ldo * EB + at) = y[i];
                        }
                    }
                };
                if (p.unit == 16) store(uint4());
                else if (p.unit == 8) store(uint2());
                else if (EB == 4 || p.unit == 4) store(uint32_t());
                else store(uint16_t());
            }
        }
        if (!ok) *abort_flag = 1;
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster_arrive();                       // neither CTA leaves while the other may reach its shared or tensor memory
    cluster_wait();
    tc_fence_after();
    if (warp == 4) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// ---------------------------------------------------------------------------------------------------
// host side

static PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    if (fn == nullptr) {
        void *ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &ptr, 12000, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
    }
    return fn;
}
// codes: rows of `bytes` bytes, `ld` apart; boxes of 128 bytes x `box` rows, 128-byte swizzle
static bool map_codes(CUtensorMap *map, const void *base, uint64_t rows, uint64_t bytes, uint64_t ld, uint32_t box) {
    PFN_cuTensorMapEncodeTiled_v12000 fn = encode_fn();
    if (fn == nullptr) return false;
    cuuint64_t dims[2] = {bytes, rows}, strides[1] = {ld};
    cuuint32_t shape[2] = {128, box}, estr[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), dims, strides, shape, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// scales: [row blocks][group blocks][512 bytes]; boxes of `tiles` x `blocks` tiles
static bool map_scales(CUtensorMap *map, const void *base, uint64_t blocks, uint64_t tiles, uint32_t box_tiles, uint32_t box_blocks) {
    PFN_cuTensorMapEncodeTiled_v12000 fn = encode_fn();
    if (fn == nullptr) return false;
    cuuint64_t dims[3] = {TILE / 4, tiles, blocks}, strides[2] = {TILE, TILE * tiles};
    cuuint32_t shape[3] = {TILE / 4, box_tiles, box_blocks}, estr[3] = {1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, const_cast<void *>(base), dims, strides, shape, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// outputs may be stored `bytes` at a time: rows begin on that boundary and are whole units
static int whole_stores(const Fp4GemmArgs &a, int bytes) {
    const int size = a.out_dtype == 2 ? 4 : 2;
    return a.N * size % bytes == 0 && a.ldo * size % bytes == 0 && reinterpret_cast<uintptr_t>(a.out) % bytes == 0;
}
static int store_unit(const Fp4GemmArgs &a) {
    int bytes = 16;
    while (!whole_stores(a, bytes)) bytes /= 2;
    return bytes;
}
template <int KIND, typename C> static bool maps(const Fp4GemmArgs &a, int b_blocks, CUtensorMap (&m)[4]) {
    const uint64_t sp = (uint64_t)cdiv(a.K, SPAN<KIND>);
    return map_codes(&m[0], a.qa, a.M, a.K / 2, a.lda, 128) && map_codes(&m[1], a.qw, a.N, a.K / 2, a.ldw, 128) &&
           map_scales(&m[2], a.sa, cdiv(a.M, 128), sp, C::TILES, 1) &&
           map_scales(&m[3], a.sw, cdiv(a.N, 128), sp, C::TILES, b_blocks);
}
// the shared-memory opt-in, once per kernel and device
template <typename K> static cudaError_t opt_in(K kernel, int bytes, bool (&done)[HN_MAX_DEV]) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= HN_MAX_DEV) return cudaErrorInvalidDevice;
    if (done[dev]) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    done[dev] = e == cudaSuccess;
    return e;
}

template <int KIND> static cudaError_t launch_wide(const Fp4GemmArgs &a, cudaStream_t st, const char **msg) {
    using C = Wide<KIND>;
    WideParams p;
    cudaError_t e = device_error_word(err_slot(st), &p.err);
    if (e != cudaSuccess) return e;
    p.o = {a.ra, a.rw, a.bias, a.bias_dtype, a.out, a.ldo, a.out_dtype};
    p.M = (int)a.M; p.N = (int)a.N; p.Kp = (int)a.K;
    p.unit = store_unit(a);
    p.raster.m_tiles = (int)cdiv(a.M, C::BM);
    p.raster.n_tiles = (int)cdiv(a.N, C::BN);
    p.tiles = p.raster.m_tiles * p.raster.n_tiles;
    // the weights of a group of column tiles: 32 MB at most, so that they stay in L2
    const int64_t fit = (32LL << 20) / (C::BN * (a.K / 2));
    p.raster.gn = (int)(fit < 1 ? 1 : fit > p.raster.n_tiles ? p.raster.n_tiles : fit);
    CUtensorMap m[4];
    if (!maps<KIND, C>(a, 2, m)) {
        *msg = "cuTensorMapEncodeTiled failed (pointer/stride alignment or driver entry point)";
        return cudaErrorInvalidValue;
    }
    int pairs = (num_sms() - a.sm_reserve) / 2;
    if (pairs > p.tiles) pairs = p.tiles;
    if (pairs < 1) pairs = 1;
    auto go = [&](auto kernel, bool (&done)[HN_MAX_DEV]) {
        cudaError_t e = opt_in(kernel, C::SMEM, done);
        if (e != cudaSuccess) return e;
        kernel<<<2 * pairs, C::THREADS, C::SMEM, st>>>(m[0], m[1], m[2], m[3], p);
        return cudaGetLastError();
    };
    static bool done2[HN_MAX_DEV], done4[HN_MAX_DEV];
    return a.out_dtype == 2 ? go(k_fp4_gemm_wide<KIND, 4>, done4) : go(k_fp4_gemm_wide<KIND, 2>, done2);
}

template <int KIND, int STAGES> static cudaError_t launch_narrow(const Fp4GemmArgs &a, int64_t tiles, int parts, cudaStream_t st, const char **msg) {
    using C = Cfg<KIND, STAGES>;
    Params p;
    cudaError_t e = device_error_word(err_slot(st), &p.err);
    if (e != cudaSuccess) return e;
    p.o = {a.ra, a.rw, a.bias, a.bias_dtype, a.out, a.ldo, a.out_dtype};
    p.M = (int)a.M; p.N = (int)a.N; p.Kp = (int)a.K;
    p.vec = whole_stores(a, a.out_dtype == 2 ? 16 : 8);
    p.m_tiles = (int)cdiv(a.M, C::BM);
    p.parts = parts;
    CUtensorMap m[4];
    if (!maps<KIND, C>(a, 1, m)) {
        *msg = "cuTensorMapEncodeTiled failed (pointer/stride alignment or driver entry point)";
        return cudaErrorInvalidValue;
    }
    static bool done[HN_MAX_DEV];
    e = opt_in(k_fp4_gemm<KIND, STAGES>, C::SMEM, done);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles * p.parts));
    cfg.blockDim = dim3(C::THREADS);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = p.parts; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k_fp4_gemm<KIND, STAGES>, m[0], m[1], m[2], m[3], p);
}

template <int KIND> static cudaError_t launch(const Fp4GemmArgs &a, cudaStream_t st, const char **msg) {
    const int sms = num_sms();
    const int64_t tiles = cdiv(a.M, 128) * cdiv(a.N, 128), kts = cdiv(a.K, KB);
    // Tiles of 128 x 128 while all of them run at once, two CTAs an SM; pairs of CTAs beyond. Measured (us, 128 x 128 / pairs):
    // 777 x 5000 x 2080 (280 tiles) 16.3 / 18.6; 1024 x 5120 x 4096 (320) 33.8 / 25.2; 2560 x 2048 x 1024 (320) 16.8 / 14.8.
    // Also pairs where SMs would get two tiles and the pairs one, in eight steps or more: 2048 x 2048 x 1024 11.6 / 11.9,
    // x 2048 14.1 / 13.4, x 16384 50.5 / 37.3; 300 x 8192 x 4096 18.9 / 16.8; but 1024 x 2048 x 16384 (128 tiles) 29.1 / 34.7. Where
    // outputs have to leave one by one, from 32 steps on: the pairs' epilogue is 4 us more then (2048 x 2041 x 2048 14.1 / 17.6)
    const bool one_round = tiles > sms && cdiv(a.M, 256) * cdiv(a.N, 256) <= sms / 2 && kts >= (store_unit(a) > 2 ? 8 : 32);
    if (tiles > 2 * sms || one_round) return launch_wide<KIND>(a, st, msg);
    // K is split over a cluster while SMs are idle and each part keeps two stages; over a second CTA on each SM only where a part
    // keeps eight. Measured (us, 1 / 2 / 4 / 8 parts): 48 x 8192 x 4096 MX 13.1 / 9.9 / 11.6 / -; 128 x 4096 x 4096 NV 16.4 / 11.5 /
    // 10.1 / 16.5; 16 x 4096 x 16384 NV 43 / 25 / 17 / 15
    int parts = 1;
    while (parts < 8 && kts >= 4 * parts && (tiles * parts * 2 <= sms || (tiles * parts * 2 <= 2 * sms && kts >= 16 * parts))) parts *= 2;
    // a CTA alone on its SM has twice the stages in flight
    if (tiles * parts <= sms) return launch_narrow<KIND, 6>(a, tiles, parts, st, msg);
    return launch_narrow<KIND, 3>(a, tiles, parts, st, msg);
}

} // namespace fp4g

cudaError_t launch_fp4_gemm(const Fp4GemmArgs &a, cudaStream_t st, const char **msg) {
    if (fp4_gemv_applies(a)) return launch_fp4_gemv(a, st);
    return a.kind == fp4::MX ? fp4g::launch<fp4::MX>(a, st, msg) : fp4g::launch<fp4::NV>(a, st, msg);
}

} // namespace hn
