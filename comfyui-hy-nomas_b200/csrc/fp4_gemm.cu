// fp4_gemm.cu - the product of two operands of 4-bit codes with block scales, on the sm_100a tensor cores.
//
//   y[m, n] = ra[m] rb[n] sum_g sa[m, g] sb[n, g] sum_{k in g} a[m, k] b[n, k]  (+ bias[n])
//
// tcgen05.mma.kind::mxf4 (scales 2^e per 32) and kind::mxf4nvf4 (e4m3 per 16) multiply the block scales in, so the accumulator
// in tensor memory is the whole sum in fp32; the row scales, the bias and the one rounding are the epilogue's.
#include <cuda.h>
#include <cudaTypedefs.h>

#include "fp4.cuh"
#include "hn_kernels.h"
#include "hn_tc.cuh"

namespace hn {
namespace fp4g {

using namespace fp4;
using namespace tc;

constexpr uint64_t WAIT_NS = 2000000000ull;     // 2 s
constexpr int KB = 256;                         // columns of a stage: 128 bytes of codes a row

// Tiles of 128 x 128 outputs. A cluster of S CTAs shares one: each takes a part of K, leaves its fp32 sums in its shared memory,
// and CTA r of the cluster adds those of its 128 / S rows, in the CTAs' order, and writes them.
template <int KIND> struct Cfg {
    static constexpr int BM = 128, BN = 128, STAGES = 3;
    static constexpr int TILES = KB / SPAN<KIND>;               // scale tiles of an operand in a stage
    static constexpr int OP = 128 * 128, SF = TILES * TILE;     // bytes of a stage: codes and scales of an operand
    static constexpr int STAGE = 2 * OP + 2 * SF;
    static constexpr int OFF_BAR = STAGES * STAGE;
    static constexpr int PITCH = BN + 4;                        // floats a row of the fp32 tile (in the stages' place)
    static_assert(BM * PITCH * 4 <= OFF_BAR, "the fp32 tile lies over the stages");
    static constexpr int OFF_MISC = OFF_BAR + 8 * (2 * STAGES + 1);
    static constexpr int SMEM = OFF_MISC + 16 + 1024;           // + alignment slack
    static constexpr int ACC = 0, SFC = BN;                     // tensor memory columns: sums, then 8 x TILES a stage
    static constexpr int COLS = 256;
    static constexpr int THREADS = 192;                         // producer, issuer, four warps that empty tensor memory
    static_assert(SFC + STAGES * 8 * TILES <= COLS, "tensor memory");
    static_assert(2 * (SMEM + 1024) <= 228 * 1024, "two CTAs an SM");
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

template <int KIND>
__global__ void __launch_bounds__(Cfg<KIND>::THREADS, 2)
    k_fp4_gemm(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
               const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSB, const Params p) {
    using C = Cfg<KIND>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t sbase = smem_u32(smem);
    const uint32_t bar_full = sbase + C::OFF_BAR, bar_empty = bar_full + 8 * C::STAGES, bar_done = bar_empty + 8 * C::STAGES;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + C::OFF_MISC);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + C::OFF_MISC + 4);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tile = blockIdx.x / p.parts, part = blockIdx.x - tile * p.parts;
    const int m0 = tile % p.m_tiles * C::BM, n0 = tile / p.m_tiles * C::BN;
    const int kts = (p.Kp + KB - 1) / KB;
    const int kt0 = (int)((int64_t)kts * part / p.parts), kt1 = (int)((int64_t)kts * (part + 1) / p.parts);

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; ++s) { mbar_init(bar_full + 8 * s, 1); mbar_init(bar_empty + 8 * s, 1); }
        mbar_init(bar_done, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
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
        int stage = 0, issued = 0;
        uint32_t phase = 0;
        for (int kt = kt0; kt < kt1; ++kt) {
            ok = warp_wait(lane, bar_empty + 8 * stage, phase ^ 1, abort_flag, WAIT_NS, p.err);
            if (!ok) break;
            if (lane == 0) {
                // boxes that run past the operand are zero-filled and count their full bytes
                const uint32_t at = sbase + stage * C::STAGE, fb = bar_full + 8 * stage;
                mbar_arrive_tx(fb, C::STAGE);
                tma_load_2d(&tmA, at, fb, kt * 128, m0);
                tma_load_2d(&tmB, at + C::OP, fb, kt * 128, n0);
                tma_load_3d(&tmSA, at + 2 * C::OP, fb, kt * C::TILES, m0 >> 7);
                tma_load_3d(&tmSB, at + 2 * C::OP + C::SF, fb, kt * C::TILES, n0 >> 7);
            }
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
                const int left = p.Kp - kt * KB;            // a stage's scale columns are its own: the MMAs that read them last
#pragma unroll                                              // are done when its operands are
                for (int j = 0; j < C::TILES; ++j) {
                    copy_scale(sf + 4 * j, sdesc_scale(at + 2 * C::OP + j * TILE));
                    copy_scale(sf + 4 * (C::TILES + j), sdesc_scale(at + 2 * C::OP + C::SF + j * TILE));
                }
                const uint64_t ad = sdesc(at), bd = sdesc(at + C::OP);
#pragma unroll
                for (int k = 0; k < KB / 64; ++k) {
                    if (64 * k >= left) break;
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
        const int rows = C::BM / p.parts, first = part * rows;
        for (int r = first + warp; r < first + rows && m0 + r < p.M; r += C::THREADS / 32) {
            const int64_t off = (int64_t)(m0 + r) * p.o.ldo + n0;
            const float ra = p.o.ra ? p.o.ra[m0 + r] : 1.0f;
            if (p.vec) {
                const int n = n0 + 4 * lane;
                const uint32_t addr = smem_u32(tile_s + r * C::PITCH + 4 * lane);
                float4 v = p.parts == 1 ? *reinterpret_cast<float4 *>(tile_s + r * C::PITCH + 4 * lane) : ld_cluster4(addr, 0);
                for (int i = 1; i < p.parts; ++i) {
                    const float4 w = ld_cluster4(addr, i);
                    v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
                }
                if (n < p.N) {
                    v.x = finish(p.o, v.x, ra, n); v.y = finish(p.o, v.y, ra, n + 1);
                    v.z = finish(p.o, v.z, ra, n + 2); v.w = finish(p.o, v.w, ra, n + 3);
                    if (p.o.out_dtype == 2)
                        *reinterpret_cast<float4 *>(static_cast<float *>(p.o.out) + off + 4 * lane) = v;
                    else
                        *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p.o.out) + off + 4 * lane) =
                            p.o.out_dtype == 0 ? make_uint2(pack_bf16_rn(v.x, v.y), pack_bf16_rn(v.z, v.w))
                                               : make_uint2(pack_f16_rn(v.x, v.y), pack_f16_rn(v.z, v.w));
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int n = lane + 32 * j;
                    const uint32_t addr = smem_u32(tile_s + r * C::PITCH + n);
                    float v = p.parts == 1 ? tile_s[r * C::PITCH + n] : ld_cluster1(addr, 0);
                    for (int i = 1; i < p.parts; ++i) v += ld_cluster1(addr, i);
                    if (n0 + n < p.N) store_result(p.o, off + n, finish(p.o, v, ra, n0 + n));
                }
            }
        }
    }
    __syncwarp();
    cluster_arrive();                               // nobody leaves while its sums are read
    cluster_wait();
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::COLS) : "memory");
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

template <int KIND> static cudaError_t launch(const Fp4GemmArgs &a, cudaStream_t st, const char **msg) {
    using C = Cfg<KIND>;
    Params p;
    cudaError_t e = device_error_word(err_slot(st), &p.err);
    if (e != cudaSuccess) return e;
    p.o = {a.ra, a.rw, a.bias, a.bias_dtype, a.out, a.ldo, a.out_dtype};
    p.M = (int)a.M; p.N = (int)a.N; p.Kp = (int)a.K;
    const int64_t out_bytes = a.out_dtype == 2 ? 16 : 8;                        // of four outputs
    p.vec = a.N % 4 == 0 && a.ldo % 4 == 0 && reinterpret_cast<uintptr_t>(a.out) % out_bytes == 0;
    p.m_tiles = (int)cdiv(a.M, C::BM);
    const int64_t tiles = p.m_tiles * cdiv(a.N, C::BN), kts = cdiv(a.K, KB);
    // K is split over a cluster while the tiles leave SMs idle
    p.parts = 1;
    while (p.parts < 8 && tiles * p.parts * 2 <= 2 * num_sms() && kts >= 4 * p.parts) p.parts *= 2;
    CUtensorMap ma, mb, msa, msb;
    const uint64_t sp = (uint64_t)cdiv(a.K, SPAN<KIND>);
    if (!map_codes(&ma, a.qa, a.M, a.K / 2, a.lda, 128) || !map_codes(&mb, a.qw, a.N, a.K / 2, a.ldw, 128) ||
        !map_scales(&msa, a.sa, cdiv(a.M, 128), sp, C::TILES, 1) || !map_scales(&msb, a.sw, cdiv(a.N, 128), sp, C::TILES, 1)) {
        *msg = "cuTensorMapEncodeTiled failed (pointer/stride alignment or driver entry point)";
        return cudaErrorInvalidValue;
    }
    static bool configured[HN_MAX_DEV];
    int dev = 0;
    e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= HN_MAX_DEV) return cudaErrorInvalidDevice;
    if (!configured[dev]) {
        e = cudaFuncSetAttribute(k_fp4_gemm<KIND>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
        if (e != cudaSuccess) return e;
        configured[dev] = true;
    }
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
    return cudaLaunchKernelEx(&cfg, k_fp4_gemm<KIND>, ma, mb, msa, msb, p);
}

} // namespace fp4g

cudaError_t launch_fp4_gemm(const Fp4GemmArgs &a, cudaStream_t st, const char **msg) {
    if (fp4_gemv_applies(a)) return launch_fp4_gemv(a, st);
    return a.kind == fp4::MX ? fp4g::launch<fp4::MX>(a, st, msg) : fp4g::launch<fp4::NV>(a, st, msg);
}

} // namespace hn
