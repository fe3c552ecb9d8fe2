// paged.cuh - what the kernels of the paged attention share: the parameters, and the line of key blocks that is cut
// into equal parts for the CTAs.
//
// A line holds the tiles of the part shared by all sequences (rows of all of them, keys [0, shared)), of the sequences' own
// keys [own_first, length), or of both. A tile is a K/V head and up to `ta` / `tb` rows; its blocks are `bk` keys each.
// The tiles' blocks follow one another: shared tiles by head and row tile, then for each sequence by head and row
// tile. CTA c of n takes blocks [c q, (c + 1) q), q = ceil(total / n): the lengths are on the device, so every CTA
// computes the cut from them, and the join computes it again. A tile inside one CTA ends there when nothing else adds to
// its rows; else each CTA's piece leaves fp32 sums, maximum and normaliser in a slot. Where whole tiles end their rows, a CTA has
// two such pieces at most, the end of a tile in slot 2 CTA and the beginning of one in 2 CTA + 1; else every piece has one,
// tile + CTA (two pieces never share it: along the line each cut raises the tile, the CTA, or both).
#pragma once
#include <cuda_fp16.h>

#include "hn_common.cuh"
#include "hn_kernels.h"

namespace hn {
namespace paged {

constexpr int HD = 128;
constexpr int MAX_B = 4096;             // sequences: their blocks' prefix sums sit in shared memory

struct Params {
    const __nv_bfloat16 *q; int64_t q_bs, q_ls, q_hs;
    __nv_bfloat16 *out; int64_t o_bs, o_ls, o_hs;
    float *lse;
    const uint8_t *k, *v;
    const float *ks, *vs;
    const int *table, *lengths, *rows;
    int slots, width, pages, page;
    int B, Lq, H, Hkv, G, shared, causal;
    float sl2;                          // |scale| * log2 e
    uint32_t flip;                      // sign bits to flip in a bf16 pair of q: a negative scale
    // the line
    int bk, ctas, min_quota;
    int nbA, nrtA, ta;                  // shared tiles: blocks, row tiles per head, rows per tile (nbA 0: not on this line)
    int has_own, nrtB, tb, own_first;   // own tiles
    int ends;                           // a whole own tile ends its rows
    int part_rows;                      // rows per slot
    float *part_o, *part_ml;            // [slots][part_rows][128], [slots][part_rows][2]
    int *sched;                         // [B + 1] prefix sums of the own blocks (of one head), written for the join
    float lse_shift;                    // the partial sums are 2^lse_shift too large
    int *err;
};

// One piece of a tile: rows [row0, row0 + its tile's), blocks [blk0, blk0 + nblk) of keys [kbeg, kend)
struct Piece {
    int own_b;          // the sequence, or -1: the shared part, rows over all sequences
    int h, row0;        // K/V head, first row
    int kbeg, kend;
    int blk0, nblk;
    int slot;           // of the partial result, or -1: the rows end here
};

__device__ __forceinline__ int seq_length(const Params &p, int b) {
    const int seq = p.rows[b];
    int len = (unsigned)seq < (unsigned)p.slots ? p.lengths[seq] : 0;
    const int most = p.width * p.page;
    len = len > most ? most : len;
    return len < 0 ? 0 : len;
}
// keys that query l of a sequence of `len` tokens sees: [0, limit)
__device__ __forceinline__ int row_limit(const Params &p, int len, int l) { return p.causal ? len - p.Lq + l + 1 : len; }

// blocks of own row tile rt: up to the last key that its last query sees
__device__ __forceinline__ int own_blocks(const Params &p, int len, int rt) {
    const int r1 = p.Lq * p.G, last = (rt + 1) * p.tb < r1 ? (rt + 1) * p.tb - 1 : r1 - 1;
    const int n = row_limit(p, len, last / p.G) - p.own_first;
    return n > 0 ? (n + p.bk - 1) / p.bk : 0;
}
// ... of all row tiles below `n_rt`
__device__ __forceinline__ int own_blocks_below(const Params &p, int len, int n_rt) {
    if (!p.causal || n_rt == 0) return n_rt ? n_rt * own_blocks(p, len, 0) : 0;
    int n = 0;
    for (int rt = 0; rt < n_rt; ++rt) n += own_blocks(p, len, rt);
    return n;
}

// pre[b] = own blocks (of one head) of the sequences before b. *lead = the sequence whose table the shared pages are looked
// up in: the first of those that hold the most of them (a listed row may be short or empty: it sees what it holds).
// `threads` threads, a multiple of 32; sums: [32] ints; lead: 8-byte aligned.
__device__ __forceinline__ void prefix_blocks(const Params &p, int *pre, int *sums, unsigned long long *lead, int threads) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int base = 0;
    if (tid == 0) *lead = 0;
    __syncthreads();
    for (int b0 = 0; b0 < p.B; b0 += threads) {
        const int len = b0 + tid < p.B ? seq_length(p, b0 + tid) : 0;
        const int n = b0 + tid < p.B && p.has_own ? own_blocks_below(p, len, p.nrtB) : 0;
        if (p.nbA && b0 + tid < p.B)
            atomicMax(lead, (unsigned long long)(len < p.shared ? len : p.shared) << 13 | (unsigned)(MAX_B - (b0 + tid)));
        int x = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) sums[warp] = x;
        __syncthreads();
        int total = 0;
        for (int i = 0; i < threads >> 5; ++i) {
            if (i == warp) x += total;
            total += sums[i];
        }
        if (b0 + tid < p.B) pre[b0 + tid] = base + x - n;
        base += total;
        __syncthreads();
    }
    if (tid == 0) {
        pre[p.B] = base;
        *lead = MAX_B - (int)(*lead & 8191);
    }
    __syncthreads();
}

// Walks the pieces of one CTA. `lead`: the sequence whose table the shared pages are looked up in; where it holds fewer than
// `shared` tokens nobody holds the rest, and the shared part ends where it does.
struct Walker {
    int64_t x, end, blocksA;
    int shared;
    __device__ __forceinline__ Walker(const Params &p, const int *pre, int lead, int cta) {
        shared = 0;
        if (p.nbA) {
            const int len = seq_length(p, lead);
            shared = len < p.shared ? len : p.shared;
        }
        blocksA = (int64_t)p.Hkv * p.nrtA * p.nbA;
        const int64_t total = blocksA + (int64_t)pre[p.B] * p.Hkv;
        const int64_t q = quota(p, total);
        x = q * cta;
        end = x + q < total ? x + q : total;
    }
    static __device__ __forceinline__ int64_t quota(const Params &p, int64_t total) {
        const int64_t q = (total + p.ctas - 1) / p.ctas;
        return q < p.min_quota ? p.min_quota : q;
    }
    __device__ bool next(const Params &p, const int *pre, int cta, Piece &w) {
        if (x >= end) return false;
        int64_t tile_end;
        int tile;
        if (x < blocksA) {
            tile = (int)(x / p.nbA);
            w.own_b = -1;
            w.h = tile / p.nrtA;
            w.row0 = (tile - w.h * p.nrtA) * p.ta;
            w.kbeg = 0; w.kend = shared;
            w.blk0 = (int)(x - (int64_t)tile * p.nbA);
            tile_end = (int64_t)(tile + 1) * p.nbA;
        } else {
            const int64_t y = x - blocksA;
            int lo = 0, hi = p.B - 1;                    // the last b with pre[b] * Hkv <= y (it has blocks)
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if ((int64_t)pre[mid] * p.Hkv <= y) lo = mid; else hi = mid - 1;
            }
            const int per_head = pre[lo + 1] - pre[lo];
            int64_t z = y - (int64_t)pre[lo] * p.Hkv;
            w.own_b = lo;
            w.h = (int)(z / per_head);
            z -= (int64_t)w.h * per_head;
            w.kbeg = p.own_first;
            w.kend = seq_length(p, lo);
            int rt = 0, nb;
            if (!p.causal) {
                nb = own_blocks(p, w.kend, 0);
                rt = (int)(z / nb);
                z -= (int64_t)rt * nb;
            } else {
                while ((nb = own_blocks(p, w.kend, rt)) <= z) { z -= nb; ++rt; }
            }
            w.row0 = rt * p.tb;
            w.blk0 = (int)z;
            tile_end = x - z + nb;
            tile = p.Hkv * p.nrtA + (lo * p.Hkv + w.h) * p.nrtB + rt;
        }
        const int64_t stop = end < tile_end ? end : tile_end;
        w.nblk = (int)(stop - x);
        const bool whole = w.blk0 == 0 && stop == tile_end && w.own_b >= 0 && p.ends;
        w.slot = whole ? -1 : p.ends ? 2 * cta + (w.blk0 == 0) : tile + cta;
        x = stop;
        return true;
    }
};

__device__ __forceinline__ void split_row(const Params &p, const Piece &w, int r, int &b, int &l, int &g) {
    const int r1 = p.Lq * p.G;
    b = w.own_b;
    if (b < 0) { b = r / r1; r -= b * r1; }
    l = r / p.G;
    g = r - l * p.G;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 1 / L of a row: 0 where nothing was seen, and a NaN stays one
__device__ __forceinline__ float inverse(float L) { return L > 0.0f ? __frcp_rn(L) : L == 0.0f ? 0.0f : L; }
__device__ __forceinline__ float row_lse(const Params &p, float M, float L) {
    return (M + lg2(L) - p.lse_shift) * 0.6931471805599453f;
}
// two biased code bytes (code + 128) of w, chosen by SEL -> two fp16 integers, exact: 0x6400 | u is 1024 + u
template <uint32_t SEL> __device__ __forceinline__ uint32_t codes_f16(uint32_t w) {
    const uint32_t u = __byte_perm(w, 0x64646464u, SEL);
    const __half2 off = __half2half2(__ushort_as_half(0x6480));       // 1152 = 1024 + 128
    __half2 x = __hsub2(*reinterpret_cast<const __half2 *>(&u), off);
    return *reinterpret_cast<uint32_t *>(&x);
}
// a power of two that brings a row of largest |q| `top` into [1, 2): 2^-e, e in [-126, 126] so that both are normal
__device__ __forceinline__ int row_exponent(float top) {
    const int e = (int)(__float_as_uint(top) >> 23) - 127;
    return e < -126 ? -126 : e > 126 ? 126 : e;
}

cudaError_t launch_tc(const Params &p, cudaStream_t st);       // the tensor-core line (paged_tc.cu); bk = 128
int tc_most_sequences();                                       // ... takes at most so many sequences

} // namespace paged
} // namespace hn
