// paged_attention.cu - attention over the paged K/V cache of sequences that share their first tokens:
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale * q_i . k_j - m_i),  j < limit_i
// limit_i = the sequence's length, or (causal) length - Lq + i + 1. A row that sees no key gives 0. With a shared part
// (the first `shared` tokens of every listed sequence are on the same pages) the rows of all sequences attend to it
// together - its K and V are read once, not once per sequence - and each sequence's rows to its own tokens; the
// two results are joined by their maxima and sums.
//
// Heads of 128, H query heads on Hkv K/V heads (H / Hkv rows per token share a head's K and V). Rows of a tile:
// (sequence,) token, group member. A tile of 16, 32 or 64 rows walks its keys in blocks of 64; the blocks of all tiles
// form one line, cut into equal parts for the CTAs, so that long and short sequences load them evenly (every CTA
// computes the cut itself from the lengths on the device). A tile that spans CTAs leaves a partial result per CTA
// (fp32 sums, maximum, normaliser), joined by k_paged_join.
//
// Bound by HBM for a token per sequence (K and V once: 2 x 256 B, int8 2 x 132 B, per key and head): 64 sequences of 1669 to 4000
// tokens (181408 in all), 8 K/V heads: bf16 126 us (743 MB, 5.9 TB/s), int8 119 us (383 MB, 3.2 TB/s: the conversion of the codes
// issues as much as the products). With 64-row tiles by the shared-memory reads of the fragments: 16 x 5 queries over 4096 shared
// and 546 to 1101 own tokens, 16 heads, bf16: 54 us and the join's 8.
// Per warp: 16 rows; m16n8k16 products, S and O in registers. The four warps split a block's keys (16-row tiles), its
// rows (64), or both (32). Blocks arrive by cp.async, STAGES deep; the smem chunks are permuted so that no read conflicts.
//  - bf16 cache: K by ldmatrix, V by its transposing form, P rounded to bf16 (both operands of a product have one type, and V's range
//    is bf16's): at most 2^-8 of the mean |v|, with the output's own rounding after it.
//  - int8 cache: codes become fp16 integers (exact: 0x6400 | (code + 128) is 1152 + code), so the scales stay outside the
//    products: x_j = (q . ck_j) * sk_j * scale + log2 sv_j (base 2), P'_j = 2^(x_j - m + 14) multiplies cv_j, and the
//    normaliser sums P'_j / sv_j. Taking the maximum over x_j keeps P' in fp16's range whatever the scales are.
//    q is brought to fp16 by a power of two per row (exact but for values 2^-24 below the row's largest).
#include <cuda_fp16.h>

#include "paged.cuh"

namespace hn {
namespace paged {

constexpr int BK = 64;                  // keys per block
constexpr int THREADS = 128;
constexpr float P_SHIFT = 14.0f;        // int8: P' <= 2^14

__device__ __forceinline__ uint32_t saddr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp16(uint32_t dst, const void *src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void *src, bool valid) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(valid ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t a) {
    uint4 r;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a) : "memory");
    return r;
}
// c += a b, 16 x 8 x 16, fp32 sums
template <bool I8>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t *a, uint32_t b0, uint32_t b1) {
    if (I8)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Bytes of one stage: K and V blocks, and the int8 scales
template <bool I8> constexpr int tile_bytes() { return BK * (I8 ? HD : 2 * HD); }
template <bool I8> constexpr int stage_bytes() { return 2 * tile_bytes<I8>() + (I8 ? 2 * BK * 4 : 0); }
template <bool I8> constexpr int stages() { return I8 ? 4 : 3; }
// the ring also holds the four warps' sums when a tile ends (4 x 16 rows x 128 fp32 + maxima and normalisers)
constexpr int END_BYTES = 4 * 16 * HD * 4 + 4 * 16 * 2 * 4;
template <bool I8> constexpr int smem_bytes() {
    return stages<I8>() * stage_bytes<I8>() > END_BYTES ? stages<I8>() * stage_bytes<I8>() : END_BYTES;
}

template <bool I8, int RG> __device__ void run_piece(const Params &p, const Piece &w, int lead, uint8_t *smem) {
    constexpr int KG = 4 / RG, KW = BK / KG, NT = KW / 8;        // key groups, keys and 8-key tiles per warp and block
    constexpr int ST = stages<I8>(), TILE = tile_bytes<I8>(), STAGE = stage_bytes<I8>();
    constexpr int CPR = I8 ? 8 : 16;                             // 16-byte chunks per row
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rg = warp % RG, kg = warp / RG, gid = lane >> 2, tq = lane & 3;
    const uint32_t sb = saddr(smem);
    const int rows = w.own_b < 0 ? p.B * p.Lq * p.G : p.Lq * p.G;

    // --- loader: block i of the piece into stage i % ST. A thread's chunks of step `it` are all in 16-key group
    // it * (128 / CPR) / 16, which lies in one page (pages and the parts' first keys are multiples of 16 tokens).
    const int seq = p.rows[w.own_b < 0 ? lead : w.own_b];
    const int *tab = p.table + (int64_t)((unsigned)seq < (unsigned)p.slots ? seq : 0) * p.width;
    constexpr int RPI = THREADS / CPR;                           // rows per step: 8 (bf16), 16 (int8)
    // The page and the place in it of the next block's four groups. The table is read a block ahead, so that no warp waits
    // for it, and the place moves on by addition (a division per group took a fifth of the loader's instructions).
    int id[4], off[4], pg = (w.kbeg + w.blk0 * BK) / p.page, at = w.kbeg + w.blk0 * BK - pg * p.page, key = w.kbeg + w.blk0 * BK;
    auto look_up = [&]() {
#pragma unroll
        for (int sub = 0; sub < 4; ++sub) {
            id[sub] = key < w.kend && pg < p.width ? tab[pg] : -1;
            off[sub] = at;
            key += 16;
            at += 16;
            if (at == p.page) { at = 0; ++pg; }
        }
    };
    look_up();
    auto load = [&](int i) {
        if (i < w.nblk) {
            const uint32_t st = sb + (uint32_t)(i % ST) * STAGE;
            const int left = w.kend - (w.kbeg + (w.blk0 + i) * BK);     // keys of the block that are there
#pragma unroll
            for (int sub = 0; sub < 4; ++sub) {
                const bool there = (unsigned)id[sub] < (unsigned)p.pages;
                const int64_t tok = there ? ((int64_t)id[sub] * p.Hkv + w.h) * p.page + off[sub] : 0;
#pragma unroll
                for (int it = 0; it < 16 / RPI; ++it) {
                    const int r = it * RPI + tid / CPR, c = tid % CPR, row = 16 * sub + r;
                    const bool ok = there && row < left;
                    const int64_t src = ok ? (tok + r) * (CPR * 16) + c * 16 : 0;
                    const int ck = I8 ? c ^ ((row & 1) << 2) : c ^ (row & 7);
                    const int cv = I8 ? c ^ (((row >> 1) & 3) << 1) : c ^ (row & 7);
                    cp16(st + row * (CPR * 16) + ck * 16, p.k + src, ok);
                    cp16(st + TILE + row * (CPR * 16) + cv * 16, p.v + src, ok);
                }
                if (I8 && tid < 32) {
                    const int r = tid & 15;
                    const bool ok = there && 16 * sub + r < left;
                    const float *sc = tid < 16 ? p.ks : p.vs;
                    cp4(st + 2 * TILE + (tid < 16 ? 0 : BK * 4) + (16 * sub + r) * 4, sc + (ok ? tok + r : 0), ok);
                }
            }
            look_up();
        }
        cp_commit();
    };
    for (int i = 0; i < ST - 1; ++i) load(i);       // on their way while q is read

    // --- the two rows of this lane: their key limits and q
    int lim[2];
    float rowscale[2];
    uint32_t qf[8][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = w.row0 + 16 * rg + gid + 8 * i;
        lim[i] = w.kend;                        // a row past the tile's end: q = 0, computed and dropped
        const __nv_bfloat16 *qp = p.q;
        const bool valid = r < rows;
        if (valid) {
            int b, l, g;
            split_row(p, w, r, b, l, g);
            lim[i] = row_limit(p, seq_length(p, b), l);
            if (lim[i] > w.kend) lim[i] = w.kend;
            qp += b * p.q_bs + l * p.q_ls + (int64_t)(w.h * p.G + g) * p.q_hs;
        }
        rowscale[i] = p.sl2;
        if (!I8) {
#pragma unroll
            for (int s = 0; s < 8; ++s) {
                qf[s][i] = valid ? *reinterpret_cast<const uint32_t *>(qp + 16 * s + 2 * tq) ^ p.flip : 0u;
                qf[s][2 + i] = valid ? *reinterpret_cast<const uint32_t *>(qp + 16 * s + 8 + 2 * tq) ^ p.flip : 0u;
            }
        } else {
            // k-step s, element j of this lane's four: d = 64 (s / 4) + 16 tq + 4 (s % 4) + j, on both operands
            uint32_t raw[16];
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    uint4 x = make_uint4(0, 0, 0, 0);
                    if (valid) x = *reinterpret_cast<const uint4 *>(qp + 64 * c + 16 * tq + 8 * u);
                    raw[8 * c + 4 * u] = x.x ^ p.flip; raw[8 * c + 4 * u + 1] = x.y ^ p.flip;
                    raw[8 * c + 4 * u + 2] = x.z ^ p.flip; raw[8 * c + 4 * u + 3] = x.w ^ p.flip;
                }
            float top = 0.0f;
#pragma unroll
            for (int j = 0; j < 16; ++j) top = fmaxf(top, fmaxf(fabsf(bf16_lo(raw[j])), fabsf(bf16_hi(raw[j]))));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int e = row_exponent(top);
            const float down = pow2i(-e);
            rowscale[i] *= pow2i(e);
#pragma unroll
            for (int s = 0; s < 8; ++s) {
                const uint32_t x0 = raw[2 * s], x1 = raw[2 * s + 1];
                qf[s][i] = pack_f16_rn(bf16_lo(x0) * down, bf16_hi(x0) * down);
                qf[s][2 + i] = pack_f16_rn(bf16_lo(x1) * down, bf16_hi(x1) * down);
            }
        }
    }
    int minlim = lim[0] < lim[1] ? lim[0] : lim[1];
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
        const int y = __shfl_xor_sync(0xffffffffu, minlim, o);
        minlim = y < minlim ? y : minlim;
    }

    float o[16][4];
#pragma unroll
    for (int j = 0; j < 16; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

    for (int i = 0; i < w.nblk; ++i) {
        cp_wait<ST - 2>();
        __syncthreads();                        // block i is here, and every warp is done with block i - 1
        load(i + ST - 1);
        const uint32_t st = sb + (uint32_t)(i % ST) * STAGE;
        const int kw = kg * KW;                 // this warp's keys in the block
        const int key0 = w.kbeg + (w.blk0 + i) * BK + kw;

        // --- S = Q K^T
        float s[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
        if (!I8) {
#pragma unroll
            for (int n = 0; n < NT; n += 2)
#pragma unroll
                for (int ks = 0; ks < 8; ++ks) {
                    uint32_t b[4];
                    const int row = kw + 8 * n + ((lane >> 4) << 3) + (lane & 7), c = 2 * ks + ((lane >> 3) & 1);
                    ldsm4(b, st + row * 256 + ((c ^ (row & 7)) << 4));
                    mma<I8>(s[n], qf[ks], b[0], b[1]);
                    mma<I8>(s[n + 1], qf[ks], b[2], b[3]);
                }
        } else {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int row = kw + 8 * n + gid;
                    const uint4 x = lds16(st + row * 128 + (((4 * c + tq) ^ ((row & 1) << 2)) << 4));
                    const uint32_t xs[4] = {x.x ^ 0x80808080u, x.y ^ 0x80808080u, x.z ^ 0x80808080u, x.w ^ 0x80808080u};
#pragma unroll
                    for (int u = 0; u < 4; ++u)
                        mma<I8>(s[n], qf[4 * c + u], codes_f16<0x4140>(xs[u]), codes_f16<0x4342>(xs[u]));
                }
        }

        // --- base-2 logits, masked; running maximum
        float inv[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            if (I8) {
                const float *sc = reinterpret_cast<const float *>(smem + (i % ST) * STAGE + 2 * TILE) + kw + 8 * n + 2 * tq;
                const float2 sk = *reinterpret_cast<const float2 *>(sc);
                float2 sv = *reinterpret_cast<const float2 *>(sc + BK);
                // a scale below 2^-100 (an all but zero row) counts as 2^-100: its values then are below 2^-93
                sv.x = sv.x < 0x1p-100f ? 0x1p-100f : sv.x;
                sv.y = sv.y < 0x1p-100f ? 0x1p-100f : sv.y;
                // (the reciprocal of a NaN is one of a number: the rows that see the key have the NaN in their logit, the others none)
                inv[n][0] = rcp(fmaxf(sv.x, 0x1p-100f));
                inv[n][1] = rcp(fmaxf(sv.y, 0x1p-100f));
                const float l0 = lg2(sv.x), l1 = lg2(sv.y);
                s[n][0] = fmaf(s[n][0], sk.x * rowscale[0], l0);
                s[n][1] = fmaf(s[n][1], sk.y * rowscale[0], l1);
                s[n][2] = fmaf(s[n][2], sk.x * rowscale[1], l0);
                s[n][3] = fmaf(s[n][3], sk.y * rowscale[1], l1);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) s[n][e] *= rowscale[e >> 1];
            }
        }
        if (key0 + KW > minlim) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (key0 + 8 * n + 2 * tq + (e & 1) >= lim[e >> 1]) s[n][e] = -INFINITY;
        }
        float al[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            float top = -INFINITY;
#pragma unroll
            for (int n = 0; n < NT; ++n) top = fmaxf(top, fmaxf(s[n][2 * r], s[n][2 * r + 1]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float mn = fmaxf(m[r], top), ref = mn == -INFINITY ? 0.0f : mn;
            al[r] = ex2(m[r] - ref);
            m[r] = mn;
            const float sub = I8 ? ref - P_SHIFT : ref;
            float sum = 0.0f;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float x = ex2(s[n][2 * r + e] - sub);
                    s[n][2 * r + e] = x;
                    sum = I8 ? fmaf(x, inv[n][e], sum) : sum + x;
                }
            l[r] = fmaf(l[r], al[r], sum);
        }
        if (__any_sync(0xffffffffu, al[0] != 1.0f || al[1] != 1.0f)) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                o[j][0] *= al[0]; o[j][1] *= al[0];
                o[j][2] *= al[1]; o[j][3] *= al[1];
            }
        }

        // --- O += P V, 16 keys at a time
#pragma unroll
        for (int n = 0; n < NT; n += 2) {
            uint32_t a[4];
            if (I8) {
                a[0] = pack_f16_rn(s[n][0], s[n][1]); a[1] = pack_f16_rn(s[n][2], s[n][3]);
                a[2] = pack_f16_rn(s[n + 1][0], s[n + 1][1]); a[3] = pack_f16_rn(s[n + 1][2], s[n + 1][3]);
            } else {
                a[0] = bf16x2_rn(s[n][0], s[n][1]); a[1] = bf16x2_rn(s[n][2], s[n][3]);
                a[2] = bf16x2_rn(s[n + 1][0], s[n + 1][1]); a[3] = bf16x2_rn(s[n + 1][2], s[n + 1][3]);
            }
            const uint32_t vt = st + TILE;
            const int kr = kw + 8 * n;
            if (!I8) {
#pragma unroll
                for (int j = 0; j < 16; j += 2) {
                    uint32_t b[4];
                    const int row = kr + (lane & 15), c = j + (lane >> 4);
                    ldsm4t(b, vt + row * 256 + ((c ^ (row & 7)) << 4));
                    mma<I8>(o[j], a, b[0], b[1]);
                    mma<I8>(o[j + 1], a, b[2], b[3]);
                }
            } else {
                // rows 2 tq, 2 tq + 1, 8 + 2 tq, 9 + 2 tq of the 16; chunk gid: n index gid of tile j is d = 16 gid + j
                uint32_t x[4][4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int row = kr + 8 * (u >> 1) + 2 * tq + (u & 1);
                    const uint4 y = lds16(vt + row * 128 + ((gid ^ (((row >> 1) & 3) << 1)) << 4));
                    x[u][0] = y.x ^ 0x80808080u; x[u][1] = y.y ^ 0x80808080u;
                    x[u][2] = y.z ^ 0x80808080u; x[u][3] = y.w ^ 0x80808080u;
                }
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const uint32_t lo0 = __byte_perm(x[0][c], x[1][c], 0x5140), hi0 = __byte_perm(x[0][c], x[1][c], 0x7362);
                    const uint32_t lo1 = __byte_perm(x[2][c], x[3][c], 0x5140), hi1 = __byte_perm(x[2][c], x[3][c], 0x7362);
                    mma<I8>(o[4 * c], a, codes_f16<0x4140>(lo0), codes_f16<0x4140>(lo1));
                    mma<I8>(o[4 * c + 1], a, codes_f16<0x4342>(lo0), codes_f16<0x4342>(lo1));
                    mma<I8>(o[4 * c + 2], a, codes_f16<0x4140>(hi0), codes_f16<0x4140>(hi1));
                    mma<I8>(o[4 * c + 3], a, codes_f16<0x4342>(hi0), codes_f16<0x4342>(hi1));
                }
            }
        }
    }
    cp_wait<0>();
    __syncthreads();

    // --- the warps' sums through shared memory, joined over the key groups
    float *so = reinterpret_cast<float *>(smem), *sm = so + 4 * 16 * HD;     // [warp][16][128], [warp][16][2]
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        const int row = 16 * warp + gid + 8 * r;
        if (tq == 0) { sm[2 * row] = m[r]; sm[2 * row + 1] = l[r]; }
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            if (I8) {
                so[row * HD + 32 * tq + j] = o[j][2 * r];
                so[row * HD + 32 * tq + 16 + j] = o[j][2 * r + 1];
            } else {
                so[row * HD + 8 * j + 2 * tq] = o[j][2 * r];
                so[row * HD + 8 * j + 2 * tq + 1] = o[j][2 * r + 1];
            }
        }
    }
    __syncthreads();
    // each warp finishes RG * 16 / 4 rows, 4 values per lane
    for (int rr = warp; rr < 16 * RG; rr += 4) {
        const int r = w.row0 + rr;
        if (r >= rows) break;
        float M = -INFINITY;
#pragma unroll
        for (int g = 0; g < KG; ++g) M = fmaxf(M, sm[2 * ((g * RG + rr / 16) * 16 + rr % 16)]);
        const float ref = M == -INFINITY ? 0.0f : M;
        float L = 0.0f;
        float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int g = 0; g < KG; ++g) {
            const int row = (g * RG + rr / 16) * 16 + rr % 16;
            const float f = ex2(sm[2 * row] - ref);
            const float4 x = *reinterpret_cast<const float4 *>(so + row * HD + 4 * lane);
            L = fmaf(f, sm[2 * row + 1], L);
            acc.x = fmaf(f, x.x, acc.x); acc.y = fmaf(f, x.y, acc.y);
            acc.z = fmaf(f, x.z, acc.z); acc.w = fmaf(f, x.w, acc.w);
        }
        if (w.slot >= 0) {
            const int64_t at = (int64_t)w.slot * p.part_rows + rr;
            *reinterpret_cast<float4 *>(p.part_o + at * HD + 4 * lane) = acc;
            if (lane == 0) *reinterpret_cast<float2 *>(p.part_ml + 2 * at) = make_float2(M, L);
        } else {
            int b, ll, g;
            split_row(p, w, r, b, ll, g);
            const int head = w.h * p.G + g;
            const float inv = inverse(L);
            uint2 y;
            y.x = bf16x2_rn(acc.x * inv, acc.y * inv);
            y.y = bf16x2_rn(acc.z * inv, acc.w * inv);
            *reinterpret_cast<uint2 *>(p.out + b * p.o_bs + ll * p.o_ls + head * p.o_hs + 4 * lane) = y;
            if (p.lse != nullptr && lane == 0)
                p.lse[((int64_t)b * p.H + head) * p.Lq + ll] = row_lse(p, M, L);
        }
    }
    __syncthreads();                        // the ring is free for the next piece
}

template <bool I8> __global__ void __launch_bounds__(THREADS, I8 ? 3 : 2) k_paged_attention(const Params p) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int sums[32];
    __shared__ unsigned long long lead;
    int *pre = reinterpret_cast<int *>(smem + smem_bytes<I8>());
    dep_launch();
    prefix_blocks(p, pre, sums, &lead, THREADS);
    if (blockIdx.x == 0)
        for (int b = threadIdx.x; b <= p.B; b += THREADS) p.sched[b] = pre[b];
    Walker walk(p, pre, (int)lead, blockIdx.x);
    Piece w;
    while (walk.next(p, pre, blockIdx.x, w)) {
        const int rows_per = w.own_b < 0 ? p.ta : p.tb;
        if (rows_per == 16) run_piece<I8, 1>(p, w, (int)lead, smem);
        else if (rows_per == 32) run_piece<I8, 2>(p, w, (int)lead, smem);
        else run_piece<I8, 4>(p, w, (int)lead, smem);
    }
    dep_wait();             // nothing here reads what the other line writes, but the join waits for this kernel only
}

// Joins the partial results of every row: out = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i. A warp takes RUN rows of a tile,
// one after the other. `a` is the line that holds the shared part (nbA 0: there is none), `b` the one that holds the own parts.
// 140800 rows of which a quarter are cut: 46 us (each row looked up in the line: 105); small calls: 5-10 us, of latency. Two CTAs an
// SM: for three ptxas spills.
template <int RUN> __global__ void __launch_bounds__(256, 2) k_paged_join(const Params a, const Params b) {
    dep_wait();
    const int lane = threadIdx.x & 31;
    const int rows = b.Lq * b.G, runs = (rows + RUN - 1) / RUN;      // of a sequence and K/V head
    const int64_t items = (int64_t)b.B * b.Hkv * runs;
    const int64_t blocksA = (int64_t)a.Hkv * a.nrtA * a.nbA, aheadB = (int64_t)b.Hkv * b.nrtA * b.nbA;
    const int64_t qA = a.nbA ? Walker::quota(a, blocksA + (int64_t)a.sched[a.B] * a.Hkv) : 1;
    const int64_t qB = Walker::quota(b, aheadB + (int64_t)b.sched[b.B] * b.Hkv);
    for (int64_t it = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); it < items; it += (int64_t)gridDim.x * 8) {
        const int64_t sh = div_nonneg(it, runs);
        const int s = (int)div_nonneg(sh, b.Hkv), h = (int)(sh - (int64_t)s * b.Hkv), r0 = (int)(it - sh * runs) * RUN;
        const int r1 = RUN == 1 || r0 + RUN < rows ? r0 + RUN : rows;
        // the own part's pieces, the same for the run's rows
        const int len = seq_length(b, s), rt = r0 / b.tb, nb = own_blocks(b, len, rt);
        const int64_t first = aheadB + (int64_t)b.sched[s] * b.Hkv +
                              (int64_t)h * (b.sched[s + 1] - b.sched[s]) + own_blocks_below(b, len, rt);
        const int own0 = nb > 0 ? (int)(first / qB) : 0, own1 = nb > 0 ? (int)((first + nb - 1) / qB) : -1;
        if (b.ends && own0 == own1) continue;   // the rows ended in their CTA
        for (int r = r0; r < r1; ++r) {
            float M = -INFINITY, L = 0.0f;
            float4 acc = make_float4(0, 0, 0, 0);
            // n pieces `step` rows apart from `at` (the first `off` further), eight at a time: their loads go out together
            auto add = [&](const Params &p, int64_t at, int64_t step, int n, int64_t off) {
                for (int i0 = 0; i0 < n; i0 += 8) {
                    float2 ml[8];
                    float4 x[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        ml[i] = make_float2(-INFINITY, 0.0f);
                        x[i] = make_float4(0, 0, 0, 0);
                        if (i0 + i < n) {
                            const int64_t row = at + (i0 + i) * step + (i == 0 && i0 == 0 ? off : 0);
                            ml[i] = *reinterpret_cast<const float2 *>(p.part_ml + 2 * row);
                            x[i] = *reinterpret_cast<const float4 *>(p.part_o + row * HD + 4 * lane);
                        }
                    }
                    float mn = M;
#pragma unroll
                    for (int i = 0; i < 8; ++i) mn = fmaxf(mn, ml[i].x);
                    const float ref = mn == -INFINITY ? 0.0f : mn, f0 = ex2(M - ref);
                    M = mn;
                    L *= f0;
                    acc.x *= f0; acc.y *= f0; acc.z *= f0; acc.w *= f0;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float f = ex2(ml[i].x - ref);
                        L = fmaf(f, ml[i].y, L);
                        acc.x = fmaf(f, x[i].x, acc.x); acc.y = fmaf(f, x[i].y, acc.y);
                        acc.z = fmaf(f, x[i].z, acc.z); acc.w = fmaf(f, x[i].w, acc.w);
                    }
                }
            };
            if (a.nbA) {
                const int64_t ra = (int64_t)s * rows + r;
                const int tile = h * a.nrtA + (int)(ra / a.ta);
                const int64_t at = (int64_t)tile * a.nbA;
                const int c0 = (int)(at / qA), c1 = (int)((at + a.nbA - 1) / qA);
                add(a, (int64_t)(tile + c0) * a.part_rows + (ra - (int64_t)(tile - h * a.nrtA) * a.ta), a.part_rows, c1 - c0 + 1, 0);
            }
            if (nb > 0) {
                const int slot = b.ends ? 2 * own0 : b.Hkv * b.nrtA + (s * b.Hkv + h) * b.nrtB + rt + own0;
                add(b, (int64_t)slot * b.part_rows + (r - rt * b.tb), b.ends ? 2 * b.part_rows : b.part_rows, own1 - own0 + 1,
                    b.ends ? b.part_rows : 0);
            }
            const int l = r / b.G, head = h * b.G + r - l * b.G;
            const float inv = inverse(L);
            uint2 y;
            y.x = bf16x2_rn(acc.x * inv, acc.y * inv);
            y.y = bf16x2_rn(acc.z * inv, acc.w * inv);
            *reinterpret_cast<uint2 *>(b.out + s * b.o_bs + l * b.o_ls + head * b.o_hs + 4 * lane) = y;
            if (b.lse != nullptr && lane == 0) b.lse[((int64_t)s * b.H + head) * b.Lq + l] = row_lse(b, M, L);
        }
    }
}

static int tile_rows(int64_t rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : 64; }
// CTAs of the streaming kernel: what fits an SM by shared memory (bf16 98 KB -> 2, int8 70 KB -> 3), times the SMs
static int stream_ctas(bool i8) { return num_sms() * (i8 ? 3 : 2); }
// Which line takes a part. A tile of the tensor cores is two groups of 128 rows over the same keys, and its launch and first blocks
// are dearer; a tile of this line is 64 rows, and every tile reads the keys' fragments again. What counts for a shared part is
// therefore K/V heads x tokens x tiles of 64 rows, from 65 rows on (up to 64 the keys go by once, at HBM's rate). Measured, us, here /
// tensor cores, bf16 and int8, own parts of 33 to 64 tokens (of 257 to 512):
//   64K   8 heads x  4096, 128 rows    35 / 42 (41 / 47)   40 / 54 (50 / 57)      8 x 1024, 512 rows   48 / 57 (85 / 93)    56 / 67 (98 / 101)
//   128K  8 heads x  8192, 128 rows    46 / 48 (50 / 55)   56 / 60 (61 / 64)      8 x 4096, 256 rows   50 / 46 (62 / 70)    57 / 57 (76 / 72)
//   192K  8 heads x 12288, 128 rows    63 / 52 (60 / 62)   68 / 67 (71 / 70)     16 x 6144,  68 rows   60 / 50 (56 / 64)    67 / 65 (71 / 69)
//   256K  8 heads x 16384, 128 rows    81 / 56 (67 / 69)   81 / 71 (85 / 77)      8 x 4096, 512 rows   93 / 63 (106 / 99)   98 / 75 (128 / 110)
//         1 head x 131072, 128 rows    84 / 68 (64 / 71)   95 / 83 (85 / 83)      4 x 32768, 68 rows   77 / 55 (55 / 56)    83 / 70 (73 / 68)
//   and far below: 1 head x 512, 136 rows 18 / 28, 19 / 34. Longer own parts move the balance to this line: they run beside the shared
//   part here, after it there.
// Own parts from 65 rows on: 2000 tokens, 8 sequences, 16 heads, 100 rows 97 / 82 and 122 / 94.
constexpr int64_t TC_SHARED_WORK = 3 << 16;
constexpr int TC_ROWS = 65;

struct Plan {
    bool shared_tc, own_tc;             // which line holds which part
    int64_t stream_slots, tc_slots;
    int64_t bytes;
    size_t tc_at, sched_at;             // byte offsets in the workspace: the second line's partials, the prefix sums
};

// The two lines of a call: `s` (this file's kernel) and `t` (paged_tc.cu). A sequence with TC_ROWS rows per K/V head or
// more walks all of its keys on the tensor-core line, the shared ones too, in tiles of its own (a tile of 256 rows is bound by its
// products, and the shared pages come from L2; with fewer rows a tile is that much emptier). Else the rows of all sequences attend
// to the shared part together, on the tensor cores if it is TC_SHARED_WORK, and the own parts stream.
static Plan plan(const PagedAttnArgs &a, Params &s, Params &t) {
    Plan pl;
    const bool i8 = a.cache.ks != nullptr;
    s.B = a.B; s.Lq = a.Lq; s.H = a.H; s.Hkv = a.cache.heads; s.G = a.H / a.cache.heads;
    s.shared = a.shared; s.causal = a.causal;
    s.nbA = s.nrtA = 0; s.ta = 16;
    s.has_own = 0; s.nrtB = 0; s.tb = 16; s.own_first = 0;
    // two blocks a CTA at least (four: 31.7 -> 35.7 us for 256 rows over 4096 keys, 8 heads; the rest within 2%)
    s.ends = 0; s.min_quota = 2;
    t = s;
    const int64_t r1 = (int64_t)a.Lq * s.G, all = r1 * a.B;
    const bool fits = a.B <= tc_most_sequences();
    pl.own_tc = fits && r1 >= TC_ROWS;
    // one sequence has nothing to share
    const bool split = a.shared > 0 && a.B > 1 && !pl.own_tc;
    pl.shared_tc = fits && split && all >= TC_ROWS && s.Hkv * (int64_t)a.shared * cdiv(all, 64) >= TC_SHARED_WORK;
    s.bk = BK; s.ctas = stream_ctas(i8);
    t.bk = 128; t.ctas = num_sms();
    Params &own = pl.own_tc ? t : s;
    own.has_own = 1;
    own.own_first = split ? a.shared : 0;
    own.ends = !split;
    own.tb = pl.own_tc ? 256 : tile_rows(r1);
    own.nrtB = (int)cdiv(r1, own.tb);
    if (split) {
        Params &sh = pl.shared_tc ? t : s;
        sh.nbA = (int)cdiv(a.shared, sh.bk);
        sh.ta = pl.shared_tc ? 256 : tile_rows(all);
        sh.nrtA = (int)cdiv(all, sh.ta);
    }
    auto slots = [&](Params &p) -> int64_t {
        p.part_rows = p.bk == 128 ? 256 : p.ta > p.tb ? p.ta : p.tb;
        const int64_t tiles = (int64_t)p.Hkv * p.nrtA + (int64_t)p.B * p.Hkv * p.nrtB;
        return !tiles ? 0 : p.ends ? 2 * p.ctas : tiles + p.ctas;
    };
    pl.stream_slots = slots(s);
    pl.tc_slots = slots(t);
    const int64_t row = (HD + 2) * 4;
    pl.tc_at = (size_t)(pl.stream_slots * s.part_rows * row);
    pl.sched_at = pl.tc_at + (size_t)(pl.tc_slots * t.part_rows * row);
    pl.bytes = (int64_t)pl.sched_at + 2 * ((int64_t)a.B + 1) * 4;
    return pl;
}

} // namespace paged

int64_t paged_attention_ws(const PagedAttnArgs &a) {
    paged::Params s, t;
    return paged::plan(a, s, t).bytes;
}

cudaError_t launch_paged_attention(const PagedAttnArgs &a, cudaStream_t st) {
    using namespace paged;
    Params s, t;
    const Plan pl = plan(a, s, t);
    const bool i8 = a.cache.ks != nullptr;
    int *err = nullptr;
    cudaError_t e = device_error_word(err_slot(st), &err);
    if (e != cudaSuccess) return e;
    for (Params *p : {&s, &t}) {
        p->q = static_cast<const __nv_bfloat16 *>(a.q); p->q_bs = a.q_bs; p->q_ls = a.q_ls; p->q_hs = a.q_hs;
        p->out = static_cast<__nv_bfloat16 *>(a.out); p->o_bs = a.o_bs; p->o_ls = a.o_ls; p->o_hs = a.o_hs;
        p->lse = a.lse;
        p->k = static_cast<const uint8_t *>(a.cache.k); p->v = static_cast<const uint8_t *>(a.cache.v);
        p->ks = a.cache.ks; p->vs = a.cache.vs;
        p->table = a.cache.meta.table; p->lengths = a.cache.meta.lengths; p->rows = a.rows;
        p->slots = a.cache.meta.slots; p->width = a.cache.meta.width; p->pages = a.cache.meta.pages;
        p->page = a.cache.meta.page;
        p->sl2 = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1e-37f);      // (a zero would make NaN of a masked -inf)
        p->flip = a.scale < 0.0f ? 0x80008000u : 0u;
        p->lse_shift = i8 ? P_SHIFT : 0.0f;
        p->err = err;
    }
    char *ws = static_cast<char *>(a.ws);
    s.part_o = reinterpret_cast<float *>(ws);
    s.part_ml = s.part_o + pl.stream_slots * s.part_rows * HD;
    t.part_o = reinterpret_cast<float *>(ws + pl.tc_at);
    t.part_ml = t.part_o + pl.tc_slots * t.part_rows * HD;
    s.sched = reinterpret_cast<int *>(ws + pl.sched_at);
    t.sched = s.sched + a.B + 1;
    if (pl.tc_slots) {
        e = launch_tc(t, st);
        if (e != cudaSuccess) return e;
    }
    if (pl.stream_slots) {
        const int smem = (i8 ? smem_bytes<true>() : smem_bytes<false>()) + (a.B + 1) * 4;
        static bool configured[HN_MAX_DEV];
        int dev = 0;
        e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return e;
        if (dev < 0 || dev >= HN_MAX_DEV) return cudaErrorInvalidDevice;
        if (!configured[dev]) {
            const int extra = (MAX_B + 1) * 4;
            e = cudaFuncSetAttribute(k_paged_attention<true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     smem_bytes<true>() + extra);
            if (e == cudaSuccess)
                e = cudaFuncSetAttribute(k_paged_attention<false>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         smem_bytes<false>() + extra);
            if (e != cudaSuccess) return e;
            configured[dev] = true;
        }
        const auto kernel = i8 ? k_paged_attention<true> : k_paged_attention<false>;
        if (pl.tc_slots) {
            e = launch_after(kernel, s.ctas, THREADS, smem, st, s);
        } else {
            kernel<<<s.ctas, THREADS, smem, st>>>(s);
            e = cudaGetLastError();
        }
        if (e != cudaSuccess) return e;
    }
    // a row a warp while that fills the GPU no more than twice; else 8 neighbouring rows (tiles are multiples of 16), whose place
    // in the line is looked up once
    const int64_t rows = (int64_t)a.B * a.Lq * a.H;
    const int run = rows <= (int64_t)num_sms() * 128 ? 1 : 8;
    int64_t grid = cdiv((int64_t)a.B * s.Hkv * cdiv((int64_t)a.Lq * s.G, run), 8);
    if (grid > (int64_t)num_sms() * 8) grid = (int64_t)num_sms() * 8;
    const bool tc_a = pl.shared_tc, tc_b = pl.own_tc;
    return launch_after(run == 1 ? k_paged_join<1> : k_paged_join<8>, (unsigned)grid, 256, 0, st, tc_a ? t : s, tc_b ? t : s);
}

} // namespace hn
