// rotary.cu - per-head RMSNorm and the rotation by position: in one pass over the heads, and on the way into the paged cache.
//
//   y = R(t) (x / sqrt(mean x^2 + eps) * w),  R(t): pairs of columns turned by t f_i, times the scaling's attention factor
//
// in fp32 from the loads to the one rounding. The first `rot` columns of a head are rotated, the others pass.
//
// Bound by HBM: each head read once and written once. A warp takes one token and several of its heads: cos and sin of the
// token's pairs are computed once, by all lanes, and shared through shared memory; the next heads are on their way while these
// are turned. Heads and rotated parts of a multiple of 16: sixteen columns a lane, chosen so that whole pairs are a lane's own,
// on packed arithmetic (20240 tokens x 32 heads of 128, bf16, with the norm: 58 us, 5.7 TB/s; one token: 2.5 us). Others: eight
// columns a lane, and in the half layout, whose partner stands in another lane, possibly from the middle of its columns on, the
// partners are loaded again, from L1 (128 with 120 rotated: 82 us, interleaved 75; 136 columns, 17 of 32 lanes at work: 142 and 127).
#include "hn_kernels.h"
#include "rotary.cuh"

namespace hn {
namespace rotary {

constexpr int WARPS = 4, CTAS = 4;           // of a block; blocks an SM
constexpr int AWARPS = 8, ACTAS = 2;         // the append's

struct Params {
    const void *x;
    int64_t x_bs, x_ls, x_hs;
    void *out;
    int64_t o_bs, o_ls, o_hs;
    const void *pos;                    // int32 or int64
    int64_t p_bs, p_ls;
    int wide;
    const void *w;                      // bf16, fp32 with w_wide, or null
    int w_wide;
    Rotation r;
    float eps;
    int B, L, H, D, per, groups;        // per: heads of a unit, a multiple of 32 / P; groups: units of a token
};

// Any head and rotated part: eight columns a lane
template <typename E, int P, bool INTER, bool NORM> __global__ void __launch_bounds__(32 * WARPS, CTAS) k_rotate8(Params p) {
    __shared__ float tables[WARPS][2 * MAX_PAIRS];
    constexpr int HEADS = 32 / P, U = 2;
    const int lane = threadIdx.x & 31, sub = lane % P;
    float *table = tables[threadIdx.x >> 5];
    const bool in = 8 * sub < p.D;
    Turn t;
    partners(p.r, sub, t);
    Weights w;
    if (NORM && in) load_weights(p.w, p.w_wide, 8 * sub, t, w);
    const float rd = 1.0f / p.D;
    const int64_t units = (int64_t)p.B * p.L * p.groups, step = (int64_t)gridDim.x * WARPS;
    for (int64_t u = (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5); u < units; u += step) {
        const int64_t token = div_nonneg(u, p.groups);
        const int first = (int)(u - token * p.groups) * p.per, last = first + p.per < p.H ? first + p.per : p.H;
        const int64_t b = div_nonneg(token, p.L), l = token - b * p.L;
        const E *x = static_cast<const E *>(p.x) + b * p.x_bs + l * p.x_ls + 8 * sub;
        E *out = static_cast<E *>(p.out) + b * p.o_bs + l * p.o_ls + 8 * sub;
        Raw8<E> raw[U];
        Raw4<E> far[U][2];                      // the partners of the lane's two runs of four (half layout)
        auto fetch = [&](int h0) {
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const int h = h0 + i * HEADS;
                raw[i].clear();
                if (in && h < last) {
                    const E *head = x + h * p.x_hs;
                    raw[i].load(head);
                    if (!INTER)
#pragma unroll
                        for (int j = 0; j < 2; ++j)
                            if (t.off[j] != 0) far[i][j].load(head + 4 * j + t.off[j]);
                }
            }
        };
        fetch(first + lane / P);                // before the table: the loads do not depend on it
        const int64_t at = b * p.p_bs + l * p.p_ls;
        turn_table(p.r, p.wide ? static_cast<const int64_t *>(p.pos)[at] : static_cast<const int32_t *>(p.pos)[at], table, lane);
        turn_of(p.r, sub, table, t);
        for (int h0 = first + lane / P; h0 - lane / P < last; h0 += U * HEADS) {
            Raw8<E> now[U];
            Raw4<E> other[U][2];
#pragma unroll
            for (int i = 0; i < U; ++i) {
                now[i] = raw[i];
                if (!INTER) { other[i][0] = far[i][0]; other[i][1] = far[i][1]; }
            }
            // the next heads' loads; out may be x, whose heads are each read, partners and all, before they are written
            if (h0 - lane / P + U * HEADS < last) fetch(h0 + U * HEADS);
            __syncwarp();
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const int h = h0 + i * HEADS;
                float v[8], o[8];
                now[i].widen(v);
                if (!INTER)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        if (t.off[j] != 0) other[i][j].widen(o + 4 * j);
                if (NORM) head_norm<P>(v, o, w, t, rd, p.eps);
                turn<INTER>(t, v, o);
                if (in && h < last) store8(out + h * p.o_hs, v);
            }
        }
    }
}

// heads and rotated parts of a multiple of 16: sixteen columns a lane
template <typename E, int P, bool INTER, bool NORM> __global__ void __launch_bounds__(32 * WARPS, CTAS) k_rotate16(Params p) {
    __shared__ __align__(16) float tables[WARPS][2 * MAX_PAIRS];
    constexpr int HEADS = 32 / P, U = 2;
    const int lane = threadIdx.x & 31, sub = lane % P;
    float *table = tables[threadIdx.x >> 5];
    const bool in = 16 * sub < p.D;
    const Lane16 at16 = lane16<INTER>(p.r, sub);
    Cols w;
    if (NORM && in) load_weights16<INTER>(p.w, p.w_wide, at16, w);
    const float rd = 1.0f / p.D;
    const int64_t units = (int64_t)p.B * p.L * p.groups, step = (int64_t)gridDim.x * WARPS;
    for (int64_t u = (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5); u < units; u += step) {
        const int64_t token = div_nonneg(u, p.groups);
        const int first = (int)(u - token * p.groups) * p.per, last = first + p.per < p.H ? first + p.per : p.H;
        const int64_t b = div_nonneg(token, p.L), l = token - b * p.L;
        const E *x = static_cast<const E *>(p.x) + b * p.x_bs + l * p.x_ls;
        E *out = static_cast<E *>(p.out) + b * p.o_bs + l * p.o_ls;
        Raw8<E> raw[U][2];
        auto fetch = [&](int h0) {
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const int h = h0 + i * HEADS;
                raw[i][0].clear();
                raw[i][1].clear();
                if (in && h < last) {
                    raw[i][0].load(x + h * p.x_hs + at16.a);
                    raw[i][1].load(x + h * p.x_hs + at16.b);
                }
            }
        };
        fetch(first + lane / P);                // before the table: the loads do not depend on it
        const int64_t at = b * p.p_bs + l * p.p_ls;
        turn_table(p.r, p.wide ? static_cast<const int64_t *>(p.pos)[at] : static_cast<const int32_t *>(p.pos)[at], table, lane);
        Turn16 t;
        turn16_of(at16, table, t);
        for (int h0 = first + lane / P; h0 - lane / P < last; h0 += U * HEADS) {
            Raw8<E> now[U][2];
#pragma unroll
            for (int i = 0; i < U; ++i) { now[i][0] = raw[i][0]; now[i][1] = raw[i][1]; }
            if (h0 - lane / P + U * HEADS < last) fetch(h0 + U * HEADS);
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const int h = h0 + i * HEADS;
                Cols v;
                widen16<INTER>(now[i], v);
                if (NORM) norm16<P>(v, w, rd, p.eps);
                turn16(at16, t, v);
                if (in && h < last) store_runs<INTER>(out + h * p.o_hs, at16, v);
            }
        }
    }
}

// a unit takes all heads of its token where there are tokens enough for all SMs, fewer where there are not; -> the grid
static unsigned plan(Params &p, int heads) {
    const int64_t tokens = (int64_t)p.B * p.L, passes = cdiv(p.H, heads), want = (int64_t)num_sms() * 32;
    int64_t each = cdiv(tokens * passes, want);
    if (each > passes) each = passes;
    p.per = (int)(each * heads);
    p.groups = (int)cdiv(p.H, p.per);
    const int64_t grid = cdiv(tokens * p.groups, WARPS), most = (int64_t)num_sms() * CTAS;
    return (unsigned)(grid < most ? grid : most);
}
template <typename E, int P> cudaError_t go(Params p, cudaStream_t st) {
    const unsigned grid = plan(p, 32 / P);
    const bool inter = p.r.layout == INTERLEAVED;
    if (inter && p.w) k_rotate8<E, P, true, true><<<grid, 32 * WARPS, 0, st>>>(p);
    else if (inter) k_rotate8<E, P, true, false><<<grid, 32 * WARPS, 0, st>>>(p);
    else if (p.w) k_rotate8<E, P, false, true><<<grid, 32 * WARPS, 0, st>>>(p);
    else k_rotate8<E, P, false, false><<<grid, 32 * WARPS, 0, st>>>(p);
    return cudaGetLastError();
}
template <typename E, int P> cudaError_t go16(Params p, cudaStream_t st) {
    const unsigned grid = plan(p, 32 / P);
    const bool inter = p.r.layout == INTERLEAVED;
    if (inter && p.w) k_rotate16<E, P, true, true><<<grid, 32 * WARPS, 0, st>>>(p);
    else if (inter) k_rotate16<E, P, true, false><<<grid, 32 * WARPS, 0, st>>>(p);
    else if (p.w) k_rotate16<E, P, false, true><<<grid, 32 * WARPS, 0, st>>>(p);
    else k_rotate16<E, P, false, false><<<grid, 32 * WARPS, 0, st>>>(p);
    return cudaGetLastError();
}
template <typename E> cudaError_t pick(const Params &p, cudaStream_t st) {
    if (p.D % 16 == 0 && p.r.rot % 16 == 0) {
        if (p.D <= 16) return go16<E, 1>(p, st);
        if (p.D <= 32) return go16<E, 2>(p, st);
        if (p.D <= 64) return go16<E, 4>(p, st);
        if (p.D <= 128) return go16<E, 8>(p, st);
        return go16<E, 16>(p, st);
    }
    if (p.D <= 16) return go<E, 2>(p, st);
    if (p.D <= 32) return go<E, 4>(p, st);
    if (p.D <= 64) return go<E, 8>(p, st);
    if (p.D <= 128) return go<E, 16>(p, st);
    return go<E, 32>(p, st);
}

// ---------------------------------------------------------------------------------------------------
// the append

struct AppendParams {
    const __nv_bfloat16 *x[3];          // q [B, n, H, 128], k and v [B, n, heads, 128]
    int64_t bs[3], ts[3], hs[3];
    __nv_bfloat16 *out;                 // rotated q, dense
    uint8_t *pool[2];                   // this layer's k and v
    float *scale[2];
    const int *rows;
    const void *pos;                    // [B, n] int32 or int64, or null: a token's place in its row
    int64_t p_bs, p_ts;
    int wide;
    const void *w[2];                   // norm weights of q and of k, bf16, fp32 with w_wide, or null
    int w_wide;
    Rotation r;
    float eps;
    int B, n, H, heads, per, groups;    // per: heads of a unit, of the token's H + 2 heads
};

// The rules of the plain append: a row whose last extend was refused, a page that several rows name, a row's listings after the
// first keep what they hold, counted. q is rotated whatever becomes of the row. A unit is a warp's share of a token: some of
// its q, k and v heads, in that order, two at a time (16 lanes each). Without loads ahead: 2 x 4400 tokens, 16 + 16 + 16 heads, 120 of
// 128 columns rotated: bf16 116 us, int8 133.
template <bool I8> __global__ void __launch_bounds__(32 * AWARPS) k_append_rotated(AppendParams p, Meta m) {
    __shared__ float tables[AWARPS][2 * MAX_PAIRS];
    const int lane = threadIdx.x & 31, sub = lane & 15, side = lane >> 4;
    float *table = tables[threadIdx.x >> 5];
    Turn t;
    partners(p.r, sub, t);
    const int all = p.H + 2 * p.heads;
    const int64_t units = (int64_t)p.B * p.n * p.groups, step = (int64_t)gridDim.x * AWARPS;
    for (int64_t u = (int64_t)blockIdx.x * AWARPS + (threadIdx.x >> 5); u < units; u += step) {
        const int64_t bt = div_nonneg(u, p.groups);
        const int first = (int)(u - bt * p.groups) * p.per, last = first + p.per < all ? first + p.per : all;
        const int b = (int)div_nonneg(bt, p.n), i = (int)(bt - (int64_t)b * p.n);
        const int row = p.rows[b];
        int page = -1, place = 0;
        int64_t at = i - p.n;
        bool again = false;
        if (last > p.H)
            for (int j = lane; j < b; j += 32) again |= p.rows[j] == row;
        if ((unsigned)row < (unsigned)m.slots) {
            at += m.lengths[row];
            const int64_t j = at / m.page;
            if (last > p.H && at >= 0 && j < m.width && m.refused[row] != m.epoch) page = m.table[(int64_t)row * m.width + j];
            place = (int)(at - j * m.page);
        }
        if ((unsigned)page < (unsigned)m.pages && m.refs[page] > 1) page = -1;
        const bool put = !__any_sync(0xffffffffu, again) && (unsigned)page < (unsigned)m.pages;
        // the token has no place of its own: counted where its k heads begin
        if (!put && lane == 0 && first <= p.H && p.H < last) atomicAdd(m.failed, p.heads);
        if (first < p.H + p.heads) {
            if (p.pos != nullptr) {
                const int64_t o = b * p.p_bs + i * p.p_ts;
                at = p.wide ? static_cast<const int64_t *>(p.pos)[o] : static_cast<const int32_t *>(p.pos)[o];
            }
            turn_table(p.r, at, table, lane);
            turn_of(p.r, sub, table, t);
        }
        for (int h0 = first; h0 < last; h0 += 2) {
            const int h = h0 + side;
            const int which = h < p.H ? 0 : h < p.H + p.heads ? 1 : 2;
            const int head = which == 0 ? h : which == 1 ? h - p.H : h - p.H - p.heads;
            const bool in = h < last && (which == 0 || put);
            float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f}, o[8];
            if (in) {
                const __nv_bfloat16 *x = p.x[which] + b * p.bs[which] + i * p.ts[which] + head * p.hs[which] + 8 * sub;
                load8(x, v);
                if (which < 2) load_partners(x, t, o);
            }
            const void *w = which < 2 ? p.w[which] : nullptr;
            if (p.w[0] != nullptr || p.w[1] != nullptr) {
                float n[8], no[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) { n[j] = v[j]; no[j] = o[j]; }
                Weights ww;
                if (w != nullptr) load_weights(w, p.w_wide, 8 * sub, t, ww);
                head_norm<16>(n, no, ww, t, 1.0f / 128, p.eps);
                if (w != nullptr)
#pragma unroll
                    for (int j = 0; j < 8; ++j) { v[j] = n[j]; o[j] = no[j]; }
            }
            if (which < 2) {
                if (t.own) turn<true>(t, v, o);
                else turn<false>(t, v, o);
            }
            const int64_t to = ((int64_t)page * p.heads + head) * m.page + place;
            if (which == 0) {
                if (in) store8(p.out + (bt * p.H + head) * 128 + 8 * sub, v);
            } else if (!I8) {
                if (in) store8(reinterpret_cast<__nv_bfloat16 *>(p.pool[which - 1]) + to * 128 + 8 * sub, v);
            }
            if (I8 && h0 + 1 >= p.H) {          // the pair has a k or v head
                float peak = nanmax_abs3(0.0f, v[0], v[1]);
#pragma unroll
                for (int j = 2; j < 8; j += 2) peak = nanmax_abs3(peak, v[j], v[j + 1]);
                peak = lanes_max<16>(peak);
                // a NaN or an infinity in the row: its scale is NaN, so that what reads it gives NaN
                const float sc = peak < INFINITY ? i8_scale(peak) : __int_as_float(0x7fffffff);
                if (in && which > 0) {
                    *reinterpret_cast<uint2 *>(p.pool[which - 1] + to * 128 + 8 * sub) =
                        quant_chunk8<0, false>(v, sc, sc >= 0x1p-90f, x2_splat(-sc), x2_splat(__frcp_rn(sc)));
                    if (sub == 0) p.scale[which - 1][to] = sc;
                }
            }
        }
    }
}

// A row of K or V (16 columns of it in this lane) as codes and scale
__device__ __forceinline__ void put_codes(uint8_t *o, float *scale, const Lane16 &l, const float (&a)[8], const float (&b)[8], bool in, bool lead) {
    float peak = nanmax_abs3(0.0f, a[0], a[1]);
#pragma unroll
    for (int j = 2; j < 8; j += 2) peak = nanmax_abs3(peak, a[j], a[j + 1]);
#pragma unroll
    for (int j = 0; j < 8; j += 2) peak = nanmax_abs3(peak, b[j], b[j + 1]);
    peak = lanes_max<8>(peak);
    // a NaN or an infinity in the row: its scale is NaN, so that what reads it gives NaN. i8_scale_bf16 is the IEEE quotient of
    // any finite fp32 peak, as i8_scale
    const float sc = peak < INFINITY ? i8_scale_bf16(peak) : __int_as_float(0x7fffffff);
    if (!in) return;
    const bool fast = sc >= 0x1p-90f;
    const uint64_t ns = x2_splat(-sc), rs = x2_splat(__frcp_rn(sc));
    *reinterpret_cast<uint2 *>(o + l.a) = quant_chunk8<0, false>(a, sc, fast, ns, rs);
    *reinterpret_cast<uint2 *>(o + l.b) = quant_chunk8<0, false>(b, sc, fast, ns, rs);
    if (lead) *scale = sc;
}

// ... with rotated parts of a multiple of 16: sixteen columns a lane, four heads of one kind (q, k or v) a pass. Each kind
// has a loop of its own, whose addresses only step on (61 us with one loop that asks for the kind). 2 x 4400 tokens, 16 + 16 + 16
// heads: int8 52 us of 28 for the bytes, bf16 51 of 33. So it is neither the quantizer nor HBM that bounds it: half of the issue slots
// are empty, and the 16 warps of an SM wait for their chains (norm, turn, peak, codes). Loads further ahead, through shared memory,
// and more warps of fewer registers changed nothing or cost more.
template <bool I8, bool INTER> __global__ void __launch_bounds__(32 * AWARPS, ACTAS) k_append_rotated16(AppendParams p, Meta m) {
    __shared__ __align__(16) float tables[AWARPS][2 * MAX_PAIRS];
    const int lane = threadIdx.x & 31, sub = lane & 7, side = lane >> 3;
    float *table = tables[threadIdx.x >> 5];
    const Lane16 at16 = lane16<INTER>(p.r, sub);
    const int nq = (p.H + 3) >> 2, nk = (p.heads + 3) >> 2, all = nq + 2 * nk;         // passes
    const int64_t units = (int64_t)p.B * p.n * p.groups, step = (int64_t)gridDim.x * AWARPS;
    for (int64_t u = (int64_t)blockIdx.x * AWARPS + (threadIdx.x >> 5); u < units; u += step) {
        const int64_t bt = div_nonneg(u, p.groups);
        const int first = (int)(u - bt * p.groups) * p.per, last = first + p.per < all ? first + p.per : all;
        const int b = (int)div_nonneg(bt, p.n), i = (int)(bt - (int64_t)b * p.n);
        // this unit's heads of each kind: [h, end) in steps of four, this lane's quarter
        const int hq = 4 * first + side, endq = min(4 * last, p.H);
        const int hk = max(4 * (first - nq), 0) + side, endk = min(4 * (last - nq), p.heads);
        const int hv = max(4 * (first - nq - nk), 0) + side, endv = min(4 * (last - nq - nk), p.heads);
        Raw8<__nv_bfloat16> raw[2];
        auto fetch = [&](const __nv_bfloat16 *x, bool in) {
            raw[0].clear();
            raw[1].clear();
            if (in) {
                raw[0].load(x + at16.a);
                raw[1].load(x + at16.b);
            }
        };
        const __nv_bfloat16 *xq = p.x[0] + b * p.bs[0] + i * p.ts[0] + hq * p.hs[0];
        const __nv_bfloat16 *xk = p.x[1] + b * p.bs[1] + i * p.ts[1] + hk * p.hs[1];
        const __nv_bfloat16 *xv = p.x[2] + b * p.bs[2] + i * p.ts[2] + hv * p.hs[2];
        // the first pass's loads, before the row is known: they do not depend on it
        if (first < nq) fetch(xq, hq < endq);
        else if (first < nq + nk) fetch(xk, hk < endk);
        else fetch(xv, hv < endv);
        const int row = p.rows[b];
        int page = -1, place = 0;
        int64_t at = i - p.n;
        bool again = false;
        if (last > nq)
            for (int j = lane; j < b; j += 32) again |= p.rows[j] == row;
        if ((unsigned)row < (unsigned)m.slots) {
            at += m.lengths[row];
            const int64_t j = at < 0 ? m.width : div_nonneg(at, m.page);
            if (last > nq && j < m.width && m.refused[row] != m.epoch) page = m.table[(int64_t)row * m.width + j];
            place = (int)(at - j * m.page);
        }
        if ((unsigned)page < (unsigned)m.pages && m.refs[page] > 1) page = -1;
        const bool put = !__any_sync(0xffffffffu, again) && (unsigned)page < (unsigned)m.pages;
        // the token has no place of its own: counted where its k heads begin
        if (!put && lane == 0 && first <= nq && nq < last) atomicAdd(m.failed, p.heads);
        const int64_t token = (int64_t)page * p.heads * m.page + place;                 // head h: h pages further
        if (first < nq + nk) {
            if (p.pos != nullptr) {
                const int64_t o = b * p.p_bs + i * p.p_ts;
                at = p.wide ? static_cast<const int64_t *>(p.pos)[o] : static_cast<const int32_t *>(p.pos)[o];
            }
            turn_table(p.r, at, table, lane);
            Turn16 t;
            turn16_of(at16, table, t);
            Cols w;
            if (first < nq) {
                if (p.w[0] != nullptr) load_weights16<INTER>(p.w[0], p.w_wide, at16, w);
                __nv_bfloat16 *out = p.out + (bt * p.H + hq) * 128;
                for (int h = hq; h - side < endq; h += 4, out += 512) {
                    Cols v;
                    widen16<INTER>(raw, v);
                    xq += 4 * p.hs[0];
                    if (h - side + 4 < endq) fetch(xq, h + 4 < endq);
                    else if (last > nq) fetch(xk, hk < endk);
                    if (p.w[0] != nullptr) norm16<8>(v, w, 1.0f / 128, p.eps);
                    turn16(at16, t, v);
                    if (h < endq) store_runs<INTER>(out, at16, v);
                }
            }
            if (last > nq) {
                if (p.w[1] != nullptr) load_weights16<INTER>(p.w[1], p.w_wide, at16, w);
                int64_t to = token + (int64_t)hk * m.page;
                for (int h = hk; h - side < endk; h += 4, to += 4 * m.page) {
                    Cols v;
                    widen16<INTER>(raw, v);
                    xk += 4 * p.hs[1];
                    if (h - side + 4 < endk) fetch(xk, h + 4 < endk);
                    else if (last > nq + nk) fetch(xv, hv < endv);
                    if (p.w[1] != nullptr) norm16<8>(v, w, 1.0f / 128, p.eps);
                    turn16(at16, t, v);
                    const bool in = put && h < endk;
                    if (I8) {
                        float c0[8], c1[8];
                        take_run<INTER>(v, 0, c0);
                        take_run<INTER>(v, 1, c1);
                        put_codes(p.pool[0] + to * 128, p.scale[0] + to, at16, c0, c1, in, sub == 0);
                    } else if (in) {
                        store_runs<INTER>(reinterpret_cast<__nv_bfloat16 *>(p.pool[0]) + to * 128, at16, v);
                    }
                }
            }
        }
        int64_t to = token + (int64_t)hv * m.page;
        for (int h = hv; h - side < endv; h += 4, to += 4 * m.page) {
            const Raw8<__nv_bfloat16> now[2] = {raw[0], raw[1]};
            xv += 4 * p.hs[2];
            if (h - side + 4 < endv) fetch(xv, h + 4 < endv);
            const bool in = put && h < endv;
            if (I8) {
                float c0[8], c1[8];
                now[0].widen(c0);
                now[1].widen(c1);
                put_codes(p.pool[1] + to * 128, p.scale[1] + to, at16, c0, c1, in, sub == 0);
            } else if (in) {
                *reinterpret_cast<uint4 *>(p.pool[1] + to * 256 + 2 * at16.a) = now[0].w;
                *reinterpret_cast<uint4 *>(p.pool[1] + to * 256 + 2 * at16.b) = now[1].w;
            }
        }
    }
}

} // namespace rotary

cudaError_t launch_rotate(const RotateArgs &a, cudaStream_t st) {
    rotary::Params p;
    p.x = a.x; p.x_bs = a.x_bs; p.x_ls = a.x_ls; p.x_hs = a.x_hs;
    p.out = a.out; p.o_bs = a.o_bs; p.o_ls = a.o_ls; p.o_hs = a.o_hs;
    p.pos = a.pos; p.p_bs = a.p_bs; p.p_ls = a.p_ls; p.wide = a.wide;
    p.w = a.w; p.w_wide = a.w_wide;
    p.r = {a.freq, a.rot, a.layout, a.factor};
    p.eps = a.eps; p.B = a.B; p.L = a.L; p.H = a.H; p.D = a.D;
    if (a.dtype == 0) return rotary::pick<__nv_bfloat16>(p, st);
    if (a.dtype == 1) return rotary::pick<__half>(p, st);
    return rotary::pick<float>(p, st);
}

cudaError_t launch_append_rotated(const CacheArgs &c, int layer, const AppendRotatedArgs &a, cudaStream_t st) {
    rotary::AppendParams p;
    const int64_t tokens = (int64_t)layer * c.meta.pages * c.heads * c.meta.page;
    const int row_bytes = c.ks ? 128 : 256;
    for (int i = 0; i < 3; ++i) {
        p.x[i] = static_cast<const __nv_bfloat16 *>(a.x[i]);
        p.bs[i] = a.bs[i]; p.ts[i] = a.ts[i]; p.hs[i] = a.hs[i];
    }
    p.out = static_cast<__nv_bfloat16 *>(a.out);
    p.pool[0] = static_cast<uint8_t *>(c.k) + tokens * row_bytes;
    p.pool[1] = static_cast<uint8_t *>(c.v) + tokens * row_bytes;
    p.scale[0] = c.ks ? c.ks + tokens : nullptr;
    p.scale[1] = c.ks ? c.vs + tokens : nullptr;
    p.rows = a.rows; p.pos = a.pos; p.p_bs = a.p_bs; p.p_ts = a.p_ts; p.wide = a.wide;
    p.w[0] = a.w[0]; p.w[1] = a.w[1]; p.w_wide = a.w_wide;
    p.r = {a.freq, a.rot, a.layout, a.factor};
    p.eps = a.eps; p.B = a.B; p.n = a.n; p.H = a.H; p.heads = c.heads;
    // passes of a token: four heads of a kind at a time, or two of any; a unit takes all of them where there are tokens enough
    const bool wide = a.rot % 16 == 0;
    const int64_t count = (int64_t)a.B * a.n, want = (int64_t)num_sms() * 32;
    const int64_t passes = wide ? cdiv(a.H, 4) + 2 * cdiv(c.heads, 4) : cdiv(a.H + 2 * c.heads, 2);
    int64_t each = cdiv(count * passes, want);
    if (each > passes) each = passes;
    p.groups = (int)cdiv(passes, each);
    p.per = (int)(wide ? each : 2 * each);
    const int64_t grid = cdiv(count * p.groups, rotary::AWARPS), most = (int64_t)num_sms() * rotary::ACTAS;
    const unsigned g = (unsigned)(grid < most ? grid : most), threads = 32 * rotary::AWARPS;
    if (wide && a.layout == rotary::INTERLEAVED) {
        if (c.ks) rotary::k_append_rotated16<true, true><<<g, threads, 0, st>>>(p, c.meta);
        else rotary::k_append_rotated16<false, true><<<g, threads, 0, st>>>(p, c.meta);
    } else if (wide) {
        if (c.ks) rotary::k_append_rotated16<true, false><<<g, threads, 0, st>>>(p, c.meta);
        else rotary::k_append_rotated16<false, false><<<g, threads, 0, st>>>(p, c.meta);
    } else {
        if (c.ks) rotary::k_append_rotated<true><<<g, threads, 0, st>>>(p, c.meta);
        else rotary::k_append_rotated<false><<<g, threads, 0, st>>>(p, c.meta);
    }
    return cudaGetLastError();
}

} // namespace hn
