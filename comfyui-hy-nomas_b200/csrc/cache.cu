// cache.cu - the paged K/V cache of forked sequences: the write of new tokens into pages, the page operations
// (extend, fork, free, compact, copy) and their metadata, all on the device and without a host synchronization.
//
// Pools: k and v [layers][pages][heads][page][128], bf16, or int8 codes with one fp32 scale per (token, head)
// ([layers][pages][heads][page], the arithmetic of hn_quantize_kv). One table serves every layer:
//   table   [slots][width]  page ids in order, -1 where there is none
//   lengths [slots]         tokens held
//   refs    [pages]         how many table entries name the page; 0 = free
//   refused [slots]         `epoch` where the row's last extend could not be met: append leaves such a row as it is
// New pages are the free ids in ascending order, handed to the requests in the order they are listed, so the
// result does not depend on timing. A request that cannot be met (no page left, table row full, an id out of
// range, a row listed twice, a child that is not empty) leaves its row as it was and adds 1 to *failed.
//
// A page operation is a plan - one CTA, which reads the reference counts and the requests and writes who gets which
// page - and a pass of many CTAs that moves the data and the table rows. The plan is O(pages + requests) on metadata of
// a few KB; the pass is one read and one write of the moved bytes, which is what bounds it. Measured (kernel alone): 8 tails of
// 33 tokens to 64 rows, 36 layers, 8 heads, int8: plan 8.1 us, pass 50 us (316 MB, 6.3 TB/s); 240 pages of 32 tokens,
// 16 layers, 8 heads, bf16: plan 5.5 us, pass 155 us (1.0 GB, 6.5 TB/s). A small fork is the two launches, 13 us.
#include "hn_common.cuh"
#include "hn_kernels.h"

namespace hn {
namespace cache {

constexpr int PLAN = 1024;              // threads of the planning CTA
constexpr int HD = 128;

__device__ __forceinline__ bool in_range(int x, int n) { return (unsigned)x < (unsigned)n; }

// exclusive prefix sum of one value per thread over the planning CTA; *total gets the sum
template <typename T> __device__ __forceinline__ T block_scan(T v, T *warp_sums, T *total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    T x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    if (warp == 0) {
        T w = warp_sums[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const T y = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += y;
        }
        warp_sums[lane] = w;
    }
    __syncthreads();
    const T base = warp ? warp_sums[warp - 1] : 0;
    *total = warp_sums[31];
    __syncthreads();
    return base + x - v;
}

// The first `want` free page ids, ascending, into `list`; returns how many there are (at most `want`). Each thread
// takes 8 consecutive ids of a chunk, so the list is in id order.
__device__ int free_pages(const int *refs, int pages, int want, int *list, int *warp_sums) {
    int found = 0;
    for (int base = 0; base < pages && found < want; base += PLAN * 8) {
        const int p0 = base + threadIdx.x * 8;
        int mine = 0;
        uint32_t bits = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (p0 + i < pages && refs[p0 + i] <= 0) { bits |= 1u << i; ++mine; }
        int total;
        int at = found + block_scan(mine, warp_sums, &total);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (bits >> i & 1) {
                if (at < want) list[at] = p0 + i;
                ++at;
            }
        found += total;
    }
    return found < want ? found : want;
}

// `claim[row]` = the first request that lists the row, for every listed row (the planning CTA's scratch)
__device__ void claim_rows(const int *rows, int n, int slots, int *claim) {
    for (int i = threadIdx.x; i < n; i += PLAN)
        if (in_range(rows[i], slots)) claim[rows[i]] = 0x7fffffff;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += PLAN)
        if (in_range(rows[i], slots)) atomicMin(&claim[rows[i]], i);
    __syncthreads();
}

// extend: every listed row grows by `tokens`, on new pages where its last one is full. Served in the order listed, up to the
// first request that there are not enough pages for: `at` counts that one too, so all after it are refused
__global__ void __launch_bounds__(PLAN) k_extend(Meta m, const int *rows, int n, int tokens, int *ws) {
    __shared__ int sums[32];
    __shared__ int64_t wide[32];            // 1024 requests may want more than 2^31 pages, though there are not so many
    int *claim = ws, *list = ws + m.slots;
    claim_rows(rows, n, m.slots, claim);
    // the pages that all requests need; a request without a row, or past the row's end, needs none and fails
    auto needs = [&](int i, int &row, int &first) -> int {
        row = rows[i];
        if (!in_range(row, m.slots) || claim[row] != i) return -1;
        const int64_t len = m.lengths[row];
        const int64_t have = (len + m.page - 1) / m.page, want = (len + tokens + m.page - 1) / m.page;
        first = (int)have;
        return len < 0 || want > m.width ? -1 : (int)(want - have);
    };
    int want = 0;
    for (int base = 0; base < n; base += PLAN) {
        const int i = base + threadIdx.x;
        int row, first;
        int64_t total;
        const int need = i < n ? needs(i, row, first) : 0;
        block_scan<int64_t>(need > 0 ? need : 0, wide, &total);
        want = total > m.pages - want ? m.pages : want + (int)total;     // no more than there are
    }
    const int have = free_pages(m.refs, m.pages, want, list, sums);
    __syncthreads();
    int64_t off = 0;
    for (int base = 0; base < n; base += PLAN) {
        const int i = base + threadIdx.x;
        int row = 0, first = 0;
        int64_t total;
        const int need = i < n ? needs(i, row, first) : 0;
        const int64_t at = off + block_scan<int64_t>(need > 0 ? need : 0, wide, &total);
        if (i < n) {
            const bool met = need >= 0 && at + need <= have;
            if (in_range(row, m.slots) && claim[row] == i) m.refused[row] = met ? 0 : m.epoch;
            if (!met) {
                atomicAdd(m.failed, 1);
            } else {
                for (int j = 0; j < need; ++j) {
                    const int p = list[at + j];
                    m.table[(int64_t)row * m.width + first + j] = p;
                    m.refs[p] = 1;
                }
                m.lengths[row] += tokens;
            }
        }
        off += total;
    }
}

// free: the listed rows drop their pages. One CTA per row; an entry is taken out of the table by an exchange, so a
// row listed twice is freed once. Integer sums: the order of the CTAs does not show.
__global__ void __launch_bounds__(256) k_free(Meta m, const int *rows, int n) {
    const int row = rows[blockIdx.x];
    if (!in_range(row, m.slots)) {
        if (threadIdx.x == 0) atomicAdd(m.failed, 1);
        return;
    }
    int *entry = m.table + (int64_t)row * m.width;
    for (int j = threadIdx.x; j < m.width; j += 256) {
        if (entry[j] < 0) continue;
        const int p = atomicExch(&entry[j], -1);
        if (in_range(p, m.pages)) atomicSub(&m.refs[p], 1);
    }
    if (threadIdx.x == 0) { m.lengths[row] = 0; m.refused[row] = 0; }
}

// fork, plan: request i gets a new page for its parent's partial last page. moves: src, dst, tokens of request i
// (dst -1: nothing to copy), and ok[i] whether the child's row is to be written.
__global__ void __launch_bounds__(PLAN) k_fork_plan(Meta m, const int *parents, const int *children, int n, int *ws) {
    dep_launch();
    __shared__ int sums[32];
    int *claim = ws, *list = claim + m.slots, *src = list + m.pages, *dst = src + n, *ntok = dst + n, *ok = ntok + n;
    for (int i = threadIdx.x; i < n; i += PLAN)
        if (in_range(parents[i], m.slots)) claim[parents[i]] = 0x7fffffff;   // a parent nobody claims
    __syncthreads();
    claim_rows(children, n, m.slots, claim);
    auto needs = [&](int i, int &a, int &c, int &len) -> int {
        a = parents[i]; c = children[i];
        if (!in_range(a, m.slots) || !in_range(c, m.slots) || claim[c] != i || claim[a] != 0x7fffffff) return -1;
        if (m.lengths[c] != 0 || m.table[(int64_t)c * m.width] >= 0) return -1;
        len = m.lengths[a];
        if (len < 0 || (int64_t)len > (int64_t)m.width * m.page) return -1;
        if (len % m.page == 0) return 0;
        // a tail without a page cannot be copied: the request takes none of the free ones
        return in_range(m.table[(int64_t)a * m.width + len / m.page], m.pages) ? 1 : -1;
    };
    const int have = free_pages(m.refs, m.pages, n < m.pages ? n : m.pages, list, sums);
    __syncthreads();
    int off = 0;
    for (int base = 0; base < n; base += PLAN) {
        const int i = base + threadIdx.x;
        int a = 0, c = 0, len = 0, total;
        int need = i < n ? needs(i, a, c, len) : 0;
        const int at = off + block_scan(need > 0 ? need : 0, sums, &total);
        if (i < n) {
            int s = -1, d = -1, t = 0;
            if (need == 1) {
                if (at < have) {
                    d = list[at];
                    s = m.table[(int64_t)a * m.width + len / m.page];
                    t = len % m.page;
                } else {
                    need = -1;
                }
            }
            if (need < 0) atomicAdd(m.failed, 1);
            else {
                if (need) m.refs[d] = 1;
                m.lengths[c] = len;
                m.refused[c] = 0;
            }
            src[i] = s; dst[i] = need < 0 ? -1 : d; ntok[i] = t; ok[i] = need >= 0;
        }
        off += total;
    }
}

// compact, plan: with n live pages, the k-th live page at or above n moves to the k-th free id below n. move_to[p]
// (p >= n) is where page p goes; src, dst list the moves, count[0] is their number.
__global__ void __launch_bounds__(PLAN) k_compact_plan(Meta m, int *ws) {
    dep_launch();
    __shared__ int sums[32];
    int *count = ws, *to = ws + 4, *src = to + m.pages, *dst = src + m.pages;
    int live = 0;
    for (int base = 0; base < m.pages; base += PLAN * 8) {
        const int p0 = base + threadIdx.x * 8;
        int mine = 0, total;
#pragma unroll
        for (int i = 0; i < 8; ++i) mine += p0 + i < m.pages && m.refs[p0 + i] > 0;
        block_scan(mine, sums, &total);
        live += total;
    }
    int holes = 0, movers = 0;
    for (int base = 0; base < m.pages; base += PLAN * 8) {
        const int p0 = base + threadIdx.x * 8;
        uint32_t hole = 0, mover = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int p = p0 + i;
            if (p >= m.pages) continue;
            const bool used = m.refs[p] > 0;
            if (p < live && !used) hole |= 1u << i;
            if (p >= live && used) mover |= 1u << i;
        }
        int total;                     // both counts in one scan: at most 8192 of each in a chunk
        const int at = block_scan(__popc(hole) | __popc(mover) << 16, sums, &total);
        int h = holes + (at & 0xffff), v = movers + (at >> 16);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (hole >> i & 1) dst[h++] = p0 + i;
            if (mover >> i & 1) src[v++] = p0 + i;
            else if (p0 + i >= live && p0 + i < m.pages) to[p0 + i] = -1;
        }
        holes += total & 0xffff;
        movers += total >> 16;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < movers; i += PLAN) {
        const int s = src[i], d = dst[i];
        to[s] = d;
        m.refs[d] = m.refs[s];
        m.refs[s] = 0;
    }
    if (threadIdx.x == 0) { count[0] = movers; count[1] = live; }
}

struct CopyParams {
    uint8_t *k, *v;                  // pools
    float *ks, *vs;                  // or null
    int layers, pages, heads, page, row_bytes;
    const int *src, *dst, *ntok;     // moves; ntok null: whole pages
    const int *count;                // their number on the device, or null
    int n;                           // ... or here
};

// One warp's run of `bytes` contiguous bytes (a multiple of 128), 8 x 16 bytes per lane in flight
__device__ __forceinline__ void warp_copy(uint8_t *d, const uint8_t *s, int bytes, int lane) {
    const uint4 *sp = reinterpret_cast<const uint4 *>(s);
    uint4 *dp = reinterpret_cast<uint4 *>(d);
    const int n = bytes >> 4;
    int i = lane;
    for (; i + 7 * 32 < n; i += 8 * 32) {
        uint4 r[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) r[j] = sp[i + 32 * j];
#pragma unroll
        for (int j = 0; j < 8; ++j) dp[i + 32 * j] = r[j];
    }
    for (; i < n; i += 32) dp[i] = sp[i];
}

// The moves' data: one warp per (move, layer, k or v, head), the run of `ntok` tokens of that head's page.
__device__ void copy_units(const CopyParams &p) {
    const int lane = threadIdx.x & 31;
    const int moves = p.count ? *p.count : p.n;
    const int64_t units = (int64_t)moves * p.layers * 2 * p.heads;
    const int64_t step = (int64_t)gridDim.x * (blockDim.x >> 5);
    for (int64_t u = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); u < units; u += step) {
        const int64_t hu = div_nonneg(u, p.heads);
        const int h = (int)(u - hu * p.heads);
        const int64_t mu = div_nonneg(hu >> 1, p.layers);
        const int l = (int)((hu >> 1) - mu * p.layers), kv = (int)(hu & 1);
        const int s = p.src[mu], d = p.dst[mu], t = p.ntok ? p.ntok[mu] : p.page;
        if (!in_range(s, p.pages) || !in_range(d, p.pages) || s == d) continue;
        const int64_t base = (int64_t)l * p.pages;
        const int64_t from = ((base + s) * p.heads + h) * p.page, to = ((base + d) * p.heads + h) * p.page;
        uint8_t *pool = kv ? p.v : p.k;
        warp_copy(pool + to * p.row_bytes, pool + from * p.row_bytes, t * p.row_bytes, lane);
        if (p.ks != nullptr) {
            float *sc = kv ? p.vs : p.ks;
            for (int i = lane; i < t; i += 32) sc[to + i] = sc[from + i];
        }
    }
}

__global__ void __launch_bounds__(256) k_copy_pages(CopyParams p) { copy_units(p); }

// fork, pass: the children's rows (full pages shared, the new tail page), then the tails' data
__global__ void __launch_bounds__(256) k_fork_pass(CopyParams p, Meta m, const int *parents, const int *children, int n,
                                                   const int *ok) {
    dep_wait();
    for (int i = blockIdx.x; i < n; i += gridDim.x) {
        if (!ok[i]) continue;
        const int a = parents[i], c = children[i], len = m.lengths[a], full = len / m.page;
        const int *from = m.table + (int64_t)a * m.width;
        int *to = m.table + (int64_t)c * m.width;
        for (int j = threadIdx.x; j < m.width; j += 256) {
            int e = -1;
            if (j < full) {
                e = from[j];
                if (in_range(e, m.pages)) atomicAdd(&m.refs[e], 1);
            } else if (j == full && len % m.page) {
                e = p.dst[i];
            }
            to[j] = e;
        }
    }
    copy_units(p);
}

// compact, pass: table entries at or above the live count follow their pages, then the pages' data
__global__ void __launch_bounds__(256) k_compact_pass(CopyParams p, Meta m, const int *ws) {
    dep_wait();
    const int live = ws[1];
    const int *to = ws + 4;
    const int64_t n = (int64_t)m.slots * m.width;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int e = m.table[i];
        if (e >= live && e < m.pages) m.table[i] = to[e];
    }
    copy_units(p);
}

struct AppendParams {
    const __nv_bfloat16 *x[2];                  // k, v [B, n, heads, 128]
    int64_t bs[2], ts[2], hs[2];                // element strides
    uint8_t *pool[2];                           // this layer's pools
    float *scale[2];
    const int *rows;
    int B, n, heads;
};

// append: the last n tokens of each listed row. A row that its last extend refused has no room for them (its last tokens are
// old ones), a page that several rows name is not one row's to write, and a row listed again is written by its first listing
// alone: such tokens are left out and counted. A warp takes the heads of one token, four K and V rows of 128 at a time
// (lanes 0-15 a K row, 16-31 the V row, 8 elements each), so that eight rows are in flight. bf16 is copied; int8 takes the
// absmax over the 16 lanes, hn_quantize_kv's scale and codes. Measured: 2 x 4400 tokens, 16 heads, int8 33 us (3.4 TB/s of
// reads and writes): the absmax stands between a row's load and its store.
template <bool I8>
__global__ void __launch_bounds__(256) k_append(AppendParams p, Meta m) {
    const int lane = threadIdx.x & 31, sub = lane & 15;
    const bool isv = lane >= 16;
    const __nv_bfloat16 *x = (isv ? p.x[1] : p.x[0]) + 8 * sub;
    const int64_t bs = isv ? p.bs[1] : p.bs[0], ts = isv ? p.ts[1] : p.ts[0], hs = isv ? p.hs[1] : p.hs[0];
    uint8_t *pool = isv ? p.pool[1] : p.pool[0];
    float *scale = isv ? p.scale[1] : p.scale[0];
    constexpr int U = 4;
    const int groups = (p.heads + U - 1) / U;               // a warp's share of a token: U heads
    const int64_t units = (int64_t)p.B * p.n * groups, step = (int64_t)gridDim.x * 8;
    for (int64_t u = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); u < units; u += step) {
        const int64_t bt = div_nonneg(u, groups);
        const int h0 = (int)(u - bt * groups) * U;
        const int b = (int)div_nonneg(bt, p.n), t = (int)(bt - (int64_t)b * p.n);
        const __nv_bfloat16 *src = x + b * bs + t * ts + h0 * hs;
        uint4 raw[U];                                       // before the table is known: the loads do not depend on it
#pragma unroll
        for (int i = 0; i < U; ++i)
            if (h0 + i < p.heads) raw[i] = ldg_stream(src + i * hs);
        const int row = p.rows[b];
        int page = -1, at = 0;
        bool again = false;
        for (int i = lane; i < b; i += 32) again |= p.rows[i] == row;
        if (in_range(row, m.slots)) {
            const int refused = m.refused[row];
            at = m.lengths[row] - p.n + t;
            const int j = at / m.page;
            if (at >= 0 && j < m.width && refused != m.epoch) page = m.table[(int64_t)row * m.width + j];
            at -= j * m.page;
        }
        if (in_range(page, m.pages) && m.refs[page] > 1) page = -1;
        if (__any_sync(0xffffffffu, again) || !in_range(page, m.pages)) {          // the token has no place of its own
            if (lane == 0 && h0 == 0) atomicAdd(m.failed, p.heads);
            continue;
        }
        const int64_t token = ((int64_t)page * p.heads + h0) * m.page + at;
#pragma unroll
        for (int i = 0; i < U; ++i) {
            if (h0 + i >= p.heads) break;
            const int64_t to = token + (int64_t)i * m.page;
            if (!I8) {
                *reinterpret_cast<uint4 *>(pool + to * (2 * HD) + 16 * sub) = raw[i];
            } else {
                const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
                float v[8], peak = 0.0f;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    v[2 * j] = bf16_lo(w[j]);
                    v[2 * j + 1] = bf16_hi(w[j]);
                    peak = nanmax_abs3(peak, v[2 * j], v[2 * j + 1]);
                }
                peak = lanes_max<16>(peak);
                // a NaN or an infinity in the row: its scale is NaN, so that what reads it gives NaN
                const float sc = peak < INFINITY ? i8_scale_bf16(peak) : __int_as_float(0x7fffffff);
                const bool fast = sc >= 0x1p-90f;
                *reinterpret_cast<uint2 *>(pool + to * HD + 8 * sub) =
                    quant_chunk8<0, false>(v, sc, fast, x2_splat(-sc), x2_splat(__frcp_rn(sc)));
                if (sub == 0) scale[to] = sc;
            }
        }
    }
}

} // namespace cache

using namespace cache;

static CopyParams copy_params(const CacheArgs &a) {
    CopyParams p;
    p.k = static_cast<uint8_t *>(a.k); p.v = static_cast<uint8_t *>(a.v);
    p.ks = a.ks; p.vs = a.vs;
    p.layers = a.layers; p.pages = a.meta.pages; p.heads = a.heads; p.page = a.meta.page;
    p.row_bytes = a.ks ? HD : 2 * HD;
    p.src = p.dst = p.ntok = p.count = nullptr;
    p.n = 0;
    return p;
}
// CTAs of 8 warps for `units` warp units, at most 6 per SM (what the registers allow): the rest is a stride loop
static unsigned copy_grid(int64_t units) {
    const int64_t want = cdiv(units, 8), most = (int64_t)num_sms() * 6;
    return (unsigned)(want < 1 ? 1 : want > most ? most : want);
}

cudaError_t launch_cache_extend(const Meta &m, const int *rows, int n, int tokens, int *ws, cudaStream_t st) {
    k_extend<<<1, PLAN, 0, st>>>(m, rows, n, tokens, ws);
    return cudaGetLastError();
}
cudaError_t launch_cache_free(const Meta &m, const int *rows, int n, cudaStream_t st) {
    k_free<<<n, 256, 0, st>>>(m, rows, n);
    return cudaGetLastError();
}
cudaError_t launch_cache_fork(const CacheArgs &a, const int *parents, const int *children, int n, int *ws, cudaStream_t st) {
    k_fork_plan<<<1, PLAN, 0, st>>>(a.meta, parents, children, n, ws);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    CopyParams p = copy_params(a);
    const int *src = ws + a.meta.slots + a.meta.pages;
    p.src = src; p.dst = src + n; p.ntok = src + 2 * n; p.n = n;
    return launch_after(k_fork_pass, copy_grid((int64_t)n * a.layers * 2 * a.heads), 256, 0, st, p, a.meta, parents, children, n,
                        src + 3 * n);
}
cudaError_t launch_cache_compact(const CacheArgs &a, int *ws, cudaStream_t st) {
    k_compact_plan<<<1, PLAN, 0, st>>>(a.meta, ws);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    CopyParams p = copy_params(a);
    p.count = ws; p.src = ws + 4 + a.meta.pages; p.dst = p.src + a.meta.pages;
    // at most half of the pages move
    return launch_after(k_compact_pass, copy_grid((int64_t)(a.meta.pages / 2) * a.layers * 2 * a.heads), 256, 0, st, p, a.meta, ws);
}
cudaError_t launch_cache_copy(const CacheArgs &a, const int *src, const int *dst, int n, cudaStream_t st) {
    CopyParams p = copy_params(a);
    p.src = src; p.dst = dst; p.n = n;
    k_copy_pages<<<copy_grid((int64_t)n * a.layers * 2 * a.heads), 256, 0, st>>>(p);
    return cudaGetLastError();
}
cudaError_t launch_cache_append(const CacheArgs &a, int layer, const void *k, int64_t k_bs, int64_t k_ts, int64_t k_hs,
                                const void *v, int64_t v_bs, int64_t v_ts, int64_t v_hs, const int *rows, int B, int n,
                                cudaStream_t st) {
    AppendParams p;
    p.x[0] = static_cast<const __nv_bfloat16 *>(k); p.x[1] = static_cast<const __nv_bfloat16 *>(v);
    p.bs[0] = k_bs; p.ts[0] = k_ts; p.hs[0] = k_hs;
    p.bs[1] = v_bs; p.ts[1] = v_ts; p.hs[1] = v_hs;
    const int64_t tokens = (int64_t)layer * a.meta.pages * a.heads * a.meta.page;
    const int row_bytes = a.ks ? HD : 2 * HD;
    p.pool[0] = static_cast<uint8_t *>(a.k) + tokens * row_bytes;
    p.pool[1] = static_cast<uint8_t *>(a.v) + tokens * row_bytes;
    p.scale[0] = a.ks ? a.ks + tokens : nullptr;
    p.scale[1] = a.ks ? a.vs + tokens : nullptr;
    p.rows = rows; p.B = B; p.n = n; p.heads = a.heads;
    int64_t grid = cdiv((int64_t)B * n * cdiv(a.heads, 4), 8);
    const int64_t most = (int64_t)num_sms() * 8;
    if (grid > most) grid = most;
    if (a.ks) k_append<true><<<(unsigned)grid, 256, 0, st>>>(p, a.meta);
    else k_append<false><<<(unsigned)grid, 256, 0, st>>>(p, a.meta);
    return cudaGetLastError();
}

} // namespace hn
