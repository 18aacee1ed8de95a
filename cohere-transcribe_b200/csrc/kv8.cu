// kv8.cu -- the 8-bit paged K/V cache (include/ct_kv8.h): rows written into
// pages, the pages' bookkeeping, and the C entry points.
#include <algorithm>
#include <atomic>

#include "kv8.cuh"
#include "kv8_attn.cuh"
#include "kv8_many.cuh"

namespace ct {
namespace kv8 {

// ---- rows -> blocks -------------------------------------------------------------
// One warp per (sequence, touched page, kv head, K or V): it reads the block's
// new rows once (16 bytes a lane, whole rows side by side), takes the largest
// magnitude as the maximum of the bit patterns without their signs (magnitudes
// order as unsigned integers, two bf16 at a time), and writes codes from the
// same registers.  Blocks with an infinity or a NaN take a path of their own.
// The loads hang together as length -> rows and page -> scale, so the rows are
// under way before the page is known.  Bound by the latency of that chain: a
// decode step of 256 sequences takes 8.3 us (1.6 MB), prompts of 56k bf16 rows
// 81 us (363 MB, 4.5 TB/s; with 6 instead of 8 CTAs per SM 86, with 10 92 us).
struct AppendArgs {
    Pool p;
    const int *table, *len, *row_start;
    int stride, n_rows, max_rows, n_seqs, layer;
    const void *src[2];
    int ld[2];
    int items;   // blocks x heads x 2 of a sequence, at most
};

template <typename T, int D, int FMT>
__global__ void __launch_bounds__(128, sizeof(T) == 4 && D == 128 ? 5 : 8) append_kernel(const AppendArgs a) {
    constexpr int EPL = 16 / sizeof(T), LPR = D / EPL, RPP = 32 / LPR, PASSES = ROWS / RPP;
    const int s = blockIdx.y, lane = threadIdx.x & 31;
    const int item = blockIdx.x * 4 + (threadIdx.x >> 5);
    if (item >= a.items) return;
    const RowSpan sp = row_span(a.len, a.row_start, s, a.n_rows, a.max_rows, a.stride * ROWS);
    if ((sp.n == 0 && sp.ok) || (!a.row_start && sp.len <= 0)) return;   // no row
    if (!sp.ok || sp.n > sp.len) {
        if (lane == 0) set_status(CT_STATUS_BAD_ARG);
        return;
    }
    const int hk = item % (2 * a.p.heads), kv = hk & 1, h = hk >> 1;
    const int p0 = sp.len - sp.n;
    const int blk = p0 / ROWS + item / (2 * a.p.heads);
    if (blk > (sp.len - 1) / ROWS) return;
    const int lo = max(p0 - blk * ROWS, 0), hi = min(sp.len - blk * ROWS, ROWS);   // the block's new rows
    const int rl = lane / LPR, c = (lane % LPR) * EPL;
    const T *src = static_cast<const T *>(a.src[kv]) +
                   ((size_t)sp.first + (blk * ROWS - p0)) * (size_t)a.ld[kv] + (size_t)h * D + c;
    uint4 x[PASSES];
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int r = i * RPP + rl;
        x[i] = make_uint4(0, 0, 0, 0);
        if (r >= lo && r < hi) x[i] = *reinterpret_cast<const uint4 *>(src + (ptrdiff_t)r * a.ld[kv]);
    }
    const int page = a.table[(size_t)s * a.stride + blk];
    const bool there = a.p.has(page);
    const size_t b = a.p.block(there ? page : 0, a.layer, kv, h);
    const int refs = a.p.refs && there ? a.p.refs[page] : 1;
    const float old = lo > 0 ? a.p.scales[b] : 0.0f;
    if (!there || refs != 1) {
        if (lane == 0) set_status(CT_STATUS_BAD_ARG);
        return;
    }
    uint32_t top = 0;                     // largest magnitude's bits
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
            top = sizeof(T) == 2 ? __vmaxu2(top, w[j] & 0x7FFF7FFFu) : max(top, w[j] & 0x7FFFFFFFu);
    }
    if (sizeof(T) == 2) top = max(top >> 16, top & 0xFFFFu) << 16;
    top = __reduce_max_sync(0xffffffffu, top);
    const bool special = top >= 0x7F800000u;   // an infinity or a NaN
    bool nan = false;
    if (special) {
        float amax = 0.0f;                // of the finite ones
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const T *e = reinterpret_cast<const T *>(&x[i]);
#pragma unroll
            for (int j = 0; j < EPL; ++j) {
                const float v = fabsf(to_f32(e[j]));
                nan |= v != v;
                if (v < INFINITY) amax = fmaxf(amax, v);
            }
        }
        top = __float_as_uint(warp_max(amax));
        nan = __any_sync(0xffffffffu, nan);
    }
    uint8_t *dst = a.p.codes + b * (ROWS * D) + c;
    float scale = block_scale<FMT>(__uint_as_float(top)), shrink = 1.0f;
    if (lo > 0) {
        nan |= old != old;
        scale = fmaxf(scale, old);
        shrink = old / scale;
    }
    const float inv = 1.0f / scale;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int r = i * RPP + rl;
        uint32_t w[EPL / 4];
        uint32_t *o = reinterpret_cast<uint32_t *>(dst + r * D);
        if (r >= lo && r < hi) {
            const T *e = reinterpret_cast<const T *>(&x[i]);
            float y[EPL];
#pragma unroll
            for (int j = 0; j < EPL; ++j) y[j] = to_f32(e[j]) * inv;   // exact: scale is a power of two
            if (special) {
#pragma unroll
                for (int j = 0; j < EPL; ++j) y[j] = y[j] != y[j] ? 0.0f : fminf(fmaxf(y[j], -448.0f), 448.0f);
            }
#pragma unroll
            for (int j = 0; j < EPL; j += 4) w[j / 4] = codes4<FMT>(y[j], y[j + 1], y[j + 2], y[j + 3], special);
        } else if (r < lo && shrink < 1.0f) {   // rows that were there: rounded to the grown scale
#pragma unroll
            for (int j = 0; j < EPL; j += 4) {
                const uint32_t u = o[j / 4];
                w[j / 4] = codes4<FMT>(code_to_f32<FMT>(u & 0xFFu) * shrink, code_to_f32<FMT>(u >> 8 & 0xFFu) * shrink,
                                       code_to_f32<FMT>(u >> 16 & 0xFFu) * shrink, code_to_f32<FMT>(u >> 24) * shrink, false);
            }
        } else {
            continue;
        }
        if (EPL == 8) *reinterpret_cast<uint2 *>(o) = make_uint2(w[0], w[EPL / 4 - 1]);
        else *o = w[0];
    }
    __syncwarp();   // every lane has read the old scale
    if (lane == 0) a.p.scales[b] = nan ? __uint_as_float(0x7FC00000u) : scale;
}

// ---- pages ----------------------------------------------------------------------
// Allocation: count the free pages of each segment and the pages each sequence
// asks for, then hand the k-th lowest free page to the k-th asked for, found by
// binary search in the prefix of needs.  Latency-bound (two launches, 4 us each
// alone); copies run at 6.2 TB/s (268 MB each way in 86 us), 32 KB a CTA.
constexpr int SEG = 4096;   // pages whose counts one CTA takes
constexpr int PT = 1024;    // threads of the counting kernels

// Exclusive scan of v over the CTA's PT threads; total to every thread.
__device__ __forceinline__ int cta_scan(int v, int &total, int *sm) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();   // sm is free again
    if (lane == 31) sm[w] = x;
    __syncthreads();
    if (w == 0) {
        int t = sm[lane], z = t;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, z, o);
            if (lane >= o) z += y;
        }
        sm[lane] = z;
    }
    __syncthreads();
    total = sm[31];
    return x - v + (w ? sm[w - 1] : 0);
}

// Sum of seg[0 .. n) over the CTA, to every thread.
__device__ __forceinline__ int cta_sum(const int *seg, int n, int *sm) {
    int v = 0, total;
    for (int i = threadIdx.x; i < n; i += PT) v += seg[i];
    cta_scan(v, total, sm);
    return total;
}

struct AllocArgs {
    Pool p;
    // reserve: table / len of the sequences, add; fork: src table / len, parents, and dst
    int *table, *len;
    int stride, n;               // stride of the table that grows, sequences that ask
    const int *add;              // reserve
    const int *src_table, *src_len, *parents;   // fork
    int src_stride, src_n;
    // workspace
    int *first;                  // [n]: table position of the first new page; < 0: refused
    int *prefix;                 // [n + 1]: pages asked for by the sequences before
    int *seg;                    // [segments]: free pages
    int nseg;
};

// Pages that sequence i asks for, and where they go.
template <bool FORK>
__device__ __forceinline__ int pages_asked(const AllocArgs &a, int i, int &first) {
    first = -1;
    if (FORK) {
        const int q = a.parents[i];
        if (q < 0) { first = 0; return 0; }
        if (q >= a.src_n) return 0;
        const int len = a.src_len[q];
        if (len <= 0) { first = 0; return 0; }
        if (len > min(a.stride, a.src_stride) * ROWS) return 0;   // before pages_of, which adds to it
        if (len % ROWS == 0) { first = 0; return 0; }
        if (!a.p.has(a.src_table[(size_t)q * a.src_stride + len / ROWS])) return 0;
        first = len / ROWS;
        return 1;
    }
    const int len = max(a.len[i], 0), add = a.add[i];
    if (add < 0 || add > a.stride * ROWS - len) return 0;
    first = pages_of(len);
    return pages_of(len + add) - first;
}

template <bool FORK>
__global__ void __launch_bounds__(PT) count_kernel(const AllocArgs a) {
    __shared__ int sm[32];
    pdl_trigger();
    if (blockIdx.x < (unsigned)a.nseg) {   // free pages of one segment
        int v = 0, total;
#pragma unroll
        for (int j = 0; j < SEG / PT; ++j) {
            const long long p = (long long)blockIdx.x * SEG + j * PT + threadIdx.x;
            if (p < a.p.n_pages) v += a.p.refs[p] == 0;
        }
        cta_scan(v, total, sm);
        if (threadIdx.x == 0) a.seg[blockIdx.x] = total;
        return;
    }
    int before = 0;
    for (int i0 = 0; i0 < a.n; i0 += PT) {
        const int i = i0 + threadIdx.x;
        int first = -1, total;
        const int v = i < a.n ? pages_asked<FORK>(a, i, first) : 0;
        const int at = cta_scan(v, total, sm);
        if (i < a.n) {
            a.first[i] = first;
            a.prefix[i] = before + at;
            if (first < 0) set_status(CT_STATUS_BAD_ARG);
        }
        before += total;
    }
    if (threadIdx.x == 0) a.prefix[a.n] = before;
}

// Page p, the o-th free one, goes to the sequence with prefix[i] <= o < prefix[i + 1].
__device__ __forceinline__ void take_page(const AllocArgs &a, int p, int o, int free_all) {
    int lo = 0, hi = a.n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.prefix[mid] <= o) lo = mid; else hi = mid;
    }
    if (a.prefix[lo + 1] > free_all) return;   // not all of its pages are there: none is taken
    a.table[(size_t)lo * a.stride + a.first[lo] + (o - a.prefix[lo])] = p;
    a.p.refs[p] = 1;
}
// The length of a sequence whose pages were there.
__device__ __forceinline__ void grow(const AllocArgs &a, int i, int free_all) {
    if (a.first[i] < 0) return;
    if (a.prefix[i + 1] > a.prefix[i] && a.prefix[i + 1] > free_all) { set_status(CT_STATUS_NO_PAGE); return; }
    a.len[i] = max(a.len[i], 0) + a.add[i];
}

// Hands the free pages out: the k-th lowest free page is the k-th asked for.
template <bool FORK>
__global__ void __launch_bounds__(PT) assign_kernel(const AllocArgs a) {
    __shared__ int sm[32];
    pdl_wait();
    const int free_all = cta_sum(a.seg, a.nseg, sm);
    int at = cta_sum(a.seg, blockIdx.x, sm);
    const int asked = a.prefix[a.n];
#pragma unroll 1
    for (int j = 0; j < SEG / PT && at < asked; ++j) {
        const long long p = (long long)blockIdx.x * SEG + j * PT + threadIdx.x;
        const int f = p < a.p.n_pages && a.p.refs[p] == 0;
        int total;
        const int o = at + cta_scan(f, total, sm);
        at += total;
        if (f && o < asked) take_page(a, (int)p, o, free_all);
    }
    if (!FORK)
        for (int i = blockIdx.x * PT + threadIdx.x; i < a.n; i += gridDim.x * PT) grow(a, i, free_all);
}

// Both steps in one CTA, for pools of at most SMALL pages: two launches less
// (a beam step of 5 beams 16.4 -> 13.0 us) while one CTA's loads are short.
constexpr int SMALL = 2 * PT;

template <bool FORK>
__global__ void __launch_bounds__(PT) alloc_kernel(const AllocArgs a) {
    __shared__ int sm[32];
    pdl_trigger();
    int free_here[SMALL / PT], free_all = 0, asked = 0;
#pragma unroll
    for (int j = 0; j < SMALL / PT; ++j) {
        const int p = j * PT + threadIdx.x;
        free_here[j] = p < a.p.n_pages && a.p.refs[p] == 0;
    }
    for (int i0 = 0; i0 < a.n; i0 += PT) {
        const int i = i0 + threadIdx.x;
        int first = -1, total;
        const int v = i < a.n ? pages_asked<FORK>(a, i, first) : 0;
        const int at = cta_scan(v, total, sm);
        if (i < a.n) {
            a.first[i] = first;
            a.prefix[i] = asked + at;
            if (first < 0) set_status(CT_STATUS_BAD_ARG);
        }
        asked += total;
    }
    if (threadIdx.x == 0) a.prefix[a.n] = asked;
    int rank[SMALL / PT];
#pragma unroll
    for (int j = 0; j < SMALL / PT; ++j) {
        int total;
        rank[j] = free_all;
        if (j * PT < a.p.n_pages) {
            rank[j] += cta_scan(free_here[j], total, sm);
            free_all += total;
        }
    }
    if (threadIdx.x == 0) a.seg[0] = free_all;
    __syncthreads();   // the prefix is written
#pragma unroll
    for (int j = 0; j < SMALL / PT; ++j)
        if (free_here[j] && rank[j] < asked) take_page(a, j * PT + threadIdx.x, rank[j], free_all);
    if (!FORK)
        for (int i = threadIdx.x; i < a.n; i += PT) grow(a, i, free_all);
}

// One page's slice of codes (16 bytes a thread) and, in slice 0, its scales.
__device__ __forceinline__ void copy_page(const Pool &p, int src, int dst, int slice, int slices) {
    const long long n16 = p.page_bytes() / 16, per = (n16 + slices - 1) / slices;
    const long long end = min(n16, (slice + 1) * per);
    const uint4 *s = reinterpret_cast<const uint4 *>(p.codes + (size_t)src * p.page_bytes());
    uint4 *d = reinterpret_cast<uint4 *>(p.codes + (size_t)dst * p.page_bytes());
    long long i = slice * per + threadIdx.x;
    for (; i + 3 * blockDim.x < end; i += 4 * blockDim.x) {
        uint4 v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = s[i + j * blockDim.x];
#pragma unroll
        for (int j = 0; j < 4; ++j) d[i + j * blockDim.x] = v[j];
    }
    for (; i < end; i += blockDim.x) d[i] = s[i];
    if (slice == 0)
        for (int j = threadIdx.x; j < p.page_scales(); j += blockDim.x)
            p.scales[(size_t)dst * p.page_scales() + j] = p.scales[(size_t)src * p.page_scales() + j];
}
// slices of about 32 KB
__host__ __forceinline__ int page_slices(const Pool &p) {
    return (int)std::min<long long>(64, std::max<long long>(1, p.page_bytes() / 32768));
}

__global__ void __launch_bounds__(256) fork_kernel(const AllocArgs a) {
    pdl_wait();
    const int i = blockIdx.x, slice = blockIdx.y;
    __shared__ int sm_total;
    if (threadIdx.x == 0) sm_total = 0;
    __syncthreads();
    const int need = a.prefix[i + 1] - a.prefix[i];
    if (need) {   // was the page there?
        int v = 0;
        for (int j = threadIdx.x; j < a.nseg; j += 256) v += a.seg[j];
        if (v) atomicAdd(&sm_total, v);
    }
    __syncthreads();
    const bool refused = a.first[i] < 0, none = need && a.prefix[i + 1] > sm_total;
    const int q = refused ? -1 : a.parents[i];
    const int len = q < 0 ? 0 : max(a.src_len[q], 0);
    if (refused || none || len == 0) {
        if (slice == 0 && threadIdx.x == 0) {
            a.len[i] = 0;
            if (none) set_status(CT_STATUS_NO_PAGE);
        }
        return;
    }
    const int *row = a.src_table + (size_t)q * a.src_stride;
    if (slice == 0) {
        for (int j = threadIdx.x; j < len / ROWS; j += 256) {
            const int p = row[j];
            a.table[(size_t)i * a.stride + j] = p;
            if (a.p.has(p)) atomicAdd(&a.p.refs[p], 1);
            else if (p != -1) set_status(CT_STATUS_BAD_ARG);
        }
        if (threadIdx.x == 0) a.len[i] = len;
    }
    if (need) copy_page(a.p, row[len / ROWS], a.table[(size_t)i * a.stride + len / ROWS], slice, gridDim.y);
}

// One holder less of page p.
__device__ __forceinline__ void release(const Pool &p, int page) {
    if (page == -1) return;   // released before
    if (!p.has(page)) { set_status(CT_STATUS_BAD_ARG); return; }
    if (atomicSub(&p.refs[page], 1) <= 0) {   // nobody held it
        atomicAdd(&p.refs[page], 1);
        set_status(CT_STATUS_BAD_ARG);
    }
}

__global__ void __launch_bounds__(128) free_kernel(const Pool p, const int *table, int *len, int n_seqs, int stride,
                                                   const int *which) {
    __shared__ int sm_len;
    const int s = which ? which[blockIdx.x] : blockIdx.x;
    if ((unsigned)s >= (unsigned)n_seqs) {
        if (threadIdx.x == 0) set_status(CT_STATUS_BAD_ARG);
        return;
    }
    if (threadIdx.x == 0) {
        if (len[s] > stride * ROWS) {      // what its row holds is not all its own
            set_status(CT_STATUS_BAD_ARG);
            sm_len = 0;
        } else {
            sm_len = atomicExch(&len[s], 0);   // an index listed twice finds 0 the second time
        }
    }
    __syncthreads();
    const int n = pages_of(max(sm_len, 0));
    for (int j = threadIdx.x; j < n; j += 128) release(p, table[(size_t)s * stride + j]);
}

__global__ void __launch_bounds__(128) trim_kernel(const Pool p, int *table, const int *len, int stride, int window,
                                                   int sinks) {
    const int s = blockIdx.x;
    const int n = len[s];
    if (n > stride * ROWS) {
        if (threadIdx.x == 0) set_status(CT_STATUS_BAD_ARG);
        return;
    }
    const int end = n > window ? (n - window) / ROWS : 0;
    for (int j = pages_of(sinks) + threadIdx.x; j < end; j += 128) {
        int *e = table + (size_t)s * stride + j;
        const int page = *e;
        if (page == -1) continue;
        *e = -1;
        release(p, page);
    }
}

struct CompactArgs {
    Pool p;
    const int *table, *len;
    int stride, n;
    int *refs_out, *table_out, *n_live;
    int *seg, *head;        // head[0] = live pages L, head[1] = live pages numbered below L
    int *dsts, *srcs, *rank;
    int nseg;
};

__global__ void __launch_bounds__(PT) count_live_kernel(const CompactArgs a) {
    __shared__ int sm[32];
    pdl_trigger();
    int v = 0, total;
#pragma unroll
    for (int j = 0; j < SEG / PT; ++j) {
        const long long p = (long long)blockIdx.x * SEG + j * PT + threadIdx.x;
        if (p < a.p.n_pages) v += a.p.refs[p] > 0;
    }
    cta_scan(v, total, sm);
    if (threadIdx.x == 0) a.seg[blockIdx.x] = total;
}

// With b(p) live pages below p: the free pages below L are numbered p - b(p),
// the live ones from L on b(p) - b(L), and equal numbers pair up.
__device__ __forceinline__ void plan_page(const CompactArgs &a, int p, int live, int b, int L) {
    if (p >= a.p.n_pages) return;
    if (p == L) a.head[1] = b;
    int rank = -1;
    if (p < L && !live) { a.dsts[p - b] = p; rank = -2; }
    if (p >= L && live) { a.srcs[b] = p; rank = b; }
    a.rank[p] = rank;
}
__device__ __forceinline__ void plan_head(const CompactArgs &a, int L) {
    a.head[0] = L;
    if (L == a.p.n_pages) a.head[1] = L;
    if (a.n_live) *a.n_live = L;
}

__global__ void __launch_bounds__(PT) plan_kernel(const CompactArgs a) {
    __shared__ int sm[32];
    pdl_wait();
    pdl_trigger();
    const int L = cta_sum(a.seg, a.nseg, sm);
    int at = cta_sum(a.seg, blockIdx.x, sm);
#pragma unroll 1
    for (int j = 0; j < SEG / PT; ++j) {
        const long long pp = (long long)blockIdx.x * SEG + j * PT + threadIdx.x;
        const int p = (int)min(pp, (long long)INT_MAX);
        const bool in = pp < a.p.n_pages;
        const int live = in && a.p.refs[p] > 0;
        int total;
        const int b = at + cta_scan(live, total, sm);
        at += total;
        if (in) plan_page(a, p, live, b, L);
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) plan_head(a, L);
}

// Both steps in one CTA, for pools of at most SMALL pages.
__global__ void __launch_bounds__(PT) plan_small_kernel(const CompactArgs a) {
    __shared__ int sm[32];
    pdl_trigger();
    int live[SMALL / PT], below[SMALL / PT], L = 0;
#pragma unroll
    for (int j = 0; j < SMALL / PT; ++j) {
        const int p = j * PT + threadIdx.x;
        live[j] = p < a.p.n_pages && a.p.refs[p] > 0;
    }
#pragma unroll
    for (int j = 0; j < SMALL / PT; ++j) {
        int total = 0;
        below[j] = L;
        if (j * PT < a.p.n_pages) below[j] += cta_scan(live[j], total, sm);
        L += total;
    }
#pragma unroll
    for (int j = 0; j < SMALL / PT; ++j) plan_page(a, j * PT + threadIdx.x, live[j], below[j], L);
    if (threadIdx.x == 0) plan_head(a, L);
}

__global__ void __launch_bounds__(256) compact_kernel(const CompactArgs a, int slices) {
    pdl_wait();
    const int L = a.head[0], bl = a.head[1], moves = L - bl;
    for (long long w = blockIdx.x; w < (long long)moves * slices; w += gridDim.x) {
        const int i = (int)(w / slices), src = a.srcs[bl + i], dst = a.dsts[i];
        copy_page(a.p, src, dst, (int)(w % slices), slices);
        if (w % slices == 0 && threadIdx.x == 0) {
            const int r = a.p.refs[src];
            a.refs_out[dst] = r;
            a.refs_out[src] = 0;
        }
    }
    const long long t0 = (long long)blockIdx.x * 256 + threadIdx.x, step = (long long)gridDim.x * 256;
    // pages that neither move nor are moved to (rank says so: refs may be refs_out,
    // and the others' entries are being rewritten above)
    for (long long p = t0; p < a.p.n_pages; p += step)
        if (a.rank[p] == -1) a.refs_out[p] = a.p.refs[p];
    for (long long e = t0; e < (long long)a.n * a.stride; e += step) {
        const int s = (int)(e / a.stride), j = (int)(e % a.stride);
        const int len = a.len[s];
        if (len > a.stride * ROWS) {
            if (j == 0) set_status(CT_STATUS_BAD_ARG);
            continue;
        }
        if (j >= pages_of(max(len, 0))) continue;
        const int p = a.table[e];
        int to = p;
        if (p != -1 && !a.p.has(p)) set_status(CT_STATUS_BAD_ARG);
        else if (p >= L && a.rank[p] >= 0) to = a.dsts[a.rank[p] - bl];
        a.table_out[e] = to;
    }
}

__global__ void __launch_bounds__(256) copy_pages_kernel(const Pool p, const int *src, const int *dst, int n) {
    const int i = blockIdx.x, from = src[i], to = dst[i];
    bool bad = !p.has(from) || !p.has(to);
    for (int j = threadIdx.x; j < n; j += 256) bad |= src[j] == to || (j != i && dst[j] == to);
    if (__syncthreads_or(bad)) {
        if (threadIdx.x == 0) set_status(CT_STATUS_BAD_ARG);
        return;
    }
    copy_page(p, from, to, blockIdx.y, gridDim.y);
}

// ---- host side ------------------------------------------------------------------
static bool aligned(const void *p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
static bool good_cache(const ct_kv8_cache *c) {
    if (!c || !c->codes || !c->scales || c->n_pages <= 0 || c->n_layers <= 0 || c->n_layers > 4096 || c->kv_heads <= 0 ||
        c->kv_heads > 4096 || (c->head_dim != 64 && c->head_dim != 128) ||
        (c->format != CT_KV8_E4M3 && c->format != CT_KV8_INT8))
        return false;
    // blocks are numbered in 31 bits
    if ((long long)c->n_pages * c->n_layers * c->kv_heads >= (1ll << 30)) return false;
    return aligned(c->codes, 16) && aligned(c->scales, 4) && aligned(c->refs, 4);
}
static bool good_seqs(const ct_kv8_seqs *s) {
    return s && s->table && s->len && s->n_seqs > 0 && s->n_seqs <= 65535 && s->table_stride > 0 &&
           s->table_stride <= (1 << 26) && aligned(s->table, 4) && aligned(s->len, 4);
}
static Pool pool_of(const ct_kv8_cache *c) {
    return Pool{c->codes, c->scales, c->refs, c->n_pages, c->n_layers, c->kv_heads, c->head_dim};
}
// rows of `width` values with stride ld: vectors of 16 bytes
static bool good_rows(const void *p, int ld, long long width, int type) {
    const int size = type == CT_KV8_F32 ? 4 : 2;
    return p && aligned(p, 16) && ld >= width && ((long long)ld * size) % 16 == 0;
}

// A kernel launch that reports a pending or a new error as a code; `pdl`: may
// start while its predecessor runs (it waits for it before it touches memory);
// `cluster`: CTAs of a cluster along x.
template <typename... P, typename... A>
static int launch_cluster(void (*k)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, bool pdl, int cluster, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    int n = 0;
    if (pdl) {
        at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        at[n].id = cudaLaunchAttributeClusterDimension;
        at[n].val.clusterDim.x = cluster;
        at[n].val.clusterDim.y = at[n].val.clusterDim.z = 1;
        ++n;
    }
    cfg.attrs = at;
    cfg.numAttrs = n;
    if (cudaLaunchKernelEx(&cfg, k, P(args)...) != cudaSuccess) {
        cudaGetLastError();
        return CT_EDEVICE;
    }
    return CT_OK;
}
template <typename... P, typename... A>
static int launch(void (*k)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, bool pdl, A... args) {
    return launch_cluster(k, grid, threads, smem, st, pdl, 1, args...);
}

// The pool as [blocks][16 rows][dim] bytes, boxes of one block, swizzled.
static int pool_map(CUtensorMap *map, const Pool &p) {
    using Encode = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static std::atomic<Encode> encode{nullptr};
    Encode f = encode.load(std::memory_order_acquire);
    if (!f) {
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess || !fn) {
            cudaGetLastError();
            return CT_EDEVICE;
        }
        f = reinterpret_cast<Encode>(fn);
        encode.store(f, std::memory_order_release);
    }
    const cuuint64_t dims[3] = {(cuuint64_t)p.dim, (cuuint64_t)ROWS, (cuuint64_t)p.n_pages * p.page_scales()};
    const cuuint64_t strides[2] = {(cuuint64_t)p.dim, (cuuint64_t)p.dim * ROWS};
    const cuuint32_t box[3] = {(cuuint32_t)p.dim, (cuuint32_t)ROWS, 1}, one[3] = {1, 1, 1};
    return f(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, p.codes, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
             p.dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? CT_OK : CT_EDEVICE;
}

// ---- attention: which kernel, which tiles, which pieces
struct AttnPlan {
    int mt;          // few_kernel: MMA columns of 8 rows; 0: many_kernel
    int tile;        // query rows of a CTA
    int tiles;       // row tiles of a sequence and kv head, at most
    int chunk, max_chunks;
    bool cluster;
    size_t ws;
};
static bool attn_plan(AttnPlan &pl, const ct_kv8_cache *c, const ct_kv8_seqs *s, int type, int n_rows, int max_rows,
                      int max_len, int heads, int causal, int window, int sinks) {
    if (!good_cache(c) || !good_seqs(s) || (type != CT_KV8_F32 && type != CT_KV8_BF16)) return false;
    if (n_rows <= 0 || max_rows <= 0 || max_rows > (1 << 20) || max_len <= 0 || max_len > (1 << 30)) return false;
    if (heads <= 0 || heads % c->kv_heads || heads / c->kv_heads > 1024) return false;
    if (window < 0 || window > (1 << 30) || sinks < 0 || sinks > (1 << 30) || (window && !causal)) return false;
    const long long rows = (long long)max_rows * (heads / c->kv_heads);   // query rows per kv head
    const int group = heads / c->kv_heads;
    // few_kernel up to 16 rows.  With 17 to 32 its CTAs (128 threads) only pay when
    // sequences and heads alone fill the SMs: 20 bf16 rows of 4 heads a group, 16
    // sequences of 20,000 keys 318 us against many_kernel's 382, 64 of 2000 keys 156
    // against 187, but 4 of 8000 keys 86 against 54 and one of 2000 33 against 29.
    // From 33 rows on it reads the cache twice: 571 us against 382.
    pl.mt = rows <= 8 ? 1 : rows <= 16 ? 2 : rows <= 32 && (long long)s->n_seqs * c->kv_heads >= 128 ? 4 : 0;
    pl.tile = pl.mt ? 8 * pl.mt : type == CT_KV8_F32 ? 128 : 256;
    const long long tiles = (rows + pl.tile - 1) / pl.tile;
    long long list = pages_of(std::min<long long>(max_len, (long long)s->table_stride * ROWS));
    if (window) {
        const long long span = (long long)window + pl.tile / group + 1;
        list = std::min(list, pages_of(sinks) + (span + ROWS - 1) / ROWS + 1);
    }
    const long long ctas = s->n_seqs * (long long)c->kv_heads * tiles;
    const long long at_once = 148 * few_ctas(pl.mt);
    long long chunk;
    if (pl.mt) {
        // Pieces of equal length, the most with which all CTAs run at once, three on an
        // SM (two of 32-row tiles), each warp with two pages at least.  4 rows of one
        // sequence of 8000 keys: 16.6 us; 22.7 with four CTAs on an SM, 36.2 with twice
        // as many as fit.  32 windows of 2048 keys, 16 rows each: 23 us, 33 with 640
        // CTAs, of which 444 fit.  A rest of up to a quarter is not cut off.
        const long long pieces = std::max({1ll, 148 * std::min(3, few_ctas(pl.mt)) / ctas, (list + FEW_CHUNK - 1) / FEW_CHUNK});
        chunk = ((list + pieces - 1) / pieces + 7) / 8 * 8;
        if (list <= chunk + chunk / 4) chunk = std::min<long long>(FEW_CHUNK, (list + 3) / 4 * 4);
    } else {
        // whole key tiles; one piece once the tiles alone give every SM a CTA
        long long pieces = std::min(std::max(1ll, 148 / ctas), std::max(1ll, list / (4 * KB)));
        // The tensor core truncates each of its fp32 sums, so an error grows with the
        // keys summed into one accumulator.  fp32 results take at most 1024 keys a
        // piece (1280 where that saves cutting, a sixteenth of them past 16,384) and
        // join the pieces with rounded sums: 14 of 12,289 fp32 calls drawn from
        // perf/operators.py (more than 16 rows per kv head) are further from 64 bits than
        // 1e-6 and 1.5 times their plain form, with pieces of 2048 keys 24 of 1412 were
        // (4 prompts of 1000 to 4097 rows take 2605 us instead of 2066).
        if (type == CT_KV8_F32 && list > 80) pieces = std::max(pieces, std::min(16ll, (list + 63) / 64));
        // However long the cache, 16,384 keys a piece (bf16 results 65,536): a step loses
        // up to 2^-22 of a sum, so 2^-12 (2^-10) of it at most.
        const long long most = type == CT_KV8_F32 ? 1024 : 4096;
        pieces = std::max(pieces, (list + most - 1) / most);
        chunk = ((list + pieces - 1) / pieces + KB - 1) / KB * KB;
    }
    pl.chunk = (int)chunk;
    pl.tiles = (int)tiles;
    pl.max_chunks = (int)((list + chunk - 1) / chunk);
    if (tiles * pl.max_chunks > INT_MAX) return false;
    // Up to 8 pieces of a kv head are one cluster when all CTAs fit the SMs at once: no
    // second kernel (one row over 376 keys: 1.5 us less).
    pl.cluster = pl.mt && pl.max_chunks > 1 && pl.max_chunks <= 8 && ctas * pl.max_chunks <= at_once;
    pl.ws = pl.max_chunks > 1 && !pl.cluster ? (size_t)n_rows * heads * pl.max_chunks * (c->head_dim + 2) * sizeof(float) : 0;
    return true;
}

template <typename T, int D, int FMT, int MT>
static int launch_few(const AttnArgs &a, const AttnPlan &pl, cudaStream_t st) {
    constexpr size_t smem = sizeof(FewSmem<T, D, MT>) + 1024;
    CUtensorMap map;
    if (pool_map(&map, a.p) != CT_OK) return CT_EDEVICE;
    if (smem > 48 * 1024 &&
        cudaFuncSetAttribute(few_kernel<T, D, FMT, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) {
        cudaGetLastError();
        return CT_EDEVICE;
    }
    int rc = launch_cluster(few_kernel<T, D, FMT, MT>, dim3(pl.max_chunks, a.p.heads, a.n_seqs), 128, smem, st, false,
                            pl.cluster ? pl.max_chunks : 1, map, a);
    if (rc == CT_OK && pl.max_chunks > 1 && !pl.cluster)
        rc = launch(join_kernel<T, D>, dim3(pl.tiles, a.p.heads, a.n_seqs), 256, 0, st, true, a, 8 * MT);
    return rc;
}
template <typename T, int D, int FMT>
static int launch_many(const AttnArgs &a, const AttnPlan &pl, cudaStream_t st) {
    constexpr size_t smem = sizeof(ManySmem<D>) + 1024;
    static_assert(smem <= 227 * 1024, "shared memory of a CTA");
    if (cudaFuncSetAttribute(many_kernel<T, D, FMT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) {
        cudaGetLastError();
        return CT_EDEVICE;
    }
    int rc = launch(many_kernel<T, D, FMT>, dim3(pl.max_chunks * pl.tiles, a.p.heads, a.n_seqs), MANY_THREADS, smem, st, false, a);
    if (rc == CT_OK && pl.max_chunks > 1)
        rc = launch(join_kernel<T, D>, dim3(pl.tiles, a.p.heads, a.n_seqs), 256, 0, st, true, a, pl.tile);
    return rc;
}
template <typename T, int D, int FMT>
static int launch_attn(const AttnArgs &a, const AttnPlan &pl, cudaStream_t st) {
    if (pl.mt == 0) return launch_many<T, D, FMT>(a, pl, st);
    if (pl.mt == 1) return launch_few<T, D, FMT, 1>(a, pl, st);
    if (pl.mt == 2) return launch_few<T, D, FMT, 2>(a, pl, st);
    return launch_few<T, D, FMT, 4>(a, pl, st);
}
template <typename T>
static int launch_attn(const AttnArgs &a, const AttnPlan &pl, int fmt, cudaStream_t st) {
    if (a.p.dim == 128)
        return fmt == CT_KV8_E4M3 ? launch_attn<T, 128, CT_KV8_E4M3>(a, pl, st) : launch_attn<T, 128, CT_KV8_INT8>(a, pl, st);
    return fmt == CT_KV8_E4M3 ? launch_attn<T, 64, CT_KV8_E4M3>(a, pl, st) : launch_attn<T, 64, CT_KV8_INT8>(a, pl, st);
}

template <typename T, int D>
static int launch_append(const AppendArgs &a, int fmt, cudaStream_t st) {
    const dim3 grid((a.items + 3) / 4, a.n_seqs);
    return fmt == CT_KV8_E4M3 ? launch(append_kernel<T, D, CT_KV8_E4M3>, grid, 128, 0, st, false, a)
                              : launch(append_kernel<T, D, CT_KV8_INT8>, grid, 128, 0, st, false, a);
}

// ---- workspace of the page operators
static int segments(const ct_kv8_cache *c) { return (c->n_pages + SEG - 1) / SEG; }
static size_t alloc_ws(const ct_kv8_cache *c, int n) { return (2 * (size_t)n + 1 + segments(c)) * sizeof(int); }
static size_t compact_ws(const ct_kv8_cache *c) { return (3 * (size_t)c->n_pages + 2 + segments(c)) * sizeof(int); }
static AllocArgs alloc_args(const ct_kv8_cache *c, const ct_kv8_seqs *s, void *ws) {
    AllocArgs a = {};
    a.p = pool_of(c);
    a.table = s->table; a.len = s->len; a.stride = s->table_stride; a.n = s->n_seqs;
    a.first = static_cast<int *>(ws);
    a.prefix = a.first + a.n;
    a.seg = a.prefix + a.n + 1;
    a.nseg = segments(c);
    return a;
}
template <bool FORK>
static int launch_alloc(AllocArgs &a, cudaStream_t st) {
    if (a.p.n_pages <= SMALL) {
        a.nseg = 1;
        return launch(alloc_kernel<FORK>, dim3(1), PT, 0, st, false, a);
    }
    int rc = launch(count_kernel<FORK>, dim3(a.nseg + 1), PT, 0, st, false, a);
    if (rc == CT_OK) rc = launch(assign_kernel<FORK>, dim3(a.nseg), PT, 0, st, true, a);
    return rc;
}
static bool good_ws(const void *ws) { return ws && aligned(ws, 256); }

}  // namespace kv8
}  // namespace ct

using namespace ct::kv8;

extern "C" int ct_kv8_append(const ct_kv8_cache *c, int layer, const ct_kv8_seqs *s, const void *k, int ldk,
                             const void *v, int ldv, int type, int n_rows, const int *row_start, int max_rows,
                             void *stream) {
    if (!good_cache(c) || !good_seqs(s) || layer < 0 || layer >= c->n_layers) return CT_EINVAL;
    if (type != CT_KV8_F32 && type != CT_KV8_BF16) return CT_EINVAL;
    const long long width = (long long)c->kv_heads * c->head_dim;
    if (!good_rows(k, ldk, width, type) || !good_rows(v, ldv, width, type)) return CT_EINVAL;
    if (n_rows <= 0 || max_rows <= 0 || max_rows > (1 << 20)) return CT_EINVAL;
    if (!row_start && (max_rows != 1 || n_rows < s->n_seqs)) return CT_EINVAL;
    if (cudaPeekAtLastError() != cudaSuccess) return CT_EDEVICE;
    AppendArgs a = {};
    a.p = pool_of(c);
    a.table = s->table; a.len = s->len; a.row_start = row_start;
    a.stride = s->table_stride; a.n_rows = n_rows; a.max_rows = max_rows; a.n_seqs = s->n_seqs; a.layer = layer;
    a.src[0] = k; a.src[1] = v;
    a.ld[0] = ldk; a.ld[1] = ldv;
    const long long items = ((max_rows + ROWS - 2) / ROWS + 1) * 2ll * c->kv_heads;
    a.items = (int)items;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (type == CT_KV8_F32)
        return c->head_dim == 128 ? launch_append<float, 128>(a, c->format, st) : launch_append<float, 64>(a, c->format, st);
    return c->head_dim == 128 ? launch_append<bf16, 128>(a, c->format, st) : launch_append<bf16, 64>(a, c->format, st);
}

extern "C" size_t ct_kv8_attn_ws_bytes(const ct_kv8_cache *c, const ct_kv8_seqs *s, int type, int n_rows, int max_rows,
                                       int max_len, int heads, int causal, int window, int sinks) {
    AttnPlan pl;
    return attn_plan(pl, c, s, type, n_rows, max_rows, max_len, heads, causal, window, sinks) ? pl.ws : 0;
}

extern "C" int ct_kv8_attn(const ct_kv8_cache *c, int layer, const ct_kv8_seqs *s, const void *q, int ldq, void *out,
                           int ldo, int type, int n_rows, const int *row_start, int max_rows, int max_len, int heads,
                           float scale, int causal, int window, int sinks, void *ws, size_t ws_bytes, void *stream) {
    AttnPlan pl;
    if (!attn_plan(pl, c, s, type, n_rows, max_rows, max_len, heads, causal, window, sinks)) return CT_EINVAL;
    if (layer < 0 || layer >= c->n_layers || !(scale > 0.0f) || !(scale < INFINITY)) return CT_EINVAL;
    const long long width = (long long)heads * c->head_dim;
    if (!good_rows(q, ldq, width, type) || !good_rows(out, ldo, width, type)) return CT_EINVAL;
    if (!row_start && (max_rows != 1 || n_rows < s->n_seqs)) return CT_EINVAL;
    if (pl.ws && !good_ws(ws)) return CT_EINVAL;
    if (ws_bytes < pl.ws) return CT_ENOMEM;
    if (cudaPeekAtLastError() != cudaSuccess) return CT_EDEVICE;
    AttnArgs a = {};
    a.p = pool_of(c);
    a.table = s->table; a.len = s->len; a.row_start = row_start;
    a.stride = s->table_stride; a.n_seqs = s->n_seqs; a.layer = layer;
    a.q = q; a.out = out; a.ldq = ldq; a.ldo = ldo;
    a.n_rows = n_rows; a.max_rows = max_rows; a.max_len = max_len;
    a.heads = heads; a.group = heads / c->kv_heads;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.causal = causal != 0; a.window = window; a.sinks = sinks;
    a.chunk = pl.chunk; a.max_chunks = pl.max_chunks; a.cluster = pl.cluster;
    a.part = static_cast<float *>(ws);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return type == CT_KV8_F32 ? launch_attn<float>(a, pl, c->format, st) : launch_attn<bf16>(a, pl, c->format, st);
}

extern "C" size_t ct_kv8_pages_ws_bytes(const ct_kv8_cache *c, int n_seqs) {
    if (!good_cache(c) || n_seqs <= 0 || n_seqs > 65535) return 0;
    return std::max(alloc_ws(c, n_seqs), compact_ws(c));
}

extern "C" int ct_kv8_reserve(const ct_kv8_cache *c, const ct_kv8_seqs *s, const int *add, void *ws, size_t ws_bytes,
                              void *stream) {
    if (!good_cache(c) || !c->refs || !good_seqs(s) || !add || !good_ws(ws)) return CT_EINVAL;
    if ((long long)s->n_seqs * s->table_stride > INT_MAX) return CT_EINVAL;   // pages asked for are summed in 32 bits
    if (ws_bytes < alloc_ws(c, s->n_seqs)) return CT_ENOMEM;
    if (cudaPeekAtLastError() != cudaSuccess) return CT_EDEVICE;
    AllocArgs a = alloc_args(c, s, ws);
    a.add = add;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return launch_alloc<false>(a, st);
}

extern "C" int ct_kv8_fork(const ct_kv8_cache *c, const ct_kv8_seqs *src, const int *parents, const ct_kv8_seqs *dst,
                           void *ws, size_t ws_bytes, void *stream) {
    if (!good_cache(c) || !c->refs || !good_seqs(src) || !good_seqs(dst) || !parents || !good_ws(ws)) return CT_EINVAL;
    const auto meet = [](const int *a, size_t na, const int *b, size_t nb) { return a < b + nb && b < a + na; };
    if (meet(src->table, (size_t)src->n_seqs * src->table_stride, dst->table, (size_t)dst->n_seqs * dst->table_stride) ||
        meet(src->len, src->n_seqs, dst->len, dst->n_seqs))
        return CT_EINVAL;
    if (ws_bytes < alloc_ws(c, dst->n_seqs)) return CT_ENOMEM;
    if (cudaPeekAtLastError() != cudaSuccess) return CT_EDEVICE;
    AllocArgs a = alloc_args(c, dst, ws);
    a.src_table = src->table; a.src_len = src->len; a.parents = parents;
    a.src_stride = src->table_stride; a.src_n = src->n_seqs;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    int rc = launch_alloc<true>(a, st);
    if (rc == CT_OK) rc = launch(fork_kernel, dim3(a.n, page_slices(a.p)), 256, 0, st, true, a);
    return rc;
}

extern "C" int ct_kv8_free(const ct_kv8_cache *c, const ct_kv8_seqs *s, const int *which, int n, void *stream) {
    if (!good_cache(c) || !c->refs || !good_seqs(s) || (which && n < 0)) return CT_EINVAL;
    if (cudaPeekAtLastError() != cudaSuccess) return CT_EDEVICE;
    const int count = which ? n : s->n_seqs;
    if (count == 0) return CT_OK;
    return launch(free_kernel, dim3(count), 128, 0, static_cast<cudaStream_t>(stream), false, pool_of(c),
                  (const int *)s->table, s->len, s->n_seqs, s->table_stride, which);
}

extern "C" int ct_kv8_trim(const ct_kv8_cache *c, const ct_kv8_seqs *s, int window, int sinks, void *stream) {
    if (!good_cache(c) || !c->refs || !good_seqs(s) || window <= 0 || window > (1 << 30) || sinks < 0 || sinks > (1 << 30))
        return CT_EINVAL;
    if (cudaPeekAtLastError() != cudaSuccess) return CT_EDEVICE;
    return launch(trim_kernel, dim3(s->n_seqs), 128, 0, static_cast<cudaStream_t>(stream), false, pool_of(c), s->table,
                  (const int *)s->len, s->table_stride, window, sinks);
}

extern "C" int ct_kv8_compact(const ct_kv8_cache *c, const ct_kv8_seqs *s, int *refs_out, int *table_out, int *n_live,
                              void *ws, size_t ws_bytes, void *stream) {
    if (!good_cache(c) || !c->refs || !good_seqs(s) || !refs_out || !table_out || !good_ws(ws)) return CT_EINVAL;
    if (ws_bytes < compact_ws(c)) return CT_ENOMEM;
    if (cudaPeekAtLastError() != cudaSuccess) return CT_EDEVICE;
    CompactArgs a = {};
    a.p = pool_of(c);
    a.table = s->table; a.len = s->len; a.stride = s->table_stride; a.n = s->n_seqs;
    a.refs_out = refs_out; a.table_out = table_out; a.n_live = n_live;
    a.dsts = static_cast<int *>(ws);
    a.srcs = a.dsts + c->n_pages;
    a.rank = a.srcs + c->n_pages;
    a.head = a.rank + c->n_pages;
    a.seg = a.head + 2;
    a.nseg = segments(c);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    int rc;
    if (c->n_pages <= SMALL) {
        rc = launch(plan_small_kernel, dim3(1), PT, 0, st, false, a);
    } else {
        rc = launch(count_live_kernel, dim3(a.nseg), PT, 0, st, false, a);
        if (rc == CT_OK) rc = launch(plan_kernel, dim3(a.nseg), PT, 0, st, true, a);
    }
    if (rc == CT_OK) rc = launch(compact_kernel, dim3(148 * 4), 256, 0, st, true, a, page_slices(a.p));
    return rc;
}

extern "C" int ct_kv8_copy_pages(const ct_kv8_cache *c, const int *src, const int *dst, int n, void *stream) {
    if (!good_cache(c) || n < 0 || n > 4096 || (n && (!src || !dst))) return CT_EINVAL;
    if (cudaPeekAtLastError() != cudaSuccess) return CT_EDEVICE;
    if (n == 0) return CT_OK;
    const Pool p = pool_of(c);
    return launch(copy_pages_kernel, dim3(n, page_slices(p)), 256, 0, static_cast<cudaStream_t>(stream), false, p, src,
                  dst, n);
}

extern "C" int ct_kv8_status(void) {
    int v = 0, zero = 0;
    if (cudaDeviceSynchronize() != cudaSuccess || cudaMemcpyFromSymbol(&v, g_ct_status, sizeof(int)) != cudaSuccess ||
        cudaMemcpyToSymbol(g_ct_status, &zero, sizeof(int)) != cudaSuccess) {
        cudaGetLastError();
        return CT_EDEVICE;
    }
    return v;
}
