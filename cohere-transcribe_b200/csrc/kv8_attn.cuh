// kv8_attn.cuh -- attention over the 8-bit paged cache (include/ct_kv8.h): the
// kernel for few query rows and the join of its pieces.
#pragma once
#include <limits.h>

#include "kv8.cuh"

namespace ct {
namespace kv8 {

struct AttnArgs {
    Pool p;
    const int *table, *len, *row_start;
    int stride, n_seqs, layer;
    const void *q;
    void *out;
    int ldq, ldo, n_rows, max_rows, max_len;
    int heads, group;       // group = heads / kv heads
    float scale_log2;       // scale * log2(e)
    int causal, window, sinks;
    int chunk;              // pages of a piece
    int max_chunks;
    float *part;            // [n_rows * heads][max_chunks][D], then [n_rows * heads][max_chunks][2]
};

// The pages that a group of query rows (token rows t_lo .. t_hi) reaches: the
// first n_sink pages and those from page `first` on.  Entry i of this list is
// page i for i < n_sink, first + i - n_sink else.
struct PageList {
    int n_sink, first, n;
    __device__ int at(int i) const { return i < n_sink ? i : first + i - n_sink; }
};
__device__ __forceinline__ PageList page_list(const AttnArgs &a, int len, int t_lo, int t_hi) {
    PageList l;
    const int end = a.causal ? min(len, t_hi + 1) : len;
    const int from = a.window ? max(0, t_lo - a.window + 1) : 0;
    l.first = from / ROWS;
    l.n_sink = min(pages_of(a.sinks), l.first);
    l.n = end > from ? l.n_sink + pages_of(end) - l.first : min(l.n_sink, pages_of(max(end, 0)));
    return l;
}
__device__ __forceinline__ bool sees(const AttnArgs &a, int t, int j, int len) {
    return j < len && (!a.causal || j <= t) && (!a.window || j > t - a.window || j < a.sinks);
}

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// x ~ hi + lo as fp16 pairs
__device__ __forceinline__ void split2(float x, float y, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&l);
}
// The power of two that brings the largest magnitude of a row into [1, 2); 1 for
// zero and non-finite ones.
__device__ __forceinline__ float row_pow2(float amax) {
    const int e = (int)(__float_as_uint(amax) >> 23);
    return (e == 0 || e == 255) ? 1.0f : __uint_as_float((uint32_t)min(max(254 - e, 1), 254) << 23);
}

template <typename T>
__device__ __forceinline__ void load8(const T *p, float (&v)[8]) {
    if (sizeof(T) == 4) {
        const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
        const uint4 a = *reinterpret_cast<const uint4 *>(p);
        const bf16 *e = reinterpret_cast<const bf16 *>(&a);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __bfloat162float(e[i]);
    }
}
template <typename T>
__device__ __forceinline__ void store4(T *p, float a, float b, float c, float d) {
    if (sizeof(T) == 4) {
        *reinterpret_cast<float4 *>(p) = make_float4(a, b, c, d);
    } else {
        const __nv_bfloat162 x = __floats2bfloat162_rn(a, b), y = __floats2bfloat162_rn(c, d);
        *reinterpret_cast<uint2 *>(p) =
            make_uint2(*reinterpret_cast<const uint32_t *>(&x), *reinterpret_cast<const uint32_t *>(&y));
    }
}

// ---- few query rows -------------------------------------------------------------
// One CTA per (piece of `chunk` pages, kv head and tile of 8 MT query rows,
// sequence); the rows of a tile are (query row, head of the group) pairs, so the
// heads that share a kv head read its codes once.  Each of the four warps takes
// every fourth page with an online softmax of its own; the warps join through
// shared memory at the end.
//
// Products on the tensor cores (m16n8k16, fp16 in, fp32 sums): codes are exact
// in fp16, and the 16 rows of the MMA hold 8 query rows twice, as the high and
// the low fp16 part of the (power-of-two scaled) query, so the sum of both
// halves carries the query with 22 bits at no extra instruction.  The
// probabilities go the same way into P.V.  Lane (g, t) = (lane / 4, lane % 4)
// holds of each operand what one or two 16-byte loads of a key row give it: a
// product over d does not care in which order the d come, so K fragments take
// 4 consecutive bytes per MMA, and the columns of V fragments are the 16 (8)
// consecutive dims that lane group g loaded.  Codes go from global memory to
// registers to the MMA, the next page's loads in flight meanwhile.
template <int D, int MT>
struct FewSmem {
    union {
        uint4 q[MT][D / 16][32];          // A fragments: hi, lo, hi, lo
        float o[4][8 * MT][D];
    };
    float m[4][8 * MT], l[4][8 * MT];
};

template <typename T, int D, int FMT, int MT>
__global__ void __launch_bounds__(128) few_kernel(const AttnArgs a) {
    constexpr int KC = D / 64;            // 16-byte loads per key row and lane
    constexpr int KS = D / 16;            // MMA steps over the head dim
    constexpr int NJ = D / 8;             // MMA column tiles over the head dim
    constexpr int VB = D / 8;             // V bytes per key and lane
    extern __shared__ __align__(16) uint8_t few_raw[];
    FewSmem<D, MT> &sm = *reinterpret_cast<FewSmem<D, MT> *>(few_raw);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int s = blockIdx.z, hk = blockIdx.y, tile = blockIdx.x / a.max_chunks, piece = blockIdx.x % a.max_chunks;
    pdl_trigger();
    const RowSpan sp = row_span(a.len, a.row_start, s, a.n_rows, a.max_rows, min(a.stride * ROWS, a.max_len));
    if (!sp.ok) {
        if (threadIdx.x == 0 && piece == 0) set_status(CT_STATUS_BAD_ARG);
        return;
    }
    const int G = a.group, M = sp.n * G, m0 = tile * 8 * MT;
    if (m0 >= M) return;
    const int len = max(sp.len, 0);
    const int t_first = len - sp.n;       // token row of query row 0 (negative: it sees nothing before row 0)
    const int t_lo = t_first + m0 / G, t_hi = t_first + (min(m0 + 8 * MT, M) - 1) / G;
    const PageList list = page_list(a, len, t_lo, t_hi);
    const int pieces = max(1, (list.n + a.chunk - 1) / a.chunk);
    if (piece >= pieces) return;

    // queries -> A fragments: warp w prepares row tile w (w < MT)
    float qf[MT];                         // per row g of each tile: scale_log2 / row's power of two
    for (int mt = 0; mt < MT; ++mt) {
        const int m = m0 + mt * 8 + g;
        float amax = 0.0f;
        float v[KC][2][8];
#pragma unroll
        for (int i = 0; i < KC; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i][e][j] = 0.0f;
                if (m < M) {
                    const T *qp = static_cast<const T *>(a.q) + (size_t)(sp.first + m / G) * a.ldq +
                                  (size_t)(hk * G + m % G) * D + (t + 4 * i) * 16 + e * 8;
                    load8(qp, v[i][e]);
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(v[i][e][j]));
            }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        const float r = row_pow2(amax);
        qf[mt] = a.scale_log2 / r;
        if (warp == (mt & 3)) {
#pragma unroll
            for (int i = 0; i < KC; ++i)
#pragma unroll
                for (int w = 0; w < 4; ++w) {   // word w of the 16-byte load: dims 4 w .. 4 w + 3 of the chunk
                    const float *x = &v[i][w >> 1][(w & 1) * 4];
                    uint4 f;
                    split2(x[0] * r, x[1] * r, f.x, f.y);
                    split2(x[2] * r, x[3] * r, f.z, f.w);
                    sm.q[mt][i * 4 + w][lane] = f;
                }
        }
    }
    __syncthreads();

    float o[MT][NJ][2];
    float m_run[MT], l_run[MT];
    int tq[MT];                           // token row of this lane's query row
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        m_run[mt] = -INFINITY;
        l_run[mt] = 0.0f;
        const int m = m0 + mt * 8 + g;
        tq[mt] = m < M ? t_first + m / G : INT_MIN / 2;   // a row of the tile's end: its results are not stored
#pragma unroll
        for (int j = 0; j < NJ; ++j) o[mt][j][0] = o[mt][j][1] = 0.0f;
    }
    const int *trow = a.table + (size_t)s * a.stride;
    const int end = min(list.n, (piece + 1) * a.chunk);
    int at = piece * a.chunk + warp;

    uint4 kr[2][KC];
    uint32_t vr[4][VB / 4];
    float ks = 0.0f, vs = 0.0f;
    bool have = false;
    auto load = [&](int i) {              // page i of the list -> registers
        have = false;
        if (i >= end) return;
        const int page = trow[list.at(i)];
        if (!a.p.has(page)) {
            if (lane == 0) set_status(CT_STATUS_BAD_ARG);
            return;                       // its rows count as not there
        }
        have = true;
        const size_t bk = a.p.block(page, a.layer, 0, hk), bv = bk + a.p.heads;
        const uint8_t *kp = a.p.codes + bk * (ROWS * D), *vp = a.p.codes + bv * (ROWS * D);
        ks = a.p.scales[bk];
        vs = a.p.scales[bv];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int c = 0; c < KC; ++c)
                kr[n][c] = *reinterpret_cast<const uint4 *>(kp + (n * 8 + g) * D + (t + 4 * c) * 16);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const uint8_t *src = vp + (2 * t + (r & 1) + (r >> 1) * 8) * D + g * VB;
            if (VB == 16) {
                const uint4 x = *reinterpret_cast<const uint4 *>(src);
                vr[r][0] = x.x; vr[r][1] = x.y; vr[r][VB / 4 - 2] = x.z; vr[r][VB / 4 - 1] = x.w;
            } else {
                const uint2 x = *reinterpret_cast<const uint2 *>(src);
                vr[r][0] = x.x; vr[r][1] = x.y;
            }
        }
    };
    load(at);
    for (; at < end; at += 4) {
        const int j0 = list.at(at) * ROWS;
        const bool ok = have;
        uint4 k[2][KC];
        uint32_t v[4][VB / 4];
        const float kscale = ks, vscale = vs;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int c = 0; c < KC; ++c) k[n][c] = kr[n][c];
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int w = 0; w < VB / 4; ++w) v[r][w] = vr[r][w];
        load(at + 4);
        if (!ok) continue;
        // every row of the tile sees the whole page
        const bool whole = j0 + ROWS <= len && (!a.causal || j0 + ROWS - 1 <= t_lo) &&
                           (!a.window || j0 > t_hi - a.window || j0 + ROWS <= a.sinks);
        if (j0 + ROWS > len) {            // rows behind the last one may hold anything
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (j0 + 2 * t + (r & 1) + (r >> 1) * 8 >= len)
#pragma unroll
                    for (int w = 0; w < VB / 4; ++w) v[r][w] = 0;
        }
        float c[MT][2][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int n = 0; n < 2; ++n) c[mt][n][0] = c[mt][n][1] = c[mt][n][2] = c[mt][n][3] = 0.0f;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            uint32_t b[2][2];
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const uint4 &x = k[n][i / 4];
                const uint32_t w = (i & 3) == 0 ? x.x : (i & 3) == 1 ? x.y : (i & 3) == 2 ? x.z : x.w;
                codes4_to_half<FMT>(w, b[n][0], b[n][1]);
            }
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                const uint4 f = sm.q[mt][i][lane];
                const uint32_t qa[4] = {f.x, f.y, f.z, f.w};
                mma_f16(c[mt][0], qa, b[0][0], b[0][1]);
                mma_f16(c[mt][1], qa, b[1][0], b[1][1]);
            }
        }
        uint32_t pa[MT][4];
        float rvs[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            const float f = qf[mt] * kscale;
            float x[4];                   // keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9
            bool any = true;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = (c[mt][e >> 1][e & 1] + c[mt][e >> 1][2 + (e & 1)]) * f;
            if (!whole) {
                any = false;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const bool see = sees(a, tq[mt], j0 + 2 * t + (e & 1) + (e >> 1) * 8, len);
                    if (!see) x[e] = -INFINITY;
                    any |= see;
                }
                any |= __shfl_xor_sync(0xffffffffu, (int)any, 1) != 0;
                any |= __shfl_xor_sync(0xffffffffu, (int)any, 2) != 0;
            }
            float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float mn = fmaxf(m_run[mt], mx);
            const float ref = mn == -INFINITY ? 0.0f : mn;
            // probabilities times 2^14: the low fp16 parts stay normal numbers
            float pr[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) pr[e] = ex2(x[e] - ref + 14.0f);
            split2(pr[0], pr[1], pa[mt][0], pa[mt][1]);
            split2(pr[2], pr[3], pa[mt][2], pa[mt][3]);
            const float corr = ex2(m_run[mt] - ref);   // 0 on the first page
            l_run[mt] = l_run[mt] * corr + ((pr[0] + pr[1]) + (pr[2] + pr[3]));
            if (__any_sync(0xffffffffu, mn != m_run[mt])) {
#pragma unroll
                for (int j = 0; j < NJ; ++j) { o[mt][j][0] *= corr; o[mt][j][1] *= corr; }
            }
            m_run[mt] = mn;
            rvs[mt] = any ? vscale : 0.0f;   // a block that a row does not see adds nothing, whatever its scale
        }
#pragma unroll
        for (int w = 0; w < VB / 4; ++w) {
            // 4 dims of keys (2 t, 2 t + 1) and (2 t + 8, 2 t + 9) as pairs over the key
            uint32_t b[4][2];
#pragma unroll
            for (int hp = 0; hp < 2; ++hp) {
                const uint32_t x = v[2 * hp][w], y = v[2 * hp + 1][w];
                codes4_to_half<FMT>(__byte_perm(x, y, 0x5140), b[0][hp], b[1][hp]);
                codes4_to_half<FMT>(__byte_perm(x, y, 0x7362), b[2][hp], b[3][hp]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    mma_f16(d, pa[mt], b[e][0], b[e][1]);
                    const int j = w * 4 + e;
                    o[mt][j][0] = fmaf(rvs[mt], d[0] + d[2], o[mt][j][0]);
                    o[mt][j][1] = fmaf(rvs[mt], d[1] + d[3], o[mt][j][1]);
                }
        }
    }

    // ---- the four warps' results -> one
    __syncthreads();                      // the queries' fragments are read
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        float l = l_run[mt];
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if (t == 0) { sm.m[warp][mt * 8 + g] = m_run[mt]; sm.l[warp][mt * 8 + g] = l; }
        float *dst = sm.o[warp][mt * 8 + g];
        // columns 2 t, 2 t + 1 of tile j: dims (2 t) * VB + j, (2 t + 1) * VB + j
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int j = 0; j < NJ; j += 4)
                *reinterpret_cast<float4 *>(dst + (2 * t + e) * VB + j) =
                    make_float4(o[mt][j][e], o[mt][j + 1][e], o[mt][j + 2][e], o[mt][j + 3][e]);
    }
    __syncthreads();
    const size_t rows_all = (size_t)a.n_rows * a.heads;
    for (int i = threadIdx.x; i < 8 * MT * (D / 4); i += 128) {
        const int row = i / (D / 4), d = (i % (D / 4)) * 4, m = m0 + row;
        if (m >= M) continue;
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) mx = fmaxf(mx, sm.m[w][row]);
        const float ref = mx == -INFINITY ? 0.0f : mx;
        float l = 0.0f;
        float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = ex2(sm.m[w][row] - ref);
            l += sm.l[w][row] * f;
            const float4 x = *reinterpret_cast<const float4 *>(&sm.o[w][row][d]);
            acc.x += x.x * f; acc.y += x.y * f; acc.z += x.z * f; acc.w += x.w * f;
        }
        const size_t r = (size_t)sp.first + m / G;
        const int h = hk * G + m % G;
        if (pieces == 1) {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;   // a row that sees nothing: zeros
            store4(static_cast<T *>(a.out) + r * a.ldo + (size_t)h * D + d, acc.x * inv, acc.y * inv, acc.z * inv,
                   acc.w * inv);
        } else {
            const size_t b = (r * a.heads + h) * a.max_chunks + piece;
            *reinterpret_cast<float4 *>(a.part + b * D + d) = acc;
            if (d == 0) *reinterpret_cast<float2 *>(a.part + rows_all * a.max_chunks * D + b * 2) = make_float2(mx, l);
        }
    }
}

// Joins the pieces of each row: a warp per row, pieces in order.
template <typename T, int D>
__global__ void __launch_bounds__(256) join_kernel(const AttnArgs a, int tile_rows) {
    pdl_wait();
    const int s = blockIdx.z, hk = blockIdx.y, tile = blockIdx.x;
    const RowSpan sp = row_span(a.len, a.row_start, s, a.n_rows, a.max_rows, min(a.stride * ROWS, a.max_len));
    const int G = a.group, M = sp.n * G, m0 = tile * tile_rows;
    if (!sp.ok || m0 >= M) return;
    const int len = max(sp.len, 0), t_first = len - sp.n;
    const PageList list = page_list(a, len, t_first + m0 / G, t_first + (min(m0 + tile_rows, M) - 1) / G);
    const int pieces = (list.n + a.chunk - 1) / a.chunk;
    if (pieces <= 1) return;
    const int lane = threadIdx.x & 31;
    constexpr int W = D / 32;             // values per lane
    for (int m = m0 + (threadIdx.x >> 5); m < min(m0 + tile_rows, M); m += 8) {
        const size_t r = (size_t)sp.first + m / G;
        const int h = hk * G + m % G;
        const size_t b = (r * a.heads + h) * a.max_chunks;
        const float2 *ml = reinterpret_cast<const float2 *>(a.part + (size_t)a.n_rows * a.heads * a.max_chunks * D) + b;
        float mx = -INFINITY;
        for (int c = lane; c < pieces; c += 32) mx = fmaxf(mx, ml[c].x);
        mx = warp_max(mx);
        const float ref = mx == -INFINITY ? 0.0f : mx;
        float l = 0.0f, acc[W];
#pragma unroll
        for (int i = 0; i < W; ++i) acc[i] = 0.0f;
#pragma unroll 4
        for (int c = 0; c < pieces; ++c) {
            const float2 x = ml[c];
            const float f = ex2(x.x - ref);
            l += x.y * f;
            const float *src = a.part + (b + c) * D + lane * W;
#pragma unroll
            for (int i = 0; i < W; ++i) acc[i] = fmaf(src[i], f, acc[i]);
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        T *dst = static_cast<T *>(a.out) + r * a.ldo + (size_t)h * D + lane * W;
        if (W == 4) {
            store4(dst, acc[0] * inv, acc[1] * inv, acc[W - 2] * inv, acc[W - 1] * inv);
        } else if (sizeof(T) == 4) {
            *reinterpret_cast<float2 *>(dst) = make_float2(acc[0] * inv, acc[1] * inv);
        } else {
            *reinterpret_cast<__nv_bfloat162 *>(dst) = __floats2bfloat162_rn(acc[0] * inv, acc[1] * inv);
        }
    }
}

}  // namespace kv8
}  // namespace ct
