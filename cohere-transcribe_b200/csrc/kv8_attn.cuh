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
    int cluster;            // few_kernel: a kv head's pieces are one cluster and join through its shared memory
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
// Chunk (16 bytes) that TMA's swizzle moves chunk 0 of `row` to, rows of D bytes:
// 128-byte rows take the 128-byte pattern, 64-byte rows the 64-byte one.
template <int D>
__device__ __forceinline__ int swz(int row) { return D == 128 ? row & 7 : (row >> 1) & 3; }

__device__ __forceinline__ void tma_load_3d(void *dst, const CUtensorMap *map, uint64_t *bar, int c0, int c1, int c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
        : "memory");
}

// The power of two that brings the largest magnitude of a row into [1, 2); 1 for
// zero and subnormal ones, NaN for an infinity: a softmax over scores of +-inf or
// NaN is NaN, also where all of them are -inf, which else hides a key.
__device__ __forceinline__ float row_pow2(float amax) {
    const int e = (int)(__float_as_uint(amax) >> 23);
    return e == 0 ? 1.0f : __uint_as_float(e == 255 ? 0x7FC00000u : (uint32_t)min(max(254 - e, 1), 253) << 23);
}
// 1 / x of a power of two in [2^-126, 2^126], without a division.
__device__ __forceinline__ float inv_pow2(float x) { return __uint_as_float(0x7F000000u - __float_as_uint(x)); }

// ---- softmax state of a row, both kernels
// Scores x are in log2.  m is the reference of the exponentials, an integer, so that
// moving it scales by exact powers of two; it moves when a score passes it by THR.
// A key's probability p = 2^(x - m + OFF) goes into the sum l, and
// p vs / 2^e (vs: the block scale of its V) as fp16 into P.V.  The exponent e of the
// unit that O is held in follows the largest product of probability and scale, not the
// scales alone: a block with a large scale and next to no probability must not push
// the others' products below what fp16 holds.  With
//   need = max over blocks (largest score - m + log2 vs),
// e is raised to need when that passes it by SLACK and comes down with every move of m.
// So the largest product lies in [2^(OFF - 1), 2^(OFF + SLACK + 1)] <= 2^15 when it is
// seen, and an fp16's absolute step is 2^-32 of it.  Scores more than 120 below m count as
// 120 in need: then vs / 2^e stays finite (such a p is 2^-111 at most).
// e stays within [-126, 126]: at 126, with vs < 2^128, need <= 127 + THR = 126 + SLACK.
constexpr float THR = 4.0f, OFF = 9.0f, SLACK = 5.0f, FAR = -120.0f;
constexpr float E_MIN = -126.0f, E_MAX = 126.0f;
// 2^x of an integer in [-127, 127]; 0 for -127: the sum's low bits hold 127 + x
__device__ __forceinline__ float pow2i(float x) { return __uint_as_float(__float_as_uint(x + 12583039.0f) << 23); }
// floor(log2 v) of v >= 0 (-127 for 0 and subnormals)
__device__ __forceinline__ float log2_floor(float v) {
    return __uint_as_float(0x4B400000u | (__float_as_uint(v) >> 23 & 0xFFu)) - 12583039.0f;
}
// Whether a row with largest new score mx, over blocks with V scales up to 2^(lv + 1), may
// have to move m or raise e (an upper bound of need decides).
__device__ __forceinline__ bool unsettled(float mx, float lv, float m, float e) {
    const float d = mx - m;
    return d > THR || fmaxf(d, FAR) + lv > e + SLACK;
}
// The new m, and what the sums so far are multiplied by for it.
__device__ __forceinline__ float move_m(float mx, float &m) {
    const bool move = mx > m + THR;                // always once a first key is seen
    const float mn = move ? ceilf(mx) : m, d = move ? fmaxf(m - mn, -300.0f) : 0.0f;
    m = mn;
    return d;                                      // a power of two's exponent
}
// The new e after m moved by d, and the exponent of what O is multiplied by (<= 0).
__device__ __forceinline__ float move_e(float need, float d, float &e) {
    const float down = fmaxf(e + d, E_MIN);
    const float en = need > down + SLACK ? fminf(ceilf(need), E_MAX) : down;
    const float f = fmaxf(d + e - en, -127.0f);
    e = en;
    return f;
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
// One CTA per (piece of `chunk` pages, kv head, sequence), for at most 8 MT rows: a
// row is a (query row, head of the group) pair, so the heads that share a kv head
// read its codes once.  Each of the four warps takes
// every fourth page, two at a time, with an online softmax of its own; the warps
// join through shared memory at the end.
//
// Products on the warp-level tensor path (m16n8k16, fp16 in, fp32 sums) with the
// cache as the 16-row operand and the query rows as the 8 columns, so that no
// half of the MMA is empty: S^T = K Q^T (16 keys x 8 rows) and O^T += V^T P^T
// (16 dims x 8 rows).  Codes are exact in fp16.  fp32 queries and probabilities
// are two fp16 each (two MMAs into the same sums), bf16 ones one (queries are
// exact: each row is scaled by a power of two).  Lane (g, t) = (lane / 4,
// lane % 4) gets of K and V what one or two 16-byte loads of a row hold: a
// product over d does not care in which order the d come, so K's fragments take
// 4 consecutive bytes per MMA, and V's 16 rows are neighbouring dims of the 16
// (8) that lane group g loaded.  P^T comes from S^T by 8 x 8 transposes.
//
// The reference of a row's exponentials and the unit of its O move seldom, so most
// pages need one vote and no shuffles.
//
// Each warp keeps a few pages in flight through a ring of its own, one TMA
// copy per K and V block; TMA's swizzle spreads both access patterns over all
// banks.
//
// Bound by HBM where there is much to read (16 rows of 32 heads over 8k to 65k keys:
// 1.19 GB in 206 us, 5.8 TB/s), otherwise by instructions and latency: a pair of pages
// takes a warp 3 to 4 thousand cycles among 16 warps, and start and join about 6
// thousand (64 fp32 rows over up to 1024 keys: 31 us for 62 MB, 36% of the issue slots
// at 11 warps per SM; one row over 376 keys: 10.3 us).
// Pages in flight per warp, and CTAs per SM.  8 rows of 128 dims: 3 pages and 4
// CTAs are 2 to 3% faster than 4 pages and 3 CTAs (attention of 16 rows over 8k to
// 65k keys 207.5 against 213.2 us).
__host__ __device__ constexpr int few_stages(int D, int MT) { return D == 128 && MT == 1 ? 3 : 4; }
__host__ __device__ constexpr int few_ctas(int MT) { return MT == 1 ? 4 : MT == 2 ? 3 : 2; }
constexpr int FEW_CHUNK = 128;            // pages of a piece at most: a lane of each warp per page

template <typename T, int D, int MT>
struct FewSmem {
    static constexpr int QW = sizeof(T) == 4 ? 4 : 2, STAGES = few_stages(D, MT);
    union {
        uint8_t kv[4][STAGES][2][ROWS * D];   // per warp: K and V blocks as TMA wrote them
        float o[4][8 * MT][D];                    // the warps' results, for the join
    };
    uint32_t q[MT][D / 16][32][QW];       // B fragments: high parts, low parts
    float qf[8 * MT];                     // per row: scale_log2 / its power of two
    float m[4][8 * MT], l[4][8 * MT];
    float2 ml[8 * MT];                    // of the CTA, for the cluster's join
    uint64_t full[4][STAGES];
};

__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

template <typename T, int D, int FMT, int MT>
__global__ void __launch_bounds__(128, few_ctas(MT)) few_kernel(const __grid_constant__ CUtensorMap map, const AttnArgs a) {
    constexpr bool TWO = sizeof(T) == 4;
    constexpr int STAGES = few_stages(D, MT);
    constexpr int KC = D / 64;            // 16-byte loads per key row and lane
    constexpr int KS = D / 16;            // MMA steps of Q.K
    constexpr int NJ = D / 16;            // MMA row tiles of P.V
    constexpr int VB = D / 8;             // V bytes per key and lane
    extern __shared__ __align__(1024) uint8_t few_raw[];
    FewSmem<T, D, MT> &sm = *reinterpret_cast<FewSmem<T, D, MT> *>((reinterpret_cast<uintptr_t>(few_raw) + 1023) & ~(uintptr_t)1023);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int s = blockIdx.z, hk = blockIdx.y, piece = blockIdx.x;
    pdl_trigger();
    if (threadIdx.x == 0) prefetch_tmap(&map);
    // Without a window the page list starts at page 0, so this lane's entry of the
    // table is known before the length is: the two loads go together.
    const int e0 = piece * a.chunk + warp, entry = e0 + 4 * lane;
    const int *trow = a.table + (size_t)s * a.stride;
    int page = -1;
    if (!a.window && lane < a.chunk / 4 && entry < a.stride) page = trow[entry];
    const RowSpan sp = row_span(a.len, a.row_start, s, a.n_rows, a.max_rows, min(a.stride * ROWS, a.max_len));
    if (!sp.ok) {
        if (threadIdx.x == 0 && piece == 0) set_status(CT_STATUS_BAD_ARG);
        return;
    }
    const int G = a.group, M = sp.n * G;       // row r: query row r / G, head r % G of the group
    if (M == 0) return;
    const float rg = __frcp_rn((float)G);
    auto row_of = [&](int r) { return (int)((r + 0.5f) * rg); };   // exact: r < 32
    const int len = max(sp.len, 0);
    const int t_lo = len - sp.n, t_hi = len - 1;   // token rows of the query rows (a negative one sees nothing before row 0)
    const PageList list = page_list(a, len, t_lo, t_hi);
    const int pieces = list.n <= a.chunk ? 1 : (list.n + a.chunk - 1) / a.chunk;
    if (piece >= pieces && !a.cluster) return;   // a cluster's CTAs all stay for its barriers

    // this warp's pages: lane i holds the i-th one's number and block scales
    const int e1 = min(list.n, (piece + 1) * a.chunk);
    const int mine = e1 > e0 ? (e1 - e0 + 3) / 4 : 0;
    if (a.window && lane < mine) page = trow[list.at(entry)];
    if (lane == 0) {
        for (int i = 0; i < STAGES; ++i) mbar_init(&sm.full[warp][i], 1);
        fence_mbar_init();
    }
    __syncwarp();
    float ks = 0.0f, vs = 0.0f;
    if (lane < mine) {
        if (a.p.has(page)) {
            const size_t b = a.p.block(page, a.layer, 0, hk);
            ks = a.p.scales[b];
            vs = a.p.scales[b + a.p.heads];
        } else {
            set_status(CT_STATUS_BAD_ARG);   // its rows count as not there
            page = -1;
        }
    }
    auto issue = [&](int i) {             // page i of this warp -> stage i % STAGES
        const int p = __shfl_sync(0xffffffffu, page, i & 31);
        if (i < mine && p >= 0 && lane == 0) {
            const int st = i % STAGES, b = (int)a.p.block(p, a.layer, 0, hk);
            mbar_expect_tx(&sm.full[warp][st], 2 * ROWS * D);
            tma_load_3d(sm.kv[warp][st][0], &map, &sm.full[warp][st], 0, 0, b);
            tma_load_3d(sm.kv[warp][st][1], &map, &sm.full[warp][st], 0, 0, b + a.p.heads);
        }
    };
#pragma unroll
    for (int i = 0; i < STAGES; ++i) issue(i);

    // queries -> B fragments: tile mt by warp mt
    if (warp < MT) {
        const int mt = warp, m = mt * 8 + g, qi = row_of(m);
        const T *qp = static_cast<const T *>(a.q) + (size_t)(sp.first + qi) * a.ldq + (size_t)(hk * G + m - qi * G) * D;
        float amax = 0.0f;
        float v[KC][2][8];
#pragma unroll
        for (int i = 0; i < KC; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i][e][j] = 0.0f;
                if (m < M) load8(qp + (KC * t + i) * 16 + e * 8, v[i][e]);
#pragma unroll
                for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(v[i][e][j]));
            }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        const float r = row_pow2(amax);
        if (t == 0) sm.qf[mt * 8 + g] = a.scale_log2 * inv_pow2(r);
#pragma unroll
        for (int i = 0; i < KC; ++i)
#pragma unroll
            for (int w = 0; w < 4; ++w) {   // word w of the 16-byte load: dims 4 w .. 4 w + 3 of the chunk
                const float *x = &v[i][w >> 1][(w & 1) * 4];
                uint32_t h0, l0, h1, l1;
                split2(x[0] * r, x[1] * r, h0, l0);
                split2(x[2] * r, x[3] * r, h1, l1);
                uint32_t *q = sm.q[mt][i * 4 + w][lane];
                q[0] = h0;
                q[1] = h1;
                if (TWO) { q[FewSmem<T, D, MT>::QW - 2] = l0; q[FewSmem<T, D, MT>::QW - 1] = l1; }
            }
    }
    __syncthreads();

    float o[MT][NJ][4];                   // dims 2 j, 2 j + 1 of the lane group's, rows 2 t, 2 t + 1: (d, r), (d, r'), (d', r), (d', r')
    float mref[MT][2], l[MT][2], eo[MT][2], qf[MT][2];
    int tq[MT][2];                        // token row of this lane's query rows
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int m = mt * 8 + 2 * t + e;
            mref[mt][e] = -INFINITY;
            l[mt][e] = 0.0f;
            eo[mt][e] = E_MIN;
            qf[mt][e] = sm.qf[mt * 8 + 2 * t + e];
            tq[mt][e] = t_lo + row_of(min(m, M - 1));
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j) o[mt][j][0] = o[mt][j][1] = o[mt][j][2] = o[mt][j][3] = 0.0f;
    }
    uint32_t loads = 0;                   // copies into each stage so far, modulo 2 (bit per stage)
    for (int it = 0; it < mine; it += 2) {
        bool there[2];
        int j0[2];
        float kscale[2], vscale[2];
        bool fail = false;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const int i = it + n, st = i % STAGES;
            kscale[n] = __shfl_sync(0xffffffffu, ks, i & 31);
            vscale[n] = __shfl_sync(0xffffffffu, vs, i & 31);
            there[n] = i < mine && __shfl_sync(0xffffffffu, page, i & 31) >= 0;
            j0[n] = list.at(e0 + 4 * i) * ROWS;
            if (there[n] && !fail) {
                fail = !__all_sync(0xffffffffu, mbar_wait(&sm.full[warp][st], (loads >> st) & 1, CT_STATUS_TIMEOUT_TMA));
                loads ^= 1u << st;
            }
        }
        if (fail) {                       // give the copies in flight once more the time to land, and stop
            for (int x = it; x < min(it + STAGES, mine); ++x)
                mbar_wait_for(&sm.full[warp][x % STAGES], (loads >> (x % STAGES)) & 1, CT_STATUS_TIMEOUT_TMA, CT_WAIT_NS / 4);
            break;
        }
        // S^T of both pages (one that is not there goes through with whatever its stage holds, unseen)
        float c[MT][2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) c[mt][n][0] = c[mt][n][1] = c[mt][n][2] = c[mt][n][3] = 0.0f;
            float small[MT][4] = {};      // the low parts' sums: the tensor core truncates, so they stay apart
            const uint8_t *kp = sm.kv[warp][(it + n) % STAGES][0];
            uint4 k[2][KC];
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int i = 0; i < KC; ++i) {
                    const int row = r * 8 + g;
                    k[r][i] = *reinterpret_cast<const uint4 *>(kp + row * D + (((KC * t + i) ^ swz<D>(row)) << 4));
                }
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                uint32_t ka[4];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const uint4 &x = k[r][i / 4];
                    const uint32_t w = (i & 3) == 0 ? x.x : (i & 3) == 1 ? x.y : (i & 3) == 2 ? x.z : x.w;
                    codes4_to_half<FMT>(w, ka[r], ka[2 + r]);
                }
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    const uint32_t *q = sm.q[mt][i][lane];
                    if (TWO) {
                        const uint4 f = *reinterpret_cast<const uint4 *>(q);
                        mma_f16(c[mt][n], ka, f.x, f.y);
                        mma_f16(small[mt], ka, f.z, f.w);
                    } else {
                        const uint2 f = *reinterpret_cast<const uint2 *>(q);
                        mma_f16(c[mt][n], ka, f.x, f.y);
                    }
                }
            }
            if (TWO) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) c[mt][n][e] += small[mt][e];
            }
        }
        // every row of the tile sees all of both pages
        bool all_whole = true;
#pragma unroll
        for (int n = 0; n < 2; ++n)
            all_whole = all_whole && there[n] && j0[n] + ROWS <= len && (!a.causal || j0[n] + ROWS - 1 <= t_lo) &&
                        (!a.window || j0[n] > t_hi - a.window || j0[n] + ROWS <= a.sinks);
        const float lv = log2_floor(fmaxf(vscale[0], vscale[1]));
        // probabilities
        uint32_t ph[MT][2][2], pl[MT][2][2];   // B fragments of P.V: keys 2 t, 2 t + 1 and 2 t + 8, 2 t + 9 of row g
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            uint32_t see = 0xFFu;         // bit 4 n + e: (key g, row 2 t), (g, 2 t + 1), (g + 8, 2 t), (g + 8, 2 t + 1) of page n
            float mx[2];
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) c[mt][n][e] *= qf[mt][e & 1] * kscale[n];
            if (all_whole) {
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    mx[e] = fmaxf(fmaxf(c[mt][0][e], c[mt][0][2 + e]), fmaxf(c[mt][1][e], c[mt][1][2 + e]));
            } else {
                mx[0] = mx[1] = -INFINITY;
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (there[n] && sees(a, tq[mt][e & 1], j0[n] + g + (e >> 1) * 8, len)) mx[e & 1] = fmaxf(mx[e & 1], c[mt][n][e]);
                        else see &= ~(1u << (4 * n + e));
                    }
            }
            if (__any_sync(0xffffffffu, unsettled(mx[0], lv, mref[mt][0], eo[mt][0]) ||
                                            unsettled(mx[1], lv, mref[mt][1], eo[mt][1]))) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
#pragma unroll
                    for (int x = 4; x < 32; x *= 2) mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], x));
                    const float d = move_m(mx[e], mref[mt][e]);
                    float need = -INFINITY;   // of the keys that this lane's row sees
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        const float ln = log2_floor(vscale[n]);
#pragma unroll
                        for (int h = 0; h < 4; h += 2)
                            if (see >> (4 * n + h + e) & 1) need = fmaxf(need, fmaxf(c[mt][n][h + e] - mref[mt][e], FAR) + ln);
                    }
#pragma unroll
                    for (int x = 4; x < 32; x *= 2) need = fmaxf(need, __shfl_xor_sync(0xffffffffu, need, x));
                    const float co = pow2i(move_e(need, d, eo[mt][e]));
                    l[mt][e] *= pow2i(fmaxf(d, -127.0f));
#pragma unroll
                    for (int j = 0; j < NJ; ++j) { o[mt][j][e] *= co; o[mt][j][2 + e] *= co; }
                }
            }
            float p[2][4], sub[2], vr[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                sub[e] = OFF - (mref[mt][e] == -INFINITY ? 0.0f : mref[mt][e]);
                vr[e] = pow2i(-eo[mt][e]);
            }
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) p[n][e] = ex2(c[mt][n][e] + sub[e & 1]);
            if (!all_whole) {
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!(see >> (4 * n + e) & 1)) p[n][e] = 0.0f;
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) l[mt][e] += (p[0][e] + p[0][2 + e]) + (p[1][e] + p[1][2 + e]);
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) p[n][e] *= vscale[n] * vr[e & 1];
            if (!all_whole) {             // a block that a row does not see adds nothing, whatever its scale
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!(see >> (4 * n + e) & 1)) p[n][e] = 0.0f;
            }
#pragma unroll
            for (int n = 0; n < 2; ++n) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t hi, lo;
                    if (TWO) {
                        split2(p[n][2 * h], p[n][2 * h + 1], hi, lo);
                        pl[mt][n][h] = transpose8(lo);
                    } else {
                        const __half2 x = __floats2half2_rn(p[n][2 * h], p[n][2 * h + 1]);
                        hi = *reinterpret_cast<const uint32_t *>(&x);
                    }
                    ph[mt][n][h] = transpose8(hi);
                }
            }
        }
        // O^T += V^T P^T
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const uint8_t *vp = sm.kv[warp][(it + n) % STAGES][1];
            uint32_t v[4][VB / 4];        // keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = 2 * t + (r & 1) + (r >> 1) * 8;
                if (VB == 16) {
                    const uint4 x = *reinterpret_cast<const uint4 *>(vp + row * D + ((g ^ swz<D>(row)) << 4));
                    v[r][0] = x.x; v[r][1] = x.y; v[r][VB / 4 - 2] = x.z; v[r][VB / 4 - 1] = x.w;
                } else {
                    const uint2 x = *reinterpret_cast<const uint2 *>(vp + row * D + (((g >> 1) ^ swz<D>(row)) << 4) + (g & 1) * 8);
                    v[r][0] = x.x; v[r][1] = x.y;
                }
            }
            if (!all_whole && (!there[n] || j0[n] + ROWS > len)) {   // what is not a row may hold anything
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (!there[n] || j0[n] + 2 * t + (r & 1) + (r >> 1) * 8 >= len)
#pragma unroll
                        for (int w = 0; w < VB / 4; ++w) v[r][w] = 0;
            }
#pragma unroll
            for (int w = 0; w < VB / 4; ++w) {
                uint32_t x[2][4];         // [key pair][dim of the word]: codes of two keys of one dim as fp16
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    codes4_to_half<FMT>(__byte_perm(v[2 * h][w], v[2 * h + 1][w], 0x5140), x[h][0], x[h][1]);
                    codes4_to_half<FMT>(__byte_perm(v[2 * h][w], v[2 * h + 1][w], 0x7362), x[h][2], x[h][3]);
                }
#pragma unroll
                for (int d = 0; d < 2; ++d) {
                    const uint32_t va[4] = {x[0][2 * d], x[0][2 * d + 1], x[1][2 * d], x[1][2 * d + 1]};
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        float (&acc)[4] = o[mt][w * 2 + d];
                        if (TWO) {        // a page's sum alone on the tensor core, small parts first; rounded into the rest
                            float x4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                            mma_f16(x4, va, pl[mt][n][0], pl[mt][n][1]);
                            mma_f16(x4, va, ph[mt][n][0], ph[mt][n][1]);
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[e] += x4[e];
                        } else {
                            mma_f16(acc, va, ph[mt][n][0], ph[mt][n][1]);
                        }
                    }
                }
            }
        }
        __syncwarp();                     // the stages are read
        issue(it + STAGES);
        issue(it + STAGES + 1);
    }

    // ---- the four warps' results -> one
    __syncthreads();                      // every warp has read its last stage
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float x = l[mt][e];
#pragma unroll
            for (int y = 4; y < 32; y *= 2) x += __shfl_xor_sync(0xffffffffu, x, y);
            const int row = mt * 8 + 2 * t + e;
            if (g == 0) { sm.m[warp][row] = mref[mt][e]; sm.l[warp][row] = x; }
            float *dst = sm.o[warp][row] + g * VB;
            // each warp's own mean of V: no sum of values can overflow (nor 2^eo / l underflow)
            const float inv = x == 0.0f ? 0.0f : 1.0f / x, E = pow2i(eo[mt][e]);
#pragma unroll
            for (int j = 0; j < NJ; j += 2)
                *reinterpret_cast<float4 *>(dst + 2 * j) =
                    make_float4(o[mt][j][e] * inv * E, o[mt][j][2 + e] * inv * E, o[mt][j + 1][e] * inv * E,
                                o[mt][j + 1][2 + e] * inv * E);
        }
    __syncthreads();
    const size_t rows_all = (size_t)a.n_rows * a.heads;
    for (int i = threadIdx.x; i < 8 * MT * (D / 4); i += 128) {
        const int row = i / (D / 4), d = (i % (D / 4)) * 4;
        if (row >= M) continue;
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) mx = fmaxf(mx, sm.m[w][row]);
        const float ref = mx == -INFINITY ? 0.0f : mx;
        float lw[4], lsum = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) lsum += lw[w] = sm.l[w][row] * ex2(sm.m[w][row] - ref);
        const float inv = lsum == 0.0f ? 0.0f : 1.0f / lsum;       // a row that sees nothing: zeros
        float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = lw[w] * inv;
            const float4 x = *reinterpret_cast<const float4 *>(&sm.o[w][row][d]);
            acc.x += x.x * f; acc.y += x.y * f; acc.z += x.z * f; acc.w += x.w * f;
        }
        if (a.cluster) {
            *reinterpret_cast<float4 *>(&sm.o[0][row][d]) = acc;   // this thread alone reads and writes this place
            if (d == 0) sm.ml[row] = make_float2(mx, lsum);
            continue;
        }
        const int qi = row_of(row), h = hk * G + row - qi * G;
        const size_t r = (size_t)sp.first + qi;
        if (pieces == 1) {
            store4(static_cast<T *>(a.out) + r * a.ldo + (size_t)h * D + d, acc.x, acc.y, acc.z, acc.w);
        } else {
            const size_t b = (r * a.heads + h) * a.max_chunks + piece;
            *reinterpret_cast<float4 *>(a.part + b * D + d) = acc;
            if (d == 0) *reinterpret_cast<float2 *>(a.part + rows_all * a.max_chunks * D + b * 2) = make_float2(mx, lsum);
        }
    }
    if (!a.cluster) return;
    // The cluster's CTAs share out the values; pieces in order.
    cluster_sync();
    for (int i = piece * 128 + threadIdx.x; i < 8 * MT * (D / 4); i += a.max_chunks * 128) {
        const int row = i / (D / 4), d = (i % (D / 4)) * 4;
        if (row >= M) break;
        float mc[8], lc[8], mx = -INFINITY, lsum = 0.0f;           // a cluster has 8 pieces at most
#pragma unroll
        for (int c = 0; c < 8; ++c)
            if (c < pieces) {
                mc[c] = dsmem_ld(dsmem_addr(smem_u32(&sm.ml[row].x), c));
                lc[c] = dsmem_ld(dsmem_addr(smem_u32(&sm.ml[row].y), c));
                mx = fmaxf(mx, mc[c]);
            }
        const float ref = mx == -INFINITY ? 0.0f : mx;
#pragma unroll
        for (int c = 0; c < 8; ++c)
            if (c < pieces) lsum += lc[c] *= ex2(mc[c] - ref);
        const float inv = lsum == 0.0f ? 0.0f : 1.0f / lsum;
        float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int c = 0; c < 8; ++c)
            if (c < pieces) {
                const float f = lc[c] * inv;
                const float4 x = dsmem_ld4(dsmem_addr(smem_u32(&sm.o[0][row][d]), c));
                acc.x = fmaf(x.x, f, acc.x); acc.y = fmaf(x.y, f, acc.y); acc.z = fmaf(x.z, f, acc.z); acc.w = fmaf(x.w, f, acc.w);
            }
        const int qi = row_of(row), h = hk * G + row - qi * G;
        store4(static_cast<T *>(a.out) + ((size_t)sp.first + qi) * a.ldo + (size_t)h * D + d, acc.x, acc.y, acc.z, acc.w);
    }
    cluster_sync();                       // nobody leaves while its results are being read
}

// Joins the pieces of each row, each of them the mean of its own V rows with the
// reference m and the sum l of its probabilities, by weights that add up to 1: a warp
// per row, pieces in order, eight loads in flight (3 us for 512 rows of two pieces;
// launch latency is hidden behind the kernel before it).
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
        for (int c = lane; c < pieces; c += 32) l += ml[c].y * ex2(ml[c].x - ref);
        l = warp_sum(l);
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int i = 0; i < W; ++i) acc[i] = 0.0f;
#pragma unroll 8
        for (int c = 0; c < pieces; ++c) {
            const float2 x = ml[c];
            const float f = x.y * ex2(x.x - ref) * inv;
            const float *src = a.part + (b + c) * D + lane * W;
#pragma unroll
            for (int i = 0; i < W; ++i) acc[i] = fmaf(src[i], f, acc[i]);
        }
        T *dst = static_cast<T *>(a.out) + r * a.ldo + (size_t)h * D + lane * W;
        if (W == 4) {
            store4(dst, acc[0], acc[1], acc[W - 2], acc[W - 1]);
        } else if (sizeof(T) == 4) {
            *reinterpret_cast<float2 *>(dst) = make_float2(acc[0], acc[1]);
        } else {
            *reinterpret_cast<__nv_bfloat162 *>(dst) = __floats2bfloat162_rn(acc[0], acc[1]);
        }
    }
}

}  // namespace kv8
}  // namespace ct
