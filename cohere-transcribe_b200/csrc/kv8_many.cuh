// kv8_many.cuh -- attention of many query rows over the 8-bit paged cache on the
// 5th-generation tensor cores (include/ct_kv8.h).
//
// One CTA per (tile of query rows, kv head, sequence, piece of the page list);
// as in the kernel for few rows, a row is a (query row, head of the group) pair.
// Two streams share the CTA's key tiles (128 keys = 8 pages); each has a
// warpgroup that owns its 128 rows (a thread per row = TMEM lane), a score tile
// S [128 x 128] and an accumulator O [128 x D] in TMEM:
//   bf16 rows: the streams are two tiles of 128 rows, both over every key tile;
//   fp32 rows: the streams are the even and the odd key tiles of the same 128
//   rows, held as high and low fp16 parts (two MMAs each for Q.K and P.V), and
//   are joined at the end like two pieces of a split.
// While one stream's rows are in their softmax the tensor core works for the
// other: step k issues P.V of item k - 2 and Q.K of item k, where items
// alternate between the streams.  Two MMAs of one thread are ordered only when they
// share accumulator and shape (the PTX ISA's list of pipelined tcgen05 pairs), so
// Q.K of item k, which overwrites the P that P.V of item k - 2 reads, waits for that
// P.V (pdone).  A commit covers all earlier MMAs of its thread: once scores are
// there (sfull), the stream's O may be rescaled and S overwritten by P.
//
// Operands: Q as fp16, each row scaled by a power of two.  Codes are exact in
// fp16: a warpgroup loads them from global memory a tile ahead, converts, and
// writes K and V alike as [key][64 dims] rows of 128 bytes with the 128-byte
// swizzle; Q.K reads K that way K-major, P.V reads V MN-major (dims
// contiguous), so nothing is transposed.  Block scales never touch the
// operands: K's multiply the scores (one factor per 16 columns), V's the
// probabilities, in units of a power of two per row that O is held in.
// P [128 x 128] fp16 replaces S in TMEM as the A operand: the 32 columns of 32
// scores hold their high parts in the first 16 and their low parts in the rest.
//
// Measured: 4 prompts of 1000 to 4097 bf16 rows, 32 heads on 8, 679 GFLOP in 955 us
// (711 TFLOP/s; 24 us of it for waiting with Q.K until P.V is finished); windowed fp32
// prompts, 62 GFLOP (every product as two MMAs), 281 us.  No unit is the bound (tensor
// pipe 34%, exponentials 37%, issue slots 41%): a stream's chain is, about 3.1
// thousand cycles of softmax and over 2 thousand until its next scores are there, per
// tile of 128 keys.  128 keys a tile keep the chain's
// fixed part small; the straight-line softmax with all scores in registers replaced
// loops over 32 of them (1450 us).
#pragma once
#include <type_traits>

#include "kv8_attn.cuh"

namespace ct {
namespace kv8 {

// Warps 0..3: MMA issue (warp 0); 4..7: codes -> fp16; 8..15: the streams.  A
// softmax thread keeps its row's 128 scores in registers, so the warpgroups
// split the launch's 4 x 128 registers per lane as 40 + 104 + 184 + 184 (the MMA
// thread is on the critical path: with 24 registers windowed fp32 prompts take 352
// us instead of 283, and its loop over the two parts stays rolled, 275).
constexpr int MANY_THREADS = 512;
constexpr int KT = 128;             // keys of a tile
constexpr int KB = KT / ROWS;       // blocks of a tile
constexpr int ABSENT = INT_MAX - 64;   // behind every length

template <int D>
struct ManySmem {
    uint8_t q[2][D / 64][128 * 128];     // [tile or part][64 dims][row]
    uint8_t kv[4][D / 64][KT * 128];     // ring: K of tile 0, V of tile 0, K of tile 1, ...
    float ks[4][KB], vs[4][KB];          // block scales of a tile
    int base[4][KB];                     // first token row of each block; ABSENT = not there
    float qf[256];                       // per row: scale_log2 / power of two of its query
    float join[3][128];
    uint64_t full[4], freed[4], sfull[2], pfull[2], pdone[2], ofull[2], qfull;
    uint32_t tmem;
};

// Bounded wait; gives up as well once any wait of the library has run out.
__device__ __forceinline__ bool many_wait(uint64_t *bar, uint32_t parity, int code) {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = globaltimer();
    for (uint32_t it = 0;; ++it) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((it & 255u) == 255u) {
            const int st = *reinterpret_cast<volatile int *>(&g_ct_status);
            if (st >= CT_STATUS_TIMEOUT_TMA && st <= CT_STATUS_TIMEOUT_FREE) return false;
            if (globaltimer() - t0 > CT_WAIT_NS) { set_status(code); return false; }
        }
    }
}

__device__ __forceinline__ void tmem_store16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
        ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
          "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_store32(uint32_t taddr, const float (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
        ::"r"(taddr), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]),
          "f"(v[8]), "f"(v[9]), "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15]),
          "f"(v[16]), "f"(v[17]), "f"(v[18]), "f"(v[19]), "f"(v[20]), "f"(v[21]), "f"(v[22]), "f"(v[23]),
          "f"(v[24]), "f"(v[25]), "f"(v[26]), "f"(v[27]), "f"(v[28]), "f"(v[29]), "f"(v[30]), "f"(v[31])
        : "memory");
}
// 128 consecutive TMEM columns, one wait for all.
__device__ __forceinline__ void tmem_load128(uint32_t taddr, float (&v)[128]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%128];\n\t"
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%129];\n\t"
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%64,%65,%66,%67,%68,%69,%70,%71,%72,%73,%74,%75,%76,%77,%78,%79,%80,%81,%82,%83,%84,%85,%86,%87,%88,%89,%90,%91,%92,%93,%94,%95}, [%130];\n\t"
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%96,%97,%98,%99,%100,%101,%102,%103,%104,%105,%106,%107,%108,%109,%110,%111,%112,%113,%114,%115,%116,%117,%118,%119,%120,%121,%122,%123,%124,%125,%126,%127}, [%131];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]),
          "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31]),
          "=f"(v[32]), "=f"(v[33]), "=f"(v[34]), "=f"(v[35]), "=f"(v[36]), "=f"(v[37]), "=f"(v[38]), "=f"(v[39]), "=f"(v[40]), "=f"(v[41]), "=f"(v[42]), "=f"(v[43]), "=f"(v[44]), "=f"(v[45]), "=f"(v[46]), "=f"(v[47]),
          "=f"(v[48]), "=f"(v[49]), "=f"(v[50]), "=f"(v[51]), "=f"(v[52]), "=f"(v[53]), "=f"(v[54]), "=f"(v[55]), "=f"(v[56]), "=f"(v[57]), "=f"(v[58]), "=f"(v[59]), "=f"(v[60]), "=f"(v[61]), "=f"(v[62]), "=f"(v[63]),
          "=f"(v[64]), "=f"(v[65]), "=f"(v[66]), "=f"(v[67]), "=f"(v[68]), "=f"(v[69]), "=f"(v[70]), "=f"(v[71]), "=f"(v[72]), "=f"(v[73]), "=f"(v[74]), "=f"(v[75]), "=f"(v[76]), "=f"(v[77]), "=f"(v[78]), "=f"(v[79]),
          "=f"(v[80]), "=f"(v[81]), "=f"(v[82]), "=f"(v[83]), "=f"(v[84]), "=f"(v[85]), "=f"(v[86]), "=f"(v[87]), "=f"(v[88]), "=f"(v[89]), "=f"(v[90]), "=f"(v[91]), "=f"(v[92]), "=f"(v[93]), "=f"(v[94]), "=f"(v[95]),
          "=f"(v[96]), "=f"(v[97]), "=f"(v[98]), "=f"(v[99]), "=f"(v[100]), "=f"(v[101]), "=f"(v[102]), "=f"(v[103]), "=f"(v[104]), "=f"(v[105]), "=f"(v[106]), "=f"(v[107]), "=f"(v[108]), "=f"(v[109]), "=f"(v[110]), "=f"(v[111]),
          "=f"(v[112]), "=f"(v[113]), "=f"(v[114]), "=f"(v[115]), "=f"(v[116]), "=f"(v[117]), "=f"(v[118]), "=f"(v[119]), "=f"(v[120]), "=f"(v[121]), "=f"(v[122]), "=f"(v[123]), "=f"(v[124]), "=f"(v[125]), "=f"(v[126]), "=f"(v[127])
        : "r"(taddr + 0u), "r"(taddr + 32u), "r"(taddr + 64u), "r"(taddr + 96u)
        : "memory");
}
// Two fp32 operations in one instruction.
__device__ __forceinline__ unsigned long long pack2(float2 a) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a.x), "f"(a.y));
    return r;
}
__device__ __forceinline__ float2 unpack2(unsigned long long r) {
    float2 a;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a.x), "=f"(a.y) : "l"(r));
    return a;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(pack2(a)), "l"(pack2(b)), "l"(pack2(c)));
    return unpack2(r);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pack2(a)), "l"(pack2(b)));
    return unpack2(r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pack2(a)), "l"(pack2(b)));
    return unpack2(r);
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// D[tmem] (+)= A[tmem] * B[smem], fp16 operands
__device__ __forceinline__ void mma_f16_ta(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                           uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Instruction descriptor, kind::f16: fp16 A / B, fp32 D; B MN-major if b_mn.
__host__ __device__ constexpr uint32_t idesc_f16(int M, int N, bool b_mn) {
    return (1u << 4) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
// MN-major operand with the 128-byte swizzle: 64 contiguous values per row, 8
// rows (of the K dimension) per 1024-byte group (SBO), the next 64 values KT
// rows further (LBO).
__device__ __forceinline__ uint64_t sw128_mn_desc(uint32_t smem_addr) {
    return (sw128_desc(smem_addr) & ~((uint64_t)0x3FFF << 16)) | ((uint64_t)((KT * 128) >> 4) << 16);
}

template <typename T, int D, int FMT>
__global__ void __launch_bounds__(MANY_THREADS, 1) many_kernel(const AttnArgs a) {
    constexpr bool TWO = sizeof(T) == 4;
    constexpr int TILE = TWO ? 128 : 256;
    constexpr int NB = D / 64;
    constexpr uint32_t COL_S = 0, COL_O = 256;  // S of stream i at 128 i, O at 256 + 128 i
    extern __shared__ __align__(1024) uint8_t many_raw[];
    ManySmem<D> &sm = *reinterpret_cast<ManySmem<D> *>((reinterpret_cast<uintptr_t>(many_raw) + 1023) & ~(uintptr_t)1023);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int s = blockIdx.z, hk = blockIdx.y, piece = blockIdx.x % a.max_chunks;
    const int tile = gridDim.x / a.max_chunks - 1 - blockIdx.x / a.max_chunks;   // long rows first
    pdl_trigger();
    const RowSpan sp = row_span(a.len, a.row_start, s, a.n_rows, a.max_rows, min(a.stride * ROWS, a.max_len));
    if (!sp.ok) {
        if (threadIdx.x == 0 && piece == 0) set_status(CT_STATUS_BAD_ARG);
        return;
    }
    const int G = a.group, M = sp.n * G, m0 = tile * TILE;
    if (m0 >= M) return;
    const int len = max(sp.len, 0), t_first = len - sp.n;
    const PageList list =
        page_list(a, len, t_first + m0 / G, t_first + (min(m0 + TILE, M) - 1) / G);
    const int pieces = max(1, (list.n + a.chunk - 1) / a.chunk);
    if (piece >= pieces) return;
    const int e0 = piece * a.chunk, e1 = min(list.n, e0 + a.chunk);
    // row r of the tile: query row i0 + (g0 + r) / G, head (g0 + r) % G of the group; g0 + r
    // < 1280, so the quotient by a float reciprocal is exact
    const int i0 = m0 / G, g0 = m0 - i0 * G;
    const float rg = 1.0f / (float)G;
    auto row_of = [&](int r) { return (int)((g0 + r + 0.5f) * rg); };
    const int nt = max(1, (e1 - e0 + KB - 1) / KB);        // key tiles (one without keys for rows that see none)
    const int items = TWO ? nt : 2 * nt;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 4; ++i) { mbar_init(&sm.full[i], 128); mbar_init(&sm.freed[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&sm.sfull[i], 1); mbar_init(&sm.pfull[i], 128); mbar_init(&sm.pdone[i], 1); mbar_init(&sm.ofull[i], 1); }
        mbar_init(&sm.qfull, 256);
        fence_mbar_init();
    }
    if (warp == 0) { tmem_alloc(&sm.tmem, 512); tmem_relinquish(); }

    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem;

    if (warp < 4) {
        // -------------------------------------------------------------- MMA issue
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        if (warp == 0 && lane == 0) {
            constexpr uint32_t id_s = idesc_f16(128, KT, false), id_o = idesc_f16(128, D, true);
            bool ok = many_wait(&sm.qfull, 0, CT_STATUS_TIMEOUT_TMA);
            for (int k = 0; k < items + 2 && ok; ++k) {
                const int i = k & 1;                       // items k - 2 and k belong to the same stream
                if (k >= 2 && k - 2 < items) {
                    const int j = TWO ? k - 2 : (k - 2) >> 1, n = 2 * j + 1;
                    ok = many_wait(&sm.full[n & 3], (n >> 2) & 1, CT_STATUS_TIMEOUT_TMA) &&
                         many_wait(&sm.pfull[i], ((k - 2) >> 1) & 1, CT_STATUS_TIMEOUT_MMA);
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t vd = sw128_mn_desc(smem_u32(sm.kv[n & 3][0]));
#pragma unroll 1
                    for (int p = TWO ? 1 : 0; p >= 0; --p)
#pragma unroll
                        for (int c = 0; c < KT / 16; ++c)
                            mma_f16_ta(tmem + COL_O + 128 * i, tmem + COL_S + 128 * i + 32 * (c >> 1) + 16 * p + 8 * (c & 1), vd + 128 * c, id_o,
                                       (k >= 4 || c || (TWO && p == 0)) ? 1u : 0u);
                    if (TWO || i) mma_commit(&sm.freed[n & 3]);
                    mma_commit(k < items ? &sm.pdone[i] : &sm.ofull[i]);
                }
                if (k < items) {
                    const int j = TWO ? k : k >> 1, n = 2 * j;
                    ok = many_wait(&sm.full[n & 3], (n >> 2) & 1, CT_STATUS_TIMEOUT_TMA) &&
                         (k < 2 || many_wait(&sm.pdone[i], ((k - 2) >> 1) & 1, CT_STATUS_TIMEOUT_MMA));
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll 1
                    for (int p = TWO ? 1 : 0; p >= 0; --p)   // the small parts first: sums are truncated at every step
#pragma unroll
                        for (int b = 0; b < NB; ++b) {
                            const uint64_t qd = sw128_desc(smem_u32(sm.q[TWO ? p : i][b]));
                            const uint64_t kd = sw128_desc(smem_u32(sm.kv[n & 3][b]));
#pragma unroll
                            for (int c = 0; c < 4; ++c)
                                mma_bf16(tmem + COL_S + 128 * i, qd + 2 * c, kd + 2 * c, id_s, ((TWO && p == 0) || b || c) ? 1u : 0u);
                        }
                    mma_commit(&sm.sfull[i]);
                    if (TWO || i) mma_commit(&sm.freed[n & 3]);
                }
            }
        }
    } else if (warp < 8) {
        // ------------------------------------------------------- codes -> fp16 tiles
        asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
        // Lane (row, 16-byte chunk of 4): 8 rows of 64 bytes a pass.  Both the loads
        // (whole sectors) and the 16-byte stores into swizzled rows (two rows' even
        // and odd chunks) meet no bank twice.
        constexpr int PASSES = 4 * NB;
        const int w = warp - 4, c = lane & 3, rl = lane >> 2;
        const int *trow = a.table + (size_t)s * a.stride;
        // Everything is fetched well before its use: page numbers two tiles ahead,
        // block scales and K codes while the V before them is converted, V codes
        // while the K before them is.
        uint4 x[2][PASSES];                                // K, V codes of the next tile to convert
        int page[2], base[2], next[2];                     // of this warp's 32 rows; next: raw table entries
        float ks = 0.0f, vs = 0.0f;                        // lane b < 2: of block b
        auto fetch = [&](int j) {
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int e = e0 + j * KB + w * 2 + b;
                next[b] = e < e1 ? trow[list.at(e)] : -1;
            }
        };
        auto resolve = [&](int j) {                        // next -> page, base of tile j; scales
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int e = e0 + j * KB + w * 2 + b;
                const bool there = e < e1 && a.p.has(next[b]);
                page[b] = there ? next[b] : -1;
                base[b] = there ? list.at(e) * ROWS : ABSENT;
                if (e < e1 && !there && lane == 0) set_status(CT_STATUS_BAD_ARG);   // its rows count as not there
            }
            const int pg = lane ? page[1] : page[0];
            ks = vs = 0.0f;
            if (lane < 2 && pg >= 0) {
                const size_t at = a.p.block(pg, a.layer, 0, hk);
                ks = a.p.scales[at];
                vs = a.p.scales[at + a.p.heads];
            }
        };
        auto load = [&](int kv) {
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const uint8_t *src = a.p.codes + a.p.block(page[b], a.layer, kv, hk) * (ROWS * D) + rl * D + c * 16;
                const int rows = len - base[b];            // rows behind the last one may hold anything
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int h = 0; h < NB; ++h) {
                        uint4 &y = x[kv][(b * 2 + i) * NB + h];
                        y = make_uint4(0, 0, 0, 0);
                        if (i * 8 + rl < rows) y = *reinterpret_cast<const uint4 *>(src + i * 8 * D + h * 64);
                    }
            }
        };
        auto convert = [&](int kv, int slot) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int h = 0; h < NB; ++h) {
                    const int r = w * 32 + i * 8 + rl;     // r & 7 = rl
                    const uint4 &y = x[kv][i * NB + h];
                    uint4 f[2];
                    codes4_to_half<FMT>(y.x, f[0].x, f[0].y);
                    codes4_to_half<FMT>(y.y, f[0].z, f[0].w);
                    codes4_to_half<FMT>(y.z, f[1].x, f[1].y);
                    codes4_to_half<FMT>(y.w, f[1].z, f[1].w);
                    uint8_t *row = &sm.kv[slot][h][r * 128];
                    *reinterpret_cast<uint4 *>(row + (((2 * c) ^ rl) << 4)) = f[0];
                    *reinterpret_cast<uint4 *>(row + (((2 * c + 1) ^ rl) << 4)) = f[1];
                }
            fence_proxy_async_smem();
            mbar_arrive(&sm.full[slot]);
        };
        fetch(0);
        resolve(0);
        load(0);
        load(1);
        if (nt > 1) fetch(1);
        for (int j = 0; j < nt; ++j) {
            const int sk = (2 * j) & 3, sv = sk + 1;       // ring slots of this tile's K and V
            const uint32_t par = ((j >> 1) - 1) & 1;
            if (j >= 2 && !many_wait(&sm.freed[sk], par, CT_STATUS_TIMEOUT_FREE)) break;
            if (lane < 2) {
                const int b = w * 2 + lane;
                sm.base[j & 3][b] = lane ? base[1] : base[0];
                sm.ks[j & 3][b] = ks;
                sm.vs[j & 3][b] = vs;
            }
            convert(0, sk);
            if (j + 1 < nt) { resolve(j + 1); load(0); }
            if (j + 2 < nt) fetch(j + 2);
            if (j >= 2 && !many_wait(&sm.freed[sv], par, CT_STATUS_TIMEOUT_FREE)) break;
            convert(1, sv);
            if (j + 1 < nt) load(1);
        }
    } else {
        // ---------------------------------------------------------------- softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");
        {
            // queries -> fp16, K-major rows of 64 dims: every load of a warp's rows in flight at once
            constexpr int EPL = 16 / sizeof(T), LPR = D / EPL, RPP = 32 / LPR, N = TILE / 8 / RPP;
            const int c = lane % LPR, r0 = (warp - 8) * (TILE / 8) + lane / LPR;
            uint4 x[N];
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const int r = r0 + n * RPP, q = row_of(r);
                x[n] = make_uint4(0, 0, 0, 0);
                if (m0 + r < M)
                    x[n] = *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.q) + (size_t)(sp.first + i0 + q) * a.ldq +
                                                            (size_t)(hk * G + g0 + r - q * G) * D + c * EPL);
            }
            float amax[N];
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const T *e = reinterpret_cast<const T *>(&x[n]);
                amax[n] = 0.0f;
#pragma unroll
                for (int j = 0; j < EPL; ++j) amax[n] = fmaxf(amax[n], fabsf(to_f32(e[j])));
            }
#pragma unroll
            for (int o = 1; o < LPR; o *= 2)
#pragma unroll
                for (int n = 0; n < N; ++n) amax[n] = fmaxf(amax[n], __shfl_xor_sync(0xffffffffu, amax[n], o));
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const T *e = reinterpret_cast<const T *>(&x[n]);
                const float p2 = row_pow2(amax[n]);
                const int r = r0 + n * RPP, rr = r & 127, d = c * EPL;
                if (c == 0) sm.qf[r] = a.scale_log2 * inv_pow2(p2);
                uint32_t hi[EPL / 2], lo[EPL / 2];
#pragma unroll
                for (int j = 0; j < EPL; j += 2) split2(to_f32(e[j]) * p2, to_f32(e[j + 1]) * p2, hi[j / 2], lo[j / 2]);
                uint8_t *dst = sm.q[TWO ? 0 : r >> 7][d >> 6] + rr * 128 + ((((d & 63) >> 3) ^ (rr & 7)) << 4) + (d & 7) * 2;
                if (TWO) {
                    *reinterpret_cast<uint2 *>(dst) = make_uint2(hi[0], hi[1]);
                    *reinterpret_cast<uint2 *>(dst + sizeof(sm.q[0])) = make_uint2(lo[0], lo[1]);
                } else {
                    *reinterpret_cast<uint4 *>(dst) = make_uint4(hi[0], hi[1], hi[EPL / 2 - 2], hi[EPL / 2 - 1]);
                }
            }
            fence_proxy_async_smem();
            mbar_arrive(&sm.qfull);
            asm volatile("bar.sync 1, 256;" ::: "memory");   // qf of every row
        }
        const int i = (warp - 8) >> 2, qw = warp & 3, ql = qw * 32 + lane;
        const uint32_t lane_off = (uint32_t)(qw * 32) << 16;
        const uint32_t ts = tmem + lane_off + COL_S + 128 * i, to = tmem + lane_off + COL_O + 128 * i;
        const int r = TWO ? ql : i * 128 + ql, m = m0 + r;
        const float rf = sm.qf[r];
        const int t = t_first + i0 + row_of((m < M ? m : M - 1) - m0);
        const int hi = a.causal ? max(0, min(len, t + 1)) : len;   // sees j < hi and (j >= lo or j < sinks)
        const int lo = a.window ? max(0, t - a.window + 1) : 0;
        float mref = -INFINITY, l = 0.0f, eo = E_MIN;      // O is held in units of 2^eo
        bool ok = true;
        const int mine = TWO ? (nt - i + 1) / 2 : nt;      // tiles of this stream
        for (int k = 0; k < mine; ++k) {
            const int j = TWO ? 2 * k + i : k;
            ok = many_wait(&sm.sfull[i], k & 1, CT_STATUS_TIMEOUT_MMA);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            const float *ks = sm.ks[j & 3], *vs = sm.vs[j & 3];
            const int *base = sm.base[j & 3];
            // whether the row sees every key of the tile
            bool every = true;
#pragma unroll
            for (int b = 0; b < KB; ++b) {
                const int j0 = base[b];
                every = every && j0 + ROWS <= hi && (j0 >= lo || j0 + ROWS <= a.sinks);
            }
            float mx = -INFINITY, vmax = 0.0f, xb[KB];     // largest score of all, of each block
            float sub, inv;
            // moves the reference and the unit when this tile asks for it
            auto settle = [&]() {
                const bool look = unsettled(mx, log2_floor(vmax), mref, eo);
                if (__any_sync(0xffffffffu, look)) {
                    const float d = move_m(mx, mref);
                    float need = -INFINITY;
#pragma unroll
                    for (int b = 0; b < KB; ++b)
                        if (xb[b] != -INFINITY) need = fmaxf(need, fmaxf(xb[b] - mref, FAR) + log2_floor(vs[b]));
                    const float co = pow2i(move_e(need, d, eo));
                    l *= pow2i(fmaxf(d, -127.0f));
                    if (k > 0 && __any_sync(0xffffffffu, co != 1.0f)) {
#pragma unroll 1
                        for (int c = 0; c < D / 32; ++c) {
                            float o[32];
                            tmem_ld32(to + 32 * c, o);
#pragma unroll
                            for (int q = 0; q < 32; ++q) o[q] *= co;
                            tmem_store32(to + 32 * c, o);
                        }
                    }
                }
                sub = OFF - (mref == -INFINITY ? 0.0f : mref);
                inv = pow2i(-eo);
            };
            auto pack = [&](const float *v, int c) {       // 32 probabilities -> TMEM, over their scores
                uint32_t phi[16], plo[16];
#pragma unroll
                for (int q = 0; q < 16; ++q) {
                    if (TWO) {
                        split2(v[2 * q], v[2 * q + 1], phi[q], plo[q]);
                    } else {
                        const __half2 p2 = __floats2half2_rn(v[2 * q], v[2 * q + 1]);
                        phi[q] = *reinterpret_cast<const uint32_t *>(&p2);
                    }
                }
                tmem_store16(ts + 32 * c, phi);
                if (TWO) tmem_store16(ts + 32 * c + 16, plo);
            };
            float2 l2[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
            // The tile's softmax as straight-line code, once without and once with hidden keys.
            auto tile_softmax = [&](auto masked) {
                constexpr bool MASKED = decltype(masked)::value;
                float v[KT];
                tmem_load128(ts, v);
#pragma unroll
                for (int b = 0; b < KB; ++b) {
                    uint32_t see = 0xFFFFu;                // bit q: key q of the block is seen
                    if (MASKED) {                          // hidden scores become -inf
                        auto below = [&](int n) { return (1u << min(max(n - base[b], 0), ROWS)) - 1u; };   // keys j < n
                        see = below(hi) & (~below(lo) | below(a.sinks));
#pragma unroll
                        for (int q = 0; q < 16; ++q)
                            if (!(see >> q & 1)) v[16 * b + q] = -INFINITY;
                    }
                    float bm[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        bm[q] = fmaxf(fmaxf(v[16 * b + q], v[16 * b + 4 + q]), fmaxf(v[16 * b + 8 + q], v[16 * b + 12 + q]));
                    const float x = fmaxf(fmaxf(bm[0], bm[1]), fmaxf(bm[2], bm[3])) * (rf * ks[b]);
                    xb[b] = -INFINITY;
                    if (!MASKED || see) {
                        xb[b] = x;
                        mx = fmaxf(mx, x);
                        vmax = fmaxf(vmax, vs[b]);
                    }
                }
                settle();
#pragma unroll
                for (int b = 0; b < KB; ++b) {
                    const float f = rf * ks[b], vr = vs[b] * inv;
                    float2 *x = reinterpret_cast<float2 *>(&v[16 * b]);
#pragma unroll
                    for (int q = 0; q < 8; ++q) {
                        const bool h0 = MASKED && x[q].x == -INFINITY, h1 = MASKED && x[q].y == -INFINITY;
                        float2 p = fma2(x[q], make_float2(f, f), make_float2(sub, sub));
                        p.x = h0 ? 0.0f : ex2(p.x);        // a hidden key adds nothing, whatever its block's scales
                        p.y = h1 ? 0.0f : ex2(p.y);
                        l2[q & 1] = add2(l2[q & 1], p);
                        p = mul2(p, make_float2(vr, vr));
                        x[q] = make_float2(h0 ? 0.0f : p.x, h1 ? 0.0f : p.y);
                    }
                    if (b & 1) pack(&v[16 * (b - 1)], b >> 1);
                }
            };
            if (__all_sync(0xffffffffu, every)) tile_softmax(std::false_type());
            else tile_softmax(std::true_type());
            l += (l2[0].x + l2[0].y) + (l2[1].x + l2[1].y);
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(&sm.pfull[i]);
        }
        // --------------------------------------------------------------- epilogue
        if (ok && mine > 0) ok = many_wait(&sm.ofull[i], 0, CT_STATUS_TIMEOUT_MMA);
        if (TWO && ok && nt > 1) ok = many_wait(&sm.ofull[1 - i], 0, CT_STATUS_TIMEOUT_MMA);   // the ring is free
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
        float *oj = reinterpret_cast<float *>(sm.kv);      // [D][128]: stream 1's O for the join
        if (TWO && nt > 1) {
            if (i == 1) {
#pragma unroll 1
                for (int c = 0; ok && c < D / 32; ++c) {
                    float v[32];
                    tmem_ld32(to + 32 * c, v);
#pragma unroll
                    for (int q = 0; q < 32; ++q) oj[(32 * c + q) * 128 + ql] = v[q];
                }
                sm.join[0][ql] = mref;
                sm.join[1][ql] = l;
                sm.join[2][ql] = eo;
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");
        }
        if (ok && (!TWO || i == 0)) {
            // The mean of this piece's V, not their sum: O / l first, then the unit, so that
            // neither the values' sum overflows nor 2^eo / l underflows.
            float f0 = 1.0f, f1 = 0.0f, e1 = 0.0f;
            const float e0 = pow2i(eo);
            if (TWO && nt > 1) {
                const float m1 = sm.join[0][ql], mn = fmaxf(mref, m1), ref = mn == -INFINITY ? 0.0f : mn;
                f0 = ex2(mref - ref);
                f1 = ex2(m1 - ref);
                l = l * f0 + sm.join[1][ql] * f1;
                e1 = pow2i(sm.join[2][ql]);
                mref = mn;
            }
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;       // a row that sees nothing: zeros
            f0 *= inv;
            f1 *= inv;
            const bool store = m < M;
            const int q = row_of(r), h = hk * G + g0 + r - q * G;
            const size_t row = (size_t)sp.first + (store ? i0 + q : 0);
            T *dst = static_cast<T *>(a.out) + row * a.ldo + (size_t)h * D;
            const size_t b = (row * a.heads + h) * a.max_chunks + piece;
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
                float v[32];
                tmem_ld32(to + 32 * c, v);
#pragma unroll
                for (int q = 0; q < 32; ++q) {
                    v[q] = v[q] * f0 * e0;
                    if (TWO && nt > 1) v[q] = fmaf(oj[(32 * c + q) * 128 + ql] * f1, e1, v[q]);
                }
                if (store) {
#pragma unroll
                    for (int q = 0; q < 32; q += 4) {
                        if (pieces == 1) store4(dst + 32 * c + q, v[q], v[q + 1], v[q + 2], v[q + 3]);
                        else *reinterpret_cast<float4 *>(a.part + b * D + 32 * c + q) = make_float4(v[q], v[q + 1], v[q + 2], v[q + 3]);
                    }
                }
            }
            if (store && pieces > 1)
                *reinterpret_cast<float2 *>(a.part + (size_t)a.n_rows * a.heads * a.max_chunks * D + b * 2) = make_float2(mref, l);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) tmem_dealloc(tmem, 512);
}

}  // namespace kv8
}  // namespace ct
