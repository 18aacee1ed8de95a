// kv8.cuh -- device helpers shared by the 8-bit cache kernels (include/ct_kv8.h).
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "../../include/ct_kv8.h"
#include "ct_common.cuh"

namespace ct {
namespace kv8 {

constexpr int ROWS = CT_KV8_ROWS;

__host__ __device__ constexpr int pages_of(int rows) { return (rows + ROWS - 1) / ROWS; }

// Address arithmetic of a pool: one layer's K (kv = 0) or V (kv = 1) block of
// page p and head h.  Offsets are 64-bit: a pool is larger than 2^31 bytes.
struct Pool {
    uint8_t *codes;
    float *scales;
    int *refs;
    int n_pages, layers, heads, dim;
    __host__ __device__ long long page_bytes() const { return 2ll * layers * heads * ROWS * dim; }
    __host__ __device__ int page_scales() const { return 2 * layers * heads; }
    __device__ size_t block(int p, int layer, int kv, int h) const {
        return (((size_t)p * layers + layer) * 2 + kv) * heads + h;
    }
    __device__ bool has(int p) const { return (unsigned)p < (unsigned)n_pages; }
};

// Rows of sequence s in this call and their first token row.
struct RowSpan {
    int first;   // first packed row
    int n;       // rows
    int len;     // token rows of the sequence, this call's included
    bool ok;
};
__device__ __forceinline__ RowSpan row_span(const int *len, const int *row_start, int s, int n_rows, int max_rows,
                                            int table_rows) {
    RowSpan r;
    r.first = row_start ? row_start[s] : s;
    r.n = row_start ? row_start[s + 1] - r.first : 1;
    r.len = len[s];
    // what the host cannot see: spans outside the packed rows, lengths beyond the table
    r.ok = r.n <= max_rows && r.first >= 0 && r.n >= 0 && r.first <= n_rows - r.n && r.len <= table_rows;
    return r;
}

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(bf16 x) { return __bfloat162float(x); }

// two codes -> fp16 pair, exact in both formats (E4M3: 4-bit exponents and
// subnormals lie inside fp16's range; int8: 1024 + (v + 128) has fp16 bits
// 0x6400 | (v + 128), and the subtraction of 1152 is exact).
template <int FMT>
__device__ __forceinline__ void codes4_to_half(uint32_t w, uint32_t &lo, uint32_t &hi) {
    if (FMT == CT_KV8_E4M3) {
        asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
            "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
            : "=r"(lo), "=r"(hi)
            : "r"(w));
    } else {
        const uint32_t u = w ^ 0x80808080u;
        const __half2 off = __floats2half2_rn(1152.0f, 1152.0f);
        uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
        __half2 ha = __hsub2(*reinterpret_cast<__half2 *>(&a), off), hb = __hsub2(*reinterpret_cast<__half2 *>(&b), off);
        lo = *reinterpret_cast<uint32_t *>(&ha);
        hi = *reinterpret_cast<uint32_t *>(&hb);
    }
}

template <int FMT>
__device__ __forceinline__ float code_to_f32(uint32_t byte) {
    if (FMT == CT_KV8_INT8) return (float)(int8_t)byte;
    __nv_fp8_e4m3 v;
    v.__x = (uint8_t)byte;
    return (float)v;
}

// Nearest codes of four values, ties to even, as one word.  E4M3 saturates.  int8:
// adding 1.5 * 2^23 rounds to the integer that the sum's low byte then holds, for
// magnitudes up to 127 (`clamp`: larger ones are cut to that first).
template <int FMT>
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d, bool clamp) {
    if (FMT == CT_KV8_E4M3) {
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
        return lo | (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3) << 16;
    }
    if (clamp) {
        a = fminf(fmaxf(a, -127.0f), 127.0f);
        b = fminf(fmaxf(b, -127.0f), 127.0f);
        c = fminf(fmaxf(c, -127.0f), 127.0f);
        d = fminf(fmaxf(d, -127.0f), 127.0f);
    }
    constexpr float magic = 12582912.0f;
    const uint32_t ab = __byte_perm(__float_as_uint(a + magic), __float_as_uint(b + magic), 0x0040);
    const uint32_t cd = __byte_perm(__float_as_uint(c + magic), __float_as_uint(d + magic), 0x0040);
    return __byte_perm(ab, cd, 0x5410);
}

// The smallest power of two that brings amax (finite, >= 0) within the codes'
// range, not below 2^-126.  E4M3: the largest code is 1.75 * 2^8; int8:
// 1.984375 * 2^6.
template <int FMT>
__device__ __forceinline__ float block_scale(float amax) {
    constexpr uint32_t frac = FMT == CT_KV8_E4M3 ? 0x600000u : 0x7E0000u;   // 0.75, 0.984375
    constexpr int shift = FMT == CT_KV8_E4M3 ? 8 : 6;
    const uint32_t b = __float_as_uint(amax);
    const int e = (int)(b >> 23) - shift + ((b & 0x7FFFFFu) > frac ? 1 : 0);   // biased
    return __uint_as_float((uint32_t)max(e, 1) << 23);
}

}  // namespace kv8
}  // namespace ct
