// Reading and writing the packed codes of the block formats, and the batch description that the cache operators share.
//
// Elements are converted by the hardware's own conversions, which round to nearest even and saturate exactly as
// `mx_quantize` does; E4M3 and E2M1 values are exact in binary16, and a value times its E8M0 scale is exact in fp32.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace mpt {

// 2^(b - 127), NaN for 0xFF
__device__ __forceinline__ float e8m0_value(uint32_t b) {
    const uint32_t u = b << 23;
    return __uint_as_float(b == 0u ? 0x00400000u : b == 255u ? 0x7FC00000u : u);
}

// the four E4M3 codes of a word -> two pairs of binary16 values
__device__ __forceinline__ void e4m3x4_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
    asm("{ .reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.rn.f16x2.e4m3x2 %0, a;\n cvt.rn.f16x2.e4m3x2 %1, b; }" : "=r"(lo), "=r"(hi) : "r"(w));
}
// the eight E2M1 codes of a word (low nibble first) -> four pairs of binary16 values
__device__ __forceinline__ void e2m1x8_to_half(uint32_t w, uint32_t (&h)[4]) {
    asm("{ .reg .b8 a, b, c, d;\n mov.b32 {a, b, c, d}, %4;\n cvt.rn.f16x2.e2m1x2 %0, a;\n cvt.rn.f16x2.e2m1x2 %1, b;\n"
        " cvt.rn.f16x2.e2m1x2 %2, c;\n cvt.rn.f16x2.e2m1x2 %3, d; }"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
}
__device__ __forceinline__ float2 half2_value(uint32_t h) { return __half22float2(*reinterpret_cast<const __half2*>(&h)); }

__device__ __forceinline__ uint32_t to_e4m3x2(float a, float b) {   // a in the low byte
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ uint32_t to_e2m1x2(float a, float b) {   // a in the low nibble
    uint16_t r;
    asm("{ .reg .b8 t;\n cvt.rn.satfinite.e2m1x2.f32 t, %2, %1;\n mov.b16 %0, {t, 0}; }" : "=h"(r) : "f"(a), "f"(b));
    return r & 0xFFu;
}

// Eight consecutive codes (of one block of 32) as fp32 values; `w` holds 8 bytes of E4M3 or 4 bytes of E2M1.
template <bool FP4>
__device__ __forceinline__ void decode8(uint2 w, float (&v)[8]) {
    uint32_t h[4];
    if (FP4) e2m1x8_to_half(w.x, h);
    else { e4m3x4_to_half(w.x, h[0], h[1]); e4m3x4_to_half(w.y, h[2], h[3]); }
#pragma unroll
    for (int i = 0; i < 4; ++i) { const float2 f = half2_value(h[i]); v[2 * i] = f.x; v[2 * i + 1] = f.y; }
}

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Eight consecutive values; `vec`: the address is a multiple of 16 bytes.
template <typename T>
__device__ __forceinline__ void load8(const T* p, bool vec, float (&v)[8]) {
    if (vec) {
        T t[8];
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(t)[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_float(t[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_float(p[i]);
    }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {   // p: a multiple of 16 bytes
    T t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = from_float<T>(v[i]);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<uint4*>(t)[i];
}

__device__ __forceinline__ float load_value(const void* p, int dtype, int64_t i) {
    return dtype == MPT_DTYPE_F32 ? static_cast<const float*>(p)[i]
         : dtype == MPT_DTYPE_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]) : __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_value(void* p, int dtype, int64_t i, float v) {
    if (dtype == MPT_DTYPE_F32) static_cast<float*>(p)[i] = v;
    else if (dtype == MPT_DTYPE_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
    else static_cast<__half*>(p)[i] = __float2half_rn(v);
}

// fp32 sums of binary16 products, 16 x 8 by 16 at a time: added to c, or begun
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// A paged MX cache and a batch of sequences in it, as kernels take them.
struct CacheView {
    uint8_t *k_codes, *k_scales, *v_codes, *v_scales;
    int heads, dim, page_shift;                // kv heads, head_dim, log2 of the tokens of a page
    int num_pages;
    const int32_t *pages, *lens, *starts;      // starts: null for the same number of new rows in each sequence
    int seqs, width, new_rows;                 // new_rows: rows of a sequence (uniform), unused otherwise
    int64_t rows;                              // new rows in all

    // Sequence and position of a new row; false where it has none (behind the last sequence, or before the first token).
    __device__ __forceinline__ bool locate(int64_t row, int& seq, int& pos) const {
        if (starts == nullptr) {
            seq = (int)((uint32_t)row / (uint32_t)new_rows);      // fewer than 2^31 rows
            const int i = (int)(row - (int64_t)seq * new_rows);
            pos = __ldg(lens + seq) - new_rows + i;
        } else {
            int lo = 0, hi = seqs;             // the first sequence that ends behind the row
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (__ldg(starts + mid + 1) > row) hi = mid; else lo = mid + 1;
            }
            seq = lo;
            if (seq >= seqs || row < __ldg(starts + seq)) { seq = -1; return false; }
            pos = __ldg(lens + seq) - __ldg(starts + seq + 1) + (int)row;
        }
        return pos >= 0;
    }
    __device__ __forceinline__ int capacity() const { return (int)min((int64_t)width << page_shift, (int64_t)0x7FFFFFFF); }
    // The number of a (token, kv head) row among the cache's rows; -1 where the token has no page.
    __device__ __forceinline__ int64_t row_of(int seq, int pos, int head) const {
        const int slot = pos >> page_shift;
        if (slot >= width) return -1;
        const int page = __ldg(pages + (int64_t)seq * width + slot);
        if (page < 0 || page >= num_pages) return -1;
        return ((((int64_t)page * heads + head) << page_shift) + (pos & ((1 << page_shift) - 1)));
    }
};

bool convert_cache(const char* who, const mpt_mx_cache* cache, const mpt_mx_batch* batch, CacheView* out);   // mxcache.cu

template <typename F>
int with_dtype(const char* who, int dtype, F&& f) {
    switch (dtype) {
        case MPT_DTYPE_F32: return f(float{});
        case MPT_DTYPE_BF16: return f(__nv_bfloat16{});
        case MPT_DTYPE_F16: return f(__half{});
    }
    set_error("%s: unknown data type %d", who, dtype);
    return MPT_ERR_INVALID_ARGUMENT;
}

}  // namespace mpt
