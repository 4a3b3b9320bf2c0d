// What the attention kernels share: the call's parameters, how row tiles map to sequences, and which tokens a row sees.
#pragma once
#include "blockcodes.cuh"

namespace mpt {

struct AttentionParams {
    CacheView c;
    const void* q;
    int dtype;
    int64_t q_seq, q_row, q_head;      // element strides of q
    int q_heads, group;                // query heads, query heads of a kv head
    float scale_log2;                  // scale * log2(e)
    int window, sinks;
    void* out;
    int zero_tail;
    int tile_rows;                     // rows of a tile
    int runs, least;                   // CTAs, and pieces of tokens that one takes at least
    float *partial, *stats;            // of row tiles that two or more CTAs share: sums [slot, row, dim], and {maximum, sum} of each row
};

// New rows of sequence s, clamped to the rows there are.
__device__ __forceinline__ int2 rows_of(const CacheView& c, int s) {
    if (c.starts == nullptr) return make_int2(s * c.new_rows, c.new_rows);
    const int lo = min(max(__ldg(c.starts + s), 0), (int)c.rows), hi = min(max(__ldg(c.starts + s + 1), 0), (int)c.rows);
    return make_int2(lo, max(hi - lo, 0));
}

// The tokens that some row of a tile sees, in pieces of STEP: first those that hold sinks, then the rest from `main0`.
template <int STEP>
struct TokenTiles {
    int sink_tiles, main0, tiles, end;        // end: behind the last token
    __device__ __forceinline__ TokenTiles(const AttentionParams& p, int low_pos, int high_pos) {
        end = min(high_pos + 1, p.c.capacity());
        int lo = p.window > 0 ? max(low_pos - p.window + 1, 0) : 0;
        main0 = lo / STEP * STEP;
        sink_tiles = p.window > 0 ? min((p.sinks + STEP - 1) / STEP, main0 / STEP) : 0;
        if (main0 >= end) {                   // only sinks are left (a table with fewer places than tokens)
            main0 = end;
            sink_tiles = min(sink_tiles, (max(end, 0) + STEP - 1) / STEP);
        }
        tiles = end <= 0 ? 0 : sink_tiles + (end - main0 + STEP - 1) / STEP;
    }
    __device__ __forceinline__ int start(int j) const { return j < sink_tiles ? j * STEP : main0 + (j - sink_tiles) * STEP; }
};

__device__ __forceinline__ bool sees(const AttentionParams& p, int pos, int t) {
    return t <= pos && (p.window <= 0 || t > pos - p.window || t < p.sinks);
}

// Rows that belong to no sequence: zeros, where the output is this library's own.
template <typename T>
__device__ __forceinline__ void zero_rows(const AttentionParams& p, int64_t lo, int64_t hi) {
    const int64_t width = (int64_t)p.q_heads * p.c.dim;
    for (int64_t row = lo + blockIdx.x; row < hi; row += gridDim.x)
        for (int64_t i = threadIdx.x; i < width; i += blockDim.x) static_cast<T*>(p.out)[row * width + i] = from_float<T>(0.f);
}
__device__ __forceinline__ void zero_outside(const AttentionParams& p) {
    if (!p.zero_tail || p.c.starts == nullptr) return;
    const int first = min(max(p.c.seqs ? __ldg(p.c.starts) : 0, 0), (int)p.c.rows);
    const int last = p.c.seqs ? min(max(__ldg(p.c.starts + p.c.seqs), 0), (int)p.c.rows) : 0;
    for (int side = 0; side < 2; ++side) {
        const int64_t lo = side ? max(last, first) : 0, hi = side ? p.c.rows : first;
        if (lo >= hi) continue;
        if (p.dtype == MPT_DTYPE_F32) zero_rows<float>(p, lo, hi);
        else if (p.dtype == MPT_DTYPE_BF16) zero_rows<__nv_bfloat16>(p, lo, hi);
        else zero_rows<__half>(p, lo, hi);
    }
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

__device__ __forceinline__ float exp2_fast(float x) {       // relative error 2^-22; exact at integers; results below 2^-126 are zero
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

}  // namespace mpt
