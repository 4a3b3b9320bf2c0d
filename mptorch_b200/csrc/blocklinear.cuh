// What the kernels of the products with packed 4-bit weights share.
#pragma once
#include "blockcodes.cuh"

namespace mpt {

struct LinearParams {
    const void* x;
    const uint8_t *codes, *scales;
    const float* global_scale;     // null: 1
    const void* bias;              // null: none
    void* y;
    int dtype, rows, n_out, n_in;
    bool x_vec;                    // x begins at a multiple of 16 bytes
};

// v * 2^e, e in [-300, 300], without leaving fp32's range on the way
__device__ __forceinline__ float scale_by_power(float v, int e) {
    const int half = e / 2, rest = e - half;
    auto power = [](int k) { return k >= -126 ? __uint_as_float((uint32_t)(min(k, 127) + 127) << 23) : __uint_as_float(0x00400000u >> min(-127 - k, 23)); };
    return v * power(half) * power(rest);
}

// The power of two that brings a row of x with the largest finite magnitude of these bits to [2^14, 2^15)
__device__ __forceinline__ int row_exponent(uint32_t top_bits) { return top_bits ? min(max(127 + 14 - (int)(top_bits >> 23), -126), 126) : 0; }

__device__ __forceinline__ void read8(const void* p, int dtype, bool vec, int64_t i, float (&v)[8]) {
    if (dtype == MPT_DTYPE_F32) load8(static_cast<const float*>(p) + i, vec, v);
    else if (dtype == MPT_DTYPE_BF16) load8(static_cast<const __nv_bfloat16*>(p) + i, vec, v);
    else load8(static_cast<const __half*>(p) + i, vec, v);
}

// The form for many rows (linear_tiles.cu)
struct TilesPlan {
    int cols, pieces, row_tiles, col_tiles, k_blocks, k_supers, runs, ring_blocks, w_stages, x_stages, columns, fold;
    int64_t units, per;
    size_t image_bytes, partial_bytes, kept_bytes, far_bytes, bytes;
};
TilesPlan tiles_plan(int64_t rows, int64_t n_out, int64_t n_in, int format, int dtype);
int launch_tiles(const LinearParams& p, const TilesPlan& pl, int format, uint8_t* workspace, cudaStream_t st);

}  // namespace mpt
