// y = x W^T + b with W held as packed E2M1 codes and group scales (MXFP4, NVFP4).
//
// One warp per output column and four rows of x at a time: a lane takes eight codes (a 32-bit word), decodes them, multiplies by
// the group's scale and by the rows' values in fp32, and the warp adds up at the end.
#include "blockcodes.cuh"

namespace mpt {
namespace {

constexpr int kWarps = 8, kRows = 4;

template <typename T, bool NV>
__global__ void __launch_bounds__(32 * kWarps) block_linear_kernel(const T* __restrict__ x, const uint8_t* __restrict__ codes,
                                                                   const uint8_t* __restrict__ scales, const float* __restrict__ global_scale,
                                                                   const T* __restrict__ bias, T* __restrict__ y, int64_t rows, int64_t n_out,
                                                                   int64_t n_in) {
    const int lane = threadIdx.x & 31;
    const int64_t n = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (n >= n_out) return;
    const uint32_t* w = reinterpret_cast<const uint32_t*>(codes + n * (n_in >> 1));
    const uint8_t* s = scales + n * (n_in / (NV ? 16 : 32));
    const float glob = global_scale != nullptr ? *global_scale : 1.0f;
    for (int64_t m0 = (int64_t)blockIdx.y * kRows; m0 < rows; m0 += (int64_t)gridDim.y * kRows) {
        float acc[kRows] = {};
        for (int64_t k = 8 * lane; k < n_in; k += 256) {
            float v[8];
            decode8<true>(make_uint2(w[k >> 3], 0u), v);
            float sc;
            if (NV) {
                uint32_t lo, hi;
                e4m3x4_to_half(s[k >> 4], lo, hi);
                sc = half2_value(lo).x;
            } else {
                sc = e8m0_value(s[k >> 5]);
            }
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                if (m0 + r >= rows) break;
                float d = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) d = fmaf(v[e], to_float(x[(m0 + r) * n_in + k + e]), d);
                acc[r] = fmaf(d, sc, acc[r]);
            }
        }
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            for (int o = 16; o > 0; o >>= 1) acc[r] += __shfl_xor_sync(0xFFFFFFFFu, acc[r], o);
            if (lane == 0 && m0 + r < rows) {
                float v = acc[r] * glob;
                if (bias != nullptr) v += to_float(bias[n]);
                y[(m0 + r) * n_out + n] = from_float<T>(v);
            }
        }
    }
}

}  // namespace
}  // namespace mpt

using namespace mpt;

extern "C" {

size_t mpt_block_linear_workspace_bytes(int64_t, int64_t, int64_t, int, int) { return 0; }

int mpt_block_linear(const void* x, const uint8_t* codes, const uint8_t* scales, const float* global_scale, const void* bias, void* y,
                     int64_t rows, int64_t n_out, int64_t n_in, int format, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
    (void)workspace; (void)workspace_bytes;
    MPT_REQUIRE(rows >= 0 && n_out >= 0 && n_in >= 0 && rows <= 0x7FFFFFFF && n_out <= 0x7FFFFFFF && n_in <= 0x7FFFFFFF, "block_linear: bad extents");
    MPT_REQUIRE(n_in % 32 == 0, "block_linear: n_in %lld is not a multiple of 32", (long long)n_in);
    MPT_REQUIRE(format == MPT_BLOCK_MXFP4 || format == MPT_BLOCK_NVFP4, "block_linear: unknown format %d", format);
    return with_dtype("block_linear", dtype, [&](auto t) -> int {
        using T = decltype(t);
        if (rows == 0 || n_out == 0) return MPT_OK;
        MPT_REQUIRE(y && (n_in == 0 || (x && codes && scales)), "block_linear: null pointer");
        MPT_REQUIRE(((uintptr_t)codes & 15u) == 0, "block_linear: the codes must begin at a multiple of 16 bytes");
        const dim3 grid((unsigned)((n_out + kWarps - 1) / kWarps), (unsigned)((rows + kRows - 1) / kRows < 256 ? (rows + kRows - 1) / kRows : 256));
        auto kern = format == MPT_BLOCK_NVFP4 ? block_linear_kernel<T, true> : block_linear_kernel<T, false>;
        kern<<<grid, 32 * kWarps, 0, as_stream(stream)>>>(static_cast<const T*>(x), codes, scales, global_scale, static_cast<const T*>(bias),
                                                        static_cast<T*>(y), rows, n_out, n_in);
        return check_launch("block_linear");
    });
}

}
