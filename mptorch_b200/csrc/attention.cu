// Attention of new tokens over a paged MX cache.
//
// One warp per (new row, query head): lane l holds the dimensions l, l + 32, ..., so that its i-th value lies in block i; one pass
// over the visible tokens with the running maximum and sum of the softmax.
#include "blockcodes.cuh"

namespace mpt {
namespace {

constexpr int kWarps = 4, kMaxBlocks = 8;

struct RowStrides { int64_t seq, row, head; };

template <bool FP4>
__device__ __forceinline__ float element(const uint8_t* codes, const uint8_t* scales, int64_t at, int dim, int d) {
    float v[8];
    if (FP4) decode8<true>(make_uint2((codes[at * (dim >> 1) + (d >> 1)] >> (4 * (d & 1))) & 15u, 0u), v);
    else decode8<false>(make_uint2(codes[at * dim + d], 0u), v);
    return v[0] * e8m0_value(scales[at * (dim >> 5) + (d >> 5)]);
}

template <typename T, bool FP4>
__global__ void __launch_bounds__(32 * kWarps) mx_attention_rows_kernel(CacheView c, const T* __restrict__ q, RowStrides qs, int q_heads, float scale,
                                                                        int window, int sinks, T* __restrict__ out, bool zero_tail) {
    const int lane = threadIdx.x & 31, nb = c.dim >> 5;
    const int64_t item = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (item >= c.rows * q_heads) return;
    const int64_t row = item / q_heads;
    const int head = (int)(item - row * q_heads), kv = head / (q_heads / c.heads);
    T* o = out + item * c.dim;
    int seq, pos;
    const bool placed = c.locate(row, seq, pos);
    if (!placed) {
        if (seq >= 0 || zero_tail) for (int i = 0; i < nb; ++i) o[lane + 32 * i] = from_float<T>(0.f);
        return;
    }
    float x[kMaxBlocks] = {}, acc[kMaxBlocks] = {}, m = -INFINITY, sum = 0.f;
    const int64_t off = c.starts == nullptr ? seq * qs.seq + (row - (int64_t)seq * c.new_rows) * qs.row : row * qs.row;
    for (int i = 0; i < nb; ++i) x[i] = to_float(q[off + head * qs.head + lane + 32 * i]);
    const int last = min(pos, c.capacity() - 1);
    for (int t = 0; t <= last; ++t) {
        if (window > 0 && (int64_t)t <= (int64_t)pos - window && t >= sinks) { t = max(t, pos - window); continue; }
        const int64_t at = c.row_of(seq, t, kv);
        if (at < 0) continue;
        float s = 0.f;
        for (int i = 0; i < nb; ++i) s = fmaf(x[i], element<FP4>(c.k_codes, c.k_scales, at, c.dim, lane + 32 * i), s);
        for (int k = 16; k > 0; k >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, k);
        s *= scale;
        const float top = fmaxf(m, s);
        const float base = top == -INFINITY ? 0.f : top, fade = expf(m - base), p = expf(s - base);
        sum = fmaf(sum, fade, p);
        for (int i = 0; i < nb; ++i) acc[i] = fmaf(acc[i], fade, p * element<FP4>(c.v_codes, c.v_scales, at, c.dim, lane + 32 * i));
        m = top;
    }
    for (int i = 0; i < nb; ++i) o[lane + 32 * i] = from_float<T>(sum == 0.f ? 0.f : acc[i] / sum);
}

}  // namespace
}  // namespace mpt

using namespace mpt;

extern "C" {

size_t mpt_mx_attention_workspace_bytes(const mpt_mx_cache*, const mpt_mx_batch*, int, int, int, int) { return 0; }

int mpt_mx_attention(const mpt_mx_cache* cache, const mpt_mx_batch* batch, const void* q, int dtype, const int64_t* q_strides, int q_heads, float scale,
                     int window, int sinks, void* out, int zero_tail, void* workspace, size_t workspace_bytes, void* stream) {
    (void)workspace; (void)workspace_bytes;
    CacheView c;
    if (!convert_cache("mx_attention", cache, batch, &c)) return MPT_ERR_INVALID_ARGUMENT;
    MPT_REQUIRE(q_heads >= 1 && q_heads % c.heads == 0, "mx_attention: %d query heads do not divide among %d kv heads", q_heads, c.heads);
    MPT_REQUIRE(window >= 0 && sinks >= 0, "mx_attention: window and sinks must not be negative");
    return with_dtype("mx_attention", dtype, [&](auto t) -> int {
        using T = decltype(t);
        if (batch->rows == 0) return MPT_OK;
        MPT_REQUIRE(q && q_strides && out, "mx_attention: null pointer");
        const RowStrides qs{q_strides[0], q_strides[1], q_strides[2]};
        auto kern = cache->elem_format == MPT_ELEM_E2M1 ? mx_attention_rows_kernel<T, true> : mx_attention_rows_kernel<T, false>;
        kern<<<(unsigned)((c.rows * q_heads + kWarps - 1) / kWarps), 32 * kWarps, 0, as_stream(stream)>>>(
            c, static_cast<const T*>(q), qs, q_heads, scale, window, sinks, static_cast<T*>(out), zero_tail != 0);
        return check_launch("mx_attention");
    });
}

}
