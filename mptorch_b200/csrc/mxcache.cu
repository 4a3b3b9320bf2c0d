// Writing new rows of K and V into the pages of an MX cache, and reading rows back.
//
// A row is the head_dim values of one token and one kv head; blocks of 32 along it share a scale 2^(floor(log2 amax) - emax),
// elements are rounded to nearest even with saturation: the codes of `mx_quantize` on the same values.
//
// Bound: HBM.  A row is read once (2 or 4 bytes an element) and its codes written once.  A thread owns eight consecutive
// elements (one or two 128-bit loads, one 8- or 4-byte store of codes), four lanes share a block and find its maximum with two
// shuffles; K and V go in one launch.
#include "blockcodes.cuh"

namespace mpt {

bool convert_cache(const char* who, const mpt_mx_cache* c, const mpt_mx_batch* b, CacheView* out) {
    if (c == nullptr || b == nullptr) { set_error("%s: null descriptor", who); return false; }
    if (c->elem_format != MPT_ELEM_E4M3 && c->elem_format != MPT_ELEM_E2M1) { set_error("%s: unknown element format %d", who, c->elem_format); return false; }
    if (c->heads < 1 || c->heads > 65535) { set_error("%s: unsupported number of kv heads %d", who, c->heads); return false; }
    if (c->dim < 32 || c->dim > 256 || c->dim % 32) { set_error("%s: head_dim %d is not a multiple of 32 up to 256", who, c->dim); return false; }
    if (c->page < 8 || c->page > 256 || (c->page & (c->page - 1))) { set_error("%s: page size %d is not a power of two from 8 to 256", who, c->page); return false; }
    if (c->num_pages < 0 || c->num_pages > 0x7FFFFFFF) { set_error("%s: bad number of pages", who); return false; }
    if (b->seqs < 0 || b->width < 0 || b->rows < 0 || (int64_t)b->width * c->page > 0x7FFFFFFF || b->rows > 0x7FFFFFFF) {
        set_error("%s: bad extents of the batch", who);
        return false;
    }
    if (b->starts == nullptr && (b->seqs == 0 ? b->rows != 0 : b->rows % b->seqs != 0)) {
        set_error("%s: %lld rows do not divide into %d sequences", who, (long long)b->rows, b->seqs);
        return false;
    }
    if (b->rows != 0 && (!c->k_codes || !c->k_scales || !c->v_codes || !c->v_scales) && c->num_pages != 0) { set_error("%s: null pointer", who); return false; }
    if (b->rows != 0 && b->seqs != 0 && (!b->lens || (!b->pages && b->width != 0))) { set_error("%s: null pointer", who); return false; }
    if (((uintptr_t)c->k_codes | (uintptr_t)c->v_codes) & 15u) { set_error("%s: the codes must begin at a multiple of 16 bytes", who); return false; }
    out->k_codes = c->k_codes; out->k_scales = c->k_scales; out->v_codes = c->v_codes; out->v_scales = c->v_scales;
    out->heads = c->heads; out->dim = c->dim;
    out->page_shift = 31 - __builtin_clz((unsigned)c->page);
    out->num_pages = (int)c->num_pages;
    out->pages = b->pages; out->lens = b->lens; out->starts = b->starts;
    out->seqs = b->seqs; out->width = b->width;
    out->new_rows = b->starts == nullptr && b->seqs > 0 ? (int)(b->rows / b->seqs) : 1;
    out->rows = b->rows;
    return true;
}

namespace {

constexpr int kThreads = 256;

// Where a new row lies in the caller's tensor (elements).
struct RowStrides { int64_t seq, row, head; };

struct Piece { int64_t row; int head, d; bool v, live; };

// Work item i: K's pieces of eight elements, then V's.  Four lanes of a block are neighbours (dim is a multiple of 32).
__device__ __forceinline__ Piece piece_of(const CacheView& c, int64_t i, int64_t per_side) {
    Piece p;
    p.live = i < 2 * per_side;
    p.v = i >= per_side;
    int64_t j = p.live ? (p.v ? i - per_side : i) : 0;
    const int per_row = c.dim >> 3;
    int64_t rh;
    if (per_side <= 0x7FFFFFFF) { rh = (uint32_t)j / (uint32_t)per_row; p.row = (uint32_t)rh / (uint32_t)c.heads; }
    else { rh = j / per_row; p.row = rh / c.heads; }
    p.d = (int)(j - rh * per_row) * 8;
    p.head = (int)(rh - p.row * c.heads);
    return p;
}

template <typename T, bool FP4>
__global__ void __launch_bounds__(kThreads) mx_cache_write_kernel(CacheView c, const T* __restrict__ k, const T* __restrict__ v, RowStrides ks,
                                                                  RowStrides vs, bool vec, int64_t per_side) {
    const int64_t total = (2 * per_side + 31) & ~(int64_t)31;      // whole warps, for the shuffles
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kThreads) {
        const Piece p = piece_of(c, i, per_side);
        int seq = 0, pos = 0;
        const bool placed = p.live && c.locate(p.row, seq, pos);
        const int64_t at = placed ? c.row_of(seq, pos, p.head) : -1;
        float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (at >= 0) {
            const RowStrides s = p.v ? vs : ks;
            const int64_t off = c.starts == nullptr ? seq * s.seq + (p.row - (int64_t)seq * c.new_rows) * s.row : p.row * s.row;
            load8((p.v ? v : k) + off + p.head * s.head + p.d, vec, x);
        }
        uint32_t amax = 0u;
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = max(amax, __float_as_uint(x[e]) & 0x7FFFFFFFu);
        amax = max(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 1));
        amax = max(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 2));
        if (at < 0) continue;
        uint32_t code, w0, w1;
        if (amax >= 0x7F800000u) {             // a NaN or an infinity poisons the block
            code = 0xFFu;
            w0 = w1 = FP4 ? 0u : 0x7F7F7F7Fu;
        } else {
            const int fl = (amax >> 23) ? (int)(amax >> 23) - 127 : (amax ? (31 - __clz((int)amax)) - 149 : -1000);
            const int e = min(max(fl - (FP4 ? 2 : 8), -127), 127);
            code = (uint32_t)(e + 127);
            const float down = -e >= -126 ? __uint_as_float((uint32_t)(127 - e) << 23) : __uint_as_float(0x00400000u);
#pragma unroll
            for (int q = 0; q < 8; ++q) x[q] = __fmul_rn(x[q], down);
            if (FP4) {
                w0 = to_e2m1x2(x[0], x[1]) | (to_e2m1x2(x[2], x[3]) << 8) | (to_e2m1x2(x[4], x[5]) << 16) | (to_e2m1x2(x[6], x[7]) << 24);
                w1 = 0u;
            } else {
                w0 = to_e4m3x2(x[0], x[1]) | (to_e4m3x2(x[2], x[3]) << 16);
                w1 = to_e4m3x2(x[4], x[5]) | (to_e4m3x2(x[6], x[7]) << 16);
            }
        }
        uint8_t* codes = p.v ? c.v_codes : c.k_codes;
        if (FP4) *reinterpret_cast<uint32_t*>(codes + at * (c.dim >> 1) + (p.d >> 1)) = w0;
        else *reinterpret_cast<uint2*>(codes + at * c.dim + p.d) = make_uint2(w0, w1);
        if ((p.d & 31) == 0) (p.v ? c.v_scales : c.k_scales)[at * (c.dim >> 5) + (p.d >> 5)] = (uint8_t)code;
    }
}

template <typename T, bool FP4>
__global__ void __launch_bounds__(kThreads) mx_cache_read_kernel(CacheView c, T* __restrict__ k, T* __restrict__ v, int64_t per_side) {
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < 2 * per_side; i += (int64_t)gridDim.x * kThreads) {
        const Piece p = piece_of(c, i, per_side);
        int seq = 0, pos = 0;
        const bool placed = c.locate(p.row, seq, pos);
        const int64_t at = placed ? c.row_of(seq, pos, p.head) : -1;
        float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (at >= 0) {
            const uint8_t* codes = p.v ? c.v_codes : c.k_codes;
            uint2 w;
            if (FP4) w = make_uint2(*reinterpret_cast<const uint32_t*>(codes + at * (c.dim >> 1) + (p.d >> 1)), 0u);
            else w = *reinterpret_cast<const uint2*>(codes + at * c.dim + p.d);
            decode8<FP4>(w, x);
            const float s = e8m0_value((p.v ? c.v_scales : c.k_scales)[at * (c.dim >> 5) + (p.d >> 5)]);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = __fmul_rn(x[e], s);
        }
        store8((p.v ? v : k) + (p.row * c.heads + p.head) * c.dim + p.d, x);
    }
}

unsigned stream_blocks(int64_t items) {
    int64_t blocks = (items + kThreads - 1) / kThreads;
    const int64_t cap = (int64_t)sm_count() * 8 * 4;
    return (unsigned)(blocks > cap ? cap : blocks < 1 ? 1 : blocks);
}

}  // namespace
}  // namespace mpt

using namespace mpt;

extern "C" {

int mpt_mx_cache_write(const mpt_mx_cache* cache, const mpt_mx_batch* batch, const void* k, const void* v, int dtype, const int64_t* k_strides,
                       const int64_t* v_strides, void* stream) {
    CacheView c;
    if (!convert_cache("mx_cache_write", cache, batch, &c)) return MPT_ERR_INVALID_ARGUMENT;
    return with_dtype("mx_cache_write", dtype, [&](auto t) -> int {
        using T = decltype(t);
        if (c.rows == 0 || c.num_pages == 0 || c.width == 0) return MPT_OK;
        MPT_REQUIRE(k && v && k_strides && v_strides, "mx_cache_write: null pointer");
        const RowStrides ks{k_strides[0], k_strides[1], k_strides[2]}, vs{v_strides[0], v_strides[1], v_strides[2]};
        const int64_t any = (int64_t)((uintptr_t)k | (uintptr_t)v) | (int64_t)sizeof(T) * (ks.row | ks.head | vs.row | vs.head | (c.starts ? 0 : ks.seq | vs.seq));
        const int64_t per_side = c.rows * c.heads * (c.dim >> 3);
        auto kern = cache->elem_format == MPT_ELEM_E2M1 ? mx_cache_write_kernel<T, true> : mx_cache_write_kernel<T, false>;
        kern<<<stream_blocks(2 * per_side), kThreads, 0, as_stream(stream)>>>(c, static_cast<const T*>(k), static_cast<const T*>(v), ks, vs, (any & 15) == 0,
                                                                           per_side);
        return check_launch("mx_cache_write");
    });
}

int mpt_mx_cache_read(const mpt_mx_cache* cache, const mpt_mx_batch* batch, void* k, void* v, int dtype, void* stream) {
    CacheView c;
    if (!convert_cache("mx_cache_read", cache, batch, &c)) return MPT_ERR_INVALID_ARGUMENT;
    return with_dtype("mx_cache_read", dtype, [&](auto t) -> int {
        using T = decltype(t);
        if (c.rows == 0) return MPT_OK;
        MPT_REQUIRE(k && v, "mx_cache_read: null pointer");
        MPT_REQUIRE((((uintptr_t)k | (uintptr_t)v) & 15u) == 0, "mx_cache_read: the outputs must begin at a multiple of 16 bytes");
        const int64_t per_side = c.rows * c.heads * (c.dim >> 3);
        auto kern = cache->elem_format == MPT_ELEM_E2M1 ? mx_cache_read_kernel<T, true> : mx_cache_read_kernel<T, false>;
        kern<<<stream_blocks(2 * per_side), kThreads, 0, as_stream(stream)>>>(c, static_cast<T*>(k), static_cast<T*>(v), per_side);
        return check_launch("mx_cache_read");
    });
}

}
