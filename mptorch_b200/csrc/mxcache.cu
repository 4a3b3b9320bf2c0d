// Writing new rows of K and V into the pages of an MX cache, and reading rows back.
//
// A row is the head_dim values of one token and one kv head; blocks of 32 along it share a scale 2^(floor(log2 amax) - emax),
// elements are rounded to nearest even with saturation: the codes of `mx_quantize` on the same values.
//
// Bound: HBM.  A row is read once (2 or 4 bytes an element) and its codes written once.  A warp takes up to 128 pieces of eight
// elements of K or of V of one token, all heads after one another, so that the token's sequence and page are looked up once; a lane has
// four pieces under way at a time, and four lanes share a block and find its maximum with two shuffles.  K and V go in one launch.
//
// Measured on a B200: seven prompts of up to 4096 tokens, 8 heads of 128, bfloat16 to and from E2M1: 71 us for both calls (25.7 for
// the bytes at the measured bandwidth); instruction issue bounds the writes (45 us) and memory latency the
// reads (23 us).  With a warp for each 32 pieces, which looks up its token each time, both took 99 us.  One token each of 32 sequences
// (12 heads of 64, float32): 26 us for both, host time.
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
    if (((uintptr_t)c->k_scales | (uintptr_t)c->v_scales) & 7u) { set_error("%s: the scales must begin at a multiple of 8 bytes", who); return false; }
    out->k_codes = c->k_codes; out->k_scales = c->k_scales; out->v_codes = c->v_codes; out->v_scales = c->v_scales;
    out->heads = c->heads; out->dim = c->dim;
    out->page_shift = 31 - __builtin_clz((unsigned)c->page);
    out->num_pages = (int)c->num_pages;
    out->pages = b->pages; out->lens = b->lens; out->starts = b->starts;
    out->seqs = b->seqs;
    out->width = c->num_pages ? b->width : 0;      // without pages there are no tokens
    out->new_rows = b->starts == nullptr && b->seqs > 0 ? (int)(b->rows / b->seqs) : 1;
    out->rows = b->rows;
    return true;
}

namespace {

constexpr int kThreads = 256;

// Where a new row lies in the caller's tensor (elements).
struct RowStrides { int64_t seq, row, head; };

constexpr int kEach = 4;                       // pieces of a lane

// Warp w: part `part` of one side of one row.
struct Unit {
    int64_t row, place;                        // place: number of the token's first row (head 0) among the cache's rows, -1 without one
    int side, first, seq;
    __device__ __forceinline__ Unit(const CacheView& c, int64_t w, int parts) {
        const int64_t rs = parts == 1 ? w : (w >> 32) ? w / parts : (uint32_t)w / (uint32_t)parts;
        first = (int)(w - rs * parts) * 32 * kEach;
        row = rs >> 1;
        side = (int)(rs & 1);
        int pos;
        place = c.locate(row, seq, pos) ? c.row_of(seq, pos, 0) : -1;
    }
};

// A lane's pieces: 32 apart, so head and dimension move by constant steps.
struct Step {
    int head, d, heads, rest, dim;
    __device__ __forceinline__ Step(int j, int dim_) : dim(dim_) {
        const uint32_t per = (uint32_t)dim >> 3;
        head = (int)((uint32_t)j / per);
        d = (j - head * (int)per) * 8;
        heads = (int)(32u / per);
        rest = (32 - heads * (int)per) * 8;
    }
    __device__ __forceinline__ void next() {
        head += heads;
        d += rest;
        if (d >= dim) { d -= dim; ++head; }
    }
};

// the larger magnitude, a NaN if one is; the sign is of no use
__device__ __forceinline__ float max_magnitude(float a, float b) {
    float r;
    asm("max.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

template <typename T, bool FP4>
__global__ void __launch_bounds__(kThreads) mx_cache_write_kernel(CacheView c, const T* __restrict__ k, const T* __restrict__ v, RowStrides ks,
                                                                  RowStrides vs, bool vec, int parts, int64_t units) {
    const int lane = threadIdx.x & 31, pieces = c.heads * (c.dim >> 3);
    const int64_t w0 = ((int64_t)blockIdx.x * kThreads + threadIdx.x) >> 5;
    if (w0 >= units) return;
    const Unit u(c, w0, parts);
    if (u.place < 0) return;
    const RowStrides s = u.side ? vs : ks;
    const T* from = (u.side ? v : k) + (c.starts == nullptr ? u.seq * s.seq + (u.row - (int64_t)u.seq * c.new_rows) * s.row : u.row * s.row);
    uint8_t* codes = u.side ? c.v_codes : c.k_codes;
    uint8_t* scales = u.side ? c.v_scales : c.k_scales;
    float x[kEach][8];
    Step at(u.first + lane, c.dim);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[i][e] = 0.f;
        if (u.first + 32 * i + lane < pieces) load8(from + at.head * s.head + at.d, vec, x[i]);
        at.next();
    }
    at = Step(u.first + lane, c.dim);
    const int64_t head_rows = (int64_t)1 << c.page_shift;
#pragma unroll
    for (int i = 0; i < kEach; ++i, at.next()) {
        if (u.first + 32 * i >= pieces) break;
        float top = x[i][0];
#pragma unroll
        for (int e = 1; e < 8; ++e) top = max_magnitude(top, x[i][e]);
        uint32_t amax = __float_as_uint(top) & 0x7FFFFFFFu;
        amax = max(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 1));
        amax = max(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 2));
        if (u.first + 32 * i + lane >= pieces) continue;
        uint32_t code, w0, w1;
        if (amax >= 0x7F800000u) {             // a NaN or an infinity poisons the block
            code = 0xFFu;
            w0 = w1 = FP4 ? 0u : 0x7F7F7F7Fu;
        } else {
            const int fl = (amax >> 23) ? (int)(amax >> 23) - 127 : (amax ? (31 - __clz((int)amax)) - 149 : -1000);
            const int e = min(max(fl - (FP4 ? 2 : 8), -127), 127);
            code = (uint32_t)(e + 127);
            const float down = -e >= -126 ? __uint_as_float((uint32_t)(127 - e) << 23) : __uint_as_float(0x00400000u);
            float q[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) q[j] = __fmul_rn(x[i][j], down);
            if (FP4) {
                w0 = to_e2m1x2(q[0], q[1]) | (to_e2m1x2(q[2], q[3]) << 8) | (to_e2m1x2(q[4], q[5]) << 16) | (to_e2m1x2(q[6], q[7]) << 24);
                w1 = 0u;
            } else {
                w0 = to_e4m3x2(q[0], q[1]) | (to_e4m3x2(q[2], q[3]) << 16);
                w1 = to_e4m3x2(q[4], q[5]) | (to_e4m3x2(q[6], q[7]) << 16);
            }
        }
        const int64_t row = u.place + at.head * head_rows;
        if (FP4) *reinterpret_cast<uint32_t*>(codes + row * (c.dim >> 1) + (at.d >> 1)) = w0;
        else *reinterpret_cast<uint2*>(codes + row * c.dim + at.d) = make_uint2(w0, w1);
        if ((at.d & 31) == 0) scales[row * (c.dim >> 5) + (at.d >> 5)] = (uint8_t)code;
    }
}

template <typename T, bool FP4>
__global__ void __launch_bounds__(kThreads) mx_cache_read_kernel(CacheView c, T* __restrict__ k, T* __restrict__ v, int parts, int64_t units) {
    const int lane = threadIdx.x & 31, pieces = c.heads * (c.dim >> 3);
    const int64_t w0 = ((int64_t)blockIdx.x * kThreads + threadIdx.x) >> 5;
    if (w0 >= units) return;
    const Unit u(c, w0, parts);
    const uint8_t* codes = u.side ? c.v_codes : c.k_codes;
    const uint8_t* scales = u.side ? c.v_scales : c.k_scales;
    T* out = (u.side ? v : k) + u.row * c.heads * c.dim;
    uint2 w[kEach];
    uint32_t s[kEach];
    Step at(u.first + lane, c.dim);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        w[i] = make_uint2(0u, 0u);
        s[i] = 127u;
        if (u.first + 32 * i + lane < pieces && u.place >= 0) {
            const int64_t row = u.place + ((int64_t)at.head << c.page_shift);
            if (FP4) w[i].x = *reinterpret_cast<const uint32_t*>(codes + row * (c.dim >> 1) + (at.d >> 1));
            else w[i] = *reinterpret_cast<const uint2*>(codes + row * c.dim + at.d);
            s[i] = scales[row * (c.dim >> 5) + (at.d >> 5)];
        }
        at.next();
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int j = u.first + 32 * i + lane;
        if (j >= pieces) break;
        float x[8];
        decode8<FP4>(w[i], x);
        const float f = e8m0_value(s[i]);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = __fmul_rn(x[e], f);
        store8(out + j * 8, x);
    }
}

// Warps' units of a call: both sides of each row, in parts of 128 pieces.
int parts_of(const CacheView& c) { return (c.heads * (c.dim >> 3) + 32 * kEach - 1) / (32 * kEach); }

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
        const int parts = parts_of(c);
        const int64_t units = 2 * c.rows * parts, blocks = (units * 32 + kThreads - 1) / kThreads;
        MPT_REQUIRE(blocks <= 0x7FFFFFFF, "%s: too many rows", "mx_cache_write");
        auto kern = cache->elem_format == MPT_ELEM_E2M1 ? mx_cache_write_kernel<T, true> : mx_cache_write_kernel<T, false>;
        kern<<<(unsigned)blocks, kThreads, 0, as_stream(stream)>>>(c, static_cast<const T*>(k), static_cast<const T*>(v), ks, vs, (any & 15) == 0, parts, units);
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
        const int parts = parts_of(c);
        const int64_t units = 2 * c.rows * parts, blocks = (units * 32 + kThreads - 1) / kThreads;
        MPT_REQUIRE(blocks <= 0x7FFFFFFF, "%s: too many rows", "mx_cache_read");
        auto kern = cache->elem_format == MPT_ELEM_E2M1 ? mx_cache_read_kernel<T, true> : mx_cache_read_kernel<T, false>;
        kern<<<(unsigned)blocks, kThreads, 0, as_stream(stream)>>>(c, static_cast<T*>(k), static_cast<T*>(v), parts, units);
        return check_launch("mx_cache_read");
    });
}

}
