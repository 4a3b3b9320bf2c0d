// y = x W^T + b for many rows of x, with W held as packed E2M1 codes and group scales (MXFP4, NVFP4): tiles of 128 rows of W by up to
// 256 columns of x on the tcgen05 tensor cores.
//
// Bound: HBM while the rows of x are few (half a byte a weight), the tensor cores beyond some 200 of them.  Two kernels, or three:
//   1. x is scaled for each row by a power of two to a largest value in [2^14, 2^15) and laid out as binary16 tiles of 64 of the sum, in
//      the layout of the products' operands in shared memory, so that a tile is one bulk copy.  float32 takes two such pieces (22
//      bits); bfloat16 and float16 one (exact unless a value is 2^-29 of the row's largest or less).
//   2. A warp copies x's tiles, a warp issues products, and eight warps turn codes into binary16 weights in shared memory: one
//      conversion and one multiplication for two of them.  NVFP4: a code times its E4M3 scale is exact (six bits).  MXFP4: a code times
//      2^(13 + e - E), E the row's largest exponent, is exact down to e = E - 36; smaller blocks count less than 2^-36 of the largest.
//      Sums are fp32 in tensor memory, those of float32's second pieces apart, and the powers of two are put back at the end.
//   3. Where there are too few tiles for the SMs the sum is split, and the parts are added up in order.
//
// Measured figures stand at the launch rule below.
#include "blocklinear.cuh"
#include "tcgen05.cuh"

namespace mpt {
namespace {

constexpr int kRowsW = 128, kBlock = 64, kWorkers = 256, kThreads = kWorkers + 64;
constexpr int kPartW = kRowsW * 128;                               // bytes of a tile of W: 128 rows of 64 weights

struct TilesParams {
    LinearParams l;
    int cols, pieces, k_blocks, splits, stages, columns;
    const uint8_t* image;              // x: [column tile][block of 64][piece][cols][128 bytes]
    int* exponent;                     // of each row of x
    float* partial;                    // [split][rows][n_out]
};

// ---- x into tiles: a CTA for a row
__global__ void __launch_bounds__(256) linear_split_kernel(const TilesParams p, uint8_t* __restrict__ image) {
    const LinearParams& l = p.l;
    const int m = blockIdx.x, ct = m / p.cols, r = m - ct * p.cols, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    __shared__ uint32_t tops[8];
    float top = 0.f;
    for (int k = 8 * threadIdx.x; k < l.n_in; k += 2048) {
        float v[8];
        read8(l.x, l.dtype, l.x_vec, (int64_t)m * l.n_in + k, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) { const float a = fabsf(v[e]); if (a < INFINITY) top = fmaxf(top, a); }
    }
    const uint32_t wtop = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(top));
    if (lane == 0) tops[warp] = wtop;
    __syncthreads();
    uint32_t all = 0u;
#pragma unroll
    for (int w = 0; w < 8; ++w) all = max(all, tops[w]);
    const int e = row_exponent(all);
    const float up = __uint_as_float((uint32_t)(127 + e) << 23);
    if (threadIdx.x == 0) p.exponent[m] = e;
    uint8_t* out = image + (int64_t)ct * p.k_blocks * p.pieces * p.cols * 128 + r * 128;
    for (int k = 8 * threadIdx.x; k < p.k_blocks * kBlock; k += 2048) {
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (k < l.n_in) read8(l.x, l.dtype, l.x_vec, (int64_t)m * l.n_in + k, v);
        __half hi[8], lo[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[i] *= up;
            hi[i] = __float2half_rn(v[i]);
            lo[i] = fabsf(v[i]) < INFINITY ? __float2half_rn((v[i] - __half2float(hi[i])) * 2048.f) : __float2half_rn(0.f);
        }
        uint8_t* to = out + (int64_t)(k / kBlock) * p.pieces * p.cols * 128 + ((((k & 63) >> 3) ^ (r & 7)) << 4);
        *reinterpret_cast<uint4*>(to) = *reinterpret_cast<uint4*>(hi);
        if (p.pieces == 2) *reinterpret_cast<uint4*>(to + p.cols * 128) = *reinterpret_cast<uint4*>(lo);
    }
}

// fp32 sums of binary16 products, M = 128
__device__ __forceinline__ uint32_t half_product_descriptor(int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | (8u << 24); }

// 2^(13 - d) as binary16, zero below 2^-24
__device__ __forceinline__ uint32_t half_weight_power(int d) { return d <= 27 ? (uint32_t)(28 - d) << 10 : d <= 37 ? 1u << (37 - d) : 0u; }

constexpr int kMaxStages = 8;

template <bool NV>
__global__ void __launch_bounds__(kThreads) linear_tiles_kernel(const TilesParams p) {
    extern __shared__ uint8_t smem_raw[];
    const LinearParams& l = p.l;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t base = (smem_at(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem = smem_raw + (base - smem_at(smem_raw));
    const int x_bytes = p.pieces * p.cols * 128, stage_bytes = kPartW + x_bytes;
    const int ct = blockIdx.x, n0 = blockIdx.y * kRowsW, split = blockIdx.z;
    const int b_lo = (int)((int64_t)p.k_blocks * split / p.splits), b_hi = (int)((int64_t)p.k_blocks * (split + 1) / p.splits), blocks = b_hi - b_lo;
    __shared__ __align__(8) uint64_t bars[3 * kMaxStages + 1];
    __shared__ uint32_t tmem_slot, failed;
    __shared__ int top_e[kRowsW];
    auto x_full = [&](int s) { return smem_at(&bars[s]); };
    auto w_full = [&](int s) { return smem_at(&bars[kMaxStages + s]); };
    auto empty = [&](int s) { return smem_at(&bars[2 * kMaxStages + s]); };
    const uint32_t done = smem_at(&bars[3 * kMaxStages]);
    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            bar_init(x_full(s), 1);
            bar_init(w_full(s), kWorkers);
            bar_init(empty(s), 1);
        }
        bar_init(done, 1);
        failed = 0u;
        fence_barrier_init();
    }
    if (warp == 9) tmem_alloc(smem_at(&tmem_slot), p.columns);
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = tmem_slot;

    if (warp == 8) {
        if (lane == 0) {
            const uint8_t* src = p.image + ((int64_t)ct * p.k_blocks + b_lo) * x_bytes;
            for (int i = 0; i < blocks; ++i) {
                const int s = i % p.stages;
                if (i >= p.stages && !bar_wait(empty(s), (i / p.stages - 1) & 1, &failed)) break;
                bar_expect(x_full(s), x_bytes);
                bulk_load(base + s * stage_bytes + kPartW, src + (int64_t)i * x_bytes, x_bytes, x_full(s));
            }
        }
        __syncwarp();
    } else if (warp == 9) {
        if (lane == 0) {
            const uint32_t desc = half_product_descriptor(p.cols);
            for (int i = 0; i < blocks; ++i) {
                const int s = i % p.stages;
                if (!bar_wait(x_full(s), (i / p.stages) & 1, &failed) || !bar_wait(w_full(s), (i / p.stages) & 1, &failed)) break;
                tmem_fence_after();
                const uint64_t w = tile_descriptor(base + s * stage_bytes, 16), x = tile_descriptor(base + s * stage_bytes + kPartW, 16);
#pragma unroll
                for (int k = 0; k < kBlock / 16; ++k) mma_ss(tmem, w + 2 * k, x + 2 * k, desc, i + k > 0);
                if (p.pieces == 2) {
#pragma unroll
                    for (int k = 0; k < kBlock / 16; ++k) mma_ss(tmem + p.cols, w + 2 * k, x + (p.cols * 128 >> 4) + 2 * k, desc, i + k > 0);
                }
                mma_commit(empty(s));
            }
            mma_commit(done);
        }
        __syncwarp();
    } else {
        // ---- weights: two threads a row, each 32 of a block's 64
        const int r = threadIdx.x >> 1, half = threadIdx.x & 1, n = n0 + r;
        const bool live = n < l.n_out;
        const int groups = l.n_in / (NV ? 16 : 32);
        const uint4* codes = reinterpret_cast<const uint4*>(l.codes + (live ? (int64_t)n * (l.n_in >> 1) : 0)) + half;
        const uint8_t* scales = l.scales + (live ? (int64_t)n * groups : 0);
        int top = 0;
        if (!NV) {
            if (live) {
                // the row's largest exponent (255 is a NaN and no exponent); bytes up to an aligned word, then words
                auto take = [&](uint32_t e) { top = max(top, e == 255u ? 0 : (int)e); };
                int k = half;
                const int head = min((int)((4 - (reinterpret_cast<uintptr_t>(scales) & 3)) & 3), groups);
                if (half == 0)
                    for (int j = 0; j < head; ++j) take(__ldg(scales + j));
                const int words = (groups - head) >> 2;
                const uint32_t* at = reinterpret_cast<const uint32_t*>(scales + head);
#pragma unroll 4
                for (k = half; k < words; k += 2) {
                    const uint32_t w = __ldg(at + k);
                    take(w & 255u); take((w >> 8) & 255u); take((w >> 16) & 255u); take(w >> 24);
                }
                if (half == 1)
                    for (int j = head + 4 * words; j < groups; ++j) take(__ldg(scales + j));
            }
            top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
            if (half == 0) top_e[r] = top;
        }
        constexpr int kAhead = 4;
        uint4 ahead[kAhead];
        uint32_t ahead_s[kAhead];
        auto fetch = [&](int i, uint4& w, uint32_t& sc) {
            const int b = b_lo + i;
            w = make_uint4(0u, 0u, 0u, 0u);
            sc = NV ? 0u : (uint32_t)top;
            if (i < blocks && live && b * 64 + half * 32 < l.n_in) {
                w = __ldg(codes + b * 2);
                if (NV) sc = __ldg(scales + b * 4 + half * 2) | ((uint32_t)__ldg(scales + b * 4 + half * 2 + 1) << 8);
                else sc = __ldg(scales + b * 2 + half);
            }
        };
#pragma unroll
        for (int a = 0; a < kAhead; ++a) fetch(a, ahead[a], ahead_s[a]);
        for (int i0 = 0; i0 < blocks; i0 += kAhead) {
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
                const int i = i0 + a;
                if (i >= blocks) break;
                const uint4 w = ahead[a];
                const uint32_t sc = ahead_s[a];
                fetch(i + kAhead, ahead[a], ahead_s[a]);
                uint32_t h[16];
                e2m1x8_to_half(w.x, *reinterpret_cast<uint32_t(*)[4]>(h));
                e2m1x8_to_half(w.y, *reinterpret_cast<uint32_t(*)[4]>(h + 4));
                e2m1x8_to_half(w.z, *reinterpret_cast<uint32_t(*)[4]>(h + 8));
                e2m1x8_to_half(w.w, *reinterpret_cast<uint32_t(*)[4]>(h + 12));
                uint32_t f[2];
                if (NV) {
                    uint32_t u;
                    e4m3x4_to_half(__byte_perm(sc, 0u, 0x0000), f[0], u);
                    e4m3x4_to_half(__byte_perm(sc, 0u, 0x1111), f[1], u);
                } else {
                    const uint32_t q = sc == 255u ? 0x7E00u : half_weight_power(top - (int)sc);
                    f[0] = f[1] = q | (q << 16);
                }
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    const __half2 v = __hmul2(*reinterpret_cast<__half2*>(&h[k]), *reinterpret_cast<__half2*>(&f[k >> 3]));
                    h[k] = *reinterpret_cast<const uint32_t*>(&v);
                }
                const int s = i % p.stages;
                if (i >= p.stages) bar_wait(empty(s), (i / p.stages - 1) & 1, &failed);
                uint8_t* to = smem + s * stage_bytes + r * 128;
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *reinterpret_cast<uint4*>(to + (((half * 4 + q) ^ (r & 7)) << 4)) = make_uint4(h[4 * q], h[4 * q + 1], h[4 * q + 2], h[4 * q + 3]);
                fence_async_proxy();
                bar_arrive(w_full(s));
            }
        }
        // ---- results: a thread has one row of W; the warps of each half every other 16 columns
        bar_wait(done, 0, &failed);
        asm volatile("bar.sync 1, %0;" ::"n"(kWorkers) : "memory");
        tmem_fence_after();
        const bool ok = *(volatile uint32_t*)&failed == 0u;
        const int rw = (warp & 3) * 32 + lane, nw = n0 + rw;
        const float glob = NV && l.global_scale != nullptr ? __ldg(l.global_scale) : 1.f;
        const float bias = l.bias != nullptr && nw < l.n_out && p.splits == 1 ? read_value(l.bias, l.dtype, nw) : 0.f;
        const int we = NV ? 0 : top_e[rw] - 140;
        for (int c0 = 16 * (warp >> 2); c0 < p.cols; c0 += 32) {
            uint32_t v[16], v2[16];
            tmem_load16(tmem + ((uint32_t)((warp & 3) * 32) << 16) + c0, v);
            if (p.pieces == 2) tmem_load16(tmem + ((uint32_t)((warp & 3) * 32) << 16) + p.cols + c0, v2);
            tmem_wait_load();
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                const int m = ct * p.cols + c0 + k;
                if (m >= l.rows) break;
                float y = __uint_as_float(v[k]);
                if (p.pieces == 2) y = fmaf(__uint_as_float(v2[k]), 0x1p-11f, y);
                y = blocks == 0 ? 0.f : scale_by_power(y, we - __ldg(p.exponent + m)) * glob;
                if (!ok) y = __uint_as_float(0x7FC00000u);
                if (nw < l.n_out) {
                    if (p.splits > 1) p.partial[((int64_t)split * l.rows + m) * l.n_out + nw] = y;
                    else write_value(l.y, l.dtype, (int64_t)m * l.n_out + nw, y + bias);
                }
            }
            __syncwarp();
        }
        tmem_fence_before();
    }
    __syncthreads();
    if (failed && threadIdx.x == 0) {                              // copies on the way write to this CTA's memory
        failed = 0u;
        for (int s = 0; s < p.stages; ++s) { bar_wait(x_full(s), 0, &failed); bar_wait(x_full(s), 1, &failed); }
    }
    __syncthreads();
    if (warp == 9) tmem_free(tmem, p.columns);
}

__global__ void __launch_bounds__(256) linear_join_kernel(const TilesParams p) {
    const LinearParams& l = p.l;
    const int64_t all = (int64_t)l.rows * l.n_out;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
        float y = 0.f;
        for (int s = 0; s < p.splits; ++s) y += p.partial[s * all + i];
        if (l.bias != nullptr) y += read_value(l.bias, l.dtype, i % l.n_out);
        write_value(l.y, l.dtype, i, y);
    }
}

}  // namespace

TilesPlan tiles_plan(int64_t rows, int64_t n_out, int64_t n_in, int dtype) {
    TilesPlan pl;
    pl.pieces = dtype == MPT_DTYPE_F32 ? 2 : 1;
    const int64_t most = 256 / pl.pieces;
    // even column tiles: of 16 columns each, as few as hold the rows
    const int64_t tiles = (rows + most - 1) / most;
    pl.cols = (int)(((rows + tiles - 1) / tiles + 15) / 16 * 16);
    pl.col_tiles = (int)((rows + pl.cols - 1) / pl.cols);
    pl.row_tiles = (int)((n_out + kRowsW - 1) / kRowsW);
    pl.k_blocks = (int)((n_in + kBlock - 1) / kBlock);
    const int stage = kPartW + pl.pieces * pl.cols * 128, sms = sm_count();
    // two CTAs on an SM where their rings leave room for it, one with a longer ring otherwise
    const int two = (110 * 1024 - 1024) / stage, one = (220 * 1024 - 1024) / stage;
    pl.stages = two >= 3 ? two : one;
    if (pl.stages > kMaxStages) pl.stages = kMaxStages;
    const int64_t ctas = (int64_t)pl.row_tiles * pl.col_tiles, slots = (two >= 3 ? 2 : 1) * (int64_t)sms;
    pl.splits = 1;
    if (ctas * 2 <= slots) {
        const int64_t want = slots / ctas, fit = pl.k_blocks / 4;
        pl.splits = (int)(want > fit ? (fit < 1 ? 1 : fit) : want);
    }
    const int used = pl.pieces * pl.cols;
    pl.columns = used <= 32 ? 32 : used <= 64 ? 64 : used <= 128 ? 128 : 256;
    pl.image_bytes = (size_t)pl.col_tiles * pl.k_blocks * pl.pieces * pl.cols * 128;
    pl.partial_bytes = pl.splits > 1 ? (size_t)pl.splits * rows * n_out * 4 : 0;
    pl.bytes = pl.image_bytes + ((size_t)rows * 4 + 255) / 256 * 256 + pl.partial_bytes;
    return pl;
}

int launch_tiles(const LinearParams& l, const TilesPlan& pl, int format, uint8_t* workspace, cudaStream_t st) {
    if (pl.row_tiles > 65535) { set_error("block_linear: more than %d outputs", 65535 * kRowsW); return MPT_ERR_INVALID_ARGUMENT; }
    TilesParams p;
    p.l = l;
    p.cols = pl.cols; p.pieces = pl.pieces; p.k_blocks = pl.k_blocks; p.splits = pl.splits; p.stages = pl.stages; p.columns = pl.columns;
    p.image = workspace;
    p.exponent = reinterpret_cast<int*>(workspace + pl.image_bytes);
    p.partial = reinterpret_cast<float*>(workspace + pl.image_bytes + ((size_t)l.rows * 4 + 255) / 256 * 256);
    linear_split_kernel<<<(unsigned)l.rows, 256, 0, st>>>(p, workspace);
    const int bytes = 1024 + pl.stages * (kPartW + pl.pieces * pl.cols * 128);
    auto kern = format == MPT_BLOCK_NVFP4 ? linear_tiles_kernel<true> : linear_tiles_kernel<false>;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return check_launch("block_linear");
    kern<<<dim3((unsigned)pl.col_tiles, (unsigned)pl.row_tiles, (unsigned)pl.splits), kThreads, bytes, st>>>(p);
    if (pl.splits > 1) {
        const int64_t blocks = ((int64_t)l.rows * l.n_out + 255) / 256, most = 8 * (int64_t)sm_count();
        linear_join_kernel<<<(unsigned)(blocks < most ? blocks : most), 256, 0, st>>>(p);
    }
    return check_launch("block_linear");
}

}  // namespace mpt
