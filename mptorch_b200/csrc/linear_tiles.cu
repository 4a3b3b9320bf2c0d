// y = x W^T + b for many rows of x, with W held as packed E2M1 codes and group scales (MXFP4, NVFP4): tiles of 128 rows of W by up to
// 256 columns of x on the tcgen05 tensor cores.
//
// Bound: HBM while the rows of x are few (half a byte a weight), the tensor cores beyond some 200 of them.  Two kernels, or three:
//   1. x is scaled for each row by a power of two to a largest value in [2^14, 2^15) and laid out as binary16 tiles of 64 of the sum, in
//      the layout of the products' operands in shared memory, so that a tile is one bulk copy.  float32 takes two such pieces (22
//      bits); bfloat16 and float16 one (exact unless a value is 2^-29 of the row's largest or less).
//   2. The pieces of 256 of the sum of all tiles (128 rows of W by up to 256 columns) are cut into equal runs, one for each SM.  A warp
//      copies x's tiles, a warp issues products, and sixteen warps turn codes into binary16 weights in shared memory, four blocks of
//      64 at a time (a warp then reads 128 bytes of each of four rows), two pieces ahead in registers: one conversion and one
//      multiplication for two weights.  NVFP4: a code times its E4M3 scale is exact (six bits).  MXFP4: a code times
//      2^(13 + e - E), E the row's largest exponent, is exact down to e = E - 36; rows with smaller blocks that are not all zeros are
//      found here and computed by a kernel at the end, in fp32 (rare, and slow: 1024 x 4096 by 4096 takes 123 us without, 200 with 40 such
//      rows, 6.6 ms with nothing else).
//      Sums are fp32 in tensor memory, those of float32's second pieces apart, and the powers of two are put back at the end.
//   3. A tile that a run ends in is left in parts, which are added up in order.
//
// Measured on a B200 (bf16 products at the measured rate and bytes at the measured bandwidth in brackets): 37 x 4096 by 11008 NVFP4
// weights, float16, 37.1 us (4.1 of bytes: the tile kernel alone takes 30, x's tiles 6 and the join 12, which overlap); 1024 x 4096 by
// 4096 MXFP4 weights, float32, 123 us (42 of products, two pieces each; 3 for the look at far blocks); 1024 x 4096 by 11008 NVFP4,
// bfloat16, 174 us (56).  What bounds it is the warps that turn codes into weights, again for every 256 columns of x (128 rows of
// float32): they wait for places in the ring and for codes on the way, with the issue slots 35 % busy and the tensor cores 36 % in the
// second of these.
#include <type_traits>

#include "blocklinear.cuh"
#include "launch.cuh"
#include "tcgen05.cuh"

namespace mpt {
namespace {

// Sixteen warps for the weights: 1024 x 4096 by 4096 MXFP4, float32, took 130 us with eight and takes 120 with sixteen.
constexpr int kRowsW = 128, kBlock = 64, kSuper = 4, kWorkers = 512, kThreads = kWorkers + 64, kRowStep = kWorkers / 8, kEach = kRowsW / kRowStep;   // codes are read in pieces of four blocks
// FOLD, float32 rows: the tensor cores cut their sums off instead of rounding them, an error that grows with the sum's length, so after
// every kFoldNv or kFoldMx pieces (1536 and 4096 of the sum) what there is is added to fp32 sums in memory and begun again.  NVFP4, 1024
// x 4096 by 4096: 3.3e-6 of the result without, 1.7e-6 with 8, 1.1e-6 with 6, 8.1e-7 with 4 (fp32 arithmetic as torch has it 1.1e-6), in
// 110, 128, 145 and 155 us.  MXFP4 loses less: 33 x 4096 by 18889 1.7e-6 without, 9152 4.4e-6 without and 1.5e-6 with 16 (torch's 1.1e-6
// and 1.6e-6), the last in 151 us; it pays more for it, since that kernel has no registers left (1024 x 4096 by 4096: 120 us without,
// 177 with 8; 4352 by 4096, the first size with 16, 182).  Those are weights of normal values; where all codes are as frequent the errors are
// twice as large (4096: 3e-6), and 1.1e-5 where all products have one sign.  bfloat16 and float16 round the result far more coarsely.
constexpr int kFoldNv = 6, kFoldMx = 16;
constexpr int kPartW = kRowsW * 128;                               // bytes of a tile of W: 128 rows of 64 weights

struct TilesParams {
    LinearParams l;
    int cols, pieces, k_blocks, col_tiles, w_stages, x_stages, columns;
    int k_supers;                      // pieces of four blocks of a tile
    int64_t units, per;                // such pieces of all tiles, and of a run
    const uint8_t* image;              // x: [column tile][block of 64][piece][cols][128 bytes]
    int* exponent;                     // of each row of x
    float* partial;                    // of tiles that are cut: [slot][column][128]
    int fold;                          // pieces after which sums are added up in memory and begun again
    float* kept;                       // there: [run][column][128]
    uint8_t* far_rows;                 // MXFP4: 1 for the rows of W that linear_far_kernel computes
};

// ---- x into tiles: a CTA for a row
__global__ void __launch_bounds__(256) linear_split_kernel(const TilesParams p, uint8_t* __restrict__ image) {
    next_may_start();
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

// 2^(13 - d) as binary16, zero where its half, the smallest code's, is below 2^-24
constexpr int kReach = 36;
__device__ __forceinline__ uint32_t half_weight_power(int d) { return d <= 27 ? (uint32_t)(28 - d) << 10 : d <= kReach ? 1u << (37 - d) : 0u; }

constexpr int kMaxStages = 12;                                      // of W's ring; x's has at most eight

// MXFP4: whether row n of W has blocks that are out of its largest exponent's reach and not all zeros
__device__ __noinline__ bool far_blocks(const LinearParams& l, int n, int c, int top, int low) {
    const int groups = l.n_in / 32;
    bool far = false;
    if (top - low > kReach)
        for (int k = c; k < groups; k += 8)
            if (top - (int)__ldg(l.scales + (int64_t)n * groups + k) > kReach) {
                const uint4 w = __ldg(reinterpret_cast<const uint4*>(l.codes + (int64_t)n * (l.n_in >> 1)) + k);
                far |= ((w.x | w.y | w.z | w.w) & 0x77777777u) != 0u;
            }
    const unsigned some = __ballot_sync(0xFFFFFFFFu, far);         // the lanes of a row are four apart
    return ((some >> (threadIdx.x & 3)) & 0x11111111u) != 0u;
}

// MXFP4: the largest exponent of row n of W, found by the eight lanes c of a row (255 is a NaN and no exponent), and whether the row is
// left to linear_far_kernel; bytes up to an aligned word, then words.
template <bool NV>
__device__ __forceinline__ int row_top(const TilesParams& p, int n, int c) {
    if (NV) return 0;
    int top = 0, low = 255;
    const int groups = p.l.n_in / 32;
    if (n < p.l.n_out) {
        const uint8_t* sc = p.l.scales + (int64_t)n * groups;
        auto take = [&](uint32_t e) {
            top = max(top, e == 255u ? 0 : (int)e);
            low = min(low, (int)e);
        };
        const int head = min((int)((4 - (reinterpret_cast<uintptr_t>(sc) & 3)) & 3), groups), words = (groups - head) >> 2;
        if (c < head) take(__ldg(sc + c));
        const uint32_t* from = reinterpret_cast<const uint32_t*>(sc + head);
#pragma unroll 4
        for (int k = c; k < words; k += 8) {
            const uint32_t w = __ldg(from + k);
            take(w & 255u); take((w >> 8) & 255u); take((w >> 16) & 255u); take(w >> 24);
        }
        if (head + 4 * words + c < groups) take(__ldg(sc + head + 4 * words + c));
    }
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
        top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
        low = min(low, __shfl_xor_sync(0xFFFFFFFFu, low, o));
    }
    const bool far = __any_sync(0xFFFFFFFFu, top - low > kReach) && far_blocks(p.l, n, c, top, low);
    if (c == 0 && n < p.l.n_out) p.far_rows[n] = far;
    return top;
}

// A tile's sums, or a run's part of them, or (`more`) those of some pieces of it, which are kept for the next ones (`carry`): a thread has one row of W; the warps of each quarter of rows take every fourth 16 columns.
constexpr uint32_t kEnded = 1u, kWhole = 2u, kCarry = 4u, kMore = 8u, kNext = 16u;     // kNext: the run's next piece is another tile's
template <bool NV, bool FOLD>
__device__ __noinline__ void tile_end(const TilesParams& p, uint32_t tmem, const int* top_e, int tile, uint32_t what, bool begins, bool ok) {
    const bool whole = what & kWhole, carry = FOLD && (what & kCarry), more = FOLD && (what & kMore);
    const LinearParams& l = p.l;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rt = tile / p.col_tiles, ct = tile - rt * p.col_tiles;
    tmem_fence_after();
    const int rw = (warp & 3) * 32 + lane, n = rt * kRowsW + rw;
    const float glob = NV && l.global_scale != nullptr ? __ldg(l.global_scale) : 1.f;
    const float bias = whole && l.bias != nullptr && n < l.n_out ? load_value(l.bias, l.dtype, n) : 0.f;
    const int we = NV ? 0 : top_e[rw] - 140;
    const bool near = we >= -60 && we <= 60;                       // no product leaves fp32's range on the way
    const float wpow = __uint_as_float((uint32_t)(127 + (near ? we : 0)) << 23);
    float* part = p.partial + (2 * (int64_t)blockIdx.x + (begins ? 0 : 1)) * p.cols * kRowsW + rw;
    float* kept = p.kept + (int64_t)blockIdx.x * p.cols * kRowsW + rw;
    for (int c0 = 16 * (warp >> 2); c0 < p.cols; c0 += kWorkers / 8) {
        uint32_t v[16], v2[16];
        float before[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) before[k] = carry && ct * p.cols + c0 + k < l.rows ? kept[(c0 + k) * kRowsW] : 0.f;
        const int m_lane = ct * p.cols + c0 + (lane & 15), mine = m_lane < l.rows ? p.exponent[m_lane] : 0;
        tmem_load16(tmem + ((uint32_t)((warp & 3) * 32) << 16) + c0, v);
        if (p.pieces == 2) tmem_load16(tmem + ((uint32_t)((warp & 3) * 32) << 16) + p.cols + c0, v2);
        tmem_wait_load();
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const int m = ct * p.cols + c0 + k, xe = __shfl_sync(0xFFFFFFFFu, mine, k);
            if (m < l.rows) {
                float y = __uint_as_float(v[k]);
                if (p.pieces == 2) y = fmaf(__uint_as_float(v2[k]), 0x1p-11f, y);
                if (near) y = y * wpow * __uint_as_float((uint32_t)(127 - xe) << 23);
                else y = scale_by_power(y, we - xe);
                y *= glob;
                if (carry) y += before[k];
                if (!ok) y = __uint_as_float(0x7FC00000u);
                if (more) kept[(c0 + k) * kRowsW] = y;
                else if (!whole) part[(c0 + k) * kRowsW] = y;
                else if (n < l.n_out) store_value(l.y, l.dtype, (int64_t)m * l.n_out + n, y + bias);
            }
        }
        __syncwarp();
    }
    tmem_fence_before();
}

// PER: blocks of a place in the rings, one or (where x's tiles are small) the four of a piece: what is waited for and handed on costs some
// hundred clocks each time.
template <bool NV, int PER, bool FOLD>
__global__ void __launch_bounds__(kThreads) linear_tiles_kernel(const __grid_constant__ TilesParams p) {
    next_may_start();
    extern __shared__ uint8_t smem_raw[];
    const LinearParams& l = p.l;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t base = (smem_at(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem = smem_raw + (base - smem_at(smem_raw));
    const int x_bytes = p.pieces * p.cols * 128, x_base = p.w_stages * PER * kPartW;
    const int64_t u0 = blockIdx.x * p.per, u1 = u0 + p.per < p.units ? u0 + p.per : p.units;
    if (u0 >= u1) {
        wait_for_previous();                                       // no CTA is done before the kernel that this one follows
        return;
    }
    __shared__ __align__(8) uint64_t bars[2 * kMaxStages + 16 + 4];
    __shared__ uint32_t tmem_slot, failed;
    __shared__ int top_e[2][kRowsW];
    auto w_full = [&](int s) { return smem_at(&bars[s]); };
    auto w_empty = [&](int s) { return smem_at(&bars[kMaxStages + s]); };
    auto x_full = [&](int s) { return smem_at(&bars[2 * kMaxStages + s]); };
    auto x_empty = [&](int s) { return smem_at(&bars[2 * kMaxStages + 8 + s]); };
    auto done = [&](int t) { return smem_at(&bars[2 * kMaxStages + 16 + (t & 1)]); };      // the sums of tile t of the run are there
    auto taken = [&](int t) { return smem_at(&bars[2 * kMaxStages + 18 + (t & 1)]); };     // and have been read
    if (threadIdx.x == 0) {
        for (int s = 0; s < p.w_stages; ++s) { bar_init(w_full(s), kWorkers / kSuper * PER); bar_init(w_empty(s), 1); }
        for (int s = 0; s < p.x_stages; ++s) { bar_init(x_full(s), 1); bar_init(x_empty(s), 1); }
        for (int t = 0; t < 2; ++t) { bar_init(done(t), 1); bar_init(taken(t), kWorkers); }
        failed = 0u;
        fence_barrier_init();
    }
    if (warp == kWorkers / 32 + 1) tmem_alloc(smem_at(&tmem_slot), p.columns);
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = tmem_slot;
    const int tile0 = (int)(u0 / p.k_supers), super0 = (int)(u0 % p.k_supers), count = (int)(u1 - u0);
    auto blocks_of = [&](int super) { return min(kSuper, p.k_blocks - super * kSuper); };

    if (warp == kWorkers / 32) {
        if (lane == 0) {
            wait_for_previous();                                   // x's tiles
            int tile = tile0, super = super0, stage = 0, turn = 0;
            bool ok = true;
            for (int i = 0; ok && i < count; ++i) {
                const uint8_t* from = p.image + ((int64_t)(tile % p.col_tiles) * p.k_blocks + super * kSuper) * x_bytes;
                const int blocks = blocks_of(super);
                for (int q = 0; q < blocks; q += PER) {
                    const uint32_t bytes = min(PER, blocks - q) * x_bytes;
                    if (turn > 0 && !(ok = bar_wait(x_empty(stage), (turn - 1) & 1, &failed))) break;
                    bar_expect(x_full(stage), bytes);
                    bulk_load(base + x_base + stage * PER * x_bytes, from + (int64_t)q * x_bytes, bytes, x_full(stage));
                    if (++stage == p.x_stages) { stage = 0; ++turn; }
                }
                if (++super == p.k_supers) { super = 0; ++tile; }
            }
        }
        __syncwarp();
    } else if (warp == kWorkers / 32 + 1) {
        {
            const bool leader = lane == 0;
            const uint32_t sums = uniform(tmem), ring = uniform(base);
            const int n = p.pieces * p.cols;                       // the pieces' columns side by side, sums apart
            const uint32_t desc = half_product_descriptor(n);
            int super = super0, fold = p.fold - super0 % p.fold, ws = 0, wt = 0, xs = 0, xt = 0, t = 0;
            bool first = true, ok = true;
            for (int i = 0; ok && i < count; ++i) {
                if (first && t > 1 && !(ok = __all_sync(0xFFFFFFFFu, bar_wait(taken(t), ((t >> 1) - 1) & 1, &failed)))) break;
                const uint32_t to = sums + (t & 1) * (p.columns >> 1);
                const int blocks = blocks_of(super);
                for (int q = 0; q < blocks; q += PER) {
                    ok = bar_wait(x_full(xs), xt & 1, &failed) && bar_wait(w_full(ws), wt & 1, &failed);
                    ok = __all_sync(0xFFFFFFFFu, ok);
                    if (!ok) break;
                    tmem_fence_after();
                    uint64_t w = tile_descriptor(ring + ws * PER * kPartW, 16), x = tile_descriptor(ring + x_base + xs * PER * x_bytes, 16);
#pragma unroll
                    for (int b = 0; b < PER; ++b) {
                        if (q + b < blocks) {
#pragma unroll
                            for (int k = 0; k < kBlock / 16; ++k) mma_ss(to, w + 2 * k, x + 2 * k, desc, !first || k > 0, leader);
                            first = false;
                            w += kPartW >> 4;
                            x += x_bytes >> 4;
                        }
                    }
                    mma_commit(w_empty(ws), leader);
                    mma_commit(x_empty(xs), leader);
                    if (++ws == p.w_stages) { ws = 0; ++wt; }
                    if (++xs == p.x_stages) { xs = 0; ++xt; }
                }
                if (++super == p.k_supers) super = 0;
                if (super == 0 || (FOLD && --fold == 0) || i + 1 == count) {
                    mma_commit(done(t), leader);
                    ++t;
                    first = true;
                    fold = p.fold;
                }
            }
        }
        __syncwarp();
    } else {
        // ---- weights: lane (c, row) takes 32 weights, half of block c / 2 of the piece, of row r and those kRowStep apart
        const int c = lane >> 2, r = warp * 4 + (lane & 3), q_mine = c >> 1, half = c & 1;
        const int groups = l.n_in / (NV ? 16 : 32);
        constexpr int kAhead = 2;
        uint4 ahead[kAhead][kEach] = {};
        uint32_t ahead_s[kAhead][kEach] = {};
        const int last = l.n_in / 32 - 1;                          // of a row's pieces of 32 weights
        int next_ct = tile0 % p.col_tiles, next_rt = tile0 / p.col_tiles, next_super = super0, next_left = count;
        const uint8_t *codes[kEach], *scales[kEach];
        auto next_rows = [&]() {
#pragma unroll
            for (int v = 0; v < kEach; ++v) {
                const int64_t n = min(next_rt * kRowsW + r + kRowStep * v, l.n_out - 1);
                codes[v] = l.codes + n * (l.n_in >> 1);
                scales[v] = l.scales + n * groups;
            }
        };
        next_rows();
        // What lies outside the matrix is read from a place inside (and scaled by zero when it is used: a choice made here would wait
        // for the load).
        auto fetch = [&](uint4 (&w)[kEach], uint32_t (&sc)[kEach]) {
            if (next_left > 0) {
                const int at = min(next_super * 8 + c, last);
                if (at >= 0) {
#pragma unroll
                    for (int v = 0; v < kEach; ++v) {
                        w[v] = __ldg(reinterpret_cast<const uint4*>(codes[v]) + at);
                        if (NV) sc[v] = __ldg(reinterpret_cast<const uint16_t*>(scales[v]) + at);
                        else sc[v] = __ldg(scales[v] + at);
                    }
                }
                --next_left;
                if (++next_super == p.k_supers) {
                    next_super = 0;
                    if (++next_ct == p.col_tiles) { next_ct = 0; ++next_rt; next_rows(); }
                }
            }
        };
#pragma unroll
        for (int a = 0; a < kAhead; ++a) fetch(ahead[a], ahead_s[a]);

        // Sums are read `ends` times in all: at the end of each tile, and after every p.fold pieces of one.
        int tile = tile0, super = super0, ends = 0, i = 0, stage = 0, turn = 0, fold = p.fold - super0 % p.fold, top[kEach];
        uint32_t ended = 0u;                                       // sums that have not been read yet, and of what they are
        uint32_t carry = 0u;                                       // kCarry, if there are kept sums of this tile
        int ct = tile0 % p.col_tiles, rt = tile0 / p.col_tiles;
        bool live[kEach];
        auto begin_rows = [&](int t, bool next) {
#pragma unroll
            for (int h = 0; h < kEach; ++h) {
                const int n = rt * kRowsW + r + kRowStep * h;
                live[h] = n < l.n_out;
                if (t == 0 || (next && ct == 0)) top[h] = row_top<NV>(p, n, c);          // otherwise the same rows again
                if (!NV && c == 0) top_e[t & 1][r + kRowStep * h] = top[h];
            }
        };
        auto end_tile = [&]() {                                    // time `ends - 1`
            bar_wait(done(ends - 1), ((ends - 1) >> 1) & 1, &failed);
            if (ends == 1) wait_for_previous();                   // the exponents of x
            asm volatile("bar.sync 1, %0;" ::"n"(kWorkers) : "memory");      // and every thread's part of top_e
            tile_end<NV, FOLD>(p, tmem + ((ends - 1) & 1) * (p.columns >> 1), top_e[(ends - 1) & 1], tile - (ended & kNext ? 1 : 0), ended, tile - (ended & kNext ? 1 : 0) == tile0, *(volatile uint32_t*)&failed == 0u);
            bar_arrive(taken(ends - 1));
            ended = 0u;
            asm volatile("bar.sync 1, %0;" ::"n"(kWorkers) : "memory");      // top_e has been read
        };
        begin_rows(0, true);
        while (i < count || ended) {
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
                const bool worked = i < count;
                if (worked) {
                    const int blocks = blocks_of(super);
                    int s = stage, t = turn;
                    if (PER == 1) {
                        s += q_mine;
                        if (s >= p.w_stages) { s -= p.w_stages; ++t; }
                    }
                    if (PER > 1 || q_mine < blocks) {
                        // (a lane does not use a place each turn, but its blocks are at most seven apart and the ring has seven places
                        // at least: the phase before the one that it waits for is over)
                        if (t > 0) bar_wait(w_empty(s), (t - 1) & 1, &failed);
                        const bool inside = super * 8 + c <= last;
#pragma unroll
                        for (int v = 0; v < kEach; ++v) {
                            const uint4 w = ahead[a][v];
                            const uint32_t sc = ahead_s[a][v];
                            const bool on = inside && live[v];
                            uint32_t h[16], f[2];
                            e2m1x8_to_half(w.x, *reinterpret_cast<uint32_t(*)[4]>(h));
                            e2m1x8_to_half(w.y, *reinterpret_cast<uint32_t(*)[4]>(h + 4));
                            e2m1x8_to_half(w.z, *reinterpret_cast<uint32_t(*)[4]>(h + 8));
                            e2m1x8_to_half(w.w, *reinterpret_cast<uint32_t(*)[4]>(h + 12));
                            if (NV) {
                                uint32_t u;
                                e4m3x4_to_half(on ? __byte_perm(sc, 0u, 0x0000) : 0u, f[0], u);
                                e4m3x4_to_half(on ? __byte_perm(sc, 0u, 0x1111) : 0u, f[1], u);
                            } else {
                                const uint32_t q = !on ? 0u : sc == 255u ? 0x7E00u : half_weight_power(top[v] - (int)sc);
                                f[0] = f[1] = q | (q << 16);
                            }
#pragma unroll
                            for (int q = 0; q < 16; ++q) {
                                const __half2 x = __hmul2(*reinterpret_cast<__half2*>(&h[q]), *reinterpret_cast<__half2*>(&f[q >> 3]));
                                h[q] = *reinterpret_cast<const uint32_t*>(&x);
                            }
                            const int row = r + kRowStep * v;
                            uint8_t* to = smem + (PER == 1 ? s : s * PER + q_mine) * kPartW + row * 128;
#pragma unroll
                            for (int q = 0; q < 4; ++q)
                                *reinterpret_cast<uint4*>(to + (((half * 4 + q) ^ (row & 7)) << 4)) = make_uint4(h[4 * q], h[4 * q + 1], h[4 * q + 2], h[4 * q + 3]);
                        }
                        fence_async_proxy();
                        bar_arrive(w_full(s));
                    }
                    fetch(ahead[a], ahead_s[a]);
                    stage += PER == 1 ? blocks : 1;
                    if (stage >= p.w_stages) { stage -= p.w_stages; ++turn; }
                    if (++super == p.k_supers) super = 0;
                    ++i;
                    --fold;
                }
                // the sums of a tile are read when the first piece of the next one is under way
                if (ended) end_tile();
                if (worked && (super == 0 || (FOLD && fold == 0) || i == count)) {
                    const bool more = FOLD && super != 0 && i < count;     // pieces of this tile
                    ended = kEnded | carry | (more ? kMore : 0u) | (super == 0 && i >= p.k_supers ? kWhole : 0u);
                    carry = more ? kCarry : 0u;
                    fold = p.fold;
                    ++ends;
                    if (!more) {
                        ++tile;
                        ended |= kNext;
                        if (++ct == p.col_tiles) { ct = 0; ++rt; }
                    }
                    if (i < count) begin_rows(ends, !more);
                    else end_tile();
                }
            }
        }
    }
    __syncthreads();
    if (failed && threadIdx.x == 0) {                              // copies on the way write to this CTA's memory
        failed = 0u;
        for (int s = 0; s < p.x_stages; ++s) { bar_wait(x_full(s), 0, &failed); bar_wait(x_full(s), 1, &failed); }
    }
    __syncthreads();
    if (warp == kWorkers / 32 + 1) tmem_free(tmem, p.columns);
}

// MXFP4: the rows of W that are marked, in fp32.  CTAs (x, .) look at rows 4096 x and on and share what there is to do: four rows of x for
// each warp and row of W at a time.
constexpr int kFarRows = 4096, kFarCols = 4;
__global__ void __launch_bounds__(256) linear_far_kernel(const TilesParams p) {
    const LinearParams& l = p.l;
    __shared__ uint16_t rows[kFarRows];                            // in order, so that all CTAs count alike
    __shared__ int of_warp[8];
    const int lane = threadIdx.x & 31, groups = l.n_in / 32, n0 = blockIdx.x * kFarRows, mine = n0 + 16 * threadIdx.x;
    wait_for_previous();
    uint32_t f[4] = {}, marked = 0u;
    if (mine < l.n_out) *reinterpret_cast<uint4*>(f) = *reinterpret_cast<const uint4*>(p.far_rows + mine);       // (the marks end at a multiple of 16 bytes)
#pragma unroll
    for (int i = 0; i < 16; ++i) marked |= mine + i < l.n_out && (f[i >> 2] >> (8 * (i & 3)) & 1u) ? 1u << i : 0u;
    int upto = __popc(marked);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xFFFFFFFFu, upto, o);
        if (lane >= o) upto += v;
    }
    if (lane == 31) of_warp[threadIdx.x >> 5] = upto;
    if (!__syncthreads_or(marked != 0u)) return;
    int count = 0, at = upto - __popc(marked);
    for (int w = 0; w < 8; ++w) {
        if (w < (int)(threadIdx.x >> 5)) at += of_warp[w];
        count += of_warp[w];
    }
    for (; marked; marked &= marked - 1) rows[at++] = (uint16_t)(16 * threadIdx.x + __ffs(marked) - 1);
    __syncthreads();
    const int each = (l.rows + 8 * kFarCols - 1) / (8 * kFarCols);
    for (int64_t item = blockIdx.y; item < (int64_t)count * each; item += gridDim.y) {
        const int64_t n = n0 + rows[item / each];
        const int m0 = ((int)(item % each) * 8 + (threadIdx.x >> 5)) * kFarCols;
        if (m0 >= l.rows) continue;
        const uint8_t *codes = l.codes + n * (l.n_in >> 1), *scales = l.scales + n * groups;
        const float bias = l.bias != nullptr ? load_value(l.bias, l.dtype, n) : 0.f;
        float sum[kFarCols] = {};
        for (int k = lane; k < l.n_in / 8; k += 32) {
            float w[8], x[kFarCols][8];
            decode8<true>(make_uint2(__ldg(reinterpret_cast<const uint32_t*>(codes) + k), 0u), w);
            const float scale = e8m0_value(__ldg(scales + (k >> 2)));
#pragma unroll
            for (int j = 0; j < kFarCols; ++j) read8(l.x, l.dtype, l.x_vec, (int64_t)min(m0 + j, l.rows - 1) * l.n_in + 8 * (int64_t)k, x[j]);
#pragma unroll
            for (int j = 0; j < kFarCols; ++j) {
                float here = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) here = fmaf(w[i], x[j][i], here);
                sum[j] = fmaf(here, scale, sum[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < kFarCols; ++j) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum[j] += __shfl_xor_sync(0xFFFFFFFFu, sum[j], o);
            if (lane == 0 && m0 + j < l.rows) store_value(l.y, l.dtype, (m0 + j) * (int64_t)l.n_out + n, sum[j] + bias);
        }
    }
}

// Adds up the tiles that runs end in: CTAs (x, .) look at the end of run x.
__global__ void __launch_bounds__(256) linear_join_kernel(const TilesParams p) {
    next_may_start();
    const LinearParams& l = p.l;
    const int64_t cut = (blockIdx.x + 1) * p.per;
    wait_for_previous();
    if (cut >= p.units || cut % p.k_supers == 0) return;           // nothing is cut here
    const int64_t tile = cut / p.k_supers, p0 = tile * p.k_supers, p1 = p0 + p.k_supers;
    if ((int64_t)blockIdx.x * p.per > p0) return;                  // an earlier CTA adds this one up
    const int last = (int)((p1 - 1) / p.per);
    const int rt = (int)(tile / p.col_tiles), ct = (int)(tile - (int64_t)rt * p.col_tiles), here = min(p.cols, l.rows - ct * p.cols);
    for (int i = blockIdx.y * 256 + threadIdx.x; i < here * kRowsW; i += gridDim.y * 256) {
        const int m = ct * p.cols + i / kRowsW, n = rt * kRowsW + i % kRowsW;
        if (n >= l.n_out) continue;
        float y = 0.f;
        for (int k = blockIdx.x; k <= last; ++k)
            y += p.partial[(2 * (int64_t)k + (k == (int)blockIdx.x && k * p.per < p0 ? 1 : 0)) * p.cols * kRowsW + i];
        if (l.bias != nullptr) y += load_value(l.bias, l.dtype, n);
        store_value(l.y, l.dtype, (int64_t)m * l.n_out + n, y);
    }
}

}  // namespace

TilesPlan tiles_plan(int64_t rows, int64_t n_out, int64_t n_in, int format, int dtype) {
    TilesPlan pl;
    pl.pieces = dtype == MPT_DTYPE_F32 ? 2 : 1;
    const int64_t most = 256 / pl.pieces;
    // even column tiles: of 16 columns each, as few as hold the rows
    const int64_t parts = (rows + most - 1) / most;
    pl.cols = (int)(((rows + parts - 1) / parts + 15) / 16 * 16);
    pl.col_tiles = (int)((rows + pl.cols - 1) / pl.cols);
    pl.row_tiles = (int)((n_out + kRowsW - 1) / kRowsW);
    pl.k_blocks = n_in > 0 ? (int)((n_in + kBlock - 1) / kBlock) : 1;
    // Rings: where x's tiles are small, places of four blocks (24 rows of 4096 by 11008 NVFP4, bfloat16: 33 us, 40 with single blocks; 64
    // rows: 41 and 48); else single blocks, since two places of four would not fit.  x's ring covers the latency of a copy with three
    // places or four, the rest is W's: seven places at least, which the wait of a worker's lane counts on.
    const int x_bytes = pl.pieces * pl.cols * 128, room = 219 * 1024;
    pl.ring_blocks = x_bytes <= 8 * 1024 ? kSuper : 1;
    pl.x_stages = pl.ring_blocks > 1 ? 2 : x_bytes <= 16 * 1024 ? 4 : 3;
    pl.w_stages = (room - pl.x_stages * pl.ring_blocks * x_bytes) / (pl.ring_blocks * kPartW);
    if (pl.w_stages > kMaxStages) pl.w_stages = kMaxStages;
    // Equal runs, one for each SM; or whole tiles, where their number leaves at most a sixteenth of the SMs' time idle: no parts and no
    // third kernel (1024 x 768 by 50257 MXFP4, bfloat16: 263 us, 303 in equal runs).
    const int64_t tiles = (int64_t)pl.row_tiles * pl.col_tiles, sms = sm_count(), rounds = (tiles + sms - 1) / sms;
    pl.k_supers = (pl.k_blocks + kSuper - 1) / kSuper;
    pl.units = tiles * pl.k_supers;
    pl.per = (pl.units + sms - 1) / sms;
    if (tiles >= sms && tiles * 16 >= rounds * sms * 15) pl.per = rounds * pl.k_supers;
    pl.runs = (int)((pl.units + pl.per - 1) / pl.per);
    const int used = pl.pieces * pl.cols;
    pl.columns = used <= 16 ? 32 : used <= 32 ? 64 : used <= 64 ? 128 : used <= 128 ? 256 : 512;      // two sets of sums
    pl.image_bytes = (size_t)pl.col_tiles * pl.k_blocks * pl.pieces * pl.cols * 128;
    pl.partial_bytes = pl.runs > 1 && pl.per % pl.k_supers ? (size_t)2 * pl.runs * pl.cols * kRowsW * 4 : 0;
    const int fold = format == MPT_BLOCK_NVFP4 ? kFoldNv : kFoldMx;
    pl.fold = pl.pieces == 2 && pl.k_supers > fold ? fold : pl.k_supers;
    pl.kept_bytes = pl.fold < pl.k_supers ? (size_t)pl.runs * pl.cols * kRowsW * 4 : 0;
    pl.far_bytes = format == MPT_BLOCK_MXFP4 ? ((size_t)n_out + 15) / 16 * 16 : 0;
    pl.bytes = pl.image_bytes + ((size_t)rows * 4 + 255) / 256 * 256 + pl.partial_bytes + pl.kept_bytes + pl.far_bytes;
    return pl;
}

int launch_tiles(const LinearParams& l, const TilesPlan& pl, int format, uint8_t* workspace, cudaStream_t st) {
    TilesParams p;
    p.l = l;
    p.cols = pl.cols; p.pieces = pl.pieces; p.k_blocks = pl.k_blocks; p.col_tiles = pl.col_tiles; p.k_supers = pl.k_supers; p.units = pl.units; p.per = pl.per; p.w_stages = pl.w_stages; p.x_stages = pl.x_stages; p.columns = pl.columns;
    p.image = workspace;
    p.exponent = reinterpret_cast<int*>(workspace + pl.image_bytes);
    p.partial = reinterpret_cast<float*>(workspace + pl.image_bytes + ((size_t)l.rows * 4 + 255) / 256 * 256);
    p.fold = pl.fold;
    p.kept = p.partial + pl.partial_bytes / 4;
    p.far_rows = pl.far_bytes ? reinterpret_cast<uint8_t*>(p.kept) + pl.kept_bytes : nullptr;
    linear_split_kernel<<<(unsigned)l.rows, 256, 0, st>>>(p, workspace);
    const int bytes = 1024 + pl.ring_blocks * (pl.w_stages * kPartW + pl.x_stages * pl.pieces * pl.cols * 128);
    const bool nv = format == MPT_BLOCK_NVFP4, single = pl.ring_blocks == 1;
    constexpr int most = 221 * 1024;                               // beside 3 kB of its own
    auto launch = [&](auto kern, bool allowed) {
        if (!allowed) return false;
        launch_after(kern, dim3((unsigned)pl.runs), dim3(kThreads), bytes, st, p);
        return true;
    };
    const bool fold = pl.fold < pl.k_supers;
    auto choose = [&](auto nv_c, auto fold_c) {
        constexpr bool kNv = decltype(nv_c)::value, kFolds = decltype(fold_c)::value;
        return single ? launch(linear_tiles_kernel<kNv, 1, kFolds>, allow_shared<linear_tiles_kernel<kNv, 1, kFolds>>(most))
                      : launch(linear_tiles_kernel<kNv, kSuper, kFolds>, allow_shared<linear_tiles_kernel<kNv, kSuper, kFolds>>(most));
    };
    using Yes = std::true_type;
    using No = std::false_type;
    const bool fine = nv ? (fold ? choose(Yes{}, Yes{}) : choose(Yes{}, No{})) : (fold ? choose(No{}, Yes{}) : choose(No{}, No{}));
    if (!fine) {
        check_launch("block_linear");
        set_error("block_linear: the kernel does not fit this device");
        return MPT_ERR_CUDA;
    }
    if (pl.partial_bytes) launch_after(linear_join_kernel, dim3((unsigned)(pl.runs - 1), 4), dim3(256), 0, st, p);
    if (pl.far_bytes) {
        const int groups = (int)(((int64_t)l.n_out + kFarRows - 1) / kFarRows), parts = 2 * sm_count() / groups;
        launch_after(linear_far_kernel, dim3((unsigned)groups, (unsigned)(parts < 1 ? 1 : parts)), dim3(256), 0, st, p);
    }
    return check_launch("block_linear");
}

}  // namespace mpt
