// Attention of chunks of new rows over a paged MX cache: 128 rows of q at a time on the tcgen05 tensor cores.
//
// Bound: the tensor cores, 4 dim operations for each pair of a row and a visible token, and beside them the exponentials (16 a
// clock on an SM).  Two kernels.  The first expands the sequences' K and V into bfloat16, where a code times its scale is exact, as
// tiles of 128 tokens in the very layout that the second one's operands have in shared memory, so that a tile is one bulk copy: it
// costs one pass over the cache (a byte read and two written an element), where expanding inside the second kernel would repeat it
// for every 128 rows.  The second is a warp that copies, a warp that issues products, and four warps with a row a thread:
//   S = Q K^T (tensor memory) -> p = exp(s - m) as bfloat16 over S's own columns -> O += P V, P read from tensor memory.
// m is moved, and O multiplied, only when a row's maximum has grown by more than 2^8 over it; p is at most 2^8 then.
//
// Accuracy.  bfloat16 queries are one operand; float16 and float32 ones are the sum of two and three bfloat16 pieces (16 and 24
// bits), and so are their weights p; sums are fp32 throughout.
//
// Measured figures stand at the launch rule below.
#include <atomic>

#include "attention.cuh"
#include "attention_chunk.cuh"
#include "tcgen05.cuh"

namespace mpt {
namespace {

constexpr int kTile = 128, kPart = 128 * 128;                     // tokens and rows of a tile; bytes of 128 rows of 64 values
constexpr int kTrailer = 256;                                     // there[4], any V block NaN, -, -, -, then a byte of blocks for each token

__host__ __device__ constexpr int parts_for(int dim) { return (dim + 63) / 64; }
__host__ __device__ constexpr int tile_bytes(int dim) { return 2 * parts_for(dim) * kPart + kTrailer; }

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float bf16_lo(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t x) { return __uint_as_float(x & 0xFFFF0000u); }

// ---- expanding.  One CTA for 128 tokens of a (sequence, kv head).
template <bool FP4>
__global__ void __launch_bounds__(256) mx_expand_kernel(const AttentionParams p, uint8_t* __restrict__ tiles, int tiles_per_seq) {
    const CacheView& c = p.c;
    const int head = blockIdx.y, t0 = blockIdx.x * kTile, nb = c.dim >> 5;
    for (int seq = blockIdx.z; seq < c.seqs; seq += gridDim.z) {
        const int n = rows_of(c, seq).y, len = __ldg(c.lens + seq), end = min(len, c.capacity());
        if (n == 0 || t0 >= end) continue;
        if (p.window > 0 && t0 + kTile <= len - n - p.window + 1 && t0 >= p.sinks) continue;    // no row sees these
        uint8_t* out = tiles + (((int64_t)seq * c.heads + head) * tiles_per_seq + blockIdx.x) * tile_bytes(c.dim);
        __shared__ int64_t row_at[kTile];
        __shared__ uint32_t there[4], any_nan;
        __shared__ uint8_t nan_blocks[kTile];
        __syncthreads();
        if (threadIdx.x == 0) any_nan = 0u;
        __syncthreads();
        if (threadIdx.x < kTile) {
            const int t = t0 + threadIdx.x;
            const int64_t row = t < end ? c.row_of(seq, t, head) : -1;
            row_at[threadIdx.x] = row;
            const uint32_t b = __ballot_sync(0xFFFFFFFFu, row >= 0);
            if ((threadIdx.x & 31) == 0) there[threadIdx.x >> 5] = b;
            uint32_t bad = 0u;
            if (row >= 0)
                for (int i = 0; i < nb; ++i) bad |= c.v_scales[row * nb + i] == 255 ? 1u << i : 0u;
            nan_blocks[threadIdx.x] = (uint8_t)bad;
            if (bad) any_nan = 1u;
        }
        __syncthreads();
        const int pieces = c.dim >> 3, row_bytes = FP4 ? c.dim >> 1 : c.dim;
        for (int i = threadIdx.x; i < kTile * pieces; i += 256) {
            const int tok = i / pieces, ch = i - tok * pieces;
            const int64_t row = row_at[tok];
            const int at = (ch >> 3) * kPart + tok * 128 + (((ch & 7) ^ (tok & 7)) << 4);
#pragma unroll
            for (int side = 0; side < 2; ++side) {
                float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                if (row >= 0) {
                    const uint8_t* from = (side ? c.v_codes : c.k_codes) + row * row_bytes + (FP4 ? ch * 4 : ch * 8);
                    const uint32_t sc = __ldg((side ? c.v_scales : c.k_scales) + row * nb + (ch >> 2));
                    uint2 w;
                    if (FP4) w = make_uint2(__ldg(reinterpret_cast<const uint32_t*>(from)), 0u);
                    else w = __ldg(reinterpret_cast<const uint2*>(from));
                    decode8<FP4>(w, x);
                    const float s = e8m0_value(sc);
                    // a block of V that is NaN takes no part in the product; its rows are told at the end
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = side && sc == 255u ? 0.f : x[e] * s;
                }
                uint4 v;
                v.x = pack_bf16(x[0], x[1]); v.y = pack_bf16(x[2], x[3]); v.z = pack_bf16(x[4], x[5]); v.w = pack_bf16(x[6], x[7]);
                *reinterpret_cast<uint4*>(out + side * parts_for(c.dim) * kPart + at) = v;
            }
        }
        uint32_t* tail = reinterpret_cast<uint32_t*>(out + 2 * parts_for(c.dim) * kPart);
        if (threadIdx.x < 4) tail[threadIdx.x] = there[threadIdx.x];
        if (threadIdx.x == 4) tail[4] = any_nan;
        if (threadIdx.x < kTile) reinterpret_cast<uint8_t*>(tail)[32 + threadIdx.x] = nan_blocks[threadIdx.x];
    }
}

// ---- attention
constexpr int kThreads = 192;                                     // four warps of rows, one that copies, one that issues products
enum { kKFull, kKEmpty, kVFull, kVEmpty, kScores, kScores2, kWeights, kWeights2, kValues, kBars };

template <int DIM, int PIECES, int NS>
struct ChunkShape {
    static constexpr int parts = parts_for(DIM), q_bytes = PIECES * parts * kPart, side = parts * kPart;
    static constexpr int smem = 1024 + q_bytes + 2 * side + 4 * kTrailer;
    // columns of tensor memory: scores (a set for each of NS), sums, and weights that do not fit over the scores
    static constexpr int sums = NS * 128, more = sums + DIM, used = more + (PIECES == 3 ? 64 * NS : 0), columns = used <= 256 ? 256 : 512;
    static_assert(used <= 512, "tensor memory");
    static_assert(smem <= 227 * 1024, "shared memory");
};

template <int DIM, int PIECES, int NS>
__global__ void __launch_bounds__(kThreads, NS == 1 ? 2 : 1) mx_attention_chunk_kernel(const AttentionParams p, const uint8_t* __restrict__ tiles, int tiles_per_seq) {
    using Shape = ChunkShape<DIM, PIECES, NS>;
    extern __shared__ uint8_t smem_raw[];
    const CacheView& c = p.c;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint8_t* smem = smem_raw + ((1024u - (smem_at(smem_raw) & 1023u)) & 1023u);
    uint8_t* q_sm = smem;
    const uint32_t q_at = smem_at(smem), k_at = q_at + Shape::q_bytes, v_at = k_at + Shape::side, tail_at = v_at + Shape::side;
    const uint8_t* tails = smem + Shape::q_bytes + 2 * Shape::side;
    __shared__ int64_t place_sm[kPlaceWords];
    __shared__ __align__(8) uint64_t bars[kBars];
    __shared__ uint32_t tmem_slot, failed;

    zero_outside(p);
    Place at;
    int64_t per;
    const int64_t total = find_place<kTile>(p, blockIdx.x, per, at, place_sm);
    int64_t left = min(per, total - blockIdx.x * per);
    if (left <= 0) return;

    auto bar = [&](int i) { return smem_at(&bars[i]); };
    if (threadIdx.x == 0) {
        for (int i = 0; i < kBars; ++i) bar_init(bar(i), i == kWeights || i == kWeights2 ? 128 : 1);
        failed = 0u;
        fence_barrier_init();
    }
    if (warp == 5) tmem_alloc(smem_at(&tmem_slot), Shape::columns);
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = tmem_slot;

    const float sign = p.scale_log2 > 0.f ? 1.f : p.scale_log2 < 0.f ? -1.f : 0.f;      // of q, so that the largest score is of the largest sum
    const float mul = p.scale_log2 == 0.f ? 1.f : fabsf(p.scale_log2);
    uint32_t it0 = 0;                                             // pieces before this segment
    bool begins = true;
    while (left > 0) {
        const int seq = at.seq, head = at.head, pieces = at.w.pieces(at.tile);
        const int take = (int)min((int64_t)(pieces - at.piece), left);
        const int2 own = rows_of(c, seq);
        const int first = at.tile * kTile, count = min(kTile, own.y * p.group - first);
        const int pos0 = __ldg(c.lens + seq) - own.y;
        const int low_pos = pos0 + first / p.group, high_pos = pos0 + (first + count - 1) / p.group;
        const TokenTiles<kTile> tt(p, low_pos, high_pos);
        const bool finished = take == pieces;
        const int j_lo = min(at.piece, tt.tiles), n = min(at.piece + take, tt.tiles) - j_lo;

        // ---- q, in pieces
        for (int i = threadIdx.x; i < kTile * (DIM / 8); i += kThreads) {
            const int r = i / (DIM / 8), ch = i - r * (DIM / 8);
            float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (r < count) {
                const int rr = first + r, tok = rr / p.group;
                const int64_t off = (c.starts == nullptr ? seq * p.q_seq + tok * p.q_row : (own.x + tok) * p.q_row) + (head * p.group + rr - tok * p.group) * p.q_head + ch * 8;
                if (PIECES == 3) load8(static_cast<const float*>(p.q) + off, p.q_vec, x);
                else if (PIECES == 2) load8(static_cast<const __half*>(p.q) + off, p.q_vec, x);
                else load8(static_cast<const __nv_bfloat16*>(p.q) + off, p.q_vec, x);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] *= sign;
#pragma unroll
            for (int k = 0; k < PIECES; ++k) {
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (k + 1 < PIECES) {       // toward zero, so that no finite value becomes infinite
                        w[e] = __byte_perm(__float_as_uint(x[2 * e]), __float_as_uint(x[2 * e + 1]), 0x7632);
                        x[2 * e] -= bf16_lo(w[e]);
                        x[2 * e + 1] -= bf16_hi(w[e]);
                    } else {
                        w[e] = pack_bf16(x[2 * e], x[2 * e + 1]);
                    }
                }
                *reinterpret_cast<uint4*>(q_sm + (k * Shape::parts + (ch >> 3)) * kPart + r * 128 + (((ch & 7) ^ (r & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
        fence_async_proxy();
        __syncthreads();

        if (warp == 4) {
            if (lane == 0) {
                const uint8_t* from = tiles + ((int64_t)seq * c.heads + head) * tiles_per_seq * tile_bytes(DIM);
                for (int i = 0; i < n; ++i) {
                    const uint32_t it = it0 + i;
                    const uint8_t* src = from + (int64_t)(tt.start(j_lo + i) / kTile) * tile_bytes(DIM);
                    if (it > 0 && !bar_wait(bar(kKEmpty), (it - 1) & 1)) { failed = 1u; break; }
                    bar_expect(bar(kKFull), Shape::side + kTrailer);
                    bulk_load(k_at, src, Shape::side, bar(kKFull));
                    bulk_load(tail_at + (it & 3) * kTrailer, src + 2 * Shape::side, kTrailer, bar(kKFull));
                    if (it > 0 && !bar_wait(bar(kVEmpty), (it - 1) & 1)) { failed = 1u; break; }
                    bar_expect(bar(kVFull), Shape::side);
                    bulk_load(v_at, src + Shape::side, Shape::side, bar(kVFull));
                }
            }
            __syncwarp();
        } else if (warp == 5) {
            if (lane == 0) {
                constexpr uint32_t score_desc = product_descriptor(128, false), value_desc = product_descriptor(DIM, true);
                auto scores = [&](int i) -> bool {
                    const uint32_t it = it0 + i;
                    if (!bar_wait(bar(kKFull), it & 1)) return false;
                    // the columns are free when the product that read the weights in them is done (the segment before is done)
                    if (i >= NS && !bar_wait(bar(kValues), (it - NS) & 1)) return false;
                    tmem_fence_after();
#pragma unroll
                    for (int k = 0; k < PIECES; ++k)
#pragma unroll
                        for (int s = 0; s < DIM / 16; ++s)
                            mma_ss(tmem + (NS == 2 ? (it & 1) * 128 : 0), tile_descriptor(q_at + (k * Shape::parts + (s >> 2)) * kPart + (s & 3) * 32, 16),
                                   tile_descriptor(k_at + (s >> 2) * kPart + (s & 3) * 32, 16), score_desc, k + s > 0);
                    mma_commit(bar(NS == 2 && (it & 1) ? kScores2 : kScores));
                    mma_commit(bar(kKEmpty));
                    return true;
                };
                bool ok = n == 0 || scores(0);
                for (int i = 0; ok && i < n; ++i) {
                    const uint32_t it = it0 + i;
                    if (NS == 2 && i + 1 < n && !(ok = scores(i + 1))) break;
                    const uint32_t turn = NS == 2 ? it & 1 : 0;
                    if (!(ok = bar_wait(bar(turn ? kWeights2 : kWeights), NS == 2 ? (it >> 1) & 1 : it & 1))) break;
                    if (!(ok = bar_wait(bar(kVFull), it & 1))) break;
                    tmem_fence_after();
#pragma unroll
                    for (int k = 0; k < PIECES; ++k) {
                        const uint32_t w = tmem + (k < 2 ? turn * 128 + k * 64 : Shape::more + turn * 64);
#pragma unroll
                        for (int s = 0; s < 8; ++s)
                            mma_ts(tmem + Shape::sums, w + s * 8, tile_descriptor(v_at + s * 2048, kPart), value_desc, i > 0 || k + s > 0);
                    }
                    mma_commit(bar(kValues));
                    mma_commit(bar(kVEmpty));
                    if (NS == 1 && i + 1 < n) ok = scores(i + 1);
                }
                if (!ok) failed = 1u;
            }
            __syncwarp();
        } else {
            const int r = threadIdx.x;                            // this thread's row
            const uint32_t mine = tmem + ((uint32_t)(warp * 32) << 16);
            const int pos = r < count ? pos0 + (first + r) / p.group : -1;
            float m = -INFINITY, l = 0.f;
            uint32_t poison = 0u;
            bool ok = true;
            for (int i = 0; i < n; ++i) {
                const uint32_t it = it0 + i, turn = NS == 2 ? it & 1 : 0, set = turn * 128;
                ok = bar_wait(bar(turn ? kScores2 : kScores), NS == 2 ? (it >> 1) & 1 : it & 1);
                if (!__all_sync(0xFFFFFFFFu, ok)) { ok = false; break; }
                tmem_fence_after();
                const uint32_t* tail = reinterpret_cast<const uint32_t*>(tails + (it & 3) * kTrailer);
                const int t0 = tt.start(j_lo + i);
                const uint4 there = *reinterpret_cast<const uint4*>(tail);
                const bool whole = (there.x & there.y & there.z & there.w) == 0xFFFFFFFFu && t0 + kTile - 1 <= low_pos && (p.window <= 0 || t0 > high_pos - p.window);
                const int upto = pos - t0, from = p.window > 0 ? pos - p.window - t0 : -1, sinks = p.sinks - t0;
                uint32_t s[64];                                   // half of the row's scores
                auto load = [&](int half) {
                    tmem_load32(mine + set + 64 * half, s);
                    tmem_load32(mine + set + 64 * half + 32, s + 32);
                    tmem_wait_load();
                    if (!whole) {
#pragma unroll
                        for (int k = 0; k < 64; ++k) {
                            const int col = 64 * half + k;
                            const uint32_t word = half == 0 ? (k < 32 ? there.x : there.y) : (k < 32 ? there.z : there.w);
                            const bool on = col <= upto && (col > from || col < sinks) && ((word >> (k & 31)) & 1u);
                            s[k] = on ? s[k] : 0xFF800000u;
                        }
                    }
                };
                if (tail[4]) {                                    // V holds blocks that are NaN
                    for (int k = 0; k < kTile; ++k) {
                        const uint32_t blocks = reinterpret_cast<const uint8_t*>(tail)[32 + k];
                        if (blocks && sees(p, pos, t0 + k)) poison |= blocks;
                    }
                }
                float top = -INFINITY, top2 = -INFINITY;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    load(half);
#pragma unroll
                    for (int k = 0; k < 64; k += 2) {
                        top = fmaxf(top, __uint_as_float(s[k]));
                        top2 = fmaxf(top2, __uint_as_float(s[k + 1]));
                    }
                }
                top = fmaxf(top, top2) * mul;
                if (__any_sync(0xFFFFFFFFu, top > m + 8.f)) {
                    const float next = fmaxf(m, top), fade = next == -INFINITY ? 1.f : exp2_fast(m - next);
                    m = next;
                    l *= fade;
                    if (i > 0) {
                        ok = bar_wait(bar(kValues), (it - 1) & 1);
                        if (!__all_sync(0xFFFFFFFFu, ok)) { ok = false; break; }
                        tmem_fence_after();
#pragma unroll
                        for (int b = 0; b < DIM; b += 32) {
                            uint32_t o[32];
                            tmem_load32(mine + Shape::sums + b, o);
                            tmem_wait_load();
#pragma unroll
                            for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * fade);
                            tmem_store32(mine + Shape::sums + b, o);
                        }
                    }
                }
                const float base = m == -INFINITY ? 0.f : m;
                // the first half's weights lie over its scores; its second pieces over the second half's scores, once these are read
                uint32_t w2[2][32];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    load(half);
                    if (PIECES > 1 && half == 1) tmem_store32(mine + set + 64, w2[0]);
                    uint32_t w[32], w3[32];
                    float sum = 0.f, sum2 = 0.f;
#pragma unroll
                    for (int e = 0; e < 64; e += 2) {
                        float a = exp2_fast(fmaf(__uint_as_float(s[e]), mul, -base)), b = exp2_fast(fmaf(__uint_as_float(s[e + 1]), mul, -base));
                        sum += a;
                        sum2 += b;
                        w[e >> 1] = pack_bf16(a, b);
                        if (PIECES > 1) {
                            a -= bf16_lo(w[e >> 1]);
                            b -= bf16_hi(w[e >> 1]);
                            w2[half][e >> 1] = pack_bf16(a, b);
                        }
                        if (PIECES > 2) w3[e >> 1] = pack_bf16(a - bf16_lo(w2[half][e >> 1]), b - bf16_hi(w2[half][e >> 1]));
                    }
                    l += sum + sum2;
                    tmem_store32(mine + set + 32 * half, w);
                    if (PIECES > 1 && half == 1) tmem_store32(mine + set + 96, w2[1]);
                    if (PIECES > 2) tmem_store32(mine + Shape::more + turn * 64 + 32 * half, w3);
                }
                tmem_wait_store();
                tmem_fence_before();
                bar_arrive(bar(turn ? kWeights2 : kWeights));
            }
            if (ok && n > 0) ok = bar_wait(bar(kValues), (it0 + n - 1) & 1);
            if (!__all_sync(0xFFFFFFFFu, ok)) { ok = false; failed = 1u; }
            tmem_fence_after();
            // ---- the row's result, or its share
            const int rr = first + r, tok = rr / p.group;
            const int64_t out_row = ((int64_t)(own.x + tok) * p.q_heads + head * p.group + rr - tok * p.group) * DIM;
            const int share = 2 * blockIdx.x + (begins ? 0 : 1);
            const float times = !ok ? __uint_as_float(0x7FC00000u) : finished ? (l == 0.f ? 0.f : __frcp_rn(l)) : 1.f;
#pragma unroll
            for (int b = 0; b < DIM; b += 32) {
                uint32_t o[32];
                if (n > 0) {
                    tmem_load32(mine + Shape::sums + b, o);
                    tmem_wait_load();
                }
                if (r < count) {
                    const bool bad = (poison >> (b >> 5)) & 1u;
#pragma unroll
                    for (int k = 0; k < 32; k += 8) {
                        float v[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] = bad ? __uint_as_float(0x7FC00000u) : (n > 0 ? __uint_as_float(o[k + e]) : 0.f) * times;
                        if (!finished) store8(p.partial + ((int64_t)share * kTile + r) * DIM + b + k, v);
                        else if (p.out_vec) {
                            if (PIECES == 3) store8(static_cast<float*>(p.out) + out_row + b + k, v);
                            else if (PIECES == 2) store8(static_cast<__half*>(p.out) + out_row + b + k, v);
                            else store8(static_cast<__nv_bfloat16*>(p.out) + out_row + b + k, v);
                        } else {
#pragma unroll
                            for (int e = 0; e < 8; ++e) store_value(p.out, p.dtype, out_row + b + k + e, v[e]);
                        }
                    }
                }
            }
            if (!finished && r < count) {
                p.stats[(share * kTile + r) * 2] = m;
                p.stats[(share * kTile + r) * 2 + 1] = l;
            }
            tmem_fence_before();
        }
        __syncthreads();
        tmem_fence_after();
        if (failed) break;
        it0 += n;
        left -= take;
        begins = false;
        if (left > 0) at.next_tile<kTile>(p);
    }
    if (failed && warp == 4 && lane == 0) {                       // copies on the way write to this CTA's memory
        bar_wait(bar(kKFull), 0); bar_wait(bar(kKFull), 1);
        bar_wait(bar(kVFull), 0); bar_wait(bar(kVFull), 1);
    }
    __syncthreads();
    if (warp == 5) tmem_free(tmem, Shape::columns);
}

template <int DIM, int PIECES, int NS>
int launch(AttentionParams p, const ChunkPlan& pl, uint8_t* tiles, cudaStream_t st) {
    using Shape = ChunkShape<DIM, PIECES, NS>;
    auto kern = mx_attention_chunk_kernel<DIM, PIECES, NS>;
    static std::atomic<int> resident[64];                         // CTAs of this kernel on an SM, by device; 0: not asked yet
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) { set_error("mx_attention: no device"); return MPT_ERR_CUDA; }
    int fit = resident[dev].load(std::memory_order_relaxed);
    if (fit == 0) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::smem) != cudaSuccess ||
            cudaOccupancyMaxActiveBlocksPerMultiprocessor(&fit, kern, kThreads, Shape::smem) != cudaSuccess || fit < 1) {
            check_launch("mx_attention");
            set_error("mx_attention: the kernel does not fit this device");
            return MPT_ERR_CUDA;
        }
        fit = fit * Shape::columns > 512 ? 512 / Shape::columns : fit;      // tensor memory: 512 columns an SM
        resident[dev].store(fit, std::memory_order_relaxed);
    }
    p.runs = pl.runs < fit * sm_count() ? pl.runs : fit * sm_count();
    kern<<<(unsigned)p.runs, kThreads, Shape::smem, st>>>(p, tiles, pl.tiles_per_seq);
    if (p.runs > 1) mx_attention_join_kernel<kTile><<<(unsigned)(p.runs - 1), 128, 0, st>>>(p);
    return check_launch("mx_attention");
}

template <int DIM>
int launch(const AttentionParams& p, const ChunkPlan& pl, uint8_t* tiles, cudaStream_t st) {
    if (p.dtype == MPT_DTYPE_BF16) {
        if constexpr (DIM <= 128) return launch<DIM, 1, 1>(p, pl, tiles, st);
        else return launch<DIM, 1, 2>(p, pl, tiles, st);
    }
    if (p.dtype == MPT_DTYPE_F16) {
        if constexpr (DIM <= 192) return launch<DIM, 2, 2>(p, pl, tiles, st);
    } else {
        if constexpr (DIM <= 128) return launch<DIM, 3, 2>(p, pl, tiles, st);
    }
    set_error("mx_attention: no chunk kernel for this size");
    return MPT_ERR_INVALID_ARGUMENT;
}

}  // namespace

bool chunk_kernel_exists(int dim, int dtype) {
    if (dim != 32 && dim != 64 && dim != 96 && dim != 128 && dim != 192 && dim != 256) return false;
    return dim <= (dtype == MPT_DTYPE_BF16 ? 256 : dtype == MPT_DTYPE_F16 ? 192 : 128);
}

ChunkPlan chunk_plan(const CacheView& c, int q_heads) {
    ChunkPlan pl;
    const int group = q_heads / c.heads;
    const int64_t tokens = (int64_t)c.width << c.page_shift;
    pl.tiles_per_seq = (int)((tokens + kTile - 1) / kTile);
    pl.tile_bytes = (size_t)c.seqs * c.heads * pl.tiles_per_seq * tile_bytes(c.dim);
    const int64_t row_tiles = c.rows * group / kTile + c.seqs, want = row_tiles * c.heads * (pl.tiles_per_seq + 1), most = 2 * (int64_t)sm_count();
    pl.runs = (int)(want < 1 ? 1 : want > most ? most : want);
    pl.partial_floats = (size_t)2 * pl.runs * kTile * c.dim;
    pl.stats_floats = (size_t)2 * pl.runs * kTile * 2;
    return pl;
}

int launch_chunk(AttentionParams p, const ChunkPlan& pl, uint8_t* tiles, bool fp4, cudaStream_t st) {
    p.tile_rows = kTile;
    p.least = 1;
    if (pl.tiles_per_seq > 0 && p.c.seqs > 0) {
        const dim3 grid((unsigned)pl.tiles_per_seq, (unsigned)p.c.heads, (unsigned)(p.c.seqs < 65535 ? p.c.seqs : 65535));
        (fp4 ? mx_expand_kernel<true> : mx_expand_kernel<false>)<<<grid, 256, 0, st>>>(p, tiles, pl.tiles_per_seq);
    }
    switch (p.c.dim) {
        case 32: return launch<32>(p, pl, tiles, st);
        case 64: return launch<64>(p, pl, tiles, st);
        case 96: return launch<96>(p, pl, tiles, st);
        case 128: return launch<128>(p, pl, tiles, st);
        case 192: return launch<192>(p, pl, tiles, st);
        case 256: return launch<256>(p, pl, tiles, st);
    }
    set_error("mx_attention: no chunk kernel for head_dim %d", p.c.dim);
    return MPT_ERR_INVALID_ARGUMENT;
}

}  // namespace mpt
