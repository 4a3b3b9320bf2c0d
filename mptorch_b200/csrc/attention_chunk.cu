// Attention of chunks of new rows over a paged MX cache: 128 rows of q at a time on the tcgen05 tensor cores.
//
// Bound: the tensor cores, 4 dim operations for each pair of a row and a visible token, and beside them the exponentials (16 a
// clock on an SM).  Two kernels.  The first expands the sequences' K and V into bfloat16, where a code times its scale is exact, as
// tiles of 128 tokens in the very layout that the second one's operands have in shared memory, so that a tile is one bulk copy: it
// costs one pass over the cache (a byte read and two written an element), where expanding inside the second kernel would repeat it
// for every 128 rows.  The second is a warp that copies, a warp that issues products, and eight warps with half a row a thread:
//   S = Q K^T (tensor memory) -> p = exp(s - m) as bfloat16 over S's own columns -> O += P V, P read from tensor memory.
// m is moved, and O multiplied, only when a row's maximum has grown by more than 2^8 over it; p is at most 2^8 then.
//
// Accuracy.  bfloat16 queries are one operand; float16 and float32 ones are the sum of two and three bfloat16 pieces (16 and 24
// bits), and so are their weights p; sums are fp32 throughout, and short ones where three pieces are worth it (kFold).  With
// bfloat16 weights the 1024-token chunks below are 2.2e-3 off, where fp32 arithmetic that is rounded to bfloat16 once is 1.7e-3 off; a
// second piece of the weights would be half as many products again.
//
// Measured on a B200: 1024-token chunks of two sequences over 8192, 32 heads on 8 of 128, E4M3, bfloat16 312 us (115.5 for the
// products at the measured rate of bfloat16; 605 TFLOP/s).  The expansion takes 18 us of it and the join of cut tiles some 10; what bounds
// the rest is the chain of a tile, product, softmax, product, two CTAs on an SM hiding each other's.  Six ragged chunks up to 300 over
// 2000, 12 heads of 64, float32: 85 us (2.9), three pieces of q and of p each, and runs of a few tiles.
#include "attention.cuh"
#include "attention_chunk.cuh"
#include "tcgen05.cuh"

namespace mpt {
namespace {

constexpr int kTile = 128, kPart = 128 * 128;                     // tokens and rows of a tile; bytes of 128 rows of 64 values
// Three pieces: the tensor cores cut their sums off instead of rounding them, an error that grows with the context.  After every fourth
// tile the sums are added to fp32 sums in registers and begun again.  384 rows over 3438, head_dim 128: 2.9e-6 of the result without,
// 1.3e-6 with every eighth, 8e-7 with every fourth (fp32 arithmetic as torch has it 1.6e-6), all of them in 220 us.
constexpr int kFold = 4;
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

constexpr float kMostBf16 = 0x1.FEp127f;

__device__ __forceinline__ uint32_t below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u; }   // the lowest n bits
// ---- expanding.  One CTA for 128 tokens of a (sequence, kv head).
template <bool FP4>
__global__ void __launch_bounds__(256) mx_expand_kernel(const AttentionParams p, uint8_t* __restrict__ tiles, int tiles_per_seq) {
    next_may_start();
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
        // a thread keeps its piece of eight values and goes through the tokens
        const int pieces = c.dim >> 3, row_bytes = FP4 ? c.dim >> 1 : c.dim, step = 256 / pieces, ch = threadIdx.x % pieces, first = threadIdx.x / pieces;
        const int side_bytes = parts_for(c.dim) * kPart;
        if (first < step) {
#pragma unroll 2
            for (int tok = first; tok < kTile; tok += step) {
                const int64_t row = row_at[tok];
                const int64_t at = max(row, (int64_t)0);
                const uint8_t *kf = c.k_codes + at * row_bytes + (FP4 ? ch * 4 : ch * 8), *vf = c.v_codes + at * row_bytes + (FP4 ? ch * 4 : ch * 8);
                uint2 kw = make_uint2(0u, 0u), vw = kw;
                uint32_t ks = 0u, vs = 0u;
                if (row >= 0) {
                    if (FP4) {
                        kw.x = __ldg(reinterpret_cast<const uint32_t*>(kf));
                        vw.x = __ldg(reinterpret_cast<const uint32_t*>(vf));
                    } else {
                        kw = __ldg(reinterpret_cast<const uint2*>(kf));
                        vw = __ldg(reinterpret_cast<const uint2*>(vf));
                    }
                    ks = __ldg(c.k_scales + at * nb + (ch >> 2));
                    vs = __ldg(c.v_scales + at * nb + (ch >> 2));
                }
                uint8_t* to = out + (ch >> 3) * kPart + tok * 128 + (((ch & 7) ^ (tok & 7)) << 4);
                auto put = [&](uint2 w, float s, bool bound, uint8_t* to) {
                    float x[8];
                    decode8<FP4>(w, x);
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] *= s;
                    if (bound) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[e] = fminf(fmaxf(x[e], -kMostBf16), kMostBf16);
                    }
                    uint4 v;
                    v.x = pack_bf16(x[0], x[1]); v.y = pack_bf16(x[2], x[3]);
                    v.z = pack_bf16(x[4], x[5]); v.w = pack_bf16(x[6], x[7]);
                    *reinterpret_cast<uint4*>(to) = v;
                };
                put(kw, e8m0_value(ks), false, to);
                // a block of V that is NaN takes no part in the product; its rows are told at the end
                if (vs == 255u) vw = make_uint2(0u, 0u);
                // (a code of 2^8 or 2^2 with a scale this large passes fp32's range; an infinity would reach rows that do not see the token)
                put(vw, vs == 255u ? 0.f : e8m0_value(vs), vs >= 247u, to + side_bytes);
            }
        }
        uint32_t* tail = reinterpret_cast<uint32_t*>(out + 2 * parts_for(c.dim) * kPart);
        if (threadIdx.x < 4) tail[threadIdx.x] = there[threadIdx.x];
        if (threadIdx.x == 4) tail[4] = any_nan;
        if (threadIdx.x < kTile) reinterpret_cast<uint8_t*>(tail)[32 + threadIdx.x] = nan_blocks[threadIdx.x];
    }
}

// ---- attention
constexpr int kRowThreads = 256, kThreads = kRowThreads + 64;     // two threads a row, each with half of the tokens; a warp that copies, one that issues products
enum { kKFull, kKEmpty, kVFull, kVEmpty, kScores, kScores2, kWeights, kWeights2, kValues, kValues2, kLast, kBars };

template <int DIM, int PIECES, int NS>
struct ChunkShape {
    static constexpr int parts = parts_for(DIM), q_bytes = PIECES * parts * kPart, side = parts * kPart;
    static constexpr int smem = 1024 + q_bytes + 2 * side + 4 * kTrailer;
    // columns of tensor memory: scores (a set for each of NS), sums, and for three pieces sums of the smaller ones (so that the tensor
    // cores, which cut sums off, do so with the large sums once a product and not three times) and weights that do not fit over the scores
    static constexpr int sums = NS * 128, small = sums + DIM, more = small + (PIECES == 3 ? DIM : 0), used = more + (PIECES == 3 ? 64 * NS : 0);
    static constexpr int columns = used <= 256 ? 256 : 512;
    static_assert(used <= 512, "tensor memory");
    static_assert(smem <= 227 * 1024, "shared memory");
};

template <int DIM, int PIECES, int NS>
__global__ void __launch_bounds__(kThreads, NS == 1 && PIECES == 1 ? 2 : 1) mx_attention_chunk_kernel(const AttentionParams p, const uint8_t* __restrict__ tiles, int tiles_per_seq) {
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
    __shared__ float tops[2][2][kTile], sums_sm[kTile];           // of alternate pieces: with two sets of scores one warp may be a piece ahead

    next_may_start();
    zero_outside(p);
    RunOf<kTile> run(p, place_sm);
    if (run.left <= 0) {
        run.end(p);
        wait_for_previous();                                      // no CTA is done before the kernel that this one follows
        return;
    }

    auto bar = [&](int i) { return smem_at(&bars[i]); };
    auto wait = [&](int i, uint32_t parity) { return bar_wait(bar(i), parity & 1u, &failed); };
    // A wait for a phase is only sound where the phase before it is known to be over.  With two sets of scores a row's weights may be
    // ready while the product with the piece before is under way, so each set has barriers of its own.
    auto values_bar = [&](uint32_t it) { return NS == 2 && (it & 1) ? kValues2 : kValues; };
    auto wait_values = [&](uint32_t it) { return wait(values_bar(it), NS == 2 ? it >> 1 : it); };
    if (threadIdx.x == 0) {
        for (int i = 0; i < kBars; ++i) bar_init(bar(i), i == kWeights || i == kWeights2 ? kRowThreads : 1);
        failed = p.fail_at == 0;
        fence_barrier_init();
    }
    if (warp == 9) tmem_alloc(smem_at(&tmem_slot), Shape::columns);
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = tmem_slot;

    const float sign = p.scale_log2 > 0.f ? 1.f : p.scale_log2 < 0.f ? -1.f : 0.f;      // of q, so that the largest score is of the largest sum
    const float mul = p.scale_log2 == 0.f ? 1.f : fabsf(p.scale_log2);
    uint32_t it0 = 0, k_copies = 0, v_copies = 0;                 // pieces before this segment; copies begun (by the thread that copies)
    for (int segment = 0; run.left > 0; ++segment) {
        // Once a wait has run out nothing more is computed: all that is left of the run gives NaN, whole row tiles and shares alike.  (Read
        // between two barriers: no wait is under way here.)
        const bool dead = *(volatile uint32_t*)&failed != 0u;
        const int seq = run.at.seq, head = run.at.head, pieces = run.at.w.pieces(run.at.tile), take = run.take(p, pieces);
        if (take == 0) break;
        const int2 own = rows_of(c, seq);
        const int first = run.at.tile * kTile, count = min(kTile, own.y * p.group - first);
        const int pos0 = __ldg(c.lens + seq) - own.y;
        const int low_pos = pos0 + first / p.group, high_pos = pos0 + (first + count - 1) / p.group;
        const TokenTiles<kTile> tt(p, low_pos, high_pos);
        const bool finished = take == pieces;
        const int j_lo = min(run.at.piece, tt.tiles), n = dead ? 0 : min(run.at.piece + take, tt.tiles) - j_lo;

        // ---- q, in pieces
#pragma unroll 1
        for (int i = dead ? kTile * (DIM / 8) : threadIdx.x; i < kTile * (DIM / 8); i += kThreads) {
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
            for (int e = 0; e < 8; ++e) x[e] = fabsf(x[e]) < INFINITY ? x[e] * sign : __uint_as_float(0x7FC00000u);      // (an infinity: the row is NaN)
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

        if (warp == 8) {
            if (lane == 0) {
                if (run.begins) wait_for_previous();                  // the expanded tiles
                const uint8_t* from = tiles + ((int64_t)seq * c.heads + head) * tiles_per_seq * tile_bytes(DIM);
                for (int i = 0; i < n; ++i) {
                    const uint32_t it = it0 + i;
                    const uint8_t* src = from + (int64_t)(tt.start(j_lo + i) / kTile) * tile_bytes(DIM);
                    if (it > 0 && !wait(kKEmpty, it - 1)) break;
                    ++k_copies;
                    bar_expect(bar(kKFull), Shape::side + kTrailer);
                    bulk_load(k_at, src, Shape::side, bar(kKFull));
                    bulk_load(tail_at + (it & 3) * kTrailer, src + 2 * Shape::side, kTrailer, bar(kKFull));
                    if (it > 0 && !wait(kVEmpty, it - 1)) break;
                    ++v_copies;
                    bar_expect(bar(kVFull), Shape::side);
                    bulk_load(v_at, src + Shape::side, Shape::side, bar(kVFull));
                }
            }
            __syncwarp();
        } else if (warp == 9) {
            {
                const bool leader = lane == 0;
                const uint32_t tm = uniform(tmem), q_u = uniform(q_at), k_u = uniform(k_at), v_u = uniform(v_at);
                constexpr uint32_t score_desc = product_descriptor(128, false), value_desc = product_descriptor(DIM, true);
                auto scores = [&](int i) -> bool {
                    const uint32_t it = it0 + i;
                    if (!__all_sync(0xFFFFFFFFu, wait(kKFull, it))) return false;
                    // the columns are free when the product that read the weights in them is done (the segment before is done)
                    if (i >= NS && !__all_sync(0xFFFFFFFFu, wait_values(it - NS))) return false;
                    tmem_fence_after();
                    const uint64_t q_desc = tile_descriptor(q_u, 16), k_desc = tile_descriptor(k_u, 16);
                    const uint32_t to = tm + (NS == 2 ? (it & 1) * 128 : 0);
#pragma unroll
                    for (int k = PIECES - 1; k >= 0; --k)             // the smallest first, while the sums are small
#pragma unroll
                        for (int s = 0; s < DIM / 16; ++s)
                            mma_ss(to, q_desc + (((k * Shape::parts + (s >> 2)) * kPart + (s & 3) * 32) >> 4), k_desc + (((s >> 2) * kPart + (s & 3) * 32) >> 4), score_desc,
                                   k < PIECES - 1 || s > 0, leader);
                    mma_commit(bar(NS == 2 && (it & 1) ? kScores2 : kScores), leader);
                    mma_commit(bar(kKEmpty), leader);
                    return true;
                };
                bool ok = n == 0 || scores(0);
                for (int i = 0; ok && i < n; ++i) {
                    const uint32_t it = it0 + i;
                    if (NS == 2 && i + 1 < n && !(ok = scores(i + 1))) break;
                    const uint32_t turn = NS == 2 ? it & 1 : 0;
                    if (!(ok = __all_sync(0xFFFFFFFFu, wait(kVFull, it)))) break;
                    if (!(ok = __all_sync(0xFFFFFFFFu, wait(turn ? kWeights2 : kWeights, NS == 2 ? it >> 1 : it)))) break;
                    tmem_fence_after();
                    const uint64_t v_desc = tile_descriptor(v_u, kPart);
#pragma unroll
                    for (int k = 0; k < PIECES; ++k) {
                        const uint32_t w = tm + (k < 2 ? turn * 128 + k * 64 : Shape::more + turn * 64);
#pragma unroll
                        for (int s = 0; s < 8; ++s)
                            mma_ts(tm + (PIECES == 3 && k > 0 ? Shape::small : Shape::sums), w + s * 8, v_desc + (s * 2048 >> 4), value_desc,
                                   (PIECES == 3 ? i % kFold > 0 : i > 0) || s > 0 || k > (PIECES == 3 ? 1 : 0), leader);
                    }
                    mma_commit(bar(values_bar(it)), leader);
                    mma_commit(bar(kVEmpty), leader);
                    if (NS == 1 && i + 1 < n) ok = scores(i + 1);
                }
            }
            __syncwarp();
        } else {
            const int half = warp >> 2, r = threadIdx.x & (kTile - 1);   // this thread's row, and its half of the tokens
            auto pair_sync = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp & 3)) : "memory"); };      // the two warps of the same rows
            const uint32_t mine = tmem + ((uint32_t)((warp & 3) * 32) << 16);
            const int pos = r < count ? pos0 + (first + r) / p.group : -1;
            float m = -INFINITY, l = 0.f;
            uint32_t poison = 0u;
            constexpr int kTotal = PIECES == 3 ? DIM / 32 : 1;    // blocks of 16 columns, which the halves take in turn
            float total[kTotal][16] = {};
            for (int i = 0; i < n; ++i) {
                const uint32_t it = it0 + i, turn = NS == 2 ? it & 1 : 0, set = turn * 128;
                if (PIECES == 3 && i > 0 && i % kFold == 0) {
                    wait_values(it - 1);
                    __syncwarp();
                    tmem_fence_after();
#pragma unroll
                    for (int j = 0; j < kTotal; ++j) {
                        uint32_t o[16], o2[16];
                        tmem_load16(mine + Shape::sums + 16 * half + 32 * j, o);
                        tmem_load16(mine + Shape::small + 16 * half + 32 * j, o2);
                        tmem_wait_load();
#pragma unroll
                        for (int k = 0; k < 16; ++k) total[j][k] += __uint_as_float(o[k]) + __uint_as_float(o2[k]);
                    }
                }
                wait(turn ? kScores2 : kScores, NS == 2 ? it >> 1 : it);
                __syncwarp();
                tmem_fence_after();
                uint32_t s[64];
                tmem_load32(mine + set + 64 * half, s);
                tmem_load32(mine + set + 64 * half + 32, s + 32);
                const uint32_t* tail = reinterpret_cast<const uint32_t*>(tails + (it & 3) * kTrailer);
                const int t0 = tt.start(j_lo + i);
                const uint4 there = *reinterpret_cast<const uint4*>(tail);
                const uint32_t any_nan = tail[4];
                const bool whole = (there.x & there.y & there.z & there.w) == 0xFFFFFFFFu && t0 + kTile - 1 <= low_pos && (p.window <= 0 || t0 > high_pos - p.window);
                tmem_wait_load();
                if (!whole) {
                    const int t1 = t0 + 64 * half, from = p.window > 0 ? pos - p.window + 1 - t1 : 0, sinks = p.window > 0 ? p.sinks - t1 : 0;
                    uint32_t seen[2];
#pragma unroll
                    for (int w = 0; w < 2; ++w)
                        seen[w] = (half ? (w ? there.w : there.z) : (w ? there.y : there.x)) & below(pos + 1 - t1 - 32 * w) &
                                  (~below(from - 32 * w) | below(sinks - 32 * w));
#pragma unroll
                    for (int k = 0; k < 64; ++k) s[k] = (seen[k >> 5] >> (k & 31)) & 1u ? s[k] : 0xFF800000u;
                }
                if (any_nan) {                                    // V holds blocks that are NaN
                    for (int k = 0; k < kTile; ++k) {
                        const uint32_t blocks = reinterpret_cast<const uint8_t*>(tail)[32 + k];
                        if (blocks && sees(p, pos, t0 + k)) poison |= blocks;
                    }
                }
                float top = -INFINITY, top2 = -INFINITY;
#pragma unroll
                for (int k = 0; k < 64; k += 2) {
                    top = fmaxf(top, __uint_as_float(s[k]));
                    top2 = fmaxf(top2, __uint_as_float(s[k + 1]));
                }
                top = fmaxf(top, top2);
                // the other half's; from here on the scores' columns are free
                tops[it & 1][half][r] = top;
                tmem_fence_before();
                pair_sync();
                tmem_fence_after();
                top = fmaxf(top, tops[it & 1][half ^ 1][r]) * mul;
                if (__any_sync(0xFFFFFFFFu, top > m + 8.f)) {
                    const float next = fmaxf(m, top), fade = next == -INFINITY ? 1.f : exp2_fast(m - next);
                    m = next;
                    l *= fade;
                    if (PIECES == 3) {
#pragma unroll
                        for (int j = 0; j < kTotal; ++j)
#pragma unroll
                            for (int k = 0; k < 16; ++k) total[j][k] *= fade;
                    }
                    if (PIECES == 3 ? i % kFold > 0 : i > 0) {
                        wait_values(it - 1);
                        __syncwarp();
                        tmem_fence_after();
                        // the halves take blocks of 16 columns in turn; few registers are free here
                        for (int b = 16 * half; b < DIM; b += 32) {
                            uint32_t o[16];
#pragma unroll
                            for (int side = 0; side < (PIECES == 3 ? 2 : 1); ++side) {
                                const uint32_t where = mine + (side ? Shape::small : Shape::sums) + b;
                                tmem_load16(where, o);
                                tmem_wait_load();
#pragma unroll
                                for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * fade);
                                tmem_store16(where, o);
                            }
                        }
                    }
                }
                const float base = m == -INFINITY ? 0.f : m;
                float sum = 0.f, sum2 = 0.f;
#pragma unroll
                for (int k = 0; k < 64; k += 32) {
                    uint32_t w[16], w2[16], w3[16];
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        float a = exp2_fast(fmaf(__uint_as_float(s[k + e]), mul, -base)), b = exp2_fast(fmaf(__uint_as_float(s[k + e + 1]), mul, -base));
                        sum += a;
                        sum2 += b;
                        w[e >> 1] = pack_bf16(a, b);
                        if (PIECES > 1) {
                            a -= bf16_lo(w[e >> 1]);
                            b -= bf16_hi(w[e >> 1]);
                            w2[e >> 1] = pack_bf16(a, b);
                        }
                        if (PIECES > 2) w3[e >> 1] = pack_bf16(a - bf16_lo(w2[e >> 1]), b - bf16_hi(w2[e >> 1]));
                    }
                    const uint32_t to = mine + 32 * half + (k >> 1);
                    tmem_store16(to + set, w);
                    if (PIECES > 1) tmem_store16(to + set + 64, w2);
                    if (PIECES > 2) tmem_store16(to + Shape::more + turn * 64, w3);
                }
                l += sum + sum2;
                tmem_wait_store();
                tmem_fence_before();
                bar_arrive(bar(turn ? kWeights2 : kWeights));
            }
            if (n > 0) wait_values(it0 + n - 1);
            if (half) sums_sm[r] = l;
            __syncwarp();
            pair_sync();
            tmem_fence_after();
            if (!half) sums_sm[r] = l += sums_sm[r];
            pair_sync();
            l = sums_sm[r];
            const bool ok = *(volatile uint32_t*)&failed == 0u;
            // ---- the row's result, or its share
            const int rr = first + r, tok = rr / p.group;
            const int64_t out_row = ((int64_t)(own.x + tok) * p.q_heads + head * p.group + rr - tok * p.group) * DIM;
            const int share = 2 * blockIdx.x + (run.begins ? 0 : 1);
            const float times = finished ? (l == 0.f ? 0.f : __frcp_rn(l)) : 1.f;
#pragma unroll(PIECES == 3 ? kTotal : 1)
            for (int b = 16 * half, j = 0; j < DIM / 32; b += 32, ++j) {      // the halves take blocks of 16 columns in turn
                uint32_t o[16];
                tmem_load16(mine + Shape::sums + b, o);
                tmem_wait_load();
                if (PIECES == 3) {
                    uint32_t o2[16];
                    tmem_load16(mine + Shape::small + b, o2);
                    tmem_wait_load();
#pragma unroll
                    for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(total[j][k] + (__uint_as_float(o[k]) + __uint_as_float(o2[k])));
                }
                if (r < count) {
                    const bool bad = (poison >> (b >> 5)) & 1u;
#pragma unroll
                    for (int k = 0; k < 16; k += 8) {
                        float v[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] = bad || !ok ? __uint_as_float(0x7FC00000u) : n > 0 ? __uint_as_float(o[k + e]) * times : 0.f;
                        if (!finished) {
                            store8(p.partial + ((int64_t)share * kTile + r) * DIM + b + k, v);
                        } else if (p.out_vec) {
                            if (PIECES == 3) store8(static_cast<float*>(p.out) + out_row + b + k, v);
                            else if (PIECES == 2) store8(static_cast<__half*>(p.out) + out_row + b + k, v);
                            else store8(static_cast<__nv_bfloat16*>(p.out) + out_row + b + k, v);
                        } else {
#pragma unroll
                            for (int e = 0; e < 8; ++e) store_value(p.out, p.dtype, out_row + b + k + e, v[e]);
                        }
                    }
                }
                __syncwarp();
            }
            if (!finished && !half && r < count) {
                p.stats[(share * kTile + r) * 2] = m;
                p.stats[(share * kTile + r) * 2 + 1] = l;
            }
            tmem_fence_before();
        }
        if (threadIdx.x == 0 && segment + 1 == p.fail_at) failed = 1u;
        __syncthreads();
        tmem_fence_after();
        it0 += n;
        run.advance(p, take, pieces);
    }
    run.end(p);
    if (*(volatile uint32_t*)&failed) {                           // copies and products on the way use this CTA's memory
        __syncthreads();
        if (threadIdx.x == 0) failed = 0u;
        __syncthreads();
        if (warp == 8 && lane == 0) {
            if (k_copies) wait(kKFull, k_copies - 1);
            if (v_copies) wait(kVFull, v_copies - 1);
        } else if (warp == 9) {
            mma_commit(bar(kLast), lane == 0);
            wait(kLast, 0);
        }
    }
    __syncthreads();
    if (warp == 9) tmem_free(tmem, Shape::columns);
}

template <int DIM, int PIECES, int NS>
int launch(AttentionParams p, const ChunkPlan& pl, uint8_t* tiles, cudaStream_t st) {
    using Shape = ChunkShape<DIM, PIECES, NS>;
    constexpr auto kern = mx_attention_chunk_kernel<DIM, PIECES, NS>;
    // CTAs on an SM, by tensor memory (512 columns), shared memory (3 kB a CTA beside the dynamic part) and registers (launch bounds)
    const int fit = Shape::columns == 256 && 2 * (Shape::smem + 3 * 1024) <= 228 * 1024 && NS == 1 && PIECES == 1 ? 2 : 1;
    if (!allow_shared<kern>(Shape::smem)) return check_launch("mx_attention");
    p.runs = pl.runs < fit * sm_count() ? pl.runs : fit * sm_count();
    p.whole = 0;
    // (without tokens nothing was expanded, and the kernel before this one is none of this call's)
    if (pl.tiles_per_seq > 0) launch_after(kern, dim3((unsigned)p.runs), dim3(kThreads), Shape::smem, st, p, tiles, pl.tiles_per_seq);
    else kern<<<(unsigned)p.runs, kThreads, Shape::smem, st>>>(p, tiles, pl.tiles_per_seq);
    if (p.runs > 1) launch_after(mx_attention_join_kernel, dim3((unsigned)(p.runs - 1), 2), dim3(512), 0, st, p);
    return check_launch("mx_attention");
}

// One set of scores where two CTAs fit an SM (bfloat16 up to 128), two sets where one CTA has the tensor memory for itself.  This choice
// and the other, 1024-token chunks of two sequences over 8192, 16 heads on 8: bfloat16 of 128 198 and 233 us, of 64 151 and 177; float32
// of 64 287 and 308, of 32 253 and 283.
template <int DIM>
int launch(const AttentionParams& p, const ChunkPlan& pl, uint8_t* tiles, cudaStream_t st) {
    if (p.dtype == MPT_DTYPE_BF16) {
        if constexpr (DIM <= 128) return launch<DIM, 1, 1>(p, pl, tiles, st);
        else return launch<DIM, 1, 2>(p, pl, tiles, st);
    }
    if (p.dtype == MPT_DTYPE_F16) {
        if constexpr (DIM <= 192) return launch<DIM, 2, 2>(p, pl, tiles, st);
    } else {
        if constexpr (DIM <= 64) return launch<DIM, 3, 2>(p, pl, tiles, st);
        else if constexpr (DIM <= 128) return launch<DIM, 3, 1>(p, pl, tiles, st);
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
    pl.stats_floats = (size_t)2 * pl.runs * kTile * 2 + (size_t)pl.runs * (sizeof(Cut) / 4);      // and the cuts
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
