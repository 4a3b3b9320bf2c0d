// What the attention kernels share: the call's parameters, how row tiles map to sequences, and which tokens a row sees.
#pragma once
#include "blockcodes.cuh"
#include "launch.cuh"

namespace mpt {

struct AttentionParams {
    CacheView c;
    const void* q;
    int dtype;
    int64_t q_seq, q_row, q_head;      // element strides of q
    bool q_vec, out_vec;               // rows of q, of out, begin at multiples of 16 bytes
    int q_heads, group;                // query heads, query heads of a kv head
    float scale_log2;                  // scale * log2(e)
    int window, sinks;
    void* out;
    int zero_tail;
    int tile_rows;                     // rows of a tile
    int runs, least;                   // CTAs, and pieces of tokens that one takes at least
    int whole;                         // row tiles of at most so many pieces are not cut
    float *partial, *stats;            // of row tiles that two or more CTAs share: sums [slot, row, dim], and {maximum, sum} of each row
    struct Cut* cuts;                  // for each run, the row tile that it has the first but not the last pieces of
    int fail_at;                       // chunks: the part of a run at which a wait is taken to have run out (-1: none; tests alone set it)
};

// A row tile that runs `run` to `last` share: the first one's slot, and two for each of the others, of which they use the first.
struct Cut { int seq, head, tile, slot, last; };           // seq: -1 for none

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

// How the work is shared out.  Row tile t of a sequence has as many pieces of STEP tokens as its last row sees, one at least (so
// that rows that see nothing are written); the pieces of all (sequence, kv head, row tile) in that order are cut into equal
// runs, one for each CTA.  A row tile that lies in one run is finished there; of one that is cut each CTA leaves its sums in a
// slot, which mx_attention_join_kernel joins.  Where there are at least as many row tiles as CTAs, short ones are not cut: an end of
// a run that falls inside of one moves to its beginning.
//
// Without a window row tile t ends at position pos0 + (R (t + 1) - 1) / G (R rows a tile, G query heads a kv head); with
// pos0 = STEP a + b that makes a + 1 + floor((t + 1 + c) / g) pieces, g = STEP G / R, c = floor((b G - 1) / R), and sums of it
// over t are closed.  With a window, with rows before the first token or with more tokens than places every tile counts the same.
struct Work {
    int tiles, base, c, g;                     // of a sequence, for each kv head; g: 0 where all tiles count `base`
    __device__ __forceinline__ int pieces(int t) const { return g ? base + (t + 1 + c) / g : base; }
    __device__ __forceinline__ int64_t upto(int t) const {        // pieces of the tiles before t
        if (g == 0) return (int64_t)t * base;
        return (int64_t)t * base + steps(t + 1 + c) - steps(1 + c);
    }
    __device__ __forceinline__ int64_t steps(int m) const {       // sum of floor(i / g) over i < m
        const int64_t q = m / g;
        return g * (q * (q - 1) / 2) + q * (m - q * g);
    }
};

template <int STEP>
__device__ __forceinline__ Work work_of(const AttentionParams& p, int seq) {
    Work w;
    const int n = rows_of(p.c, seq).y, len = __ldg(p.c.lens + seq), pos0 = len - n, end = min(len, p.c.capacity());
    w.tiles = (int)(((int64_t)n * p.group + p.tile_rows - 1) / p.tile_rows);
    w.c = w.g = 0;
    if (p.window > 0) {
        const int64_t most = ((int64_t)p.sinks + STEP - 1) / STEP + ((int64_t)p.window + p.tile_rows + STEP - 1) / STEP + 1;
        w.base = (int)max(min((int64_t)(end + STEP - 1) / STEP, most), (int64_t)1);
    } else if (pos0 < 0 || len > end) {
        w.base = max((end + STEP - 1) / STEP, 1);
    } else {
        w.base = pos0 / STEP + 1;
        const int bg = pos0 % STEP * p.group;
        w.c = bg ? (bg - 1) / p.tile_rows : -1;
        w.g = STEP * p.group / p.tile_rows;
    }
    return w;
}

// A place in the run of all pieces.
struct Place {
    int seq, head, tile, piece;
    Work w;
    template <int STEP>
    __device__ __forceinline__ void next_tile(const AttentionParams& p) {
        piece = 0;
        if (++tile < w.tiles) return;
        tile = 0;
        if (++head < p.c.heads) return;
        head = 0;
        do { w = work_of<STEP>(p, ++seq); } while (w.tiles == 0);
    }
};

constexpr int kPlaceWords = 16 + (sizeof(Place) + 7) / 8;

// Finds where run `run` begins (`place` means nothing behind the last one); `per`: pieces of a run; returns the number of all
// pieces.  Called by whole blocks of up to 512 threads; `sm` has room for kPlaceWords.
template <int STEP>
__device__ __forceinline__ int64_t find_place(const AttentionParams& p, int run, int64_t& per, Place& place, int64_t* sm) {
    const int each = (p.c.seqs + blockDim.x - 1) / blockDim.x, s0 = min((int)threadIdx.x * each, p.c.seqs), s1 = min(s0 + each, p.c.seqs);
    int64_t mine = 0;
    for (int s = s0; s < s1; ++s) {
        const Work w = work_of<STEP>(p, s);
        mine += w.upto(w.tiles);
    }
    mine *= p.c.heads;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xFFFFFFFFu, upto, o);
        if (lane >= o) upto += v;
    }
    if (lane == 31) sm[warp] = upto;
    __syncthreads();
    int64_t before = 0, total = 0;
    for (int w = 0; w < (int)blockDim.x / 32; ++w) {
        if (w < warp) before += sm[w];
        total += sm[w];
    }
    upto += before;
    per = max((total + p.runs - 1) / p.runs, (int64_t)p.least);
    const int64_t at = run * per;
    Place* out = reinterpret_cast<Place*>(sm + 16);
    if (at >= upto - mine && at < upto) {
        int64_t rest = at - (upto - mine);
        for (int s = s0; s < s1; ++s) {
            const Work w = work_of<STEP>(p, s);
            const int64_t head = w.upto(w.tiles);
            if (rest < head * p.c.heads) {
                out->seq = s;
                if (head * p.c.heads <= 0x7FFFFFFF) {
                    out->head = (int)((uint32_t)rest / (uint32_t)head);
                    rest = (uint32_t)rest % (uint32_t)head;
                } else {
                    out->head = (int)(rest / head);
                    rest %= head;
                }
                int lo = 0, hi = w.tiles - 1;                      // the last tile that begins at or before it
                while (lo < hi) {
                    const int mid = (lo + hi + 1) >> 1;
                    if (w.upto(mid) <= rest) lo = mid; else hi = mid - 1;
                }
                out->tile = lo;
                out->piece = (int)(rest - w.upto(lo));
                out->w = w;
                break;
            }
            rest -= head * p.c.heads;
        }
    }
    __syncthreads();
    place = *out;
    return total;
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

__device__ __forceinline__ float exp2_fast(float x) {       // relative error 2^-22; exact at integers; results below 2^-126 are zero
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// What a CTA has to do of its run: from its beginning, moved as above, as long as take() gives pieces.
template <int STEP>
struct RunOf {
    Place at;
    int64_t left, pos, per;                    // pieces left, number of the piece at `at` among all, pieces of a run
    bool begins = true, told = false;          // the segment stands at the beginning of the run; its cut has been written
    __device__ __forceinline__ RunOf(const AttentionParams& p, int64_t* sm) {
        const int64_t total = find_place<STEP>(p, blockIdx.x, per, at, sm);
        pos = blockIdx.x * per;
        left = min(per, total - pos);
        if (left > 0 && at.piece > 0 && at.w.pieces(at.tile) <= p.whole) {
            left += at.piece;
            pos -= at.piece;
            at.piece = 0;
        }
    }
    // pieces of the row tile at `at`, 0 at the end of the run
    __device__ __forceinline__ int take(const AttentionParams& p, int pieces) const {
        const int rest = pieces - at.piece;
        return left >= rest ? rest : left <= 0 || pieces <= p.whole ? 0 : (int)left;
    }
    __device__ __forceinline__ void advance(const AttentionParams& p, int took, int pieces) {
        if (threadIdx.x == 0 && at.piece == 0 && took < pieces) {
            p.cuts[blockIdx.x] = Cut{at.seq, at.head, at.tile, 2 * (int)blockIdx.x + (begins ? 0 : 1), (int)((pos + pieces - 1) / per)};
            told = true;
        }
        left -= took;
        pos += took;
        begins = false;
        if (left > 0) at.template next_tile<STEP>(p);
    }
    __device__ __forceinline__ void end(const AttentionParams& p) {
        if (threadIdx.x == 0 && !told) p.cuts[blockIdx.x].seq = -1;
    }
};

// Joins the row tiles that are cut: CTAs (x, .) that of which run x has the first pieces.  A warp takes a row.
__global__ void __launch_bounds__(512) mx_attention_join_kernel(const AttentionParams p);

#ifdef MPT_DEFINE_JOIN
__global__ void __launch_bounds__(512) mx_attention_join_kernel(const AttentionParams p) {
    const CacheView& c = p.c;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, dim = c.dim, nb = dim >> 5, run = blockIdx.x;
    wait_for_previous();                                           // whatever follows: this kernel is not done before the one it follows
    const Cut at = p.cuts[run];
    if (at.seq < 0) return;
    const int last = at.last;
    const int2 own = rows_of(c, at.seq);
    const int first = at.tile * p.tile_rows, count = min(p.tile_rows, own.y * p.group - first);
    auto slot_of = [&](int k) { return k == run ? at.slot : 2 * k; };
    const int warps = blockDim.x >> 5;
    for (int r = warp + warps * blockIdx.y; r < count; r += warps * gridDim.y) {
        // 32 parts at a time: a lane has the statistics of one, and the sums follow without waiting for one another
        float top = -INFINITY, sum = 0.f, v[8] = {};
        for (int k0 = run; k0 <= last; k0 += 32) {
            const int k = k0 + lane;
            float2 st = make_float2(-INFINITY, 0.f);
            if (k <= last) st = *reinterpret_cast<const float2*>(p.stats + ((int64_t)slot_of(k) * p.tile_rows + r) * 2);
            float here = fmaxf(top, st.x);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) here = fmaxf(here, __shfl_xor_sync(0xFFFFFFFFu, here, o));
            const float fade = top == -INFINITY ? (sum != sum ? sum : 0.f) : exp2_fast(top - here);
            const float w = st.x == -INFINITY ? (st.y != st.y ? st.y : 0.f) : exp2_fast(st.x - here);       // a NaN sum stays one
            float add = st.y * w;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) add += __shfl_xor_sync(0xFFFFFFFFu, add, o);
            sum = k0 == run ? add : fmaf(sum, fade, add);
            if (k0 != run)
#pragma unroll
                for (int b = 0; b < 8; ++b) v[b] *= fade;
            top = here;
            const int n = min(32, last - k0 + 1);
#pragma unroll 4
            for (int j = 0; j < n; ++j) {
                const float wj = __shfl_sync(0xFFFFFFFFu, w, j);
                const float* from = p.partial + ((int64_t)slot_of(k0 + j) * p.tile_rows + r) * dim + lane;
#pragma unroll
                for (int b = 0; b < 8; ++b)
                    if (b < nb) v[b] = fmaf(from[b * 32], wj, v[b]);
            }
        }
        const int rr = first + r, i = rr / p.group;
        const int64_t out_row = ((int64_t)(own.x + i) * p.q_heads + at.head * p.group + rr - i * p.group) * dim;
        const float inv_sum = sum == 0.f ? 0.f : __frcp_rn(sum);
#pragma unroll
        for (int b = 0; b < 8; ++b)
            if (b < nb) store_value(p.out, p.dtype, out_row + b * 32 + lane, v[b] * inv_sum);
    }
}
#endif

}  // namespace mpt
