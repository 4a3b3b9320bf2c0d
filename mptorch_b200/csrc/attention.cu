// Attention of a few new rows per sequence over a paged MX cache: single tokens, short chunks, grouped heads.
//
// Bound: HBM, the codes and scales of the visible tokens (one byte and 1/32, or half of that, an element of K and of V).  A CTA
// takes one kv head of one sequence, up to 16 columns (rows of q times their pieces) and one part of the visible tokens; its four warps
// take 32 tokens at a time, each with a ring of its own that cp.async fills, so that no warp waits for another until the end.
//
// Mathematics.  With c the element codes and e the block exponents,
//   s[t, r] = sum_b 2^e[t,b] sum_{d in b} c_k[t,d] q[r,d]        o[d, r] = sum_t c_v[t,d] (2^e[t,b(d)] p[t,r])
// Codes are exact in binary16, so both inner sums run on m16n8k16 tensor-core products of codes as they are (one conversion per two
// elements) with fp32 sums: K as the 16 x 16 operand and q^T as the 16 x 8 one, then V^T and p^T.  The scale of K multiplies a
// block's partial sums; the scale of V multiplies p, relative to a reference that moves when a scale is above it or more than 2^14 below
// it; tokens of one piece that are further apart than that are taken in two passes or more, so that neither a large V with a small weight
// nor one that a row does not see takes bits from the others.  q is scaled by a power of two to a largest value in [2^14, 2^15) and held
// as binary16: bfloat16 and float16 in one piece, exact unless a value is 2^-29 of the row's largest or less; float32 in two columns, the
// second 2^11 times what the first leaves (22 bits).  p 2^15 is rounded to binary16 (11 bits) in one piece, for float32 in two.  The
// running maximum is moved only when a tile exceeds it.  The sums of 32 tokens are added up in fp32 registers: the tensor cores cut their running sums off
// instead of rounding them, which after 20000 tokens of float32 had come to 3.9e-6 of the result, 1.5e-5 where V has one sign; now
// 3.8e-7 and 1.4e-7.
//
// Measured on a B200 (the bytes at the measured bandwidth in brackets): one token each over 16 contexts up to 32768, 32 heads on 8 of
// 128, E4M3, bfloat16 136 us (97.9: issue slots 57 % busy, DRAM 58 %; twelve warps an SM do not cover the latency of conversions and products);
// over a window of 1024 with 4 sinks, 96 sequences, 24 heads on 8 of 96, E2M1, float16 62 us (11.8: an element is half a byte, and
// the conversions are twice as many a byte); four sequences up to 1024, 12 heads of 64, float32 18.4 us (0.6: host time, two launches).
#define MPT_DEFINE_JOIN
#include "attention.cuh"
#include "attention_chunk.cuh"

namespace mpt {
namespace {

// kLeast, pieces of 32 tokens that a run has at least: with 8 four sequences of 1024 tokens take 18.4 us, with 16 22.5.
// kWhole, pieces up to which a row tile is not cut where there are as many tiles as CTAs: windows of 1024 take 59.4 us whole and 69.4 cut.
constexpr int kWarps = 4, kTok = 32, kLeast = 8, kWhole = 64;

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(live ? 16 : 0));
}
__device__ __forceinline__ void cp8(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;\n" ::"r"(dst), "l"(src), "r"(live ? 8 : 0));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t half2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ uint32_t mul_half2(uint32_t a, uint32_t b) {
    return half2_bits(__hmul2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b)));
}
// 2^-down as binary16 where down is 0 to kLevel, zero elsewhere
constexpr int kLevel = 14, kNone = -1 - kLevel;           // kNone: a reference that no exponent is in reach of
__device__ __forceinline__ uint32_t half_power(int down) { return (unsigned)down <= (unsigned)kLevel ? (uint32_t)(15 - down) << 10 : 0u; }
// 2^(ref - 127 - 15), the 15 for the weights; nothing is in reach of a negative ref
__device__ __forceinline__ float sum_power(int ref) { return __uint_as_float(ref > 15 ? (uint32_t)(ref - 15) << 23 : 1u << max(ref + 7, 0)); }

// Bytes of a token in shared memory.  A warp's reads meet no bank twice when eight K rows of four words (E2M1), four K rows of
// four double words (E4M3) and four V rows two apart fall into different quarters of the banks.
struct Layout {
    int k_pitch, v_pitch, scales, half, q_pitch, expand;      // expand: K's scales as floats, V's as pairs of binary16 powers
    constexpr __host__ __device__ Layout(int dim, bool fp4)
        : k_pitch(0), v_pitch(0), scales(0), half(0), q_pitch(0), expand(0) {
        const int nb = dim / 32, row = fp4 ? dim / 2 : dim, odd16 = ((row / 16) | 1) * 16;
        k_pitch = fp4 ? odd16 : ((row / 32) | 1) * 32;
        v_pitch = odd16;
        scales = kTok * (k_pitch > v_pitch ? k_pitch : v_pitch);
        half = scales + kTok * nb;             // K or V of 32 tokens
        q_pitch = (nb | 1) * 64;
        expand = nb * kTok * 4 + kTok / 2 * ((nb + 3) & ~3) * 4;
    }
};
__host__ __device__ __forceinline__ int smem_bytes(int dim, bool fp4, int nt) {
    const Layout l(dim, fp4);
    const int ring = kWarps * (3 * l.half + l.expand), cols = 8 * nt;
    const int merge = kWarps * cols * (dim + 4) * 4;
    return cols * l.q_pitch + (ring > merge ? ring : merge);
}

constexpr int ctas_by_registers(int nb, int nt) { return nt == 1 && nb <= 4 ? 4 : nb * nt <= 8 ? 3 : 2; }

template <int NB, bool FP4, int PIECES, int NT>
__global__ void __launch_bounds__(32 * kWarps, ctas_by_registers(NB, NT)) mx_attention_rows_kernel(const AttentionParams p) {
    constexpr int kCols = 8 * NT, kRows = kCols / PIECES, kMine = PIECES == 1 ? 2 * NT : NT;   // columns and rows of the CTA; rows that a lane holds
    extern __shared__ __align__(16) uint8_t smem[];
    const CacheView& c = p.c;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, tig = lane & 3;
    constexpr int dim = 32 * NB, nb = NB;
    constexpr Layout lay(dim, FP4);
    __shared__ int64_t place_sm[kPlaceWords];
    __shared__ float row_mul[kRows];
    next_may_start();
    zero_outside(p);
    RunOf<kTok> run(p, place_sm);
    while (run.left > 0) {
    const int seq = run.at.seq, head = run.at.head, tile = run.at.tile, pieces = run.at.w.pieces(tile), take = run.take(p, pieces);
    if (take == 0) break;
    const int2 own = rows_of(c, seq);
    const int first = tile * kRows, count = min(kRows, own.y * p.group - first);
    const int len = __ldg(c.lens + seq), pos0 = len - own.y;
    const TokenTiles<kTok> tt(p, pos0 + first / p.group, pos0 + (first + count - 1) / p.group);
    const bool finished = take == pieces;
    const int j_lo = min(run.at.piece, tt.tiles), j_hi = min(run.at.piece + take, tt.tiles);

    uint8_t* q_sm = smem;
    uint8_t* ring = smem + kCols * lay.q_pitch + warp * (3 * lay.half + lay.expand);
    float* k_scale = reinterpret_cast<float*>(ring + 3 * lay.half);                       // [block][token]
    uint32_t* v_scale = reinterpret_cast<uint32_t*>(k_scale + nb * kTok);                       // [pair of tokens][block, of four]
    constexpr int nb4 = (nb + 3) & ~3;
    const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);

    // ---- the warp's ring
    constexpr int row_bytes = FP4 ? dim / 2 : dim, chunks = row_bytes / 16, put_step = 32 / chunks;
    const int in_page = (1 << c.page_shift) - 1;
    const int put_tok = lane / chunks, put_ch = lane - put_tok * chunks;        // this lane's token and piece of 16 bytes
    auto page_of = [&](int j) -> int {          // the page of this lane's token of tile j; -1: none
        if (j >= j_hi) return -1;
        const int t = tt.start(j) + lane, slot = t >> c.page_shift;
        if (t >= tt.end || slot >= c.width) return -1;
        const int page = __ldg(c.pages + (int64_t)seq * c.width + slot);
        return page >= 0 && page < c.num_pages ? page : -1;
    };
    // K (or V) of the 32 tokens of tile j into place `slot` of the ring
    auto issue = [&](const uint8_t* codes, const uint8_t* scales, int pitch, int j, int slot, int page) {
        if (j < j_hi) {
            const uint32_t at = ring_at + slot * lay.half, to = at + put_tok * pitch + put_ch * 16;
            const int t0 = tt.start(j);
            const unsigned live = __ballot_sync(0xFFFFFFFFu, page >= 0);
            if (live == 0xFFFFFFFFu && c.page_shift >= 5) {                    // 32 rows that lie together
                const int64_t row = (((int64_t)page * c.heads + head) << c.page_shift) + (t0 & in_page) + put_tok;
                const uint8_t* src = codes + row * row_bytes + put_ch * 16;
                if (put_tok < put_step) {
#pragma unroll
                    for (int base = 0; base < kTok; base += put_step)
                        if (base + put_step <= kTok || base + put_tok < kTok) cp16(to + base * pitch, src + base * row_bytes, true);
                }
            } else {
                const int64_t mine = (((int64_t)max(page, 0) * c.heads + head) << c.page_shift) + ((t0 + lane) & in_page);
                for (int base = 0; base < kTok; base += put_step) {
                    const int tok = min(base + put_tok, kTok - 1);
                    const int64_t row = __shfl_sync(0xFFFFFFFFu, mine, tok);
                    const bool on = (live >> tok) & 1u;
                    if (put_tok < put_step && base + put_tok < kTok) cp16(to + base * pitch, codes + (on ? row * row_bytes + put_ch * 16 : 0), on);
                }
            }
            const int grp = lane / nb, pg = __shfl_sync(0xFFFFFFFFu, page, min(grp, 3) * 8);
            if (grp < 4) {                      // eight tokens' scales lie together, whatever the page size
                const int64_t row = (((int64_t)max(pg, 0) * c.heads + head) << c.page_shift) + ((t0 + grp * 8) & in_page);
                cp8(at + lay.scales + lane * 8, scales + (pg >= 0 ? row * nb + (lane - grp * nb) * 8 : 0), pg >= 0);
            }
        }
        asm volatile("cp.async.commit_group;\n" ::);
    };
    int page_put = page_of(j_lo + warp);
    unsigned there = __ballot_sync(0xFFFFFFFFu, page_put >= 0);               // which tokens of the tile there are
    issue(c.k_codes, c.k_scales, lay.k_pitch, j_lo + warp, 0, page_put);
    issue(c.v_codes, c.v_scales, lay.v_pitch, j_lo + warp, 1, page_put);
    page_put = page_of(j_lo + warp + kWarps);

    // ---- q: scaled by a power of two, as binary16 columns; one warp takes a row at a time
    for (int r = warp; r < kRows; r += kWarps) {
        const int rr = first + r, i = rr / p.group;
        float x[NB], top = 0.f;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            x[b] = 0.f;
            if (r < count) {
                const int64_t off = c.starts == nullptr ? seq * p.q_seq + i * p.q_row : (own.x + i) * p.q_row;
                x[b] = load_value(p.q, p.dtype, off + (head * p.group + rr - i * p.group) * p.q_head + b * 32 + lane);
                const float a = fabsf(x[b]);
                if (a < INFINITY) top = fmaxf(top, a);
                else x[b] = __uint_as_float(0x7FC00000u);      // an infinity gives scores of infinities and NaN alone: the row is NaN
            }
        }
        const uint32_t bits = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(top));
        const int e = bits ? min(max(127 + 14 - (int)(bits >> 23), -126), 126) : 0;
        const float up = __uint_as_float((uint32_t)(127 + e) << 23);
        if (lane == 0) row_mul[r] = p.scale_log2 * __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            {
                const float v = x[b] * up;
                const __half hi = __float2half_rn(v);
                __half* to = reinterpret_cast<__half*>(q_sm + r * PIECES * lay.q_pitch) + b * 32 + lane;
                *to = hi;
                if (PIECES == 2) {
                    const float left = (v - __half2float(hi)) * 2048.f;
                    to[lay.q_pitch / 2] = __float2half_rn(left);
                }
            }
        }
    }
    __syncthreads();

    // ---- rows of this lane
    float mul[kMine], m[kMine], l[kMine];
    int pos[kMine];
    unsigned poison[kMine];
#pragma unroll
    for (int r = 0; r < kMine; ++r) {
        const int at = PIECES == 1 ? (r >> 1) * 8 + 2 * tig + (r & 1) : r * 4 + tig;
        mul[r] = row_mul[at];
        pos[r] = at < count ? pos0 + (first + at) / p.group : -1;
        m[r] = -INFINITY;
        l[r] = 0.f;
        poison[r] = 0u;
    }
    const int low_pos = pos0 + first / p.group, high_pos = pos0 + (first + count - 1) / p.group;
    float o[NB][2][NT][4];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[b][j][n][i] = 0.f;

    int v_ref[NB];                            // the exponent that scales of V are taken relative to
#pragma unroll
    for (int b = 0; b < NB; ++b) v_ref[b] = kNone;
    // The ring has three places: while K of a tile is used, V of it and K of the warp's next tile are on the way.
    int slot = 0;
    for (int j = j_lo + warp; j < j_hi; j += kWarps) {
        const int slot_v = slot == 2 ? 0 : slot + 1, slot_k = slot_v == 2 ? 0 : slot_v + 1;
        issue(c.k_codes, c.k_scales, lay.k_pitch, j + kWarps, slot_k, page_put);
        asm volatile("cp.async.wait_group 2;\n" ::);
        __syncwarp();
        const uint8_t* k_sm = ring + slot * lay.half;
        uint8_t* v_sm = ring + slot_v * lay.half;
        const int t0 = tt.start(j);
#pragma unroll
        for (int b = 0; b < NB; ++b) k_scale[b * kTok + lane] = e8m0_value(k_sm[lay.scales + lane * nb + b]);
        __syncwarp();

        // ---- scores
        float s[2][NT][4];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[mt][n][i] = 0.f;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            {
                uint4 qb[NT];
#pragma unroll
                for (int n = 0; n < NT; ++n) qb[n] = *reinterpret_cast<const uint4*>(q_sm + (n * 8 + g) * lay.q_pitch + b * 64 + tig * 16);
#pragma unroll
                for (int mt = 0; mt < 2; ++mt) {
                    uint32_t a[4], d[4];
                    const uint8_t* row = k_sm + (mt * 16 + g) * lay.k_pitch;
                    if (FP4) {
                        e2m1x8_to_half(*reinterpret_cast<const uint32_t*>(row + b * 16 + tig * 4), a);
                        e2m1x8_to_half(*reinterpret_cast<const uint32_t*>(row + 8 * lay.k_pitch + b * 16 + tig * 4), d);
                    } else {
                        const uint2 x = *reinterpret_cast<const uint2*>(row + b * 32 + tig * 8), y = *reinterpret_cast<const uint2*>(row + 8 * lay.k_pitch + b * 32 + tig * 8);
                        e4m3x4_to_half(x.x, a[0], a[1]); e4m3x4_to_half(x.y, a[2], a[3]);
                        e4m3x4_to_half(y.x, d[0], d[1]); e4m3x4_to_half(y.y, d[2], d[3]);
                    }
                    const float s0 = k_scale[b * kTok + mt * 16 + g], s1 = k_scale[b * kTok + mt * 16 + 8 + g];
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float acc[4];
                        mma16816_first(acc, a[0], d[0], a[1], d[1], qb[n].x, qb[n].y);
                        mma16816(acc, a[2], d[2], a[3], d[3], qb[n].z, qb[n].w);
                        s[mt][n][0] = fmaf(acc[0], s0, s[mt][n][0]);
                        s[mt][n][1] = fmaf(acc[1], s0, s[mt][n][1]);
                        s[mt][n][2] = fmaf(acc[2], s1, s[mt][n][2]);
                        s[mt][n][3] = fmaf(acc[3], s1, s[mt][n][3]);
                    }
                }
            }
        }
        __syncwarp();                           // K's place is free
        // x[r][i]: row r of this lane, token g + 8 i of the tile, in units of log 2
        float x[kMine][4];
#pragma unroll
        for (int r = 0; r < kMine; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (PIECES == 1) x[r][i] = s[i >> 1][r >> 1][2 * (i & 1) + (r & 1)] * mul[r];
                else x[r][i] = fmaf(s[i >> 1][r][2 * (i & 1) + 1], 0x1p-11f, s[i >> 1][r][2 * (i & 1)]) * mul[r];
            }
        const bool whole = there == 0xFFFFFFFFu && t0 + kTok - 1 <= low_pos && (p.window <= 0 || t0 > high_pos - p.window);
        if (!whole) {
#pragma unroll
            for (int r = 0; r < kMine; ++r)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int t = g + 8 * i;
                    const bool on = ((there >> t) & 1u) && sees(p, pos[r], t0 + t);
                    x[r][i] = on ? x[r][i] : -INFINITY;
                }
        }
        bool higher = false;
#pragma unroll
        for (int r = 0; r < kMine; ++r) higher |= fmaxf(fmaxf(x[r][0], x[r][1]), fmaxf(x[r][2], x[r][3])) > m[r];
        if (__any_sync(0xFFFFFFFFu, higher)) {
#pragma unroll
            for (int r = 0; r < kMine; ++r) {
                float top = fmaxf(fmaxf(fmaxf(x[r][0], x[r][1]), fmaxf(x[r][2], x[r][3])), m[r]);
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 4));
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 8));
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 16));
                const float fade = top == -INFINITY ? 1.f : exp2_fast(m[r] - top);
                m[r] = top;
                l[r] *= fade;
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int jj = 0; jj < 2; ++jj) {
                        if (PIECES == 1) {
                            o[b][jj][r >> 1][r & 1] *= fade;
                            o[b][jj][r >> 1][2 + (r & 1)] *= fade;
                        } else {
#pragma unroll
                            for (int i = 0; i < 4; ++i) o[b][jj][r][i] *= fade;
                        }
                    }
            }
        }
        // ---- weights p 2^15, then as the second operand of the product with V
        uint32_t pw[2][NT][2];
#pragma unroll
        for (int r = 0; r < kMine; ++r) {
            const float base = (m[r] == -INFINITY ? 0.f : m[r]) - 15.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[r][i] = exp2_fast(x[r][i] - base);
                l[r] += x[r][i];
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t w;
                if (PIECES == 1) {
                    w = half2_bits(__floats2half2_rn(x[PIECES == 1 ? 2 * n : 0][i], x[PIECES == 1 ? 2 * n + 1 : 0][i]));
                } else {
                    const float v = x[n][i];
                    const __half hi = __float2half_rn(v);
                    w = half2_bits(__halves2half2(hi, __float2half_rn((v - __half2float(hi)) * 2048.f)));
                }
                pw[i >> 1][n][i & 1] = transpose8x8(w);
            }
        // ---- scales of V: each lane those of its token, relative to a reference, as binary16 powers of two
        issue(c.v_codes, c.v_scales, lay.v_pitch, j + kWarps, slot, page_put);
        asm volatile("cp.async.wait_group 2;\n" ::);
        __syncwarp();
        const bool mine = (there >> lane) & 1u;
        auto exponent = [&](int b) -> int { return mine ? (int)v_sm[lay.scales + lane * nb + b] : v_ref[b]; };
        auto zero_block = [&](int b) {
            uint32_t any = 0u;
            for (int i = 0; i < (FP4 ? 4 : 8); ++i) any |= reinterpret_cast<const uint32_t*>(v_sm + lane * lay.v_pitch)[b * (FP4 ? 4 : 8) + i];
            return (any & (FP4 ? 0x77777777u : 0x7F7F7F7Fu)) == 0u;
        };
        bool beyond = false;                    // a scale is above its reference or more than 2^kLevel below it
#pragma unroll
        for (int b = 0; b < NB; ++b) beyond |= (unsigned)(v_ref[b] - exponent(b)) > (unsigned)kLevel;
        bool levels = __any_sync(0xFFFFFFFFu, beyond);
        if (levels) {
            // a block scale of 0xFF: NaN for the rows that see the token, and nothing for those that do not
            uint32_t blocks_v = 0u;
#pragma unroll
            for (int b = 0; b < NB; ++b)
                if (exponent(b) == 255) {
                    blocks_v |= 1u << b;
                    for (int i = 0; i < (FP4 ? 4 : 8); ++i) reinterpret_cast<uint32_t*>(v_sm + lane * lay.v_pitch)[b * (FP4 ? 4 : 8) + i] = 0u;
                }
            for (uint32_t some = __ballot_sync(0xFFFFFFFFu, blocks_v != 0u); some; some &= some - 1) {
                const int t = __ffs(some) - 1;
                const uint32_t blocks = __shfl_sync(0xFFFFFFFFu, blocks_v, t);
#pragma unroll
                for (int r = 0; r < kMine; ++r)
                    if (sees(p, pos[r], t0 + t)) poison[r] |= blocks;
            }
            // new references: the largest so far where all scales are in its reach, else the largest of these
            levels = false;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const int e = mine && !((blocks_v >> b) & 1u) ? exponent(b) : kNone;
                const int top = __reduce_max_sync(0xFFFFFFFFu, e);
                const int low = __reduce_min_sync(0xFFFFFFFFu, e == kNone || (e < top - kLevel && zero_block(b)) ? 255 : e), high = max(v_ref[b], top);
                v_ref[b] = high - low <= kLevel ? high : top;
                levels |= low < top - kLevel;
            }
        }
        // Scales too far apart for one set of binary16 factors are taken in levels of 2^kLevel, the largest first: what a row adds up does
        // not depend on the scales of tokens that it does not see.
        do {
        uint32_t h[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            h[b] = half_power(v_ref[b] - exponent(b));
            h[b] |= __shfl_down_sync(0xFFFFFFFFu, h[b], 1) << 16;              // whole in the even lanes
        }
        if (!(lane & 1)) {
#pragma unroll
            for (int b = 0; b < NB; b += 4)
                *reinterpret_cast<uint4*>(v_scale + (lane >> 1) * nb4 + b) =
                    make_uint4(h[b], h[b + 1 < NB ? b + 1 : b], h[b + 2 < NB ? b + 2 : b], h[b + 3 < NB ? b + 3 : b]);
        }
        __syncwarp();

        // ---- values
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            float part[2][NT][4];                 // of these 32 tokens, added up in fp32 below
            {
#pragma unroll
                for (int mt = 0; mt < 2; ++mt) {
                    uint32_t pb[NT][2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int pair = mt * 8 + i * 4 + tig;
                        const uint32_t sc = v_scale[pair * nb4 + b];
#pragma unroll
                        for (int n = 0; n < NT; ++n) pb[n][i] = mul_half2(pw[mt][n][i], sc);
                    }
                    uint32_t a[2][4];                                               // [half of the block's 4 g .. 4 g + 3][register]
                    const uint8_t* row = v_sm + (mt * 16 + 2 * tig) * lay.v_pitch;
                    if (FP4) {
                        const uint8_t* at = row + b * 16 + g * 2;
                        const uint32_t w0 = *reinterpret_cast<const uint16_t*>(at), w1 = *reinterpret_cast<const uint16_t*>(at + lay.v_pitch);
                        const uint32_t w2 = *reinterpret_cast<const uint16_t*>(at + 8 * lay.v_pitch), w3 = *reinterpret_cast<const uint16_t*>(at + 9 * lay.v_pitch);
                        const uint32_t even = w0 | (w2 << 16), oddw = w1 | (w3 << 16);
                        uint32_t lo[4], hi[4];      // codes 0, 2 and 1, 3 of both tokens, first of the pair t, then of t + 8
                        const uint32_t x0 = (even & 0x0F0F0F0Fu) | ((oddw & 0x0F0F0F0Fu) << 4), x1 = ((even >> 4) & 0x0F0F0F0Fu) | (oddw & 0xF0F0F0F0u);
                        e2m1x8_to_half(x0, lo);
                        e2m1x8_to_half(x1, hi);
                        a[0][0] = lo[0]; a[0][1] = hi[0]; a[0][2] = lo[2]; a[0][3] = hi[2];
                        a[1][0] = lo[1]; a[1][1] = hi[1]; a[1][2] = lo[3]; a[1][3] = hi[3];
                    } else {
                        const uint8_t* at = row + b * 32 + g * 4;
                        const uint32_t w0 = *reinterpret_cast<const uint32_t*>(at), w1 = *reinterpret_cast<const uint32_t*>(at + lay.v_pitch);
                        const uint32_t w2 = *reinterpret_cast<const uint32_t*>(at + 8 * lay.v_pitch), w3 = *reinterpret_cast<const uint32_t*>(at + 9 * lay.v_pitch);
                        e4m3x4_to_half(__byte_perm(w0, w1, 0x5140), a[0][0], a[0][1]);
                        e4m3x4_to_half(__byte_perm(w2, w3, 0x5140), a[0][2], a[0][3]);
                        e4m3x4_to_half(__byte_perm(w0, w1, 0x7362), a[1][0], a[1][1]);
                        e4m3x4_to_half(__byte_perm(w2, w3, 0x7362), a[1][2], a[1][3]);
                    }
#pragma unroll
                    for (int jj = 0; jj < 2; ++jj)
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            if (mt == 0) mma16816_first(part[jj][n], a[jj][0], a[jj][1], a[jj][2], a[jj][3], pb[n][0], pb[n][1]);
                            else mma16816(part[jj][n], a[jj][0], a[jj][1], a[jj][2], a[jj][3], pb[n][0], pb[n][1]);
                        }
                }
            }
            const float up = sum_power(v_ref[b]);
#pragma unroll
            for (int jj = 0; jj < 2; ++jj)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[b][jj][n][i] = fmaf(part[jj][n][i], up, o[b][jj][n][i]);
        }
        __syncwarp();
        if (levels) {
            levels = false;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const int e = mine ? exponent(b) : 255;
                v_ref[b] = __reduce_max_sync(0xFFFFFFFFu, e < v_ref[b] - kLevel && !zero_block(b) ? e : kNone);
                levels |= v_ref[b] != kNone;
            }
        }
        } while (levels);
        slot = slot_k;
        there = __ballot_sync(0xFFFFFFFFu, page_put >= 0);
        page_put = page_of(j + 2 * kWarps);
    }
    asm volatile("cp.async.wait_group 0;\n" ::);
    __syncthreads();

    // ---- the four warps' results: sums [warp][row][dim], then maximum, sum and poisoned blocks of each row
    float* sums = reinterpret_cast<float*>(smem + kCols * lay.q_pitch);
    float* stats = sums + kWarps * kRows * dim;
#pragma unroll
    for (int r = 0; r < kMine; ++r) {
#pragma unroll
        for (int k = 4; k < 32; k <<= 1) l[r] += __shfl_xor_sync(0xFFFFFFFFu, l[r], k);
        const int at = PIECES == 1 ? (r >> 1) * 8 + 2 * tig + (r & 1) : r * 4 + tig;
        if (g == 0) {
            float* to = stats + (warp * kRows + at) * 3;
            to[0] = m[r];
            to[1] = 0x1p-15f * l[r];
            to[2] = __uint_as_float(poison[r]);
        }
#pragma unroll
        for (int b = 0; b < NB; ++b)
            {
                float* to = sums + (warp * kRows + at) * dim + b * 32 + 4 * g;
#pragma unroll
                for (int jj = 0; jj < 2; ++jj) {
                    if (PIECES == 1) {
                        to[2 * jj] = o[b][jj][r >> 1][r & 1];
                        to[2 * jj + 1] = o[b][jj][r >> 1][2 + (r & 1)];
                    } else {
                        to[2 * jj] = fmaf(o[b][jj][r][1], 0x1p-11f, o[b][jj][r][0]);
                        to[2 * jj + 1] = fmaf(o[b][jj][r][3], 0x1p-11f, o[b][jj][r][2]);
                    }
                }
            }
    }
    __syncthreads();
    const int share = 2 * blockIdx.x + (run.begins ? 0 : 1);
    for (int r = warp; r < count; r += kWarps) {
        float top = -INFINITY, w[kWarps], sum = 0.f;
        uint32_t bad = 0u;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) top = fmaxf(top, stats[(k * kRows + r) * 3]);
#pragma unroll
        for (int k = 0; k < kWarps; ++k) {
            const float* from = stats + (k * kRows + r) * 3;
            w[k] = from[0] == -INFINITY ? (from[1] != from[1] ? from[1] : 0.f) : exp2_fast(from[0] - top);   // a NaN sum stays one
            sum = fmaf(from[1], w[k], sum);
            bad |= __float_as_uint(from[2]);
        }
        const int rr = first + r, i = rr / p.group;
        const int64_t out_row = ((int64_t)(own.x + i) * p.q_heads + head * p.group + rr - i * p.group) * dim;
        const float inv_sum = sum == 0.f ? 0.f : __frcp_rn(sum);
        for (int b = 0; b < nb; ++b) {
            const int d = b * 32 + lane;
            float v = 0.f;
#pragma unroll
            for (int k = 0; k < kWarps; ++k) v = fmaf(sums[(k * kRows + r) * dim + d], w[k], v);
            if ((bad >> b) & 1u) v = __uint_as_float(0x7FC00000u);
            if (finished) store_value(p.out, p.dtype, out_row + d, v * inv_sum);
            else p.partial[((int64_t)share * kRows + r) * dim + d] = v;
        }
        if (!finished && lane == 0) {
            p.stats[(share * kRows + r) * 2] = top;
            p.stats[(share * kRows + r) * 2 + 1] = sum;
        }
    }
    __syncthreads();
    run.advance(p, take, pieces);
    }
    run.end(p);
}

// How a call is cut: columns of a tile, and CTAs.
struct Plan {
    int pieces, nt, tile_rows, runs;
    int64_t row_tiles, most_pieces;            // row tiles (about), and pieces of tokens of one at most
    size_t partial_floats, stats_floats;
};

Plan make_plan(const CacheView& c, int q_heads, int dtype, int window, int sinks) {
    Plan pl;
    const int group = q_heads / c.heads;
    pl.pieces = dtype == MPT_DTYPE_F32 ? 2 : 1;
    const int64_t per_seq = c.starts == nullptr ? (int64_t)c.new_rows * group : (c.seqs ? (c.rows * group + c.seqs - 1) / c.seqs : 0);
    // more than eight columns: a tile of 16 reads the cache once (16 sequences, four rows of 32 heads on 8 of 128 over 8192: 95 us, 109 in
    // two tiles of eight; over 1024 tokens of four sequences, where latency counts, 24 and 20)
    pl.nt = per_seq * pl.pieces > 8 ? 2 : 1;
    pl.tile_rows = 8 * pl.nt / pl.pieces;
    // at most four CTAs on each SM, and no more than there is work for if every sequence is as long as its row of the page table
    int64_t tokens = (int64_t)c.width << c.page_shift;
    if (window > 0 && tokens > (int64_t)window + sinks + 4 * kTok) tokens = (int64_t)window + sinks + 4 * kTok;
    const int64_t tiles = c.rows * group / pl.tile_rows + c.seqs, pieces = (tokens + kTok - 1) / kTok + 1, most = 4 * (int64_t)sm_count();
    const int64_t want = (tiles * c.heads * pieces + kLeast - 1) / kLeast;
    pl.runs = (int)(want < 1 ? 1 : want > most ? most : want);
    pl.row_tiles = tiles * c.heads;
    pl.most_pieces = pieces;
    pl.partial_floats = (size_t)2 * pl.runs * pl.tile_rows * c.dim;
    pl.stats_floats = (size_t)2 * pl.runs * pl.tile_rows * 2 + (size_t)pl.runs * (sizeof(Cut) / 4);      // and the cuts
    return pl;
}

// Which kernel a call takes, and the workspace it needs.  The chunk kernel from kChunkRows rows of q for a sequence and kv head on, on
// average.  It against this file's, by rows: head_dim 128, bfloat16, 16 sequences of 2048: 16 rows 62 and 66 us, 32 rows 68 and 89,
// 64 rows 79 and 164; four of 4096: 32 rows 52 and 55, 64 rows 63 and 60, 256 rows 92 and 128.  head_dim 64, float32, 16 sequences:
// 16 rows 78 and 51, 32 rows 80 and 93; four: 32 rows 47 and 43, 64 rows 52 and 62.  Where the expanded cache would pass 4 GB this
// file's kernel takes the call, which needs no such workspace.
constexpr int kChunkRows = 32;
struct CallShape {
    bool chunk;
    Plan rows;
    ChunkPlan chunks;
    size_t bytes() const {
        return chunk ? chunks.tile_bytes + 4 * (chunks.partial_floats + chunks.stats_floats) : 4 * (rows.partial_floats + rows.stats_floats);
    }
};

CallShape shape_of(const CacheView& c, int q_heads, int dtype, int window, int sinks) {
    CallShape s{};
    const int64_t per_seq = c.seqs ? c.rows * (q_heads / c.heads) / c.seqs : 0;
    if (per_seq >= kChunkRows && chunk_kernel_exists(c.dim, dtype)) {
        s.chunks = chunk_plan(c, q_heads);
        s.chunk = s.chunks.tile_bytes <= ((size_t)4 << 30);
    }
    if (!s.chunk) s.rows = make_plan(c, q_heads, dtype, window, sinks);
    return s;
}

template <int NB, bool FP4, int PIECES, int NT>
int launch_rows(AttentionParams p, const Plan& pl, cudaStream_t st) {
    const int bytes = smem_bytes(p.c.dim, FP4, NT);
    constexpr auto kern = mx_attention_rows_kernel<NB, FP4, PIECES, NT>;
    // CTAs on an SM, by registers (launch bounds) and shared memory (2 kB a CTA beside the dynamic part)
    const int by_memory = 228 * 1024 / (bytes + 2048), fit = by_memory < ctas_by_registers(NB, NT) ? (by_memory < 1 ? 1 : by_memory) : ctas_by_registers(NB, NT);
    if (!allow_shared<kern>(bytes)) return check_launch("mx_attention");
    const int most = fit * sm_count();
    p.runs = pl.runs < most ? pl.runs : most;
    p.whole = pl.row_tiles >= p.runs ? kWhole : 0;
    kern<<<(unsigned)p.runs, 32 * kWarps, bytes, st>>>(p);
    if (p.runs > 1 && pl.most_pieces > p.whole) launch_after(mx_attention_join_kernel, dim3((unsigned)(p.runs - 1), (unsigned)(p.tile_rows + 3) / 4), dim3(128), 0, st, p);
    return check_launch("mx_attention");
}

template <int NB, bool FP4>
int launch_rows(const AttentionParams& p, const Plan& pl, cudaStream_t st) {
    if (pl.pieces == 1) return pl.nt == 1 ? launch_rows<NB, FP4, 1, 1>(p, pl, st) : launch_rows<NB, FP4, 1, 2>(p, pl, st);
    return pl.nt == 1 ? launch_rows<NB, FP4, 2, 1>(p, pl, st) : launch_rows<NB, FP4, 2, 2>(p, pl, st);
}
template <bool FP4>
int launch_rows(const AttentionParams& p, const Plan& pl, cudaStream_t st) {
    switch (p.c.dim >> 5) {
        case 1: return launch_rows<1, FP4>(p, pl, st);
        case 2: return launch_rows<2, FP4>(p, pl, st);
        case 3: return launch_rows<3, FP4>(p, pl, st);
        case 4: return launch_rows<4, FP4>(p, pl, st);
        case 5: return launch_rows<5, FP4>(p, pl, st);
        case 6: return launch_rows<6, FP4>(p, pl, st);
        case 7: return launch_rows<7, FP4>(p, pl, st);
        default: return launch_rows<8, FP4>(p, pl, st);
    }
}

}  // namespace
}  // namespace mpt

using namespace mpt;

namespace {
std::atomic<int> fail_at{-1};
}

extern "C" {

void mpt_test_attention_wait_runs_out(int part) { fail_at.store(part, std::memory_order_relaxed); }

size_t mpt_mx_attention_workspace_bytes(const mpt_mx_cache* cache, const mpt_mx_batch* batch, int q_heads, int dtype, int window, int sinks) {
    CacheView c;
    if (!convert_cache("mx_attention", cache, batch, &c) || q_heads < 1 || q_heads % c.heads || c.rows == 0) return 0;
    return shape_of(c, q_heads, dtype, window, sinks).bytes();
}

int mpt_mx_attention(const mpt_mx_cache* cache, const mpt_mx_batch* batch, const void* q, int dtype, const int64_t* q_strides, int q_heads, float scale,
                     int window, int sinks, void* out, int zero_tail, void* workspace, size_t workspace_bytes, void* stream) {
    AttentionParams p{};
    if (!convert_cache("mx_attention", cache, batch, &p.c)) return MPT_ERR_INVALID_ARGUMENT;
    CacheView& c = p.c;
    MPT_REQUIRE(q_heads >= 1 && q_heads % c.heads == 0, "mx_attention: %d query heads do not divide among %d kv heads", q_heads, c.heads);
    MPT_REQUIRE(window >= 0 && sinks >= 0, "mx_attention: window and sinks must not be negative");
    MPT_REQUIRE(dtype == MPT_DTYPE_F32 || dtype == MPT_DTYPE_BF16 || dtype == MPT_DTYPE_F16, "mx_attention: unknown data type %d", dtype);
    if (c.rows == 0) return MPT_OK;
    MPT_REQUIRE(q && q_strides && out, "mx_attention: null pointer");
    MPT_REQUIRE(c.rows * q_heads <= 0x7FFFFFFF, "mx_attention: more than 2^31 - 1 rows of heads");
    const CallShape call = shape_of(c, q_heads, dtype, window, sinks);
    if (workspace_bytes < call.bytes() || !workspace || ((uintptr_t)workspace & 255u)) {
        set_error("mx_attention: a workspace of %zu bytes at a multiple of 256 is needed", call.bytes());
        return MPT_ERR_WORKSPACE;
    }
    const int64_t size = dtype == MPT_DTYPE_F32 ? 4 : 2;
    p.q = q; p.dtype = dtype;
    p.q_seq = q_strides[0]; p.q_row = q_strides[1]; p.q_head = q_strides[2];
    p.q_vec = (((int64_t)(uintptr_t)q | size * (p.q_row | p.q_head | (c.starts ? 0 : p.q_seq))) & 15) == 0;
    p.out_vec = ((uintptr_t)out & 15u) == 0;
    p.q_heads = q_heads; p.group = q_heads / c.heads;
    p.scale_log2 = (float)((double)scale * 1.4426950408889634);
    p.window = window < (1 << 30) ? window : 1 << 30;          // so that no position leaves 32 bits
    p.sinks = sinks < (1 << 30) ? sinks : 1 << 30;
    p.out = out; p.zero_tail = zero_tail;
    p.fail_at = fail_at.load(std::memory_order_relaxed);
    cudaStream_t st = as_stream(stream);
    const bool fp4 = cache->elem_format == MPT_ELEM_E2M1;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    if (call.chunk) {
        p.partial = reinterpret_cast<float*>(ws + call.chunks.tile_bytes);
        p.stats = p.partial + call.chunks.partial_floats;
        p.cuts = reinterpret_cast<Cut*>(p.stats + call.chunks.stats_floats - (size_t)call.chunks.runs * (sizeof(Cut) / 4));
        return launch_chunk(p, call.chunks, ws, fp4, st);
    }
    p.tile_rows = call.rows.tile_rows; p.least = kLeast;
    p.partial = reinterpret_cast<float*>(ws);
    p.stats = p.partial + call.rows.partial_floats;
    p.cuts = reinterpret_cast<Cut*>(p.stats + (size_t)4 * call.rows.runs * call.rows.tile_rows);
    return fp4 ? launch_rows<true>(p, call.rows, st) : launch_rows<false>(p, call.rows, st);
}

}
