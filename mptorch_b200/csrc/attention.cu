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
// block's partial sums; the scale of V multiplies p, relative to the largest of 32 tokens, and what was taken out multiplies the
// partial sums.  q is scaled by a power of two to a largest value in [2^14, 2^15) and held as binary16: bfloat16 and float16 in
// one piece, exact unless a value is 2^-29 of the row's largest or less; float32 in two columns, the second 2^11 times what the
// first leaves (22 bits).  p 2^15 is rounded to binary16 (11 bits) in one piece, for float32 in two.  The running maximum is
// moved only when a tile exceeds it.
//
// Measured figures stand at the launch rule below.
#include "attention.cuh"

namespace mpt {
namespace {

constexpr int kWarps = 4, kTok = 32;

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(live ? 16 : 0));
}
__device__ __forceinline__ void cp8(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;\n" ::"r"(dst), "l"(src), "r"(live ? 8 : 0));
}
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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
__device__ __forceinline__ uint32_t half_power(int down) {   // 2^-down as binary16, zero below 2^-24
    return down < 15 ? (uint32_t)(15 - down) << 10 : (down < 25 ? 1u << (24 - down) : 0u);
}
__device__ __forceinline__ bool has_ff(uint32_t w) {     // some byte of w is 0xFF
    const uint32_t x = ~w;
    return ((x - 0x01010101u) & ~x & 0x80808080u) != 0u;
}

// Bytes of a token in shared memory.  A warp's reads meet no bank twice when eight K rows of four words (E2M1), four K rows of
// four double words (E4M3) and four V rows two apart fall into different quarters of the banks.
struct Layout {
    int k_pitch, v_pitch, scales, stage, q_pitch;
    __host__ __device__ Layout(int dim, bool fp4) {
        const int nb = dim / 32, row = fp4 ? dim / 2 : dim, odd16 = ((row / 16) | 1) * 16;
        k_pitch = fp4 ? odd16 : ((row / 32) | 1) * 32;
        v_pitch = odd16;
        scales = kTok * (k_pitch + v_pitch);
        stage = (scales + 2 * kTok * nb + 16 + 15) / 16 * 16;
        q_pitch = (nb | 1) * 64;
    }
};
__host__ __device__ __forceinline__ int smem_bytes(int dim, bool fp4, int nt, int stages) {
    const Layout l(dim, fp4);
    const int ring = kWarps * stages * l.stage, cols = 8 * nt;
    const int merge = kWarps * cols * (dim + 4) * 4;
    return cols * l.q_pitch + (ring > merge ? ring : merge);
}

template <int NBT, bool FP4, int PIECES, int NT, int STAGES>
__global__ void __launch_bounds__(32 * kWarps) mx_attention_rows_kernel(const AttentionParams p) {
    constexpr int kCols = 8 * NT, kRows = kCols / PIECES, kMine = PIECES == 1 ? 2 * NT : NT;   // columns and rows of the CTA; rows that a lane holds
    extern __shared__ __align__(16) uint8_t smem[];
    const CacheView& c = p.c;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, tig = lane & 3;
    const int dim = c.dim, nb = dim >> 5, head = blockIdx.y, split = blockIdx.z;
    const Layout lay(dim, FP4);
    if (split == 0 && head == 0) zero_outside(p);
    int seq, tile;
    if (!find_tile(p, blockIdx.x, seq, tile)) return;
    const int2 own = rows_of(c, seq);
    const int first = tile * kRows, count = min(kRows, own.y * p.group - first);
    if (count <= 0) return;
    const int len = __ldg(c.lens + seq), pos0 = len - own.y;
    const TokenTiles<kTok> tt(p, pos0 + first / p.group, pos0 + (first + count - 1) / p.group);
    // parts of at least two tiles a warp
    const int parts = max(1, min(p.splits, tt.tiles / (2 * kWarps)));
    if (split >= parts) return;
    const int j_lo = (int)((int64_t)tt.tiles * split / parts), j_hi = (int)((int64_t)tt.tiles * (split + 1) / parts);

    uint8_t* q_sm = smem;
    uint8_t* ring = smem + kCols * lay.q_pitch + warp * STAGES * lay.stage;
    const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);

    // ---- the warp's ring
    const int row_bytes = FP4 ? dim >> 1 : dim, chunks = row_bytes >> 4, inv = 65536 / chunks + 1;
    auto page_of = [&](int j) -> int {          // the page of this lane's token of tile j; -1: none
        if (j >= j_hi) return -1;
        const int t = tt.start(j) + lane, slot = t >> c.page_shift;
        if (t >= tt.end || slot >= c.width) return -1;
        const int page = __ldg(c.pages + (int64_t)seq * c.width + slot);
        return page >= 0 && page < c.num_pages ? page : -1;
    };
    auto issue = [&](int j, int stage, int page) {
        if (j < j_hi) {
            const uint32_t at = ring_at + stage * lay.stage;
            const int t0 = tt.start(j), in_page = (1 << c.page_shift) - 1;
            for (int i = 0; i < chunks; ++i) {
                const int idx = i * 32 + lane, tok = (idx * inv) >> 16, ch = idx - tok * chunks;
                const int pg = __shfl_sync(0xFFFFFFFFu, page, tok);
                const int64_t row = (((int64_t)max(pg, 0) * c.heads + head) << c.page_shift) + ((t0 + tok) & in_page);
                const int64_t off = row * row_bytes + ch * 16;
                cp16(at + tok * lay.k_pitch + ch * 16, c.k_codes + (pg >= 0 ? off : 0), pg >= 0);
                cp16(at + kTok * lay.k_pitch + tok * lay.v_pitch + ch * 16, c.v_codes + (pg >= 0 ? off : 0), pg >= 0);
            }
            const int grp = lane / nb, pg = __shfl_sync(0xFFFFFFFFu, page, min(grp, 3) * 8);
            if (grp < 4) {                      // eight tokens' scales lie together, whatever the page size
                const int64_t row = (((int64_t)max(pg, 0) * c.heads + head) << c.page_shift) + ((t0 + grp * 8) & in_page);
                const int64_t off = pg >= 0 ? row * nb + (lane - grp * nb) * 8 : 0;
                cp8(at + lay.scales + lane * 8, c.k_scales + off, pg >= 0);
                cp8(at + lay.scales + kTok * nb + lane * 8, c.v_scales + off, pg >= 0);
            }
            const unsigned there = __ballot_sync(0xFFFFFFFFu, page >= 0);
            if (lane == 0) *reinterpret_cast<uint32_t*>(ring + stage * lay.stage + lay.scales + 2 * kTok * nb) = there;
        }
        asm volatile("cp.async.commit_group;\n" ::);
    };
    int j_put = j_lo + warp, page_put = page_of(j_put);
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) {
        issue(j_put, s, page_put);
        j_put += kWarps;
        page_put = page_of(j_put);
    }

    // ---- q: scaled by a power of two, as binary16 columns; one warp takes a row at a time
    __shared__ float row_mul[kRows];
    for (int r = warp; r < kRows; r += kWarps) {
        const int rr = first + r, i = rr / p.group;
        float x[NBT], top = 0.f;
#pragma unroll
        for (int b = 0; b < NBT; ++b) {
            x[b] = 0.f;
            if (b < nb && r < count) {
                const int64_t off = c.starts == nullptr ? seq * p.q_seq + i * p.q_row : (own.x + i) * p.q_row;
                x[b] = load_value(p.q, p.dtype, off + (head * p.group + rr - i * p.group) * p.q_head + b * 32 + lane);
                const float a = fabsf(x[b]);
                if (a < INFINITY) top = fmaxf(top, a);
            }
        }
        const uint32_t bits = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(top));
        const int e = bits ? min(max(127 + 14 - (int)(bits >> 23), -126), 126) : 0;
        const float up = __uint_as_float((uint32_t)(127 + e) << 23);
        if (lane == 0) row_mul[r] = p.scale_log2 * __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
        for (int b = 0; b < NBT; ++b) {
            if (b < nb) {
                const float v = x[b] * up;
                const __half hi = __float2half_rn(v);
                __half* to = reinterpret_cast<__half*>(q_sm + r * PIECES * lay.q_pitch) + b * 32 + lane;
                *to = hi;
                if (PIECES == 2) {
                    const float left = (v - __half2float(hi)) * 2048.f;
                    to[lay.q_pitch / 2] = fabsf(v) < INFINITY ? __float2half_rn(left) : __float2half_rn(0.f);
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
    float o[NBT][2][NT][4];
#pragma unroll
    for (int b = 0; b < NBT; ++b)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[b][j][n][i] = 0.f;

    int stage = 0;
    for (int j = j_lo + warp; j < j_hi; j += kWarps) {
        {
            int put = stage + STAGES - 1;
            if (put >= STAGES) put -= STAGES;
            issue(j_put, put, page_put);
            j_put += kWarps;
            page_put = page_of(j_put);
        }
        asm volatile("cp.async.wait_group %0;\n" ::"n"(STAGES - 1));
        __syncwarp();
        uint8_t* k_sm = ring + stage * lay.stage;
        uint8_t* v_sm = k_sm + kTok * lay.k_pitch;
        const uint8_t* ks = k_sm + lay.scales;
        const uint8_t* vs = ks + kTok * nb;
        const uint32_t there = *reinterpret_cast<const uint32_t*>(vs + kTok * nb);
        const int t0 = tt.start(j);

        // a block scale of 0xFF: what the tokens' rows of K and V hold there is NaN
        uint32_t k_nan = 0u;
        bool ff = false;
        if (lane < 4 * nb) {
            const uint2 a = reinterpret_cast<const uint2*>(ks)[lane], b = reinterpret_cast<const uint2*>(vs)[lane];
            ff = has_ff(a.x) || has_ff(a.y) || has_ff(b.x) || has_ff(b.y);
        }
        if (__any_sync(0xFFFFFFFFu, ff)) {
            bool bad_k = false;
            uint32_t bad_v = 0u;
            if ((there >> lane) & 1u)
                for (int b = 0; b < nb; ++b) {
                    bad_k |= ks[lane * nb + b] == 255;
                    if (vs[lane * nb + b] == 255) {
                        bad_v |= 1u << b;
                        for (int i = 0; i < (FP4 ? 4 : 8); ++i) reinterpret_cast<uint32_t*>(v_sm + lane * lay.v_pitch)[b * (FP4 ? 4 : 8) + i] = 0u;
                    }
                }
            k_nan = __ballot_sync(0xFFFFFFFFu, bad_k);
            for (uint32_t some = __ballot_sync(0xFFFFFFFFu, bad_v != 0u); some; some &= some - 1) {
                const int t = __ffs(some) - 1;
                const uint32_t blocks = __shfl_sync(0xFFFFFFFFu, bad_v, t);
#pragma unroll
                for (int r = 0; r < kMine; ++r)
                    if (sees(p, pos[r], t0 + t)) poison[r] |= blocks;
            }
            __syncwarp();
        }

        // ---- scores
        float s[2][NT][4];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[mt][n][i] = 0.f;
#pragma unroll
        for (int b = 0; b < NBT; ++b) {
            if (b < nb) {
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
                    // 2^-127 for a code of 0; a code of 0xFF (infinity here) is looked for above
                    const float s0 = __uint_as_float(max((uint32_t)ks[(mt * 16 + g) * nb + b] << 23, 0x00400000u));
                    const float s1 = __uint_as_float(max((uint32_t)ks[(mt * 16 + 8 + g) * nb + b] << 23, 0x00400000u));
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float acc[4] = {0.f, 0.f, 0.f, 0.f};
                        mma16816(acc, a[0], d[0], a[1], d[1], qb[n].x, qb[n].y);
                        mma16816(acc, a[2], d[2], a[3], d[3], qb[n].z, qb[n].w);
                        s[mt][n][0] = fmaf(acc[0], s0, s[mt][n][0]);
                        s[mt][n][1] = fmaf(acc[1], s0, s[mt][n][1]);
                        s[mt][n][2] = fmaf(acc[2], s1, s[mt][n][2]);
                        s[mt][n][3] = fmaf(acc[3], s1, s[mt][n][3]);
                    }
                }
            }
        }
        // x[r][i]: row r of this lane, token g + 8 i of the tile, in units of log 2
        float x[kMine][4];
#pragma unroll
        for (int r = 0; r < kMine; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (PIECES == 1) x[r][i] = s[i >> 1][r >> 1][2 * (i & 1) + (r & 1)] * mul[r];
                else x[r][i] = fmaf(s[i >> 1][r][2 * (i & 1) + 1], 0x1p-11f, s[i >> 1][r][2 * (i & 1)]) * mul[r];
            }
        const bool whole = there == 0xFFFFFFFFu && k_nan == 0u && t0 + kTok - 1 <= low_pos && (p.window <= 0 || t0 > high_pos - p.window);
        if (!whole) {
#pragma unroll
            for (int r = 0; r < kMine; ++r)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int t = g + 8 * i;
                    const bool on = ((there >> t) & 1u) && sees(p, pos[r], t0 + t);
                    if ((k_nan >> t) & 1u) x[r][i] = __uint_as_float(0x7FC00000u);
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
                for (int b = 0; b < NBT; ++b)
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
        // ---- values
#pragma unroll
        for (int b = 0; b < NBT; ++b) {
            if (b < nb) {
                uint32_t e = ((there >> lane) & 1u) ? vs[lane * nb + b] : 0u;      // this lane's token
                e = e == 255u ? 0u : e;
                const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, e);
                const int down = (int)(top - e);
                uint32_t h = half_power(min(down, 24));
                h |= __shfl_down_sync(0xFFFFFFFFu, h, 1) << 16;                     // whole in the even lanes
                // binary16 has no power below 2^-24: scales further apart take a second factor
                const bool wide = __any_sync(0xFFFFFFFFu, down > 24);
                uint32_t h2 = 0u;
                if (wide) {
                    h2 = half_power(max(down - 24, 0));
                    h2 |= __shfl_down_sync(0xFFFFFFFFu, h2, 1) << 16;
                }
                const float up = e8m0_value(top);
                float acc[2][NT][4];
#pragma unroll
                for (int jj = 0; jj < 2; ++jj)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[jj][n][i] = 0.f;
#pragma unroll
                for (int mt = 0; mt < 2; ++mt) {
                    uint32_t pb[NT][2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t sc = __shfl_sync(0xFFFFFFFFu, h, mt * 16 + i * 8 + 2 * tig);
#pragma unroll
                        for (int n = 0; n < NT; ++n) pb[n][i] = mul_half2(pw[mt][n][i], sc);
                        if (wide) {
                            const uint32_t sc2 = __shfl_sync(0xFFFFFFFFu, h2, mt * 16 + i * 8 + 2 * tig);
#pragma unroll
                            for (int n = 0; n < NT; ++n) pb[n][i] = mul_half2(pb[n][i], sc2);
                        }
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
                        for (int n = 0; n < NT; ++n) mma16816(acc[jj][n], a[jj][0], a[jj][1], a[jj][2], a[jj][3], pb[n][0], pb[n][1]);
                }
#pragma unroll
                for (int jj = 0; jj < 2; ++jj)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[b][jj][n][i] = fmaf(acc[jj][n][i], up, o[b][jj][n][i]);
            }
        }
        __syncwarp();
        if (++stage == STAGES) stage = 0;
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
            to[1] = l[r];
            to[2] = __uint_as_float(poison[r]);
        }
#pragma unroll
        for (int b = 0; b < NBT; ++b)
            if (b < nb) {
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
    const int64_t part = ((int64_t)blockIdx.x * c.heads + head) * p.splits + split;
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
            if (parts == 1) store_value(p.out, p.dtype, out_row + d, v * inv_sum);
            else p.partial[(part * kRows + r) * dim + d] = v;
        }
        if (parts > 1 && lane == 0) {
            p.stats[(part * kRows + r) * 2] = top;
            p.stats[(part * kRows + r) * 2 + 1] = sum;
        }
    }
}

// Joins the parts of each row: a warp per row.
__global__ void __launch_bounds__(128) mx_attention_join_kernel(const AttentionParams p) {
    const CacheView& c = p.c;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, dim = c.dim, nb = dim >> 5, head = blockIdx.y;
    int seq, tile;
    if (!find_tile(p, blockIdx.x, seq, tile)) return;
    const int2 own = rows_of(c, seq);
    const int first = tile * p.tile_rows, count = min(p.tile_rows, own.y * p.group - first);
    if (count <= 0) return;
    const int pos0 = __ldg(c.lens + seq) - own.y;
    const TokenTiles<kTok> tt(p, pos0 + first / p.group, pos0 + (first + count - 1) / p.group);
    const int parts = max(1, min(p.splits, tt.tiles / (2 * kWarps)));
    if (parts == 1) return;
    const int64_t part0 = ((int64_t)blockIdx.x * c.heads + head) * p.splits;
    for (int r = warp; r < count; r += 4) {
        float top = -INFINITY;
        for (int k = 0; k < parts; ++k) top = fmaxf(top, p.stats[((part0 + k) * p.tile_rows + r) * 2]);
        float sum = 0.f, v[8] = {};
        for (int k = 0; k < parts; ++k) {
            const float* st = p.stats + ((part0 + k) * p.tile_rows + r) * 2;
            const float w = st[0] == -INFINITY ? (st[1] != st[1] ? st[1] : 0.f) : exp2_fast(st[0] - top);
            sum = fmaf(st[1], w, sum);
            const float* from = p.partial + ((part0 + k) * p.tile_rows + r) * dim + lane;
#pragma unroll
            for (int b = 0; b < 8; ++b)
                if (b < nb) v[b] = fmaf(from[b * 32], w, v[b]);
        }
        const int rr = first + r, i = rr / p.group;
        const int64_t out_row = ((int64_t)(own.x + i) * p.q_heads + head * p.group + rr - i * p.group) * dim;
        const float inv_sum = sum == 0.f ? 0.f : __frcp_rn(sum);
#pragma unroll
        for (int b = 0; b < 8; ++b)
            if (b < nb) store_value(p.out, p.dtype, out_row + b * 32 + lane, v[b] * inv_sum);
    }
}

// How a call is cut: columns of a tile, row tiles, parts of the tokens.
struct Plan {
    int pieces, nt, tile_rows, tiles_per_seq, splits;
    int64_t tiles;
    size_t partial_floats, stats_floats;
};

Plan make_plan(const CacheView& c, int q_heads, int dtype, int window, int sinks) {
    Plan pl;
    const int group = q_heads / c.heads;
    pl.pieces = dtype == MPT_DTYPE_F32 ? 2 : 1;
    const int64_t per_seq = c.starts == nullptr ? (int64_t)c.new_rows * group : (c.seqs ? (c.rows * group + c.seqs - 1) / c.seqs : 0);
    pl.nt = per_seq * pl.pieces > 8 ? 2 : 1;
    pl.tile_rows = 8 * pl.nt / pl.pieces;
    pl.tiles_per_seq = (int)(((int64_t)c.new_rows * group + pl.tile_rows - 1) / pl.tile_rows);
    pl.tiles = c.starts == nullptr ? (int64_t)c.seqs * pl.tiles_per_seq : (c.rows * group + pl.tile_rows - 1) / pl.tile_rows + c.seqs;
    // parts: two waves of two CTAs on each SM, a part having two tiles for each warp at least
    int64_t tokens = (int64_t)c.width << c.page_shift;
    if (window > 0) tokens = tokens < (int64_t)window + sinks + 2 * kTok ? tokens : (int64_t)window + sinks + 2 * kTok;
    const int64_t most = tokens / kTok / (2 * kWarps), want = (4 * (int64_t)sm_count() + pl.tiles * c.heads - 1) / (pl.tiles * c.heads > 0 ? pl.tiles * c.heads : 1);
    pl.splits = (int)(want < 1 ? 1 : want > most ? (most < 1 ? 1 : most) : want);
    if (pl.splits > 64) pl.splits = 64;
    const size_t rows = (size_t)pl.tiles * c.heads * pl.splits * pl.tile_rows;
    pl.partial_floats = pl.splits > 1 ? rows * c.dim : 0;
    pl.stats_floats = pl.splits > 1 ? rows * 2 : 0;
    return pl;
}

template <int NBT, bool FP4, int PIECES, int NT>
int launch_rows(const AttentionParams& p, const Plan& pl, cudaStream_t st) {
    constexpr int STAGES = 2;
    const int bytes = smem_bytes(p.c.dim, FP4, NT, STAGES);
    auto kern = mx_attention_rows_kernel<NBT, FP4, PIECES, NT, STAGES>;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return check_launch("mx_attention");
    kern<<<dim3((unsigned)pl.tiles, (unsigned)p.c.heads, (unsigned)pl.splits), 32 * kWarps, bytes, st>>>(p);
    if (pl.splits > 1) mx_attention_join_kernel<<<dim3((unsigned)pl.tiles, (unsigned)p.c.heads), 128, 0, st>>>(p);
    return check_launch("mx_attention");
}

template <int NBT, bool FP4>
int launch_rows(const AttentionParams& p, const Plan& pl, cudaStream_t st) {
    if (pl.pieces == 1) return pl.nt == 1 ? launch_rows<NBT, FP4, 1, 1>(p, pl, st) : launch_rows<NBT, FP4, 1, 2>(p, pl, st);
    return pl.nt == 1 ? launch_rows<NBT, FP4, 2, 1>(p, pl, st) : launch_rows<NBT, FP4, 2, 2>(p, pl, st);
}
template <bool FP4>
int launch_rows(const AttentionParams& p, const Plan& pl, cudaStream_t st) {
    if (p.c.dim <= 64) return launch_rows<2, FP4>(p, pl, st);
    if (p.c.dim <= 128) return launch_rows<4, FP4>(p, pl, st);
    return launch_rows<8, FP4>(p, pl, st);
}

}  // namespace
}  // namespace mpt

using namespace mpt;

extern "C" {

size_t mpt_mx_attention_workspace_bytes(const mpt_mx_cache* cache, const mpt_mx_batch* batch, int q_heads, int dtype, int window, int sinks) {
    CacheView c;
    if (!convert_cache("mx_attention", cache, batch, &c) || q_heads < 1 || q_heads % c.heads || c.rows == 0) return 0;
    const Plan pl = make_plan(c, q_heads, dtype, window, sinks);
    return 4 * (pl.partial_floats + pl.stats_floats);
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
    const Plan pl = make_plan(c, q_heads, dtype, window, sinks);
    if (workspace_bytes < 4 * (pl.partial_floats + pl.stats_floats) || (pl.partial_floats && !workspace) || ((uintptr_t)workspace & 15u)) {
        set_error("mx_attention: a workspace of %zu bytes at a multiple of 256 is needed", 4 * (pl.partial_floats + pl.stats_floats));
        return MPT_ERR_WORKSPACE;
    }
    p.q = q; p.dtype = dtype;
    p.q_seq = q_strides[0]; p.q_row = q_strides[1]; p.q_head = q_strides[2];
    p.q_heads = q_heads; p.group = q_heads / c.heads;
    p.scale_log2 = (float)((double)scale * 1.4426950408889634);
    p.window = window; p.sinks = sinks;
    p.out = out; p.zero_tail = zero_tail;
    p.tile_rows = pl.tile_rows; p.tiles_per_seq = pl.tiles_per_seq; p.splits = pl.splits;
    p.partial = static_cast<float*>(workspace);
    p.stats = p.partial + pl.partial_floats;
    cudaStream_t st = as_stream(stream);
    return cache->elem_format == MPT_ELEM_E2M1 ? launch_rows<true>(p, pl, st) : launch_rows<false>(p, pl, st);
}

}
