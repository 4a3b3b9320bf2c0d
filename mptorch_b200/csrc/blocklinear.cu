// y = x W^T + b for a few rows of x, with W held as packed E2M1 codes and group scales (MXFP4, NVFP4).
//
// Bound: HBM, the codes and scales of W (half a byte and 1/32 or 1/16 of one for each weight).  At the measured bandwidth that is
// 46 weights a clock on each SM, which leaves less than three instructions a weight: E2M1 is exact in binary16, so codes go to
// the m16n8k16 tensor-core products after one conversion for two of them.  A CTA keeps x in shared memory and walks tiles of 16
// rows of W; one, two, four, eight or all sixteen of its warps share a tile, taking pieces of 128 of the sum in turn, each with a ring of its own
// that cp.async fills.
//
// x is scaled for each row by a power of two to a largest value in [2^14, 2^15) and held as binary16: bfloat16 and float16 in one
// column (exact unless a value is 2^-29 of the largest or less), float32 in two, the second 2^11 times what the first leaves (22
// bits).  NVFP4: a code times its E4M3 scale is exact in binary16 (six bits), so the weights are scaled and the products of a piece of
// 128 summed by the tensor cores; pieces are added up in fp32 registers, since the tensor cores cut their sums off instead of rounding
// them (two float32 rows of 9600 by 33000: 2.4e-7 of the result, 1.1e-5 with sums that run through).  MXFP4: the scale of a block multiplies the fp32 sum of its 32 products, relative to an exponent that is kept
// for each row of W and raised when a block exceeds it by 2^60, so that no range of scales overflows.
//
// Measured on a B200 (weights' bytes at the measured bandwidth in brackets): one bfloat16 row of 8192 by 28672 NVFP4 weights 39 us
// (20.2); three float32 rows of 768 by 50257 MXFP4 weights 14.4 us (3.2); one of 768 by 2304 9.7 us (0.1: host time and a launch).
// The largest has its issue slots 55 % busy and DRAM 43 %: four warps a scheduler do not cover the fixed latency between an instruction
// and the next that needs it (39 of them for 512 weights).  Copies of twice the depth changed nothing.
#include "blocklinear.cuh"
#include "launch.cuh"

namespace mpt {
namespace {

constexpr int kWarps = 16, kChunk = 128, kPitch = 80, kStages = 3;          // pitch: eight rows of four words meet no bank twice

__device__ __forceinline__ void cp_bytes(uint32_t dst, const void* src, int bytes) {   // 16
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(bytes));
}
template <int N>
__device__ __forceinline__ void cp_small(uint32_t dst, const void* src, int bytes) {   // 4 or 8
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;\n" ::"r"(dst), "l"(src), "n"(N), "r"(bytes));
}
__device__ __forceinline__ uint32_t times(uint32_t a, __half2 s) {
    const __half2 r = __hmul2(*reinterpret_cast<__half2*>(&a), s);
    return *reinterpret_cast<const uint32_t*>(&r);
}
// 2^(e - ref), zero below 2^-149
__device__ __forceinline__ float relative_power(int e, int ref) {
    const int d = e - ref;
    return d >= -126 ? __uint_as_float((uint32_t)(d + 127) << 23) : d >= -149 ? __uint_as_float(1u << (d + 149)) : 0.f;
}

__host__ __device__ constexpr int stage_bytes(bool nv) { return 16 * kPitch + 16 * (nv ? 8 : 4); }
__host__ __device__ inline int x_pitch(int n_in) { return (n_in + kChunk - 1) / kChunk * kChunk * 2 + 64; }   // whole pieces; 64 bytes behind a multiple of 128
constexpr int few_smem(int x_bytes, bool nv, int nt) { return x_bytes + kWarps * kStages * stage_bytes(nv) + kWarps * 16 * 8 * nt * 4; }   // x, rings, sums
// What few_rows admits of x, and the shared memory that the kernel is allowed: whatever is admitted can be launched.
constexpr int kMostX = 140 * 1024, kMostShared = few_smem(kMostX, true, 2);
static_assert(kMostShared + 2 * 1024 <= 227 * 1024, "2 kB for the kernel's static shared memory");

// GROUPS: one column (NVFP4), one or two (MXFP4).  The other columns of the products are used to keep the scale groups apart: column c
// has x where its group is c and zeros elsewhere, so that a column's sum over a piece of 128 is that of one group, and the scales
// multiply eight sums a row and piece instead of 128 weights.  NVFP4: eight groups of 16.  MXFP4: four blocks of 32 in columns 0 to 3,
// and in 4 to 7 those of the second column.  With and without, 8192 by 28672: NVFP4 40 and 44 us for one column (48 and 46 for two,
// which would need products of their own), MXFP4 50 and 61 for one, 51 and 63 for two.
template <bool NV, int PIECES, int NT, bool GROUPS>
__global__ void __launch_bounds__(32 * kWarps, 1) block_linear_few_kernel(const LinearParams p, int tiles, int share) {
    constexpr int kColumns = GROUPS ? NT : 8 * NT;                        // (GROUPS: NT counts columns; NVFP4 has one)
    constexpr int kScaleRow = NV ? 8 : 4;                                 // bytes of scales of a row in a piece of 128
    static_assert(!GROUPS || !NV || NT == 1);
    extern __shared__ __align__(16) uint8_t smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, tig = lane & 3;
    const int pitch = x_pitch(p.n_in), columns = p.rows * PIECES, row_bytes = p.n_in >> 1, scale_row = p.n_in / (NV ? 16 : 32);
    const int chunks = (p.n_in + kChunk - 1) / kChunk;
    const bool even = p.n_in % kChunk == 0 && (reinterpret_cast<uintptr_t>(p.scales) & 7u) == 0;     // scales can be copied by words
    uint8_t* ring = smem + columns * pitch + warp * kStages * stage_bytes(NV);
    const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
    float* sums = reinterpret_cast<float*>(smem + columns * pitch + kWarps * kStages * stage_bytes(NV));   // [warp][column][16]
    __shared__ int exponent[16], refs[kWarps][16];

    // `share` warps have a tile in common; this warp's pieces, through all of its tiles
    const int member = warp & (share - 1), team = warp / share, first_tile = team * gridDim.x + blockIdx.x, tile_step = gridDim.x * (kWarps / share);
    const int put_row = lane >> 2, put_at = put_row * kPitch + (lane & 3) * 16;
    int put_tile = first_tile, put_chunk = member;
    const uint8_t *put_codes = nullptr, *put_scales = nullptr;
    bool live0 = false, live1 = false, live_s = false;
    auto begin_tile = [&]() {                  // rows of the tile that there are
        put_chunk = member;
        live0 = put_tile * 16 + put_row < p.n_out;
        live1 = put_tile * 16 + put_row + 8 < p.n_out;
        live_s = lane < 16 && put_tile * 16 + lane < p.n_out;
        put_codes = p.codes + (live0 ? (int64_t)(put_tile * 16 + put_row) * row_bytes + member * (kChunk / 2) + (lane & 3) * 16 : 0);
        put_scales = p.scales + (live_s ? (int64_t)(put_tile * 16 + lane) * scale_row + member * kScaleRow : 0);
    };
    const bool busy = member < chunks;
    if (busy && put_tile < tiles) begin_tile();
    auto issue = [&](int stage) {
        if (busy && put_tile < tiles) {
            const uint32_t at = ring_at + stage * stage_bytes(NV);
            const bool within = put_chunk * kChunk + (lane & 3) * 32 < p.n_in;
            cp_bytes(at + put_at, live0 && within ? put_codes : p.codes, live0 && within ? 16 : 0);
            cp_bytes(at + put_at + 8 * kPitch, live1 && within ? put_codes + 8 * (int64_t)row_bytes : p.codes, live1 && within ? 16 : 0);
            if (lane < 16) {
                if (even) {
                    cp_small<kScaleRow>(at + 16 * kPitch + lane * kScaleRow, put_scales, live_s ? kScaleRow : 0);
                } else {
                    uint8_t* dst = ring + stage * stage_bytes(NV) + 16 * kPitch + lane * kScaleRow;
                    const int have = live_s ? min(kScaleRow, scale_row - put_chunk * kScaleRow) : 0;
                    for (int i = 0; i < kScaleRow; ++i) dst[i] = i < have ? put_scales[i] : (uint8_t)0;
                }
            }
            put_chunk += share;
            put_codes += share * (kChunk / 2);
            if (live_s) put_scales += share * kScaleRow;
            if (put_chunk >= chunks) {
                put_tile += tile_step;
                if (put_tile < tiles) begin_tile();
            }
        }
        asm volatile("cp.async.commit_group;\n" ::);
    };
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) issue(s);

    // ---- x: all threads together, first the rows' largest magnitudes
    __shared__ uint32_t tops[16];
    if (threadIdx.x < 16) tops[threadIdx.x] = 0u;
    __syncthreads();
    const int per_row = p.n_in >> 3, padded = chunks * (kChunk >> 3);
    float row_top = 0.f;                      // of a single row
    for (int i = threadIdx.x; i < p.rows * per_row; i += 32 * kWarps) {
        float v[8], top = 0.f;
        read8(p.x, p.dtype, p.x_vec, (int64_t)i * 8, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) { const float a = fabsf(v[e]); if (a < INFINITY) top = fmaxf(top, a); }
        if (p.rows == 1) row_top = fmaxf(row_top, top);
        else atomicMax(&tops[i / per_row], __float_as_uint(top));
    }
    if (p.rows == 1) {
        const uint32_t all = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(row_top));
        if (lane == 0) atomicMax(&tops[0], all);
    }
    __syncthreads();
    if (threadIdx.x < p.rows) exponent[threadIdx.x] = row_exponent(tops[threadIdx.x]);
    for (int i = threadIdx.x; i < p.rows * padded; i += 32 * kWarps) {
        const int m = i / padded, k = (i - m * padded) * 8;
        const float up = __uint_as_float((uint32_t)(127 + row_exponent(tops[m])) << 23);
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (k < p.n_in) read8(p.x, p.dtype, p.x_vec, (int64_t)m * p.n_in + k, v);
        __half hi[8], lo[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[e] *= up;
            hi[e] = __float2half_rn(v[e]);
            lo[e] = fabsf(v[e]) < INFINITY ? __float2half_rn((v[e] - __half2float(hi[e])) * 2048.f) : __float2half_rn(0.f);
        }
        *reinterpret_cast<uint4*>(smem + m * PIECES * pitch + k * 2) = *reinterpret_cast<uint4*>(hi);
        if (PIECES == 2) *reinterpret_cast<uint4*>(smem + (m * 2 + 1) * pitch + k * 2) = *reinterpret_cast<uint4*>(lo);
    }
    __syncthreads();

    const float glob = p.global_scale != nullptr ? __ldg(p.global_scale) : 1.f;
    const uint8_t* x_at[NT];                  // columns there are not repeat the last one; nothing is made of their sums
#pragma unroll
    for (int n = 0; n < NT; ++n) x_at[n] = smem + min(n * 8 + g, columns - 1) * pitch + tig * 16;
    // GROUPS: the block of 32 in which this lane's column is not zero, and whether it is in this lane's eight values
    const int my_block = NV ? g >> 1 : g & 3, my_column = NV ? 0 : min(g >> 2, columns - 1);
    const bool mine = NV ? (tig >> 1) == (g & 1) : true;
    int stage = 0;
    auto team_sync = [&]() {
        if (share == 1) __syncwarp();
        else asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(32 * share) : "memory");
    };
    for (int tile = first_tile; tile < tiles; tile += tile_step) {
        float acc[NT][4];
        int ref0 = 127, ref1 = 127;                                        // MXFP4: the exponents of rows g and g + 8 that the sums are relative to
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
        for (int chunk = member; chunk < chunks; chunk += share) {
            issue(stage == 0 ? kStages - 1 : stage - 1);
            asm volatile("cp.async.wait_group %0;\n" ::"n"(kStages - 1));
            __syncwarp();
            const uint8_t* w = ring + stage * stage_bytes(NV);
            const uint8_t* sc = w + 16 * kPitch;
            if constexpr (GROUPS) {
                float c[4] = {0.f, 0.f, 0.f, 0.f};
                const uint4 xv = *reinterpret_cast<const uint4*>(smem + my_column * pitch + (chunk * kChunk + my_block * 32 + tig * 8) * 2);
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    uint32_t a[4], d[4];
                    e2m1x8_to_half(*reinterpret_cast<const uint32_t*>(w + g * kPitch + b * 16 + tig * 4), a);
                    e2m1x8_to_half(*reinterpret_cast<const uint32_t*>(w + (g + 8) * kPitch + b * 16 + tig * 4), d);
                    const bool here = mine && b == my_block;
                    mma16816(c, a[0], d[0], a[1], d[1], here ? xv.x : 0u, here ? xv.y : 0u);
                    mma16816(c, a[2], d[2], a[3], d[3], here ? xv.z : 0u, here ? xv.w : 0u);
                }
                // sums of row g (and g + 8) in this lane: groups 2 tig and 2 tig + 1 (MXFP4: modulo four)
                const int at = NV ? 2 * tig : 2 * (tig & 1);
                const uint32_t b0 = *reinterpret_cast<const uint16_t*>(sc + g * kScaleRow + at), b1 = *reinterpret_cast<const uint16_t*>(sc + (g + 8) * kScaleRow + at);
                float2 f0, f1;
                if (NV) {
                    uint32_t h0, h1, unused;
                    e4m3x4_to_half(b0, h0, unused);
                    e4m3x4_to_half(b1, h1, unused);
                    f0 = half2_value(h0);
                    f1 = half2_value(h1);
                } else {
                    const int x0 = b0 & 255u, y0 = b0 >> 8, x1 = b1 & 255u, y1 = b1 >> 8;
                    if (max(x0, y0) > ref0 + 60) {
                        const float fade = relative_power(ref0, max(x0, y0));
                        ref0 = max(x0, y0);
                        acc[0][0] *= fade;
                    }
                    if (max(x1, y1) > ref1 + 60) {
                        const float fade = relative_power(ref1, max(x1, y1));
                        ref1 = max(x1, y1);
                        acc[0][1] *= fade;
                    }
                    const float nan = __uint_as_float(0x7FC00000u);
                    f0 = make_float2(x0 == 255 ? nan : relative_power(x0, ref0), y0 == 255 ? nan : relative_power(y0, ref0));
                    f1 = make_float2(x1 == 255 ? nan : relative_power(x1, ref1), y1 == 255 ? nan : relative_power(y1, ref1));
                }
                acc[0][0] = fmaf(c[0], f0.x, fmaf(c[1], f0.y, acc[0][0]));
                acc[0][1] = fmaf(c[2], f1.x, fmaf(c[3], f1.y, acc[0][1]));
            } else {
                uint2 s0, s1;
                if (NV) {
                    s0 = *reinterpret_cast<const uint2*>(sc + g * 8);
                    s1 = *reinterpret_cast<const uint2*>(sc + (g + 8) * 8);
                } else {
                    s0.x = *reinterpret_cast<const uint32_t*>(sc + g * 4);
                    s1.x = *reinterpret_cast<const uint32_t*>(sc + (g + 8) * 4);
                    // the largest of the four, as long as none is far above the reference
                    const uint32_t t0 = __vmaxu4(s0.x, s0.x >> 16), t1 = __vmaxu4(s1.x, s1.x >> 16);
                    const int top0 = max(t0 & 255u, (t0 >> 8) & 255u), top1 = max(t1 & 255u, (t1 >> 8) & 255u);
                    if (top0 > ref0 + 60) {
                        const float fade = relative_power(ref0, top0);
                        ref0 = top0;
#pragma unroll
                        for (int n = 0; n < NT; ++n) { acc[n][0] *= fade; acc[n][1] *= fade; }
                    }
                    if (top1 > ref1 + 60) {
                        const float fade = relative_power(ref1, top1);
                        ref1 = top1;
#pragma unroll
                        for (int n = 0; n < NT; ++n) { acc[n][2] *= fade; acc[n][3] *= fade; }
                    }
                }
                const int k0 = chunk * kChunk;
                float part[NT][4];                                         // NVFP4: of this piece
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    uint32_t a[4], d[4];
                    e2m1x8_to_half(*reinterpret_cast<const uint32_t*>(w + g * kPitch + b * 16 + tig * 4), a);
                    e2m1x8_to_half(*reinterpret_cast<const uint32_t*>(w + (g + 8) * kPitch + b * 16 + tig * 4), d);
                    uint4 x[NT];
#pragma unroll
                    for (int n = 0; n < NT; ++n) x[n] = *reinterpret_cast<const uint4*>(x_at[n] + (k0 + b * 32) * 2);
                    if (NV) {
                        const uint32_t sel = 0x11u * (2 * (b & 1) + (tig >> 1));     // this lane's byte, twice
                        uint32_t h0, h1, unused;
                        e4m3x4_to_half(__byte_perm(b < 2 ? s0.x : s0.y, 0u, sel), h0, unused);
                        e4m3x4_to_half(__byte_perm(b < 2 ? s1.x : s1.y, 0u, sel), h1, unused);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            a[i] = times(a[i], *reinterpret_cast<__half2*>(&h0));
                            d[i] = times(d[i], *reinterpret_cast<__half2*>(&h1));
                        }
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            if (b == 0) mma16816_first(part[n], a[0], d[0], a[1], d[1], x[n].x, x[n].y);
                            else mma16816(part[n], a[0], d[0], a[1], d[1], x[n].x, x[n].y);
                            mma16816(part[n], a[2], d[2], a[3], d[3], x[n].z, x[n].w);
                        }
                    } else {
                        const int e0 = (s0.x >> (8 * b)) & 255u, e1 = (s1.x >> (8 * b)) & 255u;
                        const float f0 = e0 == 255 ? __uint_as_float(0x7FC00000u) : relative_power(e0, ref0);
                        const float f1 = e1 == 255 ? __uint_as_float(0x7FC00000u) : relative_power(e1, ref1);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            float c[4];
                            mma16816_first(c, a[0], d[0], a[1], d[1], x[n].x, x[n].y);
                            mma16816(c, a[2], d[2], a[3], d[3], x[n].z, x[n].w);
                            acc[n][0] = fmaf(c[0], f0, acc[n][0]);
                            acc[n][1] = fmaf(c[1], f0, acc[n][1]);
                            acc[n][2] = fmaf(c[2], f1, acc[n][2]);
                            acc[n][3] = fmaf(c[3], f1, acc[n][3]);
                        }
                    }
                }
                if (NV) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[n][i] += part[n][i];
                }
            }
            __syncwarp();
            if (++stage == kStages) stage = 0;
        }
        // ---- the warps' sums
        if constexpr (GROUPS) {
            // the lanes of a row (MXFP4: of a row and column) hold parts of one sum, with exponents of their own
            if (!NV) {
                const int top0 = max(ref0, __shfl_xor_sync(0xFFFFFFFFu, ref0, 1)), top1 = max(ref1, __shfl_xor_sync(0xFFFFFFFFu, ref1, 1));
                const int all0 = max(top0, __shfl_xor_sync(0xFFFFFFFFu, top0, 2)), all1 = max(top1, __shfl_xor_sync(0xFFFFFFFFu, top1, 2));
                acc[0][0] *= relative_power(ref0, all0);
                acc[0][1] *= relative_power(ref1, all1);
                ref0 = all0;
                ref1 = all1;
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float v = acc[0][i];
                    v += __shfl_xor_sync(0xFFFFFFFFu, v, 1);
                    if (NV) v += __shfl_xor_sync(0xFFFFFFFFu, v, 2);
                    if (NV ? tig == 0 : tig == 2 * n) sums[(warp * NT + n) * 16 + g + 8 * i] = v;
                }
        } else {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) sums[(warp * 8 * NT + n * 8 + 2 * tig + (i & 1)) * 16 + g + 8 * (i >> 1)] = acc[n][i];
        }
        if (!NV && tig == 0) { refs[warp][g] = ref0; refs[warp][g + 8] = ref1; }
        team_sync();
        for (int i = member * 32 + lane; i < p.rows * 16; i += 32 * share) {
            const int m = i >> 4, r = i & 15, n = tile * 16 + r;
            int ref = 127;
            if (!NV)
                for (int w = team * share; w < team * share + share; ++w) ref = max(ref, refs[w][r]);
            float v = 0.f, v2 = 0.f;
            for (int w = team * share; w < team * share + share; ++w) {
                const float f = NV ? 1.f : relative_power(refs[w][r], ref);
                v = fmaf(sums[(w * kColumns + m * PIECES) * 16 + r], f, v);
                if (PIECES == 2) v2 = fmaf(sums[(w * kColumns + m * 2 + 1) * 16 + r], f, v2);
            }
            if (PIECES == 2) v = fmaf(v2, 0x1p-11f, v);
            if (n < p.n_out) {
                v = scale_by_power(v, (NV ? 0 : ref - 127) - exponent[m]) * glob;
                if (p.bias != nullptr) v += load_value(p.bias, p.dtype, n);
                store_value(p.y, p.dtype, (int64_t)m * p.n_out + n, v);
            }
        }
        team_sync();
    }
    asm volatile("cp.async.wait_group 0;\n" ::);
}

template <bool NV, int PIECES, int NT, bool GROUPS>
int launch_few(const LinearParams& p, cudaStream_t st) {
    const int bytes = few_smem(p.rows * PIECES * x_pitch(p.n_in), NV, NT), tiles = (p.n_out + 15) / 16;
    constexpr auto kern = block_linear_few_kernel<NV, PIECES, NT, GROUPS>;
    if (!allow_shared<kern>(kMostShared)) return check_launch("block_linear");
    // One CTA on each SM.  As many warps share a tile as take the least time: rounds of tiles times pieces of a warp, with two for the
    // end.  One row, MXFP4: 4096 by 4096 takes 10 us with eight that share, 19 where none do and 11 where all sixteen do; 768 by 50257
    // 14, 14 and 46; 8192 by 28672 50, 50 and 64.
    const int chunks = (p.n_in + kChunk - 1) / kChunk;
    int share = 1;
    int64_t least = -1;
    for (int s = 1; s <= kWarps; s *= 2) {
        const int64_t at_once = (int64_t)sm_count() * (kWarps / s), rounds = (tiles + at_once - 1) / at_once * ((chunks + s - 1) / s + 2);
        if (least < 0 || rounds < least) { least = rounds; share = s; }
    }
    kern<<<(unsigned)(tiles < sm_count() ? tiles : sm_count()), 32 * kWarps, bytes, st>>>(p, tiles, share);
    return check_launch("block_linear");
}

// Few rows: at most 16 columns (a float32 row takes two), x within the shared memory beside the rings.  This kernel against the tiles',
// 4096 by 11008, NVFP4, bfloat16: one row 13 and 28 us, eight 19 and 30, sixteen 28 and 32; MXFP4, float32, eight rows 28 and 35.
// More columns would need another set of sums for each eight, and 24 rows take the tiles 33.
bool few_rows(int64_t rows, int64_t n_in, int dtype) {
    const int64_t columns = rows * (dtype == MPT_DTYPE_F32 ? 2 : 1);
    return columns <= 16 && n_in <= 65536 && columns * x_pitch((int)n_in) <= kMostX;
}

}  // namespace
}  // namespace mpt

using namespace mpt;

extern "C" {

size_t mpt_block_linear_workspace_bytes(int64_t rows, int64_t n_out, int64_t n_in, int format, int dtype) {
    if (rows <= 0 || n_out <= 0 || n_in < 0 || rows > 0x7FFFFFFF || n_out > 0x7FFFFFFF || n_in > 0x7FFFFFFF || few_rows(rows, n_in, dtype)) return 0;
    return tiles_plan(rows, n_out, n_in, format, dtype).bytes;
}

int mpt_block_linear(const void* x, const uint8_t* codes, const uint8_t* scales, const float* global_scale, const void* bias, void* y,
                     int64_t rows, int64_t n_out, int64_t n_in, int format, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
    MPT_REQUIRE(rows >= 0 && n_out >= 0 && n_in >= 0 && rows <= 0x7FFFFF00 && n_out <= 0x7FFFFF00 && n_in <= 0x3FFFFF00, "block_linear: bad extents");
    MPT_REQUIRE(n_in % 32 == 0, "block_linear: n_in %lld is not a multiple of 32", (long long)n_in);
    MPT_REQUIRE(format == MPT_BLOCK_MXFP4 || format == MPT_BLOCK_NVFP4, "block_linear: unknown format %d", format);
    MPT_REQUIRE(dtype == MPT_DTYPE_F32 || dtype == MPT_DTYPE_BF16 || dtype == MPT_DTYPE_F16, "block_linear: unknown data type %d", dtype);
    if (rows == 0 || n_out == 0) return MPT_OK;
    MPT_REQUIRE(y && (n_in == 0 || (x && codes && scales)), "block_linear: null pointer");
    MPT_REQUIRE(((uintptr_t)codes & 15u) == 0, "block_linear: the codes must begin at a multiple of 16 bytes");
    MPT_REQUIRE(format != MPT_BLOCK_NVFP4 || ((uintptr_t)scales & 1u) == 0, "block_linear: NVFP4 scales must begin at an even address");
    LinearParams p{x, codes, scales, global_scale, bias, y, dtype, (int)rows, (int)n_out, (int)n_in, ((uintptr_t)x & 15u) == 0};
    cudaStream_t st = as_stream(stream);
    if (few_rows(rows, n_in, dtype)) {
        const bool nv = format == MPT_BLOCK_NVFP4;
        const int columns = (int)rows * (dtype == MPT_DTYPE_F32 ? 2 : 1);
        if (dtype == MPT_DTYPE_F32) {
            if (columns == 2 && !nv) return launch_few<false, 2, 2, true>(p, st);
            if (columns <= 8) return nv ? launch_few<true, 2, 1, false>(p, st) : launch_few<false, 2, 1, false>(p, st);
            return nv ? launch_few<true, 2, 2, false>(p, st) : launch_few<false, 2, 2, false>(p, st);
        }
        if (columns == 1) return nv ? launch_few<true, 1, 1, true>(p, st) : launch_few<false, 1, 1, true>(p, st);
        if (columns == 2 && !nv) return launch_few<false, 1, 2, true>(p, st);
        if (columns <= 8) return nv ? launch_few<true, 1, 1, false>(p, st) : launch_few<false, 1, 1, false>(p, st);
        return nv ? launch_few<true, 1, 2, false>(p, st) : launch_few<false, 1, 2, false>(p, st);
    }
    const TilesPlan pl = tiles_plan(rows, n_out, n_in, format, dtype);
    if (workspace_bytes < pl.bytes || !workspace || ((uintptr_t)workspace & 255u)) {
        set_error("block_linear: a workspace of %zu bytes at a multiple of 256 is needed", pl.bytes);
        return MPT_ERR_WORKSPACE;
    }
    return launch_tiles(p, pl, format, static_cast<uint8_t*>(workspace), st);
}

}
