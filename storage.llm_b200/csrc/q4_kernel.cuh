// Matrix-vector products with 4-bit weights and group scales:
//   y[r, n] = sum_g scale[n, g] sum_{k in g} value(code[n, k]) x[r, k]
// for one matrix, or by expert over the batches of the token sort (the row of
// x gathered on the way), with the gated activation of two products where a
// matrix holds gate and up rows.
//
// The floor is reading the codes and scales once.  At that rate an SM gets 46
// codes a clock and issues 128 lane instructions, so what counts is
// instructions per code: the products go to the matrix unit (m16n8k16, 16 rows
// of the matrix by 8 columns, one an instruction for 8 codes of each lane)
// even for a single row of x, each code is decoded once, two at a time, and
// everything about x is done before the loop.
//   * A block takes 16 * MT rows of one matrix, its warps every so many slices
//     of 128 columns.  Each warp streams its slices through its own ring in
//     shared memory with 16-byte asynchronous copies and meets the others once,
//     to join their sums.  Many small blocks on an SM cover each other's
//     beginnings and ends.
//   * fp32 x is cut into three bf16 terms that add up to it exactly.  One or two
//     rows of it fill up to six of the unit's eight columns, which cost nothing;
//     more rows take three tiles of columns, one a term, so that a lane makes
//     the three terms of one row from one load.  x comes straight from the first
//     cache; rows that are not aligned go through shared memory.
//   * The order of the columns inside a group does not matter as long as the
//     matrix and x agree.  The four lanes of a quad take consecutive words of
//     a row's codes inside one group, whose scale is applied to the group's
//     fp32 sum (E8M0 scales to the decoded values, which stays exact).
//   * Both codes decode exactly to bf16: integers as subnormals (c 2^-133),
//     E2M1 magnitudes shifted onto exponent and mantissa (v 2^-126); one fused
//     multiply-add brings either into range and takes the zero point off.
// Measured, with the share of a copy's 6.55 TB/s and what bounds it:
//   131,072 x 7168 integers by 128, 4 rows           110 us, 69 %   instructions
//   64 rows of 256 gated MXFP4 experts 2 x 2048 x 7168   225 us, 61 %   instructions and
//       their latency: 17 decode 8 codes; on 131,072 x 7168 one row's 99 million
//       are 90 us at full issue, 134 us as measured, with 16 warps an SM
//   128 fp32 rows of 32 MXFP4 experts 2880 x 2880     75 us, 29 %   instructions: the three
//       terms cost a third of a slice's; blocks of 9 to 16 rows go twice
//   7168 x 2048 MXFP4, one row                         5.1 us        launch and latency
//   131,072 x 7168 integers, 32 rows                 337 us, 22 %   latency: four tiles of
//       sums leave registers for 8 warps an SM
//   rows of x off 16-byte boundaries (staged in shared memory, one launch shape):
//       7168 x 2048 one row 6.3 us for 5.3, 131,072 x 7168 one row 180 for 135,
//       16,384 x 4096 8 bf16 rows 48 for 15, 4 fp32 rows 119 for 20
//   few outputs: 256 x 8192, one row 6.3 us on 16 SMs; 32 fp32 rows 46 us, four
//       passes one after the other on 8
// Slower, each by its measured time: blocks that stay for several tiles (their
// beginnings and ends no longer cover each other), warps with rows of their own
// and all columns (32 rows: 380 us), 128 registers for four tiles (479 us).
#pragma once

#include "op_common.cuh"

namespace moe_b200 {

// The launch shape a call takes (see q4_plan).
struct Q4Plan {
    int mt, nt;
    uint32_t batches, warps, smem;
    int device;
};

struct Q4Job {
    uint32_t N, K, group, groups;   // outputs, columns, columns of a scale, scales of a row
    uint32_t experts, tokens, out_rows, top_k;
    uint64_t x_stride, y_stride;
    const uint8_t* codes;
    const void* scales;
    const uint8_t* zeros;
    const void* x;
    const moe_b200_batch_t* batches;
    const uint32_t* batch_count;
    const uint32_t* perm;
    void* y;
    uint32_t* err;
    int scale_type, x_type, y_type, code, gated, act;
    int x_vec;                      // rows of x on 16-byte boundaries
    // where x goes through shared memory: its rows held at once, and of their
    // slices those of so many turns of the warps
    uint32_t pass_rows, pass_turns;
};

cudaError_t launch_q4_e2m1(const Q4Job& job, const Q4Plan& plan, cudaStream_t st);
cudaError_t launch_q4_int4(const Q4Job& job, const Q4Plan& plan, cudaStream_t st);

namespace {

__device__ __forceinline__ float scale_of_bits(int type, uint32_t s) {
    switch (type) {
        case MOE_B200_DTYPE_E8M0: return __uint_as_float(s ? s << 23 : 0x00400000u);
        case MOE_B200_DTYPE_BF16: return __uint_as_float(s << 16);
        case MOE_B200_DTYPE_F16: return __half2float(__ushort_as_half((unsigned short)s));
        default: return __uint_as_float(s);
    }
}

__device__ __forceinline__ float activate(int act, float g) {
    if (act == MOE_B200_ACT_GELU_ERF) return 0.5f * g * (1.0f + erff(g * 0.70710678118654752440f));
    if (act == MOE_B200_ACT_GELU_TANH)
        return 0.5f * g * (1.0f + tanhf(0.7978845608028654f * fmaf(0.044715f * g * g, g, g)));
    return g / (1.0f + expf(-g));
}

// A group's sum before its scale could leave fp32's range where the scaled one
// does not (128 columns of 255 |x| at most), so the weights' values enter 2^16
// smaller, which is exact, and the scale 2^16 larger, or the sum where the
// scale itself has no room.
constexpr float kGrow = 65536.0f;
__device__ __forceinline__ float add_scaled(float scale, float part, float acc) {
    return fabsf(scale) < 1e18f ? fmaf(scale * kGrow, part, acc) : fmaf(scale, part * kGrow, acc);
}

// ---------------------------------------------------------------------------
// Decoding: 8 codes of a word to four bf16 pairs, pair i = codes i and i + 4.
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint32_t hfma2_bf16(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}
// Integers minus the zero point, 2^-16 of them; `zero` = -z 2^-16 twice.  An
// integer below 256 in the low bits of a bf16 is that integer times 2^-133,
// so a code may also stay four bits up.
__device__ __forceinline__ void decode_int4(uint32_t w, uint32_t zero, uint32_t (&p)[4]) {
    const uint32_t v = w >> 8;
    p[0] = hfma2_bf16(w & 0x000f000fu, 0x7a007a00u /* 2^117 */, zero);
    p[1] = hfma2_bf16(w & 0x00f000f0u, 0x78007800u /* 2^113 */, zero);
    p[2] = hfma2_bf16(v & 0x000f000fu, 0x7a007a00u, zero);
    p[3] = hfma2_bf16(v & 0x00f000f0u, 0x78007800u, zero);
}
// E2M1 values times `unit` 2^-126.  A product makes two copies of a code, one
// with its magnitude on bits 6-8 (the value times 2^-126), one with its sign
// on bit 15.  -0 added leaves the sign of a zero alone.
__device__ __forceinline__ void decode_e2m1(uint32_t w, uint32_t unit, uint32_t (&p)[4]) {
    const uint32_t v = w >> 8;
    p[0] = hfma2_bf16(((w & 0x000f000fu) * 0x1040u) & 0x81c081c0u, unit, 0x80008000u);
    p[1] = hfma2_bf16(((w & 0x00f000f0u) * 0x0104u) & 0x81c081c0u, unit, 0x80008000u);
    p[2] = hfma2_bf16(((v & 0x000f000fu) * 0x1040u) & 0x81c081c0u, unit, 0x80008000u);
    p[3] = hfma2_bf16(((v & 0x00f000f0u) * 0x0104u) & 0x81c081c0u, unit, 0x80008000u);
}
constexpr uint32_t kUnitE2M1 = 0x76807680u;  // 2^110: v 2^-126 becomes v 2^-16

__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0)
                 : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

constexpr int kSlice = 128;            // columns of one stage: 64 bytes a row
constexpr int kRowBytes = kSlice / 2;
template <int MT>
constexpr int kDepth = MT == 1 ? 4 : (MT == 2 ? 3 : 2);  // stages of a warp's ring
template <int MT>
constexpr uint32_t kMostWarps = MT == 1 ? 16 : 8;
// Blocks of the most warps that an SM's registers have to hold.
template <int MT, int NT>
constexpr int kBlocksPerSm = NT == 4 ? 1 : (MT == 2 && NT == 1 ? 3 : 2);

// Shared memory of a block: the warps' rings, later their sums; x of `slices`
// slices by word and column.
__host__ __device__ constexpr uint32_t ring_bytes(int mt) {
    return (mt == 1 ? 4 : (mt == 2 ? 3 : 2)) * mt * 16 * kRowBytes;
}
__host__ __device__ constexpr uint32_t x_bytes(uint32_t slices, uint32_t cols) { return slices * kSlice * cols * 2; }
constexpr uint32_t kMaxPassRows = 32;
constexpr uint32_t kMostSmem = 226 * 1024;

// 8 bf16 values as pairs (i, i + 4), the order in which decode_* gives a word's
// codes.
__device__ __forceinline__ uint4 bf16_pairs(uint4 v) {
    return make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410),
                      __byte_perm(v.y, v.w, 0x7632));
}
// 8 fp32 values' upper halves, of what is left of them without the terms that
// the masks take off (upper half by upper half), as such pairs.
__device__ __forceinline__ uint4 f32_pairs(const float* p, uint32_t m1, uint32_t m2) {
    float v[8];
    load_f32<8>(p, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        v[i] -= __uint_as_float(__float_as_uint(v[i]) & m1);
        v[i] -= __uint_as_float(__float_as_uint(v[i]) & m2);
    }
    auto pair = [&](int i) { return __byte_perm(__float_as_uint(v[i]), __float_as_uint(v[i + 4]), 0x7632); };
    return make_uint4(pair(0), pair(1), pair(2), pair(3));
}
// All three terms of 8 fp32 values.
__device__ __forceinline__ void f32_terms(const float* p, uint4 (&x)[3]) {
    float v[8];
    load_f32<8>(p, v);
#pragma unroll
    for (int term = 0; term < 3; ++term) {
        auto pair = [&](int i) { return __byte_perm(__float_as_uint(v[i]), __float_as_uint(v[i + 4]), 0x7632); };
        x[term] = make_uint4(pair(0), pair(1), pair(2), pair(3));
        if (term == 2) break;
        float upper[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) upper[i] = __uint_as_float((__float_as_uint(v[i]) & 0xffff0000u) ^ 0x80000000u);
        vadd<8>(v, upper);
    }
}
// 8 values of x (term `term` of fp32 ones) as such pairs, from any address.
__device__ __forceinline__ uint4 any_pairs(const Q4Job& job, uint64_t at, uint32_t term) {
    uint32_t v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (job.x_type == MOE_B200_DTYPE_F32) {
            float f = __ldg(static_cast<const float*>(job.x) + at + i);
            if (term >= 1) f -= __uint_as_float(__float_as_uint(f) & 0xffff0000u);
            if (term == 2) f -= __uint_as_float(__float_as_uint(f) & 0xffff0000u);
            v[i] = __float_as_uint(f) >> 16;
        } else {
            v[i] = __ldg(static_cast<const uint16_t*>(job.x) + at + i);
        }
    }
    return make_uint4(v[0] | v[4] << 16, v[1] | v[5] << 16, v[2] | v[6] << 16, v[3] | v[7] << 16);
}

// The scale's type in memory, and 2^16 times a scale from its bits; `odd` where
// that leaves fp32's range.
template <int ST>
struct ScaleOf {
    using type = uint16_t;
};
template <>
struct ScaleOf<MOE_B200_DTYPE_E8M0> {
    using type = uint8_t;
};
template <>
struct ScaleOf<MOE_B200_DTYPE_F32> {
    using type = uint32_t;
};
template <int ST>
__device__ __forceinline__ float grown_scale(uint32_t s, bool& odd) {
    if constexpr (ST == MOE_B200_DTYPE_E8M0) {
        odd |= s - 1u >= 238u;
        return __uint_as_float((s + 16u) << 23);
    } else {
        const float f = scale_of_bits(ST, s) * kGrow;
        odd |= !(fabsf(f) < 3e38f);
        return f;
    }
}
template <int ST>
__device__ __forceinline__ float true_scale(const Q4Job& job, uint64_t i) {
    return scale_of_bits(ST, __ldg(static_cast<const typename ScaleOf<ST>::type*>(job.scales) + i));
}

// One product in plain fp32: for fp32 x with infinities or NaN, whose terms
// would meet as inf - inf.
__device__ __noinline__ float plain_dot(const Q4Job& job, uint64_t row, uint64_t xr) {
    float acc = 0.0f;
    for (uint32_t g = 0; g < job.groups; ++g) {
        const uint64_t s = row * job.groups + g;
        const float z = job.zeros ? (float)job.zeros[s] : 8.0f;
        float part = 0.0f;
        for (uint32_t i = 0; i < job.group; ++i) {
            const uint32_t k = g * job.group + i;
            const uint32_t c = job.codes[row * (job.K / 2) + k / 2] >> (4 * (k & 1)) & 15;
            float v = (float)c - z;
            if (job.code == MOE_B200_Q4_E2M1) {
                const uint32_t m = c & 7;
                v = m < 2 ? 0.5f * (float)m : __uint_as_float(((m >> 1) + 126) << 23 | (m & 1) << 22);
                v = c & 8 ? -v : v;
            }
            part = fmaf(v / kGrow, static_cast<const float*>(job.x)[xr * job.x_stride + k], part);
        }
        float scale;
        switch (job.scale_type) {
            case MOE_B200_DTYPE_E8M0: scale = true_scale<MOE_B200_DTYPE_E8M0>(job, s); break;
            case MOE_B200_DTYPE_F32: scale = true_scale<MOE_B200_DTYPE_F32>(job, s); break;
            case MOE_B200_DTYPE_F16: scale = true_scale<MOE_B200_DTYPE_F16>(job, s); break;
            default: scale = true_scale<MOE_B200_DTYPE_BF16>(job, s); break;
        }
        acc = add_scaled(scale, part, acc);
    }
    return acc;
}

// CODE, G, ST: the weights.  With E2M1 codes and E8M0 scales of 32 (MXFP4) the
// scales are multiplied into the decoded values (FOLD).  MT: tiles of 16 rows
// (gated: half of them gate, half up rows); NT: tiles of 8 columns; XM: how x
// comes.
enum XMode { kXBf16, kXF32, kXStaged };
template <int CODE, int G, int ST, int MT, int NT, int XM>
__global__ void __launch_bounds__(kMostWarps<MT> * 32, (kBlocksPerSm<MT, NT>))
    q4_kernel(const __grid_constant__ Q4Job job) {
    constexpr bool FOLD = CODE == MOE_B200_Q4_E2M1 && ST == MOE_B200_DTYPE_E8M0 && G == 32;
    constexpr int DEPTH = kDepth<MT>;
    constexpr bool XS = XM == kXStaged, XF32 = XM == kXF32;
    // tile nt holds term nt of 8 rows of x; the upper term's sums are kept apart
    // from those of the other two, whose share in the rounding is 2^-8
    constexpr bool BY_TERM = XF32 && NT == 3;
    constexpr int NA = BY_TERM ? 1 : NT;  // tiles of sums
    constexpr int GPS = kSlice / G;  // groups of a stage
    constexpr int WPG = G / 32;      // words of a lane in a group and row
    constexpr uint32_t ROWS = MT * 16;
    using Scale = typename ScaleOf<ST>::type;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ uint32_t pass_x_row[kMaxPassRows];  // row of x of the pass' rows; tokens: none
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const uint32_t g = lane >> 2, c = lane & 3;
    const uint32_t slices = ceil_div(job.K, (uint32_t)kSlice);
    const uint32_t terms = XF32 || (XS && job.x_type == MOE_B200_DTYPE_F32) ? 3 : 1;
    uint8_t* ring = smem + warp * ring_bytes(MT);
    uint4* xs = reinterpret_cast<uint4*>(smem + warps * ring_bytes(MT));  // [word][column][c]

    pdl_wait();
    uint32_t expert = 0, first = 0, count = job.tokens;
    if (job.batches) {
        const uint32_t batches = *job.batch_count;
        if (batches > gridDim.y && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0)
            record_error(job.err, kErrBadBatch);  // more than there can be
        if (blockIdx.y >= batches) return;
        const moe_b200_batch_t b = job.batches[blockIdx.y];
        expert = b.expert, first = b.first_sorted_index, count = b.token_count;
        if (expert >= job.experts || first > job.out_rows || count > job.out_rows - first) {
            record_error(job.err, kErrBadBatch);
            return;
        }
    }
    const uint32_t tiles = job.gated ? MT / 2 : MT;  // of outputs
    const uint32_t out_rows = tiles * 16;
    const uint32_t n0 = blockIdx.x * out_rows;
    const uint64_t gate_row = (uint64_t)expert * job.N * (job.gated ? 2 : 1) + n0, up_row = gate_row + job.N;
    const uint32_t row_bytes = job.K / 2;
    auto is_up = [&](int mt) { return job.gated && mt >= (int)tiles; };
    // row g + 8 h of tile mt, counted from the block's first; past the last
    // output, the last one again (not stored)
    auto tile_row = [&](int mt, int h) {
        return min((is_up(mt) ? mt - tiles : mt) * 16 + g + 8 * h, job.N - 1 - n0);
    };

    // Copies: lane (g, c) brings 16 bytes c of the rows g and g + 8 of each tile.
    // The ring's 64-byte rows are stored with their 16-byte pieces exchanged by
    // row, so that reads of 4, 8 or 16 bytes of 8 rows meet all banks evenly.
    const uint32_t swz = (g & 2) | (g >> 2);
    const uint32_t dst = smem_u32(ring) + g * kRowBytes + ((c ^ swz) << 4);
    uint32_t code_off[MT][2], scale_off[MT][2];  // from the block's first row
#pragma unroll
    for (int i = 0; i < MT * 2; ++i) {
        code_off[i / 2][i & 1] = tile_row(i / 2, i & 1) * row_bytes + c * 16;
        scale_off[i / 2][i & 1] = tile_row(i / 2, i & 1) * job.groups;
    }
    auto copy = [&](uint32_t slice, uint32_t slot) {
        if (slice < slices) {
            const uint32_t at = slice * kRowBytes;
            const bool real = at + c * 16 < row_bytes;  // a last slice of fewer columns
            const uint8_t* gate = job.codes + gate_row * row_bytes + at;
            const uint8_t* up = job.codes + up_row * row_bytes + at;
#pragma unroll
            for (int i = 0; i < MT * 2; ++i)
                cp_async16(dst + slot * (ROWS * kRowBytes) + i * (8 * kRowBytes),
                           (is_up(i / 2) ? up : gate) + (real ? code_off[i / 2][i & 1] : 0u), real);
        }
        cp_async_commit();
    };
    // Scales of the rows g and g + 8 of each tile: lane c of a quad holds group
    // c % GPS of the slice.
    uint32_t sbits[MT][2], zbits[MT][2];
    auto fetch_scales = [&](uint32_t slice) {
        const uint32_t q = min(slice * GPS + (c % GPS), job.groups - 1);
#pragma unroll
        for (int i = 0; i < MT * 2; ++i) {
            const uint64_t base = (is_up(i / 2) ? up_row : gate_row) * job.groups;
            const uint32_t off = scale_off[i / 2][i & 1] + q;
            sbits[i / 2][i & 1] = __ldg(static_cast<const Scale*>(job.scales) + base + off);
            zbits[i / 2][i & 1] = 8;
            if (CODE == MOE_B200_Q4_INT4 && job.zeros) zbits[i / 2][i & 1] = __ldg(job.zeros + base + off);
        }
    };
    auto x_row = [&](uint32_t r) -> uint32_t {  // row of x of the batch's row r; >= tokens: none
        return job.perm ? __ldg(job.perm + first + r) / job.top_k : first + r;
    };

    const uint32_t turns = ceil_div(slices, warps);  // slices of a warp
    const uint32_t pass_rows = XS ? job.pass_rows : (BY_TERM ? 8 : (XF32 ? NT * 8 / 3 : NT * 8));
    for (uint32_t r0 = 0; r0 < count; r0 += pass_rows) {
        const uint32_t rows = min(pass_rows, count - r0), cols = rows * terms;
#pragma unroll
        for (int d = 0; d < DEPTH - 1; ++d) copy(warp + d * warps, d);
        fetch_scales(warp);
        for (uint32_t r = threadIdx.x; r < rows; r += blockDim.x) {
            const uint32_t xr = x_row(r0 + r);
            pass_x_row[r] = min(xr, job.tokens);
            if (xr >= job.tokens) record_error(job.err, kErrBadBatch);
        }
        __syncthreads();
        // x of the slices from turn t0 on, while copies are on their way
        auto stage_x = [&](uint32_t t0) {
            const uint32_t s0 = t0 * warps, s1 = min(slices, s0 + job.pass_turns * warps);
            for (uint32_t i = threadIdx.x; i < (s1 - s0) * 4 * cols * 4; i += blockDim.x) {
                const uint32_t lc = i & 3, col = (i >> 2) % cols, word = s0 * 4 + (i >> 2) / cols;
                const uint32_t k = word / WPG * G + (lc * WPG + word % WPG) * 8;
                const uint32_t xr = pass_x_row[col / terms];
                xs[i] = k < job.K && xr < job.tokens ? any_pairs(job, xr * job.x_stride + k, col % terms)
                                                     : make_uint4(0, 0, 0, 0);
            }
            __syncthreads();
        };
        // a column that the pass does not have reads column 0 and is not stored
        uint32_t xcol[NT];
        const uint8_t* xrow[NT];
        uint32_t m1[NT], m2[NT];  // fp32: which term of x the column takes
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const uint32_t col = BY_TERM ? (g < rows ? g * 3 : 0) : (nt * 8 + g < cols ? nt * 8 + g : 0);
            if constexpr (XS) {
                xcol[nt] = col * 4 + c;
            } else {
                constexpr uint32_t size = XF32 ? 4 : 2;
                const uint32_t xr = pass_x_row[col / terms];
                xrow[nt] = static_cast<const uint8_t*>(job.x) + (xr < job.tokens ? xr : 0) * job.x_stride * size +
                           (c * (8 * WPG) + warp * kSlice) * size;  // of the warp's slice
                m1[nt] = col % terms >= 1 ? 0xffff0000u : 0u, m2[nt] = col % terms == 2 ? 0xffff0000u : 0u;
            }
        }
        float acc[MT][NA][4] = {}, lower[BY_TERM ? MT : 1][4] = {};
        uint32_t slot = 0;
        for (uint32_t turn = 0, slice = warp; turn < turns; ++turn, slice += warps) {
            if (slice >= slices && !XS) break;
            if (XS && turn % job.pass_turns == 0) {
                if (turn) __syncthreads();  // what is there has been read
                stage_x(turn);
            }
            if (slice >= slices) continue;
            // unit: what the decoding multiplies by (FOLD) or adds (integers);
            // grown: the scale times 2^16
            uint32_t unit[MT][2];
            float grown[MT][2];
            bool odd = false;  // some scale needs the careful way
#pragma unroll
            for (int i = 0; i < MT * 2; ++i) {
                const uint32_t s = sbits[i / 2][i & 1];
                if constexpr (FOLD) {
                    // 2^(s - 127 + 126) as bf16 twice; a scale above 2 is past its range
                    odd |= s > 128u;
                    unit[i / 2][i & 1] = (s + 126u) * 0x00800080u;
                } else {
                    grown[i / 2][i & 1] = grown_scale<ST>(s, odd);
                }
                if constexpr (CODE == MOE_B200_Q4_INT4)
                    unit[i / 2][i & 1] = hfma2_bf16(zbits[i / 2][i & 1] * 0x00010001u, 0xfa00fa00u /* -2^117 */, 0);
            }
            odd = __any_sync(0xffffffffu, odd);
            // x of the slice, before the wait for its codes
            const uint4* xw = xs + (slice - (XS ? turn / job.pass_turns * job.pass_turns * warps : 0u)) * 16 * cols;
            const uint32_t here = min((uint32_t)GPS, job.groups - slice * GPS);  // groups of the slice
            const bool full = here == GPS;
            constexpr bool EARLY = XM == kXBf16 && NT == 1;
            auto bf16_x = [&](int w, int nt) {
                return __ldg(reinterpret_cast<const uint4*>(xrow[nt] + (w / WPG * G + w % WPG * 8) * 2));
            };
            uint4 x_early[EARLY ? 4 : 1] = {};
            if constexpr (EARLY) {
                if (full) {
#pragma unroll
                    for (int w = 0; w < 4; ++w) x_early[w] = bf16_x(w, 0);
                } else {
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        if ((uint32_t)(w / WPG) < here) x_early[w] = bf16_x(w, 0);
                    }
                }
            }
            cp_async_wait<DEPTH - 2>();
            __syncwarp();
            copy(slice + (DEPTH - 1) * warps, slot == 0 ? DEPTH - 1 : slot - 1);
            if (slice + warps < slices) fetch_scales(slice + warps);
            const uint8_t* stage = ring + slot * (ROWS * kRowBytes) + g * kRowBytes;
            slot = slot + 1 == DEPTH ? 0 : slot + 1;
            auto load_x = [&](int word, int nt) {
                if constexpr (XS) return xw[word * 4 * cols + xcol[nt]];
                else if constexpr (EARLY) return bf16_pairs(x_early[word]);
                else if constexpr (XF32)
                    return f32_pairs(reinterpret_cast<const float*>(xrow[nt]) + word / WPG * G + word % WPG * 8, m1[nt],
                                     m2[nt]);
                else return bf16_pairs(bf16_x(word, nt));
            };
            auto of_group = [&](uint32_t v, int q) {
                return GPS == 1 ? v : __shfl_sync(0xffffffffu, v, (lane & ~3u) + q);
            };
            // the products of a group's words
            auto products = [&](int q, auto&& decode, auto& to, auto& low) {
                auto words = [&](int i, uint32_t (&w)[WPG]) {
                    const uint8_t* row = stage + i * (8 * kRowBytes);
                    if constexpr (WPG == 1) {
                        w[0] = *reinterpret_cast<const uint32_t*>(row + ((q ^ swz) << 4) + c * 4);
                    } else if constexpr (WPG == 2) {
                        const uint2 v = *reinterpret_cast<const uint2*>(row + (((2 * q + (c >> 1)) ^ swz) << 4) +
                                                                       (c & 1) * 8);
                        w[0] = v.x, w[1] = v.y;
                    } else {
                        const uint4 v = *reinterpret_cast<const uint4*>(row + ((c ^ swz) << 4));
                        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
                    }
                };
                auto tile = [&](int mt, uint32_t w0, uint32_t w1, const uint4 (&x)[NT]) {
                    uint32_t lo[4], hi[4];  // rows g and g + 8
                    decode(mt, 0, w0, lo);
                    decode(mt, 1, w1, hi);
                    const uint32_t a0[4] = {lo[0], hi[0], lo[1], hi[1]}, a1[4] = {lo[2], hi[2], lo[3], hi[3]};
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float(&d)[4] = BY_TERM && nt ? low[BY_TERM ? mt : 0] : to[mt][BY_TERM ? 0 : nt];
                        mma_bf16(d, a0, x[nt].x, x[nt].y);
                        mma_bf16(d, a1, x[nt].z, x[nt].w);
                    }
                };
                if constexpr (NT == 1) {  // x of the group's words, then tile by tile
                    uint4 x[WPG][1];
#pragma unroll
                    for (int wd = 0; wd < WPG; ++wd) x[wd][0] = load_x(q * WPG + wd, 0);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        uint32_t w0[WPG], w1[WPG];
                        words(2 * mt, w0);
                        words(2 * mt + 1, w1);
#pragma unroll
                        for (int wd = 0; wd < WPG; ++wd) tile(mt, w0[wd], w1[wd], x[wd]);
                    }
                } else {  // word by word
                    uint32_t w[MT * 2][WPG];
#pragma unroll
                    for (int i = 0; i < MT * 2; ++i) words(i, w[i]);
#pragma unroll
                    for (int wd = 0; wd < WPG; ++wd) {
                        uint4 x[NT];
                        if constexpr (BY_TERM) {
                            f32_terms(reinterpret_cast<const float*>(xrow[0]) + q * G + wd * 8, x);
                        } else {
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) x[nt] = load_x(q * WPG + wd, nt);
                        }
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) tile(mt, w[2 * mt][wd], w[2 * mt + 1][wd], x);
                    }
                }
            };
            auto scaled_group = [&](int q, bool careful) {
                float part[MT][NA][4] = {}, part_low[BY_TERM ? MT : 1][4] = {};
                uint32_t zero[MT][2];
                if constexpr (CODE == MOE_B200_Q4_INT4) {
#pragma unroll
                    for (int i = 0; i < MT * 2; ++i) zero[i / 2][i & 1] = of_group(unit[i / 2][i & 1], q);
                }
                products(q, [&](int mt, int h, uint32_t w, uint32_t (&p)[4]) {
                    if constexpr (CODE == MOE_B200_Q4_INT4) decode_int4(w, zero[mt][h], p);
                    else decode_e2m1(w, kUnitE2M1, p);
                }, part, part_low);
#pragma unroll
                for (int i = 0; i < MT * 2; ++i) {
                    const int mt = i / 2, h = i & 1;
                    float s = 0.0f;
                    if (careful) {
                        s = true_scale<ST>(job, (is_up(mt) ? up_row : gate_row) * job.groups + scale_off[mt][h] +
                                                    slice * GPS + q);
                    } else if constexpr (!FOLD) {
                        s = __uint_as_float(of_group(__float_as_uint(grown[mt][h]), q));
                    }
#pragma unroll
                    for (int j = 0; j < NA * 2; ++j) {
                        float& to = acc[mt][j / 2][2 * h + (j & 1)];
                        float v = part[mt][j / 2][2 * h + (j & 1)];
                        if constexpr (BY_TERM) v += part_low[mt][2 * h + j];
                        to = careful ? add_scaled(s, v, to) : fmaf(s, v, to);
                    }
                }
            };
            // with FOLD a slice's sum is added to the others in fp32's own rounding: the
            // matrix unit cuts where it adds, and its errors would run one way
            float of_slice[FOLD ? MT : 1][NA][4] = {};
            auto group = [&](int q) {
                if constexpr (FOLD) {
                    uint32_t u[MT][2];
#pragma unroll
                    for (int i = 0; i < MT * 2; ++i) u[i / 2][i & 1] = of_group(unit[i / 2][i & 1], q);
                    products(q, [&](int mt, int h, uint32_t w, uint32_t (&p)[4]) { decode_e2m1(w, u[mt][h], p); },
                             of_slice, lower);
                } else {
                    scaled_group(q, false);
                }
            };
            if (!odd && full) {  // nothing between the groups, so that their loads can go ahead
#pragma unroll
                for (int q = 0; q < GPS; ++q) group(q);
            } else if (!odd) {
#pragma unroll
                for (int q = 0; q < GPS - 1; ++q) {
                    if ((uint32_t)q < here) group(q);
                }
            } else {
#pragma unroll
                for (int q = 0; q < GPS; ++q) {
                    if ((uint32_t)q < here) scaled_group(q, true);
                }
            }
            if constexpr (FOLD) {
#pragma unroll
                for (int i = 0; i < MT * NA * 4; ++i) (&acc[0][0][0])[i] += (&of_slice[0][0][0])[i];
            }
#pragma unroll
            for (int nt = 0; nt < (XS ? 0 : NT); ++nt) xrow[nt] += warps * kSlice * (XF32 ? 4 : 2);
        }
        // the warps' sums, joined in their order
        cp_async_wait<0>();
        __syncwarp();
        float* mine = reinterpret_cast<float*>(ring);  // [column][row]
#pragma unroll
        for (int nt = 0; nt < NA; ++nt) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t col = nt * 8 + c * 2 + (i & 1);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    if (col < (BY_TERM ? rows : cols))
                        mine[col * ROWS + mt * 16 + g + 8 * (i / 2)] =
                            BY_TERM ? acc[mt][nt][i] + lower[BY_TERM ? mt : 0][i] : acc[mt][nt][i];
                }
            }
        }
        __syncthreads();
        auto joined = [&](uint32_t row, uint32_t r) {
            float s = 0.0f;
            for (uint32_t w = 0; w < warps; ++w) {
                const float* p = reinterpret_cast<const float*>(smem + w * ring_bytes(MT)) +
                                 (BY_TERM ? r : r * terms) * ROWS + row;
                s += !BY_TERM && terms == 3 ? p[0] + (p[ROWS] + p[2 * ROWS]) : p[0];
            }
            return s;
        };
        for (uint32_t o = threadIdx.x; o < out_rows * rows; o += blockDim.x) {
            const uint32_t n = o % out_rows, r = o / out_rows;
            const uint32_t xr = pass_x_row[r];
            if (n0 + n >= job.N || xr >= job.tokens) continue;
            float v = joined(n, r);
            if (terms == 3 && v != v) v = plain_dot(job, gate_row + n, xr);
            if (job.gated) {
                float up = joined(out_rows + n, r);
                if (terms == 3 && up != up) up = plain_dot(job, up_row + n, xr);
                v = activate(job.act, v) * up;
            }
            const uint64_t at = (uint64_t)(first + r0 + r) * job.y_stride + n0 + n;
            if (job.y_type == MOE_B200_DTYPE_F32) static_cast<float*>(job.y)[at] = v;
            else static_cast<uint16_t*>(job.y)[at] = bf16_one(v);
        }
        __syncthreads();  // the rings are free again
    }
}

template <int CODE, int G, int ST, int MT, int NT, int XM>
cudaError_t launch_q4_kernel(const Q4Job& job, const Q4Plan& p, cudaStream_t st) {
    auto* kernel = q4_kernel<CODE, G, ST, MT, NT, XM>;
    static std::atomic<uint64_t> smem_set{0};
    const cudaError_t e = allow_smem(kernel, p.device, &smem_set, kMostSmem);
    if (e != cudaSuccess) return e;
    const uint32_t blocks = ceil_div(job.N, (job.gated ? MT / 2 : MT) * 16u);
    return launch_kernel(kernel, dim3(blocks, p.batches), dim3(p.warps * 32), p.smem, st, true, job);
}

template <int CODE, int G, int ST, int XM>
cudaError_t launch_q4_shape(const Q4Job& job, const Q4Plan& p, cudaStream_t st) {
    if (p.mt == 1) return launch_q4_kernel<CODE, G, ST, 1, 1, XM>(job, p, st);
    if (p.mt == 4) return launch_q4_kernel<CODE, G, ST, 4, 1, XM>(job, p, st);
    if (p.nt == 1) return launch_q4_kernel<CODE, G, ST, 2, 1, XM>(job, p, st);
    if constexpr (XM == kXF32) {
        return launch_q4_kernel<CODE, G, ST, 2, 3, XM>(job, p, st);
    } else {
        if (p.nt == 2) return launch_q4_kernel<CODE, G, ST, 2, 2, XM>(job, p, st);
        return launch_q4_kernel<CODE, G, ST, 2, 4, XM>(job, p, st);
    }
}
template <int CODE, int G, int ST>
cudaError_t launch_q4_x(const Q4Job& job, const Q4Plan& p, cudaStream_t st) {
    if (!job.x_vec) return launch_q4_kernel<CODE, G, ST, 2, 2, kXStaged>(job, p, st);
    return job.x_type == MOE_B200_DTYPE_F32 ? launch_q4_shape<CODE, G, ST, kXF32>(job, p, st)
                                            : launch_q4_shape<CODE, G, ST, kXBf16>(job, p, st);
}
template <int CODE, int G>
cudaError_t launch_q4_scale(const Q4Job& job, const Q4Plan& p, cudaStream_t st) {
    switch (job.scale_type) {
        case MOE_B200_DTYPE_E8M0: return launch_q4_x<CODE, G, MOE_B200_DTYPE_E8M0>(job, p, st);
        case MOE_B200_DTYPE_F32: return launch_q4_x<CODE, G, MOE_B200_DTYPE_F32>(job, p, st);
        case MOE_B200_DTYPE_F16: return launch_q4_x<CODE, G, MOE_B200_DTYPE_F16>(job, p, st);
        default: return launch_q4_x<CODE, G, MOE_B200_DTYPE_BF16>(job, p, st);
    }
}
template <int CODE>
cudaError_t launch_q4_code(const Q4Job& job, const Q4Plan& p, cudaStream_t st) {
    switch (job.group) {
        case 32: return launch_q4_scale<CODE, 32>(job, p, st);
        case 64: return launch_q4_scale<CODE, 64>(job, p, st);
        default: return launch_q4_scale<CODE, 128>(job, p, st);
    }
}

}  // namespace
}  // namespace moe_b200
