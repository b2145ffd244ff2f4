// Entry point of the 4-bit matrix-vector products: argument checks and the
// launch shape (the kernel and its reasons are in q4_kernel.cuh).
#include "q4_kernel.cuh"

namespace moe_b200 {
namespace {

// The launch shape: `rows` rows of x that a matrix is likely to meet.  All
// figures in us, one token of bf16 x MXFP4 where nothing else is said.
//   mt, tiles of 16 rows a block: more share the work on x and the start of a
//   block, fewer make more blocks.  4 from four blocks an SM on (131,072 x 7168
//   integers with 4 rows: 123, with 2 tiles 130, with one 151; 49,152 x 4096: 36.5 and
//   37.2; 16,384 x 4096, two blocks: 15.7 and 15.6); one where even 2 leave a
//   quarter of the SMs without a block (2048 x 7168: 6.0 and 8.6; 4096 x 4096
//   with 4 rows, 128 blocks: 6.2 and 6.0).
//   warps, which share a block's columns: 8 while there are few blocks, 4 from
//   three an SM on (16,384 x 4096: 15.6 and 16.8; 7168 x 2048, one and a half
//   blocks: 5.2 and 5.1); 2 with four tiles of columns, whose registers hold 8
//   warps an SM (16,384 x 4096 with 32 rows: 30.5, by fours 33.2; 131,072 x
//   7168: 337 and 358).  One tile of rows: 16 (2048 x 7168: 6.0, by eights 6.6).
// By expert `rows` is the average of a batch, the host's only figure; a batch far
// above it goes through its matrix once a pass (two fp32 rows or 8 bf16 ones of
// one tile of columns).  32 matrices of 2880 x 2880: one row each 51 us in fp32
// and 45 in bf16; 20 with one row and one with 12: 85 and 38.
Q4Plan q4_plan(Q4Job& job, uint32_t rows, uint32_t batches, int sms, int device) {
    Q4Plan p = {};
    p.device = device;
    p.batches = batches;
    const uint32_t slices = ceil_div(job.K, (uint32_t)kSlice);
    const uint32_t terms = job.x_type == MOE_B200_DTYPE_F32 ? 3 : 1;
    auto blocks = [&](uint32_t mt) { return (uint64_t)ceil_div(job.N, (job.gated ? mt / 2 : mt) * 16) * batches; };
    const uint32_t cols = rows * terms;
    // fp32: three columns a row in one tile of columns, or three tiles of 8 rows
    p.nt = cols <= 8 ? 1 : (terms == 3 ? 3 : (cols <= 16 ? 2 : 4));
    p.mt = 2;
    if (p.nt == 1 && blocks(4) >= 4ull * sms) p.mt = 4;
    else if (p.nt == 1 && !job.gated && blocks(2) * 4 < 3ull * sms) p.mt = 1;
    if (!job.x_vec) p.mt = p.nt = 2;
    p.warps = std::min(p.mt == 1 ? 16u : (blocks(p.mt) < 3ull * sms ? 8u : (p.nt == 4 ? 2u : 4u)), slices);
    p.smem = p.warps * ring_bytes(p.mt);
    if (!job.x_vec) {
        // as many rows as fit, or one and where not even that fits part of it at a time
        job.pass_rows = std::min({rows, 16u / terms, kMaxPassRows});
        while (job.pass_rows > 1 && x_bytes(slices, job.pass_rows * terms) > 64 * 1024) --job.pass_rows;
        job.pass_turns = std::min(ceil_div(slices, p.warps), 160u * 1024 / x_bytes(p.warps, job.pass_rows * terms));
        p.smem += x_bytes(std::min(slices, job.pass_turns * p.warps), job.pass_rows * terms);
    }
    return p;
}

}  // namespace
}  // namespace moe_b200

using namespace moe_b200;

extern "C" {

int moe_b200_q4_matvec(moe_b200_engine_t* eng, const moe_b200_q4_cfg_t* cfg_in, const uint8_t* codes,
                       const void* scales, const uint8_t* zeros, const void* x, const moe_b200_batch_t* batches,
                       const uint32_t* batch_count, const uint32_t* perm, void* y, void* stream, char* err) {
    if (!cfg_in) {
        set_err(err, "null 4-bit config");
        return 0;
    }
    moe_b200_q4_cfg_t cfg = *cfg_in;
    if (cfg.group != 32 && cfg.group != 64 && cfg.group != 128) {
        set_err(err, "group=%u: 32, 64 or 128", cfg.group);
        return 0;
    }
    if (cfg.rows == 0 || cfg.rows > (1u << 24)) {
        set_err(err, "rows=%u outside 1..2^24", cfg.rows);
        return 0;
    }
    if (cfg.cols == 0 || cfg.cols > (1u << 20) || cfg.cols % cfg.group) {
        set_err(err, "cols=%u must be a positive multiple of the group of %u (<= 2^20)", cfg.cols, cfg.group);
        return 0;
    }
    if (cfg.code != MOE_B200_Q4_E2M1 && cfg.code != MOE_B200_Q4_INT4) {
        set_err(err, "unknown 4-bit code %d", cfg.code);
        return 0;
    }
    if (cfg.scale_type < MOE_B200_DTYPE_F32 || cfg.scale_type > MOE_B200_DTYPE_E8M0) {
        set_err(err, "unknown scale type %d", cfg.scale_type);
        return 0;
    }
    if (!row_type_ok(cfg.x_type) || !row_type_ok(cfg.y_type)) {
        set_err(err, "row types %d, %d: fp32 or bf16", cfg.x_type, cfg.y_type);
        return 0;
    }
    if (cfg.gated && (cfg.activation < MOE_B200_ACT_SILU || cfg.activation > MOE_B200_ACT_GELU_TANH)) {
        set_err(err, "unknown activation %d", cfg.activation);
        return 0;
    }
    if (cfg.experts == 0) cfg.experts = 1;
    if (cfg.experts > 1024) {
        set_err(err, "experts=%u above 1024", cfg.experts);
        return 0;
    }
    if (zeros && cfg.code != MOE_B200_Q4_INT4) {
        set_err(err, "zero points go with integer codes");
        return 0;
    }
    if (!batches) {
        if (cfg.experts != 1 || perm || batch_count) {
            set_err(err, "experts, batch_count and perm go with batches");
            return 0;
        }
        if (cfg.out_rows == 0) cfg.out_rows = cfg.tokens;
        if (cfg.out_rows != cfg.tokens) {
            set_err(err, "out_rows=%u differs from tokens=%u without batches", cfg.out_rows, cfg.tokens);
            return 0;
        }
    } else if (!batch_count) {
        set_err(err, "null batch_count");
        return 0;
    }
    if (perm && (cfg.top_k == 0 || cfg.top_k > 32)) {
        set_err(err, "top_k=%u outside 1..32", cfg.top_k);
        return 0;
    }
    if (cfg.tokens >= (1u << 31) || cfg.out_rows >= (1u << 31)) {
        set_err(err, "tokens=%u, out_rows=%u: 2^31 rows or more", cfg.tokens, cfg.out_rows);
        return 0;
    }
    if (!check_stride("x_stride", &cfg.x_stride, cfg.cols, err) ||
        !check_stride("y_stride", &cfg.y_stride, cfg.rows, err)) {
        return 0;
    }
    const uint64_t total_rows = (uint64_t)cfg.experts * cfg.rows * (cfg.gated ? 2 : 1);
    const uint64_t groups = cfg.cols / cfg.group;
    const uint32_t max_batches = batches ? std::min(cfg.experts, cfg.out_rows) : 1;
    const Span ins[] = {{"codes", codes, total_rows * (cfg.cols / 2)},
                        {"scales", scales, total_rows * groups * type_bytes(cfg.scale_type)},
                        row_span("x", x, cfg.tokens, cfg.cols, cfg.x_stride, cfg.x_type),
                        {"zeros", zeros, zeros ? total_rows * groups : 0},
                        {"batches", batches, (uint64_t)max_batches * sizeof(moe_b200_batch_t)},
                        {"batch_count", batch_count, 4},
                        {"perm", perm, (uint64_t)cfg.out_rows * 4}};
    const Span out = row_span("y", y, cfg.out_rows, cfg.rows, cfg.y_stride, cfg.y_type);
    const bool work = cfg.tokens && cfg.out_rows;
    for (int i = 0; i < 3; ++i) {
        if (work && !check_given(ins[i], err)) return 0;
    }
    if (work && !check_given(out, err)) return 0;
    if (!check_aligned(ins[0], 16, err) || !check_aligned(ins[1], type_bytes(cfg.scale_type), err) ||
        !check_aligned(ins[2], type_bytes(cfg.x_type), err) || !check_aligned(out, type_bytes(cfg.y_type), err)) {
        return 0;
    }
    for (int i = 4; i < 7; ++i) {
        if (!check_aligned(ins[i], 4, err)) return 0;
    }
    if (!check_overlap(&out, 1, ins, 7, nullptr, 0, err)) return 0;
    OnDevice on(eng, err);
    if (!on.ok) return 0;
    if (!work) return 1;
    Q4Job job = {cfg.rows, cfg.cols, cfg.group, (uint32_t)groups, cfg.experts, cfg.tokens, cfg.out_rows,
                       cfg.top_k, cfg.x_stride, cfg.y_stride, codes, scales, zeros, x, batches, batch_count, perm, y,
                       eng->err_word.as<uint32_t>(), cfg.scale_type, cfg.x_type, cfg.y_type, cfg.code, cfg.gated,
                       cfg.activation, rows_vec8(x, cfg.x_stride, cfg.x_type), 0, 0};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    // rows of x a matrix is likely to meet: all of them, or the average of a batch
    const uint32_t rows = batches ? ceil_div(cfg.out_rows, max_batches) : cfg.tokens;
    const Q4Plan plan = q4_plan(job, rows, max_batches, eng->num_sms, eng->device);
    return launched(cfg.code == MOE_B200_Q4_E2M1 ? launch_q4_e2m1(job, plan, st) : launch_q4_int4(job, plan, st),
                    "4-bit product", err);
}

}  // extern "C"
