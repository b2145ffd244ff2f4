// The edge between two blocks, forward and backward: the norm behind a block,
// its gate and residual scale, the residual add and the norm in front of the
// next block.
//
//   n = y r_y wpost (or y),  h = rs hidden + os g n,  x = h r_x wpre,
//   r = 1 / sqrt(mean(.^2) + eps)
//
// and, with D the whole gradient of h, u = dx wpre, xh = h r_x, yh = y r_y,
// H the row's length:
//
//   D  = dh + r_x (u - xh (1/H) sum(u xh))
//   dhidden = rs D,  dn = os g D
//   dy = r_y (wpost dn - yh (1/H) sum(dn wpost yh))      (dn without the norm)
//   dwpost = sum_t dn yh,  dwpre = sum_t dx xh,  dg = os D n
//
// D holds a sum over the row and dy a sum over D.  Put together,
//   sum(g n D) = sum(g n (dh + r_x u)) - r_x (1/H) sum(u xh) sum(g n xh),
// so the three sums C = sum(u xh), P = sum(g n (dh + r_x u)), Q = sum(g n xh)
// come from one reading of the row and one reduction over the block.  The
// kernel multiplies the row's roots into its scalars instead of its columns:
// with v = r_x u and m = y wpost, C = sum(v h), P = r_y sum(g m (dh + v)),
// Q = r_y r_x sum(g m h).
//
// The floor is memory traffic: a row is read once, held in registers, and
// written once.  Rates below are of a copy's 6.55 TB/s, measured with inputs
// past the second cache.
#include "op_common.cuh"

namespace moe_b200 {
namespace {

constexpr uint32_t kMaxHidden = 32768;
// Blocks of the backward kernel: what 148 SMs hold at once with blocks of a
// thread to 8 columns and 768 threads an SM (its registers allow no more), so
// that every block adds the weights' gradients up over as many rows as it can
// before one row a block goes to the workspace.  4,096 bf16 rows of 2048: 444
// blocks 37.6 us, 296 41.5, 592 47.0; of 4096: 148 blocks 72.5 us, 296 80.1
// (before later steps).
constexpr uint32_t norm_blocks(uint32_t H) {
    const uint32_t threads = (H + 255) / 256 * 32;
    return 148 * (threads < 768 ? 768 / threads : 1);
}
constexpr uint32_t kMostStages = 4;
constexpr uint32_t kMostThreads = 1024;
constexpr uint32_t kMostSmem = 220 * 1024;

struct NormJob {
    uint32_t H, T;
    uint64_t hidden_stride, y_stride, x_stride;
    const float* post_w;
    const float* pre_w;
    const void* gate;
    int gate_kind, gate_sigmoid;
    float unit_offset;  // what the norms add to their weights: 0 or 1
    float eps, rs, os, inv_h;
    uint32_t stages;     // rows of a block's ring
    int stage_weights;   // the norms' weights go to shared memory
    uint32_t* err;
};

// The reciprocal is the unit's, within one unit of the last place, of 1 or more.
__device__ __forceinline__ float sigmoid(float z) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + expf(-z)));
    return r;
}

template <int V>
__device__ __forceinline__ void load_weight(const float* w, uint32_t c, float unit_offset, float* v) {
    load_f32<V>(w + c, v);
    vadd<V>(v, unit_offset);
}
__device__ __forceinline__ float load_token_gate(const NormJob& job, uint64_t t) {
    if (job.gate_kind != MOE_B200_GATE_TOKEN) return 1.0f;
    const float z = __ldg(static_cast<const float*>(job.gate) + t);
    return job.gate_sigmoid ? sigmoid(z) : z;
}

// A row's columns of one thread: N pieces of V, blockDim.x pieces apart.
template <int V, int N, typename F>
__device__ __forceinline__ void for_pieces(uint32_t H, F&& f) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint32_t c = (threadIdx.x + i * blockDim.x) * V;
        if (c < H) f(i, c);
    }
}
// The same without a branch, so that the loads of all pieces go out together: a
// piece past the row is the last one again, read and not used (`in` false).
// Edge of 4,096 x 2043: 34 us, 61 with branches; 4,096 x 2048 14.0 and 14.9.
template <int V, int N, typename F>
__device__ __forceinline__ void all_pieces(uint32_t H, F&& f) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint32_t c = (threadIdx.x + i * blockDim.x) * V;
        f(i, min(c, H - V), c < H);
    }
}
template <int V>
__device__ __forceinline__ void zero_unless(bool in, float* v) {
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = in ? v[k] : 0.0f;
}
// A piece of a row in shared memory.
template <typename D>
__device__ __forceinline__ Raw<D, 8> staged_piece(const uint8_t* row, uint32_t c) {
    const uint4* p = reinterpret_cast<const uint4*>(row + c * sizeof(typename D::type));
    if constexpr (sizeof(Raw<D, 8>) == 32) {
        // every other four lanes take the second half first, so that eight lanes meet all banks
        const bool back = threadIdx.x & 4;
        const uint4 a = p[back], b = p[!back];
        return {back ? b : a, back ? a : b};
    } else {
        return {p[0]};
    }
}

// Sums over a block: lanes, then warps in their order.  `red` (32 values, those
// past the block's warps 0) takes the warps' sums; every thread adds them up.
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float sum_of_warps(const float* red) {
    float s = 0.0f;
    for (uint32_t w = 0; w < blockDim.x / 32; w += 4) {
        const float4 v = *reinterpret_cast<const float4*>(red + w);
        s += (v.x + v.y) + (v.z + v.w);
    }
    return s;
}
__device__ __forceinline__ double block_sum(double v, double* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    double s = 0.0;
    for (uint32_t w = 0; w < blockDim.x / 32; ++w) s += red[w];
    return s;
}
// 1 / sqrt(mean of squares + eps) of the columns that the row's threads (a
// block's, or a warp's: WARP) hold.  Squares that leave fp32's range are added
// again in double.
template <bool WARP, int N, int V>
__device__ __forceinline__ float row_rms(const float (&v)[N][V], const NormJob& job, float* red, double* wide) {
    float p2[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < N; ++i) vdot<V>(p2, v[i], v[i]);
    float p = warp_sum(p2[0] + p2[1]);
    if constexpr (!WARP) {
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = p;
        __syncthreads();
        p = sum_of_warps(red);
    }
    const float m = fmaf(p, job.inv_h, job.eps);
    if (m > 1e-30f && m < 1e38f) return rsqrtf(m);
    double d = 0.0;  // all of the row's threads
#pragma unroll
    for (int k = 0; k < N * V; ++k) d = fma((double)v[k / V][k % V], (double)v[k / V][k % V], d);
    if constexpr (WARP) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
    } else {
        d = block_sum(d, wide);
    }
    return (float)(1.0 / sqrt(d / (double)job.H + (double)job.eps));
}

// One block a row (ROWS = 1) or one warp a row, N pieces of V columns a thread.
// A row goes through three phases (loads, two sums over its threads, stores)
// that do not overlap in its own block; several blocks on an SM cover each
// other's, which is why the rows stay small: 16 columns a thread (with 32, 4,096
// x 2048 bf16 takes 15 % longer), blocks that live for one row (a persistent
// loop over rows with copies ahead measured slower), and a warp a row where
// that holds it (16,384 x 128: 6.9 us, by blocks of a warp 10.8).  Pieces of
// four columns: neighbouring lanes' fp32 values, weights among them, then lie
// side by side and a load meets half the lines that pieces of eight meet
// (16,384 x 7168, fp32 stream, bf16 rows, channel gate: 247 us, 87 %, by eights
// 262; bf16 alone is the same).  FULL: both norms and the add, without tests of
// what is there.  What bounds it is the latency of the row's phases; one row
// takes 3.4 us.
template <typename DH, typename DY, typename DX, int V, int N, bool FULL, int ROWS, uint32_t THREADS, int BLOCKS>
__global__ void __launch_bounds__(THREADS, BLOCKS)
    norm_forward_kernel(const typename DH::type* hidden, const typename DY::type* y, typename DH::type* hidden_out,
                        typename DX::type* x, float* rms_y, float* rms_x, const __grid_constant__ NormJob job) {
    __shared__ __align__(16) float red[2][32];
    __shared__ double wide[2][32];
    const bool has_y = FULL || y, has_x = FULL || x, post = FULL || job.post_w;
    const bool element = has_y && job.gate_kind == MOE_B200_GATE_ELEMENT;
    const bool channel = has_y && job.gate_kind == MOE_B200_GATE_CHANNEL;
    constexpr bool WARP = ROWS > 1;
    if constexpr (!WARP) {
        if (threadIdx.x < 64) (&red[0][0])[threadIdx.x] = 0.0f;
        if (blockDim.x == 32) (&red[0][0])[threadIdx.x + 32] = 0.0f;
        __syncthreads();
    }
    pdl_wait();
    const uint64_t t = (uint64_t)blockIdx.x * ROWS + (WARP ? threadIdx.y : 0);
    if (WARP && t >= job.T) return;
    Raw<DH, V> hr[N];
    Raw<DY, V> yr[N], gr[N];
    all_pieces<V, N>(job.H, [&](int i, uint32_t c, bool) {
        if (has_y) yr[i] = load_row<DY, V>(y + t * job.y_stride + c);
        hr[i] = load_row<DH, V>(hidden + t * job.hidden_stride + c);
        if (element) gr[i] = load_row<DY, V>(static_cast<const typename DY::type*>(job.gate) + t * job.y_stride + c);
    });
    const float tg = has_y ? load_token_gate(job, t) : 1.0f;
    float ry = 1.0f;
    if (post) {
        float n[N][V] = {};
        all_pieces<V, N>(job.H, [&](int i, uint32_t, bool in) {
            unpack(yr[i], n[i]);
            zero_unless<V>(in, n[i]);
        });
        ry = row_rms<WARP>(n, job, red[0], wide[0]);
        if (rms_y && threadIdx.x == 0) rms_y[t] = ry;
    }
    const float scale = job.os * tg;
    float h[N][V] = {};
    all_pieces<V, N>(job.H, [&](int i, uint32_t c, bool in) {
        float (&v)[V] = h[i];
        unpack(hr[i], v);
        vmul<V>(v, v, job.rs);
        if (has_y) {
            float n[V];
            unpack(yr[i], n);
            if (post) {
                float w[V];
                load_weight<V>(job.post_w, c, job.unit_offset, w);
                vmul<V>(n, n, ry);
                vmul<V>(n, n, w);
            }
            if (element || channel) {
                float g[V];
                if (element) unpack(gr[i], g);
                else load_f32<V>(static_cast<const float*>(job.gate) + c, g);
                if (job.gate_sigmoid) {
#pragma unroll
                    for (int k = 0; k < V; ++k) g[k] = sigmoid(g[k]);
                }
                vmul<V>(g, g, job.os);
                vfma<V>(v, g, n, v);
            } else {
                vfma<V>(v, n, scale, v);
            }
        }
        if ((FULL || hidden_out) && in) {
            Raw<DH, V> r;
            pack(v, r);
            store_row(hidden_out + t * job.hidden_stride + c, r);
        }
        zero_unless<V>(in, v);
    });
    if (!has_x) return;
    const float rx = row_rms<WARP>(h, job, red[1], wide[1]);
    if (rms_x && threadIdx.x == 0) rms_x[t] = rx;
    all_pieces<V, N>(job.H, [&](int i, uint32_t c, bool in) {
        float o[V], w[V];
        load_weight<V>(job.pre_w, c, job.unit_offset, w);
        vmul<V>(o, h[i], rx);
        vmul<V>(o, o, w);
        Raw<DX, V> r;
        pack(o, r);
        if (in) store_row(x + t * job.x_stride + c, r);
    });
}

// Rows that are too long for the block's registers (above 16,384 columns): h is
// kept in shared memory between its sum and x, y is read twice.  For
// completeness, not for speed.
template <typename DH, typename DY, typename DX>
__global__ void __launch_bounds__(512)
    norm_forward_long_kernel(const typename DH::type* hidden, const typename DY::type* y,
                             typename DH::type* hidden_out, typename DX::type* x, float* rms_y, float* rms_x,
                             const __grid_constant__ NormJob job) {
    extern __shared__ float row[];
    __shared__ double red[2][32];
    pdl_wait();
    const uint64_t t = blockIdx.x;
    auto value = [&](auto* d, const auto* p, uint32_t c) {
        using D = std::remove_pointer_t<decltype(d)>;
        float v[1];
        unpack(load_row<D, 1>(p + c), v);
        return v[0];
    };
    DY* dy = nullptr;
    DH* dh = nullptr;
    auto root = [&](double ss) {
        const double m = ss / (double)job.H + (double)job.eps;
        return (float)(1.0 / sqrt(m));
    };
    const typename DY::type* yt = y ? y + t * job.y_stride : nullptr;
    const float tg = y ? load_token_gate(job, t) : 1.0f;
    float ry = 1.0f;
    if (job.post_w) {
        double ss = 0.0;
        for (uint32_t c = threadIdx.x; c < job.H; c += blockDim.x) {
            const double v = value(dy, yt, c);
            ss = fma(v, v, ss);
        }
        ry = root(block_sum(ss, red[0]));
        if (rms_y && threadIdx.x == 0) rms_y[t] = ry;
    }
    double ss = 0.0;
    for (uint32_t c = threadIdx.x; c < job.H; c += blockDim.x) {
        float h = job.rs * value(dh, hidden + t * job.hidden_stride, c);
        if (y) {
            float n = value(dy, yt, c), g = tg;
            if (job.post_w) n = n * ry * (job.post_w[c] + job.unit_offset);
            if (job.gate_kind == MOE_B200_GATE_CHANNEL) g = __ldg(static_cast<const float*>(job.gate) + c);
            if (job.gate_kind == MOE_B200_GATE_ELEMENT)
                g = value(dy, static_cast<const typename DY::type*>(job.gate) + t * job.y_stride, c);
            if (job.gate_kind != MOE_B200_GATE_TOKEN && job.gate_kind && job.gate_sigmoid) g = sigmoid(g);
            h = fmaf(job.os * g, n, h);
        }
        if (hidden_out) {
            Raw<DH, 1> r;
            pack(&h, r);
            store_row(hidden_out + t * job.hidden_stride + c, r);
        }
        row[c] = h;  // this thread's own
        ss = fma((double)h, (double)h, ss);
    }
    if (!x) return;
    const float rx = root(block_sum(ss, red[1]));
    if (rms_x && threadIdx.x == 0) rms_x[t] = rx;
    for (uint32_t c = threadIdx.x; c < job.H; c += blockDim.x) {
        const float o = row[c] * rx * (job.pre_w[c] + job.unit_offset);
        Raw<DX, 1> r;
        pack(&o, r);
        store_row(x + t * job.x_stride + c, r);
    }
}

// Which sums over the tokens a backward call keeps, one slot of H values each.
struct NormSums {
    int post, pre, gate;  // slot, or -1
    int slots;
    float* part;          // [blocks][slots][H]
};

// A block's own rows of fp32 values: in shared memory (SPLIT) the first four
// values of each eight in one half of the row and the last four in the other,
// so that neighbouring threads meet neighbouring banks.
template <int V, bool SPLIT>
__device__ __forceinline__ void load_own(const float* row, uint32_t c, uint32_t H, float* v) {
    if constexpr (V == 8) {
        const float4 a = *reinterpret_cast<const float4*>(row + (SPLIT ? c / 2 : c));
        const float4 b = *reinterpret_cast<const float4*>(row + (SPLIT ? H / 2 + c / 2 : c + 4));
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
        v[0] = row[c];
    }
}
template <int V, bool SPLIT>
__device__ __forceinline__ void store_own(float* row, uint32_t c, uint32_t H, const float* v) {
    if constexpr (V == 8) {
        *reinterpret_cast<float4*>(row + (SPLIT ? c / 2 : c)) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(row + (SPLIT ? H / 2 + c / 2 : c + 4)) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        row[c] = v[0];
    }
}

// Rows t = blockIdx.x, + gridDim.x, ... of a block, so that the sums over the
// tokens stay in its shared memory.  Each column belongs to one thread, so
// those sums need no barrier; a row needs one, for C, P and Q.
// N > 0: N pieces of V columns a thread, held from the sums to the gradients.
// BULK: the rows come through a ring in shared memory by bulk copies that run
// behind the work on earlier rows.  N = 0: longer rows, read twice (the second
// time from L2), the sums over the tokens in the workspace instead.  GATE >= 0:
// both norms and the gradients of hidden, y and the norms' weights; GATE then
// is the gate's kind (a token's or none: 0), otherwise -1.
// 4,096 x 2048 bf16 with an element gate: 35.2 us, 58 % (87 us when the loads
// waited for each row and neighbouring threads' sums met the same banks).
// What bounds it: too little overlap for what each row costs.  A warp issues some
// 640 instructions for its 256 columns, a third of them the row's own, and reads
// and writes every sum over the tokens in shared memory; with 36 % of an SM's
// warps resident and a barrier every row, issue is busy in 59 % of the cycles
// and the path to shared memory in 64 %.  A thread to 16 columns would halve the
// rows' own instructions but leaves 4 blocks of 128 threads an SM: 61 us.
// Above 4096 columns one block of up to 1024 threads, spilling some of its 64
// registers, holds an SM, and beside the sums its ring often has one place, so
// that copies wait for the row before: 4,096 x 7168 with an fp32 stream, bf16
// rows and a channel gate 214 us (38 %), 8192 columns bf16 181 us (34 %).  Above
// 8192 (N = 0): 2,048 x 12,288 bf16 192 us (24 %), 16,384 columns 267 us.
// Rows that cannot be read by vectors take one column an instruction: 4,096 x
// 2043 62 us (25 %), 2,048 x 5001 140 us, 192 with branches around its loads.
// GATE >= 0 against the general kernel (us; none, channel and element gate, bf16,
// through a sigmoid): 4,096 x 2048 26 41 35 and 38 48 47; 4,096 x 4096 44 62 52
// and 52 71 67; 4,096 x 7168 97 149 and 144 183; 4,096 x 2043 55 74 73 and 95 124
// 116; 2,048 x 5001 103 140 and 220 249.  Element gates above 4096 columns
// run by the general kernel: 4,096 x 7168 173 us, 2,048 x 5001 266.
template <typename DH, typename DY, typename DX, int V, int N, bool BULK, int GATE, uint32_t THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? 3 : 1)
    norm_backward_kernel(const typename DH::type* d_hidden_out, const typename DX::type* d_x,
                         const typename DH::type* hidden_out, const typename DY::type* y, const float* rms_y,
                         const float* rms_x, typename DH::type* d_hidden, typename DY::type* d_y, void* d_gate,
                         const __grid_constant__ NormSums sums, const __grid_constant__ NormJob job) {
    constexpr int M = N ? N : 1;
    constexpr bool FULL = GATE >= 0;
    constexpr bool KEEP = N && THREADS == 512;  // the weights stay in registers
    extern __shared__ __align__(128) uint8_t ring[];  // [stages][dh, dx, h, y, gate], then the sums over the tokens
    __shared__ float red[2][THREADS / 8];  // C, P, Q of each warp
    __shared__ __align__(8) uint64_t full[kMostStages];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool has_y = FULL || y, has_x = FULL || d_x, has_dh = FULL || d_hidden_out, post = FULL || job.post_w;
    const bool element = FULL ? GATE == MOE_B200_GATE_ELEMENT : has_y && job.gate_kind == MOE_B200_GATE_ELEMENT;
    const uint32_t h_bytes = job.H * sizeof(typename DH::type), x_bytes = job.H * sizeof(typename DX::type),
                   y_bytes = job.H * sizeof(typename DY::type);
    const uint32_t at_dx = has_dh ? h_bytes : 0, at_h = at_dx + (has_x ? x_bytes : 0),
                   at_y = at_h + (has_x ? h_bytes : 0), at_g = at_y + (has_y ? y_bytes : 0);
    const uint32_t row_bytes = at_g + (element ? y_bytes : 0);
    float* acc = N ? reinterpret_cast<float*>(ring + (BULK ? job.stages * row_bytes : 0))
                   : sums.part + (uint64_t)blockIdx.x * sums.slots * job.H;
    const typename DY::type* gate = static_cast<const typename DY::type*>(job.gate);
    const bool channel = FULL ? GATE == MOE_B200_GATE_CHANNEL : job.gate_kind == MOE_B200_GATE_CHANNEL;
    const bool shared_gate = !element && !channel;
    for (uint32_t i = threadIdx.x; i < THREADS / 4; i += blockDim.x) (&red[0][0])[i] = 0.0f;
    if (BULK && threadIdx.x == 0) {
        for (uint32_t s = 0; s < job.stages; ++s) mbar_init(&full[s], 1);
        fence_mbar_init();
    }
    __syncthreads();
    pdl_wait();
    auto fetch = [&](uint64_t t, uint32_t s) {  // by one thread
        if (t >= job.T) return;
        uint8_t* to = ring + s * row_bytes;
        mbar_arrive_expect_tx(&full[s], row_bytes);
        if (has_dh) bulk_g2s(to, d_hidden_out + t * job.hidden_stride, h_bytes, &full[s]);
        if (has_x) {
            bulk_g2s(to + at_dx, d_x + t * job.x_stride, x_bytes, &full[s]);
            bulk_g2s(to + at_h, hidden_out + t * job.hidden_stride, h_bytes, &full[s]);
        }
        if (has_y) bulk_g2s(to + at_y, y + t * job.y_stride, y_bytes, &full[s]);
        if (element) bulk_g2s(to + at_g, gate + t * job.y_stride, y_bytes, &full[s]);
    };
    if (BULK && threadIdx.x == 0) {
        for (uint32_t s = 0; s < job.stages; ++s) fetch(blockIdx.x + (uint64_t)s * gridDim.x, s);
    }
    // the weights of the norms: in registers, in shared memory, or where they are
    float kept_wx[KEEP ? M : 1][V] = {}, kept_wy[KEEP ? M : 1][V] = {};
    float* staged_w = acc + sums.slots * job.H;
    const bool staged = BULK && !KEEP && job.stage_weights;
    if (staged) {
        for_pieces<V, M>(job.H, [&](int, uint32_t c) {
            float w[V];
            if (has_x) {
                load_weight<V>(job.pre_w, c, job.unit_offset, w);
                store_own<V, true>(staged_w, c, job.H, w);
            }
            if (post) {
                load_weight<V>(job.post_w, c, job.unit_offset, w);
                store_own<V, true>(staged_w + job.H, c, job.H, w);
            }
        });
    }
    auto weight = [&](int which, uint32_t c, float* w) {
        if (staged) load_own<V, true>(staged_w + which * job.H, c, job.H, w);
        else load_weight<V>(which ? job.post_w : job.pre_w, c, job.unit_offset, w);
    };
    auto weights_x = [&](int i, uint32_t c, float* w) {
        if constexpr (KEEP) {
#pragma unroll
            for (int q = 0; q < V; ++q) w[q] = kept_wx[i][q];
        } else {
            weight(0, c, w);
        }
    };
    auto weights_y = [&](int i, uint32_t c, float* w) {  // 1 without the norm
        if constexpr (KEEP) {
#pragma unroll
            for (int q = 0; q < V; ++q) w[q] = kept_wy[i][q];
        } else if (post) {
            weight(1, c, w);
        } else {
#pragma unroll
            for (int q = 0; q < V; ++q) w[q] = 1.0f;
        }
    };
    if constexpr (KEEP) {
        for_pieces<V, M>(job.H, [&](int i, uint32_t c) {
#pragma unroll
            for (int q = 0; q < V; ++q) kept_wy[i][q] = 1.0f;
            if (has_x) load_weight<V>(job.pre_w, c, job.unit_offset, kept_wx[i]);
            if (post) load_weight<V>(job.post_w, c, job.unit_offset, kept_wy[i]);
        });
    }
    bool first = true;
    auto add_product = [&](int slot, uint32_t c, const float* v, const float* w) {
        float* row = acc + (uint64_t)slot * job.H;
        float sum[V];
        if (first) {
            vmul<V>(sum, v, w);
        } else {
            load_own<V, N != 0>(row, c, job.H, sum);
            vfma<V>(sum, v, w, sum);
        }
        store_own<V, N != 0>(row, c, job.H, sum);
    };
    uint32_t turn = 0, s = 0, phase = 0;
    // the row's roots and gate, the next row's on their way meanwhile
    float ry = 1.0f, rx = 0.0f, tg = 1.0f, next_ry = 1.0f, next_rx = 0.0f, next_tg = 1.0f;
    auto roots = [&](uint64_t t) {
        if (t >= job.T) return;
        if (post) next_ry = __ldg(rms_y + t);
        if (has_x) next_rx = __ldg(rms_x + t);
        if (has_y) next_tg = load_token_gate(job, t);
    };
    roots(blockIdx.x);
    for (uint64_t t = blockIdx.x; t < job.T; t += gridDim.x, turn ^= 1) {
        ry = next_ry, rx = next_rx, tg = next_tg;
        roots(t + gridDim.x);
        auto each = [&](auto&& f) {
            if constexpr (N != 0) {
                for_pieces<V, M>(job.H, f);
            } else {
                for (uint32_t c = threadIdx.x * V; c < job.H; c += blockDim.x * V) f(0, c);
            }
        };
        // where the row is
        const typename DH::type *dh_t = d_hidden_out + t * job.hidden_stride, *h_t = hidden_out + t * job.hidden_stride;
        const typename DX::type* dx_t = d_x + t * job.x_stride;
        const typename DY::type *y_t = y + t * job.y_stride, *gate_t = gate + t * job.y_stride;
        typename DH::type* d_hidden_t = d_hidden + t * job.hidden_stride;
        typename DY::type *d_y_t = d_y + t * job.y_stride,
                          *d_gate_t = static_cast<typename DY::type*>(d_gate) + t * job.y_stride;
        // the row's pieces as they lie in memory, all loads before their first use
        Raw<DH, V> dhr[M], hr[M];
        Raw<DX, V> dxr[M];
        Raw<DY, V> yr[M], gr[M];
        auto load = [&](int i, uint32_t c) {
            if constexpr (BULK) {
                const uint8_t* at = ring + s * row_bytes;
                if (has_dh) dhr[i] = staged_piece<DH>(at, c);
                if (has_x) dxr[i] = staged_piece<DX>(at + at_dx, c), hr[i] = staged_piece<DH>(at + at_h, c);
                if (has_y) yr[i] = staged_piece<DY>(at + at_y, c);
                if (element) gr[i] = staged_piece<DY>(at + at_g, c);
            } else {
                if (has_dh) dhr[i] = load_row<DH, V>(dh_t + c);
                if (has_x) dxr[i] = load_row<DX, V>(dx_t + c), hr[i] = load_row<DH, V>(h_t + c);
                if (has_y) yr[i] = load_row<DY, V>(y_t + c);
                if (element) gr[i] = load_row<DY, V>(gate_t + c);
            }
        };
        if constexpr (BULK) {
            if (!mbar_wait(&full[s], phase, job.err, kErrTimeoutRows)) {
                // the block's copies may still land: it leaves behind them, or after as long again for each
                for (uint32_t q = 0; q < job.stages && t + (uint64_t)q * gridDim.x < job.T; ++q) {
                    const uint32_t at = s + q < job.stages ? s + q : s + q - job.stages;
                    mbar_wait(&full[at], s + q < job.stages ? phase : phase ^ 1, job.err, kErrTimeoutRows);
                }
                return;
            }
        }
        if constexpr (N != 0 && !BULK) all_pieces<V, M>(job.H, [&](int i, uint32_t c, bool) { load(i, c); });
        else if constexpr (N != 0) each(load);
        // of each column: top = dh + v, h, y, m = y wpost, and g (where it is not the row's)
        struct Cols {
            float top[V], h[V], y[V], m[V], g[V];
        };
        Cols cols[M];
        // `counted`: adds the piece to C, P, Q and to the sum for pre_w
        float C2[2] = {}, P2[2] = {}, Q2[2] = {};
        auto read = [&](int i, uint32_t c, bool counted) {
            Cols& k = cols[i];
            if (has_dh) {
                unpack(dhr[i], k.top);
            } else {
#pragma unroll
                for (int q = 0; q < V; ++q) k.top[q] = 0.0f;
            }
            if (has_x) {
                float dx[V], v[V];
                unpack(dxr[i], dx);
                unpack(hr[i], k.h);
                weights_x(i, c, v);
                vmul<V>(dx, dx, rx);
                vmul<V>(v, v, dx);
                vadd<V>(k.top, v);
                if (counted) vdot<V>(C2, v, k.h);
                if (counted && (FULL || sums.pre >= 0))
                    add_product(sums.pre, c, dx, k.h);
            } else {
#pragma unroll
                for (int q = 0; q < V; ++q) k.h[q] = 0.0f;
            }
            if (!has_y) return;
            unpack(yr[i], k.y);
            weights_y(i, c, k.m);
            vmul<V>(k.m, k.m, k.y);
            if (!shared_gate) {
                if (element) unpack(gr[i], k.g);
                else load_f32<V>(static_cast<const float*>(job.gate) + c, k.g);
                if (job.gate_sigmoid) {
#pragma unroll
                    for (int q = 0; q < V; ++q) k.g[q] = sigmoid(k.g[q]);
                }
            }
            if (!counted) return;
            if (shared_gate) {  // multiplied in afterwards
                vdot<V>(P2, k.m, k.top);
                vdot<V>(Q2, k.m, k.h);
            } else {
                float gm[V];
                vmul<V>(gm, k.m, k.g);
                vdot<V>(P2, gm, k.top);
                vdot<V>(Q2, gm, k.h);
            }
        };
        each([&](int i, uint32_t c) {
            if constexpr (N == 0) load(i, c);
            read(i, c, true);
        });
        float C = C2[0] + C2[1], P = P2[0] + P2[1], Q = Q2[0] + Q2[1];
        const float own = lanes_sum4({C, P, Q, 0.0f});
        if (lane < 4) red[turn][warp * 4 + lane] = own;
        __syncthreads();  // the other half of red is free again, and so is the row's place in the ring
        if (BULK && threadIdx.x == 0) fetch(t + (uint64_t)job.stages * gridDim.x, s);
        // a lane takes one value of every eighth warp (2,048 columns: 37.6 -> 35.2 us)
        float v = red[turn][lane];
#pragma unroll
        for (uint32_t k = 32; k < THREADS / 8; k += 32) v += red[turn][lane + k];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        C = __shfl_sync(0xffffffffu, v, 0), P = __shfl_sync(0xffffffffu, v, 1), Q = __shfl_sync(0xffffffffu, v, 2);
        // D = top + back h;  gm_d = sum of g m D
        const float back = -rx * rx * (C * job.inv_h);
        const float gm_d = fmaf(back, Q, P);
        const float scale = shared_gate ? job.os * tg : job.os;
        const float through = ry * scale;                              // e = through (g) D = r_y dn
        // dy = wpost e - mean_s y, in an order without r_y^3, which long rows of large y take to zero
        const float mean_s = (ry * through) * (ry * (gm_d * job.inv_h));
        if (shared_gate && job.gate_kind == MOE_B200_GATE_TOKEN && d_gate && threadIdx.x == 0) {
            static_cast<float*>(d_gate)[t] = job.os * ry * gm_d * (job.gate_sigmoid ? tg * (1.0f - tg) : 1.0f);
        }
        each([&](int i, uint32_t c) {
            if constexpr (N == 0) {
                load(0, c);
                read(0, c, false);
            }
            Cols& k = cols[i];
            float D[V], o[V];
            vfma<V>(D, k.h, back, k.top);
            if (FULL || d_hidden) {
                vmul<V>(o, D, job.rs);
                Raw<DH, V> r;
                pack(o, r);
                store_row(d_hidden_t + c, r);
            }
            if (!has_y) return;
            vmul<V>(D, D, through);
            if (!shared_gate) {
                if (sums.gate >= 0 || (element && d_gate)) {
                    vmul<V>(o, k.m, D);
                    float slope[V];
                    if (job.gate_sigmoid) {  // g - g g
                        vmul<V>(slope, k.g, -1.0f);
                        vfma<V>(slope, slope, k.g, k.g);
                    } else {
#pragma unroll
                        for (int q = 0; q < V; ++q) slope[q] = 1.0f;
                    }
                    if (channel) {
                        add_product(sums.gate, c, o, slope);
                    } else {
                        vmul<V>(o, o, slope);
                        Raw<DY, V> r;
                        pack(o, r);
                        store_row(d_gate_t + c, r);
                    }
                }
                vmul<V>(D, D, k.g);
            }
            // D is e now
            if (FULL || sums.post >= 0) add_product(sums.post, c, D, k.y);
            if (FULL || d_y) {
                if (post) {
                    weights_y(i, c, o);
                    vmul<V>(D, D, o);
                    vfma<V>(D, k.y, -mean_s, D);
                }
                Raw<DY, V> r;
                pack(D, r);
                store_row(d_y_t + c, r);
            }
        });
        first = false;
        if (++s == job.stages) s = 0, phase ^= 1;
    }
    if constexpr (N != 0) {
        float* part = sums.part + (uint64_t)blockIdx.x * sums.slots * job.H;
        for (int slot = 0; slot < sums.slots; ++slot) {
            for_pieces<V, M>(job.H, [&](int, uint32_t c) {
                float v[V];
                load_own<V, true>(acc + slot * job.H, c, job.H, v);
                store_own<V, false>(part + (uint64_t)slot * job.H, c, job.H, v);
            });
        }
    }
}

// out[slot][c] = the sum over the blocks' rows, in a fixed order: 32 columns a
// block, its 32 warps every 32nd row each, eight of them at a time on their
// way.  The rows come from L2; what bounds it is latency.
__global__ void __launch_bounds__(1024) norm_sums_kernel(const float* part, uint32_t blocks, uint32_t H, int slots,
                                                         float* out0, float* out1, float* out2) {
    __shared__ float red[32][33];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t c = blockIdx.x * 32 + lane;
    const int s = blockIdx.y;
    pdl_wait();
    float v = 0.0f;
    if (c < H) {
#pragma unroll 8
        for (uint32_t b = warp; b < blocks; b += 32) v += part[((uint64_t)b * slots + s) * H + c];
    }
    red[warp][lane] = v;
    __syncthreads();
    // a warp takes one column of the 32 partial sums
    v = red[lane][warp];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    const uint32_t col = blockIdx.x * 32 + warp;
    if (lane == 0 && col < H) (s == 0 ? out0 : (s == 1 ? out1 : out2))[col] = v;
}

// Threads of a row's block when each holds `each` columns; 0: too long a row.
uint32_t row_threads(uint32_t H, uint32_t each, uint32_t most) {
    const uint32_t n = round_up(ceil_div(H, each), 32);
    return n <= most ? n : 0;
}

struct Sms {
    int device, count;
};
// A ring of `row` bytes a stage beside `other` bytes: up to four stages, and as
// many blocks as an SM's shared memory and `most` threads hold.
struct Ring {
    uint32_t stages, smem;
};
Ring ring_of(uint32_t row, uint32_t other, uint32_t threads, uint32_t most, uint32_t T, int sms) {
    Ring r = {};
    // blocks of an SM so that two stages of each fit, then the stages that are left
    const uint32_t per_sm = std::max(1u, std::min(most / threads, kMostSmem / (2 * row + other + 1024)));
    const uint32_t share = kMostSmem / per_sm - 1024;
    r.stages = std::min(kMostStages, std::max(1u, (share - std::min(share, other)) / row));
    r.stages = std::min(r.stages, std::max(1u, ceil_div(T, per_sm * sms)));  // no more than rows
    r.smem = r.stages * row + other;
    return r;
}

struct NormArgs {
    const void *hidden, *y;
    void *hidden_out, *x;
    float *rms_y, *rms_x;
};
template <typename DH, typename DY, typename DX>
cudaError_t run_forward(const NormArgs& a, const NormJob& job, bool vec, const Sms& sm, cudaStream_t st) {
    static std::atomic<uint64_t> set[1];
    auto go = [&](auto kernel, std::atomic<uint64_t>* done, uint32_t smem, dim3 threads, uint32_t blocks) {
        const cudaError_t e = done ? allow_smem(kernel, sm.device, done, kMostSmem) : cudaSuccess;
        if (e != cudaSuccess) return e;
        return launch_kernel(kernel, dim3(blocks), threads, smem, st, true,
                             static_cast<const typename DH::type*>(a.hidden),
                             static_cast<const typename DY::type*>(a.y), static_cast<typename DH::type*>(a.hidden_out),
                             static_cast<typename DX::type*>(a.x), a.rms_y, a.rms_x, job);
    };
    const bool full = a.y && job.post_w && a.x;
    // rows that a warp can hold
    constexpr int R = 4;
    const dim3 warps(32, R);
    const uint32_t few = ceil_div(job.T, R);
    if (vec && job.H <= 256) {
        return full ? go(norm_forward_kernel<DH, DY, DX, 4, 2, true, R, 128, 8>, nullptr, 0, warps, few)
                    : go(norm_forward_kernel<DH, DY, DX, 4, 2, false, R, 128, 8>, nullptr, 0, warps, few);
    }
    if (vec && job.H <= 512) {
        return full ? go(norm_forward_kernel<DH, DY, DX, 4, 4, true, R, 128, 8>, nullptr, 0, warps, few)
                    : go(norm_forward_kernel<DH, DY, DX, 4, 4, false, R, 128, 8>, nullptr, 0, warps, few);
    }
    // 16 columns a thread; 8 where they are read one by one, up to 4096 of them
    if (const uint32_t n = vec ? 0 : row_threads(job.H, 8, 512)) {
        return full ? go(norm_forward_kernel<DH, DY, DX, 1, 8, true, 1, 512, 2>, nullptr, 0, n, job.T)
                    : go(norm_forward_kernel<DH, DY, DX, 1, 8, false, 1, 512, 2>, nullptr, 0, n, job.T);
    }
    if (const uint32_t n = row_threads(job.H, 16, 512)) {
        if (full && vec) return go(norm_forward_kernel<DH, DY, DX, 4, 4, true, 1, 512, 2>, nullptr, 0, n, job.T);
        return vec ? go(norm_forward_kernel<DH, DY, DX, 4, 4, false, 1, 512, 2>, nullptr, 0, n, job.T)
                   : go(norm_forward_kernel<DH, DY, DX, 1, 16, false, 1, 512, 2>, nullptr, 0, n, job.T);
    }
    if (const uint32_t n = row_threads(job.H, 32, 512)) {
        return vec ? go(norm_forward_kernel<DH, DY, DX, 4, 8, false, 1, 512, 1>, nullptr, 0, n, job.T)
                   : go(norm_forward_kernel<DH, DY, DX, 1, 32, false, 1, 512, 1>, nullptr, 0, n, job.T);
    }
    return go(norm_forward_long_kernel<DH, DY, DX>, &set[0], job.H * 4, 512, job.T);
}

struct NormBackArgs {
    const void *d_hidden_out, *d_x, *hidden_out, *y;
    const float *rms_y, *rms_x;
    void *d_hidden, *d_y, *d_gate;
    NormSums sums;
};
template <typename DH, typename DY, typename DX>
cudaError_t run_backward(const NormBackArgs& a, NormJob job, bool vec, const Sms& sm, uint32_t blocks,
                         cudaStream_t st) {
    static std::atomic<uint64_t> set[17];
    auto go = [&](auto kernel, std::atomic<uint64_t>* done, uint32_t smem, uint32_t threads) {
        const cudaError_t e = done ? allow_smem(kernel, sm.device, done, kMostSmem) : cudaSuccess;
        if (e != cudaSuccess) return e;
        return launch_kernel(kernel, dim3(blocks), dim3(threads), smem, st, true,
                             static_cast<const typename DH::type*>(a.d_hidden_out),
                             static_cast<const typename DX::type*>(a.d_x),
                             static_cast<const typename DH::type*>(a.hidden_out),
                             static_cast<const typename DY::type*>(a.y), a.rms_y, a.rms_x,
                             static_cast<typename DH::type*>(a.d_hidden), static_cast<typename DY::type*>(a.d_y),
                             a.d_gate, a.sums, job);
    };
    job.stages = 1;
    const uint32_t n = row_threads(job.H, 8, kMostThreads);
    const uint32_t acc = a.sums.slots * job.H * 4;
    const bool full = a.d_hidden_out && a.d_x && a.y && job.post_w && a.d_hidden && a.d_y && a.sums.post >= 0 &&
                      a.sums.pre >= 0;
    const int kind = !full ? -1 : (job.gate_kind == MOE_B200_GATE_TOKEN ? 0 : job.gate_kind);
    constexpr int kChannel = MOE_B200_GATE_CHANNEL, kElement = MOE_B200_GATE_ELEMENT;
    if (n && vec) {
        const uint32_t hb = job.H * sizeof(typename DH::type), yb = job.H * sizeof(typename DY::type);
        const uint32_t row = (a.d_hidden_out ? hb : 0) + (a.d_x ? hb + job.H * (uint32_t)sizeof(typename DX::type) : 0) +
                             (a.y ? yb : 0) + (a.y && job.gate_kind == MOE_B200_GATE_ELEMENT ? yb : 0);
        if (row + acc <= kMostSmem) {
            // not in the kernels that keep the weights in registers (rows of 2049 to 4096: 4,096
            // x 4096 bf16 60 us, with the weights in shared memory 62)
            job.stage_weights = (n > 512 || (n <= 256 && full)) && row + acc + 8 * job.H <= kMostSmem;
            const Ring r = ring_of(row, acc + (job.stage_weights ? 8 * job.H : 0), n, n <= 512 ? 768 : 1024, job.T,
                                   sm.count);
            job.stages = r.stages;
            if (n <= 256) {
                if (kind == 0) return go(norm_backward_kernel<DH, DY, DX, 8, 1, true, 0, 256>, &set[0], r.smem, n);
                if (kind == kChannel)
                    return go(norm_backward_kernel<DH, DY, DX, 8, 1, true, kChannel, 256>, &set[1], r.smem, n);
                if (kind == kElement)
                    return go(norm_backward_kernel<DH, DY, DX, 8, 1, true, kElement, 256>, &set[2], r.smem, n);
            }
            if (n > 256 && n <= 512) {
                if (kind == 0) return go(norm_backward_kernel<DH, DY, DX, 8, 1, true, 0, 512>, &set[14], r.smem, n);
                if (kind == kChannel)
                    return go(norm_backward_kernel<DH, DY, DX, 8, 1, true, kChannel, 512>, &set[15], r.smem, n);
                if (kind == kElement)
                    return go(norm_backward_kernel<DH, DY, DX, 8, 1, true, kElement, 512>, &set[16], r.smem, n);
            }
            if (n > 512) {
                if (kind == 0)
                    return go(norm_backward_kernel<DH, DY, DX, 8, 1, true, 0, kMostThreads>, &set[3], r.smem, n);
                if (kind == kChannel)
                    return go(norm_backward_kernel<DH, DY, DX, 8, 1, true, kChannel, kMostThreads>, &set[4], r.smem, n);
                return go(norm_backward_kernel<DH, DY, DX, 8, 1, true, -1, kMostThreads>, &set[5], r.smem, n);
            }
            return go(norm_backward_kernel<DH, DY, DX, 8, 1, true, -1, 512>, &set[6], r.smem, n);
        }
    }
    if (n && !vec) {
        if (n <= 512) {
            if (kind == 0) return go(norm_backward_kernel<DH, DY, DX, 1, 8, false, 0, 512>, &set[7], acc, n);
            if (kind == kChannel) return go(norm_backward_kernel<DH, DY, DX, 1, 8, false, kChannel, 512>, &set[8], acc, n);
            if (kind == kElement) return go(norm_backward_kernel<DH, DY, DX, 1, 8, false, kElement, 512>, &set[9], acc, n);
            return go(norm_backward_kernel<DH, DY, DX, 1, 8, false, -1, 512>, &set[10], acc, n);
        }
        if (kind == 0) return go(norm_backward_kernel<DH, DY, DX, 1, 8, false, 0, kMostThreads>, &set[11], acc, n);
        if (kind == kChannel)
            return go(norm_backward_kernel<DH, DY, DX, 1, 8, false, kChannel, kMostThreads>, &set[12], acc, n);
        return go(norm_backward_kernel<DH, DY, DX, 1, 8, false, -1, kMostThreads>, &set[13], acc, n);
    }
    return vec ? go(norm_backward_kernel<DH, DY, DX, 8, 0, false, -1, 512>, nullptr, 0, 512)
               : go(norm_backward_kernel<DH, DY, DX, 1, 0, false, -1, 512>, nullptr, 0, 512);
}

#define NORM_BY_TYPE(CALL)                                                                                      \
    (cfg.hidden_type == MOE_B200_DTYPE_F32                                                                      \
         ? (cfg.y_type == MOE_B200_DTYPE_F32                                                                    \
                ? (cfg.x_type == MOE_B200_DTYPE_F32 ? CALL(F32, F32, F32) : CALL(F32, F32, BF16))               \
                : (cfg.x_type == MOE_B200_DTYPE_F32 ? CALL(F32, BF16, F32) : CALL(F32, BF16, BF16)))            \
         : (cfg.y_type == MOE_B200_DTYPE_F32                                                                    \
                ? (cfg.x_type == MOE_B200_DTYPE_F32 ? CALL(BF16, F32, F32) : CALL(BF16, F32, BF16))             \
                : (cfg.x_type == MOE_B200_DTYPE_F32 ? CALL(BF16, BF16, F32) : CALL(BF16, BF16, BF16))))

int check_norm(const moe_b200_residual_norm_cfg_t* in, moe_b200_residual_norm_cfg_t* cfg, char* err) {
    if (!in) {
        set_err(err, "null norm config");
        return 0;
    }
    *cfg = *in;
    if (cfg->hidden == 0 || cfg->hidden > kMaxHidden) {
        set_err(err, "hidden=%u outside 1..%u", cfg->hidden, kMaxHidden);
        return 0;
    }
    if (cfg->tokens >= (1u << 31)) {
        set_err(err, "tokens=%u: 2^31 or more", cfg->tokens);
        return 0;
    }
    if (!row_type_ok(cfg->hidden_type) || !row_type_ok(cfg->y_type) || !row_type_ok(cfg->x_type)) {
        set_err(err, "row types %d, %d, %d: fp32 or bf16", cfg->hidden_type, cfg->y_type, cfg->x_type);
        return 0;
    }
    if (cfg->gate < MOE_B200_GATE_NONE || cfg->gate > MOE_B200_GATE_ELEMENT) {
        set_err(err, "unknown gate kind %d", cfg->gate);
        return 0;
    }
    return check_stride("hidden_stride", &cfg->hidden_stride, cfg->hidden, err) &&
           check_stride("y_stride", &cfg->y_stride, cfg->hidden, err) &&
           check_stride("x_stride", &cfg->x_stride, cfg->hidden, err);
}
Span gate_span(const char* name, const void* p, const moe_b200_residual_norm_cfg_t& c) {
    if (c.gate == MOE_B200_GATE_ELEMENT) return row_span(name, p, c.tokens, c.hidden, c.y_stride, c.y_type);
    return {name, p, 4ull * (c.gate == MOE_B200_GATE_TOKEN ? c.tokens : c.hidden)};
}
NormJob norm_job(const moe_b200_residual_norm_cfg_t& c, const float* post_w, const void* gate, const float* pre_w,
                 const moe_b200_engine* eng) {
    return {c.hidden, c.tokens, c.hidden_stride, c.y_stride, c.x_stride, post_w, pre_w, gate, c.gate,
            c.gate_sigmoid, c.norm_unit_offset ? 1.0f : 0.0f, c.norm_eps > 0.0f ? c.norm_eps : 1e-6f,
            c.residual_scale != 0.0f ? c.residual_scale : 1.0f, c.out_scale != 0.0f ? c.out_scale : 1.0f,
            1.0f / (float)c.hidden, 1, 0, eng->err_word.as<uint32_t>()};
}
bool norm_vec(const moe_b200_residual_norm_cfg_t& c, std::initializer_list<const void*> h,
              std::initializer_list<const void*> y, std::initializer_list<const void*> x,
              std::initializer_list<const void*> f32) {
    bool ok = c.hidden % 8 == 0;
    for (const void* p : h) ok &= rows_vec8(p, c.hidden_stride, c.hidden_type);
    for (const void* p : y) ok &= rows_vec8(p, c.y_stride, c.y_type);
    for (const void* p : x) ok &= rows_vec8(p, c.x_stride, c.x_type);
    for (const void* p : f32) ok &= aligned_to(p, 16);
    return ok;
}

constexpr int32_t kF32 = MOE_B200_DTYPE_F32;

}  // namespace
}  // namespace moe_b200

using namespace moe_b200;

extern "C" {

int moe_b200_residual_norm_forward(moe_b200_engine_t* eng, const moe_b200_residual_norm_cfg_t* cfg_in,
                                   const void* hidden, const void* y, const float* post_w, const void* gate,
                                   const float* pre_w, void* hidden_out, void* x, float* rms_y, float* rms_x,
                                   void* stream, char* err) {
    moe_b200_residual_norm_cfg_t cfg;
    if (!check_norm(cfg_in, &cfg, err)) return 0;
    const uint64_t T = cfg.tokens, H = cfg.hidden;
    const Span ins[] = {row_span("hidden", hidden, T, H, cfg.hidden_stride, cfg.hidden_type),
                        row_span("y", y, T, H, cfg.y_stride, cfg.y_type),
                        {"post_w", post_w, H * 4},
                        gate_span("gate", cfg.gate ? gate : nullptr, cfg),
                        {"pre_w", pre_w, H * 4}};
    const Span outs[] = {row_span("hidden_out", hidden_out, T, H, cfg.hidden_stride, cfg.hidden_type),
                         row_span("x", x, T, H, cfg.x_stride, cfg.x_type),
                         {"rms_y", rms_y, T * 4},
                         {"rms_x", rms_x, T * 4}};
    if (T) {  // without rows, empty buffers may have no address
        if (!check_given(ins[0], err) || (y && !check_given(outs[0], err))) return 0;
        if (!x && !y) {
            set_err(err, "neither y nor x: nothing to compute");
            return 0;
        }
        if (x && !check_given(ins[4], err)) return 0;
        if (!y && (post_w || rms_y || (gate && cfg.gate))) {
            set_err(err, "post_w, gate and rms_y go with y");
            return 0;
        }
        if (y && cfg.gate && !check_given(ins[3], err)) return 0;
        if (!post_w && rms_y) {
            set_err(err, "rms_y goes with post_w");
            return 0;
        }
        if (!x && (pre_w || rms_x)) {
            set_err(err, "pre_w and rms_x go with x");
            return 0;
        }
    }
    const int32_t in_types[] = {cfg.hidden_type, cfg.y_type, kF32,
                                cfg.gate == MOE_B200_GATE_ELEMENT ? cfg.y_type : kF32, kF32};
    const int32_t out_types[] = {cfg.hidden_type, cfg.x_type, kF32, kF32};
    for (int i = 0; i < 5; ++i) {
        if (!check_aligned(ins[i], type_bytes(in_types[i]), err)) return 0;
    }
    for (int i = 0; i < 4; ++i) {
        if (!check_aligned(outs[i], type_bytes(out_types[i]), err)) return 0;
    }
    const bool x_in_y = cfg.x_type == cfg.y_type && cfg.x_stride == cfg.y_stride;
    const char* const same[][2] = {{"hidden_out", "hidden"}, {"x", "y"}};
    if (!check_overlap(outs, 4, ins, 5, same, x_in_y ? 2 : 1, err)) return 0;
    OnDevice on(eng, err);
    if (!on.ok) return 0;
    if (T == 0) return 1;
    const NormJob job = norm_job(cfg, post_w, gate, pre_w, eng);
    const bool element = y && cfg.gate == MOE_B200_GATE_ELEMENT;
    const bool vec = norm_vec(cfg, {hidden, hidden_out}, {y, element ? gate : nullptr}, {x},
                              {post_w, pre_w, y && cfg.gate == MOE_B200_GATE_CHANNEL ? gate : nullptr});
    const NormArgs a = {hidden, y, hidden_out, x, rms_y, rms_x};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
#define CALL_NORM(DH, DY, DX) run_forward<DH, DY, DX>(a, job, vec, {eng->device, eng->num_sms}, st)
    return launched(NORM_BY_TYPE(CALL_NORM), "residual norm", err);
}

uint64_t moe_b200_residual_norm_workspace_bytes(const moe_b200_residual_norm_cfg_t* cfg_in) {
    moe_b200_residual_norm_cfg_t cfg;
    if (!check_norm(cfg_in, &cfg, nullptr)) return 0;  // the call itself says why
    const uint64_t slots = cfg.gate == MOE_B200_GATE_CHANNEL ? 3 : 2;
    return std::min<uint64_t>(cfg.tokens, norm_blocks(cfg.hidden)) * slots * cfg.hidden * 4;
}

int moe_b200_residual_norm_backward(moe_b200_engine_t* eng, const moe_b200_residual_norm_cfg_t* cfg_in,
                                    const void* d_hidden_out, const void* d_x, const void* hidden_out, const void* y,
                                    const float* post_w, const void* gate, const float* pre_w, const float* rms_y,
                                    const float* rms_x, void* d_hidden, void* d_y, float* d_post_w, void* d_gate,
                                    float* d_pre_w, void* workspace, uint64_t workspace_bytes, void* stream,
                                    char* err) {
    moe_b200_residual_norm_cfg_t cfg;
    if (!check_norm(cfg_in, &cfg, err)) return 0;
    const uint64_t T = cfg.tokens, H = cfg.hidden;
    const uint32_t blocks = std::min(cfg.tokens, norm_blocks(cfg.hidden));
    NormSums sums = {-1, -1, -1, 0, static_cast<float*>(workspace)};
    if (d_post_w) sums.post = sums.slots++;
    if (d_pre_w) sums.pre = sums.slots++;
    if (d_gate && cfg.gate == MOE_B200_GATE_CHANNEL) sums.gate = sums.slots++;
    const uint64_t need = (uint64_t)blocks * sums.slots * H * 4;
    const Span ins[] = {row_span("d_hidden_out", d_hidden_out, T, H, cfg.hidden_stride, cfg.hidden_type),
                        row_span("d_x", d_x, T, H, cfg.x_stride, cfg.x_type),
                        row_span("hidden_out", hidden_out, T, H, cfg.hidden_stride, cfg.hidden_type),
                        row_span("y", y, T, H, cfg.y_stride, cfg.y_type),
                        {"post_w", post_w, H * 4},
                        gate_span("gate", cfg.gate ? gate : nullptr, cfg),
                        {"pre_w", pre_w, H * 4},
                        {"rms_y", rms_y, T * 4},
                        {"rms_x", rms_x, T * 4}};
    const Span outs[] = {row_span("d_hidden", d_hidden, T, H, cfg.hidden_stride, cfg.hidden_type),
                         row_span("d_y", d_y, T, H, cfg.y_stride, cfg.y_type),
                         {"d_post_w", d_post_w, H * 4},
                         gate_span("d_gate", cfg.gate ? d_gate : nullptr, cfg),
                         {"d_pre_w", d_pre_w, H * 4},
                         {"workspace", workspace, need}};
    if (T) {
        if (!d_hidden_out && !d_x) {
            set_err(err, "neither d_hidden_out nor d_x is given");
            return 0;
        }
        if (d_x && (!check_given(ins[2], err) || !check_given(ins[6], err) || !check_given(ins[8], err))) return 0;
        if (d_pre_w && !d_x) {
            set_err(err, "d_pre_w needs d_x");
            return 0;
        }
        if (!y && (post_w || d_y || d_post_w || d_gate || (gate && cfg.gate))) {
            set_err(err, "post_w, gate and their gradients go with y");
            return 0;
        }
        if (y && post_w && !check_given(ins[7], err)) return 0;
        if (y && cfg.gate && !check_given(ins[5], err)) return 0;
        if (d_post_w && !check_given(ins[4], err)) return 0;
        if (!d_hidden && !d_y && !d_post_w && !d_gate && !d_pre_w) {
            set_err(err, "no gradient is asked for");
            return 0;
        }
    }
    if (d_gate && !cfg.gate) {
        set_err(err, "d_gate without a gate");
        return 0;
    }
    if (need && (!workspace || workspace_bytes < need)) {
        set_err(err, "the gradients need a workspace of %llu bytes (%llu given)", (unsigned long long)need,
                (unsigned long long)(workspace ? workspace_bytes : 0));
        return 0;
    }
    const int32_t gate_type = cfg.gate == MOE_B200_GATE_ELEMENT ? cfg.y_type : kF32;
    const int32_t in_types[] = {cfg.hidden_type, cfg.x_type, cfg.hidden_type, cfg.y_type, kF32, gate_type, kF32, kF32,
                                kF32};
    const int32_t out_types[] = {cfg.hidden_type, cfg.y_type, kF32, gate_type, kF32, kF32};
    for (int i = 0; i < 9; ++i) {
        if (!check_aligned(ins[i], type_bytes(in_types[i]), err)) return 0;
    }
    for (int i = 0; i < 6; ++i) {
        if (!check_aligned(outs[i], type_bytes(out_types[i]), err)) return 0;
    }
    if (need && !check_aligned(outs[5], 16, err)) return 0;
    const char* const same[][2] = {{"d_hidden", "d_hidden_out"}, {"d_y", "y"}};
    if (!check_overlap(outs, 6, ins, 9, same, 2, err)) return 0;
    OnDevice on(eng, err);
    if (!on.ok) return 0;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    float* const slot_out[3] = {sums.post == 0 ? d_post_w : (sums.pre == 0 ? d_pre_w : static_cast<float*>(d_gate)),
                                sums.pre == 1 ? d_pre_w : static_cast<float*>(d_gate), static_cast<float*>(d_gate)};
    if (T) {
        const NormJob job = norm_job(cfg, post_w, gate, pre_w, eng);
        const bool element = y && cfg.gate == MOE_B200_GATE_ELEMENT;
        const bool vec = norm_vec(cfg, {d_hidden_out, d_x ? hidden_out : nullptr, d_hidden},
                                  {y, d_y, element ? gate : nullptr, element ? d_gate : nullptr}, {d_x},
                                  {post_w, d_x ? pre_w : nullptr,
                                   y && cfg.gate == MOE_B200_GATE_CHANNEL ? gate : nullptr});
        const NormBackArgs a = {d_hidden_out, d_x, hidden_out, y, rms_y, rms_x, d_hidden, d_y, d_gate, sums};
#define CALL_NORM_BACK(DH, DY, DX) run_backward<DH, DY, DX>(a, job, vec, {eng->device, eng->num_sms}, blocks, st)
        if (!launched(NORM_BY_TYPE(CALL_NORM_BACK), "residual norm gradient", err)) return 0;
    }
    if (sums.slots == 0) return 1;
    return launched(launch_kernel(norm_sums_kernel, dim3(ceil_div(cfg.hidden, 32), sums.slots), dim3(1024), 0, st, true,
                                  static_cast<const float*>(sums.part), blocks, cfg.hidden, sums.slots, slot_out[0],
                                  slot_out[1], slot_out[2]),
                    "residual norm gradient", err);
}

}  // extern "C"
