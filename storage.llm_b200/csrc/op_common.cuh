// What the stand-alone operators (rows.cu, residual_norm.cu, q4.cu) share:
// rows of fp32 or bf16 read and written as fp32 values, the host's argument
// checks, and the launch on the engine's device.
#pragma once

#include <atomic>
#include <cstdint>

#include <algorithm>

#include "engine.h"

namespace moe_b200 {

// ---------------------------------------------------------------------------
// Rows as fp32 values.  V = 8: 16-byte aligned rows whose length is a multiple
// of 8 (one 16-byte access for bf16, two for fp32); V = 4: the same rows (one
// access of 8 or 16 bytes); V = 1: any row.
// ---------------------------------------------------------------------------
struct F32 {
    using type = float;
};
struct BF16 {
    using type = uint16_t;
};

__device__ __forceinline__ float bf16_lo(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t p) { return __uint_as_float(p & 0xffff0000u); }
// two values rounded to nearest even, `a` in the low half
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    uint32_t u;
    memcpy(&u, &v, 4);
    return u;
}
__device__ __forceinline__ uint16_t bf16_one(float a) { return __bfloat16_as_ushort(__float2bfloat16_rn(a)); }

// A vector as it lies in memory, so that loads can be issued well before
// their values are used.
template <typename D, int V>
struct Raw;
template <>
struct Raw<F32, 8> {
    uint4 a, b;
};
template <>
struct Raw<BF16, 8> {
    uint4 a;
};
template <>
struct Raw<F32, 4> {
    uint4 a;
};
template <>
struct Raw<BF16, 4> {
    uint2 a;
};
template <>
struct Raw<F32, 1> {
    float a;
};
template <>
struct Raw<BF16, 1> {
    uint16_t a;
};

// Each row element is used once, so loads and stores are marked as streams.
__device__ __forceinline__ Raw<F32, 8> load_raw(const float* p, F32*, Raw<F32, 8>*) {
    const uint4* q = reinterpret_cast<const uint4*>(p);
    return {__ldcs(q), __ldcs(q + 1)};
}
__device__ __forceinline__ Raw<BF16, 8> load_raw(const uint16_t* p, BF16*, Raw<BF16, 8>*) {
    return {__ldcs(reinterpret_cast<const uint4*>(p))};
}
__device__ __forceinline__ Raw<F32, 4> load_raw(const float* p, F32*, Raw<F32, 4>*) {
    return {__ldcs(reinterpret_cast<const uint4*>(p))};
}
__device__ __forceinline__ Raw<BF16, 4> load_raw(const uint16_t* p, BF16*, Raw<BF16, 4>*) {
    return {__ldcs(reinterpret_cast<const uint2*>(p))};
}
__device__ __forceinline__ Raw<F32, 1> load_raw(const float* p, F32*, Raw<F32, 1>*) { return {__ldcs(p)}; }
__device__ __forceinline__ Raw<BF16, 1> load_raw(const uint16_t* p, BF16*, Raw<BF16, 1>*) { return {__ldcs(p)}; }

template <typename D, int V>
__device__ __forceinline__ Raw<D, V> load_row(const typename D::type* p) {
    return load_raw(p, static_cast<D*>(nullptr), static_cast<Raw<D, V>*>(nullptr));
}

__device__ __forceinline__ void unpack(const Raw<F32, 8>& r, float* v) {
    v[0] = __uint_as_float(r.a.x), v[1] = __uint_as_float(r.a.y), v[2] = __uint_as_float(r.a.z);
    v[3] = __uint_as_float(r.a.w), v[4] = __uint_as_float(r.b.x), v[5] = __uint_as_float(r.b.y);
    v[6] = __uint_as_float(r.b.z), v[7] = __uint_as_float(r.b.w);
}
__device__ __forceinline__ void unpack(const Raw<BF16, 8>& r, float* v) {
    v[0] = bf16_lo(r.a.x), v[1] = bf16_hi(r.a.x), v[2] = bf16_lo(r.a.y), v[3] = bf16_hi(r.a.y);
    v[4] = bf16_lo(r.a.z), v[5] = bf16_hi(r.a.z), v[6] = bf16_lo(r.a.w), v[7] = bf16_hi(r.a.w);
}
__device__ __forceinline__ void unpack(const Raw<F32, 4>& r, float* v) {
    v[0] = __uint_as_float(r.a.x), v[1] = __uint_as_float(r.a.y);
    v[2] = __uint_as_float(r.a.z), v[3] = __uint_as_float(r.a.w);
}
__device__ __forceinline__ void unpack(const Raw<BF16, 4>& r, float* v) {
    v[0] = bf16_lo(r.a.x), v[1] = bf16_hi(r.a.x), v[2] = bf16_lo(r.a.y), v[3] = bf16_hi(r.a.y);
}
__device__ __forceinline__ void unpack(const Raw<F32, 1>& r, float* v) { v[0] = r.a; }
__device__ __forceinline__ void unpack(const Raw<BF16, 1>& r, float* v) { v[0] = bf16_lo(r.a); }

// The one rounding of an fp32 result to the row's type (round to nearest even).
__device__ __forceinline__ void pack(const float* v, Raw<F32, 8>& r) {
    r.a = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    r.b = make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]));
}
__device__ __forceinline__ void pack(const float* v, Raw<BF16, 8>& r) {
    r.a = make_uint4(bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]), bf16_pair(v[4], v[5]), bf16_pair(v[6], v[7]));
}
__device__ __forceinline__ void pack(const float* v, Raw<F32, 4>& r) {
    r.a = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
}
__device__ __forceinline__ void pack(const float* v, Raw<BF16, 4>& r) {
    r.a = make_uint2(bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]));
}
__device__ __forceinline__ void pack(const float* v, Raw<F32, 1>& r) { r.a = v[0]; }
__device__ __forceinline__ void pack(const float* v, Raw<BF16, 1>& r) { r.a = bf16_one(v[0]); }

__device__ __forceinline__ void store_row(float* p, const Raw<F32, 8>& r) {
    uint4* q = reinterpret_cast<uint4*>(p);
    __stcs(q, r.a);
    __stcs(q + 1, r.b);
}
__device__ __forceinline__ void store_row(uint16_t* p, const Raw<BF16, 8>& r) {
    __stcs(reinterpret_cast<uint4*>(p), r.a);
}
__device__ __forceinline__ void store_row(float* p, const Raw<F32, 4>& r) { __stcs(reinterpret_cast<uint4*>(p), r.a); }
__device__ __forceinline__ void store_row(uint16_t* p, const Raw<BF16, 4>& r) {
    __stcs(reinterpret_cast<uint2*>(p), r.a);
}
__device__ __forceinline__ void store_row(float* p, const Raw<F32, 1>& r) { __stcs(p, r.a); }
__device__ __forceinline__ void store_row(uint16_t* p, const Raw<BF16, 1>& r) { __stcs(p, r.a); }

// fp32 vectors of V values (weights, sums)
template <int V>
__device__ __forceinline__ void load_f32(const float* p, float* v) {
    if constexpr (V == 8) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else if constexpr (V == 4) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(p));
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    } else {
        v[0] = __ldg(p);
    }
}

// ---------------------------------------------------------------------------
// Vectors of V fp32 values; for V = 4 and 8 two values an instruction.  Nothing is
// contracted, so the general and the specialised kernels of one V give the same
// bits.  Kernels of another V give threads other columns and vdot other sums:
// their sums over a row differ in the last places.
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint64_t two(float lo, float hi) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
    return v;
}
__device__ __forceinline__ void apart(uint64_t v, float& lo, float& hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
// d = a * b
template <int V>
__device__ __forceinline__ void vmul(float* d, const float* a, const float* b) {
    if constexpr (V > 1) {
#pragma unroll
        for (int k = 0; k < V; k += 2) {
            uint64_t r;
            asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(two(a[k], a[k + 1])), "l"(two(b[k], b[k + 1])));
            apart(r, d[k], d[k + 1]);
        }
    } else {
        d[0] = __fmul_rn(a[0], b[0]);
    }
}
template <int V>
__device__ __forceinline__ void vmul(float* d, const float* a, float b) {
    const float bs[8] = {b, b, b, b, b, b, b, b};
    vmul<V>(d, a, bs);
}
// d = a * b + c
template <int V>
__device__ __forceinline__ void vfma(float* d, const float* a, const float* b, const float* c) {
    if constexpr (V > 1) {
#pragma unroll
        for (int k = 0; k < V; k += 2) {
            uint64_t r;
            asm("fma.rn.f32x2 %0, %1, %2, %3;"
                : "=l"(r)
                : "l"(two(a[k], a[k + 1])), "l"(two(b[k], b[k + 1])), "l"(two(c[k], c[k + 1])));
            apart(r, d[k], d[k + 1]);
        }
    } else {
        d[0] = fmaf(a[0], b[0], c[0]);
    }
}
template <int V>
__device__ __forceinline__ void vfma(float* d, const float* a, float b, const float* c) {
    const float bs[8] = {b, b, b, b, b, b, b, b};
    vfma<V>(d, a, bs, c);
}
// d += a
template <int V>
__device__ __forceinline__ void vadd(float* d, const float* a) {
    if constexpr (V > 1) {
#pragma unroll
        for (int k = 0; k < V; k += 2) {
            uint64_t r;
            asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(two(d[k], d[k + 1])), "l"(two(a[k], a[k + 1])));
            apart(r, d[k], d[k + 1]);
        }
    } else {
        d[0] = __fadd_rn(d[0], a[0]);
    }
}
template <int V>
__device__ __forceinline__ void vadd(float* d, float a) {
    const float as[8] = {a, a, a, a, a, a, a, a};
    vadd<V>(d, as);
}
// s += a * b, in two sums
template <int V>
__device__ __forceinline__ void vdot(float (&s)[2], const float* a, const float* b) {
    if constexpr (V > 1) {
#pragma unroll
        for (int k = 0; k < V; k += 2) {
            uint64_t r;
            asm("fma.rn.f32x2 %0, %1, %2, %3;"
                : "=l"(r)
                : "l"(two(a[k], a[k + 1])), "l"(two(b[k], b[k + 1])), "l"(two(s[0], s[1])));
            apart(r, s[0], s[1]);
        }
    } else {
        s[0] = fmaf(a[0], b[0], s[0]);
    }
}

// The lanes' sums of four values: lane l gets that of value l & 3 (six
// exchanges where one value after the other takes twenty).
__device__ __forceinline__ float lanes_sum4(const float (&v)[4]) {
    const uint32_t lane = threadIdx.x & 31;
    const bool odd = lane & 1, high = lane & 2;
    const float a = (odd ? v[1] : v[0]) + __shfl_xor_sync(0xffffffffu, odd ? v[0] : v[1], 1);
    const float b = (odd ? v[3] : v[2]) + __shfl_xor_sync(0xffffffffu, odd ? v[2] : v[3], 1);
    float s = (high ? b : a) + __shfl_xor_sync(0xffffffffu, high ? a : b, 2);
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
inline bool row_type_ok(int32_t t) { return t == MOE_B200_DTYPE_F32 || t == MOE_B200_DTYPE_BF16; }
inline uint32_t type_bytes(int32_t t) {
    return t == MOE_B200_DTYPE_F32 ? 4u : (t == MOE_B200_DTYPE_E8M0 ? 1u : 2u);
}
inline bool aligned_to(const void* p, uint64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// Device memory of one operand, for the checks of null pointers, alignment and overlap.
struct Span {
    const char* name;
    const void* p;
    uint64_t bytes;
    uint64_t row = 0, pitch = 0;  // bytes of a row and from row to row (0: one piece)
};
inline Span row_span(const char* name, const void* p, uint64_t rows, uint64_t hidden, uint64_t stride,
                     int32_t type) {
    const uint64_t b = type_bytes(type);
    return {name, p, rows ? ((rows - 1) * stride + hidden) * b : 0, hidden * b, stride * b};
}
inline bool overlap(const Span& a, const Span& b) {
    if (!a.p || !b.p || !a.bytes || !b.bytes) return false;
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(b.p);
    if (x >= y + b.bytes || y >= x + a.bytes) return false;
    if (a.pitch && a.pitch == b.pitch) {
        // two column ranges of the same wider rows
        const uint64_t d = y >= x ? (y - x) % a.pitch : (a.pitch - (x - y) % a.pitch) % a.pitch;
        return d < a.row || a.pitch - d < b.row;
    }
    return true;
}
// Refuses an output that overlaps another operand.  `same` lists pairs of
// (output, input) names that may be one and the same buffer.
inline int check_overlap(const Span* outs, int n_out, const Span* ins, int n_in, const char* const (*same)[2],
                         int n_same, char* err) {
    for (int i = 0; i < n_out; ++i) {
        for (int j = 0; j < i; ++j) {
            if (overlap(outs[i], outs[j])) {
                set_err(err, "%s overlaps %s", outs[i].name, outs[j].name);
                return 0;
            }
        }
        for (int j = 0; j < n_in; ++j) {
            if (!overlap(outs[i], ins[j])) continue;
            bool ok = false;
            for (int k = 0; k < n_same && outs[i].p == ins[j].p && outs[i].bytes == ins[j].bytes; ++k) {
                ok |= !strcmp(same[k][0], outs[i].name) && !strcmp(same[k][1], ins[j].name);
            }
            if (!ok) {
                set_err(err, "%s overlaps %s", outs[i].name, ins[j].name);
                return 0;
            }
        }
    }
    return 1;
}
inline int check_aligned(const Span& s, uint64_t bytes, char* err) {
    if (aligned_to(s.p, bytes)) return 1;
    set_err(err, "%s is not aligned to %u bytes", s.name, (unsigned)bytes);
    return 0;
}
inline int check_given(const Span& s, char* err) {
    if (s.p) return 1;
    set_err(err, "null %s", s.name);
    return 0;
}
// A row stride: 0 = rows back to back.
inline int check_stride(const char* name, uint64_t* stride, uint64_t hidden, char* err) {
    if (*stride == 0) *stride = hidden;
    if (*stride < hidden || *stride > (1ull << 40)) {
        set_err(err, "%s %llu is shorter than a row of %llu (or above 2^40)", name, (unsigned long long)*stride,
                (unsigned long long)hidden);
        return 0;
    }
    return 1;
}
// Rows that the vector kernels can take.
inline bool rows_vec8(const void* p, uint64_t stride, int32_t type) {
    return !p || (aligned_to(p, 16) && (stride * type_bytes(type)) % 16 == 0);
}

// Makes the engine's device current for one call and puts the caller's back.
class OnDevice {
  public:
    OnDevice(const moe_b200_engine* eng, char* err) {
        if (!eng) {
            set_err(err, "null engine");
            return;
        }
        cudaError_t e = cudaGetDevice(&before_);
        if (e == cudaSuccess && before_ != eng->device) {
            e = cudaSetDevice(eng->device);
            changed_ = e == cudaSuccess;
        }
        if (e != cudaSuccess) {
            set_err(err, "cannot make device %d current: %s", eng->device, cudaGetErrorString(e));
            return;
        }
        ok = true;
    }
    ~OnDevice() {
        if (changed_) cudaSetDevice(before_);
    }
    OnDevice(const OnDevice&) = delete;
    OnDevice& operator=(const OnDevice&) = delete;
    bool ok = false;

  private:
    int before_ = 0;
    bool changed_ = false;
};

inline int launched(cudaError_t e, const char* what, char* err) {
    if (e == cudaSuccess) return 1;
    set_err(err, "%s launch failed: %s", what, cudaGetErrorString(e));
    return 0;
}

// Shared memory above 48 KB has to be asked for once on each device.
template <typename Kernel>
inline cudaError_t allow_smem(Kernel* kernel, int device, std::atomic<uint64_t>* done, int bytes) {
    if (device < 64 && ((done->load(std::memory_order_relaxed) >> device) & 1u)) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && device < 64) done->fetch_or(1ull << device, std::memory_order_relaxed);
    return e;
}

}  // namespace moe_b200
