// il_logits.cuh -- what the operators on logits rows share: rows of a strided
// [B, T, V] tensor, the running softmax sums, and the warp, CTA and cluster
// reductions of them.
//
// A row z of V logits at temperature tau is reduced to
//   m = max_j z_j,   s = sum_j e_j,   u = sum_j e_j d_j
//   with d_j = (z_j - m) log2(e) / tau and e_j = 2^d_j,
// so that log sum_j exp(z_j / tau) = m / tau + ln s and the entropy of
// softmax(z / tau) is ln s - ln(2) u / s.  One pass holds (m, s, u) per thread
// and rescales s and u when m grows; partial results are joined in a fixed
// order, so that a call's results do not change from run to run.
//
// Values outside the finite numbers: -inf adds nothing (d is held at -150,
// where 2^d is 0 and d itself stays finite); a row of nothing but -inf ends
// with s = 0; NaN or +inf makes s NaN.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "il_common.cuh"
#include "il_sm100.cuh"

namespace il {

constexpr int kMaxTop = 128;         // alternatives, or the teacher's slots, of a row
constexpr int kMaxVocab = 1 << 21;   // a row split over 16 CTAs keeps its bitmap in shared memory
constexpr int kWarpVocab = 1024;     // rows up to this long are held in one warp's registers
constexpr int kRowThreads = 512;     // CTA of the longer rows
constexpr int kRowElems = 16;        // logits that a thread holds at a time
constexpr int kMaxCluster = 16;

// rows r = b*T + t of a [B, T, V] tensor whose last dimension is contiguous
struct RowsIn {
    const void* p;
    int64_t sb, st;
    uint32_t T;
};
struct RowsOut {
    void* p;
    int64_t sb, st;
    uint32_t T;
};
struct Tokens {  // [B, T] int64; p == nullptr: none
    const int64_t* p;
    int64_t sb, st, ignore;
};

__device__ __forceinline__ int64_t row_offset(int64_t sb, int64_t st, uint32_t T, uint32_t row) {
    const uint32_t b = row / T;
    return (int64_t)b * sb + (int64_t)(row - b * T) * st;
}

template <int DT>
struct Elem;
template <>
struct Elem<kF32> {
    using type = float;
    static constexpr int kVec = 4;  // elements of 16 bytes
};
template <>
struct Elem<kBF16> {
    using type = __nv_bfloat16;
    static constexpr int kVec = 8;
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class E>
__device__ __forceinline__ E from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

// 16 bytes to floats and back
template <int DT>
__device__ __forceinline__ void unpack16(const uint4& r, float* x) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (DT == kF32) {
            x[i] = __uint_as_float(w[i]);
        } else {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
}
template <int DT>
__device__ __forceinline__ uint4 pack16(const float* x) {
    uint4 r;
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (DT == kF32) {
            w[i] = __float_as_uint(x[i]);
        } else {
            const __nv_bfloat162 v = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&v);
        }
    }
    r.x = w[0], r.y = w[1], r.z = w[2], r.w = w[3];
    return r;
}
// 16 bytes of -inf
template <int DT>
__device__ __forceinline__ uint4 neg_inf16() {
    const uint32_t w = DT == kF32 ? 0xff800000u : 0xff80ff80u;
    return make_uint4(w, w, w, w);
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// max that keeps NaN
__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

constexpr float kLn2 = 0.693147180559945309f;
constexpr float kMinExp = -150.0f;

// (z - m) in units of the base-2 exponent; finite unless NaN
__device__ __forceinline__ float exponent(float z, float m, float c) { return max_nan((z - m) * c, kMinExp); }
// the value that is subtracted for a maximum m: m itself, or 0 where nothing is above -inf
__device__ __forceinline__ float shift_of(float m) { return m == -INFINITY ? 0.0f : m; }

// running sums of one thread, warp, CTA or row; s1: the sum at temperature 1
struct Sums {
    float m, s, u, s1;
};

__device__ __forceinline__ Sums no_sums() { return Sums{-INFINITY, 0.0f, 0.0f, 0.0f}; }

// c = log2(e) / tau, c1 = log2(e)
template <bool U, bool S1>
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b, float c, float c1) {
    Sums r;
    r.m = fmaxf(a.m, b.m);
    const float h = shift_of(r.m);
    const float da = exponent(a.m, h, c), db = exponent(b.m, h, c);
    const float fa = exp2_approx(da), fb = exp2_approx(db);
    r.s = a.s * fa + b.s * fb;
    r.u = 0.0f, r.s1 = 0.0f;
    if constexpr (U) r.u = fa * (a.u + a.s * da) + fb * (b.u + b.s * db);
    if constexpr (S1) r.s1 = a.s1 * exp2_approx(exponent(a.m, h, c1)) + b.s1 * exp2_approx(exponent(b.m, h, c1));
    return r;
}

// adds n values whose maximum is cm
template <int n, bool U, bool S1>
__device__ __forceinline__ void add_values(Sums& a, const float (&x)[n], float cm, float c, float c1) {
    if (cm > a.m) {
        const float h = shift_of(cm), d = exponent(a.m, h, c), f = exp2_approx(d);
        if constexpr (U) a.u = f * (a.u + a.s * d);
        a.s *= f;
        if constexpr (S1) a.s1 *= exp2_approx(exponent(a.m, h, c1));
        a.m = cm;
    }
    const float h = shift_of(a.m);
#pragma unroll
    for (int i = 0; i < n; ++i) {
        const float g = x[i] - h;
        if constexpr (U) {
            const float d = max_nan(g * c, kMinExp), e = exp2_approx(d);
            a.s += e;
            a.u = fmaf(e, d, a.u);
        } else {
            a.s += exp2_approx(g * c);
        }
        if constexpr (S1) a.s1 += exp2_approx(g * c1);
    }
}

template <bool U, bool S1>
__device__ __forceinline__ Sums warp_join(Sums a, float c, float c1) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        Sums b;
        b.m = __shfl_xor_sync(0xffffffffu, a.m, o);
        b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
        b.u = U ? __shfl_xor_sync(0xffffffffu, a.u, o) : 0.0f;
        b.s1 = S1 ? __shfl_xor_sync(0xffffffffu, a.s1, o) : 0.0f;
        // the lower lane's half first, in both lanes
        a = (threadIdx.x & o) ? join<U, S1>(b, a, c, c1) : join<U, S1>(a, b, c, c1);
    }
    return a;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// every thread's sums -> the CTA's, in all threads; part: shared, one entry a warp.
// Ends with a barrier before `part` may be written again.
template <int kThreads, bool U, bool S1>
__device__ __forceinline__ Sums cta_join(Sums a, Sums* part, float c, float c1) {
    constexpr int kWarps = kThreads / 32;
    a = warp_join<U, S1>(a, c, c1);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = a;
    __syncthreads();
    const int lane = threadIdx.x & 31;
    a = lane < kWarps ? part[lane] : no_sums();
    a = warp_join<U, S1>(a, c, c1);
    __syncthreads();
    return a;
}

__device__ __forceinline__ uint32_t ld_dsmem_u32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint64_t ld_dsmem_u64(uint32_t addr) {
    uint64_t v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
    return v;
}

// the CTAs' sums -> the row's, in every thread of the cluster, joined in rank
// order; mine: shared, one entry.  The caller has the next cluster barrier
// before `mine` is written again or the CTA ends.
template <bool U, bool S1>
__device__ __forceinline__ Sums cluster_join(const Sums& a, Sums* mine, uint32_t ctas, float c, float c1) {
    if (threadIdx.x == 0) *mine = a;
    cluster_sync();
    Sums r = no_sums();
    for (uint32_t i = 0; i < ctas; ++i) {
        const float4 v = ld_dsmem_v4(map_to_rank(smem_addr(mine), i));
        const Sums b{v.x, v.y, v.z, v.w};
        r = i == 0 ? b : join<U, S1>(r, b, c, c1);
    }
    return r;
}

// the part of a row that one of `ctas` CTAs reads: `head` logits before the
// first 16-byte boundary (rank 0), 16-byte vectors v0 .. v1 - 1 from there on,
// and `tail` logits behind the last whole vector (last rank).  Vector v starts
// at logit h0 + v * kVec, the tail at logit t0; j0 .. j1 - 1 is the whole part.
struct Segment {
    int head, tail, v0, v1, h0, t0, j0, j1;
};

template <int DT>
__device__ __forceinline__ Segment segment_of(const void* row, int V, uint32_t rank, uint32_t ctas) {
    constexpr int kVec = Elem<DT>::kVec, kSize = 16 / kVec;
    Segment g;
    const int mis = (int)(((uintptr_t)row & 15u) / kSize);
    g.h0 = min(V, mis ? kVec - mis : 0);
    const int nv = (V - g.h0) / kVec;
    g.t0 = g.h0 + nv * kVec;
    g.v0 = (int)((int64_t)nv * rank / ctas);
    g.v1 = (int)((int64_t)nv * (rank + 1) / ctas);
    g.head = rank == 0 ? g.h0 : 0;
    g.tail = rank == ctas - 1 ? V - g.t0 : 0;
    g.j0 = rank == 0 ? 0 : g.h0 + g.v0 * kVec;
    g.j1 = rank == ctas - 1 ? V : g.h0 + g.v1 * kVec;
    return g;
}

}  // namespace il
