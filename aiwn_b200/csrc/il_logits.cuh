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
//
// Rows of up to 1024 logits are a warp's, in its registers.  Longer ones are a
// CTA's of 64 to 512 threads, or where there are fewer of them than the
// SMs can hold, a cluster's of up to 16.  What bounds these is first the
// instructions of a logit (bf16, log probability and entropy: 11.5 an element
// at first, 7.9 now, of about 11 that the SMs could issue at the rate of HBM), then what
// a row costs beside its logits, which is why a row has few warps and an SM
// several rows, and for small calls the launch.  4096 x 131072 logits in bf16,
// log probability and entropy (1.07 GB, 164 us at the measured copy rate):
// 210 us with 512 threads, two vectors a step and scalar arithmetic, 184 us
// with four vectors and one fused multiply-add an exponent, 174 us (94%) with
// 768 instead of 512 threads an SM.
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
constexpr int kMaxCluster = 16;
// threads of the CTAs that an SM holds of the kernels of longer rows, which go through a row once or twice
constexpr int sm_threads(int passes) { return passes > 1 ? 512 : 768; }
constexpr float kLog2e = 1.44269504088896341f;

// rows r = b*T + t of a [B, T, V] tensor whose last dimension is contiguous; T = 1 where one stride serves all rows
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
    uint32_t T;
};

__device__ __forceinline__ int64_t row_offset(int64_t sb, int64_t st, uint32_t T, uint32_t row) {
    if (T == 1) return (int64_t)row * sb;
    const uint32_t b = row / T;
    return (int64_t)b * sb + (int64_t)(row - b * T) * st;
}

// a row that moves on by a fixed number of rows, without a division for each
struct RowAt {
    uint32_t t;
    int64_t off;
    __device__ __forceinline__ RowAt(const RowsIn& z, uint32_t row)
        : t(row % z.T), off(row_offset(z.sb, z.st, z.T, row)) {}
};
struct RowStep {
    uint32_t t;
    int64_t off, wrap;  // of b and t together; more where t passes T
    __device__ __forceinline__ RowStep(const RowsIn& z, uint32_t step)
        : t(step % z.T), off(row_offset(z.sb, z.st, z.T, step)), wrap(z.sb - (int64_t)z.T * z.st) {}
    __device__ __forceinline__ void move(RowAt& r, uint32_t T) const {
        r.t += t;
        r.off += off;
        if (r.t >= T) r.t -= T, r.off += wrap;
    }
};

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

// two floats in one 64-bit register pair: one instruction for both
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
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

__device__ __forceinline__ float sum2(uint64_t v) {
    float a, b;
    unpack2(v, a, b);
    return a + b;
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

// the sums with m raised to `top` (h = shift_of(top)); c = log2(e) / tau
template <bool U, bool S1>
__device__ __forceinline__ Sums raised(Sums a, float top, float c) {
    const float h = shift_of(top), d = exponent(a.m, h, c), f = exp2_approx(d);
    if constexpr (U) a.u = f * (a.u + a.s * d);
    a.s *= f;
    if constexpr (S1) a.s1 *= exp2_approx(exponent(a.m, h, kLog2e));
    a.m = top;
    return a;
}

template <bool U, bool S1>
__device__ __forceinline__ Sums join(Sums a, Sums b, float c) {
    const float top = fmaxf(a.m, b.m);
    a = raised<U, S1>(a, top, c);
    b = raised<U, S1>(b, top, c);
    return Sums{top, a.s + b.s, U ? a.u + b.u : 0.0f, S1 ? a.s1 + b.s1 : 0.0f};
}

// Adds n values whose maximum is cm.  They are summed among themselves first:
// a long row's small terms would be lost one by one in a sum that already holds
// the row's largest.
template <int n, bool U, bool S1>
__device__ __forceinline__ void add_values(Sums& a, const float (&x)[n], float cm, float c) {
    if (cm > a.m) a = raised<U, S1>(a, cm, c);
    const float h = shift_of(a.m);
    const uint64_t hh = pack2(-h, -h), cc = pack2(c, c), c1 = pack2(kLog2e, kLog2e);
    uint64_t s = 0, u = 0, s1 = 0;  // of the even and of the odd values
#pragma unroll
    for (int i = 0; i < n; i += 2) {
        const uint64_t g = add2(pack2(x[i], i + 1 < n ? x[i + 1 < n ? i + 1 : i] : -INFINITY), hh);
        float d, f, e0, e1;
        unpack2(mul2(g, cc), d, f);
        if constexpr (U) d = max_nan(d, kMinExp), f = max_nan(f, kMinExp);
        e0 = exp2_approx(d);
        e1 = exp2_approx(f);
        const uint64_t e = pack2(e0, e1);
        s = i ? add2(s, e) : e;
        if constexpr (U) u = i ? fma2(e, pack2(d, f), u) : mul2(e, pack2(d, f));
        if constexpr (S1) {
            unpack2(mul2(g, c1), d, f);
            const uint64_t e = pack2(exp2_approx(d), exp2_approx(f));
            s1 = i ? add2(s1, e) : e;
        }
    }
    float lo, hi;
    unpack2(s, lo, hi);
    a.s += lo + hi;
    if constexpr (U) {
        unpack2(u, lo, hi);
        a.u += lo + hi;
    }
    if constexpr (S1) {
        unpack2(s1, lo, hi);
        a.s1 += lo + hi;
    }
}

// the largest of kU 16-byte vectors' values, -inf where all are NaN
template <int DT, int kU>
__device__ __forceinline__ float max_of(const uint4 (&r)[kU]) {
    if constexpr (DT == kBF16) {
        auto word = [](uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); };
        __nv_bfloat162 m = word(r[0].x);
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            if (u) m = __hmax2(m, word(r[u].x));
            m = __hmax2(m, word(r[u].y));
            m = __hmax2(m, word(r[u].z));
            m = __hmax2(m, word(r[u].w));
        }
        return fmaxf(fmaxf(__low2float(m), __high2float(m)), -INFINITY);
    } else {
        float m = -INFINITY;
#pragma unroll
        for (int u = 0; u < kU; ++u)
            m = fmaxf(fmaxf(fmaxf(m, __uint_as_float(r[u].x)), fmaxf(__uint_as_float(r[u].y), __uint_as_float(r[u].z))),
                      __uint_as_float(r[u].w));
        return m;
    }
}

// Values below -2^100 raised to it (NaN stays): their exponential is 0 next to any maximum
// of ordinary size, and their exponent then is finite, so that 0 times it is 0.
template <int DT>
__device__ __forceinline__ uint4 floor16(const uint4& r) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
    uint32_t y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (DT == kF32) {
            y[i] = __float_as_uint(max_nan(__uint_as_float(w[i]), -1.2676506e30f));
        } else {
            const uint32_t low = 0xf180f180u;  // -2^100, twice
            const __nv_bfloat162 v = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&w[i]),
                                                 *reinterpret_cast<const __nv_bfloat162*>(&low));
            y[i] = *reinterpret_cast<const uint32_t*>(&v);
        }
    }
    return make_uint4(y[0], y[1], y[2], y[3]);
}

// the sums of a vector to the maximum m, whatever its size
template <int DT, bool U, bool S1>
__device__ __noinline__ Sums huge_vector(uint4 r, float m, float c) {
    constexpr int kVec = Elem<DT>::kVec;
    float x[kVec];
    unpack16<DT>(r, x);
    Sums a{m, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
        const float d = exponent(x[i], m, c), e = exp2_approx(d);
        a.s += e;
        if constexpr (U) a.u = fmaf(e, d, a.u);
        if constexpr (S1) a.s1 += exp2_approx(exponent(x[i], m, kLog2e));
    }
    return a;
}

// A thread's sums while a row goes by.  The exponent is taken to a whole number H next to
// m log2(e) / tau: d = z c - H is one fused multiply-add, rounded once, and a new maximum
// rescales by a power of two, without rounding.  Where |m| c is 2^22 or more (a row of nothing
// but a mask's huge negative values) such an H has no meaning, and d = (z - m) c; so it is where
// c is so small (a temperature above 10^20) that floor16's -2^100 would count for something, or so large (one below
// 10^-8) that its exponent would not be finite.
constexpr float kLeastFactor = 1e-20f, kMostFactor = 1e8f;

template <bool U, bool S1>
struct Running {
    float m, s, u, s1, h, h1;  // h, h1: -H for c and for log2(e), 0 where huge
    bool huge;

    __device__ __forceinline__ void begin(float c) {
        m = -INFINITY;
        s = u = s1 = h = h1 = 0.0f;
        huge = beyond(c);  // for what comes before the first value above -inf, too
    }
    __device__ __forceinline__ static bool beyond(float c) { return U && (c < kLeastFactor || c > kMostFactor); }
    __device__ __forceinline__ static bool is_huge(float t) { return !(fabsf(t) < 4194304.0f); }

    // The sums are next to m c, or (huge: h = h1 = 0) at m itself; the factor between any two of these forms has its
    // exponent rounded once: a product m c is rounded alone nowhere, beyond 2^22 that is by a quarter and more.
    __device__ __forceinline__ void raise(float top, float c) {
        const float t = top * c;
        const bool now = is_huge(t) || (S1 && is_huge(top * kLog2e)) || beyond(c);
        const float g = now ? 0.0f : -rintf(t), g1 = now ? 0.0f : -rintf(top * kLog2e);
        if (m != -INFINITY) {
            const float step = (huge ? m : 0.0f) - (now ? top : 0.0f);
            const float d = fmaxf(fmaf(step, c, g - h), kMinExp), f = exp2_approx(d);
            if constexpr (U) u = f * (u + s * d);
            s *= f;
            if constexpr (S1) s1 *= exp2_approx(fmaxf(fmaf(step, kLog2e, g1 - h1), kMinExp));
        }
        m = top, h = g, h1 = g1, huge = now;
    }

    // kU 16-byte vectors whose maximum is cm; they are summed among themselves first: a long row's
    // small terms would be lost one by one in a sum that already holds the row's largest
    template <int DT, int kU>
    __device__ __forceinline__ void add(const uint4 (&r)[kU], float cm, float c) {
        constexpr int kVec = Elem<DT>::kVec;
        if (cm > m) raise(cm, c);
        if (huge) {
#pragma unroll
            for (int q = 0; q < kU; ++q) {
                const Sums x = huge_vector<DT, U, S1>(r[q], shift_of(m), c);
                s += x.s, u += x.u, s1 += x.s1;
            }
        } else {
            uint64_t e = 0, f = 0, v = 0;  // of the even and the odd values
#pragma unroll
            for (int q = 0; q < kU; ++q) {
                float x[kVec];
                unpack16<DT>(U ? floor16<DT>(r[q]) : r[q], x);
#pragma unroll
                for (int i = 0; i < kVec; i += 2) {
                    const float d0 = fmaf(x[i], c, h), d1 = fmaf(x[i + 1], c, h);
                    const uint64_t a = pack2(exp2_approx(d0), exp2_approx(d1));
                    const bool first = q == 0 && i == 0;
                    e = first ? a : add2(e, a);
                    if constexpr (U) v = first ? mul2(a, pack2(d0, d1)) : fma2(a, pack2(d0, d1), v);
                    if constexpr (S1) {
                        const uint64_t b = pack2(exp2_approx(fmaf(x[i], kLog2e, h1)), exp2_approx(fmaf(x[i + 1], kLog2e, h1)));
                        f = first ? b : add2(f, b);
                    }
                }
            }
            s += sum2(e);
            if constexpr (U) u += sum2(v);
            if constexpr (S1) s1 += sum2(f);
        }
    }

    // the same sums taken to the maximum itself
    __device__ __forceinline__ Sums sums(float c) const {
        Sums r{m, s, u, s1};
        if (m != -INFINITY && !huge) {
            const float d = fmaf(m, c, h), f = exp2_approx(-d);
            if constexpr (U) r.u = f * (u - d * s);
            r.s = f * s;
            if constexpr (S1) r.s1 = exp2_approx(-fmaf(m, kLog2e, h1)) * s1;
        }
        return r;
    }
};

// lanes of a warp, all lanes get the result; kLanes = 32 or 16 (lanes 0..15 hold values)
template <int kLanes = 32>
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// the largest of the lanes' values, NaN lanes left out (NaN where there is nothing else)
__device__ __forceinline__ float warp_max(float v) {
    const uint32_t b = __float_as_uint(v);
    const uint32_t key = v != v ? 0u : b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
    const uint32_t top = __reduce_max_sync(0xffffffffu, key);
    return __uint_as_float(top ^ ((uint32_t)((int32_t)~top >> 31) | 0x80000000u));  // 0: all bits set, a NaN
}

// every lane's sums -> the warp's, in all lanes
template <bool U, bool S1>
__device__ __forceinline__ Sums warp_join(Sums a, float c) {
    a = raised<U, S1>(a, warp_max(a.m), c);
    a.s = warp_sum(a.s);
    if constexpr (U) a.u = warp_sum(a.u);
    if constexpr (S1) a.s1 = warp_sum(a.s1);
    return a;
}

// every thread's sums -> the CTA's, in all threads.  part: shared, one entry a
// warp, not written again before the CTA's next barrier but one.
template <int kThreads, bool U, bool S1>
__device__ __forceinline__ Sums cta_join(Sums a, float4* part, float c) {
    constexpr int kRowWarps = kThreads / 32;
    a = warp_join<U, S1>(a, c);
    const int lane = threadIdx.x & 31;
    if (lane == 0) part[threadIdx.x >> 5] = make_float4(a.m, a.s, a.u, a.s1);
    __syncthreads();
    const float4 v = part[lane & (kRowWarps - 1)];
    a = Sums{v.x, v.y, v.z, v.w};
    a = raised<U, S1>(a, warp_max(a.m), c);
    a.s = warp_sum<kRowWarps>(a.s);
    if constexpr (U) a.u = warp_sum<kRowWarps>(a.u);
    if constexpr (S1) a.s1 = warp_sum<kRowWarps>(a.s1);
    return a;
}

__device__ __forceinline__ uint64_t ld_dsmem_u64(uint32_t addr) {
    uint64_t v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
    return v;
}

// the CTAs' sums -> the row's, in every thread of the cluster; mine: shared, not
// written again before the cluster's next barrier but one
template <bool U, bool S1>
__device__ __forceinline__ Sums cluster_join(Sums a, float4* mine, uint32_t ctas, float c) {
    if (threadIdx.x == 0) *mine = make_float4(a.m, a.s, a.u, a.s1);
    cluster_sync();
    const uint32_t lane = threadIdx.x & 31;
    a = no_sums();
    if (lane < ctas) {
        const float4 v = ld_dsmem_v4(map_to_rank(smem_addr(mine), lane));
        a = Sums{v.x, v.y, v.z, v.w};
    }
    return warp_join<U, S1>(a, c);
}

// the part of a row that one of 2^lg CTAs reads: `head` logits before the
// first 16-byte boundary (rank 0), 16-byte vectors v0 .. v1 - 1 from there on,
// and `tail` logits behind the last whole vector (last rank).  Vector v starts
// at logit h0 + v * kVec, the tail at logit t0; j0 .. j1 - 1 is the whole part.
struct Segment {
    int head, tail, v0, v1, h0, t0, j0, j1;
};

template <int DT>
__device__ __forceinline__ Segment segment_of(const void* row, int V, uint32_t rank, uint32_t lg) {
    constexpr int kVec = Elem<DT>::kVec, kSize = 16 / kVec;
    Segment g;
    const int mis = (int)(((uintptr_t)row & 15u) / kSize);
    g.h0 = min(V, mis ? kVec - mis : 0);
    const int nv = (V - g.h0) / kVec;
    g.t0 = g.h0 + nv * kVec;
    const bool last = rank + 1 == 1u << lg;
    g.v0 = (int)(nv * rank >> lg);  // at most 2^19 vectors, 2^9 parts
    g.v1 = (int)(nv * (rank + 1) >> lg);
    g.head = rank == 0 ? g.h0 : 0;
    g.tail = last ? V - g.t0 : 0;
    g.j0 = rank == 0 ? 0 : g.h0 + g.v0 * kVec;
    g.j1 = last ? V : g.h0 + g.v1 * kVec;
    return g;
}

// ---- rows a CTA goes through, and their 16-byte vectors ahead of time -----------------

// which of 32 consecutive rows of a cluster (or CTA) are not padding: a load of a lane each
struct RowList {
    Tokens tok;
    uint32_t N, first, step, count;

    __device__ __forceinline__ RowList(const Tokens& tok_, uint32_t N_, uint32_t first_, uint32_t step_)
        : tok(tok_), N(N_), first(first_), step(step_) {
        count = first < N ? (N - first - 1) / step + 1 : 0;
    }
    __device__ __forceinline__ uint32_t row(uint32_t i) const { return first + i * step; }
    // whole warps; i: a multiple of 32.  Bit n: row i + n
    __device__ __forceinline__ uint32_t window(uint32_t i) const {
        if (!tok.p) return 0xffffffffu;
        const uint32_t n = i + (threadIdx.x & 31);
        const bool live = n < count && tok.p[row_offset(tok.sb, tok.st, tok.T, row(n))] != tok.ignore;
        return __ballot_sync(0xffffffffu, live);
    }
};

// goes through the rows of a list that are not padding
struct LiveRows {
    const RowList& list;
    const RowStep& step;
    uint32_t T, i, window;
    RowAt at;

    // whole warps
    __device__ __forceinline__ LiveRows(const RowsIn& z, const RowList& list_, const RowStep& step_)
        : list(list_), step(step_), T(z.T), i(0), at(z, list_.first) {
        window = list.window(0);
        seek();
    }
    __device__ __forceinline__ bool valid() const { return i < list.count; }
    __device__ __forceinline__ uint32_t row() const { return list.row(i); }
    __device__ __forceinline__ void next() {
        step_on();
        seek();
    }

private:
    __device__ __forceinline__ void step_on() {
        step.move(at, T);
        if ((++i & 31) == 0 && i < list.count) window = list.window(i);
    }
    __device__ __forceinline__ void seek() {
        while (i < list.count && !(window >> (i & 31) & 1u)) step_on();
    }
};

__device__ __forceinline__ void copy_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int n>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(n) : "memory");
}

// The vectors of a CTA's rows, kU of them a thread at a time, kStages steps
// ahead of their use and across the ends of rows, so that loads go on while a
// row's sums are joined.  Each thread copies what it will read itself into
// places of its own (cp.async), so that no barrier is involved.  Every row is
// gone through kPasses times.  kStages times 64 bytes a thread are under way:
// 144 KB an SM with one pass, 128 KB with two, of the 50 KB or so that its share
// of HBM's rate needs over a load's latency; the rest lasts while sums are joined.
template <int DT, int kThreads, int kPasses>
struct RowStream {
    static constexpr int kVec = Elem<DT>::kVec, kU = 4, kElems = kU * kVec, kStages = kPasses > 1 ? 4 : 3;
    static constexpr int kStep = kU * kThreads;  // vectors of a step
    static constexpr uint32_t kStepBytes = kStep * 16, kBytes = kStages * kStepBytes;
    using T = typename Elem<DT>::type;

    const RowsIn& z;
    const int V;
    const uint32_t rank, lg;
    LiveRows rows;      // at the row being loaded
    uint32_t slots;     // shared address of this thread's places
    uint32_t put, get;  // bytes
    const uint4* src;   // this thread's next vector
    int mine, steps;    // vectors and steps left of this pass
    int passes;         // left after this one

    __device__ __forceinline__ RowStream(const RowsIn& z_, int V_, const RowList& list_, const RowStep& step_,
                                         uint32_t rank_, uint32_t lg_, void* shared)
        : z(z_), V(V_), rank(rank_), lg(lg_), rows(z_, list_, step_), put(0), get(0), src(nullptr), mine(0), steps(0),
          passes(0) {
        slots = smem_addr(shared) + threadIdx.x * 16;
        begin_row();
#pragma unroll 1
        for (int n = 0; n < kStages; ++n) issue();
    }

    __device__ __forceinline__ void begin_pass(const Segment& g, const T* zr) {
        src = reinterpret_cast<const uint4*>(zr + g.h0) + g.v0 + threadIdx.x;
        mine = (g.v1 - g.v0 - (int)threadIdx.x + kThreads - 1) / kThreads;
        steps = (g.v1 - g.v0 + kStep - 1) / kStep;
    }

    __device__ __forceinline__ const T* row_at() const { return reinterpret_cast<const T*>(z.p) + rows.at.off; }

    // the first row from here on that has vectors to load; steps stays 0 if there is none
    __device__ __forceinline__ void begin_row() {
        for (; rows.valid(); rows.next()) {
            const Segment g = segment_of<DT>(row_at(), V, rank, lg);
            if (g.v0 >= g.v1) continue;
            begin_pass(g, row_at());
            passes = kPasses - 1;
            return;
        }
    }

    __device__ __forceinline__ void issue() {
        if (steps) {
            if (steps > 1) {  // a whole one
#pragma unroll
                for (int u = 0; u < kU; ++u) copy_async16(slots + put + u * (kThreads * 16), src + u * kThreads);
            } else {
#pragma unroll
                for (int u = 0; u < kU; ++u)
                    if (u < mine) copy_async16(slots + put + u * (kThreads * 16), src + u * kThreads);
            }
            src += kStep;
            mine -= kU;
            if (--steps == 0) {
                if (kPasses > 1 && passes > 0) {
                    --passes;
                    begin_pass(segment_of<DT>(row_at(), V, rank, lg), row_at());
                } else {
                    rows.next();
                    begin_row();
                }
            }
        }
        copy_commit();
        put = put + kStepBytes == kBytes ? 0 : put + kStepBytes;
    }

    // this thread's next kU vectors, of which the row has `mine`; the others are -inf
    template <bool FULL>
    __device__ __forceinline__ void take(uint4 (&r)[kU], int mine) {
        copy_wait<kStages - 1>();
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            const uint32_t from = slots + get + u * (kThreads * 16);
            if (!FULL) r[u] = neg_inf16<DT>();
            if (FULL || u < mine)
                asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                             : "=r"(r[u].x), "=r"(r[u].y), "=r"(r[u].z), "=r"(r[u].w)
                             : "r"(from)
                             : "memory");
        }
        get = get + kStepBytes == kBytes ? 0 : get + kStepBytes;
    }
};

}  // namespace il
