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
constexpr int kRowWarps = kRowThreads / 32;
constexpr int kMaxCluster = 16;
constexpr float kLog2e = 1.44269504088896341f;

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
    float s = 0.0f, u = 0.0f, s1 = 0.0f, t = 0.0f, v = 0.0f, t1 = 0.0f;  // even and odd values
#pragma unroll
    for (int i = 0; i < n; i += 2) {
        const float g = x[i] - h;
        if constexpr (U) {
            const float d = max_nan(g * c, kMinExp), e = exp2_approx(d);
            s += e;
            u = fmaf(e, d, u);
        } else {
            s += exp2_approx(g * c);
        }
        if constexpr (S1) s1 += exp2_approx(g * kLog2e);
        if (i + 1 < n) {
            const float g2 = x[i + 1] - h;
            if constexpr (U) {
                const float d = max_nan(g2 * c, kMinExp), e = exp2_approx(d);
                t += e;
                v = fmaf(e, d, v);
            } else {
                t += exp2_approx(g2 * c);
            }
            if constexpr (S1) t1 += exp2_approx(g2 * kLog2e);
        }
    }
    a.s += s + t;
    if constexpr (U) a.u += u + v;
    if constexpr (S1) a.s1 += s1 + t1;
}

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
// NaN lanes are left out
__device__ __forceinline__ float warp_max(float v) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
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
template <bool U, bool S1>
__device__ __forceinline__ Sums cta_join(Sums a, float4* part, float c) {
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

// ---- rows a CTA goes through, and their 16-byte vectors ahead of time -----------------

// the i-th row of a cluster (or CTA); which of 32 rows are not padding is found by one
// load of a lane each
struct RowList {
    Tokens tok;
    uint32_t T, N, first, step, count;
    uint32_t mask;  // of rows 32 (i / 32) ...

    __device__ __forceinline__ RowList(const Tokens& tok_, uint32_t T_, uint32_t N_, uint32_t first_, uint32_t step_)
        : tok(tok_), T(T_), N(N_), first(first_), step(step_), mask(0xffffffffu) {
        count = first < N ? (N - first - 1) / step + 1 : 0;
    }
    __device__ __forceinline__ uint32_t row(uint32_t i) const { return first + i * step; }
    // whole warps; call with i = 0 and then with every multiple of 32
    __device__ __forceinline__ void window(uint32_t i) {
        if (!tok.p) return;
        const uint32_t n = i + (threadIdx.x & 31);
        const bool live = n < count && tok.p[row_offset(tok.sb, tok.st, T, row(n))] != tok.ignore;
        mask = __ballot_sync(0xffffffffu, live);
    }
    __device__ __forceinline__ bool live(uint32_t i) const { return mask >> (i & 31) & 1u; }
};

__device__ __forceinline__ uint64_t policy_evict_first() {
    uint64_t p;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
    return p;
}
__device__ __forceinline__ uint64_t policy_evict_last() {
    uint64_t p;
    asm volatile("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(p));
    return p;
}
__device__ __forceinline__ void copy_async16(uint32_t dst, const void* src, uint64_t policy) {
    asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "l"(policy)
                 : "memory");
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
// gone through kPasses times; the last time its lines may leave the L2 first.
template <int DT, int kPasses, int kStages>
struct RowStream {
    static constexpr int kVec = Elem<DT>::kVec, kU = 2, kElems = kU * kVec;
    static constexpr int kStep = kU * kRowThreads;  // vectors of a step
    static constexpr int kBytes = kStages * kStep * 16;

    RowsIn z;
    int V;
    uint32_t rank, ctas;
    RowList list;
    uint32_t slots;  // shared address of this thread's places
    uint32_t i;      // row being loaded
    int pass, v, v0, v1, put, get;
    const uint4* body;
    uint64_t first_time, last_time;

    __device__ __forceinline__ RowStream(const RowsIn& z_, int V_, const RowList& list_, uint32_t rank_, uint32_t ctas_,
                                         void* shared)
        : z(z_), V(V_), rank(rank_), ctas(ctas_), list(list_), i(0), pass(0), v(0), v0(0), v1(0), put(0), get(0) {
        slots = smem_addr(shared) + threadIdx.x * 16;
        last_time = policy_evict_first();
        first_time = kPasses > 1 ? policy_evict_last() : last_time;
        list.window(0);
        begin_row();
#pragma unroll
        for (int n = 0; n < kStages; ++n) issue();
    }

    // to the first row from i on that has vectors to load
    __device__ __forceinline__ void begin_row() {
        for (; i < list.count;) {
            if (list.live(i)) {
                const typename Elem<DT>::type* zr = reinterpret_cast<const typename Elem<DT>::type*>(z.p) +
                                                    row_offset(z.sb, z.st, z.T, list.row(i));
                const Segment g = segment_of<DT>(zr, V, rank, ctas);
                if (g.v0 < g.v1) {
                    body = reinterpret_cast<const uint4*>(zr + g.h0);
                    v0 = g.v0, v1 = g.v1, v = g.v0;
                    return;
                }
            }
            if ((++i & 31) == 0) list.window(i);
        }
    }

    __device__ __forceinline__ void issue() {
        if (i < list.count) {
            const uint64_t policy = pass + 1 == kPasses ? last_time : first_time;
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                const int w = v + (int)threadIdx.x + u * kRowThreads;
                if (w < v1) copy_async16(slots + (put * kU + u) * (kRowThreads * 16), body + w, policy);
            }
            v += kStep;
            if (v >= v1) {
                v = v0;
                if (++pass == kPasses) {
                    pass = 0;
                    if ((++i & 31) == 0) list.window(i);
                    begin_row();
                }
            }
        }
        copy_commit();
        put = put + 1 == kStages ? 0 : put + 1;
    }

    // the next kU vectors; valid(u) tells which of them the row has (the others are -inf)
    __device__ __forceinline__ void take(uint4 (&r)[kU], int first, int end) {
        copy_wait<kStages - 1>();
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            r[u] = neg_inf16<DT>();
            if (first + (int)threadIdx.x + u * kRowThreads < end) {
                const uint32_t at = slots + (get * kU + u) * (kRowThreads * 16);
                asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                             : "=r"(r[u].x), "=r"(r[u].y), "=r"(r[u].z), "=r"(r[u].w)
                             : "r"(at)
                             : "memory");
            }
        }
        get = get + 1 == kStages ? 0 : get + 1;
    }
};

}  // namespace il
