// il_distill.cuh -- distillation of a student's logits from a teacher's top
// log probabilities, with the gradient in the same launch.
//
// A row has up to 128 slots (i, l_i): token i has probability exp(l_i) under
// the teacher at temperature tau.  With p = softmax(z / tau) of the student:
//   without tail: q = softmax(l) over the slots,  Q = 1
//                 KL = sum q_i (ln q_i - ln p_i)
//   with tail:    q_i = exp(l_i), q_r = 1 - sum q_i (not below 0),  Q = sum q_i + q_r
//                 KL = sum q_i (ln q_i - ln p_i) + q_r (ln q_r - ln p_r),
//                 p_r = the sum of p over the tokens that no slot names
//   loss = alpha tau^2 KL - (1 - alpha) ln softmax(z)_target
//   dz_j = alpha tau (p_j Q - sum_{i = j} q_i) + (1 - alpha) (softmax(z)_j - [j = target]),
//          and p_j (Q - q_r / p_r) in place of p_j Q where no slot names j.
//
// The loss reads each logit once.  The gradient is written by the same CTA
// right after the row's sums are known: it reads the row again, which the L2
// then still holds, so that a training step moves each logit over HBM once in
// and its gradient once out.
//
// With tail, p_r is never taken as 1 - sum p_i, which would lose its digits
// when the student agrees with the teacher: a bitmap of the slots in shared
// memory keeps their logits out of the running sums, which so become those of
// the rest, and the slots' own sums are joined to them.  q_r, a small
// difference of inputs, is taken in 64 bits.
#pragma once
#include "il_logits.cuh"

namespace il {

constexpr int kMean = 1, kSum = 2;  // reduction; 0: each row's loss

struct DistillArgs {
    RowsIn z;
    Tokens tok;  // targets; padded rows are tok.ignore
    RowsOut d;   // gradient, d.p == nullptr: none
    uint32_t N;
    int V, k;
    const int64_t* index;  // [N, k], < 0: empty slot
    const float* logprob;  // [N, k]
    float tau, c, alpha;
    int tail, hard;        // hard: the target's term is wanted (alpha < 1)
    float scale;           // of the gradient
    const float* scale_p;  // times *scale_p, or null
    const float* g;        // times g[0], or g[row] with g_rows, or null
    int g_rows;
    int skip_if_one;       // nothing is left to do where g[0] == 1
    float* loss;           // [N] or null
};

struct DistillRow {  // what a warp found out about a row's slots, in shared memory
    int index[kMaxTop + 1];  // the last of the k + 1: the target; -1: none
    float q[kMaxTop];
    Sums slots;              // of the slots' logits, each token once (with tail)
    float Q, rest;           // rest: q_r
    float own;               // sum q_i (ln q_i - (z_i - m0) / tau), m0 = base
    float base, used;        // used: sum of q_i over the slots
    float z_target;
    int bad;
    // gradient: e_j coef + e1_j coef1 with e_j = 2^((z_j - h) c), e1_j = 2^((z_j - h1) log2 e)
    float h, coef, h1, coef1;
    // at a slot: 2^((z - h1) c) inside - w q
    float inside, w, w_hard;
};

// One warp.  Reads the slots of a row.
template <int DT>
__device__ __forceinline__ void distill_slots(const DistillArgs& a, uint32_t row, const typename Elem<DT>::type* zr,
                                              int64_t t, DistillRow& r) {
    constexpr int kPer = kMaxTop / 32;
    const int lane = threadIdx.x & 31;
    bool bad = false;
    int j[kPer];
    float l[kPer], z[kPer], q[kPer];
#pragma unroll
    for (int n = 0; n < kPer; ++n) {
        const int i = lane + 32 * n;
        j[n] = -1;
        l[n] = -INFINITY;
        z[n] = -INFINITY;
        if (i < a.k) {
            const int64_t x = a.index[(int64_t)row * a.k + i];
            bad |= x >= a.V;
            if (x >= 0 && x < a.V) {
                j[n] = (int)x;
                l[n] = a.logprob[(int64_t)row * a.k + i];
                z[n] = to_float(zr[x]);
            }
            r.index[i] = j[n];
        }
    }
    // weights
    float Q, rest = 0.0f, shift = 0.0f, log_sum = 0.0f;
    if (a.tail) {
        double sum = 0.0;
#pragma unroll
        for (int n = 0; n < kPer; ++n) {
            const double e = j[n] >= 0 ? exp((double)l[n]) : 0.0;
            q[n] = (float)e;
            sum += e;
        }
        sum = warp_sum(sum);
        const double left = 1.0 - sum;
        rest = left > 0.0 || left != left ? (float)left : 0.0f;
        Q = (float)(left > 0.0 ? 1.0 : sum);
    } else {
        float m = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int n = 0; n < kPer; ++n) m = fmaxf(m, l[n]);
        shift = shift_of(warp_max(m));
#pragma unroll
        for (int n = 0; n < kPer; ++n) {
            q[n] = j[n] >= 0 ? expf(l[n] - shift) : 0.0f;
            sum += q[n];
        }
        sum = warp_sum(sum);
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        log_sum = sum == 0.0f ? 0.0f : logf(sum);
#pragma unroll
        for (int n = 0; n < kPer; ++n) q[n] *= inv;
        Q = sum == 0.0f ? 0.0f : 1.0f;
    }
    // sums over the slots; base: their largest logit
    float base = -INFINITY, own = 0.0f, used = 0.0f;
#pragma unroll
    for (int n = 0; n < kPer; ++n) base = fmaxf(base, z[n]);
    base = shift_of(warp_max(base));
#pragma unroll
    for (int n = 0; n < kPer; ++n) {
        const int i = lane + 32 * n;
        if (i < a.k) r.q[i] = q[n];
        used += q[n];
        own += q[n] == 0.0f ? 0.0f : q[n] * ((l[n] - shift - log_sum) - (z[n] - base) / a.tau);
    }
    used = warp_sum(used);
    own = warp_sum(own);
    __syncwarp();
    if (a.tail) {
        Sums s = no_sums();
#pragma unroll
        for (int n = 0; n < kPer; ++n) {
            if (j[n] < 0) continue;
            bool first = true;  // a token that several slots name counts once
            for (int i = 0; i < lane + 32 * n; ++i) first &= r.index[i] != j[n];
            const float x[1] = {z[n]};
            if (first) add_values<1, false, true>(s, x, z[n], a.c, 1.44269504088896341f);
        }
        s = warp_join<false, true>(s, a.c, 1.44269504088896341f);
        if (lane == 0) r.slots = s;
    }
    bad = __any_sync(0xffffffffu, bad);
    if (lane == 0) {
        r.Q = Q, r.rest = rest, r.own = own, r.base = base, r.used = used;
        r.index[a.k] = -1;
        r.z_target = 0.0f;
        if (a.hard) {
            if (t >= 0 && t < a.V) {
                r.index[a.k] = (int)t;
                r.z_target = to_float(zr[t]);
            } else {
                bad = true;
            }
        }
        r.bad = bad;
    }
    __syncwarp();
}

// One thread.  The row's loss, and what its gradient is made of.  s: the sums of
// the row, or of what no slot names (tail)
__device__ __forceinline__ float distill_row(const DistillArgs& a, uint32_t row, Sums s, DistillRow& r) {
    const float c1 = 1.44269504088896341f;
    const bool two = a.hard && a.tau != 1.0f;
    const Sums rest = s;
    if (a.tail) s = two ? join<false, true>(s, r.slots, a.c, c1) : join<false, false>(s, r.slots, a.c, c1);
    const float h = shift_of(s.m), log_s = logf(s.s);
    float kl = r.own;
    // - ln p_i = ln s - (z_i - h) / tau, and own holds - (z_i - base) / tau
    if (r.used != 0.0f) kl += r.used * (s.s == 0.0f ? INFINITY : log_s - (r.base - h) / a.tau);
    const float hr = shift_of(rest.m);
    if (a.tail && r.rest != 0.0f)
        kl += rest.s == 0.0f ? (r.rest != r.rest ? NAN : INFINITY)
                             : r.rest * (logf(r.rest) - ((hr - h) / a.tau + logf(rest.s) - log_s));
    float loss = a.alpha == 0.0f ? 0.0f : a.alpha * a.tau * a.tau * kl;
    const float s1 = two ? s.s1 : s.s;
    if (a.hard) loss -= (1.0f - a.alpha) * (s1 == 0.0f ? -INFINITY : r.z_target - h - logf(s1));
    if (r.bad) loss = NAN;
    if (a.d.p) {
        float w = a.scale * (a.scale_p ? *a.scale_p : 1.0f) * (a.g ? a.g[a.g_rows ? row : 0] : 1.0f);
        if (r.bad) w = NAN;
        const float soft = w * a.alpha * a.tau, hard = a.hard ? w * (1.0f - a.alpha) : 0.0f;
        const float inv = s.s == 0.0f ? 0.0f : 1.0f / s.s, inv1 = s1 == 0.0f ? 0.0f : 1.0f / s1;
        r.w = soft;
        r.w_hard = hard;
        r.h1 = h;
        r.coef1 = two ? hard * inv1 : 0.0f;
        r.inside = soft * r.Q * inv + (two ? 0.0f : hard * inv);
        if (a.tail) {
            const float f = exp2_approx(exponent(rest.m, h, a.c));
            r.h = hr;
            r.coef = rest.s == 0.0f ? 0.0f * w : f * r.inside - soft * r.rest / rest.s;
        } else {
            r.h = h;
            r.coef = r.inside;
        }
    }
    return loss;
}

struct DistillGrad {
    float h, coef, h1, coef1, c;
    __device__ __forceinline__ explicit DistillGrad(const DistillRow& r, float c_)
        : h(r.h), coef(r.coef), h1(r.h1), coef1(r.coef1), c(c_) {}
    template <bool S1>
    __device__ __forceinline__ float at(float z) const {
        float y = exp2_approx((z - h) * c) * coef;
        if constexpr (S1) y = fmaf(exp2_approx((z - h1) * 1.44269504088896341f), coef1, y);
        return y;
    }
};

// the slots and the target in logits j0 .. j1 - 1, after the others' gradient was written
template <class T, bool S1>
__device__ __forceinline__ void distill_grad_slots(const DistillArgs& a, const DistillRow& r, const T* zr, T* dr, int j0,
                                                   int j1, int tid, int threads) {
    const DistillGrad g(r, a.c);
    for (int i = tid; i <= a.k; i += threads) {
        const int j = r.index[i];
        if (j < j0 || j >= j1) continue;
        bool first = true;
        for (int n = 0; n < i; ++n) first &= r.index[n] != j;
        if (!first) continue;
        float q = 0.0f;  // all that is taken off at j, in the order of the slots
        for (int n = i; n < a.k; ++n)
            if (r.index[n] == j) q += r.q[n];
        const float z = to_float(zr[j]);
        float y;
        if (i < a.k) {
            y = fmaf(exp2_approx((z - r.h1) * a.c), r.inside, -r.w * q);
            if constexpr (S1) y = fmaf(exp2_approx((z - r.h1) * 1.44269504088896341f), r.coef1, y);
        } else {
            y = g.template at<S1>(z);
        }
        if (r.index[a.k] == j) y -= r.w_hard;
        dr[j] = from_float<T>(y);
    }
}

// ---- rows of at most 32 E logits: one warp a row, the row in registers --------------

template <int DT, int E, bool TAIL, bool S1>
__global__ void __launch_bounds__(256) distill_warp_kernel(DistillArgs a) {
    using T = typename Elem<DT>::type;
    if (a.skip_if_one && *a.g == 1.0f) return;
    __shared__ DistillRow rows[8];
    __shared__ uint32_t named[8][TAIL ? 32 : 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float c1 = 1.44269504088896341f;
    DistillRow& r = rows[warp];
    for (uint32_t row = blockIdx.x * 8 + warp; row < a.N; row += gridDim.x * 8) {
        const int64_t t = a.tok.p ? a.tok.p[row_offset(a.tok.sb, a.tok.st, a.z.T, row)] : 0;
        T* dr = a.d.p ? reinterpret_cast<T*>(a.d.p) + row_offset(a.d.sb, a.d.st, a.d.T, row) : nullptr;
        if (a.tok.p && t == a.tok.ignore) {
            if (dr)
                for (int j = lane; j < a.V; j += 32) dr[j] = from_float<T>(0.0f);
            if (a.loss && lane == 0) a.loss[row] = 0.0f;
            continue;
        }
        const T* zr = reinterpret_cast<const T*>(a.z.p) + row_offset(a.z.sb, a.z.st, a.z.T, row);
        float x[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int j = lane + 32 * e;
            x[e] = j < a.V ? to_float(zr[j]) : -INFINITY;
        }
        distill_slots<DT>(a, row, zr, t, r);
        Sums s = no_sums();
        {
            float y[E], cm = -INFINITY;
            if constexpr (TAIL) {
                named[warp][lane] = 0;
                __syncwarp();
                for (int i = lane; i < a.k; i += 32)
                    if (r.index[i] >= 0) atomicOr(&named[warp][r.index[i] >> 5], 1u << (r.index[i] & 31));
                __syncwarp();
            }
#pragma unroll
            for (int e = 0; e < E; ++e) {
                y[e] = x[e];
                if constexpr (TAIL)
                    if (named[warp][e] >> lane & 1u) y[e] = -INFINITY;
                cm = fmaxf(cm, y[e]);
            }
            add_values<E, false, S1>(s, y, cm, a.c, c1);
        }
        s = warp_join<false, S1>(s, a.c, c1);
        if (lane == 0) {
            const float loss = distill_row(a, row, s, r);
            if (a.loss) a.loss[row] = loss;
        }
        __syncwarp();
        if (dr) {
            const DistillGrad g(r, a.c);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int j = lane + 32 * e;
                if (j < a.V) dr[j] = from_float<T>(g.template at<S1>(x[e]));
            }
            __syncwarp();
            distill_grad_slots<T, S1>(a, r, zr, dr, 0, a.V, lane, 32);
        }
        __syncwarp();
    }
}

// ---- longer rows: a CTA, or a cluster of CTAs, a row --------------------------------

// words of the bitmap of a part of a row: its vectors' logits, 8 of the head, 8 of the tail
__host__ __device__ constexpr int distill_words(int V, int ctas) { return (V / ctas + 8 + 31) / 32 + 2; }

template <int DT, bool TAIL, bool S1>
__global__ void __launch_bounds__(kRowThreads, 2) distill_row_kernel(DistillArgs a, uint32_t ctas) {
    using T = typename Elem<DT>::type;
    constexpr int kVec = Elem<DT>::kVec, kU = kRowElems / kVec;
    if (a.skip_if_one && *a.g == 1.0f) return;
    extern __shared__ uint32_t named[];  // [distill_words]
    __shared__ DistillRow r;
    __shared__ Sums part[kRowThreads / 32];
    __shared__ __align__(16) Sums mine[2];
    const int tid = threadIdx.x;
    const uint32_t rank = blockIdx.x % ctas;
    const float c1 = 1.44269504088896341f;
    if constexpr (TAIL) {
        for (int i = tid; i < distill_words(a.V, ctas); i += kRowThreads) named[i] = 0;
        __syncthreads();
    }
    int parity = 0;
    for (uint32_t row = blockIdx.x / ctas; row < a.N; row += gridDim.x / ctas) {
        const int64_t t = a.tok.p ? a.tok.p[row_offset(a.tok.sb, a.tok.st, a.z.T, row)] : 0;
        const bool live = !(a.tok.p && t == a.tok.ignore);
        const T* zr = reinterpret_cast<const T*>(a.z.p) + row_offset(a.z.sb, a.z.st, a.z.T, row);
        T* dr = a.d.p ? reinterpret_cast<T*>(a.d.p) + row_offset(a.d.sb, a.d.st, a.d.T, row) : nullptr;
        const Segment g = segment_of<DT>(zr, a.V, rank, ctas);
        const uint4* body = reinterpret_cast<const uint4*>(zr + g.h0);
        const bool wide = (((uintptr_t)zr ^ (uintptr_t)dr) & 15u) == 0;  // 16-byte stores
        if (live) {
            // bit of a logit of this part: vectors first, then head and tail
            auto bit_of = [&](int j) {
                const int body_bits = (g.v1 - g.v0) * kVec;
                return j < g.h0 ? body_bits + j : j >= g.t0 ? body_bits + 8 + (j - g.t0) : j - g.h0 - g.v0 * kVec;
            };
            if (tid < 32) {
                distill_slots<DT>(a, row, zr, t, r);
                if constexpr (TAIL) {
                    for (int i = tid; i < a.k; i += 32)
                        if (r.index[i] >= g.j0 && r.index[i] < g.j1) {
                            const int b = bit_of(r.index[i]);
                            atomicOr(&named[b >> 5], 1u << (b & 31));
                        }
                }
            }
            if constexpr (TAIL) __syncthreads();
            auto is_named = [&](int b) { return (named[b >> 5] >> (b & 31) & 1u) != 0; };
            Sums s = no_sums();
            for (int v = g.v0; v < g.v1; v += kU * kRowThreads) {
                float x[kRowElems];
#pragma unroll
                for (int u = 0; u < kU; ++u) {
                    const int w = v + tid + u * kRowThreads;
                    unpack16<DT>(w < g.v1 ? __ldg(body + w) : neg_inf16<DT>(), x + u * kVec);
                    if constexpr (TAIL) {
                        if (w < g.v1) {
                            const int b = (w - g.v0) * kVec;
                            const uint32_t bits = named[b >> 5] >> (b & 31) & ((1u << kVec) - 1u);
                            if (bits) {
#pragma unroll
                                for (int e = 0; e < kVec; ++e)
                                    if (bits >> e & 1u) x[u * kVec + e] = -INFINITY;
                            }
                        }
                    }
                }
                float cm = x[0];
#pragma unroll
                for (int i = 1; i < kRowElems; ++i) cm = fmaxf(cm, x[i]);
                add_values<kRowElems, false, S1>(s, x, cm, a.c, c1);
            }
            if (tid < g.head + g.tail) {
                const int j = tid < g.head ? tid : g.t0 + (tid - g.head);
                float x[1] = {to_float(zr[j])};
                if constexpr (TAIL)
                    if (is_named(bit_of(j))) x[0] = -INFINITY;
                add_values<1, false, S1>(s, x, x[0], a.c, c1);
            }
            s = cta_join<kRowThreads, false, S1>(s, part, a.c, c1);
            if (ctas > 1) {
                s = cluster_join<false, S1>(s, &mine[parity], ctas, a.c, c1);
                parity ^= 1;
            }
            if (tid == 0) {
                const float loss = distill_row(a, row, s, r);
                if (a.loss && rank == 0) a.loss[row] = loss;
            }
            if constexpr (TAIL) {
                if (tid < 32)
                    for (int i = tid; i < a.k; i += 32)
                        if (r.index[i] >= g.j0 && r.index[i] < g.j1) named[bit_of(r.index[i]) >> 5] = 0;
            }
            __syncthreads();
        } else if (a.loss && rank == 0 && tid == 0) {
            a.loss[row] = 0.0f;
        }
        if (dr) {
            const DistillGrad gr(r, a.c);
            for (int v = g.v0 + tid; v < g.v1; v += kRowThreads) {
                float y[kVec];
                if (live) {
                    float x[kVec];
                    unpack16<DT>(__ldg(body + v), x);
#pragma unroll
                    for (int e = 0; e < kVec; ++e) y[e] = gr.template at<S1>(x[e]);
                } else {
#pragma unroll
                    for (int e = 0; e < kVec; ++e) y[e] = 0.0f;
                }
                T* to = dr + g.h0 + (int64_t)v * kVec;
                if (wide) {
                    __stcs(reinterpret_cast<uint4*>(to), pack16<DT>(y));
                } else {
#pragma unroll
                    for (int e = 0; e < kVec; ++e) to[e] = from_float<T>(y[e]);
                }
            }
            if (tid < g.head + g.tail) {
                const int j = tid < g.head ? tid : g.t0 + (tid - g.head);
                dr[j] = from_float<T>(live ? gr.template at<S1>(to_float(zr[j])) : 0.0f);
            }
            __syncthreads();
            if (live) distill_grad_slots<T, S1>(a, r, zr, dr, g.j0, g.j1, tid, kRowThreads);
        }
        __syncthreads();  // r is written again for the next row
    }
    if (ctas > 1) cluster_sync();  // no CTA ends while another may still read its shared memory
}

// ws[0] = 1 / (rows that are not padding, at least 1); one CTA of 1024 threads
__global__ void __launch_bounds__(1024) distill_count_kernel(Tokens tok, uint32_t T, uint32_t N, float* ws) {
    __shared__ int part[32];
    int n = 0;
    for (uint32_t row = threadIdx.x; row < N; row += 1024) n += tok.p[row_offset(tok.sb, tok.st, T, row)] != tok.ignore;
    n = __reduce_add_sync(0xffffffffu, n);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = n;
    __syncthreads();
    if (threadIdx.x < 32) {
        n = __reduce_add_sync(0xffffffffu, part[threadIdx.x]);
        if (threadIdx.x == 0) ws[0] = 1.0f / (float)(n > 1 ? n : 1);
    }
}

// loss = scale * (*scale_p) * sum of the rows' losses, in a fixed order; one CTA of 1024 threads
__global__ void __launch_bounds__(1024) distill_total_kernel(const float* rows, uint32_t N, float scale,
                                                             const float* scale_p, float* loss) {
    __shared__ float part[32];
    float v = 0.0f;
    for (uint32_t row = threadIdx.x; row < N; row += 1024) v += rows[row];
    v = warp_sum(v);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    if (threadIdx.x < 32) {
        v = warp_sum(part[threadIdx.x]);
        if (threadIdx.x == 0) *loss = v * scale * (scale_p ? *scale_p : 1.0f);
    }
}

}  // namespace il
