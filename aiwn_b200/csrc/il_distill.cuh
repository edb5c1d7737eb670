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
// difference of inputs, is taken in 64 bits; where it is less than 2^-16 and
// the student has nothing outside the slots, it is rounding and counts for 0.
//
// 8192 x 131072 bf16 with 64 slots and the gradient (4.3 GB, 658 us at the
// measured copy rate): 890 us.  The rows at work are kept to 62 MB, so that the
// second reading finds them in the L2: 148 rows of 256 KB (a CTA of 512 threads
// an SM) read 544 MB of 537 from HBM, 296 rows 871 MB and took 1007 us.  Rows of
// 128 KB take 256 threads, two rows an SM (4096 x 65536: 254 us, of 165).  What is left is
// what a row costs between its two readings (join, factors, two barriers), which
// one or two CTAs an SM do not hide: DRAM is 64% busy, the issue slots 48%.
// 4096 x 32768 bf16, 20 slots, the loss alone: 61 us (0.27 GB, 41 us at the
// measured copy rate); with 30% of the rows padding, which are not read, 53 us
// (0.19 GB, 29 us): rows are dealt out beforehand, and some CTAs keep all theirs.
#pragma once
#include "il_logits.cuh"

namespace il {

// What fp32 log probabilities leave of a mass of one by their own rounding: that of a sum over a long row is a few 2^-20
// (the largest vocabularies' bound is 2^-12, of which such sums use little).  Less than this is no bucket where the
// student has nothing outside the slots, that is 2^-150 of its mass or less: the slots then name the whole vocabulary,
// or all that a mask has left of it, and q_r ln p_r would be 1e-8 times minus infinity, or times a mask's -3e38.
constexpr double kRounding = 1.0 / 65536;

constexpr int kMean = 1;  // reduction; 2: the sum, 0: each row's loss

struct DistillArgs {
    RowsIn z;
    Tokens tok;  // targets; padded rows are tok.ignore
    RowsOut d;   // gradient, d.p == nullptr: none
    uint32_t N;
    int V, k;
    const int64_t* index;  // [N, k], < 0: empty slot
    const float* logprob;  // [N, k]
    float tau, c, alpha;
    int hard;              // the target's term is wanted (alpha < 1)
    float scale;           // of the gradient and of a whole loss
    const float* scale_p;  // times *scale_p, or null
    const float* g;        // gradient: times g[0], or g[row] with g_rows, or null
    int g_rows;
    int skip_if_one;       // nothing is left to do where g[0] == 1
    float* loss;           // [N] (each), [1], or null
    int each;
    uint32_t* ticket;      // 0 before the call, and partial sums of a whole loss, one a CTA
    float* partial;
};

struct Slot {  // a teacher's value, of one lane
    int j;     // -1: none
    float l, z;
};

// What a warp's lanes found out about their slots: with w_i = exp(l_i - top)
// (tail: exp(l_i)), mass = sum w, cross = sum w ((l_i - top) - (z_i - base) / tau)
struct SlotSums {
    float top, mass, cross, base;
    double left;  // sum of exp(l_i) in 64 bits (tail)
    Sums s;       // of the slots' logits, each token once (tail)
    int bad, again;  // a slot beyond the vocabulary; a token that an earlier slot names too
};

// a barrier of the warps that keep the slots
__device__ __forceinline__ void slot_barrier(int threads) {
    asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory");
}

template <bool TAIL>
__device__ __forceinline__ float slot_weight(float l, float top) {
    return TAIL ? expf(l) : expf(l - top);
}

// Whether the slots of this lane, lane + 32 q of those from index[base] on, are the first of index[0 ..] to name their
// tokens.  After a barrier of those who wrote `index`.
template <int n>
__device__ __forceinline__ void slot_firsts(const Slot (&x)[n], int used, const int* index, int base, bool (&first)[n]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int q = 0; q < n; ++q) {
        first[q] = true;
        if (q >= used) continue;
        const unsigned peers = __match_any_sync(0xffffffffu, x[q].j);
        first[q] = lane == __ffs(peers) - 1;
        for (int i = 0; i < base + 32 * q; ++i) first[q] &= index[i] != x[q].j;
    }
}

// n: slots of this lane; first: whether slot q is the first to name its token
template <bool TAIL, bool S1, int n>
__device__ __forceinline__ SlotSums slot_sums(const DistillArgs& a, const Slot (&x)[n], int used, bool bad,
                                              const bool (&first)[n]) {
    SlotSums r;
    float top = -INFINITY, base = -INFINITY;
#pragma unroll
    for (int q = 0; q < n; ++q)
        if (q < used) top = fmaxf(top, x[q].l), base = fmaxf(base, x[q].z);
    r.top = TAIL ? 0.0f : shift_of(warp_max(top));
    r.base = shift_of(warp_max(base));
    float mass = 0.0f, cross = 0.0f;
    double left = 0.0;
    r.s = no_sums();
#pragma unroll
    for (int q = 0; q < n; ++q) {
        if (q >= used) continue;
        const bool is = x[q].j >= 0;
        const float w = is ? slot_weight<TAIL>(x[q].l, r.top) : 0.0f;
        mass += w;
        if (w != 0.0f) cross += w * ((x[q].l - r.top) - (x[q].z - r.base) / a.tau);
        if constexpr (TAIL) {
            if (is) left += exp((double)x[q].l);
            if (is && first[q]) {
                const float y[1] = {x[q].z};
                add_values<1, false, S1>(r.s, y, x[q].z, a.c);
            }
        }
    }
    r.mass = warp_sum(mass);
    r.cross = warp_sum(cross);
    if constexpr (TAIL) {
        r.left = warp_sum(left);
        r.s = warp_join<false, S1>(r.s, a.c);
    }
    bool again = false;
#pragma unroll
    for (int q = 0; q < n; ++q) again |= x[q].j >= 0 && !first[q];
    r.bad = __any_sync(0xffffffffu, bad);
    r.again = __any_sync(0xffffffffu, again);
    return r;
}

// A row's gradient at a logit that no slot names: 2^((z - h) c) coef + 2^((z - h1) log2 e) coef1;
// at one that slots name: 2^((z - h1) c) inside + 2^((z - h1) log2 e) coef1 - soft sum of the slots' weights;
// less `hard` at the target.
struct DistillRow {
    float h, coef, h1, coef1, inside, soft, hard, top, c;
    template <bool S1>
    __device__ __forceinline__ float at(float z) const {
        float y = exp2_approx((z - h) * c) * coef;
        if constexpr (S1) y = fmaf(exp2_approx((z - h1) * kLog2e), coef1, y);
        return y;
    }
    template <bool S1>
    __device__ __forceinline__ float at_slot(float z, float weight) const {
        float y = fmaf(exp2_approx((z - h1) * c), inside, -soft * weight);
        if constexpr (S1) y = fmaf(exp2_approx((z - h1) * kLog2e), coef1, y);
        return y;
    }
};

// at() of many values, (z - h) c as one fused multiply-add: with b = -h c rounded and r = h c + b exactly, the
// exponential of z c + b is 2^r too large, which the factor takes back.  Not where |h| c is 2^22 or more.
template <bool S1>
struct DistillMany {
    float c, b, f, b1, f1;
    bool huge;
    __device__ __forceinline__ explicit DistillMany(const DistillRow& r) : c(r.c) {
        b = -(r.h * c);
        f = r.coef * exp2_approx(-fmaf(r.h, c, b));
        b1 = -(r.h1 * kLog2e);
        f1 = r.coef1 * exp2_approx(-fmaf(r.h1, kLog2e, b1));
        huge = !(fabsf(b) < 4194304.0f) || (S1 && !(fabsf(b1) < 4194304.0f));
    }
    template <int n>
    __device__ __forceinline__ void operator()(float (&x)[n]) const {
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const float z = x[i];
            x[i] = exp2_approx(fmaf(z, c, b)) * f;
            if constexpr (S1) x[i] = fmaf(exp2_approx(fmaf(z, kLog2e, b1)), f1, x[i]);
        }
    }
};

// a vector's gradient, of any size and to any address
template <int DT, bool S1>
__device__ __noinline__ void write_slowly(const DistillRow* r, uint4 z, typename Elem<DT>::type* to) {
    constexpr int kVec = Elem<DT>::kVec;
    float x[kVec];
    unpack16<DT>(z, x);
#pragma unroll
    for (int e = 0; e < kVec; ++e) to[e] = from_float<typename Elem<DT>::type>(r->template at<S1>(x[e]));
}

// What a row's sums and its slots' come to.  s: the sums of the row, or of what no slot names (tail); part: the
// slots' of `parts` warps; z_t: the target's logit, NaN for one outside the vocabulary
template <bool TAIL, bool S1>
struct DistillSums {
    Sums s, rest;
    float top, mass, inv_mass, q_rest, Q;
    bool bad;

    __device__ __forceinline__ DistillSums(const DistillArgs& a, Sums sums, const SlotSums* part, int parts, float z_t)
        : s(sums), rest(sums) {
        top = 0.0f, mass = 0.0f;
        bad = a.hard && z_t != z_t;
        if constexpr (!TAIL) {
            top = -INFINITY;
            for (int n = 0; n < parts; ++n)
                if (part[n].mass != 0.0f) top = fmaxf(top, part[n].top);
            top = shift_of(top);
        }
        double left = 1.0;
        for (int n = 0; n < parts; ++n) {
            bad |= part[n].bad != 0;
            mass = fmaf(part[n].mass, weight_of(part[n]), mass);
            if constexpr (TAIL) {
                s = join<false, S1>(s, part[n].s, a.c);
                left -= part[n].left;
            }
        }
        inv_mass = TAIL ? 1.0f : mass != 0.0f ? 1.0f / mass : 0.0f;  // NaN stays
        bool none = left < 0.0;  // no bucket
        if (TAIL && !none && left < kRounding)
            none = (rest.m - shift_of(s.m)) * a.c + log2f(rest.s) - log2f(s.s) < kMinExp;
        q_rest = !TAIL || none ? 0.0f : (float)left;  // NaN stays
        Q = TAIL ? (none ? mass : 1.0f + 0.0f * q_rest) : mass != 0.0f ? 1.0f + 0.0f * mass : 0.0f;
    }
    // of a warp's slots next to the others'
    __device__ __forceinline__ float weight_of(const SlotSums& p) const {
        return TAIL ? 1.0f : p.mass != 0.0f ? expf(p.top - top) : 0.0f;
    }

    __device__ __forceinline__ DistillRow gradient(const DistillArgs& a, uint32_t row) const {
        DistillRow r;
        float w = a.scale * (a.scale_p ? *a.scale_p : 1.0f) * (a.g ? a.g[a.g_rows ? row : 0] : 1.0f);
        if (bad) w = NAN;
        const float s1 = S1 ? s.s1 : s.s;
        const float soft = w * a.alpha * a.tau, hard = a.hard ? w * (1.0f - a.alpha) : 0.0f;
        const float inv = s.s == 0.0f ? 0.0f : 1.0f / s.s;
        r.c = a.c;
        r.h1 = shift_of(s.m);
        r.top = top;
        r.soft = soft * inv_mass;
        r.hard = hard;
        r.coef1 = S1 ? hard * (s1 == 0.0f ? 0.0f : 1.0f / s1) : 0.0f;
        r.inside = soft * Q * inv + (S1 ? 0.0f : hard * inv);
        if constexpr (TAIL) {
            const float f = exp2_approx(exponent(rest.m, r.h1, a.c));
            r.h = shift_of(rest.m);
            r.coef = rest.s == 0.0f ? 0.0f * w : f * r.inside - soft * q_rest / rest.s;
        } else {
            r.h = r.h1;
            r.coef = r.inside;
        }
        return r;
    }

    __device__ __forceinline__ float loss(const DistillArgs& a, const SlotSums* part, int parts, float z_t) const {
        const float h = shift_of(s.m), s1 = S1 ? s.s1 : s.s, log_s = logf(s.s);
        // sum q (ln q - (z - h) / tau), then + sum q (ln s)
        float kl = 0.0f, used = 0.0f;
        for (int n = 0; n < parts; ++n) {
            const float f = weight_of(part[n]);
            if (part[n].mass == 0.0f || f == 0.0f) continue;
            const float q = part[n].mass * f * inv_mass;
            kl += part[n].cross * f * inv_mass + q * ((TAIL ? 0.0f : part[n].top - top) - (part[n].base - h) / a.tau);
            used += q;
        }
        if (used != 0.0f) kl += used * (s.s == 0.0f ? INFINITY : log_s - (TAIL ? 0.0f : logf(mass)));
        if (TAIL && q_rest != 0.0f)
            kl += rest.s == 0.0f ? (q_rest != q_rest ? NAN : INFINITY)
                                 : q_rest * (logf(q_rest) - ((shift_of(rest.m) - h) / a.tau + logf(rest.s) - log_s));
        float loss = a.alpha == 0.0f ? 0.0f : a.alpha * a.tau * a.tau * kl;
        if (a.hard) loss -= (1.0f - a.alpha) * (s1 == 0.0f ? -INFINITY : z_t - h - logf(s1));
        return bad ? NAN : loss;
    }
};

// The gradient at the token of logit z of a slot of weight w (exp(l), up to the row's common factor).
// again: other slots may name it too; then the first of them writes for all.  index, logprob: the row's k slots,
// index[k] the target or -1.
template <class T, bool TAIL, bool S1>
__device__ __forceinline__ void distill_grad_slot(const DistillRow& r, const int* index, const float* logprob, int k,
                                                  int q, bool again, float z, T* dr) {
    const int j = index[q];
    float weight = slot_weight<TAIL>(logprob[q], r.top);
    if (again) {
        for (int n = 0; n < q; ++n)
            if (index[n] == j) return;
        for (int n = q + 1; n < k; ++n)
            if (index[n] == j) weight += slot_weight<TAIL>(logprob[n], r.top);
    }
    const float y = r.template at_slot<S1>(z, weight);
    dr[j] = from_float<T>(index[k] == j ? y - r.hard : y);
}

// One warp: the gradient at the target of logit z, where no slot names it
template <class T, bool S1>
__device__ __forceinline__ void distill_grad_target(const DistillRow& r, const int* index, int k, float z, T* dr) {
    const int j = index[k], lane = threadIdx.x & 31;
    bool named = false;
    for (int n = lane; n < k; n += 32) named |= index[n] == j;
    if (!__any_sync(0xffffffffu, named) && lane == 0) dr[j] = from_float<T>(r.template at<S1>(z) - r.hard);
}

// A slot as it stands in memory; false: its index is beyond the vocabulary
__device__ __forceinline__ bool read_slot(const DistillArgs& a, int64_t at, int& j, float& l) {
    const int64_t x = a.index[at];
    j = x >= 0 && x < a.V ? (int)x : -1;
    l = j >= 0 ? a.logprob[at] : -INFINITY;
    return x < a.V;
}

// The rows' losses of a CTA have been added up by thread `owner`; the last CTA adds up the CTAs', in their order.
__device__ __forceinline__ void distill_total(const DistillArgs& a, float sum, int owner, float* shared, int threads) {
    if (!a.loss || a.each) return;
    __shared__ bool last;
    if (threadIdx.x == owner) {
        a.partial[blockIdx.x] = sum;
        __threadfence();
        last = atomicAdd(a.ticket, 1u) == gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    float v = 0.0f;
    for (uint32_t i = threadIdx.x; i < gridDim.x; i += threads) v += __ldcg(a.partial + i);
    v = warp_sum(v);
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
    __syncthreads();
    if (threadIdx.x < 32) {
        v = warp_sum(threadIdx.x < (threads >> 5) ? shared[threadIdx.x] : 0.0f);
        if (threadIdx.x == 0) *a.loss = v * a.scale * (a.scale_p ? *a.scale_p : 1.0f);
    }
}

// ---- rows of at most 32 E logits: one warp a row, the row in registers --------------

template <int DT, int E, bool TAIL, bool S1>
__global__ void __launch_bounds__(256) distill_warp_kernel(DistillArgs a) {
    using T = typename Elem<DT>::type;
    constexpr int kPer = kMaxTop / 32;
    if (a.skip_if_one && *a.g == 1.0f) return;
    __shared__ int index[8][kMaxTop + 1];
    __shared__ float logprob[8][kMaxTop], total[8];
    __shared__ uint32_t named[8][TAIL ? 32 : 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int used = (a.k + 31) / 32;
    int* idx = index[warp];
    float sum = 0.0f;
    for (uint32_t row = blockIdx.x * 8 + warp; row < a.N; row += gridDim.x * 8) {
        const int64_t t = a.tok.p ? a.tok.p[row_offset(a.tok.sb, a.tok.st, a.tok.T, row)] : 0;
        const T* zr = reinterpret_cast<const T*>(a.z.p) + row_offset(a.z.sb, a.z.st, a.z.T, row);
        T* dr = a.d.p ? reinterpret_cast<T*>(a.d.p) + row_offset(a.d.sb, a.d.st, a.d.T, row) : nullptr;
        float x[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int j = lane + 32 * e;
            x[e] = j < a.V ? to_float(zr[j]) : -INFINITY;
        }
        Slot slot[kPer];
        bool bad = false;
#pragma unroll
        for (int q = 0; q < kPer; ++q) {
            slot[q] = Slot{-1, -INFINITY, -INFINITY};
            if (lane + 32 * q < a.k)
                bad |= !read_slot(a, (int64_t)row * a.k + lane + 32 * q, slot[q].j, slot[q].l);
        }
        if (a.tok.p && t == a.tok.ignore) {
            if (dr)
                for (int j = lane; j < a.V; j += 32) dr[j] = from_float<T>(0.0f);
            if (a.loss && a.each && lane == 0) a.loss[row] = 0.0f;
            continue;
        }
        const bool in = a.hard && t >= 0 && t < a.V;
        const float z_t = in ? to_float(zr[t]) : NAN;
#pragma unroll
        for (int q = 0; q < kPer; ++q) {
            if (slot[q].j >= 0) slot[q].z = to_float(zr[slot[q].j]);
            const int i = lane + 32 * q;
            if (i < a.k) idx[i] = slot[q].j, logprob[warp][i] = slot[q].l;
        }
        if (lane == 0) idx[a.k] = in ? (int)t : -1;
        if constexpr (TAIL) named[warp][lane] = 0;
        __syncwarp();
        bool first[kPer];
        slot_firsts<kPer>(slot, used, idx, 0, first);
        if constexpr (TAIL) {
#pragma unroll
            for (int q = 0; q < kPer; ++q)
                if (first[q] && slot[q].j >= 0) atomicOr(&named[warp][slot[q].j >> 5], 1u << (slot[q].j & 31));
            __syncwarp();
        }
        const SlotSums slots = slot_sums<TAIL, S1, kPer>(a, slot, used, bad, first);
        Sums s = no_sums();
        {
            float y[E], cm = -INFINITY;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                y[e] = x[e];
                if constexpr (TAIL)
                    if (named[warp][e] >> lane & 1u) y[e] = -INFINITY;
                cm = fmaxf(cm, y[e]);
            }
            s.m = warp_max(cm);
            add_values<E, false, S1>(s, y, s.m, a.c);
            s.s = warp_sum(s.s);
            if constexpr (S1) s.s1 = warp_sum(s.s1);
        }
        const DistillSums<TAIL, S1> all(a, s, &slots, 1, z_t);
        if (a.loss) {
            const float loss = all.loss(a, &slots, 1, z_t);
            sum += loss;
            if (a.each && lane == 0) a.loss[row] = loss;
        }
        if (dr) {
            const DistillRow r = all.gradient(a, row);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int j = lane + 32 * e;
                if (j < a.V) dr[j] = from_float<T>(r.template at<S1>(x[e]));
            }
            __syncwarp();
#pragma unroll
            for (int q = 0; q < kPer; ++q)
                if (slot[q].j >= 0)
                    distill_grad_slot<T, TAIL, S1>(r, idx, logprob[warp], a.k, lane + 32 * q, slots.again, slot[q].z, dr);
            if (in) distill_grad_target<T, S1>(r, idx, a.k, z_t, dr);
        }
        __syncwarp();
    }
    if (a.loss && !a.each) {
        __syncthreads();
        if (lane == 0) total[warp] = sum;
        __syncthreads();
        float v = 0.0f;
        for (int w = 0; w < 8; ++w) v += total[w];
        __syncthreads();
        distill_total(a, v, 0, total, 256);
    }
}

// ---- longer rows: a CTA, or a cluster of CTAs, a row --------------------------------

// bytes of the bitmap of a part of a row: one a vector, to the end of a step, and 16 for the row's ends
__host__ __device__ constexpr int distill_bitmap(int V, int ctas, int vec, int step) {
    return (V / vec / ctas + 1 + step - 1) / step * step + 16;
}

// a vector with -inf in place of the logits whose bits are set
template <int DT>
__device__ __forceinline__ uint4 without(const uint4& r, uint32_t bits) {
    uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (DT == kF32) {
            if (bits >> i & 1u) w[i] = 0xff800000u;
        } else {
            if (bits >> (2 * i) & 1u) w[i] = (w[i] & 0xffff0000u) | 0xff80u;
            if (bits >> (2 * i + 1) & 1u) w[i] = (w[i] & 0xffffu) | 0xff800000u;
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Of a CTA's warps the last ones keep the slots, one a lane, and are a row ahead: the slots' indices and values are
// read a row before their logits, and those (and what they come to) right after the sums of the row before.  The
// first two warps bring a row's sums and its slots' together.
template <int DT, int kThreads, bool TAIL, bool S1, bool GRAD>
__global__ void __launch_bounds__(kThreads, sm_threads(GRAD ? 2 : 1) / kThreads) distill_row_kernel(DistillArgs a, uint32_t lg) {
    using T = typename Elem<DT>::type;
    using Stream = RowStream<DT, kThreads, GRAD ? 2 : 1>;
    constexpr int kVec = Elem<DT>::kVec, kU = Stream::kU, kWarps = kThreads / 32;
    if (a.skip_if_one && *a.g == 1.0f) return;
    extern __shared__ __align__(16) unsigned char sm[];  // the stream's places, the bitmap
    uint8_t* named = sm + Stream::kBytes;
    __shared__ float4 part[2][kWarps], mine[2];
    __shared__ SlotSums slots[2][kMaxTop / 32];
    __shared__ int index[2][kMaxTop + 1];
    __shared__ float logprob[2][kMaxTop], total[kWarps];
    __shared__ DistillRow shared_row[2];
    const int tid = threadIdx.x;
    const uint32_t ctas = 1u << lg, rank = blockIdx.x & (ctas - 1);
    const int slot_warps = (a.k + 31) / 32, own = tid - (kThreads - 32 * slot_warps);  // slot of this thread
    const T* z0 = reinterpret_cast<const T*>(a.z.p);
    if constexpr (TAIL) {
        for (int i = tid; i < distill_bitmap(a.V, ctas, kVec, Stream::kStep) / 4; i += kThreads)
            reinterpret_cast<uint32_t*>(named)[i] = 0;
    }
    const RowList list(a.tok, a.N, blockIdx.x >> lg, gridDim.x >> lg);
    const RowStep step(a.z, gridDim.x >> lg);
    Stream stream(a.z, a.V, list, step, rank, lg, sm);
    // rows of padding
    if (a.tok.p && (GRAD || (a.loss && a.each))) {
        uint32_t live = 0;
        for (uint32_t i = 0; i < list.count; ++i) {
            if ((i & 31) == 0) live = list.window(i);
            if (live >> (i & 31) & 1u) continue;
            const uint32_t row = list.row(i);
            if (a.loss && a.each && rank == 0 && tid == 0) a.loss[row] = 0.0f;
            if constexpr (GRAD) {
                T* dr = reinterpret_cast<T*>(a.d.p) + row_offset(a.d.sb, a.d.st, a.d.T, row);
                const Segment g = segment_of<DT>(dr, a.V, rank, lg);
                uint4* to = reinterpret_cast<uint4*>(dr + g.h0);
                for (int v = g.v0 + tid; v < g.v1; v += kThreads) __stcs(to + v, make_uint4(0, 0, 0, 0));
                if (tid < g.head + g.tail) dr[tid < g.head ? tid : g.t0 + tid - g.head] = from_float<T>(0.0f);
            }
        }
    }
    int parity = 0;
    float sum = 0.0f;
    LiveRows at(a.z, list, step);
    LiveRows ahead = at;  // the row after the one that the slots' logits are read of
    // slot[0]: of the row that `at` will be at; now_*: the same of the row that it is at
    Slot slot[1] = {{-1, -INFINITY, -INFINITY}}, next{-1, -INFINITY, -INFINITY};
    bool ok = true, next_ok = true;
    auto read_ahead = [&] {  // this thread's slot of row `ahead`
        next = Slot{-1, -INFINITY, -INFINITY};
        next_ok = true;
        if (own >= 0 && own < a.k && ahead.valid())
            next_ok = read_slot(a, (int64_t)ahead.row() * a.k + own, next.j, next.l);
    };
    // byte and bit of a logit of this part: those of its vector; in the last 16 bytes, of the head and the tail
    const int ends_byte = TAIL ? distill_bitmap(a.V, ctas, kVec, Stream::kStep) - 16 : 0;
    auto bit_of = [&](const Segment& g, int j) {
        const int i = j - g.h0;
        return j < g.h0 ? ends_byte * 8 + j : j >= g.t0 ? ends_byte * 8 + 8 + (j - g.t0)
                                                        : (i / kVec - g.v0) * 8 + i % kVec;
    };
    uint32_t* named_words = reinterpret_cast<uint32_t*>(named);
    // the slots' indices of row `ahead` into buffer p, and their bits
    auto name = [&](int p) {
        slot[0] = next;
        ok = next_ok;
        if (own >= 0 && own < a.k) {
            index[p][own] = slot[0].j;
            logprob[p][own] = slot[0].l;
            if constexpr (TAIL) {
                const Segment g = segment_of<DT>(z0 + ahead.at.off, a.V, rank, lg);
                if (slot[0].j >= g.j0 && slot[0].j < g.j1) {
                    const int b = bit_of(g, slot[0].j);
                    atomicOr(&named_words[b >> 5], 1u << (b & 31));
                }
            }
        }
    };
    // what those slots come to; `ahead` moves on.  After a barrier of the CTA behind name()
    auto weigh = [&](int p) {
        if (own >= 0 && ahead.valid()) {
            if (slot[0].j >= 0) slot[0].z = to_float(z0[ahead.at.off + slot[0].j]);
            bool first[1];
            slot_firsts<1>(slot, 1, index[p], own & ~31, first);
            const SlotSums x = slot_sums<TAIL, S1, 1>(a, slot, 1, own < a.k && !ok, first);
            if ((tid & 31) == 0) slots[p][own >> 5] = x;
        }
        ahead.next();
        read_ahead();
    };
    read_ahead();
    __syncthreads();  // the bitmap is zero
    name(0);
    __syncthreads();
    weigh(0);
    for (; at.valid(); at.next()) {
        const uint32_t row = at.row();
        const T* zr = z0 + at.at.off;
        T* dr = GRAD ? reinterpret_cast<T*>(a.d.p) + row_offset(a.d.sb, a.d.st, a.d.T, row) : nullptr;
        const Segment g = segment_of<DT>(zr, a.V, rank, lg);
        const int ends = g.head + g.tail, end_at = tid < g.head ? tid : g.t0 + tid - g.head;
        const float end = tid < ends ? to_float(zr[end_at]) : -INFINITY;
        float z_t = 0.0f;
        const int now_j = slot[0].j;
        const float now_z = slot[0].z;
        if (tid < 64) {
            int64_t t = -1;
            if (a.hard) {
                t = a.tok.p[row_offset(a.tok.sb, a.tok.st, a.tok.T, row)];
                z_t = t >= 0 && t < a.V ? to_float(zr[t]) : NAN;
            }
            if (tid == 0) index[parity][a.k] = t >= 0 && t < a.V ? (int)t : -1;
        }
        Running<false, S1> run;
        run.begin(a.c);
        auto use = [&](uint4 (&raw)[kU], int v) {  // v: of the first vector
            if constexpr (TAIL) {
                const uint8_t* byte = named + (v - g.v0);
                uint32_t bits[kU], any = 0;
#pragma unroll
                for (int u = 0; u < kU; ++u) any |= bits[u] = byte[u * kThreads];
                if (any) {
#pragma unroll
                    for (int u = 0; u < kU; ++u)
                        if (bits[u]) raw[u] = without<DT>(raw[u], bits[u]);
                }
            }
            run.template add<DT>(raw, max_of<DT>(raw), a.c);
        };
        int left = g.v1 - g.v0;
        for (; left >= Stream::kStep; left -= Stream::kStep) {
            uint4 raw[kU];
            stream.template take<true>(raw, 0);
            stream.issue();
            use(raw, g.v1 - left + tid);
        }
        if (left > 0) {
            uint4 raw[kU];
            stream.template take<false>(raw, (left - tid + kThreads - 1) / kThreads);
            stream.issue();
            use(raw, g.v1 - left + tid);
        }
        Sums s = run.sums(a.c);
        if (tid < ends) {
            float x[1] = {end};
            if constexpr (TAIL) {
                const int b = bit_of(g, end_at);
                if (named_words[b >> 5] >> (b & 31) & 1u) x[0] = -INFINITY;
            }
            add_values<1, false, S1>(s, x, x[0], a.c);
        }
        s = cta_join<kThreads, false, S1>(s, part[parity], a.c);
        if constexpr (TAIL) {
            // all of the CTA have read the bitmap
            if (own >= 0 && own < a.k && now_j >= g.j0 && now_j < g.j1) named_words[bit_of(g, now_j) >> 5] = 0;
            if (own >= 0) slot_barrier(32 * slot_warps);
        }
        if (ctas > 1) s = cluster_join<false, S1>(s, &mine[parity], ctas, a.c);
        name(parity ^ 1);
        if (tid < 64 && (a.loss || GRAD)) {  // the first warp: the gradient, the second: the loss
            const DistillSums<TAIL, S1> all(a, s, slots[parity], slot_warps, z_t);
            if (tid >= 32) {
                const float loss = all.loss(a, slots[parity], slot_warps, z_t);
                if (rank == 0) sum += loss;
                if (a.loss && a.each && rank == 0 && tid == 32) a.loss[row] = loss;
            } else if constexpr (GRAD) {
                const DistillRow r = all.gradient(a, row);
                if (tid == 0) shared_row[parity] = r;
            }
        }
        if constexpr (GRAD || TAIL) __syncthreads();
        else if (slot_warps > 1 && own >= 0) slot_barrier(32 * slot_warps);
        weigh(parity ^ 1);
        if constexpr (GRAD) {
            const DistillRow r = shared_row[parity];
            const DistillMany<S1> many(r);
            const bool wide = (((uintptr_t)zr ^ (uintptr_t)dr) & 15u) == 0;  // 16-byte stores
            const bool plain = wide && !many.huge;
            auto write = [&](const uint4 (&raw)[kU], int v, int mine) {
                T* to = dr + g.h0 + (int64_t)v * kVec;
                if (plain) {
#pragma unroll
                    for (int u = 0; u < kU; ++u) {
                        if (u >= mine) continue;
                        float x[kVec];
                        unpack16<DT>(raw[u], x);
                        many(x);
                        __stcs(reinterpret_cast<uint4*>(to) + u * kThreads, pack16<DT>(x));
                    }
                } else {
#pragma unroll
                    for (int u = 0; u < kU; ++u)
                        if (u < mine) write_slowly<DT, S1>(&shared_row[parity], raw[u], to + u * kThreads * kVec);
                }
            };
            left = g.v1 - g.v0;
            for (; left >= Stream::kStep; left -= Stream::kStep) {
                uint4 raw[kU];
                stream.template take<true>(raw, 0);
                stream.issue();
                write(raw, g.v1 - left + tid, kU);
            }
            if (left > 0) {
                uint4 raw[kU];
                const int mine = (left - tid + kThreads - 1) / kThreads;
                stream.template take<false>(raw, mine);
                stream.issue();
                write(raw, g.v1 - left + tid, mine);
            }
            if (tid < ends) dr[end_at] = from_float<T>(r.template at<S1>(end));
            __syncthreads();
            if (own >= 0 && own < a.k && now_j >= g.j0 && now_j < g.j1) {
                bool again = false;
                for (int n = 0; n < slot_warps; ++n) again |= slots[parity][n].again != 0;
                distill_grad_slot<T, TAIL, S1>(r, index[parity], logprob[parity], a.k, own, again, now_z, dr);
            }
            if (tid < 32 && index[parity][a.k] >= g.j0 && index[parity][a.k] < g.j1)
                distill_grad_target<T, S1>(r, index[parity], a.k, z_t, dr);
        }
        parity ^= 1;
    }
    if (ctas > 1) cluster_sync();  // no CTA ends while another may still read its shared memory
    __syncthreads();
    distill_total(a, sum, 32, total, kThreads);
}

// ws[0] = 1 / (rows that are not padding, at least 1), ws[1]: the ticket, 0; one CTA of 1024 threads
__global__ void __launch_bounds__(1024) distill_begin_kernel(Tokens tok, uint32_t N, float* ws) {
    __shared__ int part[32];
    int n = 0;
    if (tok.p)
        for (uint32_t row = threadIdx.x; row < N; row += 1024)
            n += tok.p[row_offset(tok.sb, tok.st, tok.T, row)] != tok.ignore;
    n = __reduce_add_sync(0xffffffffu, n);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = n;
    __syncthreads();
    if (threadIdx.x < 32) {
        n = __reduce_add_sync(0xffffffffu, part[threadIdx.x]);
        if (threadIdx.x == 0) {
            ws[0] = 1.0f / (float)(n > 1 ? n : 1);
            reinterpret_cast<uint32_t*>(ws)[1] = 0;
        }
    }
}

}  // namespace il
