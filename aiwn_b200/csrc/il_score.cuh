// il_score.cuh -- log probabilities of given tokens, entropy and the largest
// alternatives of logits rows, and the gradient of all three.
//
//   lse = m / tau + ln s           logprob_t = (z_t - m) / tau - ln s
//   H = ln s - ln(2) u / s         top: the k largest logits, equal ones by index
//   dz_j = 1/tau ( [j = t] g + sum_i [j = idx_i] g_i - p_j (g + sum_i g_i + g_H (ln p_j + H)) )
// with (m, s, u) of il_logits.cuh.  The forward reads each logit once, the
// backward reads it once more and writes its gradient.
//
// The k largest in the same pass.  Every thread knows the maximum of the logits
// that it holds.  For the row's first logits the k-th largest of the threads'
// maxima is a lower bound of the k-th largest logit; from then on only logits
// above the bound are put into a list in shared memory, so that the work on a
// logit that is not among the largest is the comparison of its step's maximum.
// After 1, 2, 4, ... steps the bound rises to what the threads' maxima so far
// say: with j = k / warps (rounded up), the least of the warps' j-th largest.
// For logits in no particular order the list so gets a few times k entries.
// When it could run over, it is sorted and cut to k; when one step alone could
// overrun it, the bound is first taken from that step's maxima: at most k - 1
// threads then hold anything above it, and of the logits equal to it the first
// ones by index are taken.  No input needs a second pass.  List entries are
// (order-preserving bits of z) << 32 | ~index, so that all are distinct and
// equal logits go by their index.
#pragma once
#include "il_logits.cuh"

namespace il {

// unsigned order of floats; NaN counts as -inf, -0 as 0
__device__ __forceinline__ uint32_t order_key(float z) {
    const float v = z != z ? -INFINITY : z + 0.0f;
    const uint32_t b = __float_as_uint(v);
    return (int32_t)b < 0 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}

struct ScoreArgs {
    RowsIn z;
    Tokens tok;
    uint32_t N;
    int V, k;
    float tau, c;
    float* logprob;   // [N] or null
    float* entropy;   // [N]
    float2* stats;    // [N] (m, s) or null
    int64_t* top_index;   // [N, k]
    float* top_logprob;   // [N, k]
};

// the results of a row that do not need its logits: padding
__device__ __forceinline__ void score_padding(const ScoreArgs& a, uint32_t row, int tid, int threads) {
    for (int i = tid; i < a.k; i += threads) {
        a.top_index[(int64_t)row * a.k + i] = -1;
        a.top_logprob[(int64_t)row * a.k + i] = -INFINITY;
    }
    if (tid == 0) {
        if (a.logprob) a.logprob[row] = 0.0f;
        a.entropy[row] = 0.0f;
        if (a.stats) a.stats[row] = make_float2(0.0f, 1.0f);
    }
}

// ln of a probability: logit z in a row with maximum m and sum s
__device__ __forceinline__ float log_prob(float z, float m, float s, float log_s, float tau) {
    return s == 0.0f ? -INFINITY : (z - shift_of(m)) / tau - log_s;
}

// z_t: the token's logit, NaN for a token outside the vocabulary
__device__ __forceinline__ void score_write(const ScoreArgs& a, uint32_t row, float z_t, const Sums& r) {
    const float log_s = logf(r.s);
    if (a.logprob) a.logprob[row] = z_t != z_t ? NAN : log_prob(z_t, r.m, r.s, log_s, a.tau);
    a.entropy[row] = r.s == 0.0f ? 0.0f : fmaxf(log_s - kLn2 * r.u / r.s, 0.0f) + 0.0f * r.s;
    if (a.stats) a.stats[row] = make_float2(r.m, r.s);
}

// ---- rows of at most 32 E logits: one warp a row, the row in registers --------------

template <int DT, int E>
__global__ void __launch_bounds__(256) score_warp_kernel(ScoreArgs a) {
    using T = typename Elem<DT>::type;
    const int lane = threadIdx.x & 31;
    const uint32_t warps = gridDim.x * 8;
    for (uint32_t row = blockIdx.x * 8 + (threadIdx.x >> 5); row < a.N; row += warps) {
        const int64_t t = a.tok.p ? a.tok.p[row_offset(a.tok.sb, a.tok.st, a.z.T, row)] : 0;
        const T* zr = reinterpret_cast<const T*>(a.z.p) + row_offset(a.z.sb, a.z.st, a.z.T, row);
        float x[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int j = lane + 32 * e;
            x[e] = j < a.V ? to_float(zr[j]) : -INFINITY;
        }
        if (a.tok.p && t == a.tok.ignore) {
            score_padding(a, row, lane, 32);
            continue;
        }
        float best = x[0];
#pragma unroll
        for (int e = 1; e < E; ++e) best = fmaxf(best, x[e]);
        Sums r = no_sums();
        r.m = warp_max(fmaxf(best, -INFINITY));
        add_values<E, true, false>(r, x, r.m, a.c);
        r.s = warp_sum(r.s);
        r.u = warp_sum(r.u);
        if (lane == 0) score_write(a, row, a.logprob && t >= 0 && t < a.V ? to_float(zr[t]) : NAN, r);
        if (a.k == 0) continue;
        // k times the largest of the lanes' largest; what is not left is NaN, which no maximum takes
        const float log_s = logf(r.s);
        best = NAN;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            x[e] = lane + 32 * e >= a.V ? NAN : fmaxf(x[e], -INFINITY);
            best = fmaxf(best, x[e]);
        }
        float my_value = 0.0f;
        uint32_t my_index = 0;
        for (int i = 0; i < a.k; ++i) {
            const float top = warp_max(best);
            uint32_t mine = 0xffffffffu;
            if (best == top) {
#pragma unroll
                for (int e = E - 1; e >= 0; --e)
                    if (x[e] == top) mine = lane + 32 * e;
            }
            const uint32_t index = __reduce_min_sync(0xffffffffu, mine);
            if (lane == (i & 31)) my_value = top, my_index = index;
            if ((i & 31) == 31 || i == a.k - 1) {
                const int o = (i & ~31) + lane;
                if (o <= i) {
                    a.top_index[(int64_t)row * a.k + o] = my_index;
                    a.top_logprob[(int64_t)row * a.k + o] = log_prob(my_value, r.m, r.s, log_s, a.tau);
                }
            }
            if (mine == index) {
                best = NAN;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    if (lane + 32 * e == index) x[e] = NAN;
                    best = fmaxf(best, x[e]);
                }
            }
        }
    }
}

// ---- longer rows: a CTA, or a cluster of CTAs, a row --------------------------------

// entries of the list of candidates: k kept, 16 of each of k - 1 threads, k equal ones
// and 16 of a row's ends; or k and those of 16 CTAs, sorted
__host__ __device__ constexpr int top_merge(int k) {
    int n = 2;
    while (n < kMaxCluster * k) n <<= 1;
    return n;
}
__host__ __device__ constexpr int top_list(int k) {
    int n = 512;
    while (n < 18 * k + 16 || n < k + top_merge(k)) n <<= 1;
    return n;
}

// descending; n entries are in use, `list` has room up to the next power of two.  A bitonic network; up to one
// entry a thread, an entry stays in its thread's register and goes through shuffles where its partner is in the warp.
template <int kThreads>
__device__ __forceinline__ void sort_list(uint64_t* list, int n) {
    int p = 2;
    while (p < n) p <<= 1;
    const int tid = threadIdx.x;
    if (p <= kThreads) {
        if (tid < p && p <= 32) {  // one warp
            const unsigned lanes = p == 32 ? 0xffffffffu : (1u << p) - 1u;
            uint64_t x = tid < n ? list[tid] : 0;
            for (int size = 2; size <= p; size <<= 1)
                for (int d = size >> 1; d > 0; d >>= 1) {
                    const uint64_t y = __shfl_xor_sync(lanes, x, d);
                    if ((x < y) == (((tid & size) == 0) == ((tid & d) == 0))) x = y;
                }
            list[tid] = x;
        } else if (p > 32) {
            uint64_t x = tid < n ? list[tid] : 0;
            for (int size = 2; size <= p; size <<= 1)
                for (int d = size >> 1; d > 0; d >>= 1) {
                    uint64_t y;
                    if (d >= 32) {
                        __syncthreads();
                        if (tid < p) list[tid] = x;
                        __syncthreads();
                        y = tid < p ? list[tid ^ d] : x;
                    } else {
                        y = __shfl_xor_sync(0xffffffffu, x, d);
                    }
                    if ((x < y) == (((tid & size) == 0) == ((tid & d) == 0))) x = y;
                }
            __syncthreads();
            if (tid < p) list[tid] = x;
        }
        __syncthreads();
        return;
    }
    for (int i = n + tid; i < p; i += kThreads) list[i] = 0;
    __syncthreads();
    for (int size = 2; size <= p; size <<= 1)
        for (int d = size >> 1; d > 0; d >>= 1) {
            for (int i = tid; i < (p >> 1); i += kThreads) {
                const int lo = 2 * i - (i & (d - 1)), hi = lo + d;
                const uint64_t x = list[lo], y = list[hi];
                if ((x < y) == ((lo & size) == 0)) list[lo] = y, list[hi] = x;
            }
            __syncthreads();
        }
}

template <int DT, int kThreads, int kU>
struct Top {
    static constexpr int kVec = Elem<DT>::kVec, kElems = kU * kVec, kWarps = kThreads / 32;
    uint64_t* list;  // shared
    int* count;      // shared
    int* scan;       // shared, one entry a warp
    float* deposit;  // shared, two entries a warp, in turn
    int k, cap;      // cap: 16 less than the list has room for
    float bound;     // only logits above it are candidates, once `have`
    bool have;       // k logits at or above `bound`, of lower index than any to come, are listed
    int upper;       // at least *count
    int steps, due;  // of the row; where `deposit` is next made or read
    int turn;

    __device__ __forceinline__ void begin() {  // the caller's barrier follows
        have = false;
        upper = 0;
        bound = -INFINITY;
        steps = 0;
        due = 1;
        turn = 0;
        if (threadIdx.x == 0) *count = 0;
    }

    __device__ __forceinline__ void put(float z, int index) {
        list[atomicAdd(count, 1)] = ((uint64_t)order_key(z) << 32) | (uint32_t)~index;
    }

    __device__ __forceinline__ static float value(const uint4 (&r)[kU], int i) {
        const uint4& q = r[i / kVec];
        const int e = i % kVec;
        if constexpr (DT == kF32) return __uint_as_float(e == 0 ? q.x : e == 1 ? q.y : e == 2 ? q.z : q.w);
        const uint32_t w = e / 2 == 0 ? q.x : e / 2 == 1 ? q.y : e / 2 == 2 ? q.z : q.w;
        return __uint_as_float(e & 1 ? w & 0xffff0000u : w << 16);
    }

    // this thread's values above the bound
    __device__ __forceinline__ void put_above(const uint4 (&r)[kU], int first) {
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            if constexpr (DT == kBF16) {
                const __nv_bfloat162 b = __float2bfloat162_rn(bound);  // exact: a logit
                const uint32_t w[4] = {r[u].x, r[u].y, r[u].z, r[u].w};
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const uint32_t above = __hgt2_mask(*reinterpret_cast<const __nv_bfloat162*>(&w[q]), b);
                    if (above) {
                        const int at = first + u * kThreads * kVec + 2 * q;
                        if (above & 0xffffu) put(__uint_as_float(w[q] << 16), at);
                        if (above >> 16) put(__uint_as_float(w[q] & 0xffff0000u), at + 1);
                    }
                }
            } else {
#pragma unroll
                for (int e = 0; e < kVec; ++e) {
                    const float v = value(r, u * kVec + e);
                    if (v > bound) put(v, first + u * kThreads * kVec + e);
                }
            }
        }
    }

    // The row's next values: vector u of this thread, being logits first + u * kThreads * kVec + 0, 1, ..., is
    // there if bit u of `valid` is set.  cm: their maximum, all: that of all of this thread's values so far.
    __device__ __forceinline__ void add(const uint4 (&r)[kU], float cm, float all, uint32_t valid, int first) {
        const int n = __syncthreads_count(!have || cm > bound);
        ++steps;
        if (have && steps == due + 1) {  // the deposit of the step before
            const float b = deposit[turn + (threadIdx.x & (kWarps - 1))];
            bound = fmaxf(bound, -warp_max(-b));
            due *= 2;
            turn ^= kWarps;
        }
        if (n != 0) {
            if (have && upper + n * kElems <= cap) {
                upper += n * kElems;
                if (cm > bound) put_above(r, first);
            } else {
                raise(r, cm, valid, first);
            }
        }
        if (steps == due) {
            float v = all, t = -INFINITY;
            for (int j = 0; j < (k + kWarps - 1) / kWarps; ++j) {
                t = warp_max(v);
                const unsigned who = __ballot_sync(0xffffffffu, v == t);
                if ((threadIdx.x & 31) == __ffs(who) - 1) v = NAN;  // no maximum takes it again
            }
            if ((threadIdx.x & 31) == 0) deposit[turn + (threadIdx.x >> 5)] = t;
        }
    }

    __device__ __forceinline__ void raise(const uint4 (&r)[kU], float cm, uint32_t valid, int first) {
        int c = *count;
        __syncthreads();
        bool want = !have || cm > bound;
        int n = __syncthreads_count(want);
        if (c > k && c + n * kElems > cap) {
            sort_list<kThreads>(list, c);
            c = k;
            bound = fmaxf(bound, key_value((uint32_t)(list[k - 1] >> 32)));
            have = true;
            if (threadIdx.x == 0) *count = c;
            want = cm > bound;
            n = __syncthreads_count(want);
        }
        bool equal = false;
        if (!have || c + n * kElems > cap) {
            const uint32_t mine = valid ? order_key(cm) : 0u;
            uint32_t t = 0;
            // the low 16 bits of a bf16 logit's key follow from its sign
            for (int b = 31; b >= (DT == kBF16 ? 16 : 0); --b)
                if (__syncthreads_count(mine >= (t | (1u << b))) >= k) t |= 1u << b;
            if (DT == kBF16 && t && !(t & 0x80000000u)) t |= 0xffffu;
            const float f = t ? key_value(t) : -INFINITY;
            equal = !have || f > bound;
            if (equal) bound = f;
        }
        if (cm > bound) put_above(r, first);
        __syncthreads();
        if (equal) {
            int need = k - (*count - c);
            __syncthreads();
            const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                if (need <= 0) continue;
                uint32_t eq = 0;
                if (valid >> u & 1u) {
#pragma unroll
                    for (int e = 0; e < kVec; ++e) {
                        const float v = value(r, u * kVec + e);
                        eq |= (order_key(v) == order_key(bound) ? 1u : 0u) << e;
                    }
                }
                int at = __popc(eq);
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int y = __shfl_up_sync(0xffffffffu, at, o);
                    if (lane >= o) at += y;
                }
                if (lane == 31) scan[warp] = at;
                __syncthreads();
                int before = 0, total = 0;
                for (int w = 0; w < kWarps; ++w) {
                    const int y = scan[w];
                    before += w < warp ? y : 0;
                    total += y;
                }
                int rank = before + at - __popc(eq);
                for (; eq && rank < need; eq &= eq - 1, ++rank)
                    put(bound, first + u * kThreads * kVec + __ffs(eq) - 1);
                need -= total;
                __syncthreads();
            }
        }
        upper = *count;
        __syncthreads();
        have = upper >= k;
    }

    // a logit of the row's ends, after all others: of lower index than all of them, or of higher
    __device__ __forceinline__ void add_end(float z, int index, bool lower) {
        const float v = z != z ? -INFINITY : z;
        if (!have || v > bound || (lower && v == bound)) put(v, index);
    }

    // list[0 .. k - 1]: the largest, sorted; 0 where the part of the row has fewer
    __device__ __forceinline__ void finish() {
        __syncthreads();
        const int c = *count;
        sort_list<kThreads>(list, c);
        if (c < k) {
            int p = 2;
            while (p < c) p <<= 1;
            for (int i = p + threadIdx.x; i < k; i += kThreads) list[i] = 0;
            __syncthreads();
        }
    }
};

// steps that are loaded ahead, for 16 KB of them a CTA of 512 threads
template <bool TOP>
constexpr int kScoreStages = TOP ? 4 : 6;

template <int DT, int kThreads, bool TOP>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) score_row_kernel(ScoreArgs a, uint32_t lg) {
    using T = typename Elem<DT>::type;
    using Stream = RowStream<DT, kThreads, 1, kScoreStages<TOP>>;
    constexpr int kVec = Elem<DT>::kVec, kU = Stream::kU, kElems = Stream::kElems, kWarps = kThreads / 32;
    extern __shared__ __align__(16) unsigned char sm[];  // the stream's places, the list
    __shared__ float4 part[2][kWarps], mine[2];
    __shared__ int count, scan[kWarps];
    __shared__ float deposit[2 * kWarps];
    const int tid = threadIdx.x;
    const uint32_t ctas = 1u << lg, rank = blockIdx.x & (ctas - 1);
    Top<DT, kThreads, kU> top;
    top.list = reinterpret_cast<uint64_t*>(sm + Stream::kBytes);
    top.count = &count, top.scan = scan, top.deposit = deposit, top.k = a.k, top.cap = top_list(a.k) - 16;
    const RowList list(a.tok, a.z.T, a.N, blockIdx.x >> lg, gridDim.x >> lg);
    const RowStep step(a.z, gridDim.x >> lg);
    Stream stream(a.z, a.V, list, step, rank, lg, sm);
    RowAt at(a.z, list.first);
    uint32_t live = 0;
    int parity = 0;
    for (uint32_t i = 0; i < list.count; ++i, step.move(at, a.z.T)) {
        if ((i & 31) == 0) live = list.window(i);
        const uint32_t row = list.row(i);
        if (!(live >> (i & 31) & 1u)) {
            if (rank == 0) score_padding(a, row, tid, kThreads);
            continue;
        }
        const T* zr = reinterpret_cast<const T*>(a.z.p) + at.off;
        const Segment g = segment_of<DT>(zr, a.V, rank, lg);
        const int ends = g.head + g.tail, end_at = tid < g.head ? tid : g.t0 + tid - g.head;
        const float end = tid < ends ? to_float(zr[end_at]) : -INFINITY;
        int64_t t = 0;
        float z_t = 0.0f;
        if (tid == 0 && a.logprob) {
            t = a.tok.p[row_offset(a.tok.sb, a.tok.st, a.z.T, row)];
            z_t = t >= 0 && t < a.V ? to_float(zr[t]) : NAN;
        }
        if constexpr (TOP) {
            top.begin();
            __syncthreads();
        }
        Sums r = no_sums();
        for (int v = g.v0; v < g.v1; v += Stream::kStep) {
            uint4 raw[kU];
            stream.take(raw, v, g.v1);
            float x[kElems];
#pragma unroll
            for (int u = 0; u < kU; ++u) unpack16<DT>(raw[u], x + u * kVec);
            const float cm = max_of<DT>(raw);
            stream.issue();
            add_values<kElems, true, false>(r, x, cm, a.c);
            if constexpr (TOP) {
                uint32_t valid = 0;
#pragma unroll
                for (int u = 0; u < kU; ++u) valid |= (v + tid + u * kThreads < g.v1 ? 1u : 0u) << u;
                top.add(raw, cm, r.m, valid, g.h0 + (v + tid) * kVec);
            }
        }
        if (tid < ends) {
            const float x[1] = {end};
            add_values<1, true, false>(r, x, end, a.c);
            if constexpr (TOP) top.add_end(end, end_at, tid < g.head);
        }
        r = cta_join<kThreads, true, false>(r, part[parity], a.c);
        if (ctas > 1) r = cluster_join<true, false>(r, &mine[parity], ctas, a.c);
        parity ^= 1;
        if (rank == 0 && tid == 0) score_write(a, row, z_t, r);
        if constexpr (TOP) {
            top.finish();
            uint64_t* best = top.list;
            if (ctas > 1) {
                cluster_sync();
                if (rank == 0) {
                    best = top.list + a.k;
                    for (int n = tid; n < (int)ctas * a.k; n += kThreads)
                        best[n] = ld_dsmem_u64(map_to_rank(smem_addr(top.list + n % a.k), n / a.k));
                }
                cluster_sync();
                if (rank == 0) sort_list<kThreads>(best, (int)ctas * a.k);
            }
            if (rank == 0 && tid < a.k) {
                const float log_s = logf(r.s);
                a.top_index[(int64_t)row * a.k + tid] = (uint32_t)~best[tid];
                a.top_logprob[(int64_t)row * a.k + tid] =
                    log_prob(key_value((uint32_t)(best[tid] >> 32)), r.m, r.s, log_s, a.tau);
            }
            __syncthreads();
        }
    }
    if (ctas > 1) cluster_sync();  // no CTA ends while another may still read its shared memory
}

// ---- gradient -----------------------------------------------------------------------

struct ScoreGradArgs {
    RowsIn z;
    Tokens tok;
    RowsOut d;
    uint32_t N;
    int V, k;
    float tau, c;
    const float2* stats;
    const float* entropy;
    const int64_t* top_index;
    const float* g_logprob;  // [N] or null
    const float* g_entropy;  // [N] or null
    const float* g_top;      // [N, k] or null
};

struct ScoreGrad {  // of one row
    float h, inv_s, log_s, H, g, gh, all, inv_tau, c;
    __device__ __forceinline__ float at(float z) const {
        const float d = exponent(z, h, c);
        const float p = exp2_approx(d) * inv_s;
        return -p * (all + gh * (fmaf(d, kLn2, -log_s) + H));
    }
};

// a warp reads what a row's gradient needs; every lane gets it.  t: the token or -1
__device__ __forceinline__ ScoreGrad score_grad_row(const ScoreGradArgs& a, uint32_t row, int64_t t) {
    ScoreGrad r;
    const float2 st = a.stats[row];
    r.h = shift_of(st.x);
    r.inv_s = st.y == 0.0f ? 0.0f : 1.0f / st.y;
    r.log_s = st.y == 0.0f ? 0.0f : logf(st.y);
    r.H = a.entropy[row];
    r.gh = a.g_entropy ? a.g_entropy[row] : 0.0f;
    r.g = a.g_logprob ? a.g_logprob[row] : 0.0f;
    if (a.g_logprob && (t < 0 || t >= a.V)) r.g = NAN;
    float sum = 0.0f;
    if (a.g_top)
        for (int i = threadIdx.x & 31; i < a.k; i += 32) sum += a.g_top[(int64_t)row * a.k + i];
    r.all = r.g + warp_sum(sum);
    r.inv_tau = 1.0f / a.tau;
    r.c = a.c;
    return r;
}

// the given token and the alternatives, in logits j0 .. j1 - 1 of the row, after their plain
// gradient was written; thread tid of `threads`
template <class T>
__device__ __forceinline__ void score_grad_slots(const ScoreGradArgs& a, const ScoreGrad& r, uint32_t row, int64_t t,
                                                 const T* zr, T* dr, int j0, int j1, int tid, int threads) {
    const int slots = a.g_top ? a.k : 0;
    const int64_t* idx = a.top_index + (int64_t)row * a.k;
    for (int i = tid; i <= slots; i += threads) {
        if (i == slots && !a.g_logprob) break;
        const int64_t j = i < slots ? idx[i] : t;
        if (j < j0 || j >= j1) continue;
        float add;
        if (i < slots) {
            add = a.g_top[(int64_t)row * a.k + i] + (a.g_logprob && j == t ? r.g : 0.0f);
        } else {
            bool listed = false;  // then that alternative's thread has added it
            for (int q = 0; q < slots; ++q) listed |= idx[q] == t;
            if (listed) continue;
            add = r.g;
        }
        dr[j] = from_float<T>((r.at(to_float(zr[j])) + add) * r.inv_tau);
    }
}

template <int DT, int E>
__global__ void __launch_bounds__(256) score_grad_warp_kernel(ScoreGradArgs a) {
    using T = typename Elem<DT>::type;
    const int lane = threadIdx.x & 31;
    const uint32_t warps = gridDim.x * 8;
    for (uint32_t row = blockIdx.x * 8 + (threadIdx.x >> 5); row < a.N; row += warps) {
        const int64_t t = a.tok.p ? a.tok.p[row_offset(a.tok.sb, a.tok.st, a.z.T, row)] : -1;
        T* dr = reinterpret_cast<T*>(a.d.p) + row_offset(a.d.sb, a.d.st, a.d.T, row);
        if (a.tok.p && t == a.tok.ignore) {
            for (int j = lane; j < a.V; j += 32) dr[j] = from_float<T>(0.0f);
            continue;
        }
        const T* zr = reinterpret_cast<const T*>(a.z.p) + row_offset(a.z.sb, a.z.st, a.z.T, row);
        const ScoreGrad r = score_grad_row(a, row, t);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int j = lane + 32 * e;
            if (j < a.V) dr[j] = from_float<T>(r.at(to_float(zr[j])) * r.inv_tau);
        }
        __syncwarp();
        score_grad_slots<T>(a, r, row, t, zr, dr, 0, a.V, lane, 32);
    }
}

constexpr int kGradThreads = 512;

// CTA `part` of 2^lg of a row
template <int DT>
__global__ void __launch_bounds__(kGradThreads, 2) score_grad_row_kernel(ScoreGradArgs a, uint32_t lg) {
    using T = typename Elem<DT>::type;
    constexpr int kVec = Elem<DT>::kVec;
    const int tid = threadIdx.x;
    const uint32_t row = blockIdx.x >> lg;
    const int64_t t = a.tok.p ? a.tok.p[row_offset(a.tok.sb, a.tok.st, a.z.T, row)] : -1;
    const T* zr = reinterpret_cast<const T*>(a.z.p) + row_offset(a.z.sb, a.z.st, a.z.T, row);
    T* dr = reinterpret_cast<T*>(a.d.p) + row_offset(a.d.sb, a.d.st, a.d.T, row);
    const Segment g = segment_of<DT>(zr, a.V, blockIdx.x & ((1u << lg) - 1u), lg);
    const bool live = !(a.tok.p && t == a.tok.ignore);
    const bool wide = (((uintptr_t)zr ^ (uintptr_t)dr) & 15u) == 0;  // 16-byte stores
    ScoreGrad r;
    if (live) r = score_grad_row(a, row, t);
    const uint4* body = reinterpret_cast<const uint4*>(zr + g.h0);
    for (int v = g.v0 + tid; v < g.v1; v += kGradThreads) {
        float y[kVec];
        if (live) {
            float x[kVec];
            unpack16<DT>(__ldcs(body + v), x);
#pragma unroll
            for (int e = 0; e < kVec; ++e) y[e] = r.at(x[e]) * r.inv_tau;
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
    if (tid < g.head) dr[tid] = from_float<T>(live ? r.at(to_float(zr[tid])) * r.inv_tau : 0.0f);
    if (tid < g.tail) dr[g.t0 + tid] = from_float<T>(live ? r.at(to_float(zr[g.t0 + tid])) * r.inv_tau : 0.0f);
    if (!live) return;
    __syncthreads();
    score_grad_slots<T>(a, r, row, t, zr, dr, g.j0, g.j1, tid, kGradThreads);
}

}  // namespace il
