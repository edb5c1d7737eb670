// il_score.cuh -- log probabilities of given tokens, entropy and the largest
// alternatives of logits rows, and the gradient of all three.
//
//   lse = m / tau + ln s           logprob_t = (z_t - m) / tau - ln s
//   H = ln s - ln(2) u / s         top: the k largest logits, equal ones by index
//   dz_j = 1/tau ( [j = t] g + sum_i [j = idx_i] g_i - p_j (g + sum_i g_i + g_H (ln p_j + H)) )
// with (m, s, u) of il_logits.cuh.  The forward reads each logit once, the
// backward reads it once more and writes its gradient.
//
// The k largest in the same pass.  Every thread knows the maximum of the 16
// logits that it holds.  For the row's first logits the k-th largest of the
// threads' maxima is a lower bound of the k-th largest logit; from then on only
// logits above the bound are put into a list in shared memory (for logits in no
// particular order a few times k of them), so that the work on a logit that is
// not among the largest is the comparison of its thread's maximum.  When the
// list could run over, it is sorted and cut to k, and the bound rises to its
// last; when one step alone could overrun it, the bound is first taken from the
// threads' maxima again: at most (k - 1) threads then hold anything above it,
// and of the logits equal to it the first ones by index are taken.  No input
// needs a second pass.  List entries are (order-preserving bits of z) << 32 |
// ~index, so that all are distinct and equal logits go by their index.
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

// descending; n entries are in use, `list` has room up to the next power of two
__device__ __forceinline__ void sort_list(uint64_t* list, int n) {
    int p = 2;
    while (p < n) p <<= 1;
    for (int i = n + threadIdx.x; i < p; i += kRowThreads) list[i] = 0;
    __syncthreads();
    for (int size = 2; size <= p; size <<= 1)
        for (int d = size >> 1; d > 0; d >>= 1) {
            for (int i = threadIdx.x; i < (p >> 1); i += kRowThreads) {
                const int lo = 2 * i - (i & (d - 1)), hi = lo + d;
                const uint64_t x = list[lo], y = list[hi];
                if ((x < y) == ((lo & size) == 0)) list[lo] = y, list[hi] = x;
            }
            __syncthreads();
        }
}

struct Top {
    uint64_t* list;  // shared
    int* count;      // shared
    int* scan;       // shared, one entry a warp
    int k, cap;      // cap: 16 less than the list has room for
    float bound;     // only logits above it are candidates, once `have`
    bool have;       // k logits at or above `bound`, of lower index than any to come, are listed
    int upper;       // at least *count

    __device__ __forceinline__ void begin() {  // the caller's barrier follows
        have = false;
        upper = 0;
        bound = -INFINITY;
        if (threadIdx.x == 0) *count = 0;
    }

    __device__ __forceinline__ void put(float z, int index) {
        list[atomicAdd(count, 1)] = ((uint64_t)order_key(z) << 32) | (uint32_t)~index;
    }

    // kU x kV values of this thread, x[u * kV + e] being logit first + u * step + e; valid: bits of u
    template <int kU, int kV>
    __device__ __forceinline__ void add(const float (&x)[kU * kV], float cm, uint32_t valid, int first, int step) {
        bool want = !have || cm > bound;
        int n = __syncthreads_count(want);
        if (n == 0) return;
        if (have && upper + n * (kU * kV) <= cap) {
            upper += n * (kU * kV);
            if (want) {
#pragma unroll
                for (int i = 0; i < kU * kV; ++i)
                    if (x[i] > bound) put(x[i], first + (i / kV) * step + i % kV);
            }
            return;
        }
        raise<kU, kV>(x, cm, valid, first, step);
    }

    template <int kU, int kV>
    __device__ __forceinline__ void raise(const float (&x)[kU * kV], float cm, uint32_t valid, int first, int step) {
        int c = *count;
        if (c > k) {
            sort_list(list, c);
            c = k;
            bound = key_value((uint32_t)(list[k - 1] >> 32));
            have = true;
        }
        __syncthreads();
        if (threadIdx.x == 0) *count = c;
        const bool want = !have || cm > bound;
        const int n = __syncthreads_count(want);
        bool equal = false;
        if (!have || c + n * (kU * kV) > cap) {
            const uint32_t mine = valid ? order_key(cm) : 0u;
            uint32_t t = 0;
            for (int b = 31; b >= 0; --b)
                if (__syncthreads_count(mine >= (t | (1u << b))) >= k) t |= 1u << b;
            const float f = t ? key_value(t) : -INFINITY;
            equal = !have || f > bound;
            if (equal) bound = f;
        }
#pragma unroll
        for (int i = 0; i < kU * kV; ++i)
            if (x[i] > bound) put(x[i], first + (i / kV) * step + i % kV);
        __syncthreads();
        if (equal) {
            int need = k - (*count - c);
            __syncthreads();
            const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                if (need <= 0) continue;
                int eq = 0;
#pragma unroll
                for (int e = 0; e < kV; ++e) {
                    const float v = x[u * kV + e];
                    eq += (valid >> u & 1u) && !(v > bound) && order_key(v) == order_key(bound);
                }
                int at = eq;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int y = __shfl_up_sync(0xffffffffu, at, o);
                    if (lane >= o) at += y;
                }
                if (lane == 31) scan[warp] = at;
                __syncthreads();
                int before = 0, total = 0;
                for (int w = 0; w < kRowThreads / 32; ++w) {
                    const int y = scan[w];
                    before += w < warp ? y : 0;
                    total += y;
                }
                int rank = before + at - eq;
#pragma unroll
                for (int e = 0; e < kV; ++e) {
                    const float v = x[u * kV + e];
                    if ((valid >> u & 1u) && !(v > bound) && order_key(v) == order_key(bound)) {
                        if (rank < need) put(v, first + u * step + e);
                        ++rank;
                    }
                }
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
        sort_list(list, c);
        if (c < k) {
            int p = 2;
            while (p < c) p <<= 1;
            for (int i = p + threadIdx.x; i < k; i += kRowThreads) list[i] = 0;
            __syncthreads();
        }
    }
};

template <bool TOP>
constexpr int kScoreStages = TOP ? 4 : 6;

template <int DT, bool TOP>
__global__ void __launch_bounds__(kRowThreads, 2) score_row_kernel(ScoreArgs a, uint32_t ctas) {
    using T = typename Elem<DT>::type;
    using Stream = RowStream<DT, 1, kScoreStages<TOP>>;
    constexpr int kVec = Elem<DT>::kVec, kU = Stream::kU, kElems = Stream::kElems;
    extern __shared__ __align__(16) unsigned char sm[];  // the stream's places, the list
    __shared__ float4 part[2][kRowWarps], mine[2];
    __shared__ int count, scan[kRowWarps];
    const int tid = threadIdx.x;
    const uint32_t rank = blockIdx.x % ctas;
    Top top;
    top.list = reinterpret_cast<uint64_t*>(sm + Stream::kBytes);
    top.count = &count, top.scan = scan, top.k = a.k, top.cap = top_list(a.k) - 16;
    RowList list(a.tok, a.z.T, a.N, blockIdx.x / ctas, gridDim.x / ctas);
    Stream stream(a.z, a.V, list, rank, ctas, sm);
    int parity = 0;
    for (uint32_t i = 0; i < list.count; ++i) {
        if ((i & 31) == 0) list.window(i);
        const uint32_t row = list.row(i);
        if (!list.live(i)) {
            if (rank == 0) score_padding(a, row, tid, kRowThreads);
            continue;
        }
        const T* zr = reinterpret_cast<const T*>(a.z.p) + row_offset(a.z.sb, a.z.st, a.z.T, row);
        const Segment g = segment_of<DT>(zr, a.V, rank, ctas);
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
            uint32_t valid = 0;
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                unpack16<DT>(raw[u], x + u * kVec);
                valid |= (v + tid + u * kRowThreads < g.v1 ? 1u : 0u) << u;
            }
            stream.issue();
            float cm = x[0];
#pragma unroll
            for (int e = 1; e < kElems; ++e) cm = fmaxf(cm, x[e]);
            cm = fmaxf(cm, -INFINITY);  // all NaN
            add_values<kElems, true, false>(r, x, cm, a.c);
            if constexpr (TOP)
                top.template add<kU, kVec>(x, cm, valid, g.h0 + (v + tid) * kVec, kRowThreads * kVec);
        }
        if (tid < ends) {
            const float x[1] = {end};
            add_values<1, true, false>(r, x, end, a.c);
            if constexpr (TOP) top.add_end(end, end_at, tid < g.head);
        }
        r = cta_join<true, false>(r, part[parity], a.c);
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
                    for (int n = tid; n < (int)ctas * a.k; n += kRowThreads)
                        best[n] = ld_dsmem_u64(map_to_rank(smem_addr(top.list + n % a.k), n / a.k));
                }
                cluster_sync();
                if (rank == 0) sort_list(best, (int)ctas * a.k);
            }
            if (rank == 0) {
                const float log_s = logf(r.s);
                for (int n = tid; n < a.k; n += kRowThreads) {
                    a.top_index[(int64_t)row * a.k + n] = (uint32_t)~best[n];
                    a.top_logprob[(int64_t)row * a.k + n] =
                        log_prob(key_value((uint32_t)(best[n] >> 32)), r.m, r.s, log_s, a.tau);
                }
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

template <int DT>
__global__ void __launch_bounds__(kRowThreads, 2) score_grad_row_kernel(ScoreGradArgs a, uint32_t parts) {
    using T = typename Elem<DT>::type;
    constexpr int kVec = Elem<DT>::kVec;
    const int tid = threadIdx.x;
    const uint32_t row = blockIdx.x / parts;
    const int64_t t = a.tok.p ? a.tok.p[row_offset(a.tok.sb, a.tok.st, a.z.T, row)] : -1;
    const T* zr = reinterpret_cast<const T*>(a.z.p) + row_offset(a.z.sb, a.z.st, a.z.T, row);
    T* dr = reinterpret_cast<T*>(a.d.p) + row_offset(a.d.sb, a.d.st, a.d.T, row);
    const Segment g = segment_of<DT>(zr, a.V, blockIdx.x - row * parts, parts);
    const bool live = !(a.tok.p && t == a.tok.ignore);
    const bool wide = (((uintptr_t)zr ^ (uintptr_t)dr) & 15u) == 0;  // 16-byte stores
    ScoreGrad r;
    if (live) r = score_grad_row(a, row, t);
    const uint4* body = reinterpret_cast<const uint4*>(zr + g.h0);
    for (int v = g.v0 + tid; v < g.v1; v += kRowThreads) {
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
    score_grad_slots<T>(a, r, row, t, zr, dr, g.j0, g.j1, tid, kRowThreads);
}

}  // namespace il
