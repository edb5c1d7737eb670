// il_score.cuh -- log probabilities of given tokens, entropy and the largest
// alternatives of logits rows, and the gradient of all three.
//
//   lse = m / tau + ln s           logprob_t = (z_t - m) / tau - ln s
//   H = ln s - ln(2) u / s         top: the k largest logits, equal ones by index
//   dz_j = 1/tau ( [j = t] g + sum_i [j = idx_i] g_i - p_j (g + sum_i g_i + g_H (ln p_j + H)) )
// with (m, s, u) of il_logits.cuh.  The forward reads each logit once, the
// backward reads it once more and writes its gradient.
//
// The k largest.  While a row goes by, each thread keeps the maximum of every
// sixteenth (an eighth to a 64th) of what it reads, rounded up to 16 bits, and
// nothing else is done for them.  Then, with W warps and j = k / W rounded up,
// the least of the warps' j-th largest thread maxima is a bound that at least k
// logits reach, and of a row in no particular order not many more; the few
// of these that reach it are read again, and their logits that reach it are
// ranked.  Entries are (order-preserving bits of z) << 32 | ~index, so that all
// are distinct and equal logits go by their index.  Where more logits reach the
// bound than the list holds, the k-th largest of those listed is a higher bound
// for another round; where that is no higher, the list is of the logits above
// the bound, and of those equal to it the first by index fill it up to k.
// 4096 x 131072 bf16, 64 alternatives: 260 us, 174 us of them the sums'; a list
// that every logit above a running bound was put into, with a barrier a step,
// took 614 us, and reading eighths again instead of thirty-seconds 287 us.
//
// 8192 x 65536 bf16 with the gradient of log probability and entropy, a fifth
// of the rows padding (not read): forward 178 us (0.86 GB, 131 us at the
// measured copy rate), backward 310 us (1.93 GB, 296 us).  Without padding 190
// us (164) and 355 us (328).
#pragma once
#include <type_traits>

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
        const int64_t t = a.tok.p ? a.tok.p[row_offset(a.tok.sb, a.tok.st, a.tok.T, row)] : 0;
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
        // k times the largest of the lanes' largest; keys are 0 where nothing is left
        const float log_s = logf(r.s);
        uint32_t key[E], most = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            key[e] = lane + 32 * e < a.V ? order_key(x[e]) : 0u;
            most = max(most, key[e]);
        }
        uint32_t my_key = 0, my_index = 0;
        for (int i = 0; i < a.k; ++i) {
            const uint32_t top = __reduce_max_sync(0xffffffffu, most);
            uint32_t mine = 0xffffffffu;
            if (most == top) {
#pragma unroll
                for (int e = E - 1; e >= 0; --e)
                    if (key[e] == top) mine = lane + 32 * e;
            }
            const uint32_t index = __reduce_min_sync(0xffffffffu, mine);
            if (lane == (i & 31)) my_key = top, my_index = index;
            if ((i & 31) == 31 || i == a.k - 1) {
                const int o = (i & ~31) + lane;
                if (o <= i) {
                    a.top_index[(int64_t)row * a.k + o] = my_index;
                    a.top_logprob[(int64_t)row * a.k + o] = log_prob(key_value(my_key), r.m, r.s, log_s, a.tau);
                }
            }
            if (mine == index) {
                most = 0;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    if (lane + 32 * e == index) key[e] = 0;
                    most = max(most, key[e]);
                }
            }
        }
    }
}

// ---- longer rows: a CTA, or a cluster of CTAs, a row --------------------------------

// entries of the list of candidates: some times k; in a cluster also the k of each of 2^lg CTAs
__host__ __device__ constexpr int top_list(int k, int lg) {
    int n = 512;
    while (lg && n < k << lg) n <<= 1;
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

// 16 bits of a float, not below it
__device__ __forceinline__ uint16_t upper16(float v) {
    const uint32_t b = __float_as_uint(v);
    const uint32_t up = (int32_t)b >= 0 ? b + 0xffffu : b;  // away from, or towards zero
    return (uint16_t)((v == INFINITY ? b : up) >> 16);
}

// Sends every entry of list[0 .. n - 1] (all distinct) whose rank is below k to out(rank, entry): each is compared
// with all, which for a few hundred entries takes no barrier and less time than sorting them.
template <int kThreads, class Out>
__device__ __forceinline__ void rank_list(const uint64_t* list, int n, int k, Out out) {
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const uint64_t x = list[i];
        int rank = 0;
#pragma unroll 4
        for (int m = 0; m < n; ++m) rank += list[m] > x;
        if (rank < k) out(rank, x);
    }
}

// the j-th largest of the lanes' values (j: 1 .. 32)
__device__ __forceinline__ float warp_largest(float v, int j) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int d = size >> 1; d > 0; d >>= 1) {
            const float y = __shfl_xor_sync(0xffffffffu, v, d);
            v = ((lane & size) == 0) == ((lane & d) == 0) ? fmaxf(v, y) : fminf(v, y);
        }
    return __shfl_sync(0xffffffffu, v, j - 1);
}

template <int DT, int kThreads, int kU>
struct Top {
    static constexpr int kVec = Elem<DT>::kVec, kWarps = kThreads / 32, kStep = kU * kThreads;
    static constexpr int kGroups = 4096 / kThreads;  // of steps, that a row's steps are put into
    static constexpr int kHits = 128;                // that a warp reads again at a time
    struct Shared {
        uint16_t most[kGroups][kThreads];       // maxima of the groups
        uint16_t hits[kWarps][kHits];
        float deposit[2][kWarps];
        int scan[kWarps];
        int count;
    };
    using T = typename Elem<DT>::type;
    Shared* sh;
    uint64_t* list;  // shared, room for cap entries and for k
    int k, cap;

    // the least of the warps' j-th largest of their lanes' values is left by two calls with a barrier between
    __device__ __forceinline__ void offer(float all, int parity) const {
        const float t = warp_largest(all, (k + kWarps - 1) / kWarps);
        if ((threadIdx.x & 31) == 0) sh->deposit[parity][threadIdx.x >> 5] = t;
    }
    __device__ __forceinline__ float bound(int parity) const {
        return -warp_max(-sh->deposit[parity][threadIdx.x & (kWarps - 1)]);
    }

    __device__ __forceinline__ void put(float z, int index) const {
        const int at = (int)atom_add_shared_u32(smem_addr(&sh->count), 1u);
        if (at < cap) list[at] = ((uint64_t)order_key(z) << 32) | (uint32_t)~index;
    }
    __device__ __forceinline__ static bool reaches(float z, float bound, bool above) {
        return above ? z > bound : z >= bound;  // not NaN
    }

    // lists what reaches the bound in n groups of this warp
    __device__ __forceinline__ void reread(const uint4* body, const Segment& g, const uint16_t* hits, int n, int lg,
                                           float bound, bool above) const {
        // vector q of hit h is item (h << per) + q; four items of a lane are loaded at a time
        static_assert(kU == 4, "a step of a group is 4 vectors");
        const int per = 2 + lg, items = n << per;
        for (int i = threadIdx.x & 31; i < items; i += 4 * 32) {
            uint4 r[4];
            int v[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const int item = i + w * 32;
                v[w] = -1;
                if (item < items) {
                    const int h = hits[item >> per], q = item & ((1 << per) - 1);
                    const int at = g.v0 + ((h / kThreads << lg) + q / kU) * kStep + q % kU * kThreads + h % kThreads;
                    if (at < g.v1) {
                        v[w] = at;
                        r[w] = __ldg(body + at);
                    }
                }
            }
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                if (v[w] < 0) continue;
                const uint4 one[1] = {r[w]};
                if (!reaches(max_of<DT>(one), bound, above)) continue;
                float x[kVec];
                unpack16<DT>(r[w], x);
#pragma unroll
                for (int e = 0; e < kVec; ++e)
                    if (reaches(x[e], bound, above)) put(x[e], g.h0 + v[w] * kVec + e);
            }
        }
    }

    // Lists the part's logits that reach the bound (above: that are above it), sh->count of them; false: more than
    // the list holds.  sh->count is 0.  lg: log2 of the steps of a group; end, end_at, ends: this thread's logit of
    // the row's ends.
    __device__ __forceinline__ bool collect(const T* zr, const Segment& g, int lg, float end, int end_at, int ends,
                                            float bound, bool above) const {
        const int tid = threadIdx.x, lane = tid & 31;
        const uint4* body = reinterpret_cast<const uint4*>(zr + g.h0);
        const int groups = (g.v1 - g.v0 + (kStep << lg) - 1) / (kStep << lg);
        uint16_t* hits = sh->hits[tid >> 5];  // of this warp
        if (tid < ends && reaches(end, bound, above)) put(end, end_at);
        int n = 0;
        for (int i = 0; i < groups; ++i) {
            const bool hit = reaches(__uint_as_float((uint32_t)sh->most[i][tid] << 16), bound, above);
            const unsigned who = __ballot_sync(0xffffffffu, hit);
            if (hit) hits[n + __popc(who & ((1u << lane) - 1u))] = (uint16_t)(i * kThreads + tid);
            n += __popc(who);
            if (n > kHits - 32 || i == groups - 1) {
                __syncwarp();
                reread(body, g, hits, n, lg, bound, above);
                __syncwarp();
                n = 0;
            }
        }
        __syncthreads();
        return sh->count <= cap;
    }

    // the first `need` logits by index that equal the bound (-inf: NaN too)
    __device__ __forceinline__ void fill(const T* zr, const Segment& g, float bound, int need) const {
        const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
        const uint4* body = reinterpret_cast<const uint4*>(zr + g.h0);
        auto equal = [&](float z) { return z == bound || (z != z && bound == -INFINITY); };
        for (int j = 0; j < g.head; ++j)
            if (need > 0 && equal(to_float(zr[j]))) {
                if (tid == 0) put(bound, j);
                --need;
            }
        for (int v = g.v0; need > 0 && v < g.v1; v += kThreads) {
            uint32_t eq = 0;
            if (v + tid < g.v1) {
                float x[kVec];
                unpack16<DT>(__ldg(body + v + tid), x);
#pragma unroll
                for (int e = 0; e < kVec; ++e) eq |= (equal(x[e]) ? 1u : 0u) << e;
            }
            int at = __popc(eq);
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, at, o);
                if (lane >= o) at += y;
            }
            if (lane == 31) sh->scan[warp] = at;
            __syncthreads();
            int before = 0, total = 0;
            for (int w = 0; w < kWarps; ++w) {
                const int y = sh->scan[w];
                before += w < warp ? y : 0;
                total += y;
            }
            int rank = before + at - __popc(eq);
            for (; eq && rank < need; eq &= eq - 1, ++rank) put(bound, g.h0 + (v + tid) * kVec + __ffs(eq) - 1);
            need -= total;
            __syncthreads();
        }
        for (int j = g.t0; j < g.t0 + g.tail; ++j)
            if (need > 0 && equal(to_float(zr[j]))) {
                if (tid == 0) put(bound, j);
                --need;
            }
        __syncthreads();
    }

    // list[0 .. result - 1] has the k largest of the part among few others; all of the part where it has fewer than k
    __device__ __forceinline__ int find(const T* zr, const Segment& g, int lg, float end, int end_at, int ends,
                                        float bound) const {
        bool above = bound == -INFINITY;
        while (!collect(zr, g, lg, end, end_at, ends, bound, above)) {
            sort_list<kThreads>(list, cap);
            const float b = key_value((uint32_t)(list[k - 1] >> 32));
            above = !(b > bound);
            bound = b;
            __syncthreads();
            if (threadIdx.x == 0) sh->count = 0;
            __syncthreads();
        }
        if (above && sh->count < k) {
            const int need = k - sh->count;
            __syncthreads();
            fill(zr, g, bound, need);
        }
        return sh->count;
    }
};

template <int DT, int kThreads, bool TOP>
__global__ void __launch_bounds__(kThreads, sm_threads(1) / kThreads) score_row_kernel(ScoreArgs a, uint32_t lg) {
    using T = typename Elem<DT>::type;
    using Stream = RowStream<DT, kThreads, 1>;
    constexpr int kU = Stream::kU, kWarps = kThreads / 32;
    using TopOf = Top<DT, kThreads, kU>;
    extern __shared__ __align__(16) unsigned char sm[];  // the stream's places, the list
    __shared__ float4 part[2][kWarps], mine[2];
    __shared__ typename std::conditional<TOP, typename TopOf::Shared, int>::type top_shared;
    const int tid = threadIdx.x;
    const uint32_t ctas = 1u << lg, rank = blockIdx.x & (ctas - 1);
    TopOf top;
    if constexpr (TOP)
        top.sh = &top_shared, top.list = reinterpret_cast<uint64_t*>(sm + Stream::kBytes), top.k = a.k,
        top.cap = top_list(a.k, lg);
    const RowList list(a.tok, a.N, blockIdx.x >> lg, gridDim.x >> lg);
    const RowStep step(a.z, gridDim.x >> lg);
    Stream stream(a.z, a.V, list, step, rank, lg, sm);
    if constexpr (TOP) {
        if (tid == 0) top_shared.count = 0;
    }
    int parity = 0;
    if (rank == 0 && a.tok.p) {
        uint32_t live = 0;
        for (uint32_t i = 0; i < list.count; ++i) {
            if ((i & 31) == 0) live = list.window(i);
            if (!(live >> (i & 31) & 1u)) score_padding(a, list.row(i), tid, kThreads);
        }
    }
    for (LiveRows at(a.z, list, step); at.valid(); at.next()) {
        const uint32_t row = at.row();
        const T* zr = reinterpret_cast<const T*>(a.z.p) + at.at.off;
        const Segment g = segment_of<DT>(zr, a.V, rank, lg);
        const int ends = g.head + g.tail, end_at = tid < g.head ? tid : g.t0 + tid - g.head;
        const float end = tid < ends ? to_float(zr[end_at]) : -INFINITY;
        float z_t = 0.0f;
        if (tid == kThreads - 1 && a.logprob) {
            const int64_t t = a.tok.p[row_offset(a.tok.sb, a.tok.st, a.tok.T, row)];
            z_t = t >= 0 && t < a.V ? to_float(zr[t]) : NAN;
        }
        int group_lg = 0;  // kGroups groups of 2^group_lg steps are enough
        if constexpr (TOP)
            while ((Stream::kStep * TopOf::kGroups << group_lg) < g.v1 - g.v0) ++group_lg;
        Running<true, false> run;
        run.begin(a.c);
        float most = -INFINITY;
        int n = 0;
        auto use = [&](const uint4 (&raw)[kU], bool last) {
            const float cm = max_of<DT>(raw);
            run.template add<DT>(raw, cm, a.c);
            if constexpr (TOP) {
                most = fmaxf(most, cm);
                ++n;
                if ((n & ((1 << group_lg) - 1)) == 0 || last) {
                    top_shared.most[(n - 1) >> group_lg][tid] = upper16(most);
                    most = -INFINITY;
                }
            }
        };
        int left = g.v1 - g.v0;
        for (; left >= Stream::kStep; left -= Stream::kStep) {
            uint4 raw[kU];
            stream.template take<true>(raw, 0);
            stream.issue();
            use(raw, left == Stream::kStep);
        }
        if (left > 0) {
            uint4 raw[kU];
            stream.template take<false>(raw, (left - tid + kThreads - 1) / kThreads);
            stream.issue();
            use(raw, true);
        }
        Sums r = run.sums(a.c);
        if constexpr (TOP) top.offer(r.m, parity);
        if (tid < ends) {
            const float x[1] = {end};
            add_values<1, true, false>(r, x, end, a.c);
        }
        r = cta_join<kThreads, true, false>(r, part[parity], a.c);
        float bound = 0.0f;
        if constexpr (TOP) bound = top.bound(parity);
        if (ctas > 1) r = cluster_join<true, false>(r, &mine[parity], ctas, a.c);
        parity ^= 1;
        if constexpr (TOP) {
            const int c = top.find(zr, g, group_lg, end, end_at, ends, bound);
            const float log_s = logf(r.s);
            auto write = [&](int n, uint64_t x) {
                a.top_index[(int64_t)row * a.k + n] = (uint32_t)~x;
                a.top_logprob[(int64_t)row * a.k + n] = log_prob(key_value((uint32_t)(x >> 32)), r.m, r.s, log_s, a.tau);
            };
            if (ctas == 1) {
                rank_list<kThreads>(top.list, c, a.k, write);
            } else {
                uint64_t* best = top.list + top.cap;  // of this CTA, sorted
                for (int n = tid; n < a.k; n += kThreads)
                    if (n >= c) best[n] = 0;
                rank_list<kThreads>(top.list, c, a.k, [&](int n, uint64_t x) { best[n] = x; });
                cluster_sync();
                if (rank == 0)
                    for (int n = tid; n < (int)ctas * a.k; n += kThreads)
                        top.list[n] = ld_dsmem_u64(map_to_rank(smem_addr(best + n % a.k), n / a.k));
                cluster_sync();
                if (rank == 0) {
                    // an entry's rank is its place in its own list and, by halving, those in the others
                    for (int n = tid; n < (int)ctas * a.k; n += kThreads) {
                        const uint64_t x = top.list[n];
                        if (x == 0) continue;
                        int place = n % a.k;
                        for (int q = 0; q < (int)ctas && place < a.k; ++q) {
                            if (q == n / a.k) continue;
                            const uint64_t* other = top.list + q * a.k;
                            int lo = 0, hi = a.k;
                            while (lo < hi) {
                                const int mid = (lo + hi) >> 1;
                                if (other[mid] > x) lo = mid + 1;
                                else hi = mid;
                            }
                            place += lo;
                        }
                        if (place < a.k) write(place, x);
                    }
                }
            }
            if (rank == 0 && tid == kThreads - 1) score_write(a, row, z_t, r);
            __syncthreads();
            if (tid == 0) top_shared.count = 0;
        } else {
            if (rank == 0 && tid == kThreads - 1) score_write(a, row, z_t, r);
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
        // everything is asked for before the first use of any of it
        const int64_t t = a.tok.p ? a.tok.p[row_offset(a.tok.sb, a.tok.st, a.tok.T, row)] : -1;
        T* dr = reinterpret_cast<T*>(a.d.p) + row_offset(a.d.sb, a.d.st, a.d.T, row);
        const T* zr = reinterpret_cast<const T*>(a.z.p) + row_offset(a.z.sb, a.z.st, a.z.T, row);
        float x[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int j = lane + 32 * e;
            x[e] = j < a.V ? to_float(zr[j]) : 0.0f;
        }
        const ScoreGrad r = score_grad_row(a, row, t);
        const bool live = !(a.tok.p && t == a.tok.ignore);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int j = lane + 32 * e;
            if (j < a.V) dr[j] = from_float<T>(live ? r.at(x[e]) * r.inv_tau : 0.0f);
        }
        if (!live) continue;
        __syncwarp();
        score_grad_slots<T>(a, r, row, t, zr, dr, 0, a.V, lane, 32);
    }
}

// 8192 x 65536 bf16, a fifth of the rows padding: 310 us; with 512, whose parts of a row end together, 381 us
constexpr int kGradThreads = 128;

// CTA `part` of 2^lg of a row
template <int DT>
__global__ void __launch_bounds__(kGradThreads, 1024 / kGradThreads) score_grad_row_kernel(ScoreGradArgs a, uint32_t lg) {
    using T = typename Elem<DT>::type;
    constexpr int kVec = Elem<DT>::kVec;
    const int tid = threadIdx.x;
    const uint32_t row = blockIdx.x >> lg;
    const int64_t t = a.tok.p ? a.tok.p[row_offset(a.tok.sb, a.tok.st, a.tok.T, row)] : -1;
    const T* zr = reinterpret_cast<const T*>(a.z.p) + row_offset(a.z.sb, a.z.st, a.z.T, row);
    T* dr = reinterpret_cast<T*>(a.d.p) + row_offset(a.d.sb, a.d.st, a.d.T, row);
    const Segment g = segment_of<DT>(zr, a.V, blockIdx.x & ((1u << lg) - 1u), lg);
    const bool live = !(a.tok.p && t == a.tok.ignore);
    const bool wide = (((uintptr_t)zr ^ (uintptr_t)dr) & 15u) == 0;  // 16-byte stores
    ScoreGrad r;
    if (live) r = score_grad_row(a, row, t);
    const uint4* body = reinterpret_cast<const uint4*>(zr + g.h0);
    auto write = [&](int v, const uint4& raw) {
        float y[kVec];
        if (live) {
            unpack16<DT>(raw, y);
#pragma unroll
            for (int e = 0; e < kVec; ++e) y[e] = r.at(y[e]) * r.inv_tau;
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
    };
    constexpr int kAhead = 4;  // vectors of a thread that are loaded at a time
    for (int v = g.v0 + tid; v < g.v1; v += kAhead * kGradThreads) {
        uint4 raw[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (live && v + u * kGradThreads < g.v1) raw[u] = __ldcs(body + v + u * kGradThreads);
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (v + u * kGradThreads < g.v1) write(v + u * kGradThreads, raw[u]);
    }
    if (tid < g.head) dr[tid] = from_float<T>(live ? r.at(to_float(zr[tid])) * r.inv_tau : 0.0f);
    if (tid < g.tail) dr[g.t0 + tid] = from_float<T>(live ? r.at(to_float(zr[g.t0 + tid])) * r.inv_tau : 0.0f);
    if (!live) return;
    __syncthreads();
    score_grad_slots<T>(a, r, row, t, zr, dr, g.j0, g.j1, tid, kGradThreads);
}

}  // namespace il
