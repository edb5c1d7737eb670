// il_logits.cu -- entry points of the operators on a language model's logits:
// il_token_logprobs, il_distill and their gradients (include/aiwn_il.h).
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>

#include "../../include/aiwn_il.h"
#include "il_host.h"
#include "il_distill.cuh"
#include "il_score.cuh"

namespace {

using namespace il;

constexpr double kLog2e64 = 1.4426950408889634074;
// What a row costs beside its logits, as bytes of loading by one CTA.  Few rows take 13 to 16 us whatever the cluster,
// as long as it is not too wide: one row of 131072 bf16 with 20 alternatives 15 to 25 us with one CTA, 14 with 4 or 8,
// 18 with 16; 48 rows of 50021 fp32 14 to 18 us with one, 14 to 15 with 4 of 256 threads, 24 with 4 of 512; 99 rows of
// 5003 15 us with one, 21 with 4.
constexpr double kRowCost = 32768;
// bytes of rows that the L2 keeps from one pass over them to the next: 59 MB of rows at work (2048 x 50021 fp32, two
// CTAs an SM: 191 us, one: 219 us) are, 76 MB (8192 x 131072 bf16, two: 1007 us, one: 883 us) are not
constexpr double kResident = 62e6;
constexpr int64_t kMaxGrid = 8192;  // CTAs of a kernel that adds up a whole loss

// two strides as one where that serves all rows, which saves a division a row
void merge_strides(int64_t& sb, int64_t& st, int64_t B, int64_t& T) {
    if (T != 1 && (B == 1 || sb == T * st)) sb = st, T = 1;
}
template <class R, class P>
R rows_of(P* p, int64_t sb, int64_t st, int64_t B, int64_t T) {
    merge_strides(sb, st, B, T);
    return R{p, sb, st, (uint32_t)T};
}
Tokens tokens_of(const int64_t* p, int64_t sb, int64_t st, int64_t ignore, int64_t B, int64_t T) {
    merge_strides(sb, st, B, T);
    return Tokens{p, sb, st, ignore, (uint32_t)T};
}

// how a [B, T, V] operand is cut up
struct Plan {
    int regs;     // logits a lane holds, rows of one warp; 0: CTAs
    int threads;  // of a CTA
    uint32_t lg;  // 2^lg CTAs a row
    unsigned grid;
};

int check_rows(int dtype, int64_t B, int64_t T, int64_t V, double temperature) {
    if (dtype != IL_F32 && dtype != IL_BF16) return IL_ERR_DTYPE;
    if (B < 0 || T < 0 || V < 1 || V > kMaxVocab) return IL_ERR_SHAPE;
    if (B > 0 && T > (int64_t(1) << 30) / B) return IL_ERR_SHAPE;
    const float tau = (float)temperature;
    if (!(tau > 0.0f) || isinf(tau) || isinf((float)(kLog2e64 / temperature))) return IL_ERR_VALUE;
    return IL_OK;
}

// the row stride of the operands and their element size: natural alignment of the base is all that is asked
int check_align(const void* p, int dtype) { return ((uintptr_t)p & (dtype == IL_BF16 ? 1u : 3u)) ? IL_ERR_ALIGN : IL_OK; }

// Rows of more than kWarpVocab logits.  An SM holds 512 or 768 threads, in CTAs of 64 to 512: a warp's share
// of what a row costs beside its logits is the same whatever the row's length, so that shorter rows get fewer warps.
// Where all rows are at work at once and leave SMs idle, a cluster of c CTAs takes a row.  Of these the one that takes
// the shortest time by a simple count: a CTA has 1/c of a row to load at its share of the SM's rate, and the rest costs
// as much as kRowCost bytes, more for each doubling of a cluster.  A row that is gone through twice finds itself in the
// L2 the second time as long as the rows at work are not more than kResident bytes.
// shared(t, lg): bytes of shared memory of a CTA beside its stream; least: threads that it has at least.
// AIWN_IL_LOGITS=threads,ctas pins both where they can serve the row (for the tests).
template <class Shared>
Plan plan_rows(int64_t N, int64_t V, int64_t k, int dtype, int sms, int passes, int least, Shared shared) {
    Plan p{0, 256, 0, 0};
    if (V <= kWarpVocab) {
        p.regs = (int)((V + 31) / 32);
        const int64_t blocks = (N + 7) / 8, most = (int64_t)sms * 8;
        p.grid = (unsigned)(blocks < most ? blocks : most);
        return p;
    }
    const double bytes = (double)V * (dtype == IL_BF16 ? 2 : 4);
    const int stream = passes > 1 ? RowStream<kF32, 1, 2>::kBytes : RowStream<kF32, 1, 1>::kBytes;  // a thread
    double best = 0.0;
    int threads = 0, ctas = 0;
    const char* pin = getenv("AIWN_IL_LOGITS");
    if (pin && (sscanf(pin, "%d,%d", &threads, &ctas) != 2 ||
                (threads != 64 && threads != 128 && threads != 256 && threads != 512)))
        threads = ctas = 0;
    int lg0 = 0;  // the least that a CTA's part of a row allows
    while ((V >> lg0) > (1 << 18)) ++lg0;
    const int need = k > 64 ? 128 : 64;  // a slot, or an alternative, a thread
    if (threads && threads < need) threads = need;
    for (int t = need; t <= 512; t *= 2) {
        if (threads ? threads != t : t < least) continue;
        for (int lg = lg0; (1 << lg) <= kMaxCluster; ++lg) {
            const int c = 1 << lg;
            if (threads && c < ctas && 2 * c <= kMaxCluster) continue;
            if (threads && p.grid) break;
            const int64_t by_smem = 227 * 1024 / (stream * t + shared(t, lg) + 3 * 1024);
            int64_t held = by_smem < sm_threads(passes) / t ? by_smem : sm_threads(passes) / t;
            if (held < 1) continue;
            if (lg > lg0 && !threads && (N * c > sms * held || bytes / c < 16 * t)) break;
            if (passes > 1)
                while (held > 1 && (double)sms * held / c * bytes > kResident) --held;
            const int64_t clusters = (int64_t)sms * held / c, used = N < clusters ? N : clusters;
            const double rounds = (double)((N + clusters - 1) / clusters);
            const double on_sm = (double)((used * c + sms - 1) / sms);  // CTAs that share an SM
            const double rate = on_sm * t < 640 ? on_sm * t / 640.0 : 1.0;
            const double time = rounds * (bytes / c * on_sm / rate + (1 + lg) * kRowCost);
            if (p.grid == 0 || time < best) {
                best = time;
                p.threads = t;
                p.lg = lg;
                p.grid = (unsigned)(used * c);
            }
        }
    }
    return p;
}

template <class... P, class... A>
int launch(void (*kern)(P...), unsigned grid, int threads, uint32_t lg, size_t smem, cudaStream_t s, A... args) {
    if (smem > 16 * 1024)  // beyond 48 KB with the static arrays
        if (const int st = host_allow_shared((const void*)kern, smem)) return st;
    if (lg > 3 && cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) {
        cudaGetLastError();
        return IL_ERR_LAUNCH;
    }
    const uint32_t ctas = 1u << lg;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = ctas;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = ctas > 1 ? 1 : 0;
    if (cudaLaunchKernelEx(&cfg, kern, P(args)...) != cudaSuccess) {
        cudaGetLastError();
        return IL_ERR_LAUNCH;
    }
    return host_launch_status(1);
}

// f(integral constant E) for the smallest instantiated E >= regs
template <class F>
int with_regs(int regs, F f) {
#define IL_REGS(E) \
    if (regs <= E) return f(std::integral_constant<int, E>());
    IL_REGS(1) IL_REGS(2) IL_REGS(3) IL_REGS(4) IL_REGS(8) IL_REGS(16) IL_REGS(32)
#undef IL_REGS
    return IL_ERR_SHAPE;
}
template <class F>
int with_dtype(int dtype, F f) {
    return dtype == IL_BF16 ? f(std::integral_constant<int, kBF16>()) : f(std::integral_constant<int, kF32>());
}
template <class F>
int with_threads(int threads, F f) {
    if (threads == 64) return f(std::integral_constant<int, 64>());
    if (threads == 128) return f(std::integral_constant<int, 128>());
    if (threads == 256) return f(std::integral_constant<int, 256>());
    return f(std::integral_constant<int, 512>());
}
template <class F>
int with_bool(bool b, F f) {
    return b ? f(std::true_type()) : f(std::false_type());
}

}  // namespace

extern "C" {

int il_token_logprobs(const void* logits, int dtype, int64_t B, int64_t T, int64_t V, int64_t stride_b,
                      int64_t stride_t, const int64_t* tokens, int64_t tokens_b, int64_t tokens_t,
                      int64_t ignore_index, int64_t k, double temperature, float* logprob, float* entropy,
                      float* stats, int64_t* top_index, float* top_logprob, void* stream) {
    int st = check_rows(dtype, B, T, V, temperature);
    if (st) return st;
    if (k < 0 || k > kMaxTop || k > V) return IL_ERR_SHAPE;
    if (B * T == 0) return IL_OK;
    if (!logits || !entropy || (tokens && !logprob) || (k > 0 && (!top_index || !top_logprob))) return IL_ERR_NULL;
    if ((st = check_align(logits, dtype))) return st;
    if ((uintptr_t)stats & 7u) return IL_ERR_ALIGN;
    int sms = 0;
    if ((st = host_check_device(&sms))) return st;
    ScoreArgs a{};
    a.z = rows_of<RowsIn>(logits, stride_b, stride_t, B, T);
    a.tok = tokens_of(tokens, tokens_b, tokens_t, ignore_index, B, T);
    a.N = (uint32_t)(B * T), a.V = (int)V, a.k = (int)k;
    a.tau = (float)temperature, a.c = (float)(kLog2e64 / temperature);
    a.logprob = tokens ? logprob : nullptr, a.entropy = entropy, a.stats = reinterpret_cast<float2*>(stats);
    a.top_index = top_index, a.top_logprob = top_logprob;
    // more alternatives than a quarter of the lanes make the bound of their maxima a weak one (4096 x 131072 bf16, 128
    // alternatives: 627 us with 128 threads, 393 us with 256)
    const Plan p = plan_rows(a.N, V, k, dtype, sms, 1, k > 64 ? 256 : k > 32 ? 128 : 64, [&](int, int lg) {
        return k > 0 ? 9 * 1024 + 8 * (top_list(a.k, lg) + (lg ? a.k : 0)) : 0;
    });
    cudaStream_t s = (cudaStream_t)stream;
    return with_dtype(dtype, [&](auto dt) {
        if (p.regs)
            return with_regs(p.regs, [&](auto e) {
                return launch(score_warp_kernel<dt.value, e.value>, p.grid, 256, 0, 0, s, a);
            });
        return with_bool(k > 0, [&](auto top) {
            return with_threads(p.threads, [&](auto th) {
                const size_t smem = RowStream<dt.value, th.value, 1>::kBytes +
                                    (top.value ? 8 * (size_t)(top_list(a.k, (int)p.lg) + (p.lg ? a.k : 0)) : 0);
                return launch(score_row_kernel<dt.value, th.value, top.value>, p.grid, th.value, p.lg, smem, s, a, p.lg);
            });
        });
    });
}

int il_token_logprobs_backward(const void* logits, int dtype, int64_t B, int64_t T, int64_t V, int64_t stride_b,
                               int64_t stride_t, const int64_t* tokens, int64_t tokens_b, int64_t tokens_t,
                               int64_t ignore_index, int64_t k, double temperature, const float* entropy,
                               const float* stats, const int64_t* top_index, const float* g_logprob,
                               const float* g_entropy, const float* g_top, void* dlogits, int64_t dstride_b,
                               int64_t dstride_t, void* stream) {
    int st = check_rows(dtype, B, T, V, temperature);
    if (st) return st;
    if (k < 0 || k > kMaxTop || k > V) return IL_ERR_SHAPE;
    if (B * T == 0) return IL_OK;
    if (!logits || !entropy || !stats || !dlogits || (g_logprob && !tokens) || (k > 0 && g_top && !top_index))
        return IL_ERR_NULL;
    if ((st = check_align(logits, dtype)) || (st = check_align(dlogits, dtype))) return st;
    if ((uintptr_t)stats & 7u) return IL_ERR_ALIGN;
    int sms = 0;
    if ((st = host_check_device(&sms))) return st;
    ScoreGradArgs a{};
    a.z = rows_of<RowsIn>(logits, stride_b, stride_t, B, T);
    a.tok = tokens_of(tokens, tokens_b, tokens_t, ignore_index, B, T);
    a.d = rows_of<RowsOut>(dlogits, dstride_b, dstride_t, B, T);
    a.N = (uint32_t)(B * T), a.V = (int)V, a.k = (int)k;
    a.tau = (float)temperature, a.c = (float)(kLog2e64 / temperature);
    a.stats = reinterpret_cast<const float2*>(stats), a.entropy = entropy, a.top_index = top_index;
    a.g_logprob = g_logprob, a.g_entropy = g_entropy, a.g_top = k > 0 ? g_top : nullptr;
    const Plan p = plan_rows(a.N, V, 0, dtype, sms, 1, 64, [](int, int) { return 0; });
    cudaStream_t s = (cudaStream_t)stream;
    return with_dtype(dtype, [&](auto dt) {
        if (p.regs)
            return with_regs(p.regs, [&](auto e) {
                return launch(score_grad_warp_kernel<dt.value, e.value>, p.grid, 256, 0, 0, s, a);
            });
        // parts of a row of at most 32768 logits, more of them where that leaves SMs idle
        uint32_t lg = 0;
        while ((V >> lg) > 32768 || (((int64_t)a.N << lg) < 4 * sms && (V >> lg) > 4096)) ++lg;
        const int64_t grid = (int64_t)a.N << lg;
        if (grid > 0x7fffffff) return (int)IL_ERR_SHAPE;
        return launch(score_grad_row_kernel<dt.value>, (unsigned)grid, kGradThreads, 0, 0, s, a, lg);
    });
}

int64_t il_distill_workspace_bytes(int64_t N) { return N < 0 ? -1 : (kMaxGrid + 4) * 4; }

int il_distill(const void* logits, int dtype, int64_t B, int64_t T, int64_t V, int64_t stride_b, int64_t stride_t,
               const int64_t* top_index, const float* top_logprob, int64_t k, const int64_t* targets,
               int64_t targets_b, int64_t targets_t, int64_t ignore_index, double alpha, double temperature, int tail,
               int reduction, const float* g, int only_if_not_one, float* loss, void* dlogits, int64_t dstride_b,
               int64_t dstride_t, void* workspace, int64_t workspace_bytes, void* stream) {
    int st = check_rows(dtype, B, T, V, temperature);
    if (st) return st;
    if (k < 0 || k > kMaxTop || reduction < 0 || reduction > 2) return IL_ERR_SHAPE;
    if (!(alpha >= 0.0 && alpha <= 1.0)) return IL_ERR_VALUE;
    const int64_t N = B * T;
    if (N == 0 && (reduction == 0 || !loss)) return IL_OK;
    if (!loss && !dlogits) return IL_ERR_NULL;
    if (N > 0 && (!logits || (k > 0 && (!top_index || !top_logprob)) || (alpha < 1.0 && !targets))) return IL_ERR_NULL;
    if (only_if_not_one && (!g || reduction == 0)) return IL_ERR_NULL;
    if ((st = check_align(logits, dtype)) || (st = check_align(dlogits, dtype))) return st;
    const bool whole = reduction != 0;
    if (whole && (!workspace || workspace_bytes < il_distill_workspace_bytes(N))) return IL_ERR_WORKSPACE;
    if ((uintptr_t)workspace & 15u) return IL_ERR_ALIGN;
    int sms = 0;
    if ((st = host_check_device(&sms))) return st;
    cudaStream_t s = (cudaStream_t)stream;
    float* ws = reinterpret_cast<float*>(workspace);
    DistillArgs a{};
    a.z = rows_of<RowsIn>(logits, stride_b, stride_t, B, T);
    a.tok = tokens_of(targets, targets_b, targets_t, ignore_index, B, T);
    a.d = rows_of<RowsOut>(dlogits, dstride_b, dstride_t, B, T);
    a.N = (uint32_t)N, a.V = (int)V, a.k = (int)k;
    a.index = top_index, a.logprob = top_logprob;
    a.tau = (float)temperature, a.c = (float)(kLog2e64 / temperature), a.alpha = (float)alpha;
    a.hard = alpha < 1.0;
    a.scale = 1.0f;
    a.g = g, a.g_rows = reduction == 0, a.skip_if_one = only_if_not_one;
    a.loss = loss, a.each = !whole;
    if (whole) {
        a.ticket = reinterpret_cast<uint32_t*>(ws) + 1, a.partial = ws + 4;
        if (reduction == kMean) {
            if (targets) a.scale_p = ws;
            else a.scale = 1.0f / (float)(N > 1 ? N : 1);
        }
        if (loss)
            if ((st = launch(distill_begin_kernel, 1, 1024, 0, 0, s, a.tok, a.N, ws))) return st;
    }
    const Plan p = N > 0 ? plan_rows(N, V, k, dtype, sms, dlogits ? 2 : 1, 64, [&](int t, int lg) {
        return tail ? distill_bitmap(a.V, 1 << lg, dtype == IL_BF16 ? 8 : 4, 4 * t) : 0;
    }) : Plan{1, 256, 0, 1};
    const bool two = a.hard && a.tau != 1.0f;
    return with_dtype(dtype, [&](auto dt) {
        return with_bool(tail != 0, [&](auto tl) {
            return with_bool(two, [&](auto s1) {
                if (p.regs)
                    return with_regs(p.regs, [&](auto e) {
                        return launch(distill_warp_kernel<dt.value, e.value, tl.value, s1.value>, p.grid, 256, 0, 0, s, a);
                    });
                return with_bool(dlogits != nullptr, [&](auto gr) {
                    return with_threads(p.threads, [&](auto th) {
                        const size_t smem = RowStream<dt.value, th.value, gr.value ? 2 : 1>::kBytes +
                                            (tl.value ? distill_bitmap(a.V, 1 << p.lg, Elem<dt.value>::kVec,
                                                                       RowStream<dt.value, th.value, 1>::kStep)
                                                      : 0);
                        return launch(distill_row_kernel<dt.value, th.value, tl.value, s1.value, gr.value>, p.grid,
                                      th.value, p.lg, smem, s, a, p.lg);
                    });
                });
            });
        });
    });
}

}  // extern "C"
