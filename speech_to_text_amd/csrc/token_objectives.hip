// Token objectives, host side: arguments, which team takes a row, launches (include/sttfe.h, "token objectives").
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <atomic>

#include "timing.h"
#include "token_objectives.h"

namespace sttfe {
namespace {

// Rows that count, by one team.
constexpr int kRowsThreads = 1024;
__device__ int count_rows(const int64_t* __restrict__ labels, int64_t ignore, int64_t rows, int* part) {
    int n = 0;                                   // at most 2^24 rows
    for (int64_t r0 = 0; r0 < rows; r0 += 8 * kRowsThreads)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t r = r0 + i * kRowsThreads + threadIdx.x;
            const int64_t y = r < rows ? labels[r] : ignore;
            n += __popcll(__ballot(y != ignore));
        }
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = n;
    __syncthreads();
    n = 0;
    for (int i = 0; i < kRowsThreads / 64; ++i) n += part[i];
    return n;
}

// factor = weight (sum) or weight / number of rows that count (mean)
__global__ __launch_bounds__(kRowsThreads) void distill_factor_kernel(const int64_t* __restrict__ labels, int64_t ignore, int64_t rows,
                                                                      float weight, bool mean, float* __restrict__ factor) {
    __shared__ int part[kRowsThreads / 64];
    const int n = mean ? count_rows(labels, ignore, rows, part) : 1;
    if (threadIdx.x == 0) factor[0] = mean_factor(weight, n);
}

// total = factor * sum of the rows' losses, in 64 bits and in a fixed order
enum Factor { kFactorMade = 0, kFactorWeight = 1, kFactorCount = 2 };      // where the factor comes from
__global__ __launch_bounds__(kRowsThreads) void distill_total_kernel(const float* __restrict__ losses, int64_t rows,
                                                                     const int64_t* __restrict__ labels, int64_t ignore, float weight,
                                                                     int from, float* __restrict__ factor, float* __restrict__ total) {
    __shared__ int part_n[kRowsThreads / 64];
    __shared__ double part[kRowsThreads / 64];
    float f = weight;
    if (from == kFactorCount) f = mean_factor(weight, count_rows(labels, ignore, rows, part_n));
    if (from == kFactorMade) f = factor[0];
    double s = 0.0;
    for (int64_t r0 = 0; r0 < rows; r0 += 8 * kRowsThreads)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t r = r0 + i * kRowsThreads + threadIdx.x;
            s += r < rows ? (double)losses[r] : 0.0;
        }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) s += __shfl_xor(s, d, 64);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double all = 0.0;
        for (int i = 0; i < kRowsThreads / 64; ++i) all += part[i];
        total[0] = (float)(all * (double)f);
        factor[0] = f;
    }
}

int compute_units() {
    static std::atomic<int> known[64];           // by device; a device's count does not change
    int dev = 0, n = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
    n = known[dev].load(std::memory_order_relaxed);
    if (n == 0) {
        if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n < 1) n = 256;
        known[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}
// Teams of a launch over n rows: 0 = one for every segment, else that many which deal the rows among themselves: as many as the
// registers of two rows a thread leave room for.
int dealt_teams(const Plan& plan, int64_t n, bool ahead) {
    if (kTeamWaves[plan.team] < 4) return 0;
    const int teams = compute_units() * (4 * kWavesPerSimd(kTeamVpt[plan.team], ahead) / kTeamWaves[plan.team]);
    return n * plan.segs > teams ? teams : 0;
}

Distill distill_args(const int64_t* labels, int64_t ignore, const int64_t* ids, const float* teacher, int K, float tau, float alpha) {
    Distill a{labels, ids, teacher, ignore, K, tau, (float)(1.0 / (double)tau), alpha, 0.f, (float)kLog2e, 0.f, alpha != 0.f, alpha != 1.f};
    a.c = a.teacher ? (float)(kLog2e / (double)tau) : (float)kLog2e;
    a.climb = (float)(kClimb / (double)(a.label && a.c1 > a.c ? a.c1 : a.c));
    return a;
}
Mode distill_mode(const Distill& a) {
    if (!a.teacher || !a.label || a.tau == 1.f) return kOne;
    return a.tau == 2.f ? kSquare : kTwo;
}
int check_rows(const void* logits, int dtype, int64_t outer, int64_t inner, int64_t stride_outer, int64_t stride_inner, int vocab) {
    if (outer < 0 || inner < 0 || vocab < 1 || stride_outer < 0 || stride_inner < 0) return STTFE_E_INVALID_ARG;
    if (dtype != STTFE_DTYPE_F32 && dtype != STTFE_DTYPE_F16 && dtype != STTFE_DTYPE_BF16) return STTFE_E_INVALID_ARG;
    if (inner > 0 && outer > STTFE_MAX_ROWS / inner) return STTFE_E_UNSUPPORTED;
    if (vocab > STTFE_MAX_VOCAB) return STTFE_E_UNSUPPORTED;
    if (outer * inner > 0 && (!logits || ((uintptr_t)logits & (dtype == STTFE_DTYPE_F32 ? 3 : 1)))) return STTFE_E_INVALID_ARG;
    return STTFE_OK;
}

// c = log2(e) / T and T^2 stay far inside float's range.
bool temperature_ok(float t) { return t >= 1e-6f && t <= 1e6f; }
bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }       // read and written as float4

}  // namespace
}  // namespace sttfe

using namespace sttfe;

#define STTFE_BY_DTYPE(dtype, ...)                                   \
    do {                                                              \
        if ((dtype) == STTFE_DTYPE_F32) { using T = float; __VA_ARGS__; }    \
        else if ((dtype) == STTFE_DTYPE_F16) { using T = half_t; __VA_ARGS__; } \
        else { using T = bf16_t; __VA_ARGS__; }                              \
    } while (0)

extern "C" int sttfe_token_logprobs_workspace_bytes(int64_t rows, int vocab, int dtype, int top_k, size_t* bytes) {
    if (!bytes || rows < 0 || vocab < 1 || top_k < 0 || top_k > STTFE_MAX_TOP || top_k > vocab) return STTFE_E_INVALID_ARG;
    if (dtype != STTFE_DTYPE_F32 && dtype != STTFE_DTYPE_F16 && dtype != STTFE_DTYPE_BF16) return STTFE_E_INVALID_ARG;
    if (rows > STTFE_MAX_ROWS || vocab > STTFE_MAX_VOCAB) return STTFE_E_UNSUPPORTED;
    const Plan plan = row_plan(vocab, dtype);
    *bytes = plan.segs == 1 ? 0 : (size_t)rows * plan.segs * (sizeof(float4) + sizeof(uint64_t) * (size_t)top_k);
    return STTFE_OK;
}

extern "C" int sttfe_token_logprobs(const void* logits, int dtype, int64_t outer, int64_t inner, int64_t stride_outer,
                                    int64_t stride_inner, int vocab, const int64_t* labels, int64_t ignore_index,
                                    float temperature, int top_k, float* logprobs, float* entropy, float* stats,
                                    int64_t* top_ids, float* top_logprobs, void* workspace, size_t workspace_bytes, void* stream_) {
    int rc = check_rows(logits, dtype, outer, inner, stride_outer, stride_inner, vocab);
    if (rc != STTFE_OK) return rc;
    if (!temperature_ok(temperature) || top_k < 0 || top_k > STTFE_MAX_TOP || top_k > vocab) return STTFE_E_INVALID_ARG;
    const int64_t n = outer * inner;
    if (n == 0) return STTFE_OK;
    if ((logprobs && !labels) || (top_k > 0 && (!top_ids || !top_logprobs))) return STTFE_E_INVALID_ARG;
    if (!aligned16(stats) || !aligned16(workspace)) return STTFE_E_INVALID_ARG;
    size_t need = 0;
    rc = sttfe_token_logprobs_workspace_bytes(n, vocab, dtype, top_k, &need);
    if (rc != STTFE_OK) return rc;
    if (workspace_bytes < need || (need && !workspace)) return STTFE_E_WORKSPACE;
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    (void)hipGetLastError();
    const Plan plan = row_plan(vocab, dtype);
    const Rows rows{logits, (uint32_t)inner, stride_outer, stride_inner, vocab, plan.segs, plan.seg_len};
    float4* parts = static_cast<float4*>(workspace);
    const int teams = dealt_teams(plan, n, kScoreAhead(top_k > 0));
    const Score a{labels, ignore_index, (float)(kLog2e / (double)temperature), (float)(1.0 / (double)temperature),
                  (float)(kClimb / kLog2e * (double)temperature), top_k, logprobs, entropy, stats, top_ids, top_logprobs, parts, reinterpret_cast<uint64_t*>(parts + (plan.segs > 1 ? n * plan.segs : 0)), (uint32_t)n, teams > 0};
    {
        ScopedTiming t(kTimeTokenLogprobs, stream);
        STTFE_BY_DTYPE(dtype, Launch<T>::score(plan, rows, a, (unsigned)(teams ? teams : n * plan.segs), entropy || stats, stream));
        if (plan.segs > 1) STTFE_BY_DTYPE(dtype, Launch<T>::score_join(rows, a, (unsigned)n, stream));
    }
    if (hip_failed(hipGetLastError(), "token logprobs kernel launch")) return STTFE_E_LAUNCH;
    return STTFE_OK;
}

extern "C" int sttfe_token_logprobs_grad(const void* logits, int dtype, int64_t outer, int64_t inner, int64_t stride_outer,
                                         int64_t stride_inner, int vocab, const int64_t* labels, int64_t ignore_index,
                                         float temperature, const float* stats, const float* g_logprobs, const float* g_entropy,
                                         int top_k, const int64_t* top_ids, const float* g_top, void* grad, void* stream_) {
    int rc = check_rows(logits, dtype, outer, inner, stride_outer, stride_inner, vocab);
    if (rc != STTFE_OK) return rc;
    if (!temperature_ok(temperature) || top_k < 0 || top_k > STTFE_MAX_TOP || top_k > vocab) return STTFE_E_INVALID_ARG;
    const int64_t n = outer * inner;
    if (n == 0) return STTFE_OK;
    if (!stats || !aligned16(stats) || !grad || (g_logprobs && !labels) || (g_top && (top_k == 0 || !top_ids))) return STTFE_E_INVALID_ARG;
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    (void)hipGetLastError();
    const Plan plan = grad_plan(vocab, dtype);
    const Rows rows{logits, (uint32_t)inner, stride_outer, stride_inner, vocab, plan.segs, plan.seg_len};
    const ScoreGrad a{labels, ignore_index, (float)(kLog2e / (double)temperature), (float)(1.0 / (double)temperature), stats, g_logprobs,
                      g_entropy, top_k, top_ids, g_top};
    {
        ScopedTiming t(kTimeTokenLogprobsGrad, stream);
        STTFE_BY_DTYPE(dtype, Launch<T>::score_grad(rows, a, (unsigned)n, static_cast<T*>(grad), stream));
    }
    if (hip_failed(hipGetLastError(), "token logprobs gradient kernel launch")) return STTFE_E_LAUNCH;
    return STTFE_OK;
}

static int check_distill(const int64_t* labels, const int64_t* ids, const float* teacher, int K, float tau, float alpha) {
    if (!labels || !ids || !teacher || K < 1 || K > STTFE_MAX_TOP || !temperature_ok(tau) || !(alpha >= 0.f && alpha <= 1.f))
        return STTFE_E_INVALID_ARG;
    return STTFE_OK;
}

extern "C" int sttfe_distill_workspace_bytes(int64_t rows, int vocab, int dtype, size_t* bytes) {
    if (!bytes || rows < 0 || vocab < 1) return STTFE_E_INVALID_ARG;
    if (dtype != STTFE_DTYPE_F32 && dtype != STTFE_DTYPE_F16 && dtype != STTFE_DTYPE_BF16) return STTFE_E_INVALID_ARG;
    if (rows > STTFE_MAX_ROWS || vocab > STTFE_MAX_VOCAB) return STTFE_E_UNSUPPORTED;
    const Plan plan = row_plan(vocab, dtype);
    *bytes = plan.segs == 1 ? 0 : (size_t)rows * plan.segs * sizeof(float4) + (size_t)rows * 4 * sizeof(float);
    return STTFE_OK;
}

extern "C" int sttfe_distill_loss(const void* logits, int dtype, int64_t outer, int64_t inner, int64_t stride_outer,
                                  int64_t stride_inner, int vocab, const int64_t* labels, int64_t ignore_index,
                                  const int64_t* teacher_ids, const float* teacher_logits, int teacher_k, float temperature,
                                  float alpha, float weight, int reduction, float* losses, float* total, float* factor,
                                  float* stats, void* grad, void* workspace, size_t workspace_bytes, void* stream_) {
    int rc = check_rows(logits, dtype, outer, inner, stride_outer, stride_inner, vocab);
    if (rc != STTFE_OK) return rc;
    if (reduction != STTFE_REDUCE_NONE && reduction != STTFE_REDUCE_SUM && reduction != STTFE_REDUCE_MEAN) return STTFE_E_INVALID_ARG;
    const int64_t n = outer * inner;
    if (reduction != STTFE_REDUCE_NONE && (!total || !factor)) return STTFE_E_INVALID_ARG;
    if (n > 0) {
        rc = check_distill(labels, teacher_ids, teacher_logits, teacher_k, temperature, alpha);
        if (rc != STTFE_OK) return rc;
        if (!losses || !aligned16(stats) || !aligned16(workspace)) return STTFE_E_INVALID_ARG;
    }
    if (n == 0 && reduction == STTFE_REDUCE_NONE) return STTFE_OK;
    size_t need = 0;
    rc = sttfe_distill_workspace_bytes(n, vocab, dtype, &need);
    if (rc != STTFE_OK) return rc;
    if (workspace_bytes < need || (need && !workspace)) return STTFE_E_WORKSPACE;
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    (void)hipGetLastError();
    const Plan plan = row_plan(vocab, dtype);
    const Rows rows{logits, (uint32_t)inner, stride_outer, stride_inner, vocab, plan.segs, plan.seg_len};
    const Distill a = distill_args(labels, ignore_index, teacher_ids, teacher_logits, teacher_k, temperature, alpha);
    const Mode mode = distill_mode(a);
    // The factor of the gradient: from a kernel of its own where there are many rows to count, or a gradient kernel to read it.
    const bool mean = reduction == STTFE_REDUCE_MEAN, apart = grad && plan.segs > 1;
    const Factor from = reduction == STTFE_REDUCE_NONE ? kFactorWeight
                        : apart || (mean && n > kCountHere) ? kFactorMade : mean ? kFactorCount : kFactorWeight;
    if (from == kFactorMade)
        hipLaunchKernelGGL(distill_factor_kernel, dim3(1), dim3(kRowsThreads), 0, stream, labels, ignore_index, n, weight, mean, factor);
    const float* made = from == kFactorMade ? factor : nullptr;
    const float sum_weight = reduction == STTFE_REDUCE_NONE ? 1.f : weight;
    if (n > 0) {
        ScopedTiming t(kTimeDistill, stream);
        float4* parts = static_cast<float4*>(workspace);
        const int teams = dealt_teams(plan, n, kDistillAhead);
        const Out o{made, sum_weight, mean, losses, stats, parts, (uint32_t)n, teams > 0};
        if (plan.segs == 1) {
            STTFE_BY_DTYPE(dtype, Launch<T>::distill(plan, rows, a, mode, (unsigned)(teams ? teams : n), o, static_cast<T*>(grad), stream));
        } else {
            // a row over several teams: their sums, the loss from the joined sums, then the gradient in a pass of its own
            float* st = stats ? stats : reinterpret_cast<float*>(parts + n * plan.segs);
            STTFE_BY_DTYPE(dtype, {
                Launch<T>::distill(plan, rows, a, mode, (unsigned)(teams ? teams : n * plan.segs), o, static_cast<T*>(nullptr), stream);
                Launch<T>::distill_join(rows, a, mode, parts, losses, st, (unsigned)n, stream);
            });
            if (grad) {
                const Plan gp = grad_plan(vocab, dtype);
                const Rows grows{logits, (uint32_t)inner, stride_outer, stride_inner, vocab, gp.segs, gp.seg_len};
                STTFE_BY_DTYPE(dtype, Launch<T>::distill_grad(grows, a, mode, st, made, nullptr, nullptr, (unsigned)n, static_cast<T*>(grad), stream));
            }
        }
    }
    if (reduction != STTFE_REDUCE_NONE)
        hipLaunchKernelGGL(distill_total_kernel, dim3(1), dim3(kRowsThreads), 0, stream, losses, n, labels, ignore_index, weight,
                           (int)from, factor, total);
    if (hip_failed(hipGetLastError(), "distillation kernel launch")) return STTFE_E_LAUNCH;
    return STTFE_OK;
}

extern "C" int sttfe_distill_grad(const void* logits, int dtype, int64_t outer, int64_t inner, int64_t stride_outer,
                                  int64_t stride_inner, int vocab, const int64_t* labels, int64_t ignore_index,
                                  const int64_t* teacher_ids, const float* teacher_logits, int teacher_k, float temperature,
                                  float alpha, const float* stats, const float* factor, const float* g, const float* g_rows,
                                  void* grad, void* stream_) {
    int rc = check_rows(logits, dtype, outer, inner, stride_outer, stride_inner, vocab);
    if (rc != STTFE_OK) return rc;
    const int64_t n = outer * inner;
    if (n == 0) return STTFE_OK;
    rc = check_distill(labels, teacher_ids, teacher_logits, teacher_k, temperature, alpha);
    if (rc != STTFE_OK) return rc;
    if (!stats || !aligned16(stats) || !grad) return STTFE_E_INVALID_ARG;
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    (void)hipGetLastError();
    const Plan plan = grad_plan(vocab, dtype);
    const Rows rows{logits, (uint32_t)inner, stride_outer, stride_inner, vocab, plan.segs, plan.seg_len};
    const Distill a = distill_args(labels, ignore_index, teacher_ids, teacher_logits, teacher_k, temperature, alpha);
    {
        ScopedTiming t(kTimeDistillGrad, stream);
        STTFE_BY_DTYPE(dtype, Launch<T>::distill_grad(rows, a, distill_mode(a), stats, factor, g, g_rows, (unsigned)n, static_cast<T*>(grad), stream));
    }
    if (hip_failed(hipGetLastError(), "distillation gradient kernel launch")) return STTFE_E_LAUNCH;
    return STTFE_OK;
}

extern "C" int sttfe_distill_rescale(void* grad, int dtype, int64_t count, const float* g, void* stream_) {
    if (count < 0 || (dtype != STTFE_DTYPE_F32 && dtype != STTFE_DTYPE_F16 && dtype != STTFE_DTYPE_BF16)) return STTFE_E_INVALID_ARG;
    if (count == 0) return STTFE_OK;
    if (!grad || !g) return STTFE_E_INVALID_ARG;
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    (void)hipGetLastError();
    STTFE_BY_DTYPE(dtype, Launch<T>::rescale(static_cast<T*>(grad), count, g, stream));
    if (hip_failed(hipGetLastError(), "gradient rescale kernel launch")) return STTFE_E_LAUNCH;
    return STTFE_OK;
}
