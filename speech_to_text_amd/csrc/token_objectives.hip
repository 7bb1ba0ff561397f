// Token objectives: label log probabilities with entropy and top alternatives, and distillation from a teacher's top
// logits, forward and backward (include/sttfe.h, "token objectives").
//
// One row of logits z[0 .. V) per label position; T = temperature, c = log2(e) / T, all sums in float32:
//   m = max z,  S = sum 2^(c (z_j - m)),  log2 p_j = c (z_j - m) - log2 S,  H = -sum p_j ln p_j.
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <math.h>
#include <stdint.h>

#include "../../include/sttfe.h"
#include "timing.h"

namespace sttfe {
namespace {

constexpr int kThreads = 256;
constexpr float kLn2 = 0.693147180559945309f;
constexpr double kLog2e = 1.442695040888963407;

struct Rows {                      // row r = (r / inner, r % inner)
    const void* base;
    int64_t inner, stride_outer, stride_inner;
    int vocab;
};

template <typename T>
__device__ const T* row_of(const Rows& a, int64_t r) {
    return static_cast<const T*>(a.base) + (r / a.inner) * a.stride_outer + (r % a.inner) * a.stride_inner;
}

__device__ inline float to_float(float x) { return x; }
__device__ inline float to_float(__half x) { return __half2float(x); }
__device__ inline float to_float(__hip_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ inline T from_float(float x);
template <> __device__ inline float from_float<float>(float x) { return x; }
template <> __device__ inline __half from_float<__half>(float x) { return __float2half(x); }
template <> __device__ inline __hip_bfloat16 from_float<__hip_bfloat16>(float x) { return __float2bfloat16(x); }

// Order of the alternatives: value falling (NaN before everything, as torch.topk has it; -0 equals +0), index rising.
__device__ inline uint64_t order_key(float x, int index) {
    uint32_t b = __float_as_uint(x + 0.0f);
    b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    if (x != x) b = 0xFFFFFFFEu;                // above +inf, below the start of a falling search
    return ((uint64_t)b << 32) | (uint32_t)(0xFFFFFFFFu - (uint32_t)index);
}

template <typename V, typename F>
__device__ V block_reduce(V v, F f, V* scratch) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v = f(v, (V)__shfl_xor(v, d, 64));
    __syncthreads();
    if (lane == 0) scratch[wave] = v;
    __syncthreads();
    V r = scratch[0];
    for (int w = 1; w < kThreads / 64; ++w) r = f(r, scratch[w]);
    return r;
}
__device__ inline float fadd(float a, float b) { return a + b; }
__device__ inline float fmaximum(float a, float b) { return fmaxf(a, b); }
__device__ inline uint64_t umaximum(uint64_t a, uint64_t b) { return a > b ? a : b; }

template <typename T>
__global__ __launch_bounds__(kThreads) void token_logprobs_kernel(
    Rows rows, const int64_t* __restrict__ labels, int64_t ignore, float c, float inv_t, int top_k, float* __restrict__ logprobs,
    float* __restrict__ entropy, float* __restrict__ stats, int64_t* __restrict__ top_ids, float* __restrict__ top_logprobs) {
    __shared__ float sf[kThreads / 64];
    __shared__ uint64_t su[kThreads / 64];
    const int64_t r = blockIdx.x;
    const int tid = threadIdx.x, V = rows.vocab;
    const int64_t label = labels ? labels[r] : 0;
    if (labels && label == ignore) {
        if (tid == 0) {
            if (logprobs) logprobs[r] = 0.f;
            if (entropy) entropy[r] = 0.f;
        }
        for (int k = tid; k < top_k; k += kThreads) {
            top_ids[r * top_k + k] = -1;
            top_logprobs[r * top_k + k] = -INFINITY;
        }
        return;
    }
    const T* __restrict__ z = row_of<T>(rows, r);
    float m = -INFINITY;
    for (int j = tid; j < V; j += kThreads) m = fmaxf(m, to_float(z[j]));
    m = block_reduce(m, fmaximum, sf);
    float s = 0.f, w = 0.f;
    for (int j = tid; j < V; j += kThreads) {
        const float y = (to_float(z[j]) - m) * c;
        const float e = exp2f(y);
        s += e;
        w += e * fmaxf(y, -200.f);             // -inf * 0: the term of a token without probability is 0
    }
    s = block_reduce(s, fadd, sf);
    w = block_reduce(w, fadd, sf);
    const float log2s = log2f(s);
    const float h = (log2s - w / s) * kLn2;
    if (tid == 0) {
        if (logprobs) {
            float lp = NAN;                    // a label outside the vocabulary
            if (label >= 0 && label < V) lp = (to_float(z[label]) - m) * inv_t - log2s * kLn2;
            logprobs[r] = lp;
        }
        if (entropy) entropy[r] = h;
        if (stats) {
            stats[4 * r] = m;
            stats[4 * r + 1] = log2s;
            stats[4 * r + 2] = h;
        }
    }
    uint64_t last = ~0ull;
    for (int k = 0; k < top_k; ++k) {
        uint64_t best = 0;
        for (int j = tid; j < V; j += kThreads) {
            const uint64_t key = order_key(to_float(z[j]), j);
            if (key < last && key > best) best = key;
        }
        best = block_reduce(best, umaximum, su);
        last = best;
        if (tid == 0) {
            const uint32_t id = 0xFFFFFFFFu - (uint32_t)best;
            top_ids[r * top_k + k] = id;
            top_logprobs[r * top_k + k] = (to_float(z[id]) - m) * inv_t - log2s * kLn2;
        }
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void token_logprobs_grad_kernel(
    Rows rows, const int64_t* __restrict__ labels, int64_t ignore, float c, float inv_t, const float* __restrict__ stats,
    const float* __restrict__ g_logprobs, const float* __restrict__ g_entropy, int top_k, const int64_t* __restrict__ top_ids,
    const float* __restrict__ g_top, T* __restrict__ grad) {
    const int64_t r = blockIdx.x;
    const int tid = threadIdx.x, V = rows.vocab;
    T* __restrict__ out = grad + r * V;
    const int64_t label = labels ? labels[r] : -1;
    if (labels && label == ignore) {
        for (int j = tid; j < V; j += kThreads) out[j] = from_float<T>(0.f);
        return;
    }
    const T* __restrict__ z = row_of<T>(rows, r);
    const float m = stats[4 * r], log2s = stats[4 * r + 1], h = stats[4 * r + 2];
    float gl = (labels && g_logprobs) ? g_logprobs[r] : 0.f;
    if (labels && g_logprobs && (label < 0 || label >= V)) gl = NAN;
    const float gh = g_entropy ? g_entropy[r] : 0.f;
    float total = gl;
    if (g_top)
        for (int k = 0; k < top_k; ++k) total += g_top[r * top_k + k];
    for (int j = tid; j < V; j += kThreads) {
        const float y = (to_float(z[j]) - m) * c - log2s;
        const float p = exp2f(y);
        float d = -p * total;
        if (gh != 0.f) d -= gh * p * (fmaxf(y, -200.f) * kLn2 + h);
        if (j == label) d += gl;
        if (g_top)
            for (int k = 0; k < top_k; ++k)
                if (top_ids[r * top_k + k] == j) d += g_top[r * top_k + k];
        out[j] = from_float<T>(d * inv_t);
    }
}

// Softmax of the kept teacher entries (ids >= 0) at the temperature, in q; returns their sum (1, or 0 if none is kept).
__device__ float teacher_softmax(const int64_t* ids, const float* logits, int K, float inv_t, float* q, float* lnq) {
    float m = -INFINITY;                       // natural logarithms outside the sums: log2(e) times the lowest value is -inf
    for (int k = 0; k < K; ++k)
        if (ids[k] >= 0) m = fmaxf(m, logits[k]);
    if (m == -INFINITY) {
        for (int k = 0; k < K; ++k) q[k] = lnq[k] = 0.f;
        return 0.f;
    }
    float s = 0.f;
    for (int k = 0; k < K; ++k)
        if (ids[k] >= 0) s += expf((logits[k] - m) * inv_t);
    const float lns = logf(s);
    for (int k = 0; k < K; ++k) {
        lnq[k] = ids[k] >= 0 ? (logits[k] - m) * inv_t - lns : 0.f;
        q[k] = ids[k] >= 0 ? expf(lnq[k]) : 0.f;
    }
    return 1.f;
}

struct Distill {
    const int64_t* labels;
    const int64_t* ids;
    const float* logits;
    int64_t ignore;
    int K;
    float tau, alpha;
};

// What one row's gradient is multiplied by.
__device__ inline float row_weight(const float* factor, const float* g, const float* g_row, int64_t r) {
    float w = factor ? factor[0] : 1.f;
    if (g) w *= g[0];
    if (g_row) w *= g_row[r];
    return w;
}

template <typename T>
__device__ void distill_grad_row(const T* z, T* out, int V, const Distill& a, int64_t r, float m, float log2s1, float log2st,
                                 const float* q, float mass, float weight) {
    const float c1 = (float)kLog2e, ct = (float)(kLog2e / a.tau);
    const float wt = weight * a.alpha * a.tau, w1 = weight * (1.f - a.alpha);
    const int64_t label = a.labels[r];
    for (int j = threadIdx.x; j < V; j += kThreads) {
        const float x = to_float(z[j]) - m;
        float d = 0.f;
        if (a.alpha != 0.f && mass != 0.f) {
            d = wt * exp2f(x * ct - log2st);
            for (int k = 0; k < a.K; ++k)
                if (a.ids[r * a.K + k] == j) d -= wt * q[k];
        }
        if (a.alpha != 1.f) d += w1 * (exp2f(x * c1 - log2s1) - (j == label ? 1.f : 0.f));
        out[j] = from_float<T>(d);
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void distill_kernel(Rows rows, Distill a, const float* __restrict__ factor,
                                                           float* __restrict__ losses, float* __restrict__ stats, T* __restrict__ grad) {
    __shared__ float sf[kThreads / 64];
    __shared__ float q[STTFE_MAX_TOP], lnq[STTFE_MAX_TOP], mass_s;
    const int64_t r = blockIdx.x;
    const int tid = threadIdx.x, V = rows.vocab;
    const int64_t label = a.labels[r];
    T* out = grad ? grad + r * V : nullptr;
    if (label == a.ignore) {
        if (tid == 0) losses[r] = 0.f;
        if (out)
            for (int j = tid; j < V; j += kThreads) out[j] = from_float<T>(0.f);
        return;
    }
    const T* __restrict__ z = row_of<T>(rows, r);
    const float c1 = (float)kLog2e, ct = (float)(kLog2e / a.tau);
    float m = -INFINITY;
    for (int j = tid; j < V; j += kThreads) m = fmaxf(m, to_float(z[j]));
    m = block_reduce(m, fmaximum, sf);
    float s1 = 0.f, st = 0.f;
    for (int j = tid; j < V; j += kThreads) {
        const float x = to_float(z[j]) - m;
        s1 += exp2f(x * c1);
        st += exp2f(x * ct);
    }
    s1 = block_reduce(s1, fadd, sf);
    st = block_reduce(st, fadd, sf);
    float log2s1 = log2f(s1), log2st = log2f(st);
    if (tid == 0) {
        const int64_t* ids = a.ids + r * a.K;
        const float mass = teacher_softmax(ids, a.logits + r * a.K, a.K, 1.f / a.tau, q, lnq);
        float loss = 0.f;
        bool bad = label < 0 || label >= V;
        for (int k = 0; k < a.K; ++k) bad |= ids[k] >= V;
        if (a.alpha != 0.f && mass != 0.f && !bad) {
            float kl = 0.f;
            for (int k = 0; k < a.K; ++k)
                if (q[k] > 0.f) kl += q[k] * (lnq[k] - ((to_float(z[ids[k]]) - m) / a.tau - log2st * kLn2));
            loss = a.alpha * a.tau * a.tau * kl;
        }
        if (a.alpha != 1.f && !bad) loss -= (1.f - a.alpha) * (to_float(z[label]) - m - log2s1 * kLn2);
        losses[r] = bad ? NAN : loss;
        mass_s = bad ? NAN : mass;
        if (stats) {
            stats[4 * r] = m;
            stats[4 * r + 1] = bad ? NAN : log2s1;
            stats[4 * r + 2] = bad ? NAN : log2st;
        }
    }
    __syncthreads();
    if (out)
        distill_grad_row<T>(z, out, V, a, r, m, log2s1, log2st, q, mass_s, mass_s != mass_s ? NAN : row_weight(factor, nullptr, nullptr, r));
}

template <typename T>
__global__ __launch_bounds__(kThreads) void distill_grad_kernel(Rows rows, Distill a, const float* __restrict__ stats,
                                                                const float* __restrict__ factor, const float* __restrict__ g,
                                                                const float* __restrict__ g_row, T* __restrict__ grad) {
    __shared__ float q[STTFE_MAX_TOP], lnq[STTFE_MAX_TOP], mass_s;
    const int64_t r = blockIdx.x;
    const int tid = threadIdx.x, V = rows.vocab;
    T* out = grad + r * V;
    if (a.labels[r] == a.ignore) {
        for (int j = tid; j < V; j += kThreads) out[j] = from_float<T>(0.f);
        return;
    }
    if (tid == 0) mass_s = teacher_softmax(a.ids + r * a.K, a.logits + r * a.K, a.K, 1.f / a.tau, q, lnq);
    __syncthreads();
    distill_grad_row<T>(row_of<T>(rows, r), out, V, a, r, stats[4 * r], stats[4 * r + 1], stats[4 * r + 2], q, mass_s,
                        row_weight(factor, g, g_row, r));
}

// factor = weight (sum) or weight / number of rows that count (mean)
__global__ __launch_bounds__(kThreads) void distill_factor_kernel(const int64_t* __restrict__ labels, int64_t ignore, int64_t rows,
                                                                  float weight, int mean, float* __restrict__ factor) {
    __shared__ uint64_t su[kThreads / 64];
    uint64_t n = 0;
    for (int64_t r = threadIdx.x; r < rows; r += kThreads) n += labels[r] != ignore;
    n = block_reduce(n, [](uint64_t x, uint64_t y) { return x + y; }, su);
    if (threadIdx.x == 0) factor[0] = mean ? (float)((double)weight / (double)(n ? n : 1)) : weight;
}

// total = factor * sum of the rows' losses, in 64 bits and in a fixed order
__global__ __launch_bounds__(kThreads) void distill_total_kernel(const float* __restrict__ losses, int64_t rows,
                                                                 const float* __restrict__ factor, float* __restrict__ total) {
    __shared__ double sd[kThreads / 64];
    double s = 0.0;
    for (int64_t r = threadIdx.x; r < rows; r += kThreads) s += (double)losses[r];
    s = block_reduce(s, [](double x, double y) { return x + y; }, sd);
    if (threadIdx.x == 0) total[0] = (float)(s * (double)factor[0]);
}

// Gradient made for an upstream gradient of 1: nothing to do if that is what it was.
template <typename T>
__global__ __launch_bounds__(kThreads) void rescale_kernel(T* __restrict__ grad, int64_t n, const float* __restrict__ g) {
    const float f = g[0];
    if (f == 1.f) return;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kThreads)
        grad[i] = from_float<T>(to_float(grad[i]) * f);
}

int check_rows(const void* logits, int dtype, int64_t outer, int64_t inner, int64_t stride_outer, int64_t stride_inner, int vocab) {
    if (outer < 0 || inner < 0 || vocab < 1 || stride_outer < 0 || stride_inner < 0) return STTFE_E_INVALID_ARG;
    if (dtype != STTFE_DTYPE_F32 && dtype != STTFE_DTYPE_F16 && dtype != STTFE_DTYPE_BF16) return STTFE_E_INVALID_ARG;
    if (inner > 0 && outer > STTFE_MAX_ROWS / inner) return STTFE_E_UNSUPPORTED;
    if (vocab > STTFE_MAX_VOCAB) return STTFE_E_UNSUPPORTED;
    if (outer * inner > 0 && (!logits || ((uintptr_t)logits & (dtype == STTFE_DTYPE_F32 ? 3 : 1)))) return STTFE_E_INVALID_ARG;
    return STTFE_OK;
}

bool positive(float x) { return x > 0.f && x <= 3.4e38f; }

}  // namespace
}  // namespace sttfe

using namespace sttfe;

#define STTFE_BY_DTYPE(dtype, CALL)                                   \
    do {                                                              \
        if ((dtype) == STTFE_DTYPE_F32) { using T = float; CALL; }    \
        else if ((dtype) == STTFE_DTYPE_F16) { using T = __half; CALL; } \
        else { using T = __hip_bfloat16; CALL; }                      \
    } while (0)

extern "C" int sttfe_token_logprobs_workspace_bytes(int64_t rows, int vocab, int dtype, int top_k, size_t* bytes) {
    if (!bytes || rows < 0 || vocab < 1 || top_k < 0 || top_k > STTFE_MAX_TOP || top_k > vocab) return STTFE_E_INVALID_ARG;
    if (dtype != STTFE_DTYPE_F32 && dtype != STTFE_DTYPE_F16 && dtype != STTFE_DTYPE_BF16) return STTFE_E_INVALID_ARG;
    *bytes = 0;
    return STTFE_OK;
}

extern "C" int sttfe_token_logprobs(const void* logits, int dtype, int64_t outer, int64_t inner, int64_t stride_outer,
                                    int64_t stride_inner, int vocab, const int64_t* labels, int64_t ignore_index,
                                    float temperature, int top_k, float* logprobs, float* entropy, float* stats,
                                    int64_t* top_ids, float* top_logprobs, void* workspace, size_t workspace_bytes, void* stream_) {
    int rc = check_rows(logits, dtype, outer, inner, stride_outer, stride_inner, vocab);
    if (rc != STTFE_OK) return rc;
    if (!positive(temperature) || top_k < 0 || top_k > STTFE_MAX_TOP || top_k > vocab) return STTFE_E_INVALID_ARG;
    const int64_t n = outer * inner;
    if (n == 0) return STTFE_OK;
    if ((logprobs && !labels) || (top_k > 0 && (!top_ids || !top_logprobs))) return STTFE_E_INVALID_ARG;
    size_t need = 0;
    rc = sttfe_token_logprobs_workspace_bytes(n, vocab, dtype, top_k, &need);
    if (rc != STTFE_OK) return rc;
    if (workspace_bytes < need || (need && !workspace)) return STTFE_E_WORKSPACE;
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    (void)hipGetLastError();
    const Rows rows{logits, inner, stride_outer, stride_inner, vocab};
    const float c = (float)(kLog2e / (double)temperature), inv_t = (float)(1.0 / (double)temperature);
    {
        ScopedTiming t(kTimeTokenLogprobs, stream);
        STTFE_BY_DTYPE(dtype, hipLaunchKernelGGL(token_logprobs_kernel<T>, dim3((unsigned)n), dim3(kThreads), 0, stream, rows, labels,
                                                 ignore_index, c, inv_t, top_k, logprobs, entropy, stats, top_ids, top_logprobs));
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
    if (!positive(temperature) || top_k < 0 || top_k > STTFE_MAX_TOP || top_k > vocab) return STTFE_E_INVALID_ARG;
    const int64_t n = outer * inner;
    if (n == 0) return STTFE_OK;
    if (!stats || !grad || (g_logprobs && !labels) || (g_top && (top_k == 0 || !top_ids))) return STTFE_E_INVALID_ARG;
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    (void)hipGetLastError();
    const Rows rows{logits, inner, stride_outer, stride_inner, vocab};
    const float c = (float)(kLog2e / (double)temperature), inv_t = (float)(1.0 / (double)temperature);
    {
        ScopedTiming t(kTimeTokenLogprobsGrad, stream);
        STTFE_BY_DTYPE(dtype, hipLaunchKernelGGL(token_logprobs_grad_kernel<T>, dim3((unsigned)n), dim3(kThreads), 0, stream, rows, labels,
                                                 ignore_index, c, inv_t, stats, g_logprobs, g_entropy, top_k, top_ids, g_top,
                                                 static_cast<T*>(grad)));
    }
    if (hip_failed(hipGetLastError(), "token logprobs gradient kernel launch")) return STTFE_E_LAUNCH;
    return STTFE_OK;
}

static int check_distill(const int64_t* labels, const int64_t* ids, const float* teacher, int K, float tau, float alpha) {
    if (!labels || !ids || !teacher || K < 1 || K > STTFE_MAX_TOP || !positive(tau) || !(alpha >= 0.f && alpha <= 1.f))
        return STTFE_E_INVALID_ARG;
    return STTFE_OK;
}

extern "C" int sttfe_distill_workspace_bytes(int64_t rows, int vocab, int dtype, size_t* bytes) {
    if (!bytes || rows < 0 || vocab < 1) return STTFE_E_INVALID_ARG;
    if (dtype != STTFE_DTYPE_F32 && dtype != STTFE_DTYPE_F16 && dtype != STTFE_DTYPE_BF16) return STTFE_E_INVALID_ARG;
    *bytes = 0;
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
        if (!losses) return STTFE_E_INVALID_ARG;
    }
    if (n == 0 && reduction == STTFE_REDUCE_NONE) return STTFE_OK;
    size_t need = 0;
    rc = sttfe_distill_workspace_bytes(n, vocab, dtype, &need);
    if (rc != STTFE_OK) return rc;
    if (workspace_bytes < need || (need && !workspace)) return STTFE_E_WORKSPACE;
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    (void)hipGetLastError();
    const Rows rows{logits, inner, stride_outer, stride_inner, vocab};
    const Distill a{labels, teacher_ids, teacher_logits, ignore_index, teacher_k, temperature, alpha};
    if (reduction != STTFE_REDUCE_NONE)
        hipLaunchKernelGGL(distill_factor_kernel, dim3(1), dim3(kThreads), 0, stream, labels, ignore_index, n, weight,
                           reduction == STTFE_REDUCE_MEAN ? 1 : 0, factor);
    if (n > 0) {
        ScopedTiming t(kTimeDistill, stream);
        STTFE_BY_DTYPE(dtype, hipLaunchKernelGGL(distill_kernel<T>, dim3((unsigned)n), dim3(kThreads), 0, stream, rows, a,
                                                 reduction != STTFE_REDUCE_NONE ? factor : nullptr, losses, stats,
                                                 static_cast<T*>(grad)));
    }
    if (reduction != STTFE_REDUCE_NONE)
        hipLaunchKernelGGL(distill_total_kernel, dim3(1), dim3(kThreads), 0, stream, losses, n, factor, total);
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
    if (!stats || !grad) return STTFE_E_INVALID_ARG;
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    (void)hipGetLastError();
    const Rows rows{logits, inner, stride_outer, stride_inner, vocab};
    const Distill a{labels, teacher_ids, teacher_logits, ignore_index, teacher_k, temperature, alpha};
    {
        ScopedTiming t(kTimeDistillGrad, stream);
        STTFE_BY_DTYPE(dtype, hipLaunchKernelGGL(distill_grad_kernel<T>, dim3((unsigned)n), dim3(kThreads), 0, stream, rows, a, stats,
                                                 factor, g, g_rows, static_cast<T*>(grad)));
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
    const int64_t want = (count + kThreads - 1) / kThreads;
    const unsigned blocks = (unsigned)(want < 2048 ? want : 2048);
    STTFE_BY_DTYPE(dtype, hipLaunchKernelGGL(rescale_kernel<T>, dim3(blocks), dim3(kThreads), 0, stream, static_cast<T*>(grad), count, g));
    if (hip_failed(hipGetLastError(), "gradient rescale kernel launch")) return STTFE_E_LAUNCH;
    return STTFE_OK;
}
