// What token_objectives.hip (arguments, plans) and token_objectives.inc (kernels, compiled once a type) share.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/sttfe.h"

namespace sttfe {

constexpr int kMaxWaves = 8, kMaxVpt = 16;       // the largest team: waves, and 16-byte vectors a thread holds
// Whether a team that walks through rows loads the next one ahead. With alternatives to find it does not: the registers are worth
// more as a second team on the CU, whose work fills the first one's exchanges (10240 x 50021 bf16, 16 alternatives: 0.35 ms
// ahead, 0.28 ms two teams; without alternatives 0.18 ms ahead, 0.19 ms two teams, with the entropy 0.20 against 0.21).
constexpr bool kScoreAhead(bool top) { return !top; }
constexpr bool kDistillAhead = true;
constexpr int kWavesPerSimd(int vpt, bool ahead) { return vpt >= 16 && ahead ? 2 : 4; }
// Alternatives of short rows: more waves in fewer registers (100000 x 2000 bf16, 16 alternatives: 0.19 ms with 4, 0.15 with 6).
constexpr int kScoreWaves(int waves, int vpt, bool top) { return top && waves == 1 ? 6 : kWavesPerSimd(vpt, kScoreAhead(top)); }
constexpr int kGroups = 256;                     // groups of elements whose maxima bound the alternatives
constexpr int kMaxSegs = 64;                     // segments of a row: one lane each when they are joined
constexpr float kLn2 = 0.693147180559945309f;
constexpr double kLog2e = 1.442695040888963407;

using half_t = _Float16;
using bf16_t = __bf16;
struct Rows {                      // row r = (r / inner, r % inner)
    const void* base;
    uint32_t inner;
    int64_t stride_outer, stride_inner;
    int vocab, segs, seg_len;      // a row is cut into segs segments of seg_len elements (the last may be shorter)
};

constexpr double kClimb = 4.0;     // bits by which an element may exceed the reference of a wave's sums
struct Score {
    const int64_t* labels;
    int64_t ignore;
    float c, inv_t, climb;                       // log2(e) / T, 1 / T; kClimb / c
    int top_k;
    float *logprobs, *entropy, *stats;
    int64_t* top_ids;
    float* top_logprobs;
    float4* parts;                 // segments > 1: [row][segment] {m, S, W, -}
    uint64_t* keys;                //               [row][segment][top_k], falling
    uint32_t rows;
    bool dealt;
};

struct ScoreGrad {
    const int64_t* labels;
    int64_t ignore;
    float c, inv_t;
    const float *stats, *g_logprobs, *g_entropy;
    int top_k;
    const int64_t* top_ids;
    const float* g_top;
};

// Softmaxes a row needs: one (temperature 1, or only one of the two terms), two, or two of which the second is the square
// of the first (temperature 2: 2^(y) = (2^(y / 2))^2 saves an exponential of two).
enum Mode { kOne = 0, kTwo = 1, kSquare = 2 };

struct Distill {
    const int64_t* labels;
    const int64_t* ids;
    const float* logits;
    int64_t ignore;
    int K;
    float tau, inv_tau, alpha, c, c1, climb;     // c: of the first softmax, c1: of the second (or of the only one)
    bool teacher, label;                         // which terms there are
};

__host__ __device__ inline float mean_factor(float weight, int rows) { return (float)((double)weight / (double)(rows ? rows : 1)); }
constexpr int kCountHere = 1024;   // up to this many rows a mean's teams count the rows themselves: a launch less
struct Out {
    const float* factor;           // what the gradient is multiplied by; NULL: by weight, or (mean) weight / rows that count
    float weight;
    bool mean;
    float *losses, *stats;
    float4* parts;
    uint32_t rows;
    bool dealt;
};

constexpr int kGradWaves = 4, kGradVpt = 8;      // a gradient kernel's team, on a segment of at most 2048 vectors

// ---------------------------------------------------------------------------------- which team takes a row
// Limits of a launch (2^31 blocks, 2^32 threads): a team of one or two waves a row at 2^24 rows is 2^31 threads, longer rows are
// dealt; the gradients' kernels go in several launches.
static_assert((int64_t)STTFE_MAX_ROWS * 64 * 2 < (1ll << 32), "a team a row");

struct Plan {
    int team, segs, seg_len;
};

inline int elem_bytes(int dtype) { return dtype == STTFE_DTYPE_F32 ? 4 : 2; }

// Teams: waves and vectors a thread.  The smallest that holds a row in registers is taken; a row too long for the largest is cut
// into equal segments.
constexpr int kTeams = 5, kTeamWaves[kTeams] = {1, 2, 4, 4, kMaxWaves}, kTeamVpt[kTeams] = {4, 8, 8, 16, kMaxVpt};
inline Plan row_plan(int vocab, int dtype) {
    const int e = 16 / elem_bytes(dtype);
    for (int t = 0; t < kTeams; ++t)
        if (vocab / e <= kTeamVpt[t] * 64 * kTeamWaves[t]) return {t, 1, vocab};
    static_assert(STTFE_MAX_VOCAB / 4 <= kMaxSegs * kMaxVpt * 64 * kMaxWaves, "a row's segments are joined by one wave");
    const int cap = kMaxVpt * 64 * kMaxWaves * e;      // a multiple of 64: so is a segment's length, and not above it
    const int segs = (vocab + cap - 1) / cap;
    const int len = ((vocab + segs - 1) / segs + 63) / 64 * 64;
    return {kTeams - 1, (vocab + len - 1) / len, len};
}
// Gradient kernels have nothing to join: a team of kGradWaves a segment.
inline Plan grad_plan(int vocab, int dtype) {
    const int cap = kGradVpt * 64 * kGradWaves * (16 / elem_bytes(dtype));
    const int segs = (vocab + cap - 1) / cap;
    const int len = ((vocab + segs - 1) / segs + 63) / 64 * 64;
    return {-1, (vocab + len - 1) / len, len};
}

// The launches, by the type of the logits: instantiated in token_objectives_f32.hip, _f16.hip and _bf16.hip.
template <typename T>
struct Launch {
    static void score(const Plan& plan, const Rows& rows, const Score& a, unsigned blocks, bool entropy, hipStream_t stream);
    static void score_join(const Rows& rows, const Score& a, unsigned n, hipStream_t stream);
    static void score_grad(const Rows& rows, const ScoreGrad& a, unsigned n, T* grad, hipStream_t stream);
    static void distill(const Plan& plan, const Rows& rows, const Distill& a, Mode mode, unsigned blocks, const Out& o, T* grad,
                        hipStream_t stream);
    static void distill_join(const Rows& rows, const Distill& a, Mode mode, const float4* parts, float* losses, float* stats, unsigned n,
                             hipStream_t stream);
    static void distill_grad(const Rows& rows, const Distill& a, Mode mode, const float* stats, const float* factor, const float* g,
                             const float* g_rows, unsigned n, T* grad, hipStream_t stream);
    static void rescale(T* grad, int64_t count, const float* g, hipStream_t stream);
};

}  // namespace sttfe
