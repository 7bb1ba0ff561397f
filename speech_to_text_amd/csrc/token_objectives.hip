// Token objectives: label log probabilities with entropy and top alternatives, and distillation from a teacher's top
// logits, forward and backward (include/sttfe.h, "token objectives").
//
// One row of logits z[0 .. V) per label position; T = temperature, c = log2(e) / T, all sums in float32:
//   m = max z,  S = sum 2^(c (z_j - m)),  log2 p_j = c (z_j - m) - log2 S,  H = -sum p_j ln p_j.
//
// What bounds these kernels is the one read of the logits (and the one write of their gradient), with the vector ALU not
// far behind: a 50 k row of bf16 is 104 KB, 4.4 us of a CU's share of the memory rate, and an exponential, an unpacking, a
// multiply-add, a sum and half a maximum per element are 3.1 us of its vector ALU.  Hence:
//   * a row (or a segment of a longer one) is read once, into the registers of a team of 1 - 16 waves, 16 bytes a lane and
//     load, all loads in flight before the first use; the maximum, the sums, the search for the alternatives and the
//     gradient are made from the registers;
//   * every thread takes the exponentials against the maximum of ITS elements, so that one exchange through the LDS per row is
//     all the softmax costs (maximum, sums and what the alternatives need are joined there);
//   * rows start at any element (an odd vocabulary in bf16 leaves them at 2 bytes): loads and stores are 16 bytes wide at
//     element alignment, only the last vector of a row is taken element by element.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/sttfe.h"
#include "timing.h"

namespace sttfe {
namespace {

constexpr int kVpt = 8;                          // 16-byte vectors a thread holds
constexpr int kMaxWaves = 16;
constexpr int kCand = 512;                       // alternatives' candidates a team sorts at once
constexpr int kMaxSegs = 64;                     // segments of a row: one lane each when they are joined
constexpr float kLn2 = 0.693147180559945309f;
constexpr double kLog2e = 1.442695040888963407;

using half_t = _Float16;
using bf16_t = __bf16;
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef half_t f16x2 __attribute__((ext_vector_type(2)));
typedef bf16_t bf16x2 __attribute__((ext_vector_type(2)));

struct Rows {                      // row r = (r / inner, r % inner)
    const void* base;
    uint32_t inner;
    int64_t stride_outer, stride_inner;
    int vocab, segs, seg_len;      // a row is cut into segs segments of seg_len elements (the last may be shorter)
};

template <typename T>
__device__ inline const T* row_of(const Rows& a, uint32_t r) {
    return static_cast<const T*>(a.base) + (int64_t)(r / a.inner) * a.stride_outer + (int64_t)(r % a.inner) * a.stride_inner;
}

template <typename T> struct Vec {               // elements of one 16-byte vector
    static constexpr int n = 8;
};
template <> struct Vec<float> {
    static constexpr int n = 4;
};

__device__ inline void unpack(const uint4& v, float (&x)[4], float) {
    x[0] = __uint_as_float(v.x), x[1] = __uint_as_float(v.y), x[2] = __uint_as_float(v.z), x[3] = __uint_as_float(v.w);
}
__device__ inline void unpack(const uint4& v, float (&x)[8], bf16_t) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
}
__device__ inline void unpack(const uint4& v, float (&x)[8], half_t) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const f16x2 h = __builtin_bit_cast(f16x2, w[i]);
        x[2 * i] = (float)h.x;
        x[2 * i + 1] = (float)h.y;
    }
}
__device__ inline uint4 pack(const float (&x)[4], float) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
}
__device__ inline uint4 pack(const float (&x)[8], bf16_t) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){x[2 * i], x[2 * i + 1]}, bf16x2));
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ inline uint4 pack(const float (&x)[8], half_t) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){x[2 * i], x[2 * i + 1]}, f16x2));
    return make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T> __device__ inline uint4 all_minus_inf();
template <> __device__ inline uint4 all_minus_inf<float>() { return make_uint4(0xFF800000u, 0xFF800000u, 0xFF800000u, 0xFF800000u); }
template <> __device__ inline uint4 all_minus_inf<half_t>() { return make_uint4(0xFC00FC00u, 0xFC00FC00u, 0xFC00FC00u, 0xFC00FC00u); }
template <> __device__ inline uint4 all_minus_inf<bf16_t>() { return make_uint4(0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u); }

// ---------------------------------------------------------------------------------- reductions over a wave and a team
template <int CTRL, int ROW_MASK>
__device__ inline float dpp(float x, float none) {
    return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(none), __float_as_int(x), CTRL, ROW_MASK, 0xf, false));
}
template <typename F>
__device__ inline float wave_reduce(float x, float none, F f) {       // in every lane
    x = f(x, dpp<0x111, 0xf>(x, none));          // lanes of a row shifted by 1, 2, 4, 8: lane 15 has the row's result
    x = f(x, dpp<0x112, 0xf>(x, none));
    x = f(x, dpp<0x114, 0xf>(x, none));
    x = f(x, dpp<0x118, 0xf>(x, none));
    x = f(x, dpp<0x142, 0xa>(x, none));          // lane 15 to the next row, lane 31 to the upper half: lane 63 has it all
    x = f(x, dpp<0x143, 0xc>(x, none));
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}
__device__ inline float add2(float a, float b) { return a + b; }
__device__ inline float max2(float a, float b) { return fmaxf(a, b); }
__device__ inline float wave_sum(float x) { return wave_reduce(x, 0.f, add2); }
__device__ inline float wave_max(float x) { return wave_reduce(x, -INFINITY, max2); }

// The largest of WAVES neighbouring lanes, in all of them: a team has 64 such groups whatever its size.
template <int WAVES>
__device__ inline float group_max(float x) {
    if constexpr (WAVES >= 4) {
        x = fmaxf(x, dpp<0xB1, 0xf>(x, x));      // quads: lanes 1 0 3 2, then 2 3 0 1
        x = fmaxf(x, dpp<0x4E, 0xf>(x, x));
    }
    if constexpr (WAVES >= 8) x = fmaxf(x, dpp<0x141, 0xf>(x, x));      // half rows mirrored
    if constexpr (WAVES >= 16) x = fmaxf(x, dpp<0x140, 0xf>(x, x));     // rows mirrored
    return x;
}

// LDS writes before, reads after; global loads and stores in flight stay in flight (__syncthreads would wait for them).
template <int WAVES>
__device__ inline void team_sync() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if constexpr (WAVES > 1) __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Order of the alternatives: value falling (NaN before everything, as torch.topk has it; -0 equals +0), index rising.
__device__ inline uint32_t order_bits(float x) {
    uint32_t b = __float_as_uint(x + 0.0f);
    b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return x != x ? 0xFFFFFFFEu : b;             // above +inf, below the start of a falling search
}
__device__ inline float from_order_bits(uint32_t b) {
    return __uint_as_float((b & 0x80000000u) ? (b & 0x7FFFFFFFu) : ~b);     // 0xFFFFFFFE: a NaN
}
__device__ inline uint64_t order_key(float x, int index) {
    return ((uint64_t)order_bits(x) << 32) | (uint32_t)(0xFFFFFFFFu - (uint32_t)index);
}

// The k-th largest of the 64 lanes' values (k in 1 .. 64), rounded down in the bits below LOW: bit by bit from the top.
template <int LOW>
__device__ inline float kth_of_wave(float x, int k) {
    const uint32_t b = order_bits(x);
    uint64_t active = ~0ull;
    uint32_t res = 0;
#pragma unroll
    for (int bit = 31; bit >= LOW; --bit) {
        const uint64_t up = __ballot((b >> bit) & 1u) & active;
        const int n = __popcll(up);
        if (n >= k) {
            active = up;
            res |= 1u << bit;
        } else {
            k -= n;
            active &= ~up;
        }
    }
    return from_order_bits(max(res, 0x007FFFFFu));     // not below -inf: that would be a NaN
}

// ---------------------------------------------------------------------------------- a segment of a row in registers
template <typename T, int WAVES>
struct Segment {
    static constexpr int E = Vec<T>::n, THREADS = 64 * WAVES;
    uint4 v[kVpt];
    float x_tail;                  // one element of the last, incomplete vector, in the first threads; -inf elsewhere
    int n, nv;                     // elements, whole vectors

    __device__ inline int index(int i, int e) const { return (i * THREADS + (int)threadIdx.x) * E + e; }
    __device__ inline int tail_index() const { return nv * E + (int)threadIdx.x; }
    __device__ inline bool whole(int i) const { return i * THREADS + (int)threadIdx.x < nv; }
    __device__ inline bool has_tail() const { return tail_index() < n; }

    // The vectors as they were loaded: what a phase unpacked is not kept in registers for the next.
    __device__ inline void again() {
#pragma unroll
        for (int i = 0; i < kVpt; ++i) asm volatile("" : "+v"(v[i].x), "+v"(v[i].y), "+v"(v[i].z), "+v"(v[i].w));
    }

    __device__ inline void load(const T* __restrict__ p, int n_) {
        n = n_;
        nv = n / E;
#pragma unroll
        for (int i = 0; i < kVpt; ++i) {
            v[i] = all_minus_inf<T>();
            if (whole(i)) __builtin_memcpy(&v[i], p + (int64_t)index(i, 0), 16);
        }
        x_tail = -INFINITY;
        if (has_tail()) x_tail = (float)p[tail_index()];
    }
};

// Exponentials are 2^(c (x - m)): the difference first.  A single multiply-add c x - round(c m) would save an instruction, but
// c m overflows where a row's maximum is the type's lowest value, and loses what a large common offset of the logits costs.
// A thread (or wave) with nothing but -inf takes them against 0; its sums count nothing.
__device__ inline float shift_of(float m) { return m == -INFINITY ? 0.f : m; }
// log2 of what sums against `from` are multiplied by to stand against `to` >= from
__device__ inline float rebase(float c, float from, float to) { return from == -INFINITY ? -INFINITY : (from - to) * c; }

// ---------------------------------------------------------------------------------- token_logprobs
struct Score {
    const int64_t* labels;
    int64_t ignore;
    float c, inv_t;
    int top_k;
    float *logprobs, *entropy, *stats;
    int64_t* top_ids;
    float* top_logprobs;
    float4* parts;                 // segments > 1: [row][segment] {m, S, W, -}
    uint64_t* keys;                //               [row][segment][top_k], falling
};

// What a row's numbers are, from its maximum and sums (S, W against c m itself).
__device__ inline void write_row(const Score& a, uint32_t r, int64_t label, int V, float x_label, float m, float s, float w) {
    const float log2s = __log2f(s), h = (log2s - w / s) * kLn2;
    if (a.logprobs) a.logprobs[r] = (label >= 0 && label < V) ? (x_label - m) * a.inv_t - log2s * kLn2 : NAN;
    if (a.entropy) a.entropy[r] = h;
    if (a.stats) *reinterpret_cast<float4*>(a.stats + 4 * (size_t)r) = make_float4(m, log2s, h, 0.f);
}
__device__ inline void write_alternative(const Score& a, uint32_t r, int k, uint64_t key, float m, float lns, bool nan) {
    a.top_ids[(size_t)r * a.top_k + k] = (int64_t)(0xFFFFFFFFu - (uint32_t)key);
    a.top_logprobs[(size_t)r * a.top_k + k] = nan ? NAN : (from_order_bits((uint32_t)(key >> 32)) - m) * a.inv_t - lns;
}

template <typename T, int WAVES, bool ENTROPY, bool TOP>
__global__ __launch_bounds__(64 * WAVES) void score_kernel(Rows rows, Score a) {
    constexpr int E = Vec<T>::n, THREADS = 64 * WAVES;
    __shared__ float part_m[WAVES], part_s[WAVES], part_w[WAVES], groups[TOP ? 64 : 1];
    __shared__ uint64_t cand[TOP ? kCand : 1], best[TOP ? WAVES : 1];
    __shared__ int n_cand;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t r = blockIdx.x / (uint32_t)rows.segs, seg = blockIdx.x % (uint32_t)rows.segs;
    const int V = rows.vocab;
    const int64_t label = a.labels ? a.labels[r] : 0;
    if (a.labels && label == a.ignore) {
        if (seg != 0) return;
        if (tid == 0) {
            if (a.logprobs) a.logprobs[r] = 0.f;
            if (a.entropy) a.entropy[r] = 0.f;
        }
        for (int k = tid; k < a.top_k; k += THREADS) {
            a.top_ids[(size_t)r * a.top_k + k] = -1;
            a.top_logprobs[(size_t)r * a.top_k + k] = -INFINITY;
        }
        return;
    }
    const int first = (int)seg * rows.seg_len;
    const T* __restrict__ z = row_of<T>(rows, r);
    Segment<T, WAVES> x;
    x.load(z + first, min(rows.seg_len, V - first));
    float x_label = 0.f;
    if (a.logprobs && rows.segs == 1 && label >= 0 && label < V) x_label = (float)z[label];
    if (TOP && tid == 0) n_cand = 0;

    float vec_max[kVpt], mt = x.x_tail;
#pragma unroll
    for (int i = 0; i < kVpt; ++i) {
        float f[E];
        unpack(x.v[i], f, T());
        float m = f[0];
#pragma unroll
        for (int e = 1; e < E; ++e) m = fmaxf(m, f[e]);
        vec_max[i] = m;
        mt = fmaxf(mt, m);
    }
    x.again();
    const float own = shift_of(mt);
    float s[2] = {0.f, 0.f}, w[2] = {0.f, 0.f};
    auto term = [&](float f, int e) {
        const float y = (f - own) * a.c;
        const float p = __builtin_amdgcn_exp2f(y);
        s[e & 1] += p;
        if (ENTROPY) w[e & 1] = fmaf(p, fmaxf(y, -200.f), w[e & 1]);       // 2^-200 is 0 here: so is the term of a -inf
    };
#pragma unroll
    for (int i = 0; i < kVpt; ++i) {
        if (i * THREADS >= x.nv) break;
        float f[E];
        unpack(x.v[i], f, T());
#pragma unroll
        for (int e = 0; e < E; ++e) term(f[e], e);
    }
    term(x.x_tail, 0);
    float st = s[0] + s[1], wt = w[0] + w[1];
    if (TOP) x.again();

    // one exchange: the wave's maximum and sums, the groups' maxima
    const float mw = wave_max(mt);
    {
        const float d = rebase(a.c, mt, mw), f = __builtin_amdgcn_exp2f(d);
        wt = f == 0.f ? 0.f : f * (wt + st * d);
        st *= f;
    }
    st = wave_sum(st);
    if (ENTROPY) wt = wave_sum(wt);
    if (lane == 0) {
        part_m[wave] = mw;
        part_s[wave] = st;
        part_w[wave] = wt;
    }
    if (TOP) {
        const float g = group_max<WAVES>(mt);
        if (tid % WAVES == 0) groups[tid / WAVES] = g;
    }
    team_sync<WAVES>();
    float m = mw, sum = st, wsum = wt;
    if constexpr (WAVES > 1) {                   // a lane a wave, in every wave
        const int o = lane % WAVES;
        const float pm = part_m[o];
        m = wave_max(pm);
        const float d = rebase(a.c, pm, m), f = lane < WAVES ? __builtin_amdgcn_exp2f(d) : 0.f;
        if (ENTROPY) wsum = wave_sum(f == 0.f ? 0.f : f * (part_w[o] + part_s[o] * d));
        sum = wave_sum(lane < WAVES ? part_s[o] * f : 0.f);
    }
    const float seen = sum;
    if (m == -INFINITY) sum = NAN;               // nothing but -inf (or NaN)
    const float lns = __log2f(sum) * kLn2;
    if (tid == 0) {
        if (rows.segs == 1)
            write_row(a, r, label, V, x_label, m, sum, ENTROPY ? wsum : 0.f);
        else
            a.parts[(size_t)r * rows.segs + seg] = make_float4(m, seen, wsum, 0.f);
    }
    if constexpr (TOP) {
        const bool nan = sum != sum;
        uint64_t* out = a.keys + ((size_t)r * rows.segs + seg) * a.top_k;
        auto put = [&](int k, uint64_t key) {
            if (rows.segs == 1)
                write_alternative(a, r, k, key, m, lns, nan);
            else
                out[k] = key;
        };
        // The top_k-th largest of the 64 groups' maxima is a bound: top_k elements at least are not below it.
        const float bound = kth_of_wave<sizeof(T) == 2 ? 13 : 0>(groups[lane], a.top_k);
        bool slow = nan;
        if (!slow) {
            auto push = [&](float f, int j) {
                const int at = atomicAdd(&n_cand, 1);
                if (at < kCand) cand[at] = order_key(f, first + j);
            };
            if (mt >= bound) {
#pragma unroll
                for (int i = 0; i < kVpt; ++i)
                    if (vec_max[i] >= bound && x.whole(i)) {
                        float f[E];
                        unpack(x.v[i], f, T());
#pragma unroll
                        for (int e = 0; e < E; ++e)
                            if (f[e] >= bound) push(f[e], x.index(i, e));
                    }
                if (x.x_tail >= bound && x.has_tail()) push(x.x_tail, x.tail_index());
            }
            team_sync<WAVES>();
            const int n = n_cand;
            slow = n > kCand;
            if (!slow)
                for (int j = tid; j < n; j += THREADS) {
                    const uint64_t key = cand[j];
                    int rank = 0;
                    for (int q = 0; q < n; ++q) rank += cand[q] > key;
                    if (rank < a.top_k) put(rank, key);
                }
        }
        if (slow) {
            // NaN, nothing but -inf, or more equal values than candidates fit: the largest key top_k times, from the row in the
            // cache; only the thread that had it looks again
            const T* __restrict__ zs = z + first;
            const int want = min(a.top_k, x.n);
            uint64_t mine = 0, last = ~0ull;
            auto look = [&]() {
                mine = 0;
                for (int j = tid; j < x.n; j += THREADS) {
                    const uint64_t key = order_key((float)zs[j], first + j);
                    if (key < last && key > mine) mine = key;
                }
            };
            look();
            for (int k = 0; k < want; ++k) {
                uint64_t b = mine;
#pragma unroll
                for (int d = 32; d > 0; d >>= 1) {
                    const uint64_t o = __shfl_xor((unsigned long long)b, d, 64);
                    b = o > b ? o : b;
                }
                team_sync<WAVES>();
                if (lane == 0) best[wave] = b;
                team_sync<WAVES>();
                b = best[0];
#pragma unroll
                for (int i = 1; i < WAVES; ++i) b = best[i] > b ? best[i] : b;
                last = b;
                if (tid == 0) put(k, b);
                if (mine == b) look();
            }
            if (rows.segs > 1)
                for (int k = want + tid; k < a.top_k; k += THREADS) out[k] = 0;
        } else if (rows.segs > 1) {
            for (int k = x.n + tid; k < a.top_k; k += THREADS) out[k] = 0;         // a segment shorter than top_k
        }
    }
}

// Joins the segments of a row: one wave a row, one lane a segment.
__global__ __launch_bounds__(64) void score_join_kernel(Rows rows, Score a, int dtype) {
    const uint32_t r = blockIdx.x;
    const int lane = threadIdx.x;
    const int64_t label = a.labels ? a.labels[r] : 0;
    if (a.labels && label == a.ignore) return;   // written by the first segment's team
    float4 p = make_float4(-INFINITY, 0.f, 0.f, 0.f);
    if (lane < rows.segs) p = a.parts[(size_t)r * rows.segs + lane];
    const float m = wave_max(p.x);
    const float d = m == -INFINITY ? NAN : rebase(a.c, p.x, m), f = __builtin_amdgcn_exp2f(d);
    const float w = wave_sum(f == 0.f ? 0.f : f * (p.z + p.y * d)), s = wave_sum(p.y * f);
    if (lane == 0) {
        float x = 0.f;
        if (a.logprobs && label >= 0 && label < rows.vocab) {
            if (dtype == STTFE_DTYPE_F32) x = row_of<float>(rows, r)[label];
            else if (dtype == STTFE_DTYPE_F16) x = (float)row_of<half_t>(rows, r)[label];
            else x = (float)row_of<bf16_t>(rows, r)[label];
        }
        write_row(a, r, label, rows.vocab, x, m, s, w);
    }
    if (a.top_k == 0) return;
    const float lns = __log2f(s) * kLn2;
    const uint64_t* list = a.keys + ((size_t)r * rows.segs + lane) * a.top_k;
    int at = 0;
    uint64_t head = lane < rows.segs ? list[0] : 0;
    for (int k = 0; k < a.top_k; ++k) {
        uint64_t b = head;
#pragma unroll
        for (int q = 32; q > 0; q >>= 1) {
            const uint64_t o = __shfl_xor((unsigned long long)b, q, 64);
            b = o > b ? o : b;
        }
        if (lane == 0) write_alternative(a, r, k, b, m, lns, s != s);
        if (head == b) {
            ++at;
            head = at < a.top_k ? list[at] : 0;
        }
    }
}

// ---------------------------------------------------------------------------------- what single elements get beside p_j
// A list of (element, value): the label's and the alternatives' own terms of a gradient.  A bit per vector tells its owner to
// look through the list, so that every element is rounded and written once.
template <int WAVES, int E>
struct Singles {
    static constexpr int kMost = STTFE_MAX_TOP + 1, kWords = kVpt * 64 * WAVES / 32;
    int id[kMost];
    float add[kMost];
    uint32_t bits[kWords];

    __device__ inline void clear() {
        for (int w = threadIdx.x; w < kWords; w += 64 * WAVES) bits[w] = 0;
    }
    // after clear() and a team_sync(); `at` counts from the segment's first element, outside of it: not here
    __device__ inline void set(int q, int64_t at, int n, float value) {
        const bool here = at >= 0 && at < n;
        id[q] = here ? (int)at : -1;
        add[q] = value;
        if (here) atomicOr(&bits[(int)at / E / 32], 1u << ((int)at / E & 31));
    }
    __device__ inline bool any(int vec) const { return (bits[vec >> 5] >> (vec & 31)) & 1u; }
    __device__ inline void apply(float (&d)[E], int base, int count, float scale_first, float scale_last) const {
        for (int q = 0; q < count; ++q) {
            const int o = id[q] - base;
            if (id[q] >= 0 && o >= 0 && o < E) {
                const float v = add[q] * (q == count - 1 ? scale_last : scale_first);
#pragma unroll
                for (int e = 0; e < E; ++e) d[e] += o == e ? v : 0.f;
            }
        }
    }
    __device__ inline float at(int j, int count, float scale_first, float scale_last) const {
        float v = 0.f;
        for (int q = 0; q < count; ++q)
            if (id[q] == j) v += add[q] * (q == count - 1 ? scale_last : scale_first);
        return v;
    }
};

constexpr int kGradWaves = 4;                    // a gradient kernel's team, on a segment of at most kVpt * 256 vectors

struct ScoreGrad {
    const int64_t* labels;
    int64_t ignore;
    float c, inv_t;
    const float *stats, *g_logprobs, *g_entropy;
    int top_k;
    const int64_t* top_ids;
    const float* g_top;
};

template <typename T>
__device__ inline void write_zeros(T* __restrict__ out, int n, int threads) {
    constexpr int E = Vec<T>::n;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    for (int i = threadIdx.x; i < n / E; i += threads) __builtin_memcpy(out + (size_t)i * E, &zero, 16);
    const int t = n / E * E + (int)threadIdx.x;
    if (t < n) out[t] = (T)0.f;
}

template <typename T>
__global__ __launch_bounds__(64 * kGradWaves) void score_grad_kernel(Rows rows, ScoreGrad a, T* __restrict__ grad) {
    constexpr int E = Vec<T>::n, THREADS = 64 * kGradWaves;
    __shared__ Singles<kGradWaves, E> one;
    const int tid = threadIdx.x;
    const uint32_t r = blockIdx.x / (uint32_t)rows.segs, seg = blockIdx.x % (uint32_t)rows.segs;
    const int V = rows.vocab, first = (int)seg * rows.seg_len, n = min(rows.seg_len, V - first);
    T* __restrict__ out = grad + (size_t)r * V + first;
    const int64_t label = a.labels ? a.labels[r] : -1;
    if (a.labels && label == a.ignore) {
        write_zeros(out, n, THREADS);
        return;
    }
    Segment<T, kGradWaves> x;
    x.load(row_of<T>(rows, r) + first, n);
    const float4 st = *reinterpret_cast<const float4*>(a.stats + 4 * (size_t)r);
    const float m = st.x, log2s = st.y, h = st.z;
    float gl = (a.labels && a.g_logprobs) ? a.g_logprobs[r] : 0.f;
    if (a.labels && a.g_logprobs && (label < 0 || label >= V)) gl = NAN;
    const float gh = a.g_entropy ? a.g_entropy[r] : 0.f;
    const int K = a.g_top ? a.top_k : 0;
    float total = gl;
    for (int k = 0; k < K; ++k) total += a.g_top[(size_t)r * K + k];
    one.clear();
    team_sync<kGradWaves>();
    for (int q = tid; q <= K; q += THREADS) {
        if (q < K)
            one.set(q, a.top_ids[(size_t)r * K + q] - first, n, a.g_top[(size_t)r * K + q]);
        else
            one.set(q, label - first, a.g_logprobs ? n : 0, gl);
    }
    team_sync<kGradWaves>();
    // d_j = p_j (a0 + b y_j), p = 2^y inv, ln p = (y - log2 S) ln 2
    const float inv = __builtin_amdgcn_exp2f(-log2s) * a.inv_t;
    const float b = -gh * kLn2, a0 = -total - gh * fmaf(-log2s, kLn2, h);
    auto all = [&](auto ent) {
        auto value = [&](float f) {
            const float y = (f - m) * a.c;
            const float p = __builtin_amdgcn_exp2f(y) * inv;
            return ent ? p * fmaf(b, fmaxf(y, -200.f), a0) : p * a0;
        };
#pragma unroll
        for (int i = 0; i < kVpt; ++i)
            if (x.whole(i)) {
                float f[E];
                unpack(x.v[i], f, T());
#pragma unroll
                for (int e = 0; e < E; ++e) f[e] = value(f[e]);
                const int base = x.index(i, 0);
                if (one.any(base / E)) one.apply(f, base, K + 1, a.inv_t, a.inv_t);
                const uint4 w = pack(f, T());
                __builtin_memcpy(out + base, &w, 16);
            }
        if (x.has_tail()) out[x.tail_index()] = (T)(value(x.x_tail) + one.at(x.tail_index(), K + 1, a.inv_t, a.inv_t));
    };
    if (gh != 0.f)
        all(std::true_type());
    else
        all(std::false_type());
}

// ---------------------------------------------------------------------------------- distillation
// Softmaxes a row needs: one (temperature 1, or only one of the two terms), two, or two of which the second is the square
// of the first (temperature 2: 2^(y) = (2^(y / 2))^2 saves an exponential of two).
enum Mode { kOne = 0, kTwo = 1, kSquare = 2 };

struct Distill {
    const int64_t* labels;
    const int64_t* ids;
    const float* logits;
    int64_t ignore;
    int K;
    float tau, inv_tau, alpha, c, c1;            // c: of the first softmax, c1: of the second (or of the only one)
    bool teacher, label;                         // which terms there are
};

// The teacher's entry of a lane: softmax over the kept ones.
struct Entry {
    int64_t id;
    float q, lnq, mass;                          // mass: 1, or 0 if the row keeps nothing
    bool bad;                                    // some id is not in the vocabulary
};
__device__ inline Entry teacher_entry(const Distill& a, uint32_t r, int V) {
    const int lane = threadIdx.x & 63;
    Entry e{-1, 0.f, 0.f, 0.f, false};
    float t = -INFINITY;
    if (lane < a.K) {
        e.id = a.ids[(size_t)r * a.K + lane];
        if (e.id >= 0) t = a.logits[(size_t)r * a.K + lane];
    }
    e.bad = __ballot(e.id >= V) != 0;
    if (e.id < 0 || e.id >= V) e.id = -1;
    const float m = wave_max(t);
    if (m == -INFINITY && __ballot(t != t) == 0) return e;
    e.mass = 1.f;
    const float d = (t - m) * a.inv_tau;
    const float s = wave_sum(t == -INFINITY ? 0.f : __expf(d));
    const float lns = __logf(s);
    e.lnq = t == -INFINITY ? 0.f : d - lns;
    e.q = t == -INFINITY ? 0.f : __expf(d) / s;
    return e;
}

// Loss of a row, by one wave; x: the student's logit at the lane's entry.
__device__ inline float row_loss(const Distill& a, const Entry& e, float x, float x_label, float m, float lnst, float lns1) {
    float loss = 0.f;
    if (a.teacher) {
        const float kl = wave_sum(e.q > 0.f || e.q != e.q ? e.q * (e.lnq - ((x - m) * a.inv_tau - lnst)) : 0.f);
        if (e.mass != 0.f) loss = a.alpha * a.tau * a.tau * kl;
    }
    if (a.label) loss -= (1.f - a.alpha) * (x_label - m - lns1);
    return loss;
}

template <typename T, int WAVES, int MODE, bool GRAD>
__global__ __launch_bounds__(64 * WAVES) void distill_kernel(Rows rows, Distill a, const float* __restrict__ factor,
                                                             float* __restrict__ losses, float* __restrict__ stats,
                                                             float4* __restrict__ parts, T* __restrict__ grad) {
    constexpr int E = Vec<T>::n, THREADS = 64 * WAVES;
    __shared__ float part_m[WAVES], part_s[WAVES], part_w[WAVES], mass_s, bad_s;
    __shared__ Singles<GRAD ? WAVES : 1, E> one;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t r = blockIdx.x / (uint32_t)rows.segs, seg = blockIdx.x % (uint32_t)rows.segs;
    const int V = rows.vocab;
    const int64_t label = a.labels[r];
    T* __restrict__ out = GRAD ? grad + (size_t)r * V : nullptr;
    if (label == a.ignore) {
        if (tid == 0 && seg == 0) losses[r] = 0.f;
        if (GRAD) write_zeros(out, V, THREADS);
        return;
    }
    const int first = (int)seg * rows.seg_len;
    const T* __restrict__ z = row_of<T>(rows, r);
    Segment<T, WAVES> x;
    x.load(z + first, min(rows.seg_len, V - first));
    const bool whole_row = rows.segs == 1, label_ok = label >= 0 && label < V;
    const float weight = GRAD && factor ? factor[0] : 1.f;
    Entry mine{-1, 0.f, 0.f, 0.f, false};
    float x_mine = 0.f, x_label = 0.f;
    if constexpr (GRAD) {
        one.clear();
        team_sync<WAVES>();
    }
    if (whole_row && wave == 0) {
        if (label_ok) x_label = (float)z[label];
        if (a.teacher) {
            mine = teacher_entry(a, r, V);
            if (mine.id >= 0) x_mine = (float)z[mine.id];
        } else {
            mine.bad = __ballot(lane < a.K && a.ids[(size_t)r * a.K + lane] >= V) != 0;
        }
        if constexpr (GRAD) {
            if (lane < a.K) one.set(lane, mine.id, a.teacher ? V : 0, mine.q);
            if (lane == 0) one.set(a.K, label, a.label ? V : 0, 1.f);
        }
        if (lane == 0) {
            mass_s = mine.mass;
            bad_s = (mine.bad || !label_ok) ? NAN : 1.f;
        }
    }

    float mt = x.x_tail;
#pragma unroll
    for (int i = 0; i < kVpt; ++i) {
        float f[E];
        unpack(x.v[i], f, T());
#pragma unroll
        for (int e = 0; e < E; ++e) mt = fmaxf(mt, f[e]);
    }
    x.again();
    const float own = shift_of(mt);
    float s[2] = {0.f, 0.f}, w[2] = {0.f, 0.f};
    auto term = [&](float f, int e) {
        const float d = f - own, p = __builtin_amdgcn_exp2f(d * a.c);
        s[e & 1] += p;
        if (MODE == kSquare) w[e & 1] = fmaf(p, p, w[e & 1]);
        if (MODE == kTwo) w[e & 1] += __builtin_amdgcn_exp2f(d * a.c1);
    };
#pragma unroll
    for (int i = 0; i < kVpt; ++i) {
        if (i * THREADS >= x.nv) break;
        float f[E];
        unpack(x.v[i], f, T());
#pragma unroll
        for (int e = 0; e < E; ++e) term(f[e], e);
    }
    term(x.x_tail, 0);
    const float mw = wave_max(mt);
    const float st = wave_sum((s[0] + s[1]) * __builtin_amdgcn_exp2f(rebase(a.c, mt, mw)));
    const float wt = MODE == kOne ? 0.f : wave_sum((w[0] + w[1]) * __builtin_amdgcn_exp2f(rebase(a.c1, mt, mw)));
    if (lane == 0) {
        part_m[wave] = mw;
        part_s[wave] = st;
        part_w[wave] = wt;
    }
    team_sync<WAVES>();
    if (GRAD) x.again();
    float m = mw, sum = st, sum1 = wt;
    if constexpr (WAVES > 1) {                   // a lane a wave, in every wave
        const int o = lane % WAVES;
        const float pm = part_m[o];
        m = wave_max(pm);
        sum = wave_sum(lane < WAVES ? part_s[o] * __builtin_amdgcn_exp2f(rebase(a.c, pm, m)) : 0.f);
        if (MODE != kOne) sum1 = wave_sum(lane < WAVES ? part_w[o] * __builtin_amdgcn_exp2f(rebase(a.c1, pm, m)) : 0.f);
    }
    if (!whole_row) {
        if (tid == 0) parts[(size_t)r * rows.segs + seg] = make_float4(m, sum, sum1, 0.f);
        return;
    }
    if (m == -INFINITY) sum = sum1 = NAN;        // nothing but -inf (or NaN)
    const float sum_l = MODE == kOne ? sum : sum1;     // of the label's softmax
    if (wave == 0) {
        const float loss = row_loss(a, mine, x_mine, x_label, m, __log2f(sum) * kLn2, __log2f(sum_l) * kLn2);
        if (lane == 0) {
            losses[r] = loss * bad_s;
            if (stats) *reinterpret_cast<float4*>(stats + 4 * (size_t)r) = make_float4(m, __log2f(sum) * bad_s, __log2f(sum_l) * bad_s, 0.f);
        }
    }
    if constexpr (GRAD) {
        const float wk = a.teacher ? weight * a.alpha * a.tau * bad_s : 0.f, wl = a.label ? weight * (1.f - a.alpha) * bad_s : 0.f;
        float fa = a.teacher && mass_s != 0.f ? wk / sum : 0.f, fb = a.label ? wl / sum_l : 0.f;
        if (MODE == kOne) fa += fb;
        auto value = [&](float f) {
            const float d = f - m, p = __builtin_amdgcn_exp2f(d * a.c);
            if (MODE == kOne) return p * fa;
            if (MODE == kSquare) return p * fmaf(p, fb, fa);
            return fmaf(p, fa, __builtin_amdgcn_exp2f(d * a.c1) * fb);
        };
#pragma unroll
        for (int i = 0; i < kVpt; ++i)
            if (x.whole(i)) {
                float f[E];
                unpack(x.v[i], f, T());
#pragma unroll
                for (int e = 0; e < E; ++e) f[e] = value(f[e]);
                const int base = x.index(i, 0);
                if (one.any(base / E)) one.apply(f, base, a.K + 1, -wk, -wl);
                const uint4 v = pack(f, T());
                __builtin_memcpy(out + base, &v, 16);
            }
        if (x.has_tail()) out[x.tail_index()] = (T)(value(x.x_tail) + one.at(x.tail_index(), a.K + 1, -wk, -wl));
    }
}

// Joins the segments of a row: one wave a row, one lane a segment, then one lane an entry of the teacher.
template <typename T, int MODE>
__global__ __launch_bounds__(64) void distill_join_kernel(Rows rows, Distill a, const float4* __restrict__ parts,
                                                          float* __restrict__ losses, float* __restrict__ stats) {
    const uint32_t r = blockIdx.x;
    const int lane = threadIdx.x, V = rows.vocab;
    const int64_t label = a.labels[r];
    if (label == a.ignore) return;               // written by the first segment's team
    const T* __restrict__ z = row_of<T>(rows, r);
    const bool label_ok = label >= 0 && label < V;
    float4 p = make_float4(-INFINITY, 0.f, 0.f, 0.f);
    if (lane < rows.segs) p = parts[(size_t)r * rows.segs + lane];
    Entry mine{-1, 0.f, 0.f, 0.f, false};
    float x = 0.f;
    if (a.teacher) {
        mine = teacher_entry(a, r, V);
        if (mine.id >= 0) x = (float)z[mine.id];
    } else {
        mine.bad = __ballot(lane < a.K && a.ids[(size_t)r * a.K + lane] >= V) != 0;
    }
    const float m = wave_max(p.x);
    const float none = m == -INFINITY ? NAN : 0.f;
    const float sum = wave_sum(p.y * __builtin_amdgcn_exp2f(rebase(a.c, p.x, m))) + none;
    const float sum_l = MODE == kOne ? sum : wave_sum(p.z * __builtin_amdgcn_exp2f(rebase(a.c1, p.x, m))) + none;
    const float bad = mine.bad || !label_ok ? NAN : 1.f;
    const float loss = row_loss(a, mine, x, label_ok ? (float)z[label] : 0.f, m, __log2f(sum) * kLn2, __log2f(sum_l) * kLn2);
    if (lane == 0) {
        losses[r] = loss * bad;
        if (stats) *reinterpret_cast<float4*>(stats + 4 * (size_t)r) = make_float4(m, __log2f(sum) * bad, __log2f(sum_l) * bad, 0.f);
    }
}

template <typename T, int MODE>
__global__ __launch_bounds__(64 * kGradWaves) void distill_grad_kernel(Rows rows, Distill a, const float* __restrict__ stats,
                                                                       const float* __restrict__ factor, const float* __restrict__ g,
                                                                       const float* __restrict__ g_row, T* __restrict__ grad) {
    constexpr int E = Vec<T>::n, THREADS = 64 * kGradWaves;
    __shared__ Singles<kGradWaves, E> one;
    __shared__ float mass_s;
    const int tid = threadIdx.x, lane = tid & 63;
    const uint32_t r = blockIdx.x / (uint32_t)rows.segs, seg = blockIdx.x % (uint32_t)rows.segs;
    const int V = rows.vocab, first = (int)seg * rows.seg_len, n = min(rows.seg_len, V - first);
    T* __restrict__ out = grad + (size_t)r * V + first;
    const int64_t label = a.labels[r];
    if (label == a.ignore) {
        write_zeros(out, n, THREADS);
        return;
    }
    Segment<T, kGradWaves> x;
    x.load(row_of<T>(rows, r) + first, n);
    const float4 st = *reinterpret_cast<const float4*>(stats + 4 * (size_t)r);
    float weight = factor ? factor[0] : 1.f;
    if (g) weight *= g[0];
    if (g_row) weight *= g_row[r];
    one.clear();
    team_sync<kGradWaves>();
    if (tid < 64) {
        Entry mine{-1, 0.f, 0.f, 0.f, false};
        if (a.teacher) mine = teacher_entry(a, r, V);
        if (lane < a.K) one.set(lane, mine.id < 0 ? -1 : mine.id - first, a.teacher ? n : 0, mine.q);
        if (lane == 0) {
            one.set(a.K, label - first, a.label ? n : 0, 1.f);
            mass_s = mine.mass;
        }
    }
    team_sync<kGradWaves>();
    const float m = st.x, wk = a.teacher ? weight * a.alpha * a.tau : 0.f, wl = a.label ? weight * (1.f - a.alpha) : 0.f;
    float fa = a.teacher && mass_s != 0.f ? wk * __builtin_amdgcn_exp2f(-st.y) : 0.f;
    const float fb = a.label ? wl * __builtin_amdgcn_exp2f(-st.z) : 0.f;
    if (MODE == kOne) fa += fb;
    auto value = [&](float f) {
        const float d = f - m, p = __builtin_amdgcn_exp2f(d * a.c);
        if (MODE == kOne) return p * fa;
        if (MODE == kSquare) return p * fmaf(p, fb, fa);
        return fmaf(p, fa, __builtin_amdgcn_exp2f(d * a.c1) * fb);
    };
#pragma unroll
    for (int i = 0; i < kVpt; ++i)
        if (x.whole(i)) {
            float f[E];
            unpack(x.v[i], f, T());
#pragma unroll
            for (int e = 0; e < E; ++e) f[e] = value(f[e]);
            const int base = x.index(i, 0);
            if (one.any(base / E)) one.apply(f, base, a.K + 1, -wk, -wl);
            const uint4 v = pack(f, T());
            __builtin_memcpy(out + base, &v, 16);
        }
    if (x.has_tail()) out[x.tail_index()] = (T)(value(x.x_tail) + one.at(x.tail_index(), a.K + 1, -wk, -wl));
}

// factor = weight (sum) or weight / number of rows that count (mean)
constexpr int kRowsThreads = 1024;
__global__ __launch_bounds__(kRowsThreads) void distill_factor_kernel(const int64_t* __restrict__ labels, int64_t ignore, int64_t rows,
                                                                      float weight, int mean, float* __restrict__ factor) {
    __shared__ int part[kRowsThreads / 64];
    int n = 0;                                   // at most 2^24 rows
    for (int64_t r0 = 0; mean && r0 < rows; r0 += 8 * kRowsThreads)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t r = r0 + i * kRowsThreads + threadIdx.x;
            const int64_t y = r < rows ? labels[r] : ignore;
            n += __popcll(__ballot(y != ignore));
        }
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = n;
    __syncthreads();
    if (threadIdx.x == 0) {
        int all = 0;
        for (int i = 0; i < kRowsThreads / 64; ++i) all += part[i];
        factor[0] = mean ? (float)((double)weight / (double)(all ? all : 1)) : weight;
    }
}

// total = factor * sum of the rows' losses, in 64 bits and in a fixed order
__global__ __launch_bounds__(kRowsThreads) void distill_total_kernel(const float* __restrict__ losses, int64_t rows,
                                                                     const float* __restrict__ factor, float* __restrict__ total) {
    __shared__ double part[kRowsThreads / 64];
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
        total[0] = (float)(all * (double)factor[0]);
    }
}

// Gradient made for an upstream gradient of 1: nothing to do if that is what it was.
template <typename T>
__global__ __launch_bounds__(256) void rescale_kernel(T* __restrict__ grad, int64_t n, const float* __restrict__ g) {
    constexpr int E = Vec<T>::n;
    const float f = g[0];
    if (f == 1.f) return;
    const int64_t nv = n / E, at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    for (int64_t i = at; i < nv; i += (int64_t)gridDim.x * 256) {
        uint4 v;
        float x[E];
        __builtin_memcpy(&v, grad + i * E, 16);
        unpack(v, x, T());
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] *= f;
        v = pack(x, T());
        __builtin_memcpy(grad + i * E, &v, 16);
    }
    if (nv * E + at < n) grad[nv * E + at] = (T)((float)grad[nv * E + at] * f);
}

// ---------------------------------------------------------------------------------- which team takes a row
constexpr int64_t kMaxBlocks = 2147483647;

struct Plan {
    int waves, segs, seg_len;
};

int elem_bytes(int dtype) { return dtype == STTFE_DTYPE_F32 ? 4 : 2; }

// The smallest team that holds a row in registers; a row too long for the largest is cut into equal segments.
Plan row_plan(int vocab, int dtype) {
    const int e = 16 / elem_bytes(dtype);
    const int64_t vecs = vocab / e;
    for (int waves : {1, 4, 8, 16})
        if (vecs <= (int64_t)kVpt * 64 * waves) return {waves, 1, vocab};
    const int cap = kVpt * 64 * kMaxWaves * e;   // a multiple of 64: so is a segment's length, and not above it
    const int segs = (vocab + cap - 1) / cap;
    static_assert(STTFE_MAX_VOCAB / 4 <= kMaxSegs * kVpt * 64 * kMaxWaves, "a row's segments are joined by one wave");
    const int len = ((vocab + segs - 1) / segs + 63) / 64 * 64;
    return {kMaxWaves, (vocab + len - 1) / len, len};
}
// Gradient kernels have nothing to join: a team of kGradWaves a segment.
Plan grad_plan(int vocab, int dtype) {
    const int cap = kVpt * 64 * kGradWaves * (16 / elem_bytes(dtype));
    const int segs = (vocab + cap - 1) / cap;
    const int len = ((vocab + segs - 1) / segs + 63) / 64 * 64;
    return {kGradWaves, (vocab + len - 1) / len, len};
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

#define STTFE_BY_DTYPE(dtype, ...)                                   \
    do {                                                              \
        if ((dtype) == STTFE_DTYPE_F32) { using T = float; __VA_ARGS__; }    \
        else if ((dtype) == STTFE_DTYPE_F16) { using T = half_t; __VA_ARGS__; } \
        else { using T = bf16_t; __VA_ARGS__; }                              \
    } while (0)

#define STTFE_BY_WAVES(plan, ...)                                    \
    do {                                                              \
        if ((plan).waves == 1) { constexpr int W = 1; __VA_ARGS__; }         \
        else if ((plan).waves == 4) { constexpr int W = 4; __VA_ARGS__; }    \
        else if ((plan).waves == 8) { constexpr int W = 8; __VA_ARGS__; }    \
        else { constexpr int W = 16; __VA_ARGS__; }                          \
    } while (0)

namespace {
template <typename T>
void launch_score(const Plan& plan, const Rows& rows, const Score& a, unsigned blocks, bool entropy, hipStream_t stream) {
    STTFE_BY_WAVES(plan, {
        if (a.top_k && entropy) hipLaunchKernelGGL((score_kernel<T, W, true, true>), dim3(blocks), dim3(64 * W), 0, stream, rows, a);
        else if (a.top_k) hipLaunchKernelGGL((score_kernel<T, W, false, true>), dim3(blocks), dim3(64 * W), 0, stream, rows, a);
        else if (entropy) hipLaunchKernelGGL((score_kernel<T, W, true, false>), dim3(blocks), dim3(64 * W), 0, stream, rows, a);
        else hipLaunchKernelGGL((score_kernel<T, W, false, false>), dim3(blocks), dim3(64 * W), 0, stream, rows, a);
    });
}

Distill distill_args(const int64_t* labels, int64_t ignore, const int64_t* ids, const float* teacher, int K, float tau, float alpha) {
    Distill a{labels, ids, teacher, ignore, K, tau, (float)(1.0 / (double)tau), alpha, 0.f, (float)kLog2e, alpha != 0.f, alpha != 1.f};
    a.c = a.teacher ? (float)(kLog2e / (double)tau) : (float)kLog2e;
    return a;
}
Mode distill_mode(const Distill& a) {
    if (!a.teacher || !a.label || a.tau == 1.f) return kOne;
    return a.tau == 2.f ? kSquare : kTwo;
}
#define STTFE_BY_MODE(mode, ...)                                     \
    do {                                                              \
        if ((mode) == kOne) { constexpr int M = kOne; __VA_ARGS__; }         \
        else if ((mode) == kTwo) { constexpr int M = kTwo; __VA_ARGS__; }    \
        else { constexpr int M = kSquare; __VA_ARGS__; }                     \
    } while (0)

template <typename T>
void launch_distill(const Plan& plan, const Rows& rows, const Distill& a, Mode mode, unsigned blocks, const float* factor,
                    float* losses, float* stats, float4* parts, T* grad, hipStream_t stream) {
    STTFE_BY_WAVES(plan, STTFE_BY_MODE(mode, {
        if (grad) hipLaunchKernelGGL((distill_kernel<T, W, M, true>), dim3(blocks), dim3(64 * W), 0, stream, rows, a, factor, losses, stats, parts, grad);
        else hipLaunchKernelGGL((distill_kernel<T, W, M, false>), dim3(blocks), dim3(64 * W), 0, stream, rows, a, factor, losses, stats, parts, grad);
    }));
}
template <typename T>
void launch_distill_grad(const Rows& rows, const Distill& a, Mode mode, int64_t n, const float* stats, const float* factor, const float* g,
                         const float* g_rows, T* grad, hipStream_t stream) {
    STTFE_BY_MODE(mode, hipLaunchKernelGGL((distill_grad_kernel<T, M>), dim3((unsigned)(n * rows.segs)), dim3(64 * kGradWaves), 0, stream,
                                           rows, a, stats, factor, g, g_rows, grad));
}
}  // namespace

extern "C" int sttfe_token_logprobs_workspace_bytes(int64_t rows, int vocab, int dtype, int top_k, size_t* bytes) {
    if (!bytes || rows < 0 || vocab < 1 || top_k < 0 || top_k > STTFE_MAX_TOP || top_k > vocab) return STTFE_E_INVALID_ARG;
    if (dtype != STTFE_DTYPE_F32 && dtype != STTFE_DTYPE_F16 && dtype != STTFE_DTYPE_BF16) return STTFE_E_INVALID_ARG;
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
    const Plan plan = row_plan(vocab, dtype);
    if (n > kMaxBlocks / plan.segs) return STTFE_E_UNSUPPORTED;
    const Rows rows{logits, (uint32_t)inner, stride_outer, stride_inner, vocab, plan.segs, plan.seg_len};
    float4* parts = static_cast<float4*>(workspace);
    const Score a{labels, ignore_index, (float)(kLog2e / (double)temperature), (float)(1.0 / (double)temperature), top_k, logprobs, entropy,
                  stats, top_ids, top_logprobs, parts, reinterpret_cast<uint64_t*>(parts + (plan.segs > 1 ? n * plan.segs : 0))};
    {
        ScopedTiming t(kTimeTokenLogprobs, stream);
        STTFE_BY_DTYPE(dtype, launch_score<T>(plan, rows, a, (unsigned)(n * plan.segs), entropy || stats, stream));
        if (plan.segs > 1) hipLaunchKernelGGL(score_join_kernel, dim3((unsigned)n), dim3(64), 0, stream, rows, a, dtype);
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
    const Plan plan = grad_plan(vocab, dtype);
    if (n > kMaxBlocks / plan.segs) return STTFE_E_UNSUPPORTED;
    const Rows rows{logits, (uint32_t)inner, stride_outer, stride_inner, vocab, plan.segs, plan.seg_len};
    const ScoreGrad a{labels, ignore_index, (float)(kLog2e / (double)temperature), (float)(1.0 / (double)temperature), stats, g_logprobs,
                      g_entropy, top_k, top_ids, g_top};
    {
        ScopedTiming t(kTimeTokenLogprobsGrad, stream);
        STTFE_BY_DTYPE(dtype, hipLaunchKernelGGL(score_grad_kernel<T>, dim3((unsigned)(n * plan.segs)), dim3(64 * kGradWaves), 0, stream,
                                                 rows, a, static_cast<T*>(grad)));
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
        if (!losses) return STTFE_E_INVALID_ARG;
    }
    if (n == 0 && reduction == STTFE_REDUCE_NONE) return STTFE_OK;
    size_t need = 0;
    rc = sttfe_distill_workspace_bytes(n, vocab, dtype, &need);
    if (rc != STTFE_OK) return rc;
    if (workspace_bytes < need || (need && !workspace)) return STTFE_E_WORKSPACE;
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    (void)hipGetLastError();
    const Plan plan = row_plan(vocab, dtype);
    if (n > kMaxBlocks / plan.segs) return STTFE_E_UNSUPPORTED;
    const Rows rows{logits, (uint32_t)inner, stride_outer, stride_inner, vocab, plan.segs, plan.seg_len};
    const Distill a = distill_args(labels, ignore_index, teacher_ids, teacher_logits, teacher_k, temperature, alpha);
    const Mode mode = distill_mode(a);
    const float* made = reduction != STTFE_REDUCE_NONE ? factor : nullptr;
    if (reduction != STTFE_REDUCE_NONE)
        hipLaunchKernelGGL(distill_factor_kernel, dim3(1), dim3(kRowsThreads), 0, stream, labels, ignore_index, n, weight,
                           reduction == STTFE_REDUCE_MEAN ? 1 : 0, factor);
    if (n > 0) {
        ScopedTiming t(kTimeDistill, stream);
        float4* parts = static_cast<float4*>(workspace);
        if (plan.segs == 1) {
            STTFE_BY_DTYPE(dtype, launch_distill<T>(plan, rows, a, mode, (unsigned)n, made, losses, stats, parts, static_cast<T*>(grad), stream));
        } else {
            // a row over several teams: their sums, the loss from the joined sums, then the gradient in a pass of its own
            float* st = stats ? stats : reinterpret_cast<float*>(parts + n * plan.segs);
            STTFE_BY_DTYPE(dtype, {
                launch_distill<T>(plan, rows, a, mode, (unsigned)(n * plan.segs), nullptr, losses, nullptr, parts, static_cast<T*>(nullptr), stream);
                STTFE_BY_MODE(mode, hipLaunchKernelGGL((distill_join_kernel<T, M>), dim3((unsigned)n), dim3(64), 0, stream, rows, a, parts, losses, st));
            });
            if (grad) {
                const Plan gp = grad_plan(vocab, dtype);
                if (n > kMaxBlocks / gp.segs) return STTFE_E_UNSUPPORTED;
                const Rows grows{logits, (uint32_t)inner, stride_outer, stride_inner, vocab, gp.segs, gp.seg_len};
                STTFE_BY_DTYPE(dtype, launch_distill_grad<T>(grows, a, mode, n, st, made, nullptr, nullptr, static_cast<T*>(grad), stream));
            }
        }
    }
    if (reduction != STTFE_REDUCE_NONE)
        hipLaunchKernelGGL(distill_total_kernel, dim3(1), dim3(kRowsThreads), 0, stream, losses, n, factor, total);
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
    const Plan plan = grad_plan(vocab, dtype);
    if (n > kMaxBlocks / plan.segs) return STTFE_E_UNSUPPORTED;
    const Rows rows{logits, (uint32_t)inner, stride_outer, stride_inner, vocab, plan.segs, plan.seg_len};
    const Distill a = distill_args(labels, ignore_index, teacher_ids, teacher_logits, teacher_k, temperature, alpha);
    {
        ScopedTiming t(kTimeDistillGrad, stream);
        STTFE_BY_DTYPE(dtype, launch_distill_grad<T>(rows, a, distill_mode(a), n, stats, factor, g, g_rows, static_cast<T*>(grad), stream));
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
    const int64_t want = (count + 2047) / 2048;
    const unsigned blocks = (unsigned)(want < 2048 ? want : 2048);
    STTFE_BY_DTYPE(dtype, hipLaunchKernelGGL(rescale_kernel<T>, dim3(blocks), dim3(256), 0, stream, static_cast<T*>(grad), count, g));
    if (hip_failed(hipGetLastError(), "gradient rescale kernel launch")) return STTFE_E_LAUNCH;
    return STTFE_OK;
}
