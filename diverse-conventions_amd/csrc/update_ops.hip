// update_ops.hip -- what a policy-gradient update computes behind the rollout, gfx950: the clipped policy loss over logits and the clipped
// value loss, each with its gradient, and the global norm of many gradient tensors with clipping.  All of it streams: each operator is
// bound by the bytes of its inputs and outputs, and is built to read every input once (the gradient norm: once per pass).
//
// Sums over rows are kept in f64 and added in a fixed order (per-block partial sums, no atomics): the results do not depend on which
// block ran when.  Everything inside a row is f32, whatever the logits' type; a gradient is rounded once, to the logits' type.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "overcooked_ops.h"
#include "oc_internal.h"

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
// a 16-byte access at an element's own alignment: rows of an odd number of 2-byte elements start anywhere, and global memory
// instructions take any address
typedef uint32_t u32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4_a1 __attribute__((ext_vector_type(4), aligned(1)));

template <int ALIGN> struct Unaligned { typedef u32x4_a4 type; };
template <> struct Unaligned<2> { typedef u32x4_a2 type; };

template <typename T> struct Chunk {                       // 16 bytes of elements
    static constexpr int V = 16 / sizeof(T);
    union { u32x4 raw; T e[V]; };
    __device__ Chunk() {}
};

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLowest = -1e4f;                           // floor of exponents in products with 2^v, which is 0 long before
constexpr float kLargest = 3.4028235e38f;
__device__ __forceinline__ float neg_inf() { return -__builtin_inff(); }
// The hardware's own exp2, log2 and reciprocal: 1 ulp, where arguments below the normal range do not matter (a probability of 2^-127
// counts as 0 next to one of 1).  The library functions around them cost more than the memory traffic of a short row.
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float exp_fast(float x) { return exp2_fast(x * kLog2e); }
__device__ __forceinline__ float log2_fast(float x) { return __builtin_amdgcn_logf(x); }
__device__ __forceinline__ float rcp_fast(float x) { return __builtin_amdgcn_rcpf(x); }

// A row's logits as exponents of 2 relative to its largest, v = (z - m) log2 e: the difference first, so that v is 0 at the largest logit and
// carries 2^-23 of itself wherever the row lies.  (One fma with -m log2 e as its addend leaves that product's rounding in every v: 2^v is inf
// or 0 for a largest logit beyond 1e10 or so, and where wavefronts share a row each has another rounding.)
__device__ __forceinline__ float base_of(float m) { return m == neg_inf() ? 0.0f : m; }       // no possible action: exponents of -inf, not NaN
__device__ __forceinline__ float exponent_of(float z, float base) { return (z - base) * kLog2e; }

constexpr int kMaxBlocks = 2048;                           // of a launch that leaves one set of partial sums per block
constexpr int kWeightBlocks = 1024;                        // of the launch that adds up the weights
constexpr int kSums = 6;

struct PolicyLossArgs {
    const void *logits;
    const void *actions;
    const float *old_logp, *adv, *ref_logp, *weights;      // ref_logp, weights: or NULL
    const void *avail;                                     // or NULL
    void *grad;
    const float *grad_out;                                 // upstream gradient (device) or NULL = 1
    float *loss, *stats;                                   // [1], [5] or NULL
    double *weight;                                        // W: written by a forward pass, read by the backward pass
    double *weight_partials;                               // [kWeightBlocks]
    double *sums;                                          // [blocks][kSums]
    long long rows, row_stride, avail_stride;
    int n_actions, action_type, avail_u8;
    int weight_from;                                       // of the weight: see enum
    int n_weight_partials, finalize_here, want_sums;
    float clip_lo, clip_hi, entropy_coef, kl_coef, grad_scale;
};
// where a block takes the total weight from: nowhere (no gradient: the sums carry it), every block adds it up itself (few rows), the
// partial sums of the launch before, what the forward pass has left
enum { WEIGHT_NONE = 0, WEIGHT_SELF = 1, WEIGHT_PARTIALS = 2, WEIGHT_GIVEN = 3 };

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off);
    return x;
}

// Sum over the block, valid in every thread; `part`: LDS, one double per wavefront.
__device__ __forceinline__ double block_sum(double x, double *part) {
    x = wave_sum(x);
    const int waves = blockDim.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
    __syncthreads();
    x = part[0];
    for (int w = 1; w < waves; ++w) x += part[w];
    return x;
}

// The same for N values with one exchange, valid in threads 0 .. N - 1: thread i returns value i.
template <int N>
__device__ __forceinline__ double block_sums(const double (&x)[N], double (*part)[N]) {
    double y[N];
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] = x[i];
#pragma unroll
    for (int off = 32; off > 0; off >>= 1)
#pragma unroll
        for (int i = 0; i < N; ++i) y[i] += __shfl_xor(y[i], off);
    if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int i = 0; i < N; ++i) part[threadIdx.x >> 6][i] = y[i];
    __syncthreads();
    double sum = 0.0;
    if (threadIdx.x < N)
        for (int w = 0; w < static_cast<int>(blockDim.x >> 6); ++w) sum += part[w][threadIdx.x];
    return sum;
}

// The taken action of a row, -1 when it is none of 0 .. n - 1 (also a float that is NaN or lies outside [0, n): the comparison with n is one
// of whole numbers, 2^24 + 1 is no float).
__device__ __forceinline__ int checked_action(int v, int n) { return v >= 0 && v < n ? v : -1; }
__device__ __forceinline__ int checked_action(long long v, int n) { return v >= 0 && v < n ? static_cast<int>(v) : -1; }
__device__ __forceinline__ int checked_action(float f, int n) { return f >= 0.0f && f < 0x1p30f ? checked_action(static_cast<int>(f), n) : -1; }

// `first`: a row that is the same for all lanes, `i`: this lane's behind it
__device__ __forceinline__ int action_of(const PolicyLossArgs &a, long long first, uint32_t i = 0) {
    if (a.action_type == OC_ACT_F32) return checked_action((static_cast<const float *>(a.actions) + first)[i], a.n_actions);
    if (a.action_type == OC_ACT_I64) return checked_action((static_cast<const long long *>(a.actions) + first)[i], a.n_actions);
    return checked_action((static_cast<const int *>(a.actions) + first)[i], a.n_actions);
}

__device__ __forceinline__ double row_weight(const PolicyLossArgs &a, long long row) {
    if (action_of(a, row) < 0) return 0.0;
    return a.weights ? static_cast<double>(a.weights[row]) : 1.0;
}

// Weights of four rows, in 16-byte loads.
__device__ __forceinline__ double four_weights(const PolicyLossArgs &a, long long row) {
    const u32x4 w = a.weights ? *reinterpret_cast<const u32x4_a4 *>(a.weights + row) : u32x4{0x3f800000u, 0x3f800000u, 0x3f800000u, 0x3f800000u};
    int v[4];
    if (a.action_type == OC_ACT_I64) {
        const u32x4 x = reinterpret_cast<const u32x4_a4 *>(static_cast<const long long *>(a.actions) + row)[0];
        const u32x4 y = reinterpret_cast<const u32x4_a4 *>(static_cast<const long long *>(a.actions) + row)[1];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            v[i] = checked_action(static_cast<long long>(static_cast<uint64_t>(x[2 * i + 1]) << 32 | x[2 * i]), a.n_actions);
            v[2 + i] = checked_action(static_cast<long long>(static_cast<uint64_t>(y[2 * i + 1]) << 32 | y[2 * i]), a.n_actions);
        }
    } else {
        const u32x4 x = *reinterpret_cast<const u32x4_a4 *>(static_cast<const int *>(a.actions) + row);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = a.action_type == OC_ACT_F32 ? checked_action(__uint_as_float(x[i]), a.n_actions) : checked_action(static_cast<int>(x[i]), a.n_actions);
    }
    double sum[2] = {0.0, 0.0};
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i & 1] += v[i] >= 0 ? static_cast<double>(__uint_as_float(w[i])) : 0.0;
    return sum[0] + sum[1];
}

__global__ __launch_bounds__(256) void oc_policy_weight_kernel(const PolicyLossArgs a) {
    __shared__ double part[4];
    double w = 0.0;
    const long long stride = static_cast<long long>(gridDim.x) * 256;
    const long long quads = a.rows >> 2;
#pragma unroll 4
    for (long long q = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; q < quads; q += stride) w += four_weights(a, q << 2);
    if (blockIdx.x == 0 && threadIdx.x < (a.rows & 3)) w += row_weight(a, (quads << 2) + threadIdx.x);
    w = block_sum(w, part);
    if (threadIdx.x == 0) a.weight_partials[blockIdx.x] = w;
}

// 1 / total weight, 0 when there is none.
__device__ __forceinline__ float inverse_weight(const PolicyLossArgs &a, double *part) {
    double w = 0.0;
    if (a.weight_from == WEIGHT_SELF) {
        for (long long r = threadIdx.x; r < a.rows; r += blockDim.x) w += row_weight(a, r);
        w = block_sum(w, part);
    } else if (a.weight_from == WEIGHT_PARTIALS) {
        for (int i = threadIdx.x; i < a.n_weight_partials; i += blockDim.x) w += a.weight_partials[i];
        w = block_sum(w, part);
    } else if (a.weight_from == WEIGHT_GIVEN) {
        w = *a.weight;
    }
    return w != 0.0 ? static_cast<float>(1.0 / w) : 0.0f;
}

// What the rows of a thread (or of a group's first lane) add to the sums; a group's lane keeps them in LDS.
struct RowSums {
    double s[kSums];                                       // policy, entropy, kl, clipped, ratio, weight
};

// The results from the six sums: thread i has sum i.
__device__ __forceinline__ void write_result(const PolicyLossArgs &a, double mine) {
    if (threadIdx.x >= 64) return;
    const double weight = __shfl(mine, 5), inv = weight != 0.0 ? 1.0 / weight : 0.0;
    const double entropy = __shfl(mine, 1), kl = __shfl(mine, 2);
    if (threadIdx.x == 0) {
        double loss = mine;                                // a term without weight stays out, also where it is not finite
        if (a.entropy_coef != 0.0f) loss -= static_cast<double>(a.entropy_coef) * entropy;
        if (a.kl_coef != 0.0f) loss += static_cast<double>(a.kl_coef) * kl;
        *a.loss = static_cast<float>(loss * inv);
        if (a.weight) *a.weight = weight;
    }
    if (a.stats && threadIdx.x < 5) a.stats[threadIdx.x] = static_cast<float>(mine * inv);
}

__device__ __forceinline__ void finish_sums(const PolicyLossArgs &a, const RowSums &r, double (*part)[kSums]) {
    if (!a.want_sums) return;
    const double mine = block_sums(r.s, part);
    if (a.finalize_here) write_result(a, mine);
    else if (threadIdx.x < kSums) a.sums[static_cast<long long>(blockIdx.x) * kSums + threadIdx.x] = mine;
}

__global__ __launch_bounds__(1024) void oc_policy_finalize_kernel(const PolicyLossArgs a, int blocks) {
    __shared__ double part[16][kSums];
    double s[kSums] = {0, 0, 0, 0, 0, 0};
    for (int b = threadIdx.x; b < blocks; b += 1024)
#pragma unroll
        for (int i = 0; i < kSums; ++i) s[i] += a.sums[static_cast<long long>(b) * kSums + i];
    write_result(a, block_sums(s, part));
}

// One row behind its softmax, in units of log 2: `va` the exponent of the taken action, s = sum 2^v, t = sum 2^v v over the possible
// actions.  Adds to the sums; the gradient of logit j is then, times `go`, 2^v_j (a1 v_j + a0) + [j == taken] c1:
//   d loss / d lp = c1 = (w / W) (-A ratio [not clipped] + ck (1 - exp(ref - lp)));  d H / d z_j = -p_j (log p_j + H),  p_j = 2^v_j / s.
struct RowGrad {
    float c1, a1, a0;
    bool none;                                             // the row adds nothing
};

struct RowInputs { float weight, adv, old_logp, ref_logp; };

__device__ __forceinline__ RowInputs row_inputs(const PolicyLossArgs &a, long long first, uint32_t i, int action) {
    RowInputs r;
    r.weight = action < 0 ? 0.0f : a.weights ? (a.weights + first)[i] : 1.0f;
    r.adv = (a.adv + first)[i];
    r.old_logp = (a.old_logp + first)[i];
    r.ref_logp = a.ref_logp ? (a.ref_logp + first)[i] : 0.0f;
    return r;
}

__device__ __forceinline__ RowGrad row_terms(const PolicyLossArgs &a, const RowInputs &in, float inv_w, float go, bool possible, float va, float s,
                                             float t, bool leader, RowSums &sums) {
    RowGrad g = {0.0f, 0.0f, 0.0f, true};
    if (!possible) return g;
    const float log_s = log2_fast(s), inv_s = rcp_fast(s);
    // an action beyond the range of exponents has the lowest log-probability, not -inf: exp(d) - d below is inf, not inf - inf
    const float lp_any = (va - log_s) * kLn2, lp = lp_any < -kLargest ? -kLargest : lp_any;
    const float entropy = (log_s - t * inv_s) * kLn2;
    const float adv = in.adv, weight = in.weight;
    const float ratio = exp_fast(lp - in.old_logp);
    const float kept = fminf(fmaxf(ratio, a.clip_lo), a.clip_hi);
    const auto times_adv = [&](float x) { return adv == 0.0f && x == __builtin_inff() ? 0.0f : x * adv; };        // a ratio beyond f32 is a number
    const float s1 = times_adv(ratio), s2 = times_adv(kept);
    const float policy = -(s1 != s1 || s2 != s2 ? s1 + s2 : fminf(s1, s2));
    const bool cut = (adv > 0.0f && ratio > a.clip_hi) || (adv < 0.0f && ratio < a.clip_lo);
    float slope = cut ? 0.0f : -s1;
    float kl = 0.0f;
    if (a.ref_logp) {
        const float d = in.ref_logp - lp;
        float e;                                           // exp(d) - 1
        if (fabsf(d) < 0.25f) {
            // next to the reference policy exp(d) - 1 - d is about d^2 / 2, and subtracting would leave its rounding, 2^-24, of either sign: the
            // power series, cut where the next term is 2^-26 of the sum
            kl = d * d * fmaf(d, fmaf(d, fmaf(d, fmaf(d, fmaf(d, 1.0f / 5040, 1.0f / 720), 1.0f / 120), 1.0f / 24), 1.0f / 6), 0.5f);
            e = d + kl;
        } else {
            e = exp_fast(d) - 1.0f;
            kl = e - d;
        }
        if (a.kl_coef != 0.0f) slope = slope - a.kl_coef * e;
    }
    if (leader) {
        const double w = weight;
        sums.s[0] = fma(w, static_cast<double>(policy), sums.s[0]);
        sums.s[1] = fma(w, static_cast<double>(entropy), sums.s[1]);
        sums.s[2] = fma(w, static_cast<double>(kl), sums.s[2]);
        sums.s[3] += ratio < a.clip_lo || ratio > a.clip_hi ? w : 0.0;
        sums.s[4] = fma(w, static_cast<double>(ratio), sums.s[4]);
    }
    const float scale = weight * inv_w * go;
    const float ce = scale * a.entropy_coef;
    g.c1 = scale * slope;
    g.a1 = ce * kLn2 * inv_s;
    g.a0 = (ce * (entropy - log_s * kLn2) - g.c1) * inv_s;
    g.none = false;
    return g;
}

// Gradient of a logit with exponent v and e = 2^v; the taken action's c1 comes on top.
__device__ __forceinline__ float grad_of(const RowGrad &g, float v, float e) { return e * fmaf(g.a1, fmaxf(v, kLowest), g.a0); }

// -------------------------------------------------------------------------------------------------------------------------------
// Up to 16 actions: a thread has a whole row.  The block's 256 rows are one contiguous piece of memory; it is copied through LDS in
// 16-byte pieces, because lanes that each load their own 24 bytes touch every line of the piece once per load.  AM: so many values are
// held in registers.  6.55 M rows of 6 f32 with gradient: 106 us (446 MB, 4.2 TB/s) and 14 us for the weights in front; 360 vector
// instructions a row with library logarithm, exponential and division made it 204 us.
// -------------------------------------------------------------------------------------------------------------------------------
constexpr int kRowTile = 256;

template <int ALIGN>
__device__ __forceinline__ void copy_in(void *lds, const void *src, int bytes) {
    typedef typename Unaligned<ALIGN>::type U;
    const int whole = bytes & ~15;
    for (int b = threadIdx.x * 16; b < whole; b += 256 * 16)
        *reinterpret_cast<u32x4 *>(static_cast<char *>(lds) + b) = *reinterpret_cast<const U *>(static_cast<const char *>(src) + b);
    if (static_cast<int>(threadIdx.x) < bytes - whole) static_cast<char *>(lds)[whole + threadIdx.x] = static_cast<const char *>(src)[whole + threadIdx.x];
}

template <int ALIGN>
__device__ __forceinline__ void copy_out(void *dst, const void *lds, int bytes) {
    typedef typename Unaligned<ALIGN>::type U;
    const int whole = bytes & ~15;
    for (int b = threadIdx.x * 16; b < whole; b += 256 * 16)
        *reinterpret_cast<U *>(static_cast<char *>(dst) + b) = *reinterpret_cast<const u32x4 *>(static_cast<const char *>(lds) + b);
    if (static_cast<int>(threadIdx.x) < bytes - whole) static_cast<char *>(dst)[whole + threadIdx.x] = static_cast<const char *>(lds)[whole + threadIdx.x];
}

// EXACT: a row has AM values; else at most AM.
template <typename T, int AM, bool EXACT, bool GRAD>
__global__ __launch_bounds__(256) void oc_policy_loss_rows_kernel(const PolicyLossArgs a) {
    __shared__ __attribute__((aligned(16))) T rows_lds[kRowTile * AM];
    __shared__ __attribute__((aligned(16))) char avail_lds[kRowTile * AM * 4];
    __shared__ double part[4], parts[4][kSums];
    const int A = EXACT ? AM : a.n_actions;
    const float inv_w = GRAD ? inverse_weight(a, part) : 0.0f;
    const float go = GRAD ? a.grad_scale * (a.grad_out ? *a.grad_out : 1.0f) : 0.0f;
    const bool stage_avail = a.avail && a.avail_stride == A;
    const auto may_at = [&](long long at) {
        return a.avail_u8 ? static_cast<const uint8_t *>(a.avail)[at] != 0 : static_cast<const float *>(a.avail)[at] != 0.0f;
    };
    const uint32_t everything = (1u << A) - 1;
    uint32_t may_all = everything;                         // a bit per action; one mask for all rows is read once
    if (a.avail && a.avail_stride == 0) {
        may_all = 0;
        for (int j = 0; j < A; ++j) may_all |= may_at(j) ? 1u << j : 0;
    }
    RowSums sums = {};
    const long long tiles = (a.rows + kRowTile - 1) / kRowTile;
    for (long long tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const long long row0 = tile * kRowTile;
        const int n = static_cast<int>(a.rows - row0 < kRowTile ? a.rows - row0 : kRowTile);
        int me = threadIdx.x;
        asm volatile("" : "+v"(me));                       // places are computed anew, not kept in registers over the loop
        const long long row = row0 + me;
        const bool live = me < n;
        // everything that a row needs is on its way before the first wait
        const int action = live ? action_of(a, row0, me) : -1;
        RowInputs in = {0.0f, 0.0f, 0.0f, 0.0f};
        if (live) in = row_inputs(a, row0, me, action);
        if (a.row_stride == A)
            copy_in<sizeof(T) == 4 ? 4 : 2>(rows_lds, static_cast<const T *>(a.logits) + row0 * A, n * A * static_cast<int>(sizeof(T)));
        else if (live)
            for (int j = 0; j < A; ++j) rows_lds[me * A + j] = static_cast<const T *>(a.logits)[row * a.row_stride + j];
        uint32_t may = may_all;
        if (stage_avail) {
            const int size = a.avail_u8 ? 1 : 4;
            const char *src = static_cast<const char *>(a.avail) + row0 * A * size;
            if (a.avail_u8) {
                for (int b = me; b < n * A; b += 256) avail_lds[b] = src[b];
            } else {
                copy_in<4>(avail_lds, src, n * A * 4);
            }
        } else if (a.avail && a.avail_stride != 0 && live) {
            may = 0;
            for (int j = 0; j < A; ++j) may |= may_at(row * a.avail_stride + j) ? 1u << j : 0;
        }
        __syncthreads();
        float z[AM];
        float m = neg_inf(), za = neg_inf();
#pragma unroll
        for (int j = 0; j < AM; ++j) z[j] = static_cast<float>(rows_lds[me * A + (j < A ? j : 0)]);
        if (stage_avail) {
            may = 0;
            if (a.avail_u8) {
#pragma unroll
                for (int j = 0; j < AM; ++j) may |= avail_lds[me * A + (j < A ? j : 0)] != 0 ? 1u << j : 0;
            } else {
#pragma unroll
                for (int j = 0; j < AM; ++j) may |= reinterpret_cast<const float *>(avail_lds)[me * A + (j < A ? j : 0)] != 0.0f ? 1u << j : 0;
            }
            may &= everything;
        }
#pragma unroll
        for (int j = 0; j < AM; ++j) {
            z[j] = may >> j & 1 ? z[j] : neg_inf();
            za = j == action ? z[j] : za;
            m = fmaxf(m, z[j]);
        }
        RowGrad g = {0.0f, 0.0f, 0.0f, true};
        const float base = base_of(m);
        float e[AM], s = 0.0f, t = 0.0f;
        if (in.weight != 0.0f) {
            sums.s[5] += in.weight;
#pragma unroll
            for (int j = 0; j < AM; ++j) {
                const float v = exponent_of(z[j], base);
                e[j] = exp2_fast(v);
                s += e[j];
                t = fmaf(e[j], fmaxf(v, kLowest), t);
            }
            // logits that are all NaN leave m at -inf and s NaN
            g = row_terms(a, in, inv_w, go, za != neg_inf() && !(m == neg_inf() && s == 0.0f), exponent_of(za, base), s, t, true, sums);
        }
        if (GRAD) {
#pragma unroll
            for (int j = 0; j < AM; ++j) {
                if (j < A && live) {
                    float d = grad_of(g, exponent_of(z[j], base), e[j]) + (j == action ? g.c1 : 0.0f);
                    if (g.none || z[j] == neg_inf()) d = 0.0f;
                    rows_lds[me * A + j] = static_cast<T>(d);
                }
            }
            __syncthreads();
            copy_out<sizeof(T) == 4 ? 4 : 2>(static_cast<T *>(a.grad) + row0 * A, rows_lds, n * A * static_cast<int>(sizeof(T)));
        }
        __syncthreads();
    }
    finish_sums(a, sums, parts);
}

// -------------------------------------------------------------------------------------------------------------------------------
// More actions: L lanes have a row together, each C pieces of 16 bytes of it in registers (C = 0: more than fits, the row is read again
// for the gradient).  One pass: a wavefront's maximum, its sums relative to that, and, where several wavefronts share the row, one
// exchange of (maximum, sums) through LDS.  4096 rows of 32768 bf16 with gradient: 128 us, 4.2 TB/s, 82 % of a copy's rate: two
// exponentials and 19 other vector instructions an element, most of it under the memory's time (17, with one fma for an exponent: 124 us).
// -------------------------------------------------------------------------------------------------------------------------------
// Bits of -inf, in every element of a 32-bit word.  Pieces are put together as words: element by element the compiler gives each 16-bit
// value a register of its own.
template <typename T> constexpr uint32_t kNegInf = 0xff800000u;
template <> constexpr uint32_t kNegInf<__bf16> = 0xff80ff80u;
template <> constexpr uint32_t kNegInf<_Float16> = 0xfc00fc00u;

template <typename T>
__device__ __forceinline__ u32x4 rest_of_row(const T *row_ptr, int j0, int n) {
    u32x4 raw;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        uint32_t v = kNegInf<T>;
        if (sizeof(T) == 4) {
            if (j0 + w < n) v = reinterpret_cast<const uint32_t *>(row_ptr)[j0 + w];
        } else {
            if (j0 + 2 * w < n) v = (v & 0xffff0000u) | reinterpret_cast<const uint16_t *>(row_ptr)[j0 + 2 * w];
            if (j0 + 2 * w + 1 < n) v = (v & 0xffffu) | static_cast<uint32_t>(reinterpret_cast<const uint16_t *>(row_ptr)[j0 + 2 * w + 1]) << 16;
        }
        raw[w] = v;
    }
    return raw;
}

// Piece c = lane + first of a row: the row's own address and `first` are the same for all lanes, the rest is 32 bits.
template <typename T>
__device__ __forceinline__ Chunk<T> load_values(const PolicyLossArgs &a, const T *row_ptr, int first, int lane) {
    constexpr int V = Chunk<T>::V;
    typedef typename Unaligned<sizeof(T)>::type U;
    Chunk<T> x;
    if ((first + lane + 1) * V <= a.n_actions)
        x.raw = *reinterpret_cast<const U *>(reinterpret_cast<const char *>(row_ptr + static_cast<long long>(first) * V) + static_cast<uint32_t>(lane) * 16u);
    else
        x.raw = rest_of_row(row_ptr, (first + lane) * V, a.n_actions);
    return x;
}

// Unavailable actions become -inf.
template <typename T>
__device__ __forceinline__ void take_out(const PolicyLossArgs &a, Chunk<T> &x, long long row, int c) {
    constexpr int V = Chunk<T>::V;
    const int j0 = c * V;
    const long long at = row * a.avail_stride + j0;
    uint32_t may = 0;                                      // a bit per element
    if (a.avail_u8) {
        const uint8_t *src = static_cast<const uint8_t *>(a.avail) + at;
        if (j0 + V <= a.n_actions) {
            uint32_t words[V / 4];
            __builtin_memcpy(words, src, V);
#pragma unroll
            for (int i = 0; i < V; ++i) may |= (words[i / 4] >> (8 * (i & 3)) & 0xff) != 0 ? 1u << i : 0;
        } else {
            for (int i = 0; i < V && j0 + i < a.n_actions; ++i) may |= src[i] != 0 ? 1u << i : 0;
        }
    } else {
        const float *src = static_cast<const float *>(a.avail) + at;
        if (j0 + V <= a.n_actions) {
#pragma unroll
            for (int q = 0; q < V / 4; ++q) {
                const u32x4 four = reinterpret_cast<const u32x4_a4 *>(src)[q];
#pragma unroll
                for (int i = 0; i < 4; ++i) may |= (four[i] << 1) != 0 ? 1u << (q * 4 + i) : 0;         // +0 and -0 are 0
            }
        } else {
            for (int i = 0; i < V && j0 + i < a.n_actions; ++i) may |= src[i] != 0.0f ? 1u << i : 0;
        }
    }
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if (sizeof(T) == 4) {
            x.raw[w] = may >> w & 1 ? x.raw[w] : kNegInf<T>;
        } else {
            const uint32_t keep = (may >> (2 * w) & 1 ? 0xffffu : 0u) | (may >> (2 * w + 1) & 1 ? 0xffff0000u : 0u);
            x.raw[w] = (x.raw[w] & keep) | (kNegInf<T> & ~keep);
        }
    }
}

template <typename T>
__device__ __forceinline__ Chunk<T> load_chunk(const PolicyLossArgs &a, const T *row_ptr, long long row, int c) {
    Chunk<T> x = load_values<T>(a, row_ptr, 0, c);
    if (a.avail) take_out<T>(a, x, row, c);
    return x;
}

template <typename T>
__device__ __forceinline__ void store_grad(const PolicyLossArgs &a, T *row_ptr, int first, int lane, const Chunk<T> &x) {
    constexpr int V = Chunk<T>::V;
    typedef typename Unaligned<sizeof(T)>::type U;
    const int j0 = (first + lane) * V;
    if (j0 + V <= a.n_actions) {
        *reinterpret_cast<U *>(reinterpret_cast<char *>(row_ptr + static_cast<long long>(first) * V) + static_cast<uint32_t>(lane) * 16u) = x.raw;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (j0 + i < a.n_actions) row_ptr[j0 + i] = x.e[i];
    }
}

// `nan`: the row's sums or coefficients are not finite, and 0 times them is not what a masked place gets
template <typename T>
__device__ __forceinline__ Chunk<T> grad_chunk(const Chunk<T> &x, int c, int action, float base, const RowGrad &g, bool nan) {
    constexpr int V = Chunk<T>::V;
    Chunk<T> y;
    float d[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float v = exponent_of(static_cast<float>(x.e[i]), base);
        d[i] = grad_of(g, v, exp2_fast(v));
    }
    if (action / V == c) {
#pragma unroll
        for (int i = 0; i < V; ++i) d[i] += c * V + i == action ? g.c1 : 0.0f;
    }
    if (nan) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (static_cast<float>(x.e[i]) == neg_inf()) d[i] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) y.e[i] = static_cast<T>(d[i]);
    return y;
}

template <int W>
__device__ __forceinline__ float lanes_max(float x) {
#pragma unroll
    for (int off = W / 2; off > 0; off >>= 1) x = fmaxf(x, __shfl_xor(x, off));
    return x;
}

template <int W>
__device__ __forceinline__ float lanes_sum(float x) {
#pragma unroll
    for (int off = W / 2; off > 0; off >>= 1) x += __shfl_xor(x, off);
    return x;
}

template <typename T>
__device__ __forceinline__ void chunk_sums(const Chunk<T> &x, float base, float &s, float &t) {
#pragma unroll
    for (int i = 0; i < Chunk<T>::V; ++i) {
        const float v = exponent_of(static_cast<float>(x.e[i]), base), e = exp2_fast(v);
        s += e;
        t = fmaf(e, fmaxf(v, kLowest), t);
    }
}

// s and t relative to the largest logit m, taken over to a larger one.  Without a possible action so far they are 0 -- or NaN, which
// has to reach the result.
__device__ __forceinline__ void rebase(float m, float to, float &s, float &t) {
    if (m == neg_inf()) return;
    const float d = fmaxf((m - to) * kLog2e, kLowest), f = exp2_fast(d);
    t = f * fmaf(s, d, t);
    s *= f;
}

// The pieces stay in registers as they were loaded: without this the compiler keeps the converted values and the exponentials of one
// sweep for the next, twice to four times the registers, and three workgroups' worth of loads in flight become one.
template <typename T>
__device__ __forceinline__ void forget(Chunk<T> &x) { asm volatile("" : "+v"(x.raw)); }

template <typename T, int L, int C, bool GRAD>
__global__ __launch_bounds__(L < 256 ? 256 : L) __attribute__((amdgpu_waves_per_eu(C >= 16 ? 4 : 1))) void oc_policy_loss_group_kernel(const PolicyLossArgs a) {
    constexpr int B = L < 256 ? 256 : L;                   // threads of a block
    constexpr int R = B / L;                               // rows of a block
    constexpr int LW = L < 64 ? L : 64;                    // lanes of a wavefront that share a row
    constexpr int NW = L / LW;                             // wavefronts that share a row
    constexpr int V = Chunk<T>::V;
    __shared__ float merge[2][NW][4];
    __shared__ double part[B / 64], parts[B / 64][kSums];
    const float inv_w = GRAD ? inverse_weight(a, part) : 0.0f;
    const float go = GRAD ? a.grad_scale * (a.grad_out ? *a.grad_out : 1.0f) : 0.0f;
    const int lane_of_row = threadIdx.x % L;
    const int n_chunks = (a.n_actions + V - 1) / V;
    __shared__ RowSums group_sums[R];
    // a row's addresses and scalars are the wavefront's, in scalar registers, where no two rows share one
    const int group = L < 64 ? threadIdx.x / L : L < B ? __builtin_amdgcn_readfirstlane(threadIdx.x / L) : 0;
    RowSums &sums = group_sums[group];
    if (lane_of_row == 0) sums = RowSums{};
    int parity = 0;
    for (long long row = static_cast<long long>(blockIdx.x) * R + group; row < a.rows; row += static_cast<long long>(gridDim.x) * R) {
        // every row, and every sweep over it, computes its places anew: kept, the index of every element takes a register
        int lane = lane_of_row;
        asm volatile("" : "+v"(lane));
        const int action = action_of(a, row);
        const RowInputs in = row_inputs(a, row, 0, action);
        T *const grad_ptr = static_cast<T *>(a.grad) + row * a.n_actions;
        if (in.weight == 0.0f) {
            if (GRAD) {
                Chunk<T> zero;
                zero.raw = u32x4{0, 0, 0, 0};
                for (int c = lane; c < n_chunks; c += L) store_grad<T>(a, grad_ptr, 0, c, zero);
            }
            continue;
        }
        const T *row_ptr = static_cast<const T *>(a.logits) + row * a.row_stride;
        Chunk<T> x[C ? C : 1];
        if (C) {
#pragma unroll
            for (int i = 0; i < C; ++i)
                if (lane + i * L < n_chunks) x[i] = load_values<T>(a, row_ptr, i * L, lane);
        }
        float m = neg_inf(), s = 0.0f, t = 0.0f;
        float za = static_cast<float>(row_ptr[action]);
        if (a.avail) {
            const long long at = row * a.avail_stride + action;
            if (a.avail_u8 ? static_cast<const uint8_t *>(a.avail)[at] == 0 : static_cast<const float *>(a.avail)[at] == 0.0f) za = neg_inf();
        }
        if (C) {
            if (a.avail) {
                asm volatile("" : "+v"(lane));
#pragma unroll
                for (int i = 0; i < C; ++i)
                    if (lane + i * L < n_chunks) {
                        take_out<T>(a, x[i], row, lane + i * L);
                        forget(x[i]);
                        __builtin_amdgcn_sched_barrier(0);
                    }
            }
#pragma unroll
            for (int i = 0; i < C; ++i)
                if (lane + i * L < n_chunks)
#pragma unroll
                    for (int k = 0; k < V; ++k) m = fmaxf(m, static_cast<float>(x[i].e[k]));
            asm volatile("" : "+v"(lane));
            m = lanes_max<LW>(m);
            const float base = base_of(m);
#pragma unroll
            for (int i = 0; i < C; ++i)
                if (lane + i * L < n_chunks) {
                    forget(x[i]);
                    chunk_sums<T>(x[i], base, s, t);
                    __builtin_amdgcn_sched_barrier(0);
                }
        } else {
            // running maximum and sums of a lane, rescaled where a piece raises the maximum
            for (int c = lane; c < n_chunks; c += L) {
                const Chunk<T> y = load_chunk<T>(a, row_ptr, row, c);
                float mc = m;
#pragma unroll
                for (int k = 0; k < V; ++k) mc = fmaxf(mc, static_cast<float>(y.e[k]));
                if (mc > m) {
                    rebase(m, mc, s, t);
                    m = mc;
                }
                chunk_sums<T>(y, base_of(m), s, t);
            }
            const float mw = lanes_max<LW>(m);
            if (mw > m) rebase(m, mw, s, t);
            m = mw;
        }
        s = lanes_sum<LW>(s);
        t = lanes_sum<LW>(t);
        if (NW > 1) {
            const int wave = threadIdx.x >> 6;
            if ((threadIdx.x & 63) == 0) { merge[parity][wave][0] = m; merge[parity][wave][1] = s; merge[parity][wave][2] = t; }
            __syncthreads();
            float mm = neg_inf();
#pragma unroll
            for (int w = 0; w < NW; ++w) mm = fmaxf(mm, merge[parity][w][0]);
            s = 0.0f;
            t = 0.0f;
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                float sw = merge[parity][w][1], tw = merge[parity][w][2];
                rebase(merge[parity][w][0], mm, sw, tw);
                s += sw;
                t += tw;
            }
            m = mm;
            parity ^= 1;                                   // the next row's exchange does not overwrite one that is still read
        }
        if (lane == 0) sums.s[5] += in.weight;
        const float base = base_of(m);
        const bool possible = za != neg_inf() && !(m == neg_inf() && s == 0.0f);          // logits that are all NaN leave m at -inf and s NaN
        const RowGrad g = row_terms(a, in, inv_w, go, possible, exponent_of(za, base), s, t, lane == 0, sums);
        if (GRAD) {
            const bool nan = !(s + fabsf(g.c1) + fabsf(g.a1) + fabsf(g.a0) < __builtin_inff());
            asm volatile("" : "+v"(lane));
            if (C) {
#pragma unroll
                for (int i = 0; i < C; ++i) {
                    const int c = lane + i * L;
                    if (c < n_chunks) {
                        forget(x[i]);
                        Chunk<T> y = grad_chunk<T>(x[i], c, action, base, g, nan);
                        if (g.none) y.raw = u32x4{0, 0, 0, 0};
                        store_grad<T>(a, grad_ptr, i * L, lane, y);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            } else {
                for (int c = lane; c < n_chunks; c += L) {
                    Chunk<T> y = grad_chunk<T>(load_chunk<T>(a, row_ptr, row, c), c, action, base, g, nan);
                    if (g.none) y.raw = u32x4{0, 0, 0, 0};
                    store_grad<T>(a, grad_ptr, 0, c, y);
                }
            }
        }
    }
    RowSums mine = {};
    if (lane_of_row == 0) mine = sums;
    finish_sums(a, mine, parts);
}

template <typename T, bool GRAD>
void launch_policy_loss(const PolicyLossArgs &a, hipStream_t s, int *blocks) {
    // Lanes per row and 16-byte pieces per lane by the row's length (pieces of 4 f32 or 8 16-bit values)
    const int A = a.n_actions, chunks = (A + Chunk<T>::V - 1) / Chunk<T>::V;
    const auto grid = [&](int rows_per_block, int most) {
        *blocks = static_cast<int>(std::min<long long>(most, (a.rows + rows_per_block - 1) / rows_per_block));
        return dim3(*blocks);
    };
    // A row is held in registers up to 1024 lanes x 16 pieces: 64 K f32 or 128 K 16-bit actions.  Two rows or more a CU at once: 4096 pieces
    // as 512 x 8 or as 256 x 16 128 and 127 us (4096 x 32768 bf16); 6253 pieces as 512 x 16 103 us, as 1024 x 8, one row a CU, 122 us
    // (1023 x 50021 f16, forward and backward).
    const dim3 tiles = a.rows <= 2 * kRowTile ? dim3(1) : grid(kRowTile, kMaxBlocks);           // two tiles: one block, no launch to join
    if (a.rows <= 2 * kRowTile) *blocks = 1;
    if (A <= 16) {
        if (A <= 4) oc_policy_loss_rows_kernel<T, 4, false, GRAD><<<tiles, 256, 0, s>>>(a);
        else if (A == 5) oc_policy_loss_rows_kernel<T, 5, true, GRAD><<<tiles, 256, 0, s>>>(a);
        else if (A == 6) oc_policy_loss_rows_kernel<T, 6, true, GRAD><<<tiles, 256, 0, s>>>(a);
        else if (A <= 8) oc_policy_loss_rows_kernel<T, 8, false, GRAD><<<tiles, 256, 0, s>>>(a);
        else oc_policy_loss_rows_kernel<T, 16, false, GRAD><<<tiles, 256, 0, s>>>(a);
    }
    else if (chunks <= 16) oc_policy_loss_group_kernel<T, 16, 1, GRAD><<<grid(16, kMaxBlocks), 256, 0, s>>>(a);
    else if (chunks <= 64) oc_policy_loss_group_kernel<T, 16, 4, GRAD><<<grid(16, kMaxBlocks), 256, 0, s>>>(a);
    else if (chunks <= 64 * 4) oc_policy_loss_group_kernel<T, 64, 4, GRAD><<<grid(4, kMaxBlocks), 256, 0, s>>>(a);
    else if (chunks <= 256 * 4) oc_policy_loss_group_kernel<T, 256, 4, GRAD><<<grid(1, kMaxBlocks), 256, 0, s>>>(a);
    else if (chunks <= 512 * 8) oc_policy_loss_group_kernel<T, 512, 8, GRAD><<<grid(1, kMaxBlocks), 512, 0, s>>>(a);
    else if (chunks <= 512 * 16) oc_policy_loss_group_kernel<T, 512, 16, GRAD><<<grid(1, kMaxBlocks), 512, 0, s>>>(a);
    else if (chunks <= 1024 * 16) oc_policy_loss_group_kernel<T, 1024, 16, GRAD><<<grid(1, kMaxBlocks), 1024, 0, s>>>(a);
    else oc_policy_loss_group_kernel<T, 1024, 0, GRAD><<<grid(1, kMaxBlocks), 1024, 0, s>>>(a);
}

// Few rows: every block adds the weights up itself and saves the launch that does it (6 actions: 1000 rows the same, 4000 rows 19 us
// against 15, 8000 rows 25 against 15).
constexpr long long kSelfWeightRows = 1024;

template <bool GRAD>
void launch_policy_loss_type(const PolicyLossArgs &a, int type, hipStream_t s, int *blocks) {
    if (type == OC_F32) launch_policy_loss<float, GRAD>(a, s, blocks);
    else if (type == OC_BF16) launch_policy_loss<__bf16, GRAD>(a, s, blocks);
    else launch_policy_loss<_Float16, GRAD>(a, s, blocks);
}

}  // namespace

extern "C" int64_t oc_policy_loss_workspace_bytes(void) {
    return static_cast<int64_t>(kWeightBlocks + static_cast<int64_t>(kMaxBlocks) * kSums) * sizeof(double);
}

extern "C" int oc_policy_loss(const oc_policy_loss_args *p, int what, void *d_workspace, void *stream) {
    if (!p || what < OC_LOSS_FORWARD || what > OC_LOSS_BACKWARD)
        return oc_internal_fail(OC_ERR_INVALID_ARG, "oc_policy_loss: NULL arguments or an unknown pass");
    if (p->rows < 0 || p->n_actions < 1 || p->row_stride < p->n_actions || p->available_stride < 0)
        return oc_internal_fail(OC_ERR_INVALID_ARG, "oc_policy_loss: rows %lld, n_actions %d, row_stride %lld, available_stride %lld",
                                static_cast<long long>(p->rows), p->n_actions, static_cast<long long>(p->row_stride), static_cast<long long>(p->available_stride));
    if (p->logits_type < OC_F32 || p->logits_type > OC_F16 || p->action_type < OC_ACT_I32 || p->action_type > OC_ACT_F32)
        return oc_internal_fail(OC_ERR_INVALID_ARG, "oc_policy_loss: logits_type %d, action_type %d", p->logits_type, p->action_type);
    if ((p->rows > 0 && (!p->d_logits || !p->d_actions || !p->d_old_log_probs || !p->d_advantages)) ||
        (p->rows > 0 && what != OC_LOSS_FORWARD && !p->d_grad) || (what == OC_LOSS_BACKWARD ? !p->d_weight : !p->d_loss || !d_workspace))
        return oc_internal_fail(OC_ERR_INVALID_ARG, "oc_policy_loss: a required pointer is NULL");
    const uintptr_t element = p->logits_type == OC_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(p->d_logits) % element || reinterpret_cast<uintptr_t>(p->d_grad) % element ||
        reinterpret_cast<uintptr_t>(p->d_weight) % 8 || reinterpret_cast<uintptr_t>(d_workspace) % 8)
        return oc_internal_fail(OC_ERR_INVALID_ARG, "oc_policy_loss: a pointer is not aligned to its elements (workspace: 8 bytes)");
    if (p->n_actions > (1 << 28)) return oc_internal_fail(OC_ERR_UNSUPPORTED, "oc_policy_loss: n_actions %d beyond 2^28", p->n_actions);
    if (!(p->clip_param >= 0.0))
        return oc_internal_fail(OC_ERR_INVALID_ARG, "oc_policy_loss: clip_param %g", p->clip_param);
    if (p->rows == 0 && what == OC_LOSS_BACKWARD) return OC_OK;
    PolicyLossArgs a = {};
    a.logits = p->d_logits; a.actions = p->d_actions; a.old_logp = p->d_old_log_probs; a.adv = p->d_advantages;
    a.ref_logp = p->d_ref_log_probs; a.weights = p->d_active_masks; a.avail = p->d_available; a.grad = p->d_grad;
    a.grad_out = what == OC_LOSS_BACKWARD ? p->d_grad_out : nullptr;
    a.loss = p->d_loss; a.stats = p->d_stats; a.weight = p->d_weight;
    a.weight_partials = static_cast<double *>(d_workspace);
    a.sums = a.weight_partials + kWeightBlocks;
    a.rows = p->rows; a.row_stride = p->row_stride; a.avail_stride = p->available_stride;
    a.n_actions = p->n_actions; a.action_type = p->action_type; a.avail_u8 = p->available_u8 != 0;
    a.clip_lo = static_cast<float>(1.0 - p->clip_param); a.clip_hi = static_cast<float>(1.0 + p->clip_param);
    a.entropy_coef = p->entropy_coef; a.kl_coef = p->kl_coef; a.grad_scale = what == OC_LOSS_FORWARD ? 1.0f : p->grad_scale;
    const OcDeviceScope on_device(oc_device_of_pointer(what == OC_LOSS_BACKWARD ? static_cast<const void *>(p->d_weight) : p->d_loss));
    hipStream_t s = static_cast<hipStream_t>(stream);
    a.want_sums = what != OC_LOSS_BACKWARD;
    a.weight_from = what == OC_LOSS_FORWARD ? WEIGHT_NONE : what == OC_LOSS_BACKWARD ? WEIGHT_GIVEN : a.rows <= kSelfWeightRows ? WEIGHT_SELF : WEIGHT_PARTIALS;
    if (a.weight_from == WEIGHT_PARTIALS) {
        a.n_weight_partials = static_cast<int>(std::min<long long>(kWeightBlocks, (a.rows + 1023) / 1024));
        oc_policy_weight_kernel<<<dim3(a.n_weight_partials), 256, 0, s>>>(a);
    }
    int blocks = 0;
    // one block finishes by itself
    a.finalize_here = a.rows <= (a.n_actions <= 16 ? 2 * kRowTile : 1);
    if (a.rows == 0) {
        oc_policy_finalize_kernel<<<dim3(1), 1024, 0, s>>>(a, 0);
    } else {
        if (what == OC_LOSS_FORWARD) launch_policy_loss_type<false>(a, p->logits_type, s, &blocks);
        else launch_policy_loss_type<true>(a, p->logits_type, s, &blocks);
        if (a.want_sums && !a.finalize_here) oc_policy_finalize_kernel<<<dim3(1), 1024, 0, s>>>(a, blocks);
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? OC_OK : oc_internal_fail(OC_ERR_HIP, "oc_policy_loss: %s", hipGetErrorString(e));
}

// ======================================================================================================
// Clipped value loss and its gradient (train/MAPPO/r_mappo.py, cal_value_loss): per sample with target y = (return - mean) / std
//   e0 = y - v,  e1 = y - (v0 + clamp(v - v0, -c, c)),  loss = max(h(e0), h(e1)),  h(e) = e^2 / 2, or Huber's with delta;
//   d loss / d v = -h'(e0) where |v - v0| <= c or h(e0) >= h(e1), else 0 (the clamped branch does not move with v).
// 12..16 bytes read and 4 written per sample, nothing used twice: four samples per lane in one load each.  26.2 M f32 samples: forward
// 91 us (4.6 TB/s), backward 100 us (5.2 TB/s, a copy's rate).
// ======================================================================================================
namespace {

struct ValueLossArgs {
    const void *values;
    const float *preds, *returns, *weights;
    void *grad;
    const float *grad_out;
    float *loss;
    double *weight;
    double *weight_partials, *sums;                        // [kWeightBlocks], [blocks][2]
    long long n;
    float clip, delta, mean, std, grad_scale;              // clip < 0: not clipped; delta < 0: e^2 / 2
    int weight_from, n_weight_partials, finalize_here, want_sums;
};

__global__ __launch_bounds__(256) void oc_value_weight_kernel(const ValueLossArgs a) {
    __shared__ double part[4];
    double w = 0.0;
    const long long stride = static_cast<long long>(gridDim.x) * 256, n4 = a.n >> 2;
    for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < n4; i += stride) {
        const u32x4 q = reinterpret_cast<const u32x4_a4 *>(a.weights)[i];
        w += (static_cast<double>(__uint_as_float(q[0])) + __uint_as_float(q[1])) + (static_cast<double>(__uint_as_float(q[2])) + __uint_as_float(q[3]));
    }
    if (blockIdx.x == 0 && threadIdx.x < (a.n & 3)) w += a.weights[(n4 << 2) + threadIdx.x];
    w = block_sum(w, part);
    if (threadIdx.x == 0) a.weight_partials[blockIdx.x] = w;
}

__device__ __forceinline__ float value_sample(const ValueLossArgs &a, float v, float v0, float ret, float w, float scale, double &sum) {
    if (w == 0.0f) return 0.0f;
    const float y = (ret - a.mean) / a.std;
    const float e0 = y - v, step = v - v0;
    float h0, h1, slope;
    bool free_ = true;
    if (a.delta >= 0.0f) {
        h0 = fabsf(e0) <= a.delta ? 0.5f * e0 * e0 : a.delta * (fabsf(e0) - 0.5f * a.delta);
        slope = e0 > a.delta ? a.delta : e0 < -a.delta ? -a.delta : e0;       // a NaN stays
    } else {
        h0 = 0.5f * e0 * e0;
        slope = e0;
    }
    float worst = h0;
    if (a.clip >= 0.0f && !(fabsf(step) <= a.clip)) {       // also where v0 is not a number: neither is e1 then
        const float e1 = y - (v0 + copysignf(a.clip, step));
        h1 = a.delta >= 0.0f && fabsf(e1) > a.delta ? a.delta * (fabsf(e1) - 0.5f * a.delta) : 0.5f * e1 * e1;
        free_ = !(h0 < h1);
        worst = free_ ? h0 : h1;
        if (h1 != h1) worst = slope = h1;
    }
    sum += static_cast<double>(w) * static_cast<double>(worst);
    return free_ ? -scale * w * slope : 0.0f;
}

template <typename T, bool GRAD>
__global__ __launch_bounds__(256) void oc_value_loss_kernel(const ValueLossArgs a) {
    __shared__ double part[4];
    typedef T four_t __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    float scale = 0.0f;
    if (GRAD) {
        double w = 0.0;
        if (!a.weights) {
            w = static_cast<double>(a.n);
        } else if (a.weight_from == WEIGHT_SELF) {
            for (long long i = threadIdx.x; i < a.n; i += 256) w += a.weights[i];
            w = block_sum(w, part);
        } else if (a.weight_from == WEIGHT_PARTIALS) {
            for (int i = threadIdx.x; i < a.n_weight_partials; i += 256) w += a.weight_partials[i];
            w = block_sum(w, part);
        } else {
            w = *a.weight;
        }
        scale = w != 0.0 ? static_cast<float>(1.0 / w) * a.grad_scale * (a.grad_out ? *a.grad_out : 1.0f) : 0.0f;
    }
    double sum = 0.0, weight = 0.0;
    const long long n4 = a.n >> 2, stride = static_cast<long long>(gridDim.x) * 256;
    for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < n4; i += stride) {
        const four_t v = reinterpret_cast<const four_t *>(a.values)[i];
        const u32x4 v0 = reinterpret_cast<const u32x4_a4 *>(a.preds)[i], ret = reinterpret_cast<const u32x4_a4 *>(a.returns)[i];
        u32x4 w4 = {0x3f800000u, 0x3f800000u, 0x3f800000u, 0x3f800000u};
        if (a.weights) w4 = reinterpret_cast<const u32x4_a4 *>(a.weights)[i];
        four_t g;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float w = __uint_as_float(w4[k]);
            weight += static_cast<double>(w);
            g[k] = static_cast<T>(value_sample(a, static_cast<float>(v[k]), __uint_as_float(v0[k]), __uint_as_float(ret[k]), w, scale, sum));
        }
        if (GRAD) reinterpret_cast<four_t *>(a.grad)[i] = g;
    }
    if (blockIdx.x == 0 && threadIdx.x < (a.n & 3)) {
        const long long i = (n4 << 2) + threadIdx.x;
        const float w = a.weights ? a.weights[i] : 1.0f;
        weight += static_cast<double>(w);
        const float g = value_sample(a, static_cast<float>(static_cast<const T *>(a.values)[i]), a.preds[i], a.returns[i], w, scale, sum);
        if (GRAD) static_cast<T *>(a.grad)[i] = static_cast<T>(g);
    }
    if (!a.want_sums) return;
    sum = block_sum(sum, part);
    weight = block_sum(weight, part);
    if (threadIdx.x != 0) return;
    if (a.finalize_here) {
        *a.loss = static_cast<float>(weight != 0.0 ? sum / weight : 0.0);
        if (a.weight) *a.weight = weight;
    } else {
        a.sums[2 * blockIdx.x] = sum;
        a.sums[2 * blockIdx.x + 1] = weight;
    }
}

__global__ __launch_bounds__(256) void oc_value_finalize_kernel(const ValueLossArgs a, int blocks) {
    __shared__ double part[4];
    double sum = 0.0, weight = 0.0;
    for (int b = threadIdx.x; b < blocks; b += 256) {
        sum += a.sums[2 * b];
        weight += a.sums[2 * b + 1];
    }
    sum = block_sum(sum, part);
    weight = block_sum(weight, part);
    if (threadIdx.x == 0) {
        *a.loss = static_cast<float>(weight != 0.0 ? sum / weight : 0.0);
        if (a.weight) *a.weight = weight;
    }
}

template <typename T>
void launch_value_loss(const ValueLossArgs &a, int grad, int blocks, hipStream_t s) {
    if (grad) oc_value_loss_kernel<T, true><<<dim3(blocks), 256, 0, s>>>(a);
    else oc_value_loss_kernel<T, false><<<dim3(blocks), 256, 0, s>>>(a);
}

}  // namespace

extern "C" int64_t oc_value_loss_workspace_bytes(void) { return static_cast<int64_t>(kWeightBlocks + 2 * kMaxBlocks) * sizeof(double); }

extern "C" int oc_value_loss(const oc_value_loss_args *p, int what, void *d_workspace, void *stream) {
    if (!p || what < OC_LOSS_FORWARD || what > OC_LOSS_BACKWARD)
        return oc_internal_fail(OC_ERR_INVALID_ARG, "oc_value_loss: NULL arguments or an unknown pass");
    if (p->n < 0 || p->values_type < OC_F32 || p->values_type > OC_F16)
        return oc_internal_fail(OC_ERR_INVALID_ARG, "oc_value_loss: n %lld, values_type %d", static_cast<long long>(p->n), p->values_type);
    if ((p->n > 0 && (!p->d_values || !p->d_value_preds || !p->d_returns)) || (p->n > 0 && what != OC_LOSS_FORWARD && !p->d_grad) ||
        (what == OC_LOSS_BACKWARD ? !p->d_weight : !p->d_loss || !d_workspace))
        return oc_internal_fail(OC_ERR_INVALID_ARG, "oc_value_loss: a required pointer is NULL");
    const uintptr_t element = p->values_type == OC_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(p->d_values) % element || reinterpret_cast<uintptr_t>(p->d_grad) % element ||
        reinterpret_cast<uintptr_t>(p->d_weight) % 8 || reinterpret_cast<uintptr_t>(d_workspace) % 8)
        return oc_internal_fail(OC_ERR_INVALID_ARG, "oc_value_loss: a pointer is not aligned to its elements (workspace: 8 bytes)");
    if (!(p->std > 0.0f)) return oc_internal_fail(OC_ERR_INVALID_ARG, "oc_value_loss: std %g", static_cast<double>(p->std));
    if (p->n == 0 && what == OC_LOSS_BACKWARD) return OC_OK;
    ValueLossArgs a = {};
    a.values = p->d_values; a.preds = p->d_value_preds; a.returns = p->d_returns; a.weights = p->d_active_masks;
    a.grad = p->d_grad; a.grad_out = what == OC_LOSS_BACKWARD ? p->d_grad_out : nullptr; a.loss = p->d_loss; a.weight = p->d_weight;
    a.weight_partials = static_cast<double *>(d_workspace);
    a.sums = a.weight_partials + kWeightBlocks;
    a.n = p->n;
    a.clip = p->clip_param; a.delta = p->huber_delta; a.mean = p->mean; a.std = p->std;
    a.grad_scale = what == OC_LOSS_FORWARD ? 1.0f : p->grad_scale;
    a.want_sums = what != OC_LOSS_BACKWARD;
    const OcDeviceScope on_device(oc_device_of_pointer(what == OC_LOSS_BACKWARD ? static_cast<const void *>(p->d_weight) : p->d_loss));
    hipStream_t s = static_cast<hipStream_t>(stream);
    a.weight_from = what == OC_LOSS_FORWARD ? WEIGHT_NONE : what == OC_LOSS_BACKWARD ? WEIGHT_GIVEN : a.n <= kSelfWeightRows ? WEIGHT_SELF : WEIGHT_PARTIALS;
    if (a.weight_from == WEIGHT_PARTIALS && a.weights) {
        a.n_weight_partials = static_cast<int>(std::min<long long>(kWeightBlocks, (a.n + 1023) / 1024));
        oc_value_weight_kernel<<<dim3(a.n_weight_partials), 256, 0, s>>>(a);
    }
    const int blocks = static_cast<int>(std::min<long long>(kMaxBlocks, (a.n + 1023) / 1024));
    a.finalize_here = blocks == 1;
    if (a.n == 0) {
        oc_value_finalize_kernel<<<dim3(1), 256, 0, s>>>(a, 0);
    } else {
        if (p->values_type == OC_F32) launch_value_loss<float>(a, what != OC_LOSS_FORWARD, blocks, s);
        else if (p->values_type == OC_BF16) launch_value_loss<__bf16>(a, what != OC_LOSS_FORWARD, blocks, s);
        else launch_value_loss<_Float16>(a, what != OC_LOSS_FORWARD, blocks, s);
        if (a.want_sums && !a.finalize_here) oc_value_finalize_kernel<<<dim3(1), 256, 0, s>>>(a, blocks);
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? OC_OK : oc_internal_fail(OC_ERR_HIP, "oc_value_loss: %s", hipGetErrorString(e));
}

// ======================================================================================================
// Global norm of many gradient tensors and clipping (train/MAPPO/r_mappo.py clips each network's gradients with
// torch.nn.utils.clip_grad_norm_; get_gard_norm of utils/util.py is the norm alone):
//   norm = sqrt(sum g^2) over all elements of all tensors, or max |g|;  g <- g * min(1, max_norm / (norm + 1e-6)).
// Two passes, because the factor needs every element: read all, then read and write all.  The tensors' addresses travel in the kernel
// arguments of the first pass (no table to copy, nothing kept between calls), kTensors a launch; its blocks leave a note of the piece
// that they read, and the second pass is one launch over all notes, last piece first: what the caches still hold is read from there.
// The squares are added in f64: neither 1e-30 nor 1e30 leaves the range, and the order of the sums does not show.  The second pass adds
// up the first one's partial sums in every block (many: a launch between them does).  566 M elements, bf16 among f32 (1.13 GB): 245 + 8 +
// 411 us, 4.6 TB/s read, then 5.5 TB/s.
// ======================================================================================================
namespace {

constexpr int kTensors = 120;                              // kernel arguments stay below 4 KB
constexpr int kNormBlocks = 16384;                         // pieces that the elements are cut into, beside one per tensor: short ones, so that
                                                           // the last round of blocks is short (4096 pieces: 275 us for 1.13 GB instead of 245)
constexpr int kJoinHere = 1024;                            // up to so many partial sums every block of the second pass adds up by itself, which
                                                           // saves a launch of 5 us where that is half of the call; 14900 in every block: 441 us
                                                           // for the second pass instead of 411
constexpr long long kPiece = 4096;                         // and their unit

struct Piece {                                             // what a block of the first pass has read
    const void *src;
    void *dst;
    int n, type;
};

struct NormArgs {
    const void *src[kTensors];
    void *dst[kTensors];
    long long numel[kTensors];
    int first_block[kTensors + 1];                         // of this launch
    uint8_t type[kTensors];
    long long piece;
    double *partials;                                      // of the whole call
    Piece *notes;
    int n, block0, inf_norm;
};
static_assert(sizeof(NormArgs) <= 4096, "kernel arguments");

struct ClipArgs {
    const double *partials;
    const Piece *notes;
    float *norm;
    float max_norm;
    int n_partials, inf_norm, in_place;
    int joined;                                            // *norm holds the norm already
};

__device__ __forceinline__ int tensor_of_block(const NormArgs &a, int block) {
    int lo = 0, hi = a.n;                                  // first_block[lo] <= block < first_block[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.first_block[mid] <= block) lo = mid; else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ double join(double x, double y, int inf_norm) {
    if (!inf_norm) return x + y;
    return x != x || y != y ? x + y : fmax(x, y);           // a NaN stays
}

__device__ __forceinline__ double block_join(double x, int inf_norm, double *part) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) x = join(x, __shfl_xor(x, off), inf_norm);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
    __syncthreads();
    return join(join(part[0], part[1], inf_norm), join(part[2], part[3], inf_norm), inf_norm);
}

template <typename T>
__device__ __forceinline__ double norm_of_piece(const T *p, long long n, int inf_norm) {
    constexpr int V = 16 / sizeof(T);
    typedef typename Unaligned<sizeof(T)>::type U;
    double sum[4] = {0, 0, 0, 0};
    const long long chunks = n / V;
    const auto take = [&](const Chunk<T> &c) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const float f = static_cast<float>(c.e[k]);
            if (inf_norm) {
                sum[k & 3] = join(sum[k & 3], static_cast<double>(fabsf(f)), 1);
            } else {
                const double d = static_cast<double>(f);
                sum[k & 3] = fma(d, d, sum[k & 3]);
            }
        }
    };
    long long i = threadIdx.x;
    for (; i + 768 < chunks; i += 1024) {                  // four loads in flight
        Chunk<T> c[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) c[u].raw = reinterpret_cast<const U *>(p)[i + 256 * u];
#pragma unroll
        for (int u = 0; u < 4; ++u) take(c[u]);
    }
    for (; i < chunks; i += 256) {
        Chunk<T> c;
        c.raw = reinterpret_cast<const U *>(p)[i];
        take(c);
    }
    for (long long j = chunks * V + threadIdx.x; j < n; j += 256) {
        const double d = static_cast<double>(static_cast<float>(p[j]));
        sum[0] = inf_norm ? join(sum[0], fabs(d), 1) : fma(d, d, sum[0]);
    }
    return join(join(sum[0], sum[1], inf_norm), join(sum[2], sum[3], inf_norm), inf_norm);
}

__global__ __launch_bounds__(256) void oc_grad_norm_kernel(const NormArgs a) {
    __shared__ double part[4];
    const int t = tensor_of_block(a, blockIdx.x);
    const long long from = (static_cast<long long>(blockIdx.x) - a.first_block[t]) * a.piece;
    const long long n = a.numel[t] - from < a.piece ? a.numel[t] - from : a.piece;
    double x = 0.0;
    if (n > 0) {
        if (a.type[t] == OC_F32) x = norm_of_piece(static_cast<const float *>(a.src[t]) + from, n, a.inf_norm);
        else if (a.type[t] == OC_BF16) x = norm_of_piece(static_cast<const __bf16 *>(a.src[t]) + from, n, a.inf_norm);
        else x = norm_of_piece(static_cast<const _Float16 *>(a.src[t]) + from, n, a.inf_norm);
    }
    x = block_join(x, a.inf_norm, part);
    if (threadIdx.x == 0) {
        const long long size = a.type[t] == OC_F32 ? 4 : 2;
        a.partials[a.block0 + blockIdx.x] = x;
        a.notes[a.block0 + blockIdx.x] = Piece{static_cast<const char *>(a.src[t]) + from * size, static_cast<char *>(a.dst[t]) + from * size,
                                               static_cast<int>(n), a.type[t]};
    }
}

__device__ __forceinline__ float total_norm(const ClipArgs &a, double *part) {
    double x = 0.0;
#pragma unroll 8
    for (int i = threadIdx.x; i < a.n_partials; i += 256) x = join(x, a.partials[i], a.inf_norm);
    x = block_join(x, a.inf_norm, part);
    return static_cast<float>(a.inf_norm ? x : sqrt(x));
}

template <typename T>
__device__ __forceinline__ void scale_piece(const T *src, T *dst, long long n, float f) {
    constexpr int V = 16 / sizeof(T);
    typedef typename Unaligned<sizeof(T)>::type U;
    const long long chunks = n / V;
    const auto scaled = [&](Chunk<T> c) {
#pragma unroll
        for (int k = 0; k < V; ++k) c.e[k] = static_cast<T>(static_cast<float>(c.e[k]) * f);
        return c.raw;
    };
    long long i = threadIdx.x;
    for (; i + 768 < chunks; i += 1024) {
        Chunk<T> c[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) c[u].raw = reinterpret_cast<const U *>(src)[i + 256 * u];
#pragma unroll
        for (int u = 0; u < 4; ++u) reinterpret_cast<U *>(dst)[i + 256 * u] = scaled(c[u]);
    }
    for (; i < chunks; i += 256) {
        Chunk<T> c;
        c.raw = reinterpret_cast<const U *>(src)[i];
        reinterpret_cast<U *>(dst)[i] = scaled(c);
    }
    for (long long j = chunks * V + threadIdx.x; j < n; j += 256) dst[j] = static_cast<T>(static_cast<float>(src[j]) * f);
}

__global__ __launch_bounds__(1024) void oc_grad_join_kernel(const ClipArgs a) {
    __shared__ double part[16];
    double x = 0.0;
#pragma unroll 8
    for (int i = threadIdx.x; i < a.n_partials; i += 1024) x = join(x, a.partials[i], a.inf_norm);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) x = join(x, __shfl_xor(x, off), a.inf_norm);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
        for (int w = 1; w < 16; ++w) x = join(x, part[w], a.inf_norm);
        *a.norm = static_cast<float>(a.inf_norm ? x : sqrt(x));
    }
}

__global__ __launch_bounds__(256) void oc_grad_clip_kernel(const ClipArgs a) {
    __shared__ double part[4];
    const float norm = a.joined ? *a.norm : total_norm(a, part);
    if (!a.joined && blockIdx.x == 0 && threadIdx.x == 0) *a.norm = norm;
    if (a.max_norm < 0.0f || a.n_partials == 0) return;    // the norm alone, or no element at all
    const float factor = a.max_norm / (norm + 1e-6f);
    const float f = factor > 1.0f ? 1.0f : factor;         // a NaN norm makes every gradient NaN, as the product does
    if (a.in_place && f == 1.0f) return;                   // nothing to clip: the gradients stay as they are
    const Piece p = a.notes[a.n_partials - 1 - blockIdx.x];
    if (p.type == OC_F32) scale_piece(static_cast<const float *>(p.src), static_cast<float *>(p.dst), p.n, f);
    else if (p.type == OC_BF16) scale_piece(static_cast<const __bf16 *>(p.src), static_cast<__bf16 *>(p.dst), p.n, f);
    else scale_piece(static_cast<const _Float16 *>(p.src), static_cast<_Float16 *>(p.dst), p.n, f);
}

}  // namespace

extern "C" int64_t oc_grad_norm_workspace_bytes(int32_t n_tensors) {
    return n_tensors < 0 ? -1 : (static_cast<int64_t>(kNormBlocks) + n_tensors) * static_cast<int64_t>(sizeof(double) + sizeof(Piece));
}

extern "C" int oc_grad_norm_clip(int32_t n_tensors, const void *const *d_grads, void *const *d_out, const int64_t *numel, const int32_t *types,
                                 float max_norm, int inf_norm, float *d_norm, void *d_workspace, void *stream) {
    if (n_tensors < 0 || !d_norm || !d_workspace || (n_tensors > 0 && (!d_grads || !numel || !types)))
        return oc_internal_fail(OC_ERR_INVALID_ARG, "oc_grad_norm_clip: n_tensors %d or a required pointer is NULL", n_tensors);
    if (reinterpret_cast<uintptr_t>(d_workspace) % 8 || max_norm != max_norm)
        return oc_internal_fail(OC_ERR_INVALID_ARG, "oc_grad_norm_clip: workspace not aligned to 8 bytes, or max_norm is NaN");
    long long total = 0;
    for (int i = 0; i < n_tensors; ++i) {
        if (numel[i] < 0 || types[i] < OC_F32 || types[i] > OC_F16)
            return oc_internal_fail(OC_ERR_INVALID_ARG, "oc_grad_norm_clip: tensor %d has %lld elements of type %d", i, static_cast<long long>(numel[i]), types[i]);
        const uintptr_t element = types[i] == OC_F32 ? 4 : 2;
        const uintptr_t src = reinterpret_cast<uintptr_t>(d_grads[i]), dst = d_out ? reinterpret_cast<uintptr_t>(d_out[i]) : src;
        if (numel[i] > 0 && (!src || !dst || src % element || dst % element))
            return oc_internal_fail(OC_ERR_INVALID_ARG, "oc_grad_norm_clip: tensor %d is NULL or not aligned to its elements", i);
        total += numel[i];
    }
    // pieces of one size: at most kNormBlocks of them, and one more per tensor for its rest
    const long long piece = std::max<long long>(kPiece, ((total + kNormBlocks - 1) / kNormBlocks + kPiece - 1) / kPiece * kPiece);
    if (piece > 0x7fffffffLL) return oc_internal_fail(OC_ERR_UNSUPPORTED, "oc_grad_norm_clip: %lld elements", total);
    const OcDeviceScope on_device(oc_device_of_pointer(d_norm));
    hipStream_t s = static_cast<hipStream_t>(stream);
    double *partials = static_cast<double *>(d_workspace);
    Piece *notes = reinterpret_cast<Piece *>(partials + kNormBlocks + n_tensors);
    int block0 = 0;
    for (int i = 0; i < n_tensors;) {
        NormArgs a;
        a.n = 0;
        a.piece = piece; a.partials = partials; a.notes = notes; a.block0 = block0; a.inf_norm = inf_norm != 0;
        int blocks = 0;
        for (; i < n_tensors && a.n < kTensors; ++i) {
            if (numel[i] == 0) continue;
            a.src[a.n] = d_grads[i];
            a.dst[a.n] = d_out ? d_out[i] : const_cast<void *>(d_grads[i]);
            a.numel[a.n] = numel[i];
            a.type[a.n] = static_cast<uint8_t>(types[i]);
            a.first_block[a.n++] = blocks;
            blocks += static_cast<int>((numel[i] + piece - 1) / piece);
        }
        if (!blocks) continue;
        a.first_block[a.n] = blocks;
        oc_grad_norm_kernel<<<dim3(blocks), 256, 0, s>>>(a);
        block0 += blocks;
    }
    const ClipArgs c = {partials, notes, d_norm, max_norm, block0, inf_norm != 0, d_out == nullptr, block0 > kJoinHere || max_norm < 0.0f};
    if (c.joined) oc_grad_join_kernel<<<dim3(1), 1024, 0, s>>>(c);
    if (max_norm >= 0.0f) oc_grad_clip_kernel<<<dim3(block0 ? block0 : 1), 256, 0, s>>>(c);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? OC_OK : oc_internal_fail(OC_ERR_HIP, "oc_grad_norm_clip: %s", hipGetErrorString(e));
}
