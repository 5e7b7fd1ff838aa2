// Routing rows to experts: scores, the choice, its weights and their gradient, and the rows listed by expert.
//
// With logits l[row, e] and an optional bias b[e]
//     s = softmax(l) or sigmoid(l),   key = s + b   (without a bias key = l, which orders like s),
// the experts of the best `top_groups` of `n_groups` equal groups stay (a group ranks by its largest key, or by the sum of
// its two largest values s + b), the top_k largest keys of those are chosen, the lowest index first among equals, and
//     w_j = scale * s_j      or, renormalised,   w_j = scale * s_j / sum over the chosen i of s_i.
// An expert whose logit or key is -inf or NaN is never chosen; where fewer than top_k are left the id is -1, the weight 0.
#include "mps.h"

#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <cmath>

#include "mps_internal.h"
#include "mps_tc.cuh"
#include "mps_types.cuh"

namespace cg = cooperative_groups;
using mps::fail;
using mps::to_f32;

namespace {

#define RT_CUDA(call)                                                                               \
    do {                                                                                            \
        cudaError_t e_ = (call);                                                                    \
        if (e_ != cudaSuccess) return fail(MPS_ERR_CUDA, "%s: %s", #call, cudaGetErrorString(e_));  \
    } while (0)

__device__ int g_status;
__global__ void clear_status(int bits) { atomicAnd(&g_status, ~bits); }

constexpr int kMaxExperts = 1024;   // 32 keys per lane
constexpr int kMaxTop = 32;         // one chosen expert per lane
constexpr int kMaxGroups = 32;      // one bit per expert group
constexpr int kRouteWarps = 4;
constexpr unsigned kAll = 0xffffffffu;

struct RouteArgs {
    int n_rows, n_experts, top_k, n_groups, per_group, top_groups, group_top;
    unsigned group_inverse;  // 2^32 / per_group rounded up: experts stay below 2^16, so mulhi by it is the quotient (0: per_group 1)
    bool renormalise;
    float scale;
};

template <typename F>
__device__ __forceinline__ F neg_inf();
template <>
__device__ __forceinline__ float neg_inf<float>() { return -INFINITY; }
template <>
__device__ __forceinline__ double neg_inf<double>() { return -(double)INFINITY; }

__device__ __forceinline__ float sigmoid(float x) {  // exp of a number <= 0 only: no overflow, and small scores keep their digits
    const float e = expf(x < 0.0f ? x : -x);
    return (x < 0.0f ? e : 1.0f) / (1.0f + e);
}

template <typename F>
__device__ __forceinline__ F warp_sum(F v) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(kAll, v, d);
    return v;
}

template <typename F>
__device__ __forceinline__ F warp_max(F v) {
#pragma unroll
    for (int d = 16; d; d >>= 1) {
        const F o = __shfl_xor_sync(kAll, v, d);
        v = o > v ? o : v;
    }
    return v;
}

// fp32 -> unsigned with the same order (no NaN comes in; -0 counts as 0)
__device__ __forceinline__ unsigned ordered(float v) {
    const unsigned b = __float_as_uint(v + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// the largest (value, lowest index) of the warp's candidates
__device__ __forceinline__ void warp_best(float &v, int &at) {
    const unsigned mine = ordered(v), top = __reduce_max_sync(kAll, mine);
    at = (int)__reduce_min_sync(kAll, mine == top ? (unsigned)at : 0x7fffffffu);
    v = __uint_as_float(top & 0x80000000u ? top ^ 0x80000000u : ~top);
}
__device__ __forceinline__ void warp_best(double &v, int &at) {  // by the two halves of an integer that orders like the double
    const long long bits = __double_as_longlong(v + 0.0);
    const unsigned long long o = bits < 0 ? ~(unsigned long long)bits : (unsigned long long)bits | 1ull << 63;
    const unsigned hi = (unsigned)(o >> 32), top_hi = __reduce_max_sync(kAll, hi);
    const unsigned lo = hi == top_hi ? (unsigned)o : 0u, top_lo = __reduce_max_sync(kAll, lo);
    at = (int)__reduce_min_sync(kAll, hi == top_hi && lo == top_lo ? (unsigned)at : 0x7fffffffu);
    const unsigned long long top = (unsigned long long)top_hi << 32 | top_lo;
    v = __longlong_as_double((long long)(top >> 63 ? top ^ 1ull << 63 : ~top));
}

// Sigmoid and exponential of the keys, which only have to order.  __expf is off by (2 + 1.173 |x|) 2^-23 of the result, which
// keeps 1 / (1 + e^-x) within 5e-7 (|x| e^-|x| is bounded; below -80 the score counts as e^-80).
__device__ __forceinline__ float key_sigmoid(float x) { return __fdividef(1.0f, 1.0f + __expf(fminf(-x, 80.0f))); }
__device__ __forceinline__ double key_sigmoid(double x) {
    const double e = exp(x < 0 ? x : -x);
    return (x < 0 ? e : 1.0) / (1.0 + e);
}
__device__ __forceinline__ float key_exp(float x) { return __expf(x); }
__device__ __forceinline__ double key_exp(double x) { return exp(x); }
__device__ __forceinline__ float key_div(float x, float y) { return __fdividef(x, y); }
__device__ __forceinline__ double key_div(double x, double y) { return x / y; }

// How far apart two fp32 keys must be for their order to be that of the exact ones.  A sigmoid is off by at most 5e-7 (the
// errors above), a softmax by 3e-6 (its denominator adds up to 37 roundings), a key s + b by another half unit of itself; twice
// that for two keys.
template <bool SIGMOID>
__device__ __forceinline__ float clearance(float key) { return (SIGMOID ? 1e-6f : 6e-6f) + 2.5e-7f * fabsf(key); }
// How far a group's fp32 rank may be off: half of that for each of the keys it is made of, which may cancel, and the sum's rounding.
template <bool SIGMOID>
__device__ __forceinline__ float rank_error(float one, float two, bool both) {
    return 0.5f * clearance<SIGMOID>(one) + (both ? 0.5f * clearance<SIGMOID>(two) + 6e-8f * fabsf(one + two) : 0.0f);
}

// Keeps the experts of the best groups: key of the others becomes -inf.  `cells` is this warp's shared row of n_experts
// (+ padding) values.  Returns false where fp32 cannot tell the last group kept from the first one dropped.
template <bool SIGMOID, typename F, int VPL>
__device__ __forceinline__ bool keep_groups(F (&key)[VPL], const F (&value)[VPL], const RouteArgs &a, F *cells, int lane) {
    // groups are contiguous runs of experts; `parts` lanes share a group, each scanning every parts-th member
    int parts = 32;
    while (parts * a.n_groups > 32) parts >>= 1;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        const int e = lane + 32 * i;
        if (e < a.n_experts) cells[e + (e >> 5)] = value[i];
    }
    __syncwarp();
    const int g = lane / parts;
    F one = neg_inf<F>(), two = neg_inf<F>();
    if (g < a.n_groups)
        for (int m = lane % parts; m < a.per_group; m += parts) {
            const int e = g * a.per_group + m;
            const F v = cells[e + (e >> 5)];
            if (v > one) { two = one; one = v; }
            else if (v > two) two = v;
        }
    for (int d = 1; d < parts; d <<= 1) {
        const F o1 = __shfl_xor_sync(kAll, one, d), o2 = __shfl_xor_sync(kAll, two, d);
        const F low = one < o1 ? one : o1;
        one = one > o1 ? one : o1;
        two = two > o2 ? two : o2;
        two = two > low ? two : low;
    }
    F rank = one;
    const bool both = a.group_top == 2 && two > neg_inf<F>();
    if (both) rank = one + two;
    if (g >= a.n_groups || lane % parts) rank = neg_inf<F>();
    const F own = rank;
    unsigned kept = 0;
    for (int j = 0; j < a.top_groups; ++j) {
        F best = rank;
        int at = lane;
        warp_best(best, at);
        if (!(best > neg_inf<F>())) break;
        kept |= 1u << (at / parts);
        if (lane == at) rank = neg_inf<F>();
    }
    bool clear = true;
    if (sizeof(F) == 4) {
        const float off = rank_error<SIGMOID>((float)one, (float)two, both);
        const float least = -warp_max(rank != own ? off - (float)own : -INFINITY), most = warp_max(rank > neg_inf<F>() ? (float)rank + off : -INFINITY);
        // the sum of two keys of the type's lowest or largest value has left fp32, though neither key has
        const bool beyond = (float)one > -INFINITY && !(fabsf((float)own) < INFINITY) && g < a.n_groups && lane % parts == 0;
        const bool none_beyond = !__any_sync(kAll, beyond);
        clear = least > most && none_beyond;
    }
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        const int e = lane + 32 * i;
        const int at = a.group_inverse ? (int)__umulhi((unsigned)e, a.group_inverse) : e;
        if (e < a.n_experts && !((kept >> at) & 1)) key[i] = neg_inf<F>();
    }
    return clear;
}

// The top_k largest keys: lane j returns the j-th expert (or -1) in `mine`.  Every lane keeps the best two of its keys at hand, so
// that most picks cost two warp reductions and no pass over the keys.  EXACT keys are compared as they are; others must be
// `clearance` apart unless they belong to equal logits and equal biases, and so must the last pick and every key that is left (not
// the next one alone: behind one that equals the last pick there may be one that only seems to).  Returns false where they are not.
template <bool EXACT, bool SIGMOID, typename F, int VPL, typename T>
__device__ __forceinline__ bool choose(F (&key)[VPL], const RouteArgs &a, const T *logits, const float *bias, int lane, int &mine) {
    F one, two;
    int one_at, two_at;
    auto scan = [&]() {  // the lane's best two, the lower index first among equals
        one = two = neg_inf<F>();
        one_at = two_at = 0;
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            const bool first = key[i] > one, second = key[i] > two;
            two = first ? one : second ? key[i] : two;
            two_at = first ? one_at : second ? i : two_at;
            one = first ? key[i] : one;
            one_at = first ? i : one_at;
        }
    };
    scan();
    mine = -1;
    bool clear = true;
    float prev = INFINITY;
    int prev_at = -1;
    auto equal = [&](int e, int o) { return to_f32(logits[e]) == to_f32(logits[o]) && bias[e] == bias[o]; };
    for (int j = 0; j < a.top_k; ++j) {
        F best = one;
        int at = lane + 32 * one_at;
        warp_best(best, at);
        if (!(best > neg_inf<F>())) {
            prev_at = -1;  // nothing is left
            break;
        }
        if (!EXACT) {
            const float v = (float)best;
            clear = !(prev_at >= 0 && prev - v <= clearance<SIGMOID>(v)) || equal(prev_at, at);
            if (!clear) break;
            prev = v;
            prev_at = at;
        }
        if (lane == j) mine = at;
        if ((at & 31) == lane) {
#pragma unroll
            for (int i = 0; i < VPL; ++i)
                if (i == one_at) key[i] = neg_inf<F>();
            if (two > neg_inf<F>()) {
                one = two;
                one_at = two_at;
                two = neg_inf<F>();
            } else scan();
        }
    }
    if (!EXACT && clear && prev_at >= 0 && __any_sync(kAll, prev - (float)one <= clearance<SIGMOID>((float)one))) {
        bool close = false;
#pragma unroll
        for (int i = 0; i < VPL; ++i)
            if (key[i] > neg_inf<F>() && prev - (float)key[i] <= clearance<SIGMOID>((float)key[i])) close = close || !equal(prev_at, lane + 32 * i);
        clear = !__any_sync(kAll, close);
    }
    return clear;
}

// keys and group values of one row in F; -inf where the expert may not be chosen
template <typename F, int VPL, bool SIGMOID>
__device__ __forceinline__ void row_keys(const float (&l)[VPL], const float (&b)[VPL], bool has_bias, bool need_score, F (&key)[VPL], F (&value)[VPL]) {
    F peak = neg_inf<F>(), total = 0;
    if (need_score && !SIGMOID) {
#pragma unroll
        for (int i = 0; i < VPL; ++i)
            if ((F)l[i] > peak) peak = (F)l[i];
        peak = warp_max(peak);
#pragma unroll
        for (int i = 0; i < VPL; ++i)
            if (l[i] > -INFINITY) total += key_exp((F)l[i] - peak);
        total = warp_sum(total);
    }
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        const bool open = l[i] > -INFINITY;
        F s = 0;
        if (need_score && open) {
            s = SIGMOID ? key_sigmoid((F)l[i]) : key_div(key_exp((F)l[i] - peak), total);
        }
        F k = has_bias ? s + (F)b[i] : (F)l[i];
        if (!open || !(k > neg_inf<F>())) k = neg_inf<F>();
        key[i] = k;
        value[i] = has_bias || !need_score ? k : (open ? s : neg_inf<F>());
    }
}

// A row decided exactly (logits as they are, scores in fp64): lane j returns the j-th expert.  Out of line, so that the few rows that need it do not cost the
// others their registers.
template <typename T, int VPL, bool SIGMOID>
__device__ __noinline__ int decide_exactly(const RouteArgs &a, const T *line, const float *bias, double *cells, int lane) {
    float l[VPL], b[VPL];
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        const int e = lane + 32 * i;
        l[i] = e < a.n_experts ? to_f32(line[e]) : -INFINITY;
        b[i] = bias && e < a.n_experts ? bias[e] : 0.0f;
        if (l[i] != l[i]) l[i] = -INFINITY;
    }
    int mine;
    if (!bias && (a.n_groups == 1 || a.group_top == 1)) {  // the logits themselves are compared
        float key[VPL], value[VPL];
        row_keys<float, VPL, SIGMOID>(l, b, false, false, key, value);
        if (a.n_groups > 1) keep_groups<SIGMOID>(key, value, a, (float *)cells, lane);
        choose<true, SIGMOID>(key, a, line, bias, lane, mine);
        return mine;
    }
    double key[VPL], value[VPL];
    row_keys<double, VPL, SIGMOID>(l, b, bias != nullptr, true, key, value);
    if (a.n_groups > 1) keep_groups<SIGMOID>(key, value, a, cells, lane);
    choose<true, SIGMOID>(key, a, line, bias, lane, mine);
    return mine;
}

// One warp per row.  The row's logits stay in registers (lane + 32 i); the choice runs on fp32 keys, and a row in which two
// keys that decide it lie closer together than fp32 can tell is decided again on fp64 keys.  That keeps the choice the
// definition's at a fraction of the cost of fp64 throughout.
template <typename T, int VPL, bool SIGMOID>
__global__ void __launch_bounds__(32 * kRouteWarps, VPL <= 8 ? 8 : 1) route_kernel(const RouteArgs a, const T *__restrict__ logits, const float *__restrict__ bias,
                                                                int *__restrict__ ids, float *__restrict__ weights) {
    extern __shared__ double s_cells[];
    mps::let_next_launch_start();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int pitch = a.n_experts + (a.n_experts >> 5) + 1;
    double *cells = s_cells + (size_t)warp * pitch;
    const bool has_bias = bias != nullptr, grouped = a.n_groups > 1;
    const bool need_score = has_bias || (grouped && a.group_top == 2);
    float b[VPL];
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        const int e = lane + 32 * i;
        b[i] = has_bias && e < a.n_experts ? bias[e] : 0.0f;
    }
    for (long long row = (long long)blockIdx.x * kRouteWarps + warp; row < a.n_rows; row += (long long)gridDim.x * kRouteWarps) {
        const T *line = logits + row * a.n_experts;
        float l[VPL], peak = 0.0f, total = 1.0f;
        bool nan = false;
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            const int e = lane + 32 * i;
            l[i] = e < a.n_experts ? to_f32(line[e]) : -INFINITY;
            nan = nan || !(SIGMOID ? l[i] <= INFINITY : l[i] < INFINITY);  // the row's scores are not numbers: neither are its weights
            if (l[i] != l[i]) l[i] = -INFINITY;
        }
        nan = __any_sync(kAll, nan);
        if (!SIGMOID && !a.renormalise) {  // the denominator of the weights
            peak = l[0];
            total = 0.0f;
#pragma unroll
            for (int i = 1; i < VPL; ++i) peak = fmaxf(peak, l[i]);
            peak = warp_max(peak);
#pragma unroll
            for (int i = 0; i < VPL; ++i)
                if (l[i] > -INFINITY) total += expf(l[i] - peak);
            total = warp_sum(total);
        }
        float key[VPL], value[VPL];
        row_keys<float, VPL, SIGMOID>(l, b, has_bias, need_score, key, value);
        bool clear = true;
        int mine;
        if (grouped) {
            clear = keep_groups<SIGMOID>(key, value, a, (float *)cells, lane);
            if (!need_score) clear = true;  // logits compare exactly
        }
        if (has_bias) clear = choose<false, SIGMOID>(key, a, line, bias, lane, mine) && clear;
        else choose<true, SIGMOID>(key, a, line, bias, lane, mine);
        if (!clear) mine = decide_exactly<T, VPL, SIGMOID>(a, line, bias, cells, lane);
        // weights of the chosen, lane j the j-th
        const bool live = mine >= 0;
        const float lm = live ? to_f32(line[mine]) : -INFINITY;
        float w;
        // the chosen scores' ratios: by exponentials of differences where the scores are exponentials (softmax, or a sigmoid so
        // far down that 1 + e^l is 1), so that they do not underflow together
        if (a.renormalise) {
            const float top = warp_max(lm);
            w = !SIGMOID || top < -30.0f ? (live ? expf(lm - top) : 0.0f) : (live ? sigmoid(lm) : 0.0f);
            w = w / warp_sum(w);
        } else w = SIGMOID ? (live ? sigmoid(lm) : 0.0f) : expf(lm - peak) / total;
        if (lane < a.top_k) {
            ids[row * a.top_k + lane] = mine;
            weights[row * a.top_k + lane] = nan ? NAN : live ? w * a.scale : 0.0f;
        }
    }
}

// the fp32 key of an expert, all of its bits
template <typename T, bool SIGMOID>
__device__ __forceinline__ float whole_key(const T *line, const float *bias, float peak, float total, int e) {
    const float x = to_f32(line[e]);
    return bias ? (SIGMOID ? key_sigmoid(x) : key_div(key_exp(x - peak), total)) + bias[e] : x;
}

// Whether one of `count` experts from `first` that was not picked, and is not equal to the last pick by what its key is made of, may
// belong before it.  Out of line: few rows ask.
template <typename T, bool SIGMOID>
__device__ __noinline__ bool may_be_lost(const T *line, const float *bias, float peak, float total, int first, int count, int last, const int *picks, int top_k) {
    const float key = whole_key<T, SIGMOID>(line, bias, peak, total, last);
    for (int e = first; e < first + count; ++e) {
        const float k = whole_key<T, SIGMOID>(line, bias, peak, total, e);
        if (!(to_f32(line[e]) > -INFINITY && k > -INFINITY && key - k <= (bias ? clearance<SIGMOID>(k) : 0.0f))) continue;
        if (to_f32(line[e]) == to_f32(line[last]) && (!bias || bias[e] == bias[last])) continue;
        bool picked = false;
        for (int r = 0; r < top_k; ++r) picked = picked || picks[r] == e;
        if (!picked) return true;
    }
    return false;
}

// Many rows: eight lanes per row, four rows per warp, so that a pick's reductions serve four rows.  A lane holds a contiguous
// eighth of the experts (a part of one group: 1, 2, 4 or 8 groups) as integers that order like the keys, the low five bits
// replaced by the place in the lane: the lane's best is one integer maximum, equal keys go to the lower place by themselves, and
// taking an expert out is a comparison with the value that won.  Keys that differ in the five bits only count as close (of
// 16-bit logits without a bias they are zeros); where a key that is left may be as large as the last pick, every one is looked at
// again.  16384 rows of 256 experts, top 8 of 4 of 8 groups:
// 30 us, 42 with a warp per row (which keeps fewer rows, other group counts and more experts).
constexpr int kOctetRows = 2048;  // from here on there are rows enough for a B200's 148 SMs

template <typename T, int VPL, bool SIGMOID>
__global__ void __launch_bounds__(32 * kRouteWarps, 6) route_octet_kernel(const RouteArgs a, const T *__restrict__ logits, const float *__restrict__ bias,
                                                                      int *__restrict__ ids, float *__restrict__ weights, bool vectors) {
    extern __shared__ double s_cells[];
    __shared__ int s_pick[kRouteWarps][4][kMaxTop];
    mps::let_next_launch_start();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane & 7, quad = lane >> 3;
    double *cells = s_cells + (size_t)warp * (a.n_experts + (a.n_experts >> 5) + 1);
    const int chunk = a.n_experts >> 3, first = sub * chunk, per_group = 8 / a.n_groups;  // lanes per group
    const bool has_bias = bias != nullptr, grouped = a.n_groups > 1, need_score = has_bias || (grouped && a.group_top == 2);
    const bool whole = sizeof(T) == 2 && !has_bias;  // the five bits lose nothing
    auto row_max = [](float v) {
#pragma unroll
        for (int d = 1; d < 8; d <<= 1) v = fmaxf(v, __shfl_xor_sync(kAll, v, d));
        return v;
    };
    auto row_sum = [](float v) {
#pragma unroll
        for (int d = 1; d < 8; d <<= 1) v += __shfl_xor_sync(kAll, v, d);
        return v;
    };
    auto key_of = [](unsigned packed) {  // the key, up to the five bits
        const unsigned o = packed & ~31u;
        return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
    };
    const long long rows_of_grid = (long long)gridDim.x * kRouteWarps * 4;
    for (long long row0 = ((long long)blockIdx.x * kRouteWarps + warp) * 4; row0 < a.n_rows; row0 += rows_of_grid) {
        const long long row = row0 + quad;
        const bool live = row < a.n_rows;
        const T *line = logits + (live ? row : 0) * a.n_experts;
        float l[VPL];
        if (vectors) {  // a lane's experts in 16-byte pieces
            constexpr int N = mps::Pack<T>::N < VPL ? mps::Pack<T>::N : VPL;
#pragma unroll
            for (int i = 0; i < VPL; i += N) {
                mps::Pack<T> p = {};
                if (i < chunk) p = *reinterpret_cast<const mps::Pack<T> *>(line + first + i);
#pragma unroll
                for (int j = 0; j < N; ++j) l[i + j] = live && i < chunk ? to_f32(p.v[j]) : -INFINITY;
            }
        } else {
#pragma unroll
            for (int i = 0; i < VPL; ++i) l[i] = live && i < chunk ? to_f32(line[first + i]) : -INFINITY;
        }
        bool nan = false;
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            nan = nan || !(SIGMOID ? l[i] <= INFINITY : l[i] < INFINITY);
            if (l[i] != l[i]) l[i] = -INFINITY;
        }
        nan = (__ballot_sync(kAll, nan) >> (quad * 8) & 0xff) != 0;
        float peak = -INFINITY, total = 0.0f, total_w = 0.0f;
        if (!SIGMOID && (need_score || !a.renormalise)) {
#pragma unroll
            for (int i = 0; i < VPL; ++i) peak = fmaxf(peak, l[i]);
            peak = row_max(peak);
            if (need_score) {
#pragma unroll
                for (int i = 0; i < VPL; ++i)
                    if (l[i] > -INFINITY) total += key_exp(l[i] - peak);
                total = row_sum(total);
            }
            if (!a.renormalise) {  // the denominator of the weights
#pragma unroll
                for (int i = 0; i < VPL; ++i)
                    if (l[i] > -INFINITY) total_w += expf(l[i] - peak);
                total_w = row_sum(total_w);
            }
        }
        // keys, and the lane's two largest group values
        unsigned key[VPL];
        float one = -INFINITY, two = -INFINITY;
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            const bool open = l[i] > -INFINITY;
            float s = 0.0f;
            if (need_score) s = SIGMOID ? key_sigmoid(l[i]) : key_div(key_exp(l[i] - peak), total);
            const float k = has_bias ? s + (i < chunk ? bias[first + i] : 0.0f) : l[i];
            const bool in = open && k > -INFINITY;
            key[i] = in ? (ordered(k) & ~31u) | (31 - i) : 0u;
            if (grouped) {
                const float v = in ? (has_bias || !need_score ? k : s) : -INFINITY;
                two = fmaxf(two, fminf(one, v));
                one = fmaxf(one, v);
            }
        }
        bool clear = true;
        if (grouped) {
            for (int d = 1; d < per_group; d <<= 1) {
                const float o1 = __shfl_xor_sync(kAll, one, d), o2 = __shfl_xor_sync(kAll, two, d);
                two = fmaxf(fmaxf(two, o2), fminf(one, o1));
                one = fmaxf(one, o1);
            }
            const bool both = a.group_top == 2 && two > -INFINITY;
            const float rank = both ? one + two : one;
            int better = 0;
            for (int d = per_group; d < 8; d += per_group) {  // every other group once
                const float o = __shfl_xor_sync(kAll, rank, d);
                if (o > rank || (o == rank && (sub ^ d) < sub)) ++better;
            }
            const bool kept = better < a.top_groups && rank > -INFINITY;
            if (need_score) {  // logits compare exactly
                const float off = rank_error<SIGMOID>(one, two, both);
                const float least = -row_max(kept ? off - rank : -INFINITY), most = row_max(!kept && rank > -INFINITY ? rank + off : -INFINITY);
                const bool beyond = one > -INFINITY && !(fabsf(rank) < INFINITY);  // see keep_groups
                const unsigned lanes_beyond = __ballot_sync(kAll, beyond);  // by all lanes: rows differ in what they compare
                clear = least > most && !(lanes_beyond >> (quad * 8) & 0xff);
            }
            if (!kept) {
#pragma unroll
                for (int i = 0; i < VPL; ++i) key[i] = 0u;
            }
        }
        // picks
        unsigned best = 0u, prev = 0u;
#pragma unroll
        for (int i = 0; i < VPL; ++i) best = max(best, key[i]);
        int prev_at = -1;
        for (int j = 0; j < a.top_k; ++j) {
            unsigned top = (best & ~31u) | (best ? 8 - sub : 0);  // the lower lane among equals
#pragma unroll
            for (int d = 1; d < 8; d <<= 1) top = max(top, __shfl_xor_sync(kAll, top, d));
            const int owner = 8 - (int)(top & 31u);  // 8: none left in this row
            const unsigned won = __shfl_sync(kAll, best, (quad << 3) | (owner & 7));
            const int at = owner < 8 ? owner * chunk + 31 - (int)(won & 31u) : -1;
            if (at >= 0 && prev_at >= 0 && !whole) {
                const float p = key_of(prev), v = key_of(top);
                bool close = (prev & ~31u) == (top & ~31u);
                if (has_bias && p - v <= clearance<SIGMOID>(v) + 8e-6f * fmaxf(fabsf(p), fabsf(v))) {  // within the five bits: by the whole keys
                    const float k = whole_key<T, SIGMOID>(line, bias, peak, total, at);
                    close = close || whole_key<T, SIGMOID>(line, bias, peak, total, prev_at) - k <= clearance<SIGMOID>(k);
                }
                if (close) clear = clear && to_f32(line[prev_at]) == to_f32(line[at]) && (!has_bias || bias[prev_at] == bias[at]);
            }
            prev = top;
            prev_at = at;
            if (sub == 0) s_pick[warp][quad][j] = at;
            if (!__any_sync(kAll, at >= 0 && clear)) {
                for (int r = j + 1; sub == 0 && r < a.top_k; ++r) s_pick[warp][quad][r] = -1;
                break;
            }
            if (sub == owner) {
                best = 0u;
#pragma unroll
                for (int i = 0; i < VPL; ++i) {
                    key[i] = key[i] == won ? 0u : key[i];
                    best = max(best, key[i]);
                }
            }
        }
        if (!whole) {
            // the best key that is left to this lane, against the last pick: as far as the five bits tell
            bool close = false;
            if (prev_at >= 0 && clear && best) {
                const float p = key_of(prev), v = key_of(best);
                close = has_bias ? p - v <= clearance<SIGMOID>(v) + 8e-6f * fmaxf(fabsf(p), fabsf(v)) : (prev & ~31u) == (best & ~31u);
            }
            if (__any_sync(kAll, close)) {
                __syncwarp();  // the picks are read below
                if (close) close = may_be_lost<T, SIGMOID>(line, bias, peak, total, first, chunk, prev_at, s_pick[warp][quad], a.top_k);
            }
            const unsigned lanes_close = __ballot_sync(kAll, close);
            clear = clear && !(lanes_close >> (quad * 8) & 0xff);
        }
        __syncwarp();
        // rows that fp32 keys do not decide, by the whole warp
        const unsigned unclear = __ballot_sync(kAll, live && !clear);
        for (int q = 0; q < 4; ++q)
            if (unclear >> (8 * q) & 0xff) {
                const int mine = decide_exactly<T, VPL / 4, SIGMOID>(a, logits + (row0 + q) * a.n_experts, bias, cells, lane);
                if (lane < a.top_k) s_pick[warp][q][lane] = mine;
                __syncwarp();
            }
        // weights of the chosen, a lane every eighth
        float lm[kMaxTop / 8], w[kMaxTop / 8], top = -INFINITY, sum = 0.0f;
        int mine[kMaxTop / 8];
#pragma unroll
        for (int i = 0; i < kMaxTop / 8; ++i) {
            const int j = sub + 8 * i;
            mine[i] = j < a.top_k ? s_pick[warp][quad][j] : -1;
            lm[i] = mine[i] >= 0 ? to_f32(line[mine[i]]) : -INFINITY;
            top = fmaxf(top, lm[i]);
        }
        if (a.renormalise) top = row_max(top);
#pragma unroll
        for (int i = 0; i < kMaxTop / 8; ++i) {
            w[i] = 0.0f;
            if (mine[i] < 0) continue;
            if (a.renormalise) w[i] = !SIGMOID || top < -30.0f ? expf(lm[i] - top) : sigmoid(lm[i]);
            else w[i] = SIGMOID ? sigmoid(lm[i]) : expf(lm[i] - peak) / total_w;
            sum += w[i];
        }
        if (a.renormalise) sum = row_sum(sum);
#pragma unroll
        for (int i = 0; i < kMaxTop / 8; ++i) {
            const int j = sub + 8 * i;
            if (live && j < a.top_k) {
                ids[row * a.top_k + j] = mine[i];
                const float v = a.renormalise ? w[i] / sum : w[i];
                weights[row * a.top_k + j] = nan ? NAN : mine[i] >= 0 ? v * a.scale : 0.0f;
            }
        }
        __syncwarp();
    }
}

// Gradient by the logits, all of the row written.  With r = the chosen scores' shares and g = the weights' gradient:
//   renormalised: dl_j = scale r_j (g_j - sum_i g_i r_i) (times 1 - s_j for a sigmoid), nothing for the others;
//   softmax:      dl_e = scale p_e (g_e - sum_i g_i p_i);      sigmoid: dl_j = scale g_j s_j (1 - s_j).
// One warp per row; the row is put together in shared memory, the chosen one after the other, so that an expert named twice gets
// both contributions in the order of the choices.
template <typename T, bool SIGMOID>
__global__ void __launch_bounds__(32 * kRouteWarps) route_backward_kernel(const RouteArgs a, const T *__restrict__ logits, const int *__restrict__ ids,
                                                                         const float *__restrict__ d_weights, T *__restrict__ d_logits) {
    extern __shared__ float s_rows[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float *cells = s_rows + (size_t)warp * a.n_experts;
    const bool dense = !SIGMOID && !a.renormalise;
    for (long long row = (long long)blockIdx.x * kRouteWarps + warp; row < a.n_rows; row += (long long)gridDim.x * kRouteWarps) {
        const T *line = logits + row * a.n_experts;
        int id = -1;
        float g = 0.0f;
        if (lane < a.top_k) {
            id = ids[row * a.top_k + lane];
            if (id >= a.n_experts) {
                atomicOr(&g_status, mps::kStatusBadIndex);
                id = -1;
            }
            if (id >= 0) g = d_weights[row * a.top_k + lane];
        }
        const float l = id >= 0 ? to_f32(line[id]) : -INFINITY;
        float own;
        if (dense) {
            float p = -INFINITY, t = 0.0f;
            for (int e = lane; e < a.n_experts; e += 32) {
                const float v = to_f32(line[e]);
                cells[e] = v;
                p = v > p || v != v ? v : p;
            }
            const float peak = warp_max(p);
            for (int e = lane; e < a.n_experts; e += 32) {
                const float v = cells[e], x = v != -INFINITY ? expf(v - peak) : 0.0f;
                cells[e] = x;
                t += x;
            }
            const float total = warp_sum(t);
            own = l != -INFINITY ? a.scale * g * (expf(l - peak) / total) : 0.0f;
            const float common = warp_sum(own);
            for (int e = lane; e < a.n_experts; e += 32) cells[e] = total > 0.0f || total != total ? -(cells[e] / total) * common : 0.0f;
        } else {
            const float s = SIGMOID ? (id >= 0 ? sigmoid(l) : 0.0f) : 0.0f, slope = SIGMOID ? sigmoid(-l) : 1.0f;
            if (a.renormalise) {
                const float top = warp_max(l);
                float share;
                if (!SIGMOID || top < -30.0f) {
                    const float e = l != -INFINITY ? expf(l - top) : 0.0f, sum = warp_sum(e);
                    share = sum != 0.0f ? e / sum : 0.0f;
                } else share = s / warp_sum(s);
                own = a.scale * share * (g - warp_sum(g * share)) * (id >= 0 ? slope : 0.0f);
            } else own = id >= 0 ? a.scale * g * s * slope : 0.0f;
            for (int e = lane; e < a.n_experts; e += 32) cells[e] = 0.0f;
        }
        __syncwarp();
        for (int j = 0; j < a.top_k; ++j) {
            if (lane == j && id >= 0) cells[id] += own;
            __syncwarp();
        }
        for (int e = lane; e < a.n_experts; e += 32) d_logits[row * a.n_experts + e] = mps::from_f32<T>(cells[e]);
        __syncwarp();
    }
}

// Rows listed by group: a stable counting sort of the pairs (row, choice) by id in one launch of one cluster.  The pairs are cut
// into one contiguous run per warp of the cluster; a warp counts its run's ids in shared memory, the counts are scanned over
// warps, blocks (distributed shared memory) and groups, and the warp walks its run again, 32 pairs at a time, and places every
// pair: lanes of equal id find one another by a ballot per bit of the id, so there is one order and no atomics in it (match.any
// for the same took 45 us for 131,072 pairs of 256 groups).  A block first sorts its own pairs in shared memory and then writes
// whole runs per group: scattered 4-byte writes straight to memory took 30 of 37 us there.  With `rest` the pairs without a
// group form one group more, the last.
constexpr int kGroupThreads = 1024, kGroupWarps = kGroupThreads / 32, kGroupMax = 1024;
constexpr int kGroupCluster = 16;
constexpr int kSortedMax = 16384;  // pairs a block sorts in shared memory

struct GroupArgs {
    long long n_pairs;
    int per_row, n_groups, sorted;  // sorted: pairs a block has room for (0: written straight to memory)
    bool rest;
    const int *ids;
    int *group_ptr, *slot_row, *slot_of;
};

__global__ void __launch_bounds__(kGroupThreads) group_kernel(const GroupArgs a) {
    extern __shared__ int s_int[];
    const int columns = a.n_groups + (a.rest ? 1 : 0), none = a.rest ? a.n_groups : -1;
    int *count = s_int;                           // [warps][columns], later the next free place of the block's sorted pairs
    int *total = count + kGroupWarps * columns;   // this block's pairs per column
    int *local = total + columns;                 // where a column starts among the block's sorted pairs (columns + 1)
    int *global = local + columns + 1;            // and among all
    int *sorted = global + columns;
    __shared__ int s_scan[kGroupWarps], s_own[kGroupWarps];
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank(), blocks = (int)cluster.num_blocks();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int steps = (int)((a.n_pairs + 31) / 32), runs = blocks * kGroupWarps, run = rank * kGroupWarps + warp;
    const int lo = (int)((long long)steps * run / runs), hi = (int)((long long)steps * (run + 1) / runs);
    int *own = count + warp * columns;
    mps::let_next_launch_start();
    for (int g = lane; g < columns; g += 32) own[g] = 0;
    __syncwarp();
    const int bits = columns > 1 ? 32 - __clz(columns - 1) : 0;  // of an id
    auto lanes_of = [&](int id) {                               // lanes with this lane's id, for an id >= 0
        unsigned same = __ballot_sync(kAll, id >= 0);
        for (int b = 0; b < bits; ++b) {
            const unsigned set = __ballot_sync(kAll, id >> b & 1);
            same &= id >> b & 1 ? set : ~set;
        }
        return same;
    };
    mps::wait_for_launch_before();
    constexpr int kBatch = 8;  // loads in flight
    int batch[kBatch];
    auto load = [&](int s) {
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const long long i = (long long)(s + j) * 32 + lane;
            const bool in = s + j < hi && i < a.n_pairs;
            batch[j] = in ? a.ids[i] : -1;
            if ((unsigned)batch[j] >= (unsigned)a.n_groups) {
                if (batch[j] >= 0) atomicOr(&g_status, mps::kStatusBadIndex);
                batch[j] = in ? none : -1;
            }
        }
    };
    for (int s = lo; s < hi; s += kBatch) {
        load(s);
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
            if (batch[j] >= 0) atomicAdd(&own[batch[j]], 1);  // counts only: their order does not show
    }
    __syncthreads();
    for (int g = tid; g < columns; g += kGroupThreads) {
        int sum = 0;
#pragma unroll
        for (int w = 0; w < kGroupWarps; ++w) {
            const int c = count[w * columns + g];
            count[w * columns + g] = sum;
            sum += c;
        }
        total[g] = sum;
    }
    cluster.sync();
    // exclusive scans over the columns: of this block's totals and of all blocks'
    int before = 0, all = 0, mine = 0;
    if (tid < a.n_groups) {
        mine = total[tid];
        for (int r = 0; r < blocks; ++r) {
            const int c = cluster.map_shared_rank(total, r)[tid];
            if (r < rank) before += c;
            all += c;
        }
    }
    int scan = all, scan_own = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(kAll, scan, d), q = __shfl_up_sync(kAll, scan_own, d);
        if (lane >= d) {
            scan += o;
            scan_own += q;
        }
    }
    if (lane == 31) {
        s_scan[warp] = scan;
        s_own[warp] = scan_own;
    }
    __syncthreads();
    if (warp == 0) {
        int v = s_scan[lane], q = s_own[lane];
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(kAll, v, d), u = __shfl_up_sync(kAll, q, d);
            if (lane >= d) {
                v += o;
                q += u;
            }
        }
        s_scan[lane] = v;
        s_own[lane] = q;
    }
    __syncthreads();
    const int start = scan - all + (warp ? s_scan[warp - 1] : 0), start_own = scan_own - mine + (warp ? s_own[warp - 1] : 0);
    const int used = s_scan[kGroupWarps - 1], used_own = s_own[kGroupWarps - 1];
    if (tid < a.n_groups) {
        local[tid] = start_own;
        global[tid] = start + before;
        if (rank == 0) {
            a.group_ptr[tid] = start;
            if (tid == a.n_groups - 1) a.group_ptr[a.n_groups] = used;
        }
    }
    if (tid == 0) {
        local[a.n_groups] = used_own;
        if (a.rest) {  // behind the groups
            int ahead = used;
            for (int r = 0; r < rank; ++r) ahead += cluster.map_shared_rank(total, r)[a.n_groups];
            global[a.n_groups] = ahead;
            local[columns] = used_own + total[a.n_groups];
            if (rank == 0) a.group_ptr[columns] = (int)a.n_pairs;
        }
    }
    cluster.sync();  // also: no block leaves while another still reads its totals
    for (int s = lo; s < hi; s += kBatch) {
        load(s);
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            if (s + j >= hi) break;
            const long long i = (long long)(s + j) * 32 + lane;
            const int id = batch[j];
            const unsigned same = lanes_of(id);
            int at = -1;
            if (id >= 0) at = own[id] + __popc(same & ((1u << lane) - 1));  // among the block's pairs of the column
            __syncwarp();
            if (id >= 0 && lane == __ffs(same) - 1) own[id] += __popc(same);
            __syncwarp();
            if (i < a.n_pairs) {
                const int slot = id >= 0 ? global[id] + at : -1;
                if (a.slot_of) a.slot_of[i] = slot;
                if (id >= 0) {
                    if (a.sorted) sorted[local[id] + at] = (int)i / a.per_row;
                    else a.slot_row[slot] = (int)i / a.per_row;
                }
                if (!a.rest && i >= used) a.slot_row[i] = -1;
            }
        }
    }
    if (a.sorted) {
        __syncthreads();
        for (int g = warp; g < columns; g += kGroupWarps)
            for (int j = local[g] + lane; j < local[g + 1]; j += 32) a.slot_row[global[g] + j - local[g]] = sorted[j];
    }
}

int launch_group(long long n_pairs, int per_row, int n_groups, bool rest, const int *ids, int *ptr, int *row, int *slot, bool follows, cudaStream_t st) {
    const int columns = n_groups + (rest ? 1 : 0);
    const int blocks = n_pairs > 16384 ? kGroupCluster : n_pairs > 2048 ? 8 : 1;
    const long long runs = blocks * kGroupWarps, most = ((n_pairs + 31) / 32 + runs - 1) / runs * 32 * kGroupWarps;  // pairs of a block
    const GroupArgs a = {n_pairs, per_row, n_groups, most <= kSortedMax ? (int)most : 0, rest, ids, ptr, row, slot};
    const size_t smem = ((size_t)(kGroupWarps + 3) * columns + 1 + a.sorted) * sizeof(int);
    if (smem > 40 * 1024)
        RT_CUDA(cudaFuncSetAttribute(group_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     (int)(((kGroupWarps + 3) * (kGroupMax + 1) + 1 + kSortedMax) * sizeof(int))));
    if (blocks > 8) RT_CUDA(cudaFuncSetAttribute(group_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = blocks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // see mps_tc.cuh
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(kGroupThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = follows ? 2 : 1;
    RT_CUDA(cudaLaunchKernelEx(&cfg, group_kernel, a));
    return MPS_OK;
}

// Blocks for `want` blocks' worth of rows: no more than the device has room for at once, each then walks over its share.
template <typename Kernel>
int resident_blocks(Kernel kernel, long long want, size_t smem, unsigned *blocks) {
    int sms, per_sm = 1;
    if (int rc = mps::sm_count(&sms)) return rc;
    if (want > sms) RT_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, 32 * kRouteWarps, smem));
    const long long room = (long long)sms * per_sm;
    *blocks = (unsigned)(want < room ? want : room);
    return MPS_OK;
}

template <typename T, bool SIGMOID>
int launch_route(const RouteArgs &a, const void *logits, const float *bias, int *ids, float *weights, cudaStream_t st) {
    const size_t smem = (size_t)kRouteWarps * (a.n_experts + (a.n_experts >> 5) + 1) * sizeof(double);
    const int per_lane = (a.n_experts + 31) / 32;
    if (a.n_rows >= kOctetRows && a.n_experts % 8 == 0 && a.n_experts <= 256 && a.n_groups <= 8 && 8 % a.n_groups == 0) {
        const long long want = ((long long)a.n_rows + 4 * kRouteWarps - 1) / (4 * kRouteWarps);
        unsigned grid;
        const bool vectors = a.n_experts / 8 * sizeof(T) % 16 == 0 && ((uintptr_t)logits & 15) == 0;
#define RT_LAUNCH(V)                                                                                                                          \
    do {                                                                                                                                      \
        if (int rc = resident_blocks(route_octet_kernel<T, V, SIGMOID>, want, smem, &grid)) return rc;                                        \
        route_octet_kernel<T, V, SIGMOID><<<grid, 32 * kRouteWarps, smem, st>>>(a, (const T *)logits, bias, ids, weights, vectors);           \
    } while (0)
        if (a.n_experts <= 64) RT_LAUNCH(8);
        else if (a.n_experts <= 128) RT_LAUNCH(16);
        else RT_LAUNCH(32);
#undef RT_LAUNCH
        RT_CUDA(cudaGetLastError());
        return MPS_OK;
    }
    const long long want = ((long long)a.n_rows + kRouteWarps - 1) / kRouteWarps;
    unsigned blocks;
#define RT_LAUNCH(V)                                                                                                       \
    do {                                                                                                                   \
        if (int rc = resident_blocks(route_kernel<T, V, SIGMOID>, want, smem, &blocks)) return rc;                         \
        route_kernel<T, V, SIGMOID><<<blocks, 32 * kRouteWarps, smem, st>>>(a, (const T *)logits, bias, ids, weights);     \
    } while (0)
    if (per_lane <= 1) RT_LAUNCH(1);
    else if (per_lane <= 2) RT_LAUNCH(2);
    else if (per_lane <= 4) RT_LAUNCH(4);
    else if (per_lane <= 8) RT_LAUNCH(8);
    else if (per_lane <= 16) RT_LAUNCH(16);
    else RT_LAUNCH(32);
#undef RT_LAUNCH
    RT_CUDA(cudaGetLastError());
    return MPS_OK;
}

int check_spec(const char *who, int n_rows, const mps_route_spec *spec, int dtype, RouteArgs *a) {
    if (!spec) return fail(MPS_ERR_ARG, "%s: spec is NULL", who);
    if (n_rows < 0) return fail(MPS_ERR_ARG, "%s: n_rows = %d", who, n_rows);
    if (dtype != MPS_F32 && dtype != MPS_F16 && dtype != MPS_BF16) return fail(MPS_ERR_ARG, "%s: unknown dtype %d", who, dtype);
    if (spec->score != MPS_SCORE_SOFTMAX && spec->score != MPS_SCORE_SIGMOID) return fail(MPS_ERR_ARG, "%s: unknown score %d", who, spec->score);
    if (spec->n_experts < 1 || spec->top_k < 1 || spec->n_groups < 1 || spec->n_experts % spec->n_groups)
        return fail(MPS_ERR_ARG, "%s: %d experts, top %d, %d groups (experts must divide into the groups)", who, spec->n_experts, spec->top_k,
                    spec->n_groups);
    if (spec->top_groups < 1 || spec->top_groups > spec->n_groups || (spec->group_top != 1 && spec->group_top != 2))
        return fail(MPS_ERR_ARG, "%s: top_groups %d of %d, group_top %d (1 or 2)", who, spec->top_groups, spec->n_groups, spec->group_top);
    if (spec->top_k > spec->n_experts / spec->n_groups * spec->top_groups)
        return fail(MPS_ERR_ARG, "%s: top %d of %d experts in the groups kept", who, spec->top_k, spec->n_experts / spec->n_groups * spec->top_groups);
    if (!std::isfinite(spec->scale)) return fail(MPS_ERR_ARG, "%s: scale is not finite", who);
    if (spec->n_experts > kMaxExperts || spec->top_k > kMaxTop || spec->n_groups > kMaxGroups)
        return fail(MPS_ERR_UNSUPPORTED, "%s: at most %d experts, top %d, %d groups", who, kMaxExperts, kMaxTop, kMaxGroups);
    if ((long long)n_rows * spec->top_k >= 1LL << 31) return fail(MPS_ERR_UNSUPPORTED, "%s: rows * top_k does not fit 31 bits", who);
    *a = RouteArgs{n_rows, spec->n_experts, spec->top_k, spec->n_groups, spec->n_experts / spec->n_groups, spec->top_groups, spec->group_top,
                   spec->n_experts == spec->n_groups ? 0u : (unsigned)(((1ull << 32) + spec->n_experts / spec->n_groups - 1) / (spec->n_experts / spec->n_groups)),
                   spec->renormalise != 0, spec->scale};
    return MPS_OK;
}

bool misaligned(const void *p, size_t size) { return ((uintptr_t)p & (size - 1)) != 0; }

}  // namespace

namespace mps {
int sm_count(int *n) {
    static PerDevice<int> known;
    int dev = 0;
    RT_CUDA(cudaGetDevice(&dev));
    if ((*n = known.get(dev))) return MPS_OK;
    RT_CUDA(cudaDeviceGetAttribute(n, cudaDevAttrMultiProcessorCount, dev));
    known.put(dev, *n);
    return MPS_OK;
}
int take_route_status(void *stream, int *status) {
    cudaStream_t st = (cudaStream_t)stream;
    RT_CUDA(cudaMemcpyFromSymbolAsync(status, g_status, sizeof(int), 0, cudaMemcpyDeviceToHost, st));
    RT_CUDA(cudaStreamSynchronize(st));
    if (*status) {  // see mps_routed_check
        clear_status<<<1, 1, 0, st>>>(*status);
        RT_CUDA(cudaGetLastError());
        RT_CUDA(cudaStreamSynchronize(st));
    }
    return MPS_OK;
}
int list_rows_and_rest(int n_rows, int n_groups, const int32_t *ids, int32_t *group_ptr, int32_t *slot_row, void *stream) {
    return launch_group(n_rows, 1, n_groups, true, ids, group_ptr, slot_row, nullptr, false, (cudaStream_t)stream);
}
}  // namespace mps

extern "C" int mps_group_rows(int32_t n_rows, int32_t per_row, int32_t n_groups, const int32_t *d_ids, int32_t *d_group_ptr, int32_t *d_slot_row,
                              int32_t *d_slot_of, void *stream) {
    if (n_rows < 0 || per_row < 1 || n_groups < 1) return fail(MPS_ERR_ARG, "mps_group_rows: %d rows, %d per row, %d groups", n_rows, per_row, n_groups);
    const long long pairs = (long long)n_rows * per_row;
    if (!d_group_ptr || (pairs > 0 && (!d_ids || !d_slot_row || !d_slot_of))) return fail(MPS_ERR_ARG, "mps_group_rows: NULL pointer");
    if (n_groups > kGroupMax) return fail(MPS_ERR_UNSUPPORTED, "mps_group_rows: at most %d groups", kGroupMax);
    if (pairs >= 1LL << 31) return fail(MPS_ERR_UNSUPPORTED, "mps_group_rows: rows * per_row does not fit 31 bits");
    if (misaligned(d_ids, 4) || misaligned(d_group_ptr, 4) || misaligned(d_slot_row, 4) || misaligned(d_slot_of, 4))
        return fail(MPS_ERR_ALIGN, "mps_group_rows: pointers must be 4-byte aligned");
    return launch_group(pairs, per_row, n_groups, false, d_ids, d_group_ptr, d_slot_row, d_slot_of, false, (cudaStream_t)stream);
}

extern "C" int mps_route(int32_t n_rows, const mps_route_spec *spec, int dtype, const void *d_logits, const float *d_bias, int32_t *d_ids,
                         float *d_weights, int32_t *d_group_ptr, int32_t *d_slot_row, int32_t *d_slot_of, void *stream) {
    RouteArgs a;
    if (int rc = check_spec("mps_route", n_rows, spec, dtype, &a)) return rc;
    const bool list = d_group_ptr || d_slot_row || d_slot_of;
    if (n_rows > 0 && (!d_logits || !d_ids || !d_weights)) return fail(MPS_ERR_ARG, "mps_route: NULL pointer");
    if (list && (!d_group_ptr || (n_rows > 0 && (!d_slot_row || !d_slot_of))))
        return fail(MPS_ERR_ARG, "mps_route: the three group arrays go together (all or none NULL)");
    if (misaligned(d_logits, dtype == MPS_F32 ? 4 : 2) || misaligned(d_bias, 4) || misaligned(d_ids, 4) || misaligned(d_weights, 4) ||
        misaligned(d_group_ptr, 4) || misaligned(d_slot_row, 4) || misaligned(d_slot_of, 4))
        return fail(MPS_ERR_ALIGN, "mps_route: a pointer is not aligned to its element size");
    cudaStream_t st = (cudaStream_t)stream;
    if (n_rows > 0) {
        const bool sig = spec->score == MPS_SCORE_SIGMOID;
        int rc;
        if (dtype == MPS_F32) rc = sig ? launch_route<float, true>(a, d_logits, d_bias, d_ids, d_weights, st) : launch_route<float, false>(a, d_logits, d_bias, d_ids, d_weights, st);
        else if (dtype == MPS_F16) rc = sig ? launch_route<__half, true>(a, d_logits, d_bias, d_ids, d_weights, st) : launch_route<__half, false>(a, d_logits, d_bias, d_ids, d_weights, st);
        else rc = sig ? launch_route<__nv_bfloat16, true>(a, d_logits, d_bias, d_ids, d_weights, st) : launch_route<__nv_bfloat16, false>(a, d_logits, d_bias, d_ids, d_weights, st);
        if (rc) return rc;
    }
    if (list) return launch_group((long long)n_rows * a.top_k, a.top_k, a.n_experts, false, d_ids, d_group_ptr, d_slot_row, d_slot_of, n_rows > 0, st);
    return MPS_OK;
}

template <typename T>
static int launch_route_backward(const RouteArgs &a, bool sigmoid_score, const void *logits, const int *ids, const float *d_weights, void *d_logits,
                                 cudaStream_t st) {
    const long long want = ((long long)a.n_rows + kRouteWarps - 1) / kRouteWarps;
    const size_t smem = (size_t)kRouteWarps * a.n_experts * sizeof(float);
    unsigned blocks;
    if (int rc = sigmoid_score ? resident_blocks(route_backward_kernel<T, true>, want, smem, &blocks) : resident_blocks(route_backward_kernel<T, false>, want, smem, &blocks))
        return rc;
    if (sigmoid_score) route_backward_kernel<T, true><<<blocks, 32 * kRouteWarps, smem, st>>>(a, (const T *)logits, ids, d_weights, (T *)d_logits);
    else route_backward_kernel<T, false><<<blocks, 32 * kRouteWarps, smem, st>>>(a, (const T *)logits, ids, d_weights, (T *)d_logits);
    RT_CUDA(cudaGetLastError());
    return MPS_OK;
}

extern "C" int mps_route_backward(int32_t n_rows, const mps_route_spec *spec, int dtype, const void *d_logits, const int32_t *d_ids,
                                  const float *d_dweights, void *d_dlogits, void *stream) {
    RouteArgs a;
    if (int rc = check_spec("mps_route_backward", n_rows, spec, dtype, &a)) return rc;
    if (n_rows == 0) return MPS_OK;
    if (!d_logits || !d_ids || !d_dweights || !d_dlogits) return fail(MPS_ERR_ARG, "mps_route_backward: NULL pointer");
    const size_t size = dtype == MPS_F32 ? 4 : 2;
    if (misaligned(d_logits, size) || misaligned(d_dlogits, size) || misaligned(d_ids, 4) || misaligned(d_dweights, 4))
        return fail(MPS_ERR_ALIGN, "mps_route_backward: a pointer is not aligned to its element size");
    const bool sig = spec->score == MPS_SCORE_SIGMOID;
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == MPS_F32) return launch_route_backward<float>(a, sig, d_logits, d_ids, d_dweights, d_dlogits, st);
    if (dtype == MPS_F16) return launch_route_backward<__half>(a, sig, d_logits, d_ids, d_dweights, d_dlogits, st);
    return launch_route_backward<__nv_bfloat16>(a, sig, d_logits, d_ids, d_dweights, d_dlogits, st);
}
