// Routing of tokens to experts, and the plan that puts the (token, expert) pairs into one bucket per expert.
//
//   moe_route_k(logits, bias, ids, weights, rows, n_exp, topk, n_group, topk_group, group_top, score, renorm, scale, dtype)
//       score 0: s = softmax(logits) over the experts, 1: s = 1 / (1 + exp(-logit)).
//       The order of the experts of a token is that of  key = logit  without a bias (the order of s, free of
//       rounding) and of  key = s + bias  with one (the bias balances the load; it does not enter the weights).
//       n_group > 1: the experts are n_group runs of neighbours; a group is worth its largest s (+ bias), or with
//       group_top = 2 the sum of its two largest, and only the experts of the topk_group best groups stay.
//       ids[t, j], j < topk: the experts of the topk largest keys, descending, equal keys by ascending index;
//       weights[t, j] = s[ids], divided by their sum when renorm is set, times scale.
//       A logit of -inf or NaN (or such a bias) takes the expert out; a choice without a candidate is id -1, weight 0.
//   moe_route_plan_k(logits, bias, ids, weights, bucket_rows, base, offsets, rows, ..., dtype)
//       moe_route_k and moe_plan_k behind each other; few tokens in one launch.
//   moe_plan_k(ids, weights, bucket_rows, base, offsets, rows, n_exp, topk)
//       counting sort of the pairs by expert, stable by pair index: offsets[n_exp + 1] bounds the buckets,
//       bucket_rows[slot] is the token of a slot, base[t, j] the slot of a pair.  A pair whose id is out of range or
//       whose weight is 0 gets no slot: its base is 0 and its weight is set to 0.  Slots behind offsets[n_exp] are
//       not written.  (The device form of MoEExperts.route; reference python/k100lc_kernels/model.py:620-720.)
//
// The grid given by the caller is ignored; the arguments fix the work.
//
// A warp takes a token and holds its experts in registers, neighbours to a lane, so that a group is a run of lanes: scores, a
// sort of the lane's keys, the groups' worths by shuffles, and topk rounds of a warp-wide maximum over the lanes' best.
// Measured (B200): one token of 128 experts 7.2 us (a launch), 48 of 256 in groups 11.9, 3001 of 60 14.3, 16384 of 256 (bf16,
// sigmoid, bias, 4 of 8 groups, 8 choices) 48 us, 219 GB/s.  Bound by instructions: 1140 of a warp for a token, issued in 58 % of
// the cycles; the bytes would take 1.6 us.  (16384 tokens of 256 equal logits, f32, 39 us: see decide_again.)
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "device_utils.cuh"
#include "fm_internal.h"

namespace fm {
namespace {

constexpr int kMaxExperts = 1024, kMaxTopk = 32, kMaxGroups = 32;

struct RouteParams {
    const void* logits;
    const float* bias;
    int* ids;
    float* weights;
    int rows, n_exp, topk, n_group, topk_group, group_top, group_size;
    int group_lanes;           // lanes to a group when that is a power of two of whole lanes, else 0
    int dtype;
    bool sigmoid, renorm, vector;
    float scale;
    // moe_route_plan_k
    int *bucket_rows, *base, *offsets, *hist;
};

__device__ __forceinline__ float logit_at(const float* p, size_t i) { return p[i]; }
__device__ __forceinline__ float logit_at(const __nv_bfloat16* p, size_t i) { return __bfloat162float(p[i]); }
__device__ __forceinline__ float logit_at(const __half* p, size_t i) { return __half2float(p[i]); }

// Keys as unsigned integers of the same order; 0 stands for "no candidate".  (x + 0 makes -0 equal to +0.)
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    return x > -INFINITY ? b ^ ((uint32_t)((int)b >> 31) | 0x80000000u) : 0u;        // false for NaN as well
}
__device__ __forceinline__ uint64_t ordered(double x) {
    const uint64_t b = (uint64_t)__double_as_longlong(x + 0.0);
    return x > -INFINITY ? b ^ ((uint64_t)((long long)b >> 63) | 0x8000000000000000ull) : 0ull;
}
__device__ __forceinline__ float key_value(uint32_t u) { return u ? __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u) : -INFINITY; }
__device__ __forceinline__ double key_value(uint64_t u) {
    return u ? __longlong_as_double((long long)(u & 0x8000000000000000ull ? u ^ 0x8000000000000000ull : ~u)) : -INFINITY;
}
__device__ __forceinline__ uint64_t warp_max(uint64_t v) {
    const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32));
    const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
    return (uint64_t)hi << 32 | lo;
}

__device__ __forceinline__ float exp2f_approx(float x) {
    float d;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(x));
    return d;
}
__device__ __forceinline__ float rcp_approx(float x) {
    float d;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(x));
    return d;
}

// Two fp32 keys of at most this magnitude are told apart for certain when they are this far from each other.
// sigmoid: exp is within 2^-22 and, its argument x log2(e) being rounded, within |x| 2^-24, of which s (1 - s) <= 1/4 reaches
// the score; 1 + exp rounds by 2^-24, the reciprocal by 2^-23: 3e-7 together, twice that for two scores.  softmax: a sum of up
// to 1024 exps (32 in turn, then five halvings) is within 37 * 2^-24 of its value besides: 2.8e-6, twice that.  Adding the
// bias rounds by 2^-24 of the key, the position in its lowest bits takes up to VPL steps of 2^-23.
template <int VPL>
__device__ __forceinline__ float resolution(const RouteParams& p, float most) {
    return (!p.bias && p.group_top == 1 ? 0.f : p.sigmoid ? 1e-6f : 6e-6f) + (VPL + 2) * 1.1920929e-7f * most;
}

// ---- the decision in fp64: lane's experts lane * VPL + i, plain loops; taken for the few tokens that fp32 cannot decide
template <int VPL>
__device__ __forceinline__ int decide64(const RouteParams& p, const float* __restrict__ xs, double* stage) {
    const int lane = threadIdx.x & 31;
    double s[VPL];
    float x[VPL];
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < VPL; i++) {
        x[i] = xs[i];
        m = fmaxf(m, x[i]);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    double z = 0.0;
#pragma unroll
    for (int i = 0; i < VPL; i++) {
        if (p.sigmoid) s[i] = 1.0 / (1.0 + exp(-(double)x[i]));
        else {
            s[i] = !(x[i] > -INFINITY) ? 0.0 : x[i] == m ? 1.0 : exp((double)x[i] - (double)m);
            z += s[i];
        }
    }
    if (!p.sigmoid) {
#pragma unroll
        for (int o = 16; o; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
    }
    uint64_t key[VPL];
#pragma unroll
    for (int i = 0; i < VPL; i++) {
        const int e = lane * VPL + i;
        if (!p.sigmoid) s[i] = s[i] / z;
        if (p.bias && e < p.n_exp) s[i] += (double)p.bias[e];
        key[i] = x[i] > -INFINITY ? ordered(p.bias ? s[i] : (double)x[i]) : 0ull;
    }
    if (p.n_group > 1) {
        const bool by_key = !p.bias && p.group_top == 1;              // (the order of the logits is that of the scores)
#pragma unroll
        for (int i = 0; i < VPL; i++)
            if (lane * VPL + i < p.n_exp) stage[lane * VPL + i] = !key[i] ? -INFINITY : by_key ? (double)x[i] : s[i];
        __syncwarp();
        uint64_t w = 0;
        if (lane < p.n_group) {
            double a = -INFINITY, b = -INFINITY;
            for (int k = 0; k < p.group_size; k++) {
                const double v = stage[lane * p.group_size + k];
                if (v > a) { b = a; a = v; }
                else if (v > b) b = v;
            }
            w = ordered(p.group_top == 2 && b > -INFINITY ? a + b : a);
        }
        __syncwarp();
        uint32_t kept = 0;
        for (int k = 0; k < p.topk_group; k++) {
            const uint64_t best = warp_max(w);
            if (best == 0) break;
            const int g = __ffs(__ballot_sync(0xffffffffu, w == best)) - 1;
            kept |= 1u << g;
            if (lane == g) w = 0;
        }
#pragma unroll
        for (int i = 0; i < VPL; i++) {
            const int e = lane * VPL + i;
            if (e < p.n_exp && !((kept >> (e / p.group_size)) & 1u)) key[i] = 0;
        }
    }
    int mine = -1;
    for (int j = 0; j < p.topk; j++) {
        uint64_t best = 0;
#pragma unroll
        for (int i = 0; i < VPL; i++) best = key[i] > best ? key[i] : best;
        const uint64_t top = warp_max(best);
        if (top == 0) break;
        const int from = __ffs(__ballot_sync(0xffffffffu, best == top)) - 1;
        int at = 0;
        if (lane == from) {
#pragma unroll
            for (int i = VPL - 1; i >= 0; i--)
                if (key[i] == top) at = i;
#pragma unroll
            for (int i = 0; i < VPL; i++)
                if (i == at) key[i] = 0;
        }
        at = __shfl_sync(0xffffffffu, at, from);
        if (lane == j) mine = from * VPL + at;
    }
    return mine;
}

// ---- the decision in fp32
// exp and 1 / x to 2^-21 at least: good enough to order by (see `resolution`), not for the weights
__device__ __forceinline__ float fast_exp(float x) { return exp2f_approx(x * 1.4426950f); }

// A key carries its position in the lane in its lowest bits, the first highest, so that a lane's keys are distinct, equal
// values keep the order of their indices, and a sort moves one word.  The bits cost the key at most 2^-18 of its value;
// `resolution` allows for it.  (16-bit logits have no bits there.)
template <int VPL>
__device__ __forceinline__ uint32_t key_of(float v, int i) {
    const uint32_t o = ordered(v);
    return o ? (o & ~(uint32_t)(VPL - 1)) | (uint32_t)(VPL - 1 - i) : 0u;
}
template <int VPL>
__device__ __forceinline__ float value_of(uint32_t key) { return key_value(key & ~(uint32_t)(VPL - 1)); }

// Whether an expert of the lane that is not chosen may have a larger key than `tie`, the first left out, from other inputs: by
// the logits where they are the keys, by what fp32 can tell (the keys as route_token forms them) where there is a bias.  Equal
// inputs on both sides of the cut are in the order of their index, but say nothing about the keys behind them.  (Experts of
// groups that were dropped count as well: at worst the token is decided in fp64.)
// id, value: the lane's choice and its key; m, z: maximum and sum of the softmax.
template <int VPL, typename T>
__device__ __forceinline__ bool hidden_by_tie(const RouteParams& p, size_t row, const float* xs, int id, float value, float m, float z) {
    const int lane = threadIdx.x & 31, tie = __shfl_sync(0xffffffffu, id, p.topk);       // (topk < 32)
    const float logit = logit_at(reinterpret_cast<const T*>(p.logits), row * p.n_exp + tie), bias = p.bias ? p.bias[tie] : 0.f;
    value = __shfl_sync(0xffffffffu, value, p.topk);
    uint32_t chosen = 0;
    for (int j = 0; j < p.topk; j++) {
        const int e = __shfl_sync(0xffffffffu, id, j);
        if (e / VPL == lane) chosen |= 1u << (e % VPL);
    }
    const float r = 1.f / z;
    bool hidden = false;
#pragma unroll 1
    for (int i = 0; i < VPL; i++) {
        const float x = xs[i];
        if (!(x > -INFINITY) || (chosen >> i & 1u)) continue;
        if (!p.bias) {
            hidden |= x > logit;
            continue;
        }
        const float b = p.bias[lane * VPL + i], s = p.sigmoid ? rcp_approx(1.f + fast_exp(-x)) : x == m ? r : fast_exp(x - m) * r, key = s + b;
        hidden |= !(x == logit && b == bias) && !(value - key > resolution<VPL>(p, fmaxf(fabsf(value), key > -INFINITY ? fabsf(key) : 0.f)));
    }
    return __any_sync(0xffffffffu, hidden);
}

// What the few tokens come to that fp32 may not decide: `near`, or else equal inputs on both sides of the cut and more keys close
// behind them.
template <int VPL, typename T>
__device__ __noinline__ int decide_again(const RouteParams& p, size_t row, const float* xs, int id, float value, float m, float z, bool near, double* stage) {
    if (!near && !hidden_by_tie<VPL, T>(p, row, xs, id, value, m, z)) return id;
    return decide64<VPL>(p, xs, stage);
}

// Sorts the lane's keys, descending: Batcher's odd-even merge sort (1968).
template <int VPL>
__device__ __forceinline__ void sort_lane(uint32_t (&k)[VPL]) {
#pragma unroll
    for (int p = 1; p < VPL; p <<= 1)
#pragma unroll
        for (int q = p; q >= 1; q >>= 1)
#pragma unroll
            for (int j = q % p; j + q < VPL; j += 2 * q)
#pragma unroll
                for (int i = 0; i < q; i++)
                    if (i + j + q < VPL && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
                        const uint32_t hi = max(k[i + j], k[i + j + q]), lo = min(k[i + j], k[i + j + q]);
                        k[i + j] = hi;
                        k[i + j + q] = lo;
                    }
}

// The largest keys of the warp in order, from the lanes' sorted lists: lane j gets the j-th position (-1: none) and key.
template <int VPL>
__device__ __forceinline__ int pick(int rounds, uint32_t (&key)[VPL], uint32_t& kept) {
    const int lane = threadIdx.x & 31;
    int whose = -1;
    kept = 0;
    for (int j = 0; j < rounds; j++) {
        const uint32_t best = key[0] & ~(uint32_t)(VPL - 1);
        const uint32_t top = __reduce_max_sync(0xffffffffu, best);
        if (top == 0) break;
        const int from = __ffs(__ballot_sync(0xffffffffu, best == top)) - 1;
        const uint32_t k = __shfl_sync(0xffffffffu, key[0], from);
        const bool hit = lane == from;                                // its next one moves up
#pragma unroll
        for (int i = 0; i + 1 < VPL; i++) key[i] = hit ? key[i + 1] : key[i];
        key[VPL - 1] = hit ? 0u : key[VPL - 1];
        if (lane == j) {
            whose = from;
            kept = k;
        }
    }
    return whose < 0 ? -1 : whose * VPL + (VPL - 1 - (int)(kept & (uint32_t)(VPL - 1)));
}

// Which groups stay, as a mask of the lanes that speak for them (the first of a group).  a, b: the two best of the lane's group (group_lanes > 0) or of group `lane`.  gap: the distance
// between the worst group kept and the best one dropped; most: the largest magnitude of the numbers that make the groups' worths.
__device__ __forceinline__ uint32_t best_groups(const RouteParams& p, float a, float b, float& gap, float& most) {
    const int lane = threadIdx.x & 31, lanes = p.group_lanes;
    for (int o = 1; o < lanes; o <<= 1) {
        const float oa = __shfl_xor_sync(0xffffffffu, a, o), ob = __shfl_xor_sync(0xffffffffu, b, o);
        b = fmaxf(fminf(a, oa), fmaxf(b, ob));
        a = fmaxf(a, oa);
    }
    const int group = lanes > 0 ? lane / lanes : lane;
    const bool speaks = group < p.n_group && (lanes <= 1 || lane % lanes == 0);          // one lane of a group speaks for it
    uint32_t w = speaks ? ordered(p.group_top == 2 && b > -INFINITY ? a + b : a) : 0u;
    uint32_t kept = 0, last = 0, next = 0;
    if (p.n_group <= 4 * p.topk_group) {                              // a group's rank is the number of better ones
        int rank = 0;
        for (int g = 0; g < p.n_group; g++) {
            const uint32_t t = __shfl_sync(0xffffffffu, w, lanes > 0 ? g * lanes : g);
            rank += t > w || (t == w && g < group);
        }
        kept = __ballot_sync(0xffffffffu, speaks && rank < p.topk_group && w != 0);
        last = __reduce_max_sync(0xffffffffu, speaks && rank == p.topk_group - 1 ? w : 0u);
        next = __reduce_max_sync(0xffffffffu, speaks && rank == p.topk_group ? w : 0u);
    } else {
        uint32_t left = w;
        for (int k = 0; k < p.topk_group; k++) {
            last = __reduce_max_sync(0xffffffffu, left);
            if (last == 0) break;                                     // the other groups are empty
            const uint32_t who = __ballot_sync(0xffffffffu, left == last);
            kept |= who & (0u - who);                                 // the first
            if ((who & (0u - who)) >> lane & 1u) left = 0;
        }
        next = __reduce_max_sync(0xffffffffu, left);
    }
    const float l = last ? key_value(last) : INFINITY, n = key_value(next);
    gap = l - n;
    // (of a group's two numbers one may be large and negative: their magnitudes bound the error of the sum)
    const float size = speaks ? fmaxf(fabsf(a), b > -INFINITY ? fabsf(b) : 0.f) : 0.f;
    most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(size < INFINITY ? size : 0.f)));
    return kept;
}

template <int VPL, typename T>
__device__ __forceinline__ void load_logits(const RouteParams& p, size_t row, float (&x)[VPL]) {
    const int lane = threadIdx.x & 31;
    const T* in = reinterpret_cast<const T*>(p.logits) + row * p.n_exp + lane * VPL;
    constexpr int PER = 16 / (int)sizeof(T);
    if (VPL % PER == 0 && p.n_exp == 32 * VPL && p.vector) {          // whole 16-byte words
#pragma unroll
        for (int i = 0; i < VPL; i += PER) {
            const uint4 w = *reinterpret_cast<const uint4*>(in + i);
            const T* t = reinterpret_cast<const T*>(&w);
#pragma unroll
            for (int k = 0; k < PER; k++) x[(i + k) % VPL] = logit_at(t, k);
        }
    } else {
#pragma unroll
        for (int i = 0; i < VPL; i++) x[i] = lane * VPL + i < p.n_exp ? logit_at(in, i) : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < VPL; i++)
        if (!(x[i] > -INFINITY)) x[i] = -INFINITY;                    // NaN: never chosen
}

// Quotients of scores w some of which are below 2^-92 and may leave fp32's range (c: the lane's logit, -inf: no choice): all are
// formed over exp(from), from being the largest chosen logit (of sigmoids: at most 0).  The sigmoid over it is
// exp(c - from) / (1 + exp(c)) for c <= 0, and the second factor is 1 to fp32 below -64.
__device__ __noinline__ float small_quotient(bool sigmoid, float c, float m, float w) {
    const float most = key_value(__reduce_max_sync(0xffffffffu, ordered(c))), from = fminf(most, 0.f);
    if (!sigmoid) w = m == INFINITY ? w : c == most ? 1.f : expf(c - most);
    else if (from < 0.f) w = __fdiv_rn(expf(c - from), 1.f + expf(c));
    else if (c < -64.f) w = expf(c);
    if (!(c > -INFINITY)) w = 0.f;
    const float sum = warp_sum(w);
    return sum > 0.f ? __fdiv_rn(w, sum) : 0.f;
}

// One token: lane j < topk gets its j-th expert and weight.  Keys are formed and ordered in fp32; a token where two that
// matter lie within the error of fp32 is decided again in fp64, so that the choice is that of the keys in fp64 at fp32's cost.
// bias: the lane's.
template <int VPL, typename T>
__device__ __forceinline__ void route_token(const RouteParams& p, size_t row, const float (&bias)[VPL], double* stage, int& id, float& weight) {
    const int lane = threadIdx.x & 31;
    float x[VPL], s[VPL];                                             // logits; scores to order by
    load_logits<VPL, T>(p, row, x);
    float m = 0.f, z = 1.f;
    const bool by_score = !p.bias && p.n_group > 1 && p.group_top == 2, need = p.bias || by_score;
    if (!p.sigmoid) {
        m = -INFINITY;
#pragma unroll
        for (int i = 0; i < VPL; i++) m = fmaxf(m, x[i]);
        m = key_value(__reduce_max_sync(0xffffffffu, ordered(m)));
        if (need || !p.renorm) {
            z = 0.f;
#pragma unroll
            for (int i = 0; i < VPL; i++) {                           // (an infinite maximum is its own score)
                s[i] = !(x[i] > -INFINITY) ? 0.f : x[i] == m ? 1.f : p.renorm ? fast_exp(x[i] - m) : expf(x[i] - m);
                z += s[i];
            }
            z = warp_sum(z);
            const float r = 1.f / z;
#pragma unroll
            for (int i = 0; i < VPL; i++) s[i] *= r;
        }
    } else if (need) {
#pragma unroll
        for (int i = 0; i < VPL; i++) s[i] = rcp_approx(1.f + fast_exp(-x[i]));
    }
    uint32_t key[VPL], kept;
#pragma unroll
    for (int i = 0; i < VPL; i++) key[i] = key_of<VPL>(!p.bias ? x[i] : x[i] > -INFINITY ? s[i] + bias[i] : -INFINITY, i);
    const bool check = p.bias || sizeof(T) == 4;                      // (16-bit logits themselves are exact keys)
    bool near = false, tie = false;
    float a = -INFINITY, b = -INFINITY;                               // the two best of the lane
    if (by_score) {
#pragma unroll
        for (int i = 0; i < VPL; i++) {
            const float t = key[i] ? s[i] : -INFINITY;
            b = fmaxf(b, fminf(a, t));
            a = fmaxf(a, t);
        }
    }
    if (p.n_group > 1 && p.group_lanes == 0) {                        // groups that do not end with lanes
        float* list = reinterpret_cast<float*>(stage);
#pragma unroll
        for (int i = 0; i < VPL; i++)
            if (lane * VPL + i < p.n_exp) list[lane * VPL + i] = by_score && key[i] ? s[i] : value_of<VPL>(key[i]);
        __syncwarp();
        a = b = -INFINITY;
        if (lane < p.n_group)
            for (int k = 0; k < p.group_size; k++) {
                const float t = list[lane * p.group_size + k];
                b = fmaxf(b, fminf(a, t));
                a = fmaxf(a, t);
            }
        __syncwarp();
        float gap, most;
        const uint32_t groups = best_groups(p, a, b, gap, most);
        near = (check || by_score) && !(gap > 2.f * resolution<VPL>(p, most));       // (a group's worth is a sum of two)
#pragma unroll
        for (int i = 0; i < VPL; i++) {
            const int e = lane * VPL + i;
            if (e < p.n_exp && !((groups >> (e / p.group_size)) & 1u)) key[i] = 0;       // (lane g speaks for group g)
        }
    }
    sort_lane<VPL>(key);
    if (p.n_group > 1 && p.group_lanes > 0) {
        if (!by_score) {
            a = value_of<VPL>(key[0]);
            if (VPL > 1) b = value_of<VPL>(key[VPL > 1 ? 1 : 0]);
        }
        float gap, most;
        const uint32_t groups = best_groups(p, a, b, gap, most);
        near = (check || by_score) && !(gap > 2.f * resolution<VPL>(p, most));
        if (!((groups >> (lane & ~(p.group_lanes - 1))) & 1u)) {
#pragma unroll
            for (int i = 0; i < VPL; i++) key[i] = 0;
        }
    }
    id = pick<VPL>(min(p.topk + (check ? 1 : 0), 32), key, kept);
    if (check) {
        const float v = value_of<VPL>(kept), prev = __shfl_up_sync(0xffffffffu, v, 1);
        const int before = __shfl_up_sync(0xffffffffu, id, 1);
        const bool close = lane > 0 && lane <= p.topk && id >= 0 && !(prev - v > resolution<VPL>(p, fmaxf(fabsf(v), fabsf(prev))));
        near = near || p.topk == 32;                                  // (the key after 32 choices has no lane to compare it in)
        if (__any_sync(0xffffffffu, close)) {                         // equal inputs are equal keys: the order of the index is right
            const T* in = reinterpret_cast<const T*>(p.logits) + row * p.n_exp;
            const bool equal = close && logit_at(in, id) == logit_at(in, before) && (!p.bias || p.bias[id] == p.bias[before]);
            near = near || __any_sync(0xffffffffu, close && !equal);
            if (__any_sync(0xffffffffu, equal && lane == p.topk)) {   // is there more behind (`pick` took its own off the lists)
                const float at = __shfl_sync(0xffffffffu, v, p.topk & 31), rest = value_of<VPL>(__reduce_max_sync(0xffffffffu, key[0]));
                tie = !(at - rest > resolution<VPL>(p, fmaxf(fabsf(at), rest > -INFINITY ? fabsf(rest) : 0.f)));
            }
        }
    }
    if (near || tie) {
        float copy[VPL];                                              // (an array whose address is taken lives in memory)
#pragma unroll
        for (int i = 0; i < VPL; i++) copy[i] = x[i];
        id = decide_again<VPL, T>(p, row, copy, id, value_of<VPL>(kept), m, z, near, stage);
    }
    if (lane >= p.topk) id = -1;
    // the weight of the lane's choice, from its logit
    float w = 0.f, c = -INFINITY;
    if (id >= 0) {
        c = logit_at(reinterpret_cast<const T*>(p.logits), row * p.n_exp + id);
        if (p.sigmoid) w = __frcp_rn(1.f + expf(-c));
        else w = c == m ? 1.f : expf(c - m);
        if (!p.sigmoid && !p.renorm) w = __fdiv_rn(w, z);
    }
    if (p.renorm) {
        // (a score below 2^-92 makes the sum -inf: it may be too small for fp32 where its quotient is not)
        const float sum = warp_sum(id >= 0 && w < 0x1p-92f ? -INFINITY : w);
        w = sum > 0.f ? __fdiv_rn(w, sum) : small_quotient(p.sigmoid, c, m, w);
    } else if (p.sigmoid && c < -64.f) {
        w = id >= 0 ? expf(c) : 0.f;                                  // (1 + exp(-c) ends with fp32's range)
    }
    weight = w * p.scale;
}

// ------------------------------------------------------------------------------------------------------ the plan
// The slot of a pair is
//   (pairs of smaller experts) + (pairs of its expert in earlier blocks, warps, batches and lanes),
// so the order is that of the pair indices whatever the scheduling: no atomic decides a position.
constexpr int kThreads = 512;                       // of the counting kernel

__device__ __forceinline__ int pair_expert(int id, float w, int n_exp) { return id >= 0 && id < n_exp && w != 0.f ? id : -1; }

// Exclusive scan of total[0 .. n) into first[0 .. n); returns the sum.  All threads call it; total and first may be one.
__device__ __forceinline__ int block_scan(const int* total, int* first, int n, int* part) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    int carry = 0;
    for (int e0 = 0; e0 < n; e0 += blockDim.x) {
        const int e = e0 + (int)threadIdx.x, v = e < n ? total[e] : 0;
        int inc = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += t;
        }
        __syncthreads();
        if (lane == 31) part[warp] = inc;
        __syncthreads();
        int lower = carry;
        for (int k = 0; k < warps; k++) {
            if (k < warp) lower += part[k];
            carry += part[k];
        }
        if (e < n) first[e] = lower + inc - v;
    }
    __syncthreads();
    return carry;
}

// Places the pairs [lo, hi) of this block.  first[e]: the slot of its first pair of expert e; cnt: [warps][n_exp].
__device__ __forceinline__ void place_pairs(const int* ids, float* w, int* bucket_rows, int* base, int lo, int hi, int n_exp, int topk, const int* first,
                                            int* cnt) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const int per = ((hi - lo + warps - 1) / warps + 31) & ~31, i0 = lo + warp * per, i1 = min(i0 + per, hi);
    int* mine = cnt + warp * n_exp;
    for (int e = lane; e < n_exp; e += 32) mine[e] = 0;
    __syncwarp();
    for (int i = i0 + lane; i < i1; i += 32) {
        const int e = pair_expert(__ldcg(ids + i), __ldcg(w + i), n_exp);
        if (e >= 0) atomicAdd(&mine[e], 1);                           // (integers: the order does not matter)
    }
    __syncthreads();
    for (int e = threadIdx.x; e < n_exp; e += blockDim.x) {
        int at = first[e];
        for (int k = 0; k < warps; k++) {
            const int h = cnt[k * n_exp + e];
            cnt[k * n_exp + e] = at;
            at += h;
        }
    }
    __syncthreads();
    for (int j0 = i0; j0 < i1; j0 += 32) {
        const int i = j0 + lane;
        const int e = i < i1 ? pair_expert(__ldcg(ids + i), __ldcg(w + i), n_exp) : -1;
        const uint32_t peers = __match_any_sync(0xffffffffu, e);
        const int rank = __popc(peers & ((1u << lane) - 1u));
        const int slot = e >= 0 ? mine[e] + rank : 0;
        __syncwarp();
        if (e >= 0 && rank == 0) mine[e] += __popc(peers);
        __syncwarp();
        if (i < i1) {
            base[i] = slot;
            if (e >= 0) bucket_rows[slot] = i / topk;
            else w[i] = 0.f;
        }
    }
}

__device__ unsigned g_blocks_done;                   // blocks of a fused launch that have finished; back at 0 when it ends

// Block b routes the tokens [b * tokens, (b + 1) * tokens), a warp a token at a time.  With a plan: few pairs are placed by
// the block that finishes last (fuse), otherwise every block counts its pairs of each expert for plan_place_kernel.
template <int VPL, typename T>
__global__ void __launch_bounds__(VPL <= 8 ? 1024 : 512, 1)
route_kernel(const RouteParams p, int tokens, bool fuse) {
    extern __shared__ double dyn[];                                   // [warps][n_exp] where there are groups; then ints
    __shared__ int next, part[32];
    __shared__ bool last;
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    double* stage = dyn + (p.n_group > 1 ? (size_t)warp * p.n_exp : 0);
    int* count = reinterpret_cast<int*>(dyn + (p.n_group > 1 ? (size_t)warps * p.n_exp : 0));
    if (p.hist)
        for (int e = threadIdx.x; e < p.n_exp; e += blockDim.x) count[e] = 0;
    if (threadIdx.x == 0) next = warps;
    float bias[VPL];
#pragma unroll
    for (int i = 0; i < VPL; i++) bias[i] = p.bias && lane * VPL + i < p.n_exp ? p.bias[lane * VPL + i] : 0.f;
    __syncthreads();
    const int row0 = blockIdx.x * tokens, rows = min(tokens, p.rows - row0);
    for (int t = warp; t < rows;) {                                   // (whichever warp is free takes the next token)
        const size_t row = (size_t)row0 + t;
        int id;
        float w;
        route_token<VPL, T>(p, row, bias, stage, id, w);
        if (lane < p.topk) {
            p.ids[row * p.topk + lane] = id;
            p.weights[row * p.topk + lane] = w;
            if (p.hist && pair_expert(id, w, p.n_exp) >= 0) atomicAdd(&count[id], 1);
        }
        if (lane == 0) t = atomicAdd(&next, 1);
        t = __shfl_sync(0xffffffffu, t, 0);
    }
    if (p.hist) {
        __syncthreads();
        for (int e = threadIdx.x; e < p.n_exp; e += blockDim.x) p.hist[(size_t)blockIdx.x * p.n_exp + e] = count[e];
    }
    if (fuse) {
        if (gridDim.x > 1) {
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) last = atomicInc(&g_blocks_done, gridDim.x - 1) == gridDim.x - 1;
            __syncthreads();
            if (!last) return;
            __threadfence();
        } else {
            __syncthreads();
        }
        const int pairs = p.rows * p.topk;
        int* total = count;                                           // [n_exp], then the warps' counts
        int* cnt = count + p.n_exp;
        for (int e = threadIdx.x; e < p.n_exp; e += blockDim.x) total[e] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < pairs; i += blockDim.x) {
            const int e = pair_expert(__ldcg(p.ids + i), __ldcg(p.weights + i), p.n_exp);
            if (e >= 0) atomicAdd(&total[e], 1);
        }
        __syncthreads();
        const int sum = block_scan(total, total, p.n_exp, part);
        for (int e = threadIdx.x; e < p.n_exp; e += blockDim.x) p.offsets[e] = total[e];
        if (threadIdx.x == 0) p.offsets[p.n_exp] = sum;
        place_pairs(p.ids, p.weights, p.bucket_rows, p.base, 0, pairs, p.n_exp, p.topk, total, cnt);
    }
    pdl_launch_dependents();
}

// hist[block][n_exp] of pairs that are given
__global__ void __launch_bounds__(kThreads)
plan_count_kernel(const int* ids, const float* w, int* hist, int pairs, int n_exp, int per_block) {
    extern __shared__ int count[];
    pdl_wait();
    for (int e = threadIdx.x; e < n_exp; e += kThreads) count[e] = 0;
    __syncthreads();
    const int lo = blockIdx.x * per_block, hi = min(lo + per_block, pairs);
    for (int i = lo + threadIdx.x; i < hi; i += kThreads) {
        const int e = pair_expert(ids[i], w[i], n_exp);
        if (e >= 0) atomicAdd(&count[e], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < n_exp; e += kThreads) hist[(size_t)blockIdx.x * n_exp + e] = count[e];
    pdl_launch_dependents();
}

// Launched while the kernel in front ends (what that writes is read through no path that may be read ahead of pdl_wait).
// Every block adds up the counts of all blocks (blockDim / n_exp threads to an expert) and places its own pairs.
__global__ void __launch_bounds__(1024)
plan_place_kernel(const int* ids, float* w, int* __restrict__ bucket_rows, int* __restrict__ base, int* __restrict__ offsets, const int* hist, int pairs, int n_exp, int topk, int per_block) {
    extern __shared__ int sm[];
    int* total = sm;                                                  // [n_exp]
    int* first = sm + n_exp;                                          // [n_exp] first the pairs of earlier blocks
    int* cnt = sm + 2 * n_exp;                                        // [warps][n_exp]
    __shared__ int part[32];
    pdl_wait();
    for (int e = threadIdx.x; e < 2 * n_exp; e += blockDim.x) sm[e] = 0;
    __syncthreads();
    const int split = max((int)blockDim.x / n_exp, 1), blocks = gridDim.x;
    for (int i = threadIdx.x; i < n_exp * split; i += blockDim.x) {
        const int e = i % n_exp, s = i / n_exp;
        int all = 0, before = 0;
#pragma unroll 16
        for (int b = s; b < blocks; b += split) {
            const int h = __ldcg(hist + (size_t)b * n_exp + e);
            all += h;
            if (b < (int)blockIdx.x) before += h;
        }
        if (all) {
            atomicAdd(&total[e], all);
            if (before) atomicAdd(&first[e], before);
        }
    }
    __syncthreads();
    const int sum = block_scan(total, total, n_exp, part);
    for (int e = threadIdx.x; e < n_exp; e += blockDim.x) {
        if (blockIdx.x == 0) offsets[e] = total[e];
        first[e] += total[e];
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) offsets[n_exp] = sum;
    __syncthreads();
    const int lo = blockIdx.x * per_block;
    place_pairs(ids, w, bucket_rows, base, lo, min(lo + per_block, pairs), n_exp, topk, first, cnt);
    pdl_launch_dependents();
}

// ------------------------------------------------------------------------------------------------------- host side
// Pairs that the last block of the routing places itself, instead of a second launch: 256 experts, 8 choices, in us for 384
// pairs 8.9 against 12.5, for 1024 10.6 against 11.8, for 2048 14.1 against 11.8.
constexpr int kFusePairs = 1024;
constexpr int kFuseExperts = 256;

template <typename T>
cudaError_t run_route(const LaunchCtx& c, const RouteParams& p, int blocks, int tokens, bool fuse) {
    const int vpl = (p.n_exp + 31) / 32, most = vpl <= 8 ? 32 : 16;
    int warps = tokens < most ? tokens : most;
    if (fuse && warps < 8) warps = 8;                                 // (they place the pairs)
    const size_t smem = (p.n_group > 1 ? (size_t)warps * p.n_exp * 8 : 0) + (p.hist ? (size_t)p.n_exp * 4 : 0) + (fuse ? (size_t)p.n_exp * 4 * (1 + warps) : 0);
    auto kern = vpl <= 1   ? route_kernel<1, T>
                : vpl <= 2 ? route_kernel<2, T>
                : vpl <= 4 ? route_kernel<4, T>
                : vpl <= 8 ? route_kernel<8, T>
                : vpl <= 16 ? route_kernel<16, T>
                            : route_kernel<32, T>;
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
    }
    return launch_kernel(kern, dim3((unsigned)blocks), dim3(warps * 32), smem, c.stream, pdl_enabled(), p, tokens, fuse);
}
cudaError_t run_route_of(const LaunchCtx& c, const RouteParams& p, int blocks, int tokens, bool fuse) {
    return p.dtype == 0 ? run_route<float>(c, p, blocks, tokens, fuse) : p.dtype == 1 ? run_route<__nv_bfloat16>(c, p, blocks, tokens, fuse) : run_route<__half>(c, p, blocks, tokens, fuse);
}

int run_place(const char* kn, const LaunchCtx& c, const int* ids, float* w, int* bucket_rows, int* base, int* offsets, const int* hist, int pairs, int n_exp,
              int topk, int blocks, int per_block) {
    const size_t smem = (size_t)n_exp * 4 * (2 + 32);
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(plan_place_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return cuda_fail(kn, e);
    }
    const cudaError_t e = launch_kernel(plan_place_kernel, dim3(blocks), dim3(1024), smem, c.stream, true, ids, w, bucket_rows, base, offsets, hist,
                                        pairs, n_exp, topk, per_block);
    return e == cudaSuccess ? after_launch(kn) : cuda_fail(kn, e);
}

// arguments of the choice; `a` begins with rows
int read_route(const char* kn, RouteParams& p, const uint64_t* a) {
    p.rows = arg_i32(a[0]);
    p.n_exp = arg_i32(a[1]);
    p.topk = arg_i32(a[2]);
    p.n_group = arg_i32(a[3]);
    p.topk_group = arg_i32(a[4]);
    p.group_top = arg_i32(a[5]);
    const int score = arg_i32(a[6]), renorm = arg_i32(a[7]);
    p.scale = arg_f32(a[8]);
    p.dtype = arg_i32(a[9]);
    FM_REQUIRE(p.rows >= 0 && p.n_exp >= 1 && p.n_exp <= kMaxExperts, kn, "rows=%d n_exp=%d: 1..%d experts", p.rows, p.n_exp, kMaxExperts);
    FM_REQUIRE(p.n_group >= 1 && p.n_group <= kMaxGroups && p.n_exp % p.n_group == 0, kn, "n_group=%d must divide n_exp=%d and be at most %d",
               p.n_group, p.n_exp, kMaxGroups);
    FM_REQUIRE(p.topk_group >= 1 && p.topk_group <= p.n_group, kn, "topk_group=%d of %d groups", p.topk_group, p.n_group);
    FM_REQUIRE(p.topk >= 1 && p.topk <= kMaxTopk && p.topk <= p.n_exp / p.n_group * p.topk_group, kn,
               "topk=%d: at most %d, and at most the experts of the kept groups", p.topk, kMaxTopk);
    FM_REQUIRE(p.group_top == 1 || p.group_top == 2, kn, "group_top=%d: 1 or 2", p.group_top);
    FM_REQUIRE((score == 0 || score == 1) && (renorm == 0 || renorm == 1), kn, "score=%d renorm=%d: 0 or 1", score, renorm);
    FM_REQUIRE(p.dtype >= 0 && p.dtype <= 2, kn, "dtype=%d: 0 f32, 1 bf16, 2 f16", p.dtype);
    p.sigmoid = score == 1;
    p.renorm = renorm == 1;
    p.group_size = p.n_exp / p.n_group;
    int vpl = 1;
    while (vpl * 32 < p.n_exp) vpl *= 2;
    const int lanes = p.group_size / vpl;
    p.group_lanes = p.group_size % vpl == 0 && (lanes & (lanes - 1)) == 0 ? lanes : 0;
    const size_t es = p.dtype == 0 ? 4 : 2, pairs = (size_t)p.rows * p.topk;
    FM_REQUIRE(pairs <= (1u << 30), kn, "rows * topk = %zu: at most 2^30 pairs", pairs);
    if (p.rows == 0) return FM_OK;
    FM_REQUIRE(aligned(p.logits, es) && aligned(p.bias, 4) && aligned(p.ids, 4) && aligned(p.weights, 4), kn, "misaligned pointer");
    FM_RANGE(p.logits, (size_t)p.rows * p.n_exp * es, kn, "logits");
    if (p.bias) FM_RANGE(p.bias, (size_t)p.n_exp * 4, kn, "bias");
    FM_RANGE(p.ids, pairs * 4, kn, "ids");
    FM_RANGE(p.weights, pairs * 4, kn, "weights");
    p.vector = aligned(p.logits, 16) && (size_t)p.n_exp * es % 16 == 0;
    return FM_OK;
}

// blocks of a routing launch: one to an SM, a token to a block at least
void route_shape(const LaunchCtx& c, int rows, int& blocks, int& tokens) {
    tokens = (rows + c.sm_count - 1) / c.sm_count;
    blocks = (rows + tokens - 1) / tokens;
}

int launch_route(const LaunchCtx& c, const uint64_t* a) {
    const char* kn = "moe_route_k";
    RouteParams p = {};
    p.logits = arg_ptr<const void>(a[0]);
    p.bias = arg_ptr<const float>(a[1]);
    p.ids = arg_ptr<int>(a[2]);
    p.weights = arg_ptr<float>(a[3]);
    const int rc = read_route(kn, p, a + 4);
    if (rc != FM_OK || p.rows == 0) return rc;
    int blocks, tokens;
    route_shape(c, p.rows, blocks, tokens);
    const cudaError_t e = run_route_of(c, p, blocks, tokens, false);
    return e == cudaSuccess ? after_launch(kn) : cuda_fail(kn, e);
}

// ranges of a plan's arrays
int check_plan(const char* kn, const int* bucket_rows, const int* base, const int* offsets, size_t pairs, int n_exp) {
    FM_REQUIRE(aligned(bucket_rows, 4) && aligned(base, 4) && aligned(offsets, 4), kn, "misaligned pointer");
    FM_RANGE(bucket_rows, pairs * 4, kn, "bucket_rows");
    FM_RANGE(base, pairs * 4, kn, "base");
    FM_RANGE(offsets, (size_t)(n_exp + 1) * 4, kn, "offsets");
    return FM_OK;
}

int no_rows(const char* kn, const LaunchCtx& c, int* offsets, int n_exp) {
    const cudaError_t e = cudaMemsetAsync(offsets, 0, (size_t)(n_exp + 1) * 4, c.stream);
    return e == cudaSuccess ? FM_OK : cuda_fail(kn, e);
}

int launch_route_plan(const LaunchCtx& c, const uint64_t* a) {
    const char* kn = "moe_route_plan_k";
    RouteParams p = {};
    p.logits = arg_ptr<const void>(a[0]);
    p.bias = arg_ptr<const float>(a[1]);
    p.ids = arg_ptr<int>(a[2]);
    p.weights = arg_ptr<float>(a[3]);
    p.bucket_rows = arg_ptr<int>(a[4]);
    p.base = arg_ptr<int>(a[5]);
    p.offsets = arg_ptr<int>(a[6]);
    int rc = read_route(kn, p, a + 7);
    if (rc != FM_OK) return rc;
    const size_t pairs = (size_t)p.rows * p.topk;
    if ((rc = check_plan(kn, p.bucket_rows, p.base, p.offsets, pairs, p.n_exp)) != FM_OK) return rc;
    if (p.rows == 0) return no_rows(kn, c, p.offsets, p.n_exp);
    int blocks, tokens;
    route_shape(c, p.rows, blocks, tokens);
    const bool fuse = pairs <= kFusePairs && p.n_exp <= kFuseExperts;
    if (!fuse) {
        p.hist = static_cast<int*>(engine_scratch((size_t)blocks * p.n_exp * 4));
        FM_REQUIRE(p.hist, kn, "the engine workspace cannot grow to %zu bytes here (inside a capture: raise FM_SCRATCH_MB)", (size_t)blocks * p.n_exp * 4);
    }
    const cudaError_t e = run_route_of(c, p, blocks, tokens, fuse);
    if (e != cudaSuccess) return cuda_fail(kn, e);
    rc = after_launch(kn);
    if (rc != FM_OK || fuse) return rc;
    return run_place(kn, c, p.ids, p.weights, p.bucket_rows, p.base, p.offsets, p.hist, (int)pairs, p.n_exp, p.topk, blocks, tokens * p.topk);
}

int launch_plan(const LaunchCtx& c, const uint64_t* a) {
    const char* kn = "moe_plan_k";
    const int* ids = arg_ptr<const int>(a[0]);
    float* w = arg_ptr<float>(a[1]);
    int* bucket_rows = arg_ptr<int>(a[2]);
    int* base = arg_ptr<int>(a[3]);
    int* offsets = arg_ptr<int>(a[4]);
    const int rows = arg_i32(a[5]), n_exp = arg_i32(a[6]), topk = arg_i32(a[7]);
    FM_REQUIRE(rows >= 0 && n_exp >= 1 && n_exp <= kMaxExperts && topk >= 1 && topk <= kMaxTopk, kn,
               "rows=%d n_exp=%d topk=%d: 1..%d experts, 1..%d choices", rows, n_exp, topk, kMaxExperts, kMaxTopk);
    const size_t pairs = (size_t)rows * topk;
    FM_REQUIRE(pairs <= (1u << 30), kn, "rows * topk = %zu: at most 2^30 pairs", pairs);
    FM_REQUIRE(aligned(ids, 4) && aligned(w, 4), kn, "misaligned pointer");
    FM_RANGE(ids, pairs * 4, kn, "ids");
    FM_RANGE(w, pairs * 4, kn, "weights");
    const int rc = check_plan(kn, bucket_rows, base, offsets, pairs, n_exp);
    if (rc != FM_OK) return rc;
    if (rows == 0) return no_rows(kn, c, offsets, n_exp);
    const int most = c.sm_count;
    int per_block = (int)((pairs + most - 1) / most);
    if (per_block < 512) per_block = 512;
    const int blocks = (int)((pairs + per_block - 1) / per_block);
    int* hist = static_cast<int*>(engine_scratch((size_t)blocks * n_exp * 4));
    FM_REQUIRE(hist, kn, "the engine workspace cannot grow to %zu bytes here (inside a capture: raise FM_SCRATCH_MB)", (size_t)blocks * n_exp * 4);
    const cudaError_t e = launch_kernel(plan_count_kernel, dim3(blocks), dim3(kThreads), (size_t)n_exp * 4, c.stream, pdl_enabled(), ids, w, hist, (int)pairs,
                                        n_exp, per_block);
    if (e != cudaSuccess) return cuda_fail(kn, e);
    const int rc2 = after_launch(kn);
    if (rc2 != FM_OK) return rc2;
    return run_place(kn, c, ids, w, bucket_rows, base, offsets, hist, (int)pairs, n_exp, topk, blocks, per_block);
}

const KernelEntry kRoute[] = {
    {"moe_route_k", 14, launch_route, "ppppiiiiiiiifi"},
    {"moe_plan_k", 8, launch_plan, "pppppiii"},
    {"moe_route_plan_k", 17, launch_route_plan, "pppppppiiiiiiiifi"},
};

}  // namespace

const KernelEntry* moe_route_kernels(int* n) {
    *n = (int)(sizeof(kRoute) / sizeof(kRoute[0]));
    return kRoute;
}

}  // namespace fm
