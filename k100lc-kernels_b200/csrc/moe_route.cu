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
//   moe_plan_k(ids, weights, bucket_rows, base, offsets, rows, n_exp, topk)
//       counting sort of the pairs by expert, stable by pair index: offsets[n_exp + 1] bounds the buckets,
//       bucket_rows[slot] is the token of a slot, base[t, j] the slot of a pair.  A pair whose id is out of range or
//       whose weight is 0 gets no slot: its base is 0 and its weight is set to 0.  Slots behind offsets[n_exp] are
//       not written.  (The device form of MoEExperts.route; reference python/k100lc_kernels/model.py:620-720.)
//
// The grid given by the caller is ignored; the arguments fix the work.
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
    bool sigmoid, renorm;
    float scale;
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
__device__ __forceinline__ uint32_t warp_max(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }
__device__ __forceinline__ uint64_t warp_max(uint64_t v) {
    const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32));
    const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
    return (uint64_t)hi << 32 | lo;
}

__device__ __forceinline__ float exp_of(float x) { return expf(x); }
__device__ __forceinline__ double exp_of(double x) { return exp(x); }
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
using fm::warp_sum;

template <typename R> struct KeyOf;
template <> struct KeyOf<float> { typedef uint32_t type; };
template <> struct KeyOf<double> { typedef uint64_t type; };

// Two fp32 keys of at most this magnitude are told apart for certain when they are this far from each other: exp and
// the division are within 2^-22, a sum of up to 1024 scores (32 in turn, then five halvings) within 37 * 2^-24 of their
// values, which are at most 1; adding the bias rounds by at most 2^-24 of the key.
__device__ __forceinline__ float resolution(float most) { return 7.6293945e-6f + 2.3841858e-7f * most; }

// s of the lane's experts (expert i * 32 + lane) in precision R
template <typename R, int VPL>
__device__ __forceinline__ void scores(const float (&x)[VPL], bool sigmoid, R (&s)[VPL]) {
    if (sigmoid) {
#pragma unroll
        for (int i = 0; i < VPL; i++) s[i] = R(1) / (R(1) + exp_of(-(R)x[i]));
        return;
    }
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < VPL; i++) m = fmaxf(m, x[i]);
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    R z = 0;
#pragma unroll
    for (int i = 0; i < VPL; i++) {
        s[i] = x[i] == m ? R(1) : x[i] > -INFINITY ? exp_of((R)x[i] - (R)m) : R(0);   // (an infinite maximum is its own score)
        if (!(x[i] > -INFINITY)) s[i] = 0;
        z += s[i];
    }
    z = warp_sum(z);
#pragma unroll
    for (int i = 0; i < VPL; i++) s[i] = s[i] / z;
}

// Takes the experts of all but the best groups out of the keys.  `s`: the values that make a group's worth.  Returns
// the distance between the worst group kept and the best one dropped (for the caller's decision whether R resolves it).
template <typename R, int VPL>
__device__ __forceinline__ R limit_groups(const RouteParams& p, typename KeyOf<R>::type (&key)[VPL], const R (&s)[VPL], R* stage) {
    typedef typename KeyOf<R>::type Key;
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < VPL; i++)
        if (i * 32 + lane < p.n_exp) stage[i * 32 + lane] = key[i] ? s[i] : -INFINITY;
    __syncwarp();
    R worth = -INFINITY;
    if (lane < p.n_group) {
        R a = -INFINITY, b = -INFINITY;
        int j = lane % p.group_size;                                  // (lanes start apart: fewer bank conflicts)
        for (int k = 0; k < p.group_size; k++) {
            const R v = stage[lane * p.group_size + j];
            if (v > a) { b = a; a = v; }
            else if (v > b) b = v;
            if (++j == p.group_size) j = 0;
        }
        worth = p.group_top == 2 && p.group_size > 1 ? (b > -INFINITY ? a + b : a) : a;
    }
    __syncwarp();
    Key w = ordered(worth);
    uint32_t kept = 0;
    R last = 0, next = -INFINITY;
    for (int k = 0; k <= p.topk_group && k < p.n_group; k++) {
        const Key best = warp_max(w);
        if (k == p.topk_group) { next = key_value(best); break; }
        if (best == 0) { last = INFINITY; break; }                    // the other groups are empty
        const int g = __ffs(__ballot_sync(0xffffffffu, w == best)) - 1;
        kept |= 1u << g;
        last = key_value(best);
        if (lane == g) w = 0;
    }
#pragma unroll
    for (int i = 0; i < VPL; i++)
        if (!((kept >> ((i * 32 + lane) / p.group_size & 31)) & 1u)) key[i] = 0;
    return last - next;
}

// The topk experts of the token in order: lane j returns the j-th (-1: none).  `near` becomes true when two keys that
// follow each other are closer than fp32 tells apart and do not come from equal inputs (checked for R = float only).
template <typename R, int VPL>
__device__ __forceinline__ int pick(const RouteParams& p, typename KeyOf<R>::type (&key)[VPL], const float (&x)[VPL], bool check, bool& near) {
    typedef typename KeyOf<R>::type Key;
    const int lane = threadIdx.x & 31;
    int mine = -1;
    float px = 0.f, pb = 0.f;
    R prev = INFINITY;
    for (int j = 0; j < p.topk + (check ? 1 : 0); j++) {
        Key best = 0;
        int at = 0;
#pragma unroll
        for (int i = 0; i < VPL; i++)
            if (key[i] > best) { best = key[i]; at = i; }
        const Key top = warp_max(best);
        if (top == 0) break;
        const int e = (int)__reduce_min_sync(0xffffffffu, best == top ? (uint32_t)(at * 32 + lane) : 0xffffffffu);
        float ex = 0.f;
#pragma unroll
        for (int i = 0; i < VPL; i++)
            if (i * 32 + lane == e) { key[i] = 0; ex = x[i]; }
        if (check) {
            ex = __shfl_sync(0xffffffffu, ex, e & 31);
            const float eb = p.bias[e];
            const R v = key_value(top);
            if (j > 0 && !(prev - v > resolution((float)fmaxf(fabsf((float)v), fabsf((float)prev)))) && !(ex == px && eb == pb)) near = true;
            prev = v;
            px = ex;
            pb = eb;
        }
        if (j < p.topk && lane == j) mine = e;
    }
    return mine;
}

// One warp per token.  With a bias the keys are rounded sums: they are formed in fp32 first, and a token where two
// keys (or the last group kept and the first one dropped) lie within the error of fp32 is decided again in fp64, so
// that the choice is that of the exact keys at fp32's cost.
template <typename T, int VPL>
__global__ void __launch_bounds__(128)
route_kernel(const RouteParams p) {
    extern __shared__ double stage_all[];
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row = blockIdx.x * 4 + warp;
    if (row >= p.rows) return;
    double* stage = stage_all + (size_t)warp * p.n_exp;
    const T* in = reinterpret_cast<const T*>(p.logits) + (size_t)row * p.n_exp;
    float x[VPL];
#pragma unroll
    for (int i = 0; i < VPL; i++) {
        const int e = i * 32 + lane;
        x[i] = e < p.n_exp ? logit_at(in, e) : -INFINITY;
        if (!(x[i] > -INFINITY)) x[i] = -INFINITY;                    // NaN: never chosen
    }
    float s[VPL];
    scores<float, VPL>(x, p.sigmoid, s);
    uint32_t key[VPL];
    int mine;
    if (!p.bias) {
#pragma unroll
        for (int i = 0; i < VPL; i++) key[i] = ordered(x[i]);
        bool near = false;
        if (p.n_group > 1 && p.group_top == 1) limit_groups<float, VPL>(p, key, x, reinterpret_cast<float*>(stage));
        else if (p.n_group > 1) {
            const float gap = limit_groups<float, VPL>(p, key, s, reinterpret_cast<float*>(stage));
            near = !(gap > 2.f * resolution(1.f));
        }
        if (near) {
            double sd[VPL];
            uint64_t kd[VPL];
            scores<double, VPL>(x, p.sigmoid, sd);
#pragma unroll
            for (int i = 0; i < VPL; i++) kd[i] = ordered((double)x[i]);
            limit_groups<double, VPL>(p, kd, sd, stage);
#pragma unroll
            for (int i = 0; i < VPL; i++) key[i] = kd[i] ? ordered(x[i]) : 0u;
        }
        mine = pick<float, VPL>(p, key, x, false, near);
    } else {
        float v[VPL];
#pragma unroll
        for (int i = 0; i < VPL; i++) {
            const int e = i * 32 + lane;
            v[i] = x[i] > -INFINITY ? s[i] + p.bias[e] : -INFINITY;
            key[i] = ordered(v[i]);
        }
        bool near = false;
        if (p.n_group > 1) {
            float most = 0.f;                                         // the largest finite key: what fp32 resolves
#pragma unroll
            for (int i = 0; i < VPL; i++)
                if (key[i]) most = fmaxf(most, fabsf(v[i]));
#pragma unroll
            for (int o = 16; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
            const float gap = limit_groups<float, VPL>(p, key, v, reinterpret_cast<float*>(stage));
            near = !(gap > 2.f * resolution(most));                   // (a group's worth is a sum of two)
        }
        if (!near) mine = pick<float, VPL>(p, key, x, true, near);
        if (near) {
            double vd[VPL];
            uint64_t kd[VPL];
            scores<double, VPL>(x, p.sigmoid, vd);
#pragma unroll
            for (int i = 0; i < VPL; i++) {
                vd[i] = x[i] > -INFINITY ? vd[i] + (double)p.bias[i * 32 + lane] : -INFINITY;
                kd[i] = ordered(vd[i]);
            }
            if (p.n_group > 1) limit_groups<double, VPL>(p, kd, vd, stage);
            mine = pick<double, VPL>(p, kd, x, false, near);
        }
    }
    // the scores of the chosen, from the lanes that hold them
    float w = 0.f;
    for (int j = 0; j < p.topk; j++) {
        const int e = __shfl_sync(0xffffffffu, mine, j);
        float v = 0.f;
#pragma unroll
        for (int i = 0; i < VPL; i++)
            if (i * 32 + lane == e) v = s[i];
        v = __shfl_sync(0xffffffffu, v, e & 31);
        if (lane == j && e >= 0) w = v;
    }
    if (p.renorm) {
        const float sum = warp_sum(lane < p.topk ? w : 0.f);
        w = sum > 0.f ? w / sum : 0.f;
    }
    if (lane < p.topk) {
        p.ids[(size_t)row * p.topk + lane] = mine;
        p.weights[(size_t)row * p.topk + lane] = w * p.scale;
    }
    pdl_launch_dependents();
}

template <typename T>
cudaError_t run_route(const LaunchCtx& c, const RouteParams& p) {
    const dim3 grid((unsigned)((p.rows + 3) / 4)), block(128);
    const size_t smem = p.n_group > 1 ? (size_t)4 * p.n_exp * 8 : 0;
    const int vpl = (p.n_exp + 31) / 32;
#define FM_ROUTE(V) return launch_kernel(route_kernel<T, V>, grid, block, smem, c.stream, pdl_enabled(), p)
    if (vpl <= 1) FM_ROUTE(1);
    if (vpl <= 2) FM_ROUTE(2);
    if (vpl <= 4) FM_ROUTE(4);
    if (vpl <= 8) FM_ROUTE(8);
    if (vpl <= 16) FM_ROUTE(16);
    FM_ROUTE(32);
#undef FM_ROUTE
}

int launch_route(const LaunchCtx& c, const uint64_t* a) {
    const char* kn = "moe_route_k";
    RouteParams p;
    p.logits = arg_ptr<const void>(a[0]);
    p.bias = arg_ptr<const float>(a[1]);
    p.ids = arg_ptr<int>(a[2]);
    p.weights = arg_ptr<float>(a[3]);
    p.rows = arg_i32(a[4]);
    p.n_exp = arg_i32(a[5]);
    p.topk = arg_i32(a[6]);
    p.n_group = arg_i32(a[7]);
    p.topk_group = arg_i32(a[8]);
    p.group_top = arg_i32(a[9]);
    const int score = arg_i32(a[10]), renorm = arg_i32(a[11]), dtype = arg_i32(a[13]);
    p.scale = arg_f32(a[12]);
    FM_REQUIRE(p.rows >= 0 && p.n_exp >= 1 && p.n_exp <= kMaxExperts, kn, "rows=%d n_exp=%d: 1..%d experts", p.rows, p.n_exp, kMaxExperts);
    FM_REQUIRE(p.n_group >= 1 && p.n_group <= kMaxGroups && p.n_exp % p.n_group == 0, kn, "n_group=%d must divide n_exp=%d and be at most %d",
               p.n_group, p.n_exp, kMaxGroups);
    FM_REQUIRE(p.topk_group >= 1 && p.topk_group <= p.n_group, kn, "topk_group=%d of %d groups", p.topk_group, p.n_group);
    FM_REQUIRE(p.topk >= 1 && p.topk <= kMaxTopk && p.topk <= p.n_exp / p.n_group * p.topk_group, kn,
               "topk=%d: at most %d, and at most the experts of the kept groups", p.topk, kMaxTopk);
    FM_REQUIRE(p.group_top == 1 || p.group_top == 2, kn, "group_top=%d: 1 or 2", p.group_top);
    FM_REQUIRE((score == 0 || score == 1) && (renorm == 0 || renorm == 1), kn, "score=%d renorm=%d: 0 or 1", score, renorm);
    FM_REQUIRE(dtype >= 0 && dtype <= 2, kn, "dtype=%d: 0 f32, 1 bf16, 2 f16", dtype);
    p.sigmoid = score == 1;
    p.renorm = renorm == 1;
    p.group_size = p.n_exp / p.n_group;
    if (p.rows == 0) return FM_OK;
    const size_t es = dtype == 0 ? 4 : 2, pairs = (size_t)p.rows * p.topk;
    FM_REQUIRE(pairs <= 0x7fffffff, kn, "rows * topk exceeds 2^31 - 1");
    FM_REQUIRE(aligned(p.logits, es) && aligned(p.bias, 4) && aligned(p.ids, 4) && aligned(p.weights, 4), kn, "misaligned pointer");
    FM_RANGE(p.logits, (size_t)p.rows * p.n_exp * es, kn, "logits");
    if (p.bias) FM_RANGE(p.bias, (size_t)p.n_exp * 4, kn, "bias");
    FM_RANGE(p.ids, pairs * 4, kn, "ids");
    FM_RANGE(p.weights, pairs * 4, kn, "weights");
    const cudaError_t e = dtype == 0 ? run_route<float>(c, p) : dtype == 1 ? run_route<__nv_bfloat16>(c, p) : run_route<__half>(c, p);
    return e == cudaSuccess ? after_launch(kn) : cuda_fail(kn, e);
}

// ------------------------------------------------------------------------------------------------------ the plan
// A block takes kChunk consecutive pairs, a warp kChunk / 8 of them in batches of 32.  The slot of a pair is
//   (pairs of smaller experts) + (pairs of its expert in earlier blocks, warps, batches and lanes),
// so the order is that of the pair indices whatever the scheduling: no atomics decide a position.
constexpr int kPlanThreads = 256, kPlanWarps = kPlanThreads / 32, kChunk = 2048, kPerWarp = kChunk / kPlanWarps;

__device__ __forceinline__ int pair_expert(const int* ids, const float* w, int i, int pairs, int n_exp) {
    if (i >= pairs) return -1;
    const int e = ids[i];
    return e >= 0 && e < n_exp && w[i] != 0.f ? e : -1;
}

// hist[block][n_exp]
__global__ void __launch_bounds__(kPlanThreads)
plan_count_kernel(const int* __restrict__ ids, const float* __restrict__ w, int* __restrict__ hist, int pairs, int n_exp) {
    extern __shared__ int count[];
    pdl_wait();
    for (int e = threadIdx.x; e < n_exp; e += kPlanThreads) count[e] = 0;
    __syncthreads();
    const int lo = blockIdx.x * kChunk;
    for (int i = lo + threadIdx.x; i < lo + kChunk; i += kPlanThreads) {
        const int e = pair_expert(ids, w, i, pairs, n_exp);
        if (e >= 0) atomicAdd(&count[e], 1);                          // (integers: the order does not matter)
    }
    __syncthreads();
    for (int e = threadIdx.x; e < n_exp; e += kPlanThreads) hist[(size_t)blockIdx.x * n_exp + e] = count[e];
    pdl_launch_dependents();
}

__global__ void __launch_bounds__(kPlanThreads)
plan_place_kernel(const int* __restrict__ ids, float* __restrict__ w, int* __restrict__ bucket_rows, int* __restrict__ base,
                  int* __restrict__ offsets, const int* __restrict__ hist, int pairs, int n_exp, int topk) {
    extern __shared__ int sm[];
    int* start = sm;                                                  // [n_exp] first slot of this block's pairs
    int* cnt = sm + n_exp;                                            // [kPlanWarps][n_exp]
    __shared__ int warp_total[kPlanWarps];
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int i = threadIdx.x; i < kPlanWarps * n_exp; i += kPlanThreads) cnt[i] = 0;
    // totals per expert over all blocks and over the earlier ones; exclusive scan over the experts
    int carry = 0;
    for (int e0 = 0; e0 < n_exp; e0 += kPlanThreads) {
        const int e = e0 + threadIdx.x;
        int total = 0, before = 0;
        if (e < n_exp)
            for (int b = 0; b < (int)gridDim.x; b++) {
                const int h = hist[(size_t)b * n_exp + e];
                if (b < (int)blockIdx.x) before += h;
                total += h;
            }
        int inc = total;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += t;
        }
        __syncthreads();
        if (lane == 31) warp_total[warp] = inc;
        __syncthreads();
        int lower = carry, all = 0;
        for (int k = 0; k < kPlanWarps; k++) {
            if (k < warp) lower += warp_total[k];
            all += warp_total[k];
        }
        if (e < n_exp) {
            start[e] = lower + inc - total + before;
            if (blockIdx.x == 0) {
                offsets[e] = lower + inc - total;
                if (e == n_exp - 1) offsets[n_exp] = lower + inc;
            }
        }
        carry += all;
    }
    __syncthreads();
    // this warp's pairs per expert
    const int lo = blockIdx.x * kChunk + warp * kPerWarp;
    for (int i = lo + lane; i < lo + kPerWarp; i += 32) {
        const int e = pair_expert(ids, w, i, pairs, n_exp);
        if (e >= 0) atomicAdd(&cnt[warp * n_exp + e], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < n_exp; e += kPlanThreads) {
        int at = start[e];
        for (int k = 0; k < kPlanWarps; k++) {
            const int h = cnt[k * n_exp + e];
            cnt[k * n_exp + e] = at;
            at += h;
        }
    }
    __syncthreads();
    for (int i0 = lo; i0 < lo + kPerWarp && i0 < pairs; i0 += 32) {
        const int i = i0 + lane;
        const int e = pair_expert(ids, w, i, pairs, n_exp);
        const uint32_t peers = __match_any_sync(0xffffffffu, e);
        const int rank = __popc(peers & ((1u << lane) - 1u));
        int slot = 0;
        if (e >= 0) slot = cnt[warp * n_exp + e] + rank;
        __syncwarp();
        if (e >= 0 && rank == 0) cnt[warp * n_exp + e] += __popc(peers);
        __syncwarp();
        if (i < pairs) {
            base[i] = slot;
            if (e >= 0) bucket_rows[slot] = i / topk;
            else w[i] = 0.f;
        }
    }
    pdl_launch_dependents();
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
    FM_REQUIRE(pairs <= 0x7fffffff - kChunk, kn, "rows * topk exceeds what 32-bit slots can name");
    FM_REQUIRE(aligned(ids, 4) && aligned(w, 4) && aligned(bucket_rows, 4) && aligned(base, 4) && aligned(offsets, 4), kn, "misaligned pointer");
    FM_RANGE(ids, pairs * 4, kn, "ids");
    FM_RANGE(w, pairs * 4, kn, "weights");
    FM_RANGE(bucket_rows, pairs * 4, kn, "bucket_rows");
    FM_RANGE(base, pairs * 4, kn, "base");
    FM_RANGE(offsets, (size_t)(n_exp + 1) * 4, kn, "offsets");
    const int blocks = pairs ? (int)((pairs + kChunk - 1) / kChunk) : 1;   // (no rows: the offsets are still written)
    int* hist = static_cast<int*>(engine_scratch((size_t)blocks * n_exp * 4));
    FM_REQUIRE(hist, kn, "the engine workspace cannot grow to %zu bytes here (inside a capture: raise FM_SCRATCH_MB)", (size_t)blocks * n_exp * 4);
    cudaError_t e = launch_kernel(plan_count_kernel, dim3(blocks), dim3(kPlanThreads), (size_t)n_exp * 4, c.stream, pdl_enabled(), ids, w,
                                  hist, (int)pairs, n_exp);
    if (e != cudaSuccess) return cuda_fail(kn, e);
    const int rc = after_launch(kn);
    if (rc != FM_OK) return rc;
    e = launch_kernel(plan_place_kernel, dim3(blocks), dim3(kPlanThreads), (size_t)n_exp * 4 * (1 + kPlanWarps), c.stream, pdl_enabled(), ids, w,
                      bucket_rows, base, offsets, hist, (int)pairs, n_exp, topk);
    return e == cudaSuccess ? after_launch(kn) : cuda_fail(kn, e);
}

const KernelEntry kRoute[] = {
    {"moe_route_k", 14, launch_route, "ppppiiiiiiiifi"},
    {"moe_plan_k", 8, launch_plan, "pppppiii"},
};

}  // namespace

const KernelEntry* moe_route_kernels(int* n) {
    *n = (int)(sizeof(kRoute) / sizeof(kRoute[0]));
    return kRoute;
}

}  // namespace fm
