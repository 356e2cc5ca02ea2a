// What the kernels of the W4A8 product with an epilogue share: the arguments, the walk over the buckets of a plan, and
// the epilogue.
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

#include "fm_internal.h"

namespace fm {
namespace linear {

constexpr int kMaxExperts = 1024;

struct Params {
    const uint8_t* wq;         // [n_exp][N or 2N][K/2]
    const __half* ws;          // [n_exp][N or 2N][K/128]
    const int8_t *ae, *ao;     // [xrows][K/2]
    const float* asc;          // [xrows][K/128]
    const int* asu;            // [xrows][K/128]
    const float* bias;         // [n_exp][N or 2N] or nullptr
    const float* residual;     // rows of ldr values or nullptr
    float* y;                  // rows of ldy values
    const int* bucket_rows;    // [m] or nullptr: slot s takes row s of x
    const int* offsets;        // [n_exp + 1], or nullptr: one bucket of m rows
    long long ldy, ldr;
    int n_exp, m, xrows, N, K, act;
    bool gated;
};

__device__ __forceinline__ float rcp_approx(float x) {
    float d;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(x));
    return d;
}
__device__ __forceinline__ float exp_approx(float x) {               // (results below 2^-126 are 0)
    float d;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(x * 1.44269504f));
    return d;
}
// 1 / (1 + exp(-v)): the reciprocal and the power of two to one or two units in the last place
__device__ __forceinline__ float logistic(float v) { return rcp_approx(1.f + exp_approx(-v)); }
// 1 + erf(t), erf by Abramowitz and Stegun 7.1.26 (to 1.5e-7): erfcf takes three times as many instructions, which the tiles,
// whose accumulators wait meanwhile, spent a third of their time in
__device__ __forceinline__ float one_plus_erf(float t) {
    const float z = fabsf(t), k = rcp_approx(fmaf(0.3275911f, z, 1.f));
    const float q = k * fmaf(k, fmaf(k, fmaf(k, fmaf(k, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f), 0.254829592f) * exp_approx(-z * z);
    return t < 0.f ? q : 2.f - q;
}
template <int ACT>
__device__ __forceinline__ float activate(float v) {
    if (ACT == 1) return v < 0.f ? 0.f : v;                          // (NaN stays NaN)
    if (ACT == 2) return v * logistic(v);
    if (ACT == 3) return 0.5f * v * one_plus_erf(v * 0.70710678f);
    if (ACT == 4) return v * logistic(1.5957691f * (v + 0.044715f * v * v * v));      // 1 + tanh(t) = 2 / (1 + exp(-2t))
    return v;
}
template <int ACT, int N>
__device__ __forceinline__ void activate_all(float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = activate<ACT>(v[i]);
}
// N values at a time, so that the choice of the activation is one branch and the values overlap
template <int N>
__device__ __forceinline__ void activate_n(int act, float (&v)[N]) {
    switch (act) {
        case 1: activate_all<1>(v); break;
        case 2: activate_all<2>(v); break;
        case 3: activate_all<3>(v); break;
        case 4: activate_all<4>(v); break;
        default: break;
    }
}
// A unit is one tile of weight rows times one chunk of a bucket's rows; units of a chunk differ in the tile last.
struct Unit { int expert, tile, first, count; };
struct Buckets { int part[33]; };

// bounds of bucket e, held to [0, m]
__device__ __forceinline__ int bound(const Params& p, int e) { return min(max(p.offsets[e], 0), p.m); }

// Number of units; ends[e] becomes the number of units of the experts up to e.  0 for a damaged plan (bounds that fall or lie
// outside of [0, m]): nothing is read or written by it.  All threads of the CTA call it.
__device__ __forceinline__ int count_units(const Params& p, int cols, int tiles, int* ends, Buckets* bk) {
    if (!p.offsets) return (p.m + cols - 1) / cols * tiles;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    int carry = 0, damaged = 0;
    for (int e0 = 0; e0 < p.n_exp; e0 += blockDim.x) {
        const int e = e0 + (int)threadIdx.x;
        int v = 0;
        if (e < p.n_exp) {
            const int lo = p.offsets[e], hi = p.offsets[e + 1];
            damaged |= lo < 0 || hi < lo || hi > p.m;
            v = damaged ? 0 : (hi - lo + cols - 1) / cols * tiles;
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += t;
        }
        __syncthreads();
        if (lane == 31) bk->part[warp] = v;
        __syncthreads();
        int all = 0;
        for (int k = 0; k < warps; k++) {
            if (k < warp) v += bk->part[k];
            all += bk->part[k];
        }
        if (e < p.n_exp) ends[e] = carry + v;
        carry += all;
    }
    return __syncthreads_or(damaged) ? 0 : carry;
}

// TILE_LAST: the units of a bucket walk its chunks of rows first (they share a tile of weights), otherwise its tiles first
// (they share rows of x).
template <bool TILE_LAST>
__device__ __forceinline__ Unit find_unit_by(const Params& p, int u, int cols, int tiles, const int* ends) {
    Unit r;
    int lo = 0, begin = 0, end = p.m;
    if (p.offsets) {
        int hi = p.n_exp - 1;                                         // first expert whose units end behind u
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (ends[mid] > u) hi = mid;
            else lo = mid + 1;
        }
        if (lo) u -= ends[lo - 1];
        begin = bound(p, lo);
        end = bound(p, lo + 1);
    }
    const int chunks = (end - begin + cols - 1) / cols;
    r.expert = lo;
    const int i = TILE_LAST ? u / chunks : u / tiles, j = u - i * (TILE_LAST ? chunks : tiles);
    r.tile = TILE_LAST ? i : j;
    r.first = begin + (TILE_LAST ? j : i) * cols;
    r.count = min(cols, end - r.first);
    return r;
}

__device__ __forceinline__ Unit find_unit(const Params& p, int u, int cols, int tiles, const int* ends) { return find_unit_by<true>(p, u, cols, tiles, ends); }
__device__ __forceinline__ Unit find_unit_of_chunk(const Params& p, int u, int cols, int tiles, const int* ends) {
    return find_unit_by<false>(p, u, cols, tiles, ends);
}

// row of x that column c of the unit takes, or -1
__device__ __forceinline__ long long x_row(const Params& p, const Unit& u, int c) {
    if (c >= u.count) return -1;
    if (!p.bucket_rows) return u.first + c;
    const int r = p.bucket_rows[u.first + c];
    return r >= 0 && r < p.xrows ? r : -1;
}

// the tensor-core tiles (linear_w4a8_tc.cu); arguments checked
int run_tiles(const char* kn, const LaunchCtx& c, const Params& p);

}  // namespace linear
}  // namespace fm
