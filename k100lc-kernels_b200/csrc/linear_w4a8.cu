// W4A8 product with an epilogue, for one weight matrix and for a stack of experts, any number of rows.
//
//   linear_w4a8_k(wq, ws, ae, ao, asc, asu, bias, residual, y, M, N, K, ldy, ldr, act, gated)
//       y[m, n] = act(v[m, n]) + residual[m, n]            v = sum_g (f16(ws[n, g]) * asc[m, g]) * float(I[m, n, g]) + bias[n]
//       gated:  y[m, n] = act(v[m, n]) * v[m, N + n] + residual[m, n]   (2N weight rows: N gate rows, then N up rows)
//   moe_linear_w4a8_k(wq, ws, ae, ao, asc, asu, bias, bucket_rows, offsets, y, n_exp, pairs, xrows, N, K, ldy, act, gated)
//       the same for every expert e of a plan (moe_plan_k): slot s of bucket [offsets[e], offsets[e + 1]) takes the
//       codes of row bucket_rows[s] (bucket_rows = 0: of row s), the weights and the bias of expert e, and writes
//       y[s].  Rows behind offsets[n_exp] are not written.
//
//   I[m, n, g] = sum_{k in 128-group g} w[n, k] * q[m, k] is the exact integer of the by-name GEMVs, the codes are those of
//   quant_act; act: 0 none, 1 relu, 2 silu, 3 gelu (erf), 4 gelu (tanh).  bias and residual may be 0; the residual may
//   be y itself.  The grid given by the caller is ignored.
//
// A warp owns 16 weight rows (gated: 8 gate rows and the 8 up rows beside them, so that a lane holds both factors) and
// multiplies one 128-group at a time with mma.sync m16n8k32, the rows of x being the columns of B.  The four lanes that
// share a fragment row read the 64 bytes of its group as one 16-byte word each; a word's low and high nibbles are the
// even and odd k, which is how the codes are stored, so both operands go from memory to the MMA without a shuffle.
// Nibbles enter as u = nibble ^ 8 (u8 x s8), the accumulators start at -8 * sum(q).
#include <cuda_fp16.h>

#include "device_utils.cuh"
#include "fm_internal.h"
#include "linear_w4a8.cuh"

namespace fm {
namespace linear {
namespace {

constexpr int kWarps = 8, kThreads = kWarps * 32;

__device__ __forceinline__ void mma_u8s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t lo_u(uint32_t w) { return (w & 0x0F0F0F0Fu) ^ 0x08080808u; }
__device__ __forceinline__ uint32_t hi_u(uint32_t w) { return ((w >> 4) & 0x0F0F0F0Fu) ^ 0x08080808u; }
__device__ __forceinline__ uint32_t word(const uint4& v, int j) { return j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w; }

// NT: fragments of eight rows of x that share the weights in registers
template <int NT, bool GATED>
__global__ void __launch_bounds__(kThreads)
rows_kernel(const Params p, int wk) {
    __shared__ float join[kWarps][NT][4][32];
    __shared__ Buckets bk;
    extern __shared__ int ends[];                                     // [n_exp] units up to and including expert e
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, fr = lane >> 2, fq = lane & 3;
    constexpr int COLS = 8 * NT, ROWS = GATED ? 8 : 16;
    const int tiles = (p.N + ROWS - 1) / ROWS, G = p.K / 128;
    const int total = count_units(p, COLS, tiles, ends, &bk);
    const int per_cta = kWarps / wk, sub = warp / wk, part = warp % wk;
    for (int u0 = blockIdx.x * per_cta; u0 < total; u0 += gridDim.x * per_cta) {
        const int u = u0 + sub;
        const bool live = u < total;
        Unit un = {0, 0, 0, 0, 0};
        if (live) un = find_unit(p, u, COLS, tiles, ends);
        const int n0 = un.tile * ROWS;
        float acc[NT][4];
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) acc[t][i] = 0.f;
        if (live) {
            // the two weight rows of this lane's fragment (rows past the end repeat the last one and are not stored)
            const int ra = min(n0 + fr, p.N - 1), rb = GATED ? p.N + ra : min(n0 + 8 + fr, p.N - 1);
            const size_t row0 = (size_t)un.expert * (GATED ? 2 * p.N : p.N);
            const uint8_t* wa = p.wq + (row0 + ra) * (size_t)(p.K / 2) + fq * 16;
            const uint8_t* wb = p.wq + (row0 + rb) * (size_t)(p.K / 2) + fq * 16;
            const __half* sa = p.ws + (row0 + ra) * (size_t)G;
            const __half* sb = p.ws + (row0 + rb) * (size_t)G;
            const int8_t *xe[NT], *xo[NT];                            // codes of column fr; nullptr: no such row
            const float* cs[NT][2];                                   // scales of columns 2 fq and 2 fq + 1
            const int* cu[NT][2];
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const long long r = x_row(p, un, t * 8 + fr);
                xe[t] = r < 0 ? nullptr : p.ae + (size_t)r * (p.K / 2) + fq * 16;
                xo[t] = r < 0 ? nullptr : p.ao + (size_t)r * (p.K / 2) + fq * 16;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const long long c = x_row(p, un, t * 8 + fq * 2 + h);
                    cs[t][h] = c < 0 ? nullptr : p.asc + (size_t)c * G;
                    cu[t][h] = c < 0 ? nullptr : p.asu + (size_t)c * G;
                }
            }
#pragma unroll 2
            for (int g = part; g < G; g += wk) {
                const uint4 va = ld_stream_v4(wa + (size_t)g * 64), vb = ld_stream_v4(wb + (size_t)g * 64);
                const float fa = __half2float(sa[g]), fb = __half2float(sb[g]);
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    const uint4 z = make_uint4(0, 0, 0, 0);
                    const uint4 e = xe[t] ? *reinterpret_cast<const uint4*>(xe[t] + (size_t)g * 64) : z;
                    const uint4 o = xo[t] ? *reinterpret_cast<const uint4*>(xo[t] + (size_t)g * 64) : z;
                    const float s0 = cs[t][0] ? cs[t][0][g] : 0.f, s1 = cs[t][1] ? cs[t][1][g] : 0.f;
                    const int u0q = cu[t][0] ? -8 * cu[t][0][g] : 0, u1q = cu[t][1] ? -8 * cu[t][1][g] : 0;
                    int c[4] = {u0q, u1q, u0q, u1q};
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        mma_u8s8(c, lo_u(word(va, j)), lo_u(word(vb, j)), hi_u(word(va, j)), hi_u(word(vb, j)), word(e, j), word(o, j));
                    acc[t][0] = fmaf((float)c[0], fa * s0, acc[t][0]);
                    acc[t][1] = fmaf((float)c[1], fa * s1, acc[t][1]);
                    acc[t][2] = fmaf((float)c[2], fb * s0, acc[t][2]);
                    acc[t][3] = fmaf((float)c[3], fb * s1, acc[t][3]);
                }
            }
        }
        if (wk > 1) {                                                 // add the K parts, in the order of the parts
            __syncthreads();
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) join[warp][t][i][lane] = acc[t][i];
            __syncthreads();
            if (part == 0) {
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        for (int k = 1; k < wk; k++) acc[t][i] += join[warp + k][t][i][lane];
            }
        }
        if (live && part == 0) {
            const float* bias = p.bias ? p.bias + (size_t)un.expert * (GATED ? 2 * p.N : p.N) : nullptr;
            const int na = n0 + fr, nb = GATED ? p.N + na : na + 8;   // the lane's two weight rows
            const bool has_a = na < p.N, has_b = GATED ? has_a : nb < p.N;
            const float ba = bias && has_a ? bias[na] : 0.f, bb = bias && has_b ? bias[nb] : 0.f;
            const long long end = (long long)un.first + un.count;
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const long long m = (long long)un.first + t * 8 + fq * 2;
                float v[2] = {acc[t][0] + ba, acc[t][1] + ba}, w[2] = {acc[t][2] + bb, acc[t][3] + bb};
                if (m >= end) continue;
                if (GATED) {
                    if (has_a) finish<2, true>(p, m, 1, end, na, v, w);
                } else {
                    if (has_a) finish<2, false>(p, m, 1, end, na, v, v);
                    if (has_b) finish<2, false>(p, m, 1, end, nb, w, w);
                }
            }
        }
    }
    pdl_launch_dependents();
}

template <int NT>
cudaError_t run_rows(const LaunchCtx& c, const Params& p) {
    const int cols = 8 * NT, rows = p.gated ? 8 : 16, tiles = (p.N + rows - 1) / rows, G = p.K / 128;
    // the K dimension is split over the warps of a CTA while a warp keeps at least four groups
    int wk = 1;
    while (wk < kWarps && G / (wk * 2) >= 4) wk *= 2;
    long long chunks = (p.m + cols - 1) / cols;
    if (p.offsets) chunks = p.n_exp < p.m ? chunks + p.n_exp : p.m;   // every bucket may end in a part of a chunk
    const long long units = chunks * tiles;
    long long grid = (units + kWarps / wk - 1) / (kWarps / wk);
    if (grid > c.sm_count * 8LL) grid = c.sm_count * 8LL;
    const size_t smem = p.offsets ? (size_t)p.n_exp * 4 : 0;
    return p.gated ? launch_kernel(rows_kernel<NT, true>, dim3((unsigned)grid), dim3(kThreads), smem, c.stream, pdl_enabled(), p, wk)
                   : launch_kernel(rows_kernel<NT, false>, dim3((unsigned)grid), dim3(kThreads), smem, c.stream, pdl_enabled(), p, wk);
}

int run(const char* kn, const LaunchCtx& c, const Params& p) {
    // rows per bucket, were all experts equally popular
    const int per = p.offsets ? p.m / (p.n_exp < p.m ? p.n_exp : p.m) : p.m;
    if (per >= 16) return run_tiles(kn, c, p);
    const cudaError_t e = p.m <= 8 || p.offsets ? run_rows<1>(c, p) : run_rows<2>(c, p);
    return e == cudaSuccess ? after_launch(kn) : cuda_fail(kn, e);
}

// what both entries check: weights, codes of `xrows` rows, `m` output rows
int check(const char* kn, const Params& p, int n_exp, long long xrows) {
    FM_REQUIRE(p.N >= 1 && p.K >= 128 && p.K % 128 == 0, kn, "N=%d K=%d: K must be a positive multiple of 128", p.N, p.K);
    FM_REQUIRE(p.act >= 0 && p.act <= 4, kn, "act=%d: 0 none, 1 relu, 2 silu, 3 gelu, 4 gelu (tanh)", p.act);
    FM_REQUIRE(p.ldy >= p.N && (!p.residual || p.ldr >= p.N), kn, "ldy=%lld ldr=%lld: rows of %d values overlap", p.ldy, p.ldr, p.N);
    FM_REQUIRE(p.N <= (1 << 28) && p.K <= (1 << 24), kn, "N=%d K=%d is too large", p.N, p.K);
    FM_REQUIRE(aligned(p.wq, 16) && aligned(p.ae, 16) && aligned(p.ao, 16), kn, "wq, ae and ao must be 16-byte aligned");
    FM_REQUIRE(aligned(p.ws, 2) && aligned(p.asc, 4) && aligned(p.asu, 4) && aligned(p.bias, 4) && aligned(p.residual, 4) && aligned(p.y, 4), kn,
               "misaligned pointer");
    const size_t wr = (size_t)n_exp * p.N * (p.gated ? 2 : 1), G = p.K / 128;
    FM_RANGE(p.wq, wr * (p.K / 2), kn, "wq");
    FM_RANGE(p.ws, wr * G * 2, kn, "ws");
    FM_RANGE(p.ae, (size_t)xrows * (p.K / 2), kn, "ae");
    FM_RANGE(p.ao, (size_t)xrows * (p.K / 2), kn, "ao");
    FM_RANGE(p.asc, (size_t)xrows * G * 4, kn, "asc");
    FM_RANGE(p.asu, (size_t)xrows * G * 4, kn, "asu");
    if (p.bias) FM_RANGE(p.bias, wr * 4, kn, "bias");
    FM_RANGE(p.y, ((size_t)(p.m - 1) * p.ldy + p.N) * 4, kn, "y");
    if (p.residual) {
        FM_RANGE(p.residual, ((size_t)(p.m - 1) * p.ldr + p.N) * 4, kn, "residual");
        // element by element it may be y itself; shifted against y, values would be read after they were replaced
        const uintptr_t y = reinterpret_cast<uintptr_t>(p.y), r = reinterpret_cast<uintptr_t>(p.residual);
        const bool apart = r >= y + ((size_t)(p.m - 1) * p.ldy + p.N) * 4 || y >= r + ((size_t)(p.m - 1) * p.ldr + p.N) * 4;
        FM_REQUIRE(apart || (r == y && p.ldr == p.ldy), kn, "the residual overlaps y without being y");
    }
    return FM_OK;
}

int launch_linear(const LaunchCtx& c, const uint64_t* a) {
    const char* kn = "linear_w4a8_k";
    Params p = {};
    p.wq = arg_ptr<const uint8_t>(a[0]);
    p.ws = arg_ptr<const __half>(a[1]);
    p.ae = arg_ptr<const int8_t>(a[2]);
    p.ao = arg_ptr<const int8_t>(a[3]);
    p.asc = arg_ptr<const float>(a[4]);
    p.asu = arg_ptr<const int>(a[5]);
    p.bias = arg_ptr<const float>(a[6]);
    p.residual = arg_ptr<const float>(a[7]);
    p.y = arg_ptr<float>(a[8]);
    p.m = arg_i32(a[9]);
    p.N = arg_i32(a[10]);
    p.K = arg_i32(a[11]);
    p.ldy = arg_i32(a[12]);
    p.ldr = arg_i32(a[13]);
    p.act = arg_i32(a[14]);
    FM_REQUIRE(p.m >= 0 && (arg_i32(a[15]) == 0 || arg_i32(a[15]) == 1), kn, "M=%d gated=%d", p.m, arg_i32(a[15]));
    p.gated = arg_i32(a[15]) == 1;
    p.n_exp = 1;
    if (p.m == 0) return FM_OK;
    const int rc = check(kn, p, 1, p.m);
    return rc != FM_OK ? rc : run(kn, c, p);
}

int launch_moe_linear(const LaunchCtx& c, const uint64_t* a) {
    const char* kn = "moe_linear_w4a8_k";
    Params p = {};
    p.wq = arg_ptr<const uint8_t>(a[0]);
    p.ws = arg_ptr<const __half>(a[1]);
    p.ae = arg_ptr<const int8_t>(a[2]);
    p.ao = arg_ptr<const int8_t>(a[3]);
    p.asc = arg_ptr<const float>(a[4]);
    p.asu = arg_ptr<const int>(a[5]);
    p.bias = arg_ptr<const float>(a[6]);
    p.bucket_rows = arg_ptr<const int>(a[7]);
    p.offsets = arg_ptr<const int>(a[8]);
    p.y = arg_ptr<float>(a[9]);
    p.n_exp = arg_i32(a[10]);
    p.m = arg_i32(a[11]);
    const int xrows = arg_i32(a[12]);
    p.N = arg_i32(a[13]);
    p.K = arg_i32(a[14]);
    p.ldy = arg_i32(a[15]);
    p.act = arg_i32(a[16]);
    FM_REQUIRE(p.m >= 0 && xrows >= 0 && (arg_i32(a[17]) == 0 || arg_i32(a[17]) == 1), kn, "pairs=%d xrows=%d gated=%d", p.m, xrows, arg_i32(a[17]));
    p.gated = arg_i32(a[17]) == 1;
    p.xrows = xrows;
    FM_REQUIRE(p.n_exp >= 1 && p.n_exp <= kMaxExperts, kn, "n_exp=%d: 1..%d", p.n_exp, kMaxExperts);
    if (p.m == 0) return FM_OK;
    FM_REQUIRE(xrows >= 1 && (p.bucket_rows || xrows >= p.m), kn, "xrows=%d: without bucket_rows every one of the %d slots has a row of its own", xrows, p.m);
    const int rc = check(kn, p, p.n_exp, xrows);
    if (rc != FM_OK) return rc;
    FM_REQUIRE(p.offsets && aligned(p.offsets, 4) && aligned(p.bucket_rows, 4), kn, "misaligned pointer");
    FM_RANGE(p.offsets, (size_t)(p.n_exp + 1) * 4, kn, "offsets");
    if (p.bucket_rows) FM_RANGE(p.bucket_rows, (size_t)p.m * 4, kn, "bucket_rows");
    return run(kn, c, p);
}

const KernelEntry kLinear[] = {
    {"linear_w4a8_k", 16, launch_linear, "pppppppppiiiiiii"},
    {"moe_linear_w4a8_k", 18, launch_moe_linear, "ppppppppppiiiiiiii"},
};

}  // namespace
}  // namespace linear

const KernelEntry* linear_kernels(int* n) {
    *n = (int)(sizeof(linear::kLinear) / sizeof(linear::kLinear[0]));
    return linear::kLinear;
}

}  // namespace fm
