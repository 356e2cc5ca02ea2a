// W4A8 product with an epilogue, for one weight matrix and for a stack of experts, any number of rows.
//
//   linear_w4a8_k(wq, ws, ae, ao, asc, asu, bias, residual, y, M, N, K, ldy, ldr, act, gated)
//       y[m, n] = act(v[m, n]) + residual[m, n]            v = sum_g (f16(ws[n, g]) * asc[m, g]) * float(I[m, n, g]) + bias[n]
//       gated:  y[m, n] = act(v[m, n]) * v[m, N + n] + residual[m, n]   (2N weight rows: N gate rows, then N up rows)
//   moe_linear_w4a8_k(wq, ws, ae, ao, asc, asu, bias, bucket_rows, offsets, y, n_exp, pairs, xrows, N, K, ldy, act, gated)
//       the same for every expert e of a plan (moe_plan_k): slot s of bucket [offsets[e], offsets[e + 1]) takes the
//       codes of row bucket_rows[s] (bucket_rows = 0: of row s), the weights and the bias of expert e, and writes
//       y[s].  Rows behind offsets[n_exp] are not written.  A bucket_rows[s] outside of [0, xrows) stands for a row of zeros.
//
//   I[m, n, g] = sum_{k in 128-group g} w[n, k] * q[m, k] is the exact integer of the by-name GEMVs, the codes are those of
//   quant_act (asu, the sums of the codes, is not needed here); act: 0 none, 1 relu, 2 silu, 3 gelu (erf), 4 gelu (tanh).  bias
//   and residual may be 0; the residual may be y itself.  The grid given by the caller is ignored.
//
// A warp owns 16 weight rows (gated: 8 gate rows and the 8 up rows beside them, so that a lane holds both factors) and
// multiplies one 128-group at a time with mma.sync m16n8k32, the rows of x being the columns of B.  The four lanes that
// share a weight row read the 64 bytes of its group as one 16-byte word each; a word's low and high nibbles are the even
// and odd k, which is how the codes are stored, so both operands go from memory to the MMA without a shuffle.  Nibbles
// enter in the upper half of their byte, as the int8 value 16 w (one or two logic instructions a word, no sum of the codes
// to correct by); the 16 is divided out at the end, exactly.
// Bound by HBM.  A warp asks for a group of its next chunk (four groups: 256 bytes of every row) as soon as it has multiplied
// that group of the current one, so that 4 KB a warp are on their way at any time, across the ends of its units too.  Where
// there are fewer units than warps the K dimension is split over the warps of a team and their partial sums meet in shared
// memory.  Measured (B200, cold weights): one row of 17408 x 5120 12.3 us (11.0 in a graph, 4.2 TB/s; 8 rows 11.9), five rows of
// 5120 x 17408 18.3 us (16.0), 33 tokens through 8 of 64 experts of 5120 x 1024 35 to 38 us (4.6 to 5 TB/s, 0.70 to 0.76 of a copy's rate): what is left
// is the time from a launch to the first weights and the last unit's tail.
#include <cuda_fp16.h>

#include "device_utils.cuh"
#include "fm_internal.h"
#include "linear_w4a8.cuh"

namespace fm {
namespace linear {
namespace {

constexpr int kMaxWarps = 8, kCtasPerSm = 2;        // at 128 registers a thread
constexpr int CH = 4;                               // groups of a chunk
constexpr int COLS = 8;                             // rows of x of a unit

__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_s8_first(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));
}
// read-once data, and the 256 bytes around it on their way to L2
__device__ __forceinline__ uint4 ld_stream_256(const void* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t lo16(uint32_t w) { return (w << 4) & 0xF0F0F0F0u; }
__device__ __forceinline__ uint32_t hi16(uint32_t w) { return w & 0xF0F0F0F0u; }
__device__ __forceinline__ uint32_t word(const uint4& v, int j) { return j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w; }

// y[m + i, n] for the N sums v (gated: gates v, ups u); rows from `end` on are left alone.  The bias is in the
// sums already.  All residuals are read before the first value is written: an element is the residual of itself only.
template <int N, bool GATED>
__device__ __forceinline__ void finish(const Params& p, long long m, long long end, int n, float (&v)[N], const float (&u)[N]) {
    float r[N];
#pragma unroll
    for (int i = 0; i < N; i++) r[i] = p.residual && m + i < end ? p.residual[(m + i) * p.ldr + n] : 0.f;
    activate_n(p.act, v);
#pragma unroll
    for (int i = 0; i < N; i++)
        if (m + i < end) {
            float o = GATED ? v[i] * u[i] : v[i];
            if (p.residual) o += r[i];
            p.y[(m + i) * p.ldy + n] = o;
        }
}

// wk warps, a team, share a unit; blockDim = 32 * wk * (teams of a CTA), and every team has a run of units of its own.
// WHOLE: K is a multiple of 512; otherwise the groups past the end of a row repeat its last one with scale 0.
// GATHER: a slot's row of x is named by the plan, which may name none; its sums are 0 then.  (The two flags for that, kept without
// GATHER as well, made 33 tokens through 8 of 64 experts of 5120 x 1024 in bucket order take 38.4 us instead of 37.0; flags that
// zero the scales as they are loaded, one token through 8 gated experts 14.2 us instead of 13.5.)
template <bool GATED, bool WHOLE, bool GATHER>
__global__ void __launch_bounds__(kMaxWarps * 32, kCtasPerSm)
rows_kernel(const Params p, int wk) {
    __shared__ float join[2][kMaxWarps][4][32];
    __shared__ Buckets bk;
    extern __shared__ int ends[];                                     // [n_exp] units up to and including expert e
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, fr = lane >> 2, fq = lane & 3;
    constexpr int ROWS = GATED ? 8 : 16;
    const int tiles = (p.N + ROWS - 1) / ROWS, G = p.K / 128, chunks = (G + CH - 1) / CH;
    const int total = count_units(p, COLS, tiles, ends, &bk);
    const int per_cta = (int)(blockDim.x >> 5) / wk, team = warp / wk, part = warp % wk;
    const int teams = per_cta * (int)gridDim.x, me = (int)blockIdx.x * per_cta + team;
    const int c0 = chunks * part / wk, c1 = chunks * (part + 1) / wk;
    int u = (int)((long long)total * me / teams);
    const int u1 = (int)((long long)total * (me + 1) / teams);
    if (u >= u1) return;                                              // (a team's barrier is its own)

    uint4 wa[CH], wb[CH], e[CH], o[CH];
    unsigned short sa[CH], sb[CH];
    float f0[CH], f1[CH];                                             // scales of columns 2 fq and 2 fq + 1
    const uint8_t *pa, *pb;
    const __half *qa, *qb;
    const int8_t *xe, *xo;                                            // codes of column fr (no such row: those of row 0)
    const float *x0, *x1;
    bool no0, no1;                                                    // no row of x for columns 2 fq and 2 fq + 1: their sums are 0
    auto start = [&](const Unit& n) {                                 // chunk c0 of a unit
        // (rows past the end repeat the last one and are not stored)
        const int n0 = n.tile * ROWS, ra = min(n0 + fr, p.N - 1), rb = GATED ? p.N + ra : min(n0 + 8 + fr, p.N - 1), g = c0 * CH;
        const size_t row0 = (size_t)n.expert * (GATED ? 2 * p.N : p.N);
        pa = p.wq + (row0 + ra) * (size_t)(p.K / 2) + g * 64 + fq * 16;
        pb = p.wq + (row0 + rb) * (size_t)(p.K / 2) + g * 64 + fq * 16;
        qa = p.ws + (row0 + ra) * (size_t)G + g;
        qb = p.ws + (row0 + rb) * (size_t)G + g;
        const size_t r = (size_t)max(x_row(p, n, fr), 0ll) * (p.K / 2) + g * 64 + fq * 16;
        xe = p.ae + r;
        xo = p.ao + r;
        const long long r0 = x_row(p, n, 2 * fq), r1 = x_row(p, n, 2 * fq + 1);
        no0 = r0 < 0;
        no1 = r1 < 0;
        x0 = p.asc + (size_t)max(r0, 0ll) * G + g;
        x1 = p.asc + (size_t)max(r1, 0ll) * G + g;
    };
    auto load = [&](int j, int last) {                                // group j of the chunk, whose last group is `last`
        const int at = WHOLE ? j : min(j, last);
        wa[j] = ld_stream_256(pa + at * 64);
        wb[j] = ld_stream_256(pb + at * 64);
        sa[j] = __half_as_ushort(qa[at]);
        sb[j] = __half_as_ushort(qb[at]);
        e[j] = *reinterpret_cast<const uint4*>(xe + at * 64);
        o[j] = *reinterpret_cast<const uint4*>(xo + at * 64);
        f0[j] = WHOLE || j <= last ? x0[at] : 0.f;
        f1[j] = WHOLE || j <= last ? x1[at] : 0.f;
    };
    Unit un = find_unit_of_chunk(p, u, COLS, tiles, ends);
    start(un);
#pragma unroll
    for (int j = 0; j < CH; j++) load(j, G - 1 - c0 * CH);
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    int buf = 0;
    while (true) {
        Unit nu = un;
        const bool zero0 = no0, zero1 = no1;                          // (of this unit; `start` goes on to the next)
        const bool more = u + 1 < u1;
        for (int c = c0; c < c1; c++) {
            const bool ends_unit = c + 1 == c1;
            if (!ends_unit) {
                pa += CH * 64;
                pb += CH * 64;
                qa += CH;
                qb += CH;
                xe += CH * 64;
                xo += CH * 64;
                x0 += CH;
                x1 += CH;
            } else if (more) {
                if (++nu.tile == tiles) nu = find_unit_of_chunk(p, u + 1, COLS, tiles, ends);        // (otherwise the same rows of x)
                start(nu);
            }
            const bool fetch = !ends_unit || more;
            const int last = G - 1 - (ends_unit ? c0 : c + 1) * CH;
#pragma unroll
            for (int j = 0; j < CH; j++) {
                int d[4];
                mma_s8_first(d, lo16(wa[j].x), lo16(wb[j].x), hi16(wa[j].x), hi16(wb[j].x), e[j].x, o[j].x);
                mma_s8(d, lo16(wa[j].y), lo16(wb[j].y), hi16(wa[j].y), hi16(wb[j].y), e[j].y, o[j].y);
                mma_s8(d, lo16(wa[j].z), lo16(wb[j].z), hi16(wa[j].z), hi16(wb[j].z), e[j].z, o[j].z);
                mma_s8(d, lo16(wa[j].w), lo16(wb[j].w), hi16(wa[j].w), hi16(wb[j].w), e[j].w, o[j].w);
                const float fa = __half2float(__ushort_as_half(sa[j])), fb = __half2float(__ushort_as_half(sb[j]));
                acc[0] = fmaf((float)d[0], fa * f0[j], acc[0]);
                acc[1] = fmaf((float)d[1], fa * f1[j], acc[1]);
                acc[2] = fmaf((float)d[2], fb * f0[j], acc[2]);
                acc[3] = fmaf((float)d[3], fb * f1[j], acc[3]);
                if (fetch) load(j, last);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) acc[i] *= 0.0625f;
        if (wk > 1) {                                                 // add the parts, in their order
#pragma unroll
            for (int i = 0; i < 4; i++) join[buf][warp][i][lane] = acc[i];
            asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(wk * 32) : "memory");          // (two buffers: one barrier a unit)
            if (part == 0)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    for (int k = 1; k < wk; k++) acc[i] += join[buf][warp + k][i][lane];
            buf ^= 1;
        }
        if (GATHER && zero0) acc[0] = acc[2] = 0.f;
        if (GATHER && zero1) acc[1] = acc[3] = 0.f;
        if (part == 0) {
            const int n0 = un.tile * ROWS;
            const float* bias = p.bias ? p.bias + (size_t)un.expert * (GATED ? 2 * p.N : p.N) : nullptr;
            const int na = n0 + fr, nb = GATED ? p.N + na : na + 8;   // the lane's two weight rows
            const bool has_a = na < p.N, has_b = GATED ? has_a : nb < p.N;
            const float ba = bias && has_a ? bias[na] : 0.f, bb = bias && has_b ? bias[nb] : 0.f;
            const long long m = (long long)un.first + fq * 2, end = (long long)un.first + un.count;
            float v[2] = {acc[0] + ba, acc[1] + ba}, w[2] = {acc[2] + bb, acc[3] + bb};
            if (m < end) {
                if (GATED) {
                    if (has_a) finish<2, true>(p, m, end, na, v, w);
                } else {
                    if (has_a) finish<2, false>(p, m, end, na, v, v);
                    if (has_b) finish<2, false>(p, m, end, nb, w, w);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) acc[i] = 0.f;
        if (!more) break;
        un = nu;
        u++;
    }
    pdl_launch_dependents();
}

int run_rows(const char* kn, const LaunchCtx& c, const Params& p) {
    const int rows = p.gated ? 8 : 16, tiles = (p.N + rows - 1) / rows, parts = (p.K / 128 + CH - 1) / CH;
    long long chunks = (p.m + COLS - 1) / COLS;
    if (p.offsets) chunks = p.n_exp < p.m ? chunks + p.n_exp : p.m;   // every bucket may end in a part of a chunk
    const long long units = chunks * tiles, slots = (long long)c.sm_count * kCtasPerSm * kMaxWarps;
    FM_REQUIRE(units < (1ll << 30), kn, "%lld tiles are too many for one call", units);
    // the K dimension is split over warps while all of them stay resident at once, each keeps a chunk and every team has one
    // unit at most (320 units of 5120 x 17408, 5 rows: 17.1 us with 7 warps a team, of which 24 of 296 had two units, 16.2 with 4)
    int wk = (int)(slots / units < kMaxWarps ? slots / units : kMaxWarps);
    while (wk > 1 && (long long)c.sm_count * kCtasPerSm * (kMaxWarps / wk) < units) wk--;
    if (wk > parts) wk = parts;
    if (wk < 1) wk = 1;
    const int per_cta = kMaxWarps / wk;
    long long grid = (units + per_cta - 1) / per_cta;
    if (grid > c.sm_count * kCtasPerSm) grid = c.sm_count * kCtasPerSm;
    const size_t smem = p.offsets ? (size_t)p.n_exp * 4 : 0;
    const bool whole = p.K % 512 == 0;
    auto kern = !p.bucket_rows ? (p.gated ? (whole ? rows_kernel<true, true, false> : rows_kernel<true, false, false>)
                                          : (whole ? rows_kernel<false, true, false> : rows_kernel<false, false, false>))
                               : (p.gated ? (whole ? rows_kernel<true, true, true> : rows_kernel<true, false, true>)
                                          : (whole ? rows_kernel<false, true, true> : rows_kernel<false, false, true>));
    const cudaError_t e = launch_kernel(kern, dim3((unsigned)grid), dim3(wk * per_cta * 32), smem, c.stream, pdl_enabled(), p, wk);
    return e == cudaSuccess ? after_launch(kn) : cuda_fail(kn, e);
}

// Rows or tiles, whichever promises to be done first.  The rows kernel passes over the weights of a bucket once for every 8 rows:
// counted at 5.7 MB a microsecond, measured 3.3 (5120 x 17408, whose few units leave warps idle: 32 to 56 rows all take 54 us) to
// 5.8 (the experts below).  A tile is counted at 0.35 us for a 128-group, one wave of tiles after the other, 2.5 us later than the
// rows kernel starts, measured 0.35 to 0.42.  (Buckets as if all experts were equally popular, half a piece added for the rest of
// each.)
// Measured, rows against tiles: 17408 x 5120 at 16 rows 19.0 and 22.3 us, at 17 rows 27.3 and 23.1; 5120 x 17408 at 32 rows 53.4
// and 53.3, at 40 53.8 and 59.4, at 48 53.8 and 59.2 (the last that goes to the rows kernel), at 56 54.0 and 59.5, at 64 73.8 and
// 59.5; 5120 x 5120 at 48 rows 20.5 and 20.8, at 64 25.4 and 22.6; 2048 x 2048 at 48 rows 8.2 and 12.4, at 128 12.3 and 14.5; 8 of
// 64 gated experts of 1024 x 5120 at 72 tokens 94 and 109, at 128 142 and 114.
bool rows_first(const LaunchCtx& c, const Params& p) {
    const long long used = !p.offsets ? 1 : p.n_exp < p.m ? p.n_exp : p.m, rows = p.gated ? 64 : 128;
    auto pieces = [&](int of) {
        if (!p.offsets) return (p.m + of - 1ll) / of;
        const long long n = p.m / of + used / 2;
        return n < used ? used : n;
    };
    const double bytes = (double)pieces(COLS) * p.N * (p.gated ? p.K : p.K / 2);
    const long long tiles = pieces(128) * ((p.N + rows - 1) / rows), steps = (tiles + c.sm_count - 1) / c.sm_count * (p.K / 128);
    return bytes <= 2e6 * (7 + steps);
}

int run(const char* kn, const LaunchCtx& c, const Params& p) { return rows_first(c, p) ? run_rows(kn, c, p) : run_tiles(kn, c, p); }

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
