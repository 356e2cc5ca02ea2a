// The W4A8 product with an epilogue on the fifth-generation tensor cores, for buckets of many rows (the entries and the
// arithmetic are those of linear_w4a8.cu).
//
// D^T[weight row][row of x] = W . x^T: 128 weight rows (gated: 64 gate rows and the 64 up rows beside them) are the 128
// lanes of an accumulator, up to 128 rows of a bucket its columns, so that a short bucket costs a narrow MMA and not a
// padded tile.  tcgen05.mma.kind::i8 forms the exact integer of a 128-group; the weights enter as 16 w, a nibble in the
// upper half of its byte, which takes two logic instructions for eight of them, and the 16 is divided out of their scale.
// (kind::f16, whose fp32 accumulators need no conversion, took 526 us where this took 480 for 2048 x 17408 x 5120: its
// expansion takes nine instructions for eight weights, its rows of x twice the bytes, and its A operand leaves tensor memory
// for two accumulators instead of three.)
//
// Roles of the 16 warps of the persistent CTA, joined by mbarriers (every wait is bounded):
//   * one warp copies packed weight tiles (128 rows x 64 bytes, two TMA boxes) into a ring;
//   * four warps expand them: a thread owns a weight row, reads its 64 bytes and writes 128 to tensor memory, from where
//     the MMA takes its A operand; it also fetches the scale of its row and of one row of x, some steps ahead;
//   * one warp copies the rows of x by TMA, put into bucket order by a small kernel in front, or their even and odd codes from
//     where they are;
//   * two warps issue the MMAs of the even and the odd groups, into three accumulators in turn;
//   * eight warps, four for the even and four for the odd groups, drain the accumulators: C[m, n] = fmaf(float(I), ws * asc,
//     C) in registers, then the epilogue.
//
// Measured (B200): 2048 x 17408 x 5120 with bias and gelu 361 to 368 us, 1.0 POP/s; the experts' gate and up projections of 1999
// tokens, 8 of 64 experts of 1024 x 5120, 426 to 434 us; 77 gated rows of 6144 x 5120 24.6 us.  What bounds it is the epilogue: a
// step of 128 x 128 sums takes its two sets 2000 clocks each (1000 a step; the MMAs 256), of which 1300 load, convert, scale and
// add and the rest waits for barriers that are there and starts the next step; a tile ends with 5000 clocks in which nothing is
// multiplied.  Measured and dropped: 16 columns loaded ahead of the 16 in work (396 us against 361), 8 ahead of 8 (486 against
// 443 then), conversion by adding 1.5 * 2^23 for all sums (477 against 443) or half of them (402 against 379), sets that share the
// columns instead of the steps (575 against 443).  Few rows are bound by the expansion, 700 clocks a step for its chain of waits;
// the next step's weights loaded ahead did not shorten it (27.9 us against 26.3 then).
#include <cuda.h>

#include "device_utils.cuh"
#include "fm_internal.h"
#include "linear_w4a8.cuh"
#include "tc_utils.cuh"

namespace fm {
namespace linear {
namespace {
using namespace tc;

constexpr int kCols = 128;                          // rows of x per tile
constexpr int RING = 4;                             // stages of A (tensor memory), B (shared memory) and "step done" barriers
constexpr int NACC = 3;                             // accumulators
constexpr int BP = 8;                               // stages of packed weights
constexpr int SLOTS = 16;                           // stages of scales (reuse distance: see where they are fetched)
constexpr int kAhead = 6;                           // steps between issuing a fetch of scales and their use
constexpr int B_BYTES = kCols * 128, BP_BYTES = 128 * 64;
constexpr int WEIGHT_WARP = 0, MMA_WARP = 1, ROW_WARP = 3, EXP_WARP0 = 4, EPI_WARP0 = 8, kThreads = 16 * 32;
// 512 threads start with 128 registers each; the shares below add up to no more
constexpr int kRegsIssue = 72, kRegsExpand = 72, kRegsEpilogue = 184;
static_assert(kRegsIssue + kRegsExpand + 2 * kRegsEpilogue <= 512, "register shares of the four warpgroups");
static_assert(SLOTS > kAhead + RING + NACC + 1, "see where the scales are fetched");
constexpr int kOutPitch = 68;                       // values between weight rows of the sums on their way out (16-byte words, no two of eight rows in a bank)
constexpr int kSpin = 1 << 17;
constexpr uint32_t kTmemCols = 512, kTmemA = NACC * kCols;   // accumulators, then A: 4 x 32 columns
static_assert(NACC * kCols + RING * 32 <= 512, "tensor memory");

struct __align__(16) Control {
    uint64_t bp_full[BP], bp_free[BP];
    uint64_t a_full[RING], b_full[RING], done[RING];
    uint64_t acc_full[2 * NACC], acc_free[2 * NACC], drain[2];
    uint32_t tmem_base;
    volatile int abort;
};

// 0, or the code of the first bounded wait that ran out: 21 packed stage not free, 22 accumulator not drained, 23 weights not
// expanded, 24 rows of x not landed, 25 and 27 step not done (copy, expansion), 26 packed weights not landed, 28 accumulator
// not complete.  Read and cleared by fm_gemm_status().
__device__ int g_status;

__device__ __forceinline__ bool wait(uint32_t b, uint32_t parity, Control* ctl, int code) {
    for (int i = 0; i < kSpin; i++) {
        if (mbar_try_wait_at(b, parity)) return true;
        if ((i & 63) == 63 && ctl->abort) return false;
    }
    ctl->abort = 1;
    atomicCAS(&g_status, 0, code);
    return false;
}
// the same by all lanes of a warp, which leave it with one answer (their next instructions are warp-wide)
__device__ __forceinline__ bool wait_warp(uint32_t b, uint32_t parity, Control* ctl, int code) {
    if (__all_sync(0xffffffffu, mbar_try_wait_at(b, parity))) return true;
    return __all_sync(0xffffffffu, wait(b, parity, ctl, code));
}

// two barriers in the time of one when both are ready
__device__ __forceinline__ bool wait_warp2(uint32_t b0, uint32_t parity0, int code0, uint32_t b1, uint32_t parity1, int code1, Control* ctl) {
    const bool r0 = mbar_try_wait_at(b0, parity0), r1 = mbar_try_wait_at(b1, parity1);
    if (__all_sync(0xffffffffu, r0 && r1)) return true;
    return wait_warp(b0, parity0, ctl, code0) && wait_warp(b1, parity1, ctl, code1);
}

// kind::i8: s32 accumulator, s8 operands, both K-major, M = 128
__device__ __forceinline__ uint32_t instr_desc(int n) { return 2u << 4 | 1u << 7 | 1u << 10 | (uint32_t)(n >> 3) << 17 | (uint32_t)(128 >> 4) << 24; }

// Eight two's-complement nibbles of a word -> 16 times their value as bytes, the even k of a group before the odd ones, as the
// codes of x are stored.
__device__ __forceinline__ void expand_word(uint32_t w, uint32_t* o) {
    o[0] = (w << 4) & 0xF0F0F0F0u;
    o[16] = w & 0xF0F0F0F0u;
}

// Rows of x into bucket order, [m][K] with the even codes of a group before its odd ones, and their scales, [K/128][m]; slot s
// of a plan takes row bucket_rows[s], and scale 0 if there is no such row.  A thread moves 32 k of a row, one in four of them
// the scale of the group too; slots behind the last bucket are skipped.  (The tiles are launched meanwhile, as far as their first
// wait.)
__global__ void __launch_bounds__(256)
order_codes_kernel(const Params p, int8_t* __restrict__ out, float* __restrict__ scales) {
    pdl_wait();
    pdl_launch_dependents();
    const unsigned per_row = p.K / 32, G = p.K / 128;
    const long long n = (long long)(p.offsets ? bound(p, p.n_exp) : p.m) * per_row;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) {
        const long long slot = n < (1ll << 32) ? (unsigned)i / per_row : i / per_row;
        const unsigned c = (unsigned)(i - slot * per_row);
        const long long row = p.bucket_rows ? p.bucket_rows[slot] : slot;
        const bool is = !p.bucket_rows || (row >= 0 && row < p.xrows);
        if (c % 4 == 0) scales[(size_t)(c / 4) * p.m + slot] = is ? p.asc[row * G + c / 4] : 0.f;
        if (!is) continue;
        int8_t* dst = out + slot * p.K + c / 4 * 128 + c % 4 * 16;
        *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(p.ae + row * (p.K / 2) + c * 16);
        *reinterpret_cast<uint4*>(dst + 64) = *reinterpret_cast<const uint4*>(p.ao + row * (p.K / 2) + c * 16);
    }
}

__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool take) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(take ? 4 : 0) : "memory");
}
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// weight row of lane `row` of a tile (a row past the end repeats the last one and is not stored)
template <bool GATED>
__device__ __forceinline__ size_t weight_row(const Params& p, const Unit& u, int row) {
    if (!GATED) return (size_t)u.expert * p.N + min(u.tile * 128 + row, p.N - 1);
    return (size_t)u.expert * 2 * p.N + (row < 64 ? 0 : p.N) + min(u.tile * 64 + (row & 63), p.N - 1);
}

// A wait names a phase by its parity, so a waiter must see every phase of its barrier: one phase late or early, the parity is
// the same and the wait passes at once.  The copy and expansion roles wait for the step that frees the stage they are about to
// fill, step by step.  The issuers and the sets of the epilogue take every other step: of the stages, an even number, each has
// its own; the three accumulators change hands, so each has two pairs of barriers, for the even and the odd steps: step it
// fills acc_full[it % 6], is drained by acc_free[it % 6] and takes over from step it - 3.
//
// Position in a ring of N stages and the parity of its phase there.  A wait for the other parity passes at once in the first
// round: the phase before a barrier's first counts as complete.
template <int N>
struct Ring {
    uint32_t s = 0, ph = 0;
    __device__ __forceinline__ void next() {
        s = s + 1 == N ? 0 : s + 1;
        ph ^= s == 0 ? 1u : 0u;
    }
    __device__ __forceinline__ void next2() {                         // two steps on
        s = s + 2 >= N ? s + 2 - N : s + 2;
        ph ^= s < 2 ? 1u : 0u;
    }
};

// boxes of 128, 64, 32 and 16 rows of x: a group's codes put in order, or (direct) its even and its odd ones from where they are
struct RowMaps { CUtensorMap box[4], odd[4]; };
struct Scales { const float* at; long long row, group; };            // of slot s and group g: at[s * row + g * group]

// GATED: 64 gate rows and 64 up rows make a tile.
template <bool GATED>
__global__ void __launch_bounds__(kThreads, 1)
tile_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ RowMaps map_x, const Scales scales, const bool direct, const Params p) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t* bring = smem;                                           // RING x [128 rows][128 bytes], or even and odd codes [128 rows][64 bytes]
    uint8_t* wring = bring + RING * B_BYTES;                         // BP x [128 rows][64 bytes]
    float* sring = reinterpret_cast<float*>(wring + BP * BP_BYTES);  // SLOTS x [128]
    uint32_t* wsring = reinterpret_cast<uint32_t*>(sring + SLOTS * kCols);   // SLOTS x [128]: the word that holds the weight row's scale
    float* xch = reinterpret_cast<float*>(wsring + SLOTS * 128);     // a set's [128 rows][64 columns] of sums on their way out, twice
    Control* ctl = reinterpret_cast<Control*>(xch + 2 * 128 * kOutPitch);
    int* ends = reinterpret_cast<int*>(ctl + 1);                     // [n_exp]
    __shared__ Buckets bk;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int ROWS = GATED ? 64 : 128;
    const int G = p.K / 128, tiles = (p.N + ROWS - 1) / ROWS;

    if (threadIdx.x == 0) {
        for (int i = 0; i < BP; i++) {
            mbar_init(&ctl->bp_full[i], 1);
            mbar_init(&ctl->bp_free[i], 4);
        }
        for (int i = 0; i < RING; i++) {
            mbar_init(&ctl->a_full[i], 4);
            mbar_init(&ctl->b_full[i], 1);
            mbar_init(&ctl->done[i], 1);
        }
        for (int i = 0; i < 2 * NACC; i++) {
            mbar_init(&ctl->acc_full[i], 1);
            mbar_init(&ctl->acc_free[i], 4);
        }
        for (int i = 0; i < 2; i++) mbar_init(&ctl->drain[i], 1);
        ctl->abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == MMA_WARP) tmem_alloc(&ctl->tmem_base, kTmemCols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ctl->tmem_base;
    pdl_wait();
    const int total = count_units(p, kCols, tiles, ends, &bk);

    const uint32_t bring_s = smem_u32(bring), wring_s = smem_u32(wring), sring_s = smem_u32(sring), wsring_s = smem_u32(wsring);
    const uint32_t bp_full = smem_u32(ctl->bp_full), bp_free = smem_u32(ctl->bp_free), a_full = smem_u32(ctl->a_full), b_full = smem_u32(ctl->b_full);
    const uint32_t done = smem_u32(ctl->done), acc_full = smem_u32(ctl->acc_full), acc_free = smem_u32(ctl->acc_free);
    if (warp < EXP_WARP0) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsIssue));
        // In these roles the whole warp walks the steps and one lane is elected to issue: a single lane that waits alone polls
        // its barrier dozens of times a step, and descriptors stay in uniform registers.
        if (warp == WEIGHT_WARP) {
            // ================================================================ packed weights
            Ring<BP> r;
            int it = 0;
            bool ok = true;
            for (int u = blockIdx.x; u < total && ok; u += gridDim.x) {
                const Unit un = find_unit(p, u, kCols, tiles, ends);
                const int y0 = un.expert * (GATED ? 2 * p.N : p.N) + un.tile * ROWS, y1 = y0 + (GATED ? p.N : 64);
                for (int g = 0; g < G; g++, it++, r.next()) {
                    if (!(ok = wait_warp(bp_free + r.s * 8, r.ph ^ 1, ctl, 21))) break;
                    if (elect_one()) {
                        const uint32_t bar = bp_full + r.s * 8, dst = wring_s + r.s * BP_BYTES;
                        mbar_expect_tx_at(bar, BP_BYTES);
                        tma_2d_at(dst, &map_w, g * 64, y0, bar);
                        tma_2d_at(dst + BP_BYTES / 2, &map_w, g * 64, y1, bar);
                    }
                    __syncwarp();
                }
            }
            if (ctl->abort)                                          // copies in flight land before the memory is given up
                for (int j = it > BP ? it - BP : 0; j < it; j++)
                    for (int i = 0; i < kSpin && !mbar_try_wait(&ctl->bp_full[j % BP], (j / BP) & 1); i++) {}
        } else if (warp == ROW_WARP) {
            // ================================================================ rows of x
            // A count of rows is a sum of boxes of 128, 64, 32 and 16: a box costs its issue, about 100 clocks, whatever it holds
            // (16-row boxes throughout, 16 instructions a step, bound the tile at 1800 clocks; four-row gathers at 6000).
            const int width = direct ? 64 : 128;
            Ring<RING> r;
            int it = 0;
            bool ok = true;
            for (int u = blockIdx.x; u < total && ok; u += gridDim.x) {
                const Unit un = find_unit(p, u, kCols, tiles, ends);
                const int n16 = (un.count + 15) & ~15;
                for (int g = 0; g < G; g++, it++, r.next()) {
                    if (!(ok = wait_warp(done + r.s * 8, r.ph ^ 1, ctl, 25))) break;
                    if (elect_one()) {
                        const uint32_t bar = b_full + r.s * 8;
                        mbar_expect_tx_at(bar, (uint32_t)n16 * 128);
                        uint32_t dst = bring_s + r.s * B_BYTES;
                        int at = un.first;
#pragma unroll
                        for (int b = 0; b < 4; b++)
                            if (n16 & (128 >> b)) {
                                tma_2d_at(dst, &map_x.box[b], g * width, at, bar);
                                if (direct) tma_2d_at(dst + B_BYTES / 2, &map_x.odd[b], g * width, at, bar);
                                at += 128 >> b;
                                dst += (128 >> b) * width;
                            }
                    }
                    __syncwarp();
                }
            }
            if (ctl->abort)
                for (int j = it > RING ? it - RING : 0; j < it; j++)
                    for (int i = 0; i < kSpin && !mbar_try_wait(&ctl->b_full[j % RING], (j / RING) & 1); i++) {}
        } else {
            // ================================================================ MMA issuers: even and odd steps
            const uint32_t par = warp - MMA_WARP;
            const uint64_t bdesc0 = direct ? smem_desc_sw64(bring_s) : smem_desc_sw128(bring_s);
            const uint32_t odd = direct ? B_BYTES / 2 >> 4 : 64 >> 4;
            Ring<RING> r;
            Ring<2 * NACC> acc;
            uint32_t parity = 0;                                     // of the first step of the tile
            if (par) {
                r.next();
                acc.next();
            }
            bool ok = true;
            for (int u = blockIdx.x; u < total && ok; u += gridDim.x) {
                const Unit un = find_unit(p, u, kCols, tiles, ends);
                const uint32_t idesc = instr_desc((un.count + 15) & ~15);
                for (int g = par ^ parity; g < G; g += 2, r.next2(), acc.next2()) {
                    if (!(ok = wait_warp2(a_full + r.s * 8, r.ph, 23, b_full + r.s * 8, r.ph, 24, ctl))) break;
                    const uint32_t late = acc.s >= NACC, d_at = late ? acc.s - NACC : acc.s;
                    if (!(ok = wait_warp(acc_free + (late ? d_at : d_at + NACC) * 8, acc.ph ^ 1 ^ late, ctl, 22))) break;
                    tc_fence_after();
                    const uint64_t bd = bdesc0 + (uint64_t)(r.s * (B_BYTES >> 4));
                    const uint32_t d = tmem + d_at * kCols, a = tmem + kTmemA + r.s * 32;
                    if (elect_one()) {
#pragma unroll
                        for (int j = 0; j < 4; j++)                  // 32 k each: 8 columns of A, 32 bytes of B
                            tc_mma_i8_ts(d, a + j * 8, bd + (j >> 1) * odd + (j & 1) * 2, idesc, j > 0);
                        tc_commit_at(acc_full + acc.s * 8);
                        tc_commit_at(done + r.s * 8);
                    }
                    __syncwarp();
                }
                parity ^= G & 1;
            }
            // nothing this warp issued may still run when tensor memory is released (the lane that issued commits: elect.sync
            // names the same lane of a full warp every time)
            if (elect_one()) tc_commit(&ctl->drain[par]);
            for (int i = 0; i < kSpin && !mbar_try_wait(&ctl->drain[par], 0); i++) {}
        }
    } else if (warp < EPI_WARP0) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsExpand));
        // ==================================================================== expansion of the weights
        const uint32_t q = warp & 3, row = q * 32 + lane;
        const uint32_t a0 = tmem + ((uint32_t)(q * 32) << 16) + kTmemA;
        const uint32_t x = ((row >> 1) & 3) << 4;                    // 64-byte swizzle: chunk ^= (row / 2) % 4
        const uint32_t w0 = wring_s + row * 64 + x, w1 = wring_s + row * 64 + (16 ^ x), w2 = wring_s + row * 64 + (32 ^ x), w3 = wring_s + row * 64 + (48 ^ x);
        // A lane fetches the scale of the row of x that is its column and the aligned word around the scale of its weight row,
        // kAhead steps before the expansion that publishes them.  (A copy has at least four bytes, two groups; a lane copies
        // each word once, into the slot of the step that first needs it.  Allocations are whole words.)  With two steps, less
        // than the memory's latency, the MMAs waited; one warp that fetched for all took 700 clocks a step.
        // This warp has seen the MMAs up to step it - 1 - RING done, which were issued after the accumulators up to step
        // it - 1 - RING - NACC had been drained, so nobody reads the slot of step it + kAhead - SLOTS or the one before any more.
        int fu = blockIdx.x, fg = 0;                                 // next to fetch
        const float* sc = nullptr;
        uintptr_t wsc = 0;
        bool has = false;
        Ring<SLOTS> slot;
        auto fetch = [&]() {
            if (fu < total) {
                if (fg == 0) {
                    const Unit un = find_unit(p, fu, kCols, tiles, ends);
                    has = (int)row < un.count;
                    sc = scales.at + (un.first + (has ? (long long)row : 0)) * scales.row;
                    wsc = reinterpret_cast<uintptr_t>(p.ws + weight_row<GATED>(p, un, row) * G);
                }
                const uint32_t at = (slot.s * 128 + row) * 4;
                cp_async4(sring_s + at, sc, has);
                if (fg == 0 || !(wsc & 2)) cp_async4(wsring_s + at, reinterpret_cast<const void*>(wsc & ~(uintptr_t)3), true);
                sc += scales.group;
                wsc += 2;
                slot.next();
                if (++fg == G) {
                    fg = 0;
                    fu += gridDim.x;
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        for (int i = 0; i < kAhead; i++) fetch();
        Ring<BP> rp;
        Ring<RING> r;
        bool ok = true;
        for (int u = blockIdx.x; u < total && ok; u += gridDim.x) {
            for (int g = 0; g < G; g++, rp.next(), r.next()) {
                if (!(ok = wait_warp2(bp_full + rp.s * 8, rp.ph, 26, done + r.s * 8, r.ph ^ 1, 27, ctl))) break;
                const uint32_t at = rp.s * BP_BYTES;
                const uint4 w[4] = {lds128(w0 + at), lds128(w1 + at), lds128(w2 + at), lds128(w3 + at)};
                tc_fence_after();
                uint32_t o[32];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    expand_word(w[j].x, o + 4 * j);
                    expand_word(w[j].y, o + 4 * j + 1);
                    expand_word(w[j].z, o + 4 * j + 2);
                    expand_word(w[j].w, o + 4 * j + 3);
                }
                tmem_st32(a0 + r.s * 32, o);
                fetch();
                cp_async_wait<kAhead>();
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();                                        // (every lane has its words in registers, and A is written)
                if (lane == 0) {
                    mbar_arrive_at(bp_free + rp.s * 8);
                    mbar_arrive_at(a_full + r.s * 8);
                }
            }
        }
        cp_async_wait<0>();
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsEpilogue));
        // ==================================================================== epilogue
        // Two sets of four warps, one for the even and one for the odd steps, so that a set has two step times for its chain of
        // waits, loads and sums; a tile's two partial sums meet on their way out.  warp: lanes 32 q .. of the accumulators
        const uint32_t set = (warp - EPI_WARP0) >> 2, q = warp & 3, row = q * 32 + lane;
        const uint32_t d0 = tmem + ((uint32_t)(q * 32) << 16), sw0 = wsring_s + row * 4;
        float *const mine = xch + set * (128 * kOutPitch), *const theirs = xch + (set ^ 1) * (128 * kOutPitch);
        Ring<SLOTS> r;
        Ring<2 * NACC> acc;
        uint32_t parity = 0;                                         // of the first step of the tile
        if (set) {
            r.next();
            acc.next();
        }
        for (int u = blockIdx.x; u < total; u += gridDim.x) {
            const Unit un = find_unit(p, u, kCols, tiles, ends);
            const int n0 = un.tile * ROWS, chunks = (un.count + 15) >> 4;
            // which half of its word the scale of a group is: by the group's parity, one for the set's groups of a tile
            const uint32_t shift = ((uint32_t)(reinterpret_cast<uintptr_t>(p.ws + weight_row<GATED>(p, un, row) * G) >> 1) ^ set ^ parity) << 4 & 16;
            const float bias = p.bias ? p.bias[weight_row<GATED>(p, un, row)] : 0.f;
            bool ok = true;
            uint64_t C[8][8];                                        // pairs of neighbouring columns
#pragma unroll
            for (int a = 0; a < 8; a++)
#pragma unroll
                for (int j = 0; j < 8; j++) C[a][j] = 0;
            for (int g = set ^ parity; g < G; g += 2, r.next2(), acc.next2()) {
                if (!(ok = wait_warp(acc_full + acc.s * 8, acc.ph, ctl, 28))) break;
                tc_fence_after();
                const uint32_t slot = r.s * 512, sb = sring_s + slot, d = d0 + (acc.s >= NACC ? acc.s - NACC : acc.s) * kCols;
                const uint32_t s = __float_as_uint(__half2float(__ushort_as_half((unsigned short)(lds32(sw0 + (g && shift ? (r.s - 1) % SLOTS * 512 : slot)) >> shift))) * 0.0625f);
                const uint64_t s2 = pack2(s, s);
#pragma unroll
                for (int a = 0; a < 8; a++) {
                    if (a >= chunks) break;
                    uint64_t f[8];
                    uint32_t v[16];
#pragma unroll
                    for (int j = 0; j < 8; j += 2) {
                        const uint4 b = lds128(sb + a * 64 + j * 8);
                        f[j] = mul2p(s2, pack2(b.x, b.y));
                        f[j + 1] = mul2p(s2, pack2(b.z, b.w));
                    }
                    tmem_ld16_now(d + a * 16, v);
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        fma2p(C[a][j], pack2(__float_as_uint((float)(int)v[2 * j]), __float_as_uint((float)(int)v[2 * j + 1])), f[j]);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_at(acc_free + acc.s * 8);
            }
            parity ^= G & 1;
            // The sets swap half of their partial sums through shared memory, set k keeping the 16-column pieces a with a % 2 ==
            // k, and put the sums of those there as well, so that the loop with the activation is rolled and there once: code that
            // runs once a tile is fetched once a tile.  (Unrolled over the registers it was 60 KB, and fetching that took 1.7
            // times as long as the tile's products; four loops of 32 columns took 15000 clocks of 57000.)  A warp that gave up a
            // wait takes part in the barriers all the same; the last one of the tile tells all.
            const int t = threadIdx.x & 127;
            const long long end = (long long)un.first + un.count;
            auto first_of = [&](int i) { return (long long)un.first + ((i & 48) * 2 + set * 16 + (i & 15)); };      // row of sum i
#pragma unroll
            for (int a = 0; a < 8; a += 2) {                         // (by static index: C stays in registers)
                if (a >= chunks) break;
#pragma unroll
                for (int j = 0; j < 8; j += 2)
                    *reinterpret_cast<ulonglong2*>(theirs + row * kOutPitch + a * 8 + 2 * j) = make_ulonglong2(set ? C[a][j] : C[a + 1][j], set ? C[a][j + 1] : C[a + 1][j + 1]);
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");
            const uint64_t bias2 = pack2(__float_as_uint(bias), __float_as_uint(bias));
#pragma unroll
            for (int a = 0; a < 8; a += 2) {
                if (a >= chunks) break;
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    ulonglong2* at = reinterpret_cast<ulonglong2*>(mine + row * kOutPitch + a * 8 + 2 * j);
                    const ulonglong2 o = *at;
                    *at = make_ulonglong2(add2p(o.x, add2p(set ? C[a + 1][j] : C[a][j], bias2)), add2p(o.y, add2p(set ? C[a + 1][j + 1] : C[a][j + 1], bias2)));
                }
            }
            if (GATED) asm volatile("bar.sync %0, 128;" ::"r"(2 + set) : "memory");          // gate lane gr meets up lane 64 + gr
            const int n = n0 + (GATED ? t & 63 : (int)row);
            if (n < p.N) {
                float* sums = mine + (n - n0) * kOutPitch;
                const bool keep = p.residual != nullptr;             // (for the loop below)
#pragma unroll 1
                for (int i = GATED ? t >> 6 << 4 : 0; i < 64 && (GATED || !keep || p.act); i += GATED ? 32 : 16) {
                    const long long m = first_of(i);
                    if (m >= end) break;
                    float v[16];
#pragma unroll
                    for (int k = 0; k < 16; k++) v[k] = sums[i + k];
                    activate_n(p.act, v);
                    if (GATED) {
#pragma unroll
                        for (int k = 0; k < 16; k++) v[k] *= sums[64 * kOutPitch + i + k];
                    }
                    if (keep) {
#pragma unroll
                        for (int k = 0; k < 16; k++) sums[i + k] = v[k];
                    } else {
                        const int left = (int)(end - m);
                        float* y = p.y + m * p.ldy + n;
                        if (left >= 16) {
#pragma unroll
                            for (int k = 0; k < 16; k++) y[k * p.ldy] = v[k];
                        } else {
#pragma unroll
                            for (int k = 0; k < 15; k++)
                                if (k < left) y[k * p.ldy] = v[k];
                        }
                    }
                }
                // the residual in a loop of its own, 16 loads on their way: one latency for every four rows was twice the products'
                // time at 1228 x 10187 x 1536.  An element is the residual of itself only, read by the thread that writes it.
                if (keep) {
#pragma unroll 1
                    for (int i = GATED ? t >> 6 << 4 : 0; i < 64; i += GATED ? 32 : 16) {
                        const long long m = first_of(i);
                        const int left = (int)(end - m);
                        if (left <= 0) break;
                        const float* r = p.residual + m * p.ldr + n;
                        float* y = p.y + m * p.ldy + n;
                        float add[16];
#pragma unroll
                        for (int j = 0; j < 16; j++) add[j] = j < left ? r[j * p.ldr] : 0.f;
#pragma unroll
                        for (int j = 0; j < 16; j++)
                            if (j < left) y[j * p.ldy] = sums[i + j] + add[j];
                    }
                }
            }
            int all;
            asm volatile("{\n.reg .pred p, q;\nsetp.ne.s32 p, %1, 0;\nbar.red.and.pred q, 1, 256, p;\nselp.s32 %0, 1, 0, q;\n}" : "=r"(all) : "r"((int)ok) : "memory");
            if (!all) break;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == MMA_WARP) tmem_dealloc(tmem, kTmemCols);
    pdl_launch_dependents();
}

size_t smem_bytes(const Params& p) {
    return 1024 + RING * B_BYTES + BP * BP_BYTES + SLOTS * (kCols + 128) * 4 + 2 * 128 * kOutPitch * 4 + sizeof(Control) + (size_t)p.n_exp * 4;
}

}  // namespace

int run_tiles(const char* kn, const LaunchCtx& c, const Params& p) {
    const int per_tile = p.gated ? 64 : 128;
    long long chunks = (p.m + kCols - 1) / kCols;
    if (p.offsets) chunks = chunks + p.n_exp < p.m ? chunks + p.n_exp : p.m;
    const long long units = chunks * ((p.N + per_tile - 1) / per_tile);
    FM_REQUIRE(units < (1ll << 30), kn, "%lld tiles are too many for one call", units);
    // Rows that stay where they are can be read from there, half a group a box and every scale from a line of its own, which
    // costs a step some 2 %; the kernel that orders them costs 2 to 3 us.  (77 rows, 40 steps: 24.6 us and 26.5; 2048 rows, 600
    // steps: 373 and 363.)
    const bool direct = !p.bucket_rows && (units + c.sm_count - 1) / c.sm_count * (p.K / 128) <= 200;
    const long long rows = direct && p.offsets ? p.xrows : p.m;
    const int8_t* x = p.ae;
    Scales scales = {p.asc, p.K / 128, 1};
    cudaError_t e;
    if (!direct) {
        const size_t codes = (size_t)p.m * p.K, bytes = codes + (size_t)p.m * (p.K / 128) * 4;
        int8_t* ordered = static_cast<int8_t*>(engine_scratch(bytes));
        FM_REQUIRE(ordered, kn, "the engine workspace cannot grow to %zu bytes here (inside a capture: raise FM_SCRATCH_MB)", bytes);
        float* by_group = reinterpret_cast<float*>(ordered + codes);
        size_t blocks = ((size_t)p.m * (p.K / 32) + 255) / 256;
        if (blocks > (size_t)c.sm_count * 16) blocks = (size_t)c.sm_count * 16;
        e = launch_kernel(order_codes_kernel, dim3((unsigned)blocks), dim3(256), 0, c.stream, pdl_enabled(), p, ordered, by_group);
        if (e != cudaSuccess) return cuda_fail(kn, e);
        const int rc = after_launch(kn);
        if (rc != FM_OK) return rc;
        x = ordered;
        scales = {by_group, 1, p.m};
    }
    CUtensorMap map_w;
    RowMaps map_x = {};
    const uint64_t wrows = (uint64_t)p.n_exp * p.N * (p.gated ? 2 : 1), width = direct ? p.K / 2 : p.K;
    bool ok = wrows < 0x7fffffff && encode_bytes_box_map(&map_w, p.wq, wrows, (uint64_t)p.K / 2, 64, 64);
    for (int b = 0; b < 4; b++) {
        ok = ok && encode_bytes_box_map(&map_x.box[b], x, (uint64_t)rows, width, direct ? 64 : 128, 128 >> b);
        if (direct) ok = ok && encode_bytes_box_map(&map_x.odd[b], p.ao, (uint64_t)rows, width, 64, 128 >> b);
    }
    FM_REQUIRE(ok, kn, "the tensor maps of %llu rows of weights and %lld rows of x were refused (K=%d)", (unsigned long long)wrows, rows, p.K);
    auto kern = p.gated ? tile_kernel<true> : tile_kernel<false>;
    const size_t smem = smem_bytes(p);
    if ((e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem)) != cudaSuccess) return cuda_fail(kn, e);
    const unsigned grid = (unsigned)(units < c.sm_count ? units : c.sm_count);
    e = launch_kernel(kern, dim3(grid), dim3(kThreads), smem, c.stream, !direct || pdl_enabled(), map_w, map_x, scales, direct, p);
    return e == cudaSuccess ? after_launch(kn) : cuda_fail(kn, e);
}

}  // namespace linear

int linear_read_status() {
    int v = 0;
    const int zero = 0;
    if (cudaMemcpyFromSymbol(&v, linear::g_status, sizeof(int)) != cudaSuccess) return -1;
    if (v) cudaMemcpyToSymbol(linear::g_status, &zero, sizeof(int));
    return v;
}

}  // namespace fm
