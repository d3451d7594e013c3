// gated_ff_tc.cu - the products of the gated feed-forward block on 16-bit tensors:
// tcgen05 CTA pairs, operands read as they lie in memory.
//
// Every product of the block (gated_ff.cuh) is D[M x N] = A B with A's rows and
// B's columns contiguous along the sum (k-major: x, h, dg, du, dy; Wd^T, Wg^T, Wu^T
// in the backward pass) or across it (mn-major: the weights in the forward pass;
// x^T, h^T, dg, du, dy under the weights' gradients).  16-bit MMAs take both from
// shared memory, so nothing is transposed or packed first.
//
// Two CTAs of a cluster (tcgen05 cta_group::2) compute a 256 x 256 tile; CTA r
// holds rows [128 r, 128 r + 128) of A and of D, and half of B's columns.  Stages
// hold 64 of the sum: 16 KB of A and of B per CTA, each as two boxes of 64 rows
// (k-major: 64 rows of 64 of the sum; mn-major: 64 of the sum for 64 rows), 8 KB
// with 128-byte swizzle:
//   k-major   8-row groups 1024 bytes apart; an MMA's 16 of the sum are 32 bytes
//             along the rows
//   mn-major  8-groups of the sum 1024 bytes apart, the second 64 rows 8192; an
//             MMA's 16 of the sum are 2048 bytes further
// For the gated pair of products CTA 0 loads 128 columns of Wg and CTA 1 the same
// columns of Wu: one accumulator holds 128 columns of g beside 128 of u, the
// epilogue threads find both for their row, and neither goes through memory.
// dh's epilogue reads g and u and writes dg, du and h; dh itself stays in TMEM.
// dx sums two products in one accumulator; it and the three weights' gradients share
// one launch.
//
// Roles as in the f32 kernels (sgemm_tc.cu): warp 0 TMA, warp 1 MMA (CTA 0 of the
// pair issues), warps 2-9 epilogue.  The f32 accumulator stays in TMEM for up to kFfRun
// of the sum: its additions truncate, which takes 1.1e-4 from a sum of that many terms of
// one sign (gated_ff.cuh).  A longer sum comes in runs, which the epilogue warps add up,
// rounding to nearest, while the MMAs fill the other accumulator (LONG: 128 values a
// lane, in local memory; a run takes 70 us and more, its drain a few).  Two
// accumulators: a tile's epilogue overlaps the next tile's MMAs.  When the last wave would keep
// at most half of the pairs busy its tiles run as two column halves.  Products of
// few tiles and a long sum are split along it into f32 parts, which a second kernel
// adds up in order.  Each kernel is launched while the one before it drains
// (programmatic dependent launch) and waits for it before it touches memory.
//
// Bound by the tensor cores, and at length by the 1000 W cap: 4096 rows of 4096 -> 8192
// in bf16 take 583 us forward (1.41 PFLOP/s) and 1.17 ms backward (1.41) one at a time,
// 610-690 us and 1.3-1.4 ms in a loop, where cuBLAS holds 1.41 PFLOP/s too.  Few tiles
// are bound by one tile's way: 3 us to the first stage, 0.26-0.4 us a stage, and 4-6 us
// of epilogue.
#include <algorithm>
#include <atomic>
#include <cstdint>
#include <cstring>

#include "gated_ff_pair.cuh"
#include "zg_gemm_internal.h"

namespace zg {
namespace {

constexpr int kThreads = 320, kEpiWarps = 8;
constexpr int kBK = 64, kBox = 64;             // of the sum per stage; rows per box
constexpr int kRun = kFfRun / kBK;             // stages in a run
constexpr int kBoxBytes = kBox * 128;          // 8 KB
constexpr int kOperandBytes = 2 * kBoxBytes;   // 128 rows
constexpr int kStageBytes = 2 * kOperandBytes; // A and B: 32 KB per CTA
// Stages: five; dh's epilogue, which also holds blocks of g and u, leaves room for
// four.
constexpr int kStageCount[3] = {5, 5, 4};
constexpr int kBlock32 = 32 * kPitch<float>;
constexpr int kBlock16 = 32 * kPitch<__half>;
constexpr int kTurnBytes[3] = {kBlock32, kBlock32, kBlock16 + 2 * kBlock32};
constexpr int smem_bytes(int epi) {
    return kStageCount[epi] * kStageBytes + kEpiWarps * kTurnBytes[epi] + 1024 /*align*/ +
           256 /*bars*/;
}
static_assert(smem_bytes(2) <= 232448, "shared memory of an SM");
constexpr uint32_t kTmemCols = 512;

struct alignas(64) PairProblem {
    CUtensorMap a[2], b[2];
    void* c;
    void* c2;
    void* c3;
    float* pre_g;
    float* pre_u;
    int64_t ldc;
    int M, N;
    int nkb[2];  // stages of the two sums
    int a_mn, b_mn;
    int vec_c, vec_pre;
    int splits;     // of the sum; with more than one, parts[s] = c, planes of M x ldp f32
    int64_t plane;  // elements of one
    int tiles;      // of this problem and those before it, each split counted
};

struct PairArgs {
    PairProblem p[kMaxProblems];
    int count;
    int full_units, split;
    Deal deal;
    uint32_t* status;
};

__device__ __forceinline__ uint64_t smem_desc(uint32_t saddr, uint32_t lbo) {
    return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) |
           (static_cast<uint64_t>((lbo >> 4) & 0x3FFFu) << 16) |
           (static_cast<uint64_t>(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// kind::f16 instruction descriptor: f32 D, M = 256, N, types and majors.
template <class T>
__device__ __forceinline__ uint32_t instr_desc(int n, int a_mn, int b_mn) {
    const uint32_t type = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    return (1u << 4) | (type << 7) | (type << 10) | (static_cast<uint32_t>(a_mn) << 15) |
           (static_cast<uint32_t>(b_mn) << 16) | (static_cast<uint32_t>(n >> 3) << 17) |
           (static_cast<uint32_t>(256 >> 4) << 24);
}

// Two 64-row boxes (one when `rows` is 64) of an operand, rows from r0, the sum
// from i0.
__device__ __forceinline__ void load_operand(uint8_t* smem, const CUtensorMap* map, int mn, int r0,
                                             int i0, int rows, uint32_t bar) {
    for (int b = 0; b < rows; b += kBox)
        tma_load_2d_pair(smem + b * 128, map, mn ? r0 + b : i0, mn ? i0 : r0 + b, bar);
}

// A unit of work: a tile, or a column half of one of the last tiles.
struct Unit {
    const PairProblem* p;
    int m0, n0, width;  // width: columns of D in TMEM, 256 or 128
    int part, kb0, kb1;
};
template <int EPI>
__device__ __forceinline__ Unit unit_of(const PairArgs& args, int u) {
    const bool half = u >= args.full_units && args.split > 1;
    const int tile = half ? args.full_units + (u - args.full_units) / 2 : u;
    int i = 0;
    while (i + 1 < args.count && tile >= args.p[i].tiles) ++i;
    const PairProblem& p = args.p[i];
    constexpr int cols = EPI == kFfGated ? 128 : 256;  // columns of the output
    const int mt = (p.M + 255) / 256, nt = (p.N + cols - 1) / cols;
    const int t = tile - (i ? args.p[i - 1].tiles : 0);
    Unit w;
    w.p = &p;
    w.part = EPI == kFfStore ? t / (mt * nt) : 0;
    const int nkb = p.nkb[0] + p.nkb[1];
    w.kb0 = nkb * w.part / p.splits;
    w.kb1 = nkb * (w.part + 1) / p.splits;
    int mi, ni;
    raster(t - w.part * mt * nt, mt, nt, mi, ni);
    w.m0 = mi * 256;
    w.n0 = ni * cols + (half ? ((u - args.full_units) & 1) * (cols / 2) : 0);
    w.width = half ? 128 : 256;
    return w;
}

// A lane's row of 32 values as 16-bit pairs, for the tensors' type.
template <class T>
__device__ __forceinline__ uint32_t pair16(float lo, float hi) {
    T t[2] = {FfElem<T>::put(lo), FfElem<T>::put(hi)};
    uint32_t w;
    __builtin_memcpy(&w, t, 4);
    return w;
}

// The reverse for f32, asynchronous: copies the block's rows into `turn`, zeros
// outside the matrix.  Pieces as flush_block's.
__device__ __forceinline__ void fetch_block(const float* src, int64_t ld, int rows, int cols,
                                            bool vec, uint8_t* turn, int lane) {
    const uint32_t to = smem_u32(turn);
    if (vec) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int r = (j * 32 + lane) / 8, piece = lane % 8;
            const bool in = r < rows && piece * 4 < cols;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                             to + r * kPitch<float> + piece * 16),
                         "l"(in ? src + r * ld + piece * 4 : src), "r"(in ? 16 : 0)
                         : "memory");
        }
    } else {
#pragma unroll 4
        for (int r = 0; r < 32; ++r) {
            const bool in = r < rows && lane < cols;
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(
                             to + r * kPitch<float> + lane * 4),
                         "l"(in ? src + r * ld + lane : src), "r"(in ? 4 : 0)
                         : "memory");
        }
    }
}

// LONG: a unit's sum may take several runs.
template <int EPI, int ACT, class T, bool LONG>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    ff_pair_kernel(const __grid_constant__ PairArgs args) {
    constexpr int kStages = kStageCount[EPI];
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                               ~uintptr_t(1023));
    uint8_t* turns = smem + kStages * kStageBytes;
    uint64_t* full = reinterpret_cast<uint64_t*>(turns + kEpiWarps * kTurnBytes[EPI]);
    uint64_t* empty = full + kStages;
    uint64_t* acc_full = empty + kStages;
    uint64_t* acc_empty = acc_full + 2;
    uint64_t* drain = acc_empty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    const int pair = blockIdx.x >> 1;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], 2 * kEpiWarps);
        }
        mbar_init(drain, 1);
        fence_mbar_init();
    }
    if (warp == 1) tmem_alloc_pair(tmem_slot, kTmemCols);
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    // after the allocation: a dependent CTA must not hold TMEM that this grid waits for
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // what the kernel before this one wrote may be read from here on
    asm volatile("griddepcontrol.wait;\n\tfence.proxy.async.global;" ::: "memory");

    if (warp == 0) {
        // ---------------- TMA producer (both CTAs) ----------------
        if (lane == 0) {
            int it = 0;
            bool ok = true;
            for (int j = 0, u; ok && (u = unit_at(args.deal, pair, j)) >= 0; ++j) {
                const Unit w = unit_of<EPI>(args, u);
                const PairProblem& p = *w.p;
                const int b_rows = w.width / 2;
                // gated: CTA 0 takes Wg's columns, CTA 1 the same columns of Wu
                const int b0 = EPI == kFfGated ? w.n0 : w.n0 + b_rows * static_cast<int>(rank);
                for (int kb = w.kb0; kb < w.kb1; ++kb, ++it) {
                    const int s = it % kStages;
                    if (!mbar_wait_bounded(&empty[s], ((it / kStages) & 1) ^ 1, args.status,
                                           kErrFfProducer)) {
                        ok = false;
                        break;
                    }
                    if (leader)
                        mbar_arrive_expect_tx(&full[s], 2 * (kOperandBytes + b_rows * 128));
                    const uint32_t bar = mapa_shared(&full[s], 0);
                    uint8_t* st = smem + s * kStageBytes;
                    const int seg = kb < p.nkb[0] ? 0 : 1;
                    const int i0 = (kb - (seg ? p.nkb[0] : 0)) * kBK;
                    load_operand(st, &p.a[seg], p.a_mn, w.m0 + 128 * static_cast<int>(rank), i0,
                                 128, bar);
                    load_operand(st + kOperandBytes, &p.b[EPI == kFfGated ? rank : seg], p.b_mn,
                                 b0, i0, b_rows, bar);
                }
            }
            // no copy may still be landing at exit: wait until the last stages were read
            for (int i = it > kStages ? it - kStages : 0; i < it; ++i)
                mbar_wait_bounded(&empty[i % kStages], (i / kStages) & 1, args.status, kErrFfDrain);
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer (CTA 0) ----------------
        if (leader && lane == 0) {
            bool ok = true;
            int it = 0, n = 0;  // stages and runs so far
            for (int j = 0, u; ok && (u = unit_at(args.deal, pair, j)) >= 0; ++j) {
                const Unit w = unit_of<EPI>(args, u);
                const PairProblem& p = *w.p;
                const uint32_t idesc = instr_desc<T>(w.width, p.a_mn, p.b_mn);
                const uint32_t a_step = p.a_mn ? 2048 : 32, b_step = p.b_mn ? 2048 : 32;
                for (int k0 = w.kb0; k0 < w.kb1 && ok; k0 += kRun, ++n) {
                    const int buf = n & 1;
                    const uint32_t d_tmem = tmem_base + buf * 256;
                    if (n >= 2 && !mbar_wait_bounded(&acc_empty[buf], ((n >> 1) - 1) & 1,
                                                     args.status, kErrFfMma)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const int k1 = LONG ? min(w.kb1, k0 + kRun) : w.kb1;
                    for (int kb = k0; kb < k1; ++kb, ++it) {
                        const int s = it % kStages;
                        if (!mbar_wait_bounded(&full[s], (it / kStages) & 1, args.status,
                                               kErrFfMma)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        const uint32_t a = smem_u32(smem + s * kStageBytes), b = a + kOperandBytes;
#pragma unroll
                        for (int i = 0; i < kBK / 16; ++i)
                            mma_f16_ss_pair(d_tmem, smem_desc(a + i * a_step, kBoxBytes),
                                            smem_desc(b + i * b_step, kBoxBytes), idesc,
                                            kb != k0 || i != 0);
                        mma_commit_pair(&empty[s], 0x3);
                    }
                    if (ok) mma_commit_pair(&acc_full[buf], 0x3);
                    if (!LONG) break;
                }
                if (!LONG) ++n;
            }
            if (!ok) {
                mma_commit_pair(drain, 0x1);
                mbar_wait_bounded(drain, 0, args.status, kErrFfDrain);
            }
        }
    } else {
        // ---------------- epilogue (warps 2..9, both CTAs) ----------------
        const int q = warp & 3, half = (warp - 2) >> 2;
        const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
        const uint32_t leader_empty0 = mapa_shared(&acc_empty[0], 0);
        const uint32_t leader_empty1 = mapa_shared(&acc_empty[1], 0);
        uint8_t* turn = turns + (warp - 2) * kTurnBytes[EPI];
        uint8_t *turn_g = turn + kBlock16, *turn_u = turn_g + kBlock32;  // dh's epilogue
        // what the runs before a sum's last one came to: D's columns of this warp, Wu's
        // from 64 on in the gated form
        float held[LONG ? 128 : 1];
        int n = 0;
        for (int j = 0, u; (u = unit_at(args.deal, pair, j)) >= 0; ++j, ++n) {
            const Unit w = unit_of<EPI>(args, u);
            const PairProblem& p = *w.p;
            const int64_t row0 = w.m0 + 128 * static_cast<int>(rank) + q * 32;
            const int rows = static_cast<int>(min(p.M - row0, static_cast<int64_t>(32)));
            // columns of the output this warp covers
            const int span = EPI == kFfGated ? w.width / 4 : w.width / 2;
            const int begin = half * span, end = begin + span;
            auto fetch = [&](int c0) {
                // a block that lies outside altogether is not even addressed
                const int cols = min(p.N - w.n0 - c0, 32);
                const int64_t pre = rows > 0 && cols > 0 ? row0 * p.N + w.n0 + c0 : 0;
                fetch_block(p.pre_g + pre, p.N, rows, cols, p.vec_pre, turn_g, lane);
                fetch_block(p.pre_u + pre, p.N, rows, cols, p.vec_pre, turn_u, lane);
            };
            if (EPI == kFfSlope) fetch(begin);  // on its way while the sums finish
            const bool many = LONG && w.kb1 - w.kb0 > kRun;
            auto add_held = [&](auto& r, int at) {
                if (many) {
#pragma unroll
                    for (int e = 0; e < static_cast<int>(sizeof(r) / sizeof(r[0])); ++e)
                        r[e] = __float_as_uint(held[at + e] + __uint_as_float(r[e]));
                }
            };
            bool lost = false;
            for (int k0 = w.kb0; many && k0 + kRun < w.kb1; k0 += kRun, ++n) {
                const bool here = mbar_wait_bounded(&acc_full[n & 1], (n >> 1) & 1, args.status,
                                                    kErrFfEpilogue);
                if ((lost = !__all_sync(0xffffffffu, here))) break;
                tc_fence_after();
                for (int at = 0; at < (EPI == kFfGated ? 2 : 1) * span; at += 16) {
                    const bool up = EPI == kFfGated && at >= span;  // Wu's half
                    const int in = up ? at - span : at;
                    uint32_t r[16];
                    tmem_ld_32x32b_x16(lane_base + (n & 1) * 256 + (up ? w.width / 2 : 0) + begin + in,
                                       r);
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        float& h = held[(up ? 64 : 0) + in + e];
                        h = k0 == w.kb0 ? __uint_as_float(r[e]) : h + __uint_as_float(r[e]);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(n & 1 ? leader_empty1 : leader_empty0);
            }
            if (lost) break;
            const int buf = n & 1;
            const bool got = mbar_wait_bounded(&acc_full[buf], (n >> 1) & 1, args.status,
                                               kErrFfEpilogue);
            // the TMEM loads below are warp-collective: the warp gives up together
            if (!__all_sync(0xffffffffu, got)) break;
            tc_fence_after();
            const uint32_t d = lane_base + buf * 256;
            constexpr int kStep = EPI == kFfStore ? 64 : 32;  // columns a turn
            for (int c0 = begin; c0 < end; c0 += kStep) {
                const int col = w.n0 + c0, cols = p.N - col;
                const int64_t at = row0 * p.ldc + col, pre = row0 * p.N + col;
                T* c = static_cast<T*>(p.c) + at;
                uint8_t* mine32 = turn + lane * kPitch<float>;
                uint8_t* mine16 = turn + lane * kPitch<T>;
                auto f = [](uint32_t x) { return __uint_as_float(x); };
                const int own = c0 - begin;  // of the columns in `held`
                // 32 columns of D from `from` on, as they are, to an f32 matrix
                auto put32 = [&](uint32_t from, int at, float* to, int64_t ld, int width, bool vec) {
                    __syncwarp();
#pragma unroll 1
                    for (int i = 0; i < 32; i += 16) {
                        uint32_t r[16];
                        tmem_ld_32x32b_x16(from + i, r);
                        add_held(r, at + i);
#pragma unroll
                        for (int e = 0; e < 16; e += 4)
                            *reinterpret_cast<uint4*>(mine32 + (i + e) * 4) =
                                make_uint4(r[e], r[e + 1], r[e + 2], r[e + 3]);
                    }
                    __syncwarp();
                    flush_block<float, 32>(to, ld, rows, width, vec, turn, kPitch<float>, 16, lane);
                };
                if (EPI == kFfStore && p.splits > 1) {
                    float* part = static_cast<float*>(p.c) + w.part * p.plane + at;
#pragma unroll 1
                    for (int h = 0; h < 64; h += 32)
                        put32(d + c0 + h, own + h, part + h, p.ldc, cols - h, true);
                } else if (EPI == kFfStore) {
                    __syncwarp();
#pragma unroll 1
                    for (int i = 0; i < 64; i += 16) {
                        uint32_t r[16];
                        tmem_ld_32x32b_x16(d + c0 + i, r);
                        add_held(r, own + i);
                        uint32_t o[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) o[e] = pair16<T>(f(r[2 * e]), f(r[2 * e + 1]));
                        *reinterpret_cast<uint4*>(mine32 + i * 2) =
                            make_uint4(o[0], o[1], o[2], o[3]);
                        *reinterpret_cast<uint4*>(mine32 + i * 2 + 16) =
                            make_uint4(o[4], o[5], o[6], o[7]);
                    }
                    __syncwarp();
                    flush_block<T, 64>(c, p.ldc, rows, cols, p.vec_c, turn, kPitch<float>, 16, lane);
                }
                if (EPI == kFfGated) {
                    const uint32_t u0 = d + w.width / 2 + c0;
                    if (p.pre_g) {
#pragma unroll 1
                        for (int which = 0; which < 2; ++which)
                            put32(which ? u0 : d + c0, which ? 64 + own : own,
                                  (which ? p.pre_u : p.pre_g) + pre, p.N, cols, p.vec_pre);
                    }
                    __syncwarp();
#pragma unroll 1
                    for (int i = 0; i < 32; i += 8) {
                        uint32_t g[8], x[8], o[4];
                        tmem_ld_32x32b_2x8(d + c0 + i, u0 + i, g, x);
                        add_held(g, own + i);
                        add_held(x, 64 + own + i);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            o[e] = pair16<T>(
                                activate<ACT, true>(f(g[2 * e])).a * f(x[2 * e]),
                                activate<ACT, true>(f(g[2 * e + 1])).a * f(x[2 * e + 1]));
                        *reinterpret_cast<uint4*>(mine16 + i * 2) =
                            make_uint4(o[0], o[1], o[2], o[3]);
                    }
                    __syncwarp();
                    flush_block<T, 32>(c, p.ldc, rows, cols, p.vec_c, turn, kPitch<T>, 16, lane);
                }
                if (EPI == kFfSlope) {
                    uint8_t* my_g = turn_g + lane * kPitch<float>;
                    const uint8_t* my_u = turn_u + lane * kPitch<float>;
                    asm volatile("cp.async.wait_all;" ::: "memory");
                    __syncwarp();
                    // dg to `turn`; du and h take the places of the g they came from
#pragma unroll 1
                    for (int i = 0; i < 32; i += 8) {
                        uint32_t r[8], o[12];
                        tmem_ld_32x32b_x8(d + c0 + i, r);
                        add_held(r, own + i);
                        float g[8], x[8];
#pragma unroll
                        for (int e = 0; e < 8; e += 4) {
                            const float4 g4 = *reinterpret_cast<const float4*>(my_g + (i + e) * 4);
                            const float4 u4 = *reinterpret_cast<const float4*>(my_u + (i + e) * 4);
                            g[e] = g4.x, g[e + 1] = g4.y, g[e + 2] = g4.z, g[e + 3] = g4.w;
                            x[e] = u4.x, x[e + 1] = u4.y, x[e + 2] = u4.z, x[e + 3] = u4.w;
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float v[3][2];
#pragma unroll
                            for (int q = 0; q < 2; ++q) {
                                const ActValue a = activate<ACT, true>(g[2 * e + q]);
                                const float dh = f(r[2 * e + q]), u = x[2 * e + q];
                                v[0][q] = dh * u * a.slope;
                                v[1][q] = dh * a.a;
                                v[2][q] = a.a * u;
                            }
#pragma unroll
                            for (int t = 0; t < 3; ++t) o[4 * t + e] = pair16<T>(v[t][0], v[t][1]);
                        }
                        *reinterpret_cast<uint4*>(mine16 + i * 2) =
                            make_uint4(o[0], o[1], o[2], o[3]);
                        *reinterpret_cast<uint4*>(my_g + i * 4) =
                            make_uint4(o[4], o[5], o[6], o[7]);
                        *reinterpret_cast<uint4*>(my_g + i * 4 + 16) =
                            make_uint4(o[8], o[9], o[10], o[11]);
                    }
                    __syncwarp();
#pragma unroll 1
                    for (int t = 2; t >= 0; --t) {
                        // the next block's g and u, while dg is stored
                        if (t == 0) {
                            __syncwarp();
                            if (c0 + 32 < end) fetch(c0 + 32);
                        }
                        void* to = t == 2 ? p.c3 : t == 1 ? p.c2 : p.c;
                        flush_block<T, 32>(static_cast<T*>(to) + at, p.ldc, rows, cols, p.vec_c,
                                           t == 0 ? turn : turn_g + (t - 1) * 16,
                                           t == 0 ? kPitch<T> : kPitch<float>, t == 0 ? 16 : 32,
                                           lane);
                    }
                    __syncwarp();
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(buf ? leader_empty1 : leader_empty0);
        }
        if (EPI == kFfSlope) asm volatile("cp.async.wait_all;" ::: "memory");  // gave up early
    }

    tc_fence_before();
    cluster_sync();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, kTmemCols);
    }
}

// ---- host ----------------------------------------------------------------------
// An operand as 64 x 64 boxes: inner dimension along the memory.
int operand_map(CUtensorMap* map, uint32_t dtype, const FfOperand& o, int rows, int sum) {
    return encode_16bit_map(map, dtype, o.p, o.mn ? rows : sum, o.mn ? sum : rows, o.ld, kBox, kBox);
}

template <int EPI, int ACT, class T, bool LONG>
int launch_runs(const PairArgs& args, cudaStream_t s) {
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = allow_smem(ff_pair_kernel<EPI, ACT, T, LONG>, smem_bytes(EPI), done);
    if (e != cudaSuccess) return cuda_status(e, "gated_ff shared memory");
    return launch_dependent("gated_ff", ff_pair_kernel<EPI, ACT, T, LONG>, 2 * args.deal.pairs,
                            kThreads, smem_bytes(EPI), s, args);
}
template <int EPI, int ACT, class T>
int launch(const PairArgs& args, cudaStream_t s) {
    for (int i = 0; i < args.count; ++i) {
        const PairProblem& p = args.p[i];
        if ((p.nkb[0] + p.nkb[1] + p.splits - 1) / p.splits > kRun)
            return launch_runs<EPI, ACT, T, true>(args, s);
    }
    return launch_runs<EPI, ACT, T, false>(args, s);
}

template <class T>
int launch_epi(FfEpilogue epi, int act, const PairArgs& a, cudaStream_t s) {
    if (epi == kFfStore) return launch<kFfStore, ZG_ACT_RELU, T>(a, s);
    if (epi == kFfGated) switch (act) {
            case ZG_ACT_SILU: return launch<kFfGated, ZG_ACT_SILU, T>(a, s);
            case ZG_ACT_GELU: return launch<kFfGated, ZG_ACT_GELU, T>(a, s);
            case ZG_ACT_GELU_TANH: return launch<kFfGated, ZG_ACT_GELU_TANH, T>(a, s);
            default: return launch<kFfGated, ZG_ACT_RELU, T>(a, s);
        }
    switch (act) {
        case ZG_ACT_SILU: return launch<kFfSlope, ZG_ACT_SILU, T>(a, s);
        case ZG_ACT_GELU: return launch<kFfSlope, ZG_ACT_GELU, T>(a, s);
        case ZG_ACT_GELU_TANH: return launch<kFfSlope, ZG_ACT_GELU_TANH, T>(a, s);
        default: return launch<kFfSlope, ZG_ACT_RELU, T>(a, s);
    }
}

}  // namespace

uint64_t ff_split_bytes(const FfProduct* products, int count) {
    return split_bytes(products, count, kBK);
}

int ff_pair(uint32_t dtype, FfEpilogue epi, int act, const FfProduct* products, int count,
            float* parts, cudaStream_t s) {
    PairArgs args;
    std::memset(&args, 0, sizeof(args));
    args.count = count;
    int rc = status_word(&args.status), tiles = 0;
    int splits[kMaxProblems] = {1, 1, 1, 1};
    if (epi == kFfStore) splits_of(products, count, kBK, splits);
    SumArgs sum;
    sum.count = 0;
    const int cols = epi == kFfGated ? 128 : 256;
    for (int i = 0; i < count && !rc; ++i) {
        const FfProduct& f = products[i];
        PairProblem& p = args.p[i];
        p.M = f.M, p.N = f.N;
        p.a_mn = f.a[0].mn, p.b_mn = f.b[0].mn;
        p.c = f.c, p.c2 = f.c2, p.c3 = f.c3, p.ldc = f.ldc;
        p.pre_g = f.pre_g, p.pre_u = f.pre_u;
        p.vec_c = f.ldc % 8 == 0 && aligned16(f.c) && aligned16(f.c2) && aligned16(f.c3);
        p.vec_pre = f.N % 4 == 0 && aligned16(f.pre_g) && aligned16(f.pre_u);
        for (int seg = 0; seg < 2; ++seg) p.nkb[seg] = (f.k[seg] + kBK - 1) / kBK;
        p.splits = splits[i];
        if (splits[i] > 1) {  // f32 parts first
            p.c = parts;
            add_parts(sum, f, splits[i], parts);
            p.plane = sum.m[sum.count - 1].plane, p.ldc = sum.m[sum.count - 1].ldp;
        }
        rc = operand_map(&p.a[0], dtype, f.a[0], f.M, f.k[0]);
        if (!rc) rc = operand_map(&p.b[0], dtype, f.b[0], f.N, f.k[0]);
        if (!rc && f.k[1]) rc = operand_map(&p.a[1], dtype, f.a[1], f.M, f.k[1]);
        if (!rc && f.b[1].p) rc = operand_map(&p.b[1], dtype, f.b[1], f.N, f.k[1] ? f.k[1] : f.k[0]);
        const int64_t total =
            tiles + static_cast<int64_t>((f.M + 255) / 256) * ((f.N + cols - 1) / cols) * splits[i];
        if (total > (1 << 29)) return set_error(ZG_ERR_DISPATCH, "gated_ff: too many tiles");
        p.tiles = tiles = static_cast<int>(total);
    }
    if (rc) return rc;
    // the last wave's tiles in halves, where the units are of one kind
    const int pairs = sm_pairs(), rem = tiles % pairs;
    args.split = count == 1 && rem > 0 && 2 * rem <= pairs ? 2 : 1;
    args.full_units = args.split > 1 ? tiles - rem : tiles;
    auto unit_time = [&](int i) {  // in stages; an epilogue takes about eight
        return (args.p[i].nkb[0] + args.p[i].nkb[1]) / splits[i] + 8;
    };
    args.deal = deal_of(args.full_units + (tiles - args.full_units) * args.split, pairs,
                        args.p[0].tiles, count > 1 ? unit_time(0) / unit_time(1) : 0);
    rc = dtype == ZG_DTYPE_BF16 ? launch_epi<__nv_bfloat16>(epi, act, args, s)
                                : launch_epi<__half>(epi, act, args, s);
    if (rc) return rc;
    return dtype == ZG_DTYPE_BF16 ? launch_sum<__nv_bfloat16>(sum, s) : launch_sum<__half>(sum, s);
}

}  // namespace zg
