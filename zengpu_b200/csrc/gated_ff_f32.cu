// gated_ff_f32.cu - the products of the gated feed-forward block on f32 tensors in the
// TF32X3 mode: tcgen05 CTA pairs on split-precision operand planes (sgemm_tc.cu: x =
// hi + lo in tf32, every 16 of the sum one 128-byte row of 16 hi and 16 lo; three
// kind::tf32 products hi lo + lo hi + hi hi), several products to a launch and long
// sums split; and the elementwise work between them, which writes h, dg and du
// straight as the next products' planes.
//
// The tensor core's f32 additions truncate, so a sum that stays in TMEM loses about
// half a unit of the last place an addition, always downwards.  Here it stays for 48
// of the sum, 18 additions (sgemm_tc.cu: 512, 192); sixteen epilogue warps then add
// it to f32 registers, rounding to nearest, 64 columns a lane, while the MMAs fill
// the other accumulator.  Two chained products so end within 1.1e-6 of float64, about
// what plain f32 sums give.  A drain reads 128 KB of TMEM per SM, 2000 cycles and
// more beside the MMAs, whose chunk takes 2500; with 32 of the sum a chunk the MMAs
// would wait for it (a training pass 1.3 times as long).
//
// Tiles, pairs and roles as gated_ff_tc.cu, 256 x 256 with 16 of the sum a stage.  A
// training pass of 2048 rows, 1024 -> 4096, takes 0.92 ms: 168 useful TFLOP/s, 0.75 ms
// of it in the products (206), whose ceiling is a sixth of the bf16 rate, 279.
#include <cstdint>
#include <cstring>

#include "gated_ff_pair.cuh"
#include "zg_gemm_internal.h"

namespace zg {
namespace {

constexpr int kThreads = 64 + 32 * 16, kEpi = 16;
constexpr int kBK = 16, kStages = 4, kChunk = 3;  // of the sum; stages; stages a chunk
constexpr int kOperandBytes = 128 * 128, kStageBytes = 2 * kOperandBytes;
constexpr int kTurnBytes = 32 * kPitch<float>;
constexpr int kSmem = kStages * kStageBytes + kEpi * kTurnBytes + 1024 + 256;
constexpr uint32_t kTmemCols = 512;

struct alignas(64) F32Problem {
    CUtensorMap a, b;
    float* c;
    int64_t ldc, plane;  // plane: elements of a part of a split sum
    int M, N, nkb, vec_c, splits, tiles;
};
struct F32Args {
    F32Problem p[kMaxProblems];
    int count;
    Deal deal;
    uint32_t* status;
};

__device__ __forceinline__ uint64_t plane_desc(uint32_t saddr) {
    return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) | (1ull << 16) |
           (static_cast<uint64_t>(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
constexpr uint32_t kIdesc = (1u << 4) | (2u << 7) | (2u << 10) | ((256u >> 3) << 17) |
                            ((256u >> 4) << 24);

struct F32Unit {
    const F32Problem* p;
    int m0, n0, part, kb0, kb1;
};
__device__ __forceinline__ F32Unit f32_unit(const F32Args& args, int u) {
    int i = 0;
    while (i + 1 < args.count && u >= args.p[i].tiles) ++i;
    const F32Problem& p = args.p[i];
    const int mt = (p.M + 255) / 256, nt = (p.N + 255) / 256;
    const int t = u - (i ? args.p[i - 1].tiles : 0);
    F32Unit w;
    w.p = &p;
    w.part = t / (mt * nt);
    w.kb0 = p.nkb * w.part / p.splits;
    w.kb1 = p.nkb * (w.part + 1) / p.splits;
    int mi, ni;
    raster(t - w.part * mt * nt, mt, nt, mi, ni);
    w.m0 = mi * 256, w.n0 = ni * 256;
    return w;
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    ff_f32_kernel(const __grid_constant__ F32Args args) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                               ~uintptr_t(1023));
    uint8_t* turns = smem + kStages * kStageBytes;
    uint64_t* full = reinterpret_cast<uint64_t*>(turns + kEpi * kTurnBytes);
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
            mbar_init(&acc_empty[b], 2 * kEpi);
        }
        mbar_init(drain, 1);
        fence_mbar_init();
    }
    if (warp == 1) tmem_alloc_pair(tmem_slot, kTmemCols);
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;\n\tfence.proxy.async.global;" ::: "memory");

    if (warp == 0) {
        if (lane == 0) {
            int it = 0;
            bool ok = true;
            for (int j = 0, u; ok && (u = unit_at(args.deal, pair, j)) >= 0; ++j) {
                const F32Unit w = f32_unit(args, u);
                const int half = 128 * static_cast<int>(rank);
                for (int kb = w.kb0; kb < w.kb1; ++kb, ++it) {
                    const int s = it % kStages;
                    if (!mbar_wait_bounded(&empty[s], ((it / kStages) & 1) ^ 1, args.status,
                                           kErrFfProducer)) {
                        ok = false;
                        break;
                    }
                    if (leader) mbar_arrive_expect_tx(&full[s], 2 * kStageBytes);
                    const uint32_t bar = mapa_shared(&full[s], 0);
                    uint8_t* st = smem + s * kStageBytes;
                    tma_load_2d_pair(st, &w.p->a, kb * 32, w.m0 + half, bar);
                    tma_load_2d_pair(st + kOperandBytes, &w.p->b, kb * 32, w.n0 + half, bar);
                }
            }
            for (int i = it > kStages ? it - kStages : 0; i < it; ++i)
                mbar_wait_bounded(&empty[i % kStages], (i / kStages) & 1, args.status, kErrFfDrain);
        }
    } else if (warp == 1) {
        if (leader && lane == 0) {
            bool ok = true;
            int it = 0, n = 0;  // stages and chunks so far
            for (int j = 0, u; ok && (u = unit_at(args.deal, pair, j)) >= 0; ++j) {
                const F32Unit w = f32_unit(args, u);
                for (int kc = w.kb0; kc < w.kb1 && ok; kc += kChunk, ++n) {
                    const int buf = n & 1;
                    const uint32_t d = tmem_base + buf * 256;
                    if (n >= 2 && !mbar_wait_bounded(&acc_empty[buf], ((n >> 1) - 1) & 1,
                                                     args.status, kErrFfMma)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    for (int kb = kc; kb < min(w.kb1, kc + kChunk); ++kb, ++it) {
                        const int s = it % kStages;
                        if (!mbar_wait_bounded(&full[s], (it / kStages) & 1, args.status,
                                               kErrFfMma)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        const uint32_t a = smem_u32(smem + s * kStageBytes), b = a + kOperandBytes;
#pragma unroll
                        for (int i = 0; i < 2; ++i) {  // 8 of the sum: 32 bytes; lo 64 on
                            const uint32_t o = i * 32;
                            mma_tf32_ss_pair(d, plane_desc(a + 64 + o), plane_desc(b + o), kIdesc,
                                             kb != kc || i != 0);
                            mma_tf32_ss_pair(d, plane_desc(a + o), plane_desc(b + 64 + o), kIdesc, 1);
                            mma_tf32_ss_pair(d, plane_desc(a + o), plane_desc(b + o), kIdesc, 1);
                        }
                        mma_commit_pair(&empty[s], 0x3);
                    }
                    if (ok) mma_commit_pair(&acc_full[buf], 0x3);
                }
            }
            if (!ok) {
                mma_commit_pair(drain, 0x1);
                mbar_wait_bounded(drain, 0, args.status, kErrFfDrain);
            }
        }
    } else {
        const int q = warp & 3, group = (warp - 2) >> 2;
        const uint32_t lanes = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
        const uint32_t d0 = group * 64;  // a lane's columns of D
        const uint32_t leader_empty0 = mapa_shared(&acc_empty[0], 0);
        const uint32_t leader_empty1 = mapa_shared(&acc_empty[1], 0);
        uint8_t* turn = turns + (warp - 2) * kTurnBytes;
        bool ok = true;
        int n = 0;
        for (int j = 0, u; ok && (u = unit_at(args.deal, pair, j)) >= 0; ++j) {
            const F32Unit w = f32_unit(args, u);
            const F32Problem& p = *w.p;
            float acc[64] = {};
            for (int kc = w.kb0; kc < w.kb1; kc += kChunk, ++n) {
                const int buf = n & 1;
                bool got = true;  // one lane polls: 512 would crowd the barrier
                if (lane == 0)
                    got = mbar_wait_bounded(&acc_full[buf], (n >> 1) & 1, args.status,
                                            kErrFfEpilogue);
                if (!__all_sync(0xffffffffu, got)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
#pragma unroll
                for (int i = 0; i < 64; i += 16) {
                    uint32_t r[16];
                    tmem_ld_32x32b_x16(lanes + buf * 256 + d0 + i, r);
                    if (i == 48) {  // all of the accumulator is in registers
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive_cluster(buf ? leader_empty1 : leader_empty0);
                    }
#pragma unroll
                    for (int e = 0; e < 16; ++e) acc[i + e] += __uint_as_float(r[e]);
                }
            }
            if (!ok) break;
            const int64_t row0 = w.m0 + 128 * static_cast<int>(rank) + q * 32;
            const int rows = static_cast<int>(min(p.M - row0, static_cast<int64_t>(32)));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int col = w.n0 + group * 64 + 32 * h, cols = min(p.N - col, 32);
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 32; i += 4)
                    *reinterpret_cast<float4*>(turn + lane * kPitch<float> + i * 4) =
                        make_float4(acc[32 * h + i], acc[32 * h + i + 1], acc[32 * h + i + 2],
                                    acc[32 * h + i + 3]);
                __syncwarp();
                flush_block<float, 32>(p.c + w.part * p.plane + row0 * p.ldc + col, p.ldc, rows,
                                       cols, p.vec_c, turn, kPitch<float>, 16, lane);
            }
        }
    }

    tc_fence_before();
    cluster_sync();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, kTmemCols);
    }
}

// ---- between the products ------------------------------------------------------------
// A CTA takes 32 rows (m) x 96 columns (f) of g, u (and dh): three blocks of 32 x 32,
// two warps each for half the rows.  A value's planes are blocks of 16 along the next
// sum: along f for h, dg and du, along m for their transposes, which go through a
// shared tile.  Bound by HBM: 8 bytes read and 8 written for an h, 12 read and 40
// written for a dh.
struct ActArgs {
    const float* g;
    const float* u;
    const float* dh;
    float* rows[2];    // h; or dg and du
    float* turned[3];  // transposes of dg, du, h
    int64_t ld_rows, ld_turned;
    int M, N;
};

// Lane l of 16 puts value l of a block of 16 (hi, then lo 16 floats on).
__device__ __forceinline__ void put_plane(float* row, int k, float x) {
    const float h = to_tf32(x);
    float* p = row + (k >> 4) * 32 + (k & 15);
    p[0] = h;
    p[16] = to_tf32(__fsub_rn(x, h));
}

constexpr int kActCols = 96, kActThreads = 2 * kActCols;
template <int ACT, bool SLOPE>
__global__ void __launch_bounds__(kActThreads) ff_planes_kernel(const ActArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    __shared__ float tile[SLOPE ? kActCols / 32 : 1][SLOPE ? 3 : 1][32][33];
    const int lane = threadIdx.x & 31, block = threadIdx.x / 64, half = threadIdx.x / 32 & 1;
    const int col = blockIdx.y * kActCols + block * 32 + lane;
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * 32;
    const int kpad = (a.N + 15) / 16 * 16;
    float g[16], u[16], d[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int64_t row = row0 + half * 16 + r, at = row * a.N + col;
        const bool in = row < a.M && col < a.N;
        g[r] = in ? __ldcs(a.g + at) : 0.0f;
        u[r] = in ? __ldcs(a.u + at) : 0.0f;
        d[r] = SLOPE && in ? __ldcs(a.dh + at) : 0.0f;
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int64_t row = row0 + half * 16 + r;
        const bool in = row < a.M && col < kpad;
        const ActValue v = activate<ACT, false>(g[r]);
        if (!SLOPE) {
            if (in) put_plane(a.rows[0] + row * a.ld_rows, col, v.a * u[r]);
            continue;
        }
        const float dg = d[r] * u[r] * v.slope, du = d[r] * v.a;
        if (in) {
            put_plane(a.rows[0] + row * a.ld_rows, col, dg);
            put_plane(a.rows[1] + row * a.ld_rows, col, du);
        }
        if (SLOPE) {
            tile[block][0][half * 16 + r][lane] = dg;
            tile[block][1][half * 16 + r][lane] = du;
            tile[block][2][half * 16 + r][lane] = v.a * u[r];
        }
    }
    if (!SLOPE) return;
    __syncthreads();
    // a row of the transpose per turn, its 32 of m along the lanes
    const int mpad = (a.M + 15) / 16 * 16;
    const int m = static_cast<int>(row0) + lane;
#pragma unroll 4
    for (int r = 0; r < 16; ++r) {
        const int c = half * 16 + r, f = blockIdx.y * kActCols + block * 32 + c;
        if (f >= a.N || m >= mpad) continue;
#pragma unroll
        for (int t = 0; t < 3; ++t)
            put_plane(a.turned[t] + f * a.ld_turned, m, tile[SLOPE ? block : 0][SLOPE ? t : 0][lane][c]);
    }
}

template <int ACT, bool SLOPE>
int launch_planes(const ActArgs& a, cudaStream_t s) {
    const dim3 grid((a.M + 31) / 32, (a.N + kActCols - 1) / kActCols);
    if (grid.y > 65535u) return set_error(ZG_ERR_DISPATCH, "gated_ff: too many columns");
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kActThreads);
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cuda_status(cudaLaunchKernelEx(&cfg, ff_planes_kernel<ACT, SLOPE>, a),
                       "gated_ff activation");
}

template <bool SLOPE>
int launch_planes_act(int act, const ActArgs& a, cudaStream_t s) {
    switch (act) {
        case ZG_ACT_SILU: return launch_planes<ZG_ACT_SILU, SLOPE>(a, s);
        case ZG_ACT_GELU: return launch_planes<ZG_ACT_GELU, SLOPE>(a, s);
        case ZG_ACT_GELU_TANH: return launch_planes<ZG_ACT_GELU_TANH, SLOPE>(a, s);
        default: return launch_planes<ZG_ACT_RELU, SLOPE>(a, s);
    }
}

int plane_map(CUtensorMap* map, const FfOperand& o, int rows, int nkb) {
    return encode_f32_map(map, o.p, static_cast<uint64_t>(nkb) * 32, rows, o.ld, 32, 128,
                          CU_TENSOR_MAP_SWIZZLE_128B);
}

}  // namespace

uint64_t ff_f32_split_bytes(const FfProduct* products, int count) {
    return split_bytes(products, count, 64);
}

int ff_f32(const FfProduct* products, int count, float* parts, cudaStream_t s) {
    F32Args args;
    std::memset(&args, 0, sizeof(args));
    args.count = count;
    int rc = status_word(&args.status), tiles = 0;
    int splits[kMaxProblems];
    splits_of(products, count, 64, splits);
    SumArgs sum;
    sum.count = 0;
    for (int i = 0; i < count && !rc; ++i) {
        const FfProduct& f = products[i];
        F32Problem& p = args.p[i];
        p.M = f.M, p.N = f.N, p.nkb = (f.k[0] + kBK - 1) / kBK, p.splits = splits[i];
        p.c = static_cast<float*>(f.c), p.ldc = f.ldc;
        p.vec_c = f.ldc % 4 == 0 && aligned16(f.c);
        if (splits[i] > 1) {
            p.c = parts, p.vec_c = 1;
            add_parts(sum, f, splits[i], parts);
            p.plane = sum.m[sum.count - 1].plane, p.ldc = sum.m[sum.count - 1].ldp;
        }
        rc = plane_map(&p.a, f.a[0], f.M, p.nkb);
        if (!rc) rc = plane_map(&p.b, f.b[0], f.N, p.nkb);
        const int64_t total =
            tiles + static_cast<int64_t>((f.M + 255) / 256) * ((f.N + 255) / 256) * splits[i];
        if (total > (1 << 29)) return set_error(ZG_ERR_DISPATCH, "gated_ff: too many tiles");
        p.tiles = tiles = static_cast<int>(total);
    }
    if (rc) return rc;
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = allow_smem(ff_f32_kernel, kSmem, done);
    if (e != cudaSuccess) return cuda_status(e, "gated_ff shared memory");
    auto unit_time = [&](int i) { return args.p[i].nkb / splits[i] + 8; };  // in stages
    args.deal = deal_of(tiles, sm_pairs(), args.p[0].tiles,
                        count > 1 ? unit_time(0) / unit_time(1) : 0);
    rc = launch_dependent("gated_ff", ff_f32_kernel, 2 * args.deal.pairs, kThreads, kSmem, s, args);
    return rc ? rc : launch_sum<float>(sum, s);
}

int ff_f32_act(int act, const float* g, const float* u, int m, int n, const FfOperand& h,
               cudaStream_t s) {
    ActArgs a{};
    a.g = g, a.u = u, a.M = m, a.N = n;
    a.rows[0] = static_cast<float*>(const_cast<void*>(h.p)), a.ld_rows = h.ld;
    return launch_planes_act<false>(act, a, s);
}

int ff_f32_slope(int act, const float* g, const float* u, const float* dh, int m, int n,
                 const FfOperand& dg, const FfOperand& du, const FfOperand (&turned)[3],
                 cudaStream_t s) {
    ActArgs a{};
    a.g = g, a.u = u, a.dh = dh, a.M = m, a.N = n;
    a.rows[0] = static_cast<float*>(const_cast<void*>(dg.p)), a.ld_rows = dg.ld;
    a.rows[1] = static_cast<float*>(const_cast<void*>(du.p));
    for (int t = 0; t < 3; ++t)
        a.turned[t] = static_cast<float*>(const_cast<void*>(turned[t].p));
    a.ld_turned = turned[0].ld;
    return launch_planes_act<true>(act, a, s);
}

}  // namespace zg
