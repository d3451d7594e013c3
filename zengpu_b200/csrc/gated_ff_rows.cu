// gated_ff_rows.cu - the forward products of the gated feed-forward block for few
// rows (tokens being decoded), 16-bit tensors: every weight is read once, and the
// time is that of reading them.
//
// The weights take the MMA's M side: D^T[128 columns of W x rows of x] = W^T x^T, so
// a tile wastes nothing on missing rows: the MMA's N is the rows rounded up to
// 16, 32 or 64.  W is read as it lies (mn-major, see gated_ff_tc.cu), x or h as
// the k-major B operand.  The gated product holds two accumulators, of Wg and Wu.
//
// A CTA takes 128 columns and a part of the sum; the CTAs of a cluster share the
// columns and split the sum, then add their partial results through distributed
// shared memory, in rank order, so the result does not depend on timing.  Each CTA
// finishes the rows r with r % cluster size == its rank.
//
// Bound by HBM: what counts is bytes in flight, a ring of 64-of-the-sum stages (32 KB
// of weights for the gated pair, 16 KB for Wd) of up to 110 KB per CTA, two CTAs to
// an SM.  y's kernel is launched while h's still runs (programmatic dependent
// launch): it fills its ring with Wd, which nobody writes meanwhile, before it waits
// for h.  4096 -> 12288: one token 54 us for 302 MB (5.6 TB/s), 16 rows 57, 48 rows 64-67: what
// grows is the cluster's exchange of the rows' partial sums, in both kernels, and past
// 32 rows the gated ring holds two stages.
#include <algorithm>
#include <atomic>
#include <cstdint>
#include <cstring>
#include <type_traits>

#include "gated_ff.cuh"
#include "zg_gemm_internal.h"

namespace zg {
namespace {

constexpr int kRowsThreads = 192;  // TMA, MMA, four epilogue warps
constexpr int kRowsMaxStages = 12;
constexpr int kSumStep = 64;
constexpr int kColumns = 128;  // of W per CTA
constexpr int kWeightBytes = kColumns * kSumStep * 2;

struct alignas(64) RowsArgs {
    CUtensorMap w[2], x;
    void* c;
    float* pre_g;
    float* pre_u;
    int64_t ldc;
    int M, N, nkb, stages;
    int vec;  // rows of c, pre_g and pre_u: four columns at a time are aligned
    uint32_t* status;
};

__device__ __forceinline__ uint64_t rows_desc(uint32_t saddr, uint32_t lbo) {
    return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) |
           (static_cast<uint64_t>((lbo >> 4) & 0x3FFFu) << 16) |
           (static_cast<uint64_t>(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t mine, uint32_t rank) {
    float4 v;
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(mine), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(a)
                 : "memory");
    return v;
}

__host__ __device__ constexpr uint32_t tmem_columns(int n) {
    return n <= 32 ? 32 : n <= 64 ? 64 : 128;
}

// GATED: c = act(x Wg) * (x Wu), and the two products to pre_g, pre_u unless null.
// Otherwise c = x W.  ROWS: the MMA's N.
template <bool GATED, int ACT, class T, int ROWS>
__global__ void __launch_bounds__(kRowsThreads)
    ff_rows_kernel(const __grid_constant__ RowsArgs args) {
    constexpr int kMats = GATED ? 2 : 1;
    constexpr int kStage = kMats * kWeightBytes + ROWS * 128;
    constexpr uint32_t kCols = tmem_columns(kMats * ROWS);
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                               ~uintptr_t(1023));
    __shared__ uint64_t full[kRowsMaxStages], empty[kRowsMaxStages], acc_full, drain;
    __shared__ uint32_t tmem_slot;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int stages = args.stages;
    const int split = gridDim.x, rank = blockIdx.x;  // the grid's x is the cluster
    const int n0 = blockIdx.y * kColumns;
    const int kb0 = static_cast<int>(static_cast<int64_t>(args.nkb) * rank / split);
    const int kb1 = static_cast<int>(static_cast<int64_t>(args.nkb) * (rank + 1) / split);

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(&acc_full, 1);
        mbar_init(&drain, 1);
        fence_mbar_init();
    }
    if (warp == 0 && lane == 0) {
        prefetch_tensormap(&args.w[0]);
        if (GATED) prefetch_tensormap(&args.w[1]);
        prefetch_tensormap(&args.x);
    }
    if (warp == 1) tmem_alloc(&tmem_slot, kCols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    // after the allocation: a dependent CTA must not hold TMEM that this grid waits for
    if (GATED) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    if (warp == 0) {
        if (lane == 0) {
            auto weights = [&](int kb) {
                const int s = (kb - kb0) % stages;
                uint8_t* st = smem + s * kStage;
                mbar_arrive_expect_tx(&full[s], kStage);
                for (int w = 0; w < kMats; ++w)
                    for (int h = 0; h < 2; ++h)
                        tma_load_2d(st + w * kWeightBytes + h * (kWeightBytes / 2), &args.w[w],
                                    n0 + 64 * h, kb * kSumStep, &full[s]);
            };
            auto rows = [&](int kb) {
                const int s = (kb - kb0) % stages;
                tma_load_2d(smem + s * kStage + kMats * kWeightBytes, &args.x, kb * kSumStep, 0,
                            &full[s]);
            };
            int issued = kb0;
            const int ahead = min(kb1, kb0 + stages);
            for (; issued < ahead; ++issued) weights(issued);
            // x or h may still be in the making by the kernel before
            if (!GATED)
                asm volatile("griddepcontrol.wait;\n\tfence.proxy.async.global;" ::: "memory");
            for (int kb = kb0; kb < ahead; ++kb) rows(kb);
            for (; issued < kb1; ++issued) {
                const int it = issued - kb0;
                if (!mbar_wait_bounded(&empty[it % stages], ((it / stages) & 1) ^ 1, args.status,
                                       kErrFfProducer))
                    break;
                weights(issued);
                rows(issued);
            }
            // no copy may still be landing when the ring is reused or the CTA ends
            const int n = issued - kb0;
            for (int i = max(0, n - stages); i < n; ++i)
                mbar_wait_bounded(&full[i % stages], (i / stages) & 1, args.status, kErrFfDrain);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t type = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
            constexpr uint32_t idesc = (1u << 4) | (type << 7) | (type << 10) | (1u << 15) |
                                       (static_cast<uint32_t>(ROWS >> 3) << 17) | (8u << 24);
            bool ok = true;
            for (int kb = kb0; kb < kb1 && ok; ++kb) {
                const int it = kb - kb0, s = it % stages;
                if (!mbar_wait_bounded(&full[s], (it / stages) & 1, args.status, kErrFfMma)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t st = smem_u32(smem + s * kStage);
#pragma unroll
                for (int i = 0; i < kSumStep / 16; ++i)
#pragma unroll
                    for (int w = 0; w < kMats; ++w)
                        mma_f16_ss(tmem + w * ROWS,
                                   rows_desc(st + w * kWeightBytes + i * 2048, kWeightBytes / 2),
                                   rows_desc(st + kMats * kWeightBytes + i * 32, 16), idesc,
                                   (it | i) != 0);
                mma_commit(&empty[s]);
            }
            if (ok) {
                mma_commit(&acc_full);
            } else {
                mma_commit(&drain);
                mbar_wait_bounded(&drain, 0, args.status, kErrFfDrain);
            }
        }
    }

    // ---------------- results ----------------
    const int q = warp & 3;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(q * 32) << 16);
    const int column = q * 32 + lane;
    auto finish = [&](int row, int col, float g, float u) {
        if (col >= args.N || row >= args.M) return;
        T* c = static_cast<T*>(args.c) + row * args.ldc + col;
        if (GATED) {
            if (args.pre_g) {
                const int64_t pre = static_cast<int64_t>(row) * args.N + col;
                args.pre_g[pre] = g;
                args.pre_u[pre] = u;
            }
            *c = FfElem<T>::put(activate<ACT, true>(g).a * u);
        } else {
            *c = FfElem<T>::put(g);
        }
    };
    auto finish4 = [&](int row, int col, float4 g, float4 u) {
        if (args.vec && col + 4 <= args.N) {
            const float v[4] = {g.x, g.y, g.z, g.w}, w[4] = {u.x, u.y, u.z, u.w};
            T t[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                t[e] = FfElem<T>::put(GATED ? activate<ACT, true>(v[e]).a * w[e] : v[e]);
            uint2 q;
            __builtin_memcpy(&q, t, 8);
            *reinterpret_cast<uint2*>(static_cast<T*>(args.c) + row * args.ldc + col) = q;
            if (GATED && args.pre_g) {
                const int64_t pre = static_cast<int64_t>(row) * args.N + col;
                *reinterpret_cast<float4*>(args.pre_g + pre) = g;
                *reinterpret_cast<float4*>(args.pre_u + pre) = u;
            }
        } else {
            finish(row, col, g.x, u.x);
            finish(row, col + 1, g.y, u.y);
            finish(row, col + 2, g.z, u.z);
            finish(row, col + 3, g.w, u.w);
        }
    };
    bool ok = true;
    if (warp >= 2) {
        ok = mbar_wait_bounded(&acc_full, 0, args.status, kErrFfEpilogue);
        ok = __all_sync(0xffffffffu, ok);  // the TMEM loads are warp-collective
        tc_fence_after();
        if (ok && split == 1) {
#pragma unroll
            for (int r0 = 0; r0 < ROWS; r0 += 16) {
                if (r0 >= args.M) break;
                uint32_t g[16], u[16];
                tmem_ld_32x32b_x16(lanes + r0, g);
                if (GATED) tmem_ld_32x32b_x16(lanes + ROWS + r0, u);
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    finish(r0 + i, n0 + column, __uint_as_float(g[i]),
                           GATED ? __uint_as_float(u[i]) : 0.0f);
            }
        }
    }
    if (split > 1) {
        // The ring is free: every copy has landed (the producer waited) and every MMA
        // has read it (acc_full).  Its memory takes the partial results.
        float* part = reinterpret_cast<float*>(smem);
        if (warp >= 2 && ok) {
#pragma unroll
            for (int w = 0; w < kMats; ++w)
#pragma unroll
                for (int r0 = 0; r0 < ROWS; r0 += 16) {
                    if (r0 >= args.M) break;
                    uint32_t v[16];
                    tmem_ld_32x32b_x16(lanes + w * ROWS + r0, v);
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        part[(w * ROWS + r0 + i) * kColumns + column] = __uint_as_float(v[i]);
                }
        }
        cluster_sync();
        if (warp >= 2) {
            // A warp to a row, four columns to a lane, the loads of several ranks
            // and rows in flight together (one from another SM takes about 300 ns).
            // After an expired wait the sums mean nothing, as the status word says, but
            // are in bounds.
            const uint32_t at = smem_u32(part) + lane * 16;
            constexpr int kBatch = ROWS == 16 ? 1 : 2;
            const int col = n0 + lane * 4, step = split * 4;
            for (int row = rank + split * (warp - 2); row < args.M; row += kBatch * step) {
                float4 g[kBatch], u[kBatch];
#pragma unroll
                for (int i = 0; i < kBatch; ++i) g[i] = u[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
                for (int p = 0; p < split; ++p) {
                    float4 x[kBatch], z[kBatch];
#pragma unroll
                    for (int i = 0; i < kBatch; ++i) {
                        const int r = min(row + i * step, args.M - 1);  // loaded, not stored
                        x[i] = ld_cluster_f32x4(at + r * (kColumns * 4), p);
                        if (GATED) z[i] = ld_cluster_f32x4(at + (ROWS + r) * (kColumns * 4), p);
                    }
#pragma unroll
                    for (int i = 0; i < kBatch; ++i) {
                        g[i].x += x[i].x, g[i].y += x[i].y, g[i].z += x[i].z, g[i].w += x[i].w;
                        if (GATED)
                            u[i].x += z[i].x, u[i].y += z[i].y, u[i].z += z[i].z, u[i].w += z[i].w;
                    }
                }
#pragma unroll
                for (int i = 0; i < kBatch; ++i)
                    if (row + i * step < args.M) finish4(row + i * step, col, g[i], u[i]);
            }
        }
        cluster_sync();  // nobody leaves while its memory is read
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, kCols);
    }
}

// ---- host ----------------------------------------------------------------------
int rows_sms() {
    int dev = 0, sms = 148;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    return sms > 0 ? sms : 148;
}

template <bool GATED, int ACT, class T, int ROWS>
int launch_rows(RowsArgs& args, cudaStream_t s) {
    constexpr int kStage = (GATED ? 2 : 1) * kWeightBytes + ROWS * 128;
    constexpr int kPart = (GATED ? 2 : 1) * ROWS * kColumns * 4;
    const int tiles = (args.N + kColumns - 1) / kColumns, sms = rows_sms();
    int split = 1;
    // as many CTAs as two to an SM, and more where a CTA's part were longer than a run may be
    while (split < 8 && 2 * split <= args.nkb &&
           (2 * split * tiles <= 2 * sms || args.nkb > split * (kFfRun / kSumStep)))
        split *= 2;
    const int per = (args.nkb + split - 1) / split;
    // two CTAs to an SM, or with fewer CTAs than SMs one that holds more of its weights
    // before h arrives
    const int ring = (!GATED && split * tiles <= sms ? 200 : 110) * 1024;
    args.stages = std::min(std::min(std::max(ring / kStage, 2), kRowsMaxStages), per);
    // TMEM holds four CTAs (128 columns at most), which 56 KB of shared memory each ensure;
    // with 64 rows' short rings (two stages) a third CTA took 2 us more than two
    constexpr int kLeast = (ROWS > 32 ? 104 : 56) * 1024;
    const int smem = std::max({args.stages * kStage, split > 1 ? kPart : 0, kLeast}) + 1024;
    auto kernel = ff_rows_kernel<GATED, ACT, T, ROWS>;
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    const uint64_t bit = dev < 64 ? uint64_t{1} << dev : 0;
    if (e == cudaSuccess && !(done.load(std::memory_order_acquire) & bit)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 202 * 1024);
        if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
    }
    if (e != cudaSuccess) return cuda_status(e, "gated_ff shared memory");
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {static_cast<unsigned>(split), 1, 1};
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(split, tiles);
    cfg.blockDim = dim3(kRowsThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = GATED ? 1 : 2;
    return cuda_status(cudaLaunchKernelEx(&cfg, kernel, args), "gated_ff rows");
}

template <bool GATED, int ACT, class T>
int launch_rows_n(RowsArgs& a, cudaStream_t s) {
    if (a.M <= 16) return launch_rows<GATED, ACT, T, 16>(a, s);
    if (a.M <= 32) return launch_rows<GATED, ACT, T, 32>(a, s);
    return launch_rows<GATED, ACT, T, 64>(a, s);
}

template <class T>
int launch_rows_act(bool gated, int act, RowsArgs& a, cudaStream_t s) {
    if (!gated) return launch_rows_n<false, ZG_ACT_RELU, T>(a, s);
    switch (act) {
        case ZG_ACT_SILU: return launch_rows_n<true, ZG_ACT_SILU, T>(a, s);
        case ZG_ACT_GELU: return launch_rows_n<true, ZG_ACT_GELU, T>(a, s);
        case ZG_ACT_GELU_TANH: return launch_rows_n<true, ZG_ACT_GELU_TANH, T>(a, s);
        default: return launch_rows_n<true, ZG_ACT_RELU, T>(a, s);
    }
}

}  // namespace

int ff_rows(uint32_t dtype, bool gated, int act, const FfProduct& f, cudaStream_t s) {
    RowsArgs args;
    std::memset(&args, 0, sizeof(args));
    args.c = f.c, args.ldc = f.ldc, args.pre_g = f.pre_g, args.pre_u = f.pre_u;
    args.vec = f.ldc % 4 == 0 && (reinterpret_cast<uintptr_t>(f.c) & 7) == 0 &&
               (!f.pre_g || f.N % 4 == 0);
    args.M = f.M, args.N = f.N, args.nkb = (f.k[0] + kSumStep - 1) / kSumStep;
    const int rows = f.M <= 16 ? 16 : f.M <= 32 ? 32 : 64;
    int rc = status_word(&args.status);
    for (int w = 0; w < (gated ? 2 : 1) && !rc; ++w)
        rc = encode_16bit_map(&args.w[w], dtype, f.b[w].p, f.N, f.k[0], f.b[w].ld, 64, kSumStep);
    if (!rc) rc = encode_16bit_map(&args.x, dtype, f.a[0].p, f.k[0], f.M, f.a[0].ld, 64, rows);
    if (rc) return rc;
    return dtype == ZG_DTYPE_BF16 ? launch_rows_act<__nv_bfloat16>(gated, act, args, s)
                                  : launch_rows_act<__half>(gated, act, args, s);
}

}  // namespace zg
