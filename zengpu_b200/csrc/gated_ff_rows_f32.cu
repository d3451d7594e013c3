// gated_ff_rows_f32.cu - the forward products of the gated feed-forward block for
// few rows of f32 tensors, on the CUDA cores: every weight is read once, as it lies
// (any size, any pitch), where the tensor-core modes would first write it out again
// as operand planes.  Every mode takes this form for up to kFfRowsF32 rows; its sums
// are plain f32 FMAs.
//
// A CTA takes 128 columns of W (of Wg and of Wu for the gated product) and a part of
// the sum; the CTAs of a cluster share the columns and split the sum.  Weights and
// the piece of x come through a ring of stages of 32 of the sum (cp.async, 16 bytes
// where the pitch allows it, else 4).  A lane holds four columns; the eight warps are
// dealt out to groups of eight rows (of 1, 2 or 4, up to that many) and, where those are
// fewer, to parts of the stage: 8 rows x 4 columns x 2 products a thread, 64 FMAs for four 16-byte reads of shared
// memory (two of them the eight rows' x, four of the sum at a time).  Partial results meet in shared memory, across the
// cluster as in gated_ff_rows.cu, in a fixed order.
//
// Up to 4 rows the weights' 4 bytes each bound it: 4096 -> 12288 takes 111 us for one token
// (604 MB, 5.5 TB/s) and 125 for 4.  Beyond, 8 rows take 165, 16 rows 234 and 32 rows 362.
// The f32 pipe is part of that (8 rows a weight are 16 cycles of an SM's 128 lanes for 1 KB
// of weights, which HBM delivers in 44; 32 rows are 64 cycles, 135 us); the rest is
// latency, a barrier of the CTA for every 32 of the sum, and unequal dealing: the split of
// the sum is a power of two, so that h's 96 tiles are 192 CTAs on 148 SMs.
// From 33 rows on the tensor cores are faster (2048 -> 6144: 217 us at 33 rows, 64 rows
// here took 230).
#include <algorithm>
#include <atomic>
#include <cstdint>

#include "gated_ff.cuh"

namespace zg {
namespace {

constexpr int kRThreads = 256, kRWarps = 8, kRCols = 128, kRStep = 32;
constexpr int kXPitch = kRStep + 4;  // floats of a row of x in a stage
// About 100 KB of weights in flight, two CTAs to an SM.
__host__ __device__ constexpr int ring_stages(int mats) { return mats == 2 ? 3 : 5; }

struct RowsF32Args {
    const float* x;
    const float* w[2];
    float* c;
    float* pre_g;
    float* pre_u;
    int64_t ldx, ldw, ldc;
    int M, N, K;
    int vec_w, vec_x;  // 16-byte aligned rows
};

// Copies the first `count` of four floats, zeros after them.
__device__ __forceinline__ void copy16(uint32_t to, const float* from, int count) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from),
                 "r"(4 * count)
                 : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const float* from, bool in) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from),
                 "r"(in ? 4 : 0)
                 : "memory");
}
__device__ __forceinline__ float4 ld_rank(uint32_t mine, uint32_t rank) {
    float4 v;
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(mine), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(a)
                 : "memory");
    return v;
}

// ROWS: 1, 2, 4, 8, 16 or 32.
template <bool GATED, int ACT, int ROWS>
__global__ void __launch_bounds__(kRThreads, 2)
    ff_rows_f32_kernel(const __grid_constant__ RowsF32Args a) {
    constexpr int kMats = GATED ? 2 : 1;
    constexpr int kOwn = ROWS < 8 ? ROWS : 8;  // rows of a warp
    constexpr int kRowGroups = ROWS / kOwn, kSumGroups = kRWarps / kRowGroups;
    constexpr int kStages = ring_stages(kMats);
    constexpr int kWFloats = kMats * kRStep * kRCols, kStageFloats = kWFloats + ROWS * kXPitch;
    extern __shared__ float4 ring4[];
    float* ring = reinterpret_cast<float*>(ring4);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = gridDim.x, rank = blockIdx.x;
    const int n0 = blockIdx.y * kRCols;
    const int steps = (a.K + kRStep - 1) / kRStep;
    const int s0 = static_cast<int>(static_cast<int64_t>(steps) * rank / split);
    const int s1 = static_cast<int>(static_cast<int64_t>(steps) * (rank + 1) / split);
    const int row0 = warp % kRowGroups * kOwn, part = warp / kRowGroups;

    auto load = [&](int step) {
        if (step < s1) {
            const uint32_t st = smem_u32(ring + (step - s0) % kStages * kStageFloats);
            const int k0 = step * kRStep;
#pragma unroll
            for (int w = 0; w < kMats; ++w) {
                const float* from = w ? a.w[1] : a.w[0];
                const uint32_t to = st + w * kRStep * kRCols * 4;
                if (a.vec_w) {
#pragma unroll
                    for (int i = 0; i < kRStep * kRCols / 4 / kRThreads; ++i) {
                        const int k = i * (kRThreads * 4 / kRCols) + threadIdx.x / (kRCols / 4);
                        const int c = threadIdx.x % (kRCols / 4) * 4;
                        const bool in = k0 + k < a.K && n0 + c < a.N;
                        copy16(to + (k * kRCols + c) * 4,
                               in ? from + (k0 + k) * a.ldw + n0 + c : from, in ? 4 : 0);
                    }
                } else {
#pragma unroll 4
                    for (int i = 0; i < kRStep * kRCols / kRThreads; ++i) {
                        const int k = i * (kRThreads / kRCols) + threadIdx.x / kRCols;
                        const int c = threadIdx.x % kRCols;
                        const bool in = k0 + k < a.K && n0 + c < a.N;
                        copy4(to + (k * kRCols + c) * 4,
                              in ? from + (k0 + k) * a.ldw + n0 + c : from, in);
                    }
                }
            }
            const uint32_t to = st + kWFloats * 4;
            if (a.vec_x) {
                for (int j = threadIdx.x; j < ROWS * (kRStep / 4); j += kRThreads) {
                    const int r = j / (kRStep / 4), k = j % (kRStep / 4) * 4;
                    // a row of h goes on past the sum, with what scratch memory held
                    const int in = r < a.M ? max(min(a.K - (k0 + k), 4), 0) : 0;
                    copy16(to + (r * kXPitch + k) * 4, in ? a.x + r * a.ldx + k0 + k : a.x, in);
                }
            } else {
                for (int j = threadIdx.x; j < ROWS * kRStep; j += kRThreads) {
                    const int r = j / kRStep, k = j % kRStep;
                    const bool in = k0 + k < a.K && r < a.M;
                    copy4(to + (r * kXPitch + k) * 4, in ? a.x + r * a.ldx + k0 + k : a.x, in);
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };

    float acc[kMats][kOwn][4] = {};
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (int i = 0; i < kStages - 1; ++i) load(s0 + i);
    for (int step = s0; step < s1; ++step) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
        __syncthreads();  // the stage has landed, and the one before it is free
        load(step + kStages - 1);
        const float* st = ring + (step - s0) % kStages * kStageFloats;
#pragma unroll
        for (int i = 0; i < kRStep / 4 / kSumGroups; ++i) {
            const int k = (part + i * kSumGroups) * 4;
            float x[kOwn][4];
#pragma unroll
            for (int r = 0; r < kOwn; ++r) {
                const float4 v =
                    *reinterpret_cast<const float4*>(st + kWFloats + (row0 + r) * kXPitch + k);
                x[r][0] = v.x, x[r][1] = v.y, x[r][2] = v.z, x[r][3] = v.w;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int w = 0; w < kMats; ++w) {
                    const float4 v = *reinterpret_cast<const float4*>(
                        st + (w * kRStep + k + e) * kRCols + lane * 4);
#pragma unroll
                    for (int r = 0; r < kOwn; ++r) {
                        acc[w][r][0] = fmaf(x[r][e], v.x, acc[w][r][0]);
                        acc[w][r][1] = fmaf(x[r][e], v.y, acc[w][r][1]);
                        acc[w][r][2] = fmaf(x[r][e], v.z, acc[w][r][2]);
                        acc[w][r][3] = fmaf(x[r][e], v.w, acc[w][r][3]);
                    }
                }
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    // partial results [sum group][product][row][column] take the ring's place
#pragma unroll
    for (int w = 0; w < kMats; ++w)
#pragma unroll
        for (int r = 0; r < kOwn; ++r)
            *reinterpret_cast<float4*>(ring + ((part * kMats + w) * ROWS + row0 + r) * kRCols +
                                       lane * 4) =
                make_float4(acc[w][r][0], acc[w][r][1], acc[w][r][2], acc[w][r][3]);
    if (split > 1) cluster_sync();
    else __syncthreads();
    const uint32_t at = smem_u32(ring) + lane * 16;
    for (int row = rank + split * warp; row < a.M; row += split * kRWarps) {
        float4 g = make_float4(0.0f, 0.0f, 0.0f, 0.0f), u = g;
        for (int p = 0; p < split; ++p)
#pragma unroll
            for (int q = 0; q < kSumGroups; ++q) {
                const float4 v = ld_rank(at + (q * kMats * ROWS + row) * kRCols * 4, p);
                g.x += v.x, g.y += v.y, g.z += v.z, g.w += v.w;
                if (GATED) {
                    const float4 z = ld_rank(at + ((q * kMats + 1) * ROWS + row) * kRCols * 4, p);
                    u.x += z.x, u.y += z.y, u.z += z.z, u.w += z.w;
                }
            }
        const float gs[4] = {g.x, g.y, g.z, g.w}, us[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int col = n0 + lane * 4 + e;
            if (col >= a.N) break;
            if (GATED && a.pre_g) {
                const int64_t pre = static_cast<int64_t>(row) * a.N + col;
                a.pre_g[pre] = gs[e];
                a.pre_u[pre] = us[e];
            }
            a.c[row * a.ldc + col] = GATED ? activate<ACT, false>(gs[e]).a * us[e] : gs[e];
        }
    }
    if (split > 1) cluster_sync();  // nobody leaves while its memory is read
}

template <bool GATED, int ACT, int ROWS>
int launch_rows(const RowsF32Args& a, cudaStream_t s) {
    constexpr int kMats = GATED ? 2 : 1;
    constexpr int kSmem = std::max(ring_stages(kMats) * (kMats * kRStep * kRCols + ROWS * kXPitch),
                                   kMats * std::min(ROWS, 8) * kRWarps * kRCols) * 4;
    const int tiles = (a.N + kRCols - 1) / kRCols, steps = (a.K + kRStep - 1) / kRStep;
    int split = 1;
    // two CTAs of an SM, a few stages for each part of the sum at least
    while (split < 8 && 2 * split * tiles <= 2 * 148 && 6 * split <= steps) split *= 2;
    auto kernel = ff_rows_f32_kernel<GATED, ACT, ROWS>;
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    const uint64_t bit = dev < 64 ? uint64_t{1} << dev : 0;
    if (e == cudaSuccess && !(done.load(std::memory_order_acquire) & bit)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
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
    cfg.blockDim = dim3(kRThreads);
    cfg.dynamicSmemBytes = kSmem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cuda_status(cudaLaunchKernelEx(&cfg, kernel, a), "gated_ff rows");
}

template <bool GATED, int ACT>
int launch_rows_n(const RowsF32Args& a, cudaStream_t s) {
    if (a.M <= 1) return launch_rows<GATED, ACT, 1>(a, s);
    if (a.M <= 2) return launch_rows<GATED, ACT, 2>(a, s);
    if (a.M <= 4) return launch_rows<GATED, ACT, 4>(a, s);
    if (a.M <= 8) return launch_rows<GATED, ACT, 8>(a, s);
    if (a.M <= 16) return launch_rows<GATED, ACT, 16>(a, s);
    return launch_rows<GATED, ACT, 32>(a, s);
}

}  // namespace

int ff_rows_f32(bool gated, int act, const FfProduct& f, cudaStream_t s) {
    RowsF32Args a{};
    a.x = static_cast<const float*>(f.a[0].p), a.ldx = f.a[0].ld;
    a.w[0] = static_cast<const float*>(f.b[0].p), a.w[1] = static_cast<const float*>(f.b[1].p);
    a.ldw = f.b[0].ld;
    a.c = static_cast<float*>(f.c), a.ldc = f.ldc;
    a.pre_g = f.pre_g, a.pre_u = f.pre_u;
    a.M = f.M, a.N = f.N, a.K = f.k[0];
    a.vec_x = a.ldx % 4 == 0 && (reinterpret_cast<uintptr_t>(a.x) & 15) == 0;
    a.vec_w = a.ldw % 4 == 0 &&
            ((reinterpret_cast<uintptr_t>(a.w[0]) | reinterpret_cast<uintptr_t>(a.w[1])) & 15) == 0;
    if (!gated) return launch_rows_n<false, ZG_ACT_RELU>(a, s);
    switch (act) {
        case ZG_ACT_SILU: return launch_rows_n<true, ZG_ACT_SILU>(a, s);
        case ZG_ACT_GELU: return launch_rows_n<true, ZG_ACT_GELU>(a, s);
        case ZG_ACT_GELU_TANH: return launch_rows_n<true, ZG_ACT_GELU_TANH>(a, s);
        default: return launch_rows_n<true, ZG_ACT_RELU>(a, s);
    }
}

}  // namespace zg
