// gated_ff_pair.cuh - what the tensor-core kernels of the gated feed-forward block
// share (gated_ff_tc.cu for 16-bit tensors, gated_ff_f32.cu): the order of the
// tiles, the epilogues' way to memory, and split sums.
#pragma once

#include <algorithm>
#include <atomic>

#include "gated_ff.cuh"

namespace zg {
namespace {

constexpr int kMaxProblems = 3;
constexpr int kPairsSold = 74;  // SM pairs of a B200: what split sums are dealt out for

// Grouped raster, as sgemm_tc.cu's (eight row tiles before the next column).
__device__ __forceinline__ void raster(int tile, int mt, int nt, int& mi, int& ni) {
    const int group = tile / (8 * nt), first = group * 8;
    const int gm = min(mt - first, 8), r = tile - group * 8 * nt;
    mi = first + r % gm;
    ni = r / gm;
}

// An epilogue warp turns blocks of 32 x 32 between "a row per lane" (TMEM) and
// "neighbours along a row" (memory) through shared memory of its own, with rows of
// 144 bytes (f32) or 80 (16 bits): an odd number of 16-byte pieces, so that accesses
// of either kind meet no bank twice.
template <class T> constexpr int kPitch = sizeof(T) * 32 + 16;

// Stores a warp's 32 x 32 block of T, row `lane` in the words of v, at `dst` (its
// row 0, column 0); `rows` and `cols` of it lie inside the matrix.  vec: 16-byte
// pieces of rows; otherwise (odd pitch or base) neighbours side by side.
template <class T>
__device__ __forceinline__ void store_block(T* dst, int64_t ld, int rows, int cols, bool vec,
                                            const uint32_t (&v)[8 * sizeof(T)], uint8_t* turn,
                                            int lane) {
    constexpr int kPer = 16 / sizeof(T), kPieces = 32 / kPer, kTurnPitch = kPitch<T>;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kPieces; ++i)
        *reinterpret_cast<uint4*>(turn + lane * kTurnPitch + i * 16) =
            make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    __syncwarp();
    if (vec) {
#pragma unroll
        for (int j = 0; j < kPieces; ++j) {
            const int r = (j * 32 + lane) / kPieces, piece = lane % kPieces;
            if (r < rows && piece * kPer < cols)
                *reinterpret_cast<uint4*>(dst + r * ld + piece * kPer) =
                    *reinterpret_cast<const uint4*>(turn + r * kTurnPitch + piece * 16);
        }
    } else if (sizeof(T) == 2) {
        // two rows a turn, 16 lanes each, in aligned words of two elements: 2 l and
        // 2 l + 1, or in a row that starts inside a word one further, and then
        // elements 0 and 31 alone
        const int l = lane & 15;
        for (int r = lane >> 4; r < rows; r += 2) {
            T* to = dst + r * ld;
            const T* from = reinterpret_cast<const T*>(turn + r * kTurnPitch);
            const int odd = (reinterpret_cast<uintptr_t>(to) >> 1) & 1, e = 2 * l + odd;
            if (e + 1 < min(cols, 32)) {
                T pair[2] = {from[e], from[e + 1]};
                uint32_t word;
                __builtin_memcpy(&word, pair, 4);
                *reinterpret_cast<uint32_t*>(to + e) = word;
            } else if (e < cols) {
                to[e] = from[e];
            }
            if (odd && l == 0 && cols > 0) to[0] = from[0];
        }
    } else if (lane < cols) {
        for (int r = 0; r < rows; ++r)
            dst[r * ld + lane] = reinterpret_cast<const T*>(turn + r * kTurnPitch)[lane];
    }
}

// Adds up the parts of split sums, in order, and rounds: four elements a thread.
struct SumArgs {
    struct {
        const float* part;
        void* c;
        int64_t plane, groups;  // groups of this matrix and those before it
        int N, ldp;
    } m[kMaxProblems];
    int count, splits;
};
template <class T>
__global__ void __launch_bounds__(256) ff_sum_kernel(const __grid_constant__ SumArgs a) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int64_t step = static_cast<int64_t>(gridDim.x) * 256;
    for (int64_t g = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
         g < a.m[a.count - 1].groups; g += step) {
        int i = 0;
        while (g >= a.m[i].groups) ++i;
        const auto& m = a.m[i];
        const int64_t at = (g - (i ? a.m[i - 1].groups : 0)) * 4;
        const int64_t row = at / m.ldp;
        const int col = static_cast<int>(at - row * m.ldp);
        float4 sum = __ldcs(reinterpret_cast<const float4*>(m.part + at));
        for (int s = 1; s < a.splits; ++s) {
            const float4 x = __ldcs(reinterpret_cast<const float4*>(m.part + s * m.plane + at));
            sum.x += x.x, sum.y += x.y, sum.z += x.z, sum.w += x.w;
        }
        T* c = static_cast<T*>(m.c) + row * m.N + col;
        const float v[4] = {sum.x, sum.y, sum.z, sum.w};
        if (m.N % 4 == 0 && (reinterpret_cast<uintptr_t>(m.c) & (4 * sizeof(T) - 1)) == 0) {
            struct alignas(4 * sizeof(T)) Four {
                T t[4];
            } q;
#pragma unroll
            for (int e = 0; e < 4; ++e) q.t[e] = FfElem<T>::put(v[e]);
            *reinterpret_cast<Four*>(c) = q;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (col + e < m.N) c[e] = FfElem<T>::put(v[e]);
        }
    }
}

// ---- host ----------------------------------------------------------------------
inline int sm_pairs() {
    int dev = 0, sms = 148;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    return std::max((sms > 0 ? sms : 148) / 2, 1);
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Into how many parts products of few 256 x 256 tiles split their sums, stages of
// `step`: as many as the SM pairs take, sixteen at most, four stages each at least.
inline int splits_of(const FfProduct* products, int count, int step) {
    int64_t tiles = 0;
    int nkb = 1 << 30;
    for (int i = 0; i < count; ++i) {
        const FfProduct& f = products[i];
        tiles += static_cast<int64_t>((f.M + 255) / 256) * ((f.N + 255) / 256);
        nkb = std::min(nkb, (f.k[0] + step - 1) / step + (f.k[1] + step - 1) / step);
    }
    return static_cast<int>(
        std::max<int64_t>(1, std::min<int64_t>({16, kPairsSold / std::max<int64_t>(tiles, 1), nkb / 4})));
}
inline uint64_t split_bytes(const FfProduct* products, int count, int splits) {
    if (splits == 1) return 0;
    uint64_t elems = 0;
    for (int i = 0; i < count; ++i)
        elems += static_cast<uint64_t>(products[i].M) * ((products[i].N + 3) / 4 * 4);
    return elems * splits * 4;
}

template <class Kernel>
cudaError_t allow_smem(Kernel* kernel, int bytes, std::atomic<uint64_t>& done) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    const uint64_t bit = dev < 64 ? uint64_t{1} << dev : 0;
    if (e != cudaSuccess || (done.load(std::memory_order_acquire) & bit)) return e;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
    return e;
}

}  // namespace
}  // namespace zg
