// gated_ff_pair.cuh - what the tensor-core kernels of the gated feed-forward block
// share (gated_ff_tc.cu for 16-bit tensors, gated_ff_f32.cu): the order of the
// tiles, the epilogues' way to memory, and split sums.
#pragma once

#include <algorithm>
#include <atomic>

#include "gated_ff.cuh"

namespace zg {
namespace {

constexpr int kMaxProblems = 4;  // of a launch: dx and the three weights' gradients
constexpr int kPairsSold = 74;  // SM pairs of a B200: what split sums are dealt out for

// Grouped raster, as sgemm_tc.cu's (eight row tiles before the next column).
__device__ __forceinline__ void raster(int tile, int mt, int nt, int& mi, int& ni) {
    const int group = tile / (8 * nt), first = group * 8;
    const int gm = min(mt - first, 8), r = tile - group * 8 * nt;
    mi = first + r % gm;
    ni = r / gm;
}

// Which unit of work an SM pair takes in its turn j: its own remainder of the units,
// unless the first `longs` of them take much longer than the others (dx's sum is 2 f
// long, the weights' gradients' m).  Then the long ones are dealt out first, and the
// pairs that got one less take `extra` short ones before the rest go around.
struct Deal {
    int units, pairs, longs, extra;
};
__device__ __forceinline__ int unit_at(const Deal& d, int pair, int j) {
    const int over = d.longs % d.pairs;  // pairs with one long unit more
    const int own = d.longs / d.pairs + (pair < over);
    if (j < own) return pair + j * d.pairs;
    j -= own;
    int rest = d.longs;
    if (over) {
        if (pair >= over) {
            if (j < d.extra) return rest + (pair - over) * d.extra + j;
            j -= d.extra;
        }
        rest += d.extra * (d.pairs - over);
    }
    const int u = rest + (pair - over + d.pairs) % d.pairs + j * d.pairs;
    return u < d.units ? u : -1;
}

// An epilogue warp turns blocks of 32 x 32 between "a row per lane" (TMEM) and
// "neighbours along a row" (memory) through shared memory of its own, with rows of
// 144 bytes (f32) or 80 (16 bits): an odd number of 16-byte pieces, so that accesses
// of either kind meet no bank twice.
template <class T> constexpr int kPitch = sizeof(T) * 32 + 16;

// Stores a warp's block of 32 rows and COLS columns of T from shared memory, rows `pitch`
// bytes apart and their 16-byte pieces `step`, to `dst` (its row 0, column 0); `rows`
// rows and `cols` columns of it lie inside the matrix.  vec: 16-byte pieces of rows;
// otherwise (odd pitch or base) neighbours side by side.
template <class T, int COLS>
__device__ __forceinline__ void flush_block(T* dst, int64_t ld, int rows, int cols, bool vec,
                                            const uint8_t* turn, int pitch, int step, int lane) {
    constexpr int kPer = 16 / sizeof(T), kPieces = COLS / kPer;
    if (vec) {
#pragma unroll 4
        for (int j = 0; j < kPieces; ++j) {
            const int r = (j * 32 + lane) / kPieces, piece = lane % kPieces;
            if (r < rows && piece * kPer < cols)
                *reinterpret_cast<uint4*>(dst + r * ld + piece * kPer) =
                    *reinterpret_cast<const uint4*>(turn + r * pitch + piece * step);
        }
    } else if constexpr (sizeof(T) == 2) {
        // COLS / 2 lanes to a row, in aligned words of two elements: 2 l and 2 l + 1, or in
        // a row that starts inside a word one further, and then the first and the last
        // element alone
        constexpr int kLanes = COLS / 2;
        const int l = lane % kLanes, most = min(cols, COLS);
        auto word = [&](int r, int w) {
            return *reinterpret_cast<const uint32_t*>(turn + r * pitch + w / 4 * step + w % 4 * 4);
        };
        auto low = [](uint32_t w) {
            T t;
            __builtin_memcpy(&t, &w, 2);
            return t;
        };
#pragma unroll 4
        for (int r = lane / kLanes; r < rows; r += 32 / kLanes) {
            T* to = dst + r * ld;
            const int odd = (reinterpret_cast<uintptr_t>(to) >> 1) & 1, e = 2 * l + odd;
            const uint32_t first = word(r, l);
            // the word after a row's last is its padding, read and not stored
            const uint32_t pair = odd ? __funnelshift_r(first, word(r, l + 1), 16) : first;
            if (e + 1 < most) *reinterpret_cast<uint32_t*>(to + e) = pair;
            else if (e < most) to[e] = low(pair);
            if (odd && l == 0 && cols > 0) to[0] = low(first);
        }
    } else if (lane < cols) {
#pragma unroll 4
        for (int r = 0; r < rows; ++r)
            dst[r * ld + lane] = *reinterpret_cast<const T*>(turn + r * pitch + lane * 4);
    }
}

// Adds up the parts of split sums, in order, and rounds: four elements a thread.  The
// parts are mostly still in L2 (4-6 us for 2 M values in four parts).
struct SumArgs {
    struct {
        const float* part;
        void* c;
        int64_t plane, groups;  // groups of this matrix and those before it
        int N, ldp, splits;
    } m[kMaxProblems];
    int count;
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
        for (int s = 1; s < m.splits; ++s) {
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

// Into how many parts each product of a launch splits its sum, in stages of `step`:
// as many as leave no unit with more than an SM pair's share of all the stages, but
// sixteen at most, and four stages to a part at least.
inline void splits_of(const FfProduct* products, int count, int step, int (&splits)[kMaxProblems]) {
    int64_t tiles[kMaxProblems], nkb[kMaxProblems], all = 0;
    for (int i = 0; i < count; ++i) {
        const FfProduct& f = products[i];
        tiles[i] = static_cast<int64_t>((f.M + 255) / 256) * ((f.N + 255) / 256);
        nkb[i] = (f.k[0] + step - 1) / step + (f.k[1] + step - 1) / step;
        all += tiles[i] * nkb[i];
    }
    const int64_t share = std::max<int64_t>((all + kPairsSold - 1) / kPairsSold, 1);
    for (int i = 0; i < count; ++i)
        splits[i] = static_cast<int>(std::max<int64_t>(
            1, std::min<int64_t>({16, (nkb[i] + share / 2) / share, nkb[i] / 4})));
}
inline uint64_t split_bytes(const FfProduct* products, int count, int step) {
    int splits[kMaxProblems];
    splits_of(products, count, step, splits);
    uint64_t bytes = 0;
    for (int i = 0; i < count; ++i)
        if (splits[i] > 1)
            bytes += static_cast<uint64_t>(products[i].M) * ((products[i].N + 3) / 4 * 4) *
                     splits[i] * 4;
    return bytes;
}
// Notes a split product for ff_sum_kernel; its parts begin at `parts`, which moves on.
inline void add_parts(SumArgs& sum, const FfProduct& f, int splits, float*& parts) {
    const int ldp = (f.N + 3) / 4 * 4;
    const int64_t plane = static_cast<int64_t>(f.M) * ldp;
    const int64_t before = sum.count ? sum.m[sum.count - 1].groups : 0;
    sum.m[sum.count++] = {parts, f.c, plane, before + plane / 4, f.N, ldp, splits};
    parts += plane * splits;
}
template <class T>
int launch_sum(const SumArgs& sum, cudaStream_t s) {
    if (!sum.count) return ZG_OK;
    const int64_t groups = sum.m[sum.count - 1].groups;
    return launch_dependent("gated_ff sum", ff_sum_kernel<T>,
                            static_cast<unsigned>(std::min<int64_t>((groups + 255) / 256, 148 * 16)),
                            256, 0, s, sum);
}

// The deal for `units`, of which the first `longs` take `ratio` times the others' time.
inline Deal deal_of(int units, int pairs, int longs, int ratio) {
    Deal d{units, std::min(units, pairs), 0, 0};
    if (ratio >= 2 && longs < units) {
        d.longs = longs;
        const int less = d.pairs - longs % d.pairs;
        d.extra = std::min(ratio, (units - longs) / less);
    }
    return d;
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
