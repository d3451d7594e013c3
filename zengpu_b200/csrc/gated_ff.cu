// gated_ff.cu - the gated feed-forward block y = (act(x Wg) * (x Wu)) Wd and its
// backward pass (formulas and roundings: gated_ff.cuh), beside the fused GEMM +
// bias + ReLU.  The reference has no gated layer and no backward pass; its
// op_graph_lower chain (examples/op_graph_lower.rs:39-68) is the ungated,
// forward-only form.
#include <algorithm>
#include <cstdint>
#include <initializer_list>

#include "gated_ff.cuh"
#include "zg_gemm_internal.h"

namespace zg {
namespace {

// ---- CUDA-core product ------------------------------------------------------------
// The SIMT_FP32 mode: 64 x 64 of D per CTA, 4 x 4 per thread (twice for the gated
// pair), operands of any layout through shared memory 16 of the sum at a time.  f32
// throughout; bound by the f32 pipe, of which it reaches a quarter (18 TFLOP/s on a
// 2048 x 1024 x 4096 training pass): the mode is the accuracy anchor, not a fast path.
constexpr int kTile = 64, kStep = 16;

__device__ __forceinline__ void load_panel(float (&sh)[kStep][kTile + 4], const FfOperand& o,
                                           int rows, int r0, int k, int i0) {
    // the thread order follows the operand's contiguous direction
    for (int e = threadIdx.x; e < kTile * kStep; e += 256) {
        const int r = o.mn ? e % kTile : e / kStep, i = o.mn ? e / kTile : e % kStep;
        float v = 0.0f;
        if (r0 + r < rows && i0 + i < k)
            v = static_cast<const float*>(
                o.p)[o.mn ? (i0 + i) * o.ld + r0 + r : (r0 + r) * o.ld + i0 + i];
        sh[i][r] = v;
    }
}

template <int EPI, int ACT>
__global__ void __launch_bounds__(256) ff_simt_kernel(const FfProduct p) {
    __shared__ float sa[kStep][kTile + 4], sb[2][kStep][kTile + 4];
    const int m0 = blockIdx.x * kTile, n0 = blockIdx.y * kTile;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    float acc[2][4][4] = {};
    for (int seg = 0; seg < (EPI == kFfStore ? 2 : 1); ++seg) {
        for (int i0 = 0; i0 < p.k[seg]; i0 += kStep) {
            load_panel(sa, p.a[seg], p.M, m0, p.k[seg], i0);
            load_panel(sb[0], p.b[seg], p.N, n0, p.k[seg], i0);
            if (EPI == kFfGated) load_panel(sb[1], p.b[1], p.N, n0, p.k[0], i0);
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kStep; ++i) {
                float a[4], b[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) a[r] = sa[i][ty * 4 + r];
#pragma unroll
                for (int w = 0; w < (EPI == kFfGated ? 2 : 1); ++w) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) b[c] = sb[w][i][tx * 4 + c];
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int c = 0; c < 4; ++c) acc[w][r][c] = fmaf(a[r], b[c], acc[w][r][c]);
                }
            }
            __syncthreads();
        }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int64_t row = m0 + ty * 4 + r;
        if (row >= p.M) break;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int col = n0 + tx * 4 + c;
            if (col >= p.N) break;
            const int64_t at = row * p.ldc + col, pre = row * p.N + col;
            const float x = acc[0][r][c];
            if (EPI == kFfStore) static_cast<float*>(p.c)[at] = x;
            if (EPI == kFfGated) {
                const float u = acc[1][r][c];
                static_cast<float*>(p.c)[at] = activate<ACT, false>(x).a * u;
                if (p.pre_g) {
                    p.pre_g[pre] = x;
                    p.pre_u[pre] = u;
                }
            }
            if (EPI == kFfSlope) {
                const float u = p.pre_u[pre];
                const ActValue v = activate<ACT, false>(p.pre_g[pre]);
                static_cast<float*>(p.c)[at] = x * u * v.slope;
                static_cast<float*>(p.c2)[at] = x * v.a;
                static_cast<float*>(p.c3)[at] = v.a * u;
            }
        }
    }
}

template <int EPI>
int launch_simt(int act, const FfProduct& p, cudaStream_t s) {
    const dim3 grid((p.M + kTile - 1) / kTile, (p.N + kTile - 1) / kTile);
    if (grid.y > 65535u) return set_error(ZG_ERR_DISPATCH, "gated_ff: too many columns");
    if constexpr (EPI == kFfStore) {
        ff_simt_kernel<EPI, ZG_ACT_RELU><<<grid, 256, 0, s>>>(p);
    } else {
        switch (act) {
            case ZG_ACT_SILU: ff_simt_kernel<EPI, ZG_ACT_SILU><<<grid, 256, 0, s>>>(p); break;
            case ZG_ACT_GELU: ff_simt_kernel<EPI, ZG_ACT_GELU><<<grid, 256, 0, s>>>(p); break;
            case ZG_ACT_GELU_TANH:
                ff_simt_kernel<EPI, ZG_ACT_GELU_TANH><<<grid, 256, 0, s>>>(p);
                break;
            default: ff_simt_kernel<EPI, ZG_ACT_RELU><<<grid, 256, 0, s>>>(p); break;
        }
    }
    return cuda_status(cudaGetLastError(), "gated_ff");
}

}  // namespace

int ff_simt(FfEpilogue epi, int act, const FfProduct& p, cudaStream_t s) {
    switch (epi) {
        case kFfStore: return launch_simt<kFfStore>(act, p, s);
        case kFfGated: return launch_simt<kFfGated>(act, p, s);
        default: return launch_simt<kFfSlope>(act, p, s);
    }
}

namespace {

uint64_t round_up(uint64_t x, uint64_t a) { return (x + a - 1) / a * a; }

struct FfCall {
    uint32_t dtype;
    int mode, act;
    int m, k, f, d;
    uint64_t size;  // bytes of an element
    bool backward;
};

// 16-bit rows copied to a pitch that is a multiple of 8 (16 bytes, the tensor
// maps' rule), for sizes that are not: up to five tensors in one launch.  HBM bound:
// 49 us for 139 MB read and as much written (5.7 TB/s).
struct PadCopy {
    const uint16_t* src;
    uint16_t* dst;
    int64_t rows;
    int cols, ld;
};
struct PadCopies {
    PadCopy t[5];
    int64_t first[6];  // first group of eight elements of each tensor
    int count;
};

__global__ void __launch_bounds__(256) pad_rows_kernel(const __grid_constant__ PadCopies c) {
    const int64_t step = static_cast<int64_t>(gridDim.x) * 256;
    for (int64_t g = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; g < c.first[c.count];
         g += step) {
        int i = 0;
        while (g >= c.first[i + 1]) ++i;
        const PadCopy& t = c.t[i];
        const int64_t at = (g - c.first[i]) * 8;
        const int64_t row = at / t.ld;
        const int col = static_cast<int>(at - row * t.ld);
        const uint16_t* src = t.src + row * t.cols + col;
        uint4 q;
        if (col + 8 > t.cols) {
            uint16_t v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = col + e < t.cols ? src[e] : 0;
            __builtin_memcpy(&q, v, 16);
        } else if ((reinterpret_cast<uintptr_t>(src) & 2) == 0) {
            const uint32_t* w = reinterpret_cast<const uint32_t*>(src);
            q = make_uint4(w[0], w[1], w[2], w[3]);
        } else {  // three words inside, an element on either side
            const uint32_t* w = reinterpret_cast<const uint32_t*>(src + 1);
            const uint32_t a = src[0], b = w[0], c = w[1], d = w[2], e = src[7];
            q = make_uint4(a | (b << 16), (b >> 16) | (c << 16), (c >> 16) | (d << 16),
                           (d >> 16) | (e << 16));
        }
        *reinterpret_cast<uint4*>(t.dst + at) = q;
    }
}

void shape_y(const FfCall& c, FfProduct& p) { p.M = c.m, p.N = c.d, p.k[0] = c.f, p.ldc = c.d; }
void shape_grads(const FfCall& c, FfProduct (&p)[4]) {  // dx, dWg, dWu, dWd
    p[0].M = c.m, p[0].N = c.k, p[0].k[0] = p[0].k[1] = c.f, p[0].ldc = c.k;
    for (int i = 1; i < 4; ++i) p[i].k[0] = c.m;
    p[1].M = p[2].M = c.k, p[1].N = p[2].N = c.f, p[1].ldc = p[2].ldc = c.f;
    p[3].M = c.f, p[3].N = c.d, p[3].ldc = c.d;
}

// Workspace: h, then for the backward pass dg and du, [m, f] each; then padded
// copies of the 16-bit inputs that need them.
enum { kX, kWg, kWu, kWd, kDy, kInputs };
struct FfLayout {
    int64_t ld_f;
    uint64_t plane, total;
    bool pad[kInputs];
    uint64_t at[kInputs];
    uint64_t parts;  // of split sums
};
FfLayout ff_layout(const FfCall& c) {
    FfLayout l;
    l.ld_f = static_cast<int64_t>(round_up(c.f, 8));
    l.plane = round_up(static_cast<uint64_t>(c.m) * l.ld_f * c.size, 256);
    l.total = l.plane * (c.backward ? 3 : 1);
    const int rows[kInputs] = {c.m, c.k, c.k, c.f, c.m}, cols[kInputs] = {c.k, c.f, c.f, c.d, c.d};
    for (int i = 0; i < kInputs; ++i) {
        l.pad[i] = c.size == 2 && cols[i] % 8 != 0 && (c.backward || i != kDy);
        l.at[i] = l.total;
        if (l.pad[i]) l.total += round_up(rows[i] * round_up(cols[i], 8) * c.size, 256);
    }
    l.parts = l.total;
    if (c.size == 2) {
        FfProduct y, grads[4];
        shape_y(c, y), shape_grads(c, grads);
        l.total += c.backward ? ff_split_bytes(grads, 4) : ff_split_bytes(&y, 1);
    }
    return l;
}

struct FfInput {
    const void* p;
    int64_t ld;
};

// The inputs as the products read them: where they lie, or padded.
int place_inputs(const FfCall& c, const FfLayout& l, uint8_t* ws, const void* const* src,
                 FfInput* out, cudaStream_t s) {
    const int rows[kInputs] = {c.m, c.k, c.k, c.f, c.m}, cols[kInputs] = {c.k, c.f, c.f, c.d, c.d};
    PadCopies pc;
    pc.count = 0;
    pc.first[0] = 0;
    for (int i = 0; i < kInputs; ++i) {
        out[i] = {src[i], cols[i]};
        if (!l.pad[i]) continue;
        PadCopy& t = pc.t[pc.count];
        t.src = static_cast<const uint16_t*>(src[i]);
        t.dst = reinterpret_cast<uint16_t*>(ws + l.at[i]);
        t.rows = rows[i], t.cols = cols[i], t.ld = static_cast<int>(round_up(cols[i], 8));
        pc.first[pc.count + 1] = pc.first[pc.count] + t.rows * (t.ld / 8);
        ++pc.count;
        out[i] = {t.dst, t.ld};
    }
    if (!pc.count) return ZG_OK;
    const int64_t blocks = (pc.first[pc.count] + 255) / 256;
    pad_rows_kernel<<<static_cast<unsigned>(std::min<int64_t>(blocks, 148 * 16)), 256, 0, s>>>(pc);
    return cuda_status(cudaGetLastError(), "gated_ff padding");
}

// The forward pass of few rows (gated_ff_rows.cu, gated_ff_rows_f32.cu), whose grids
// take 65535 tiles of 128 columns, and whose 16-bit sums eight runs.
bool few_rows(const FfCall& c) {
    return c.m <= (c.size == 2 ? kFfRows : kFfRowsF32) && std::max(c.f, c.d) <= 65535 * 128 &&
           (c.size == 4 || std::max(c.k, c.f) <= 8 * kFfRun);
}
bool f32_tensor(const FfCall& c) { return c.size == 4 && c.mode != ZG_GEMM_SIMT_FP32; }

// ---- f32 on the tensor cores -----------------------------------------------------
// The split-precision GEMMs of sgemm_tc.cu on operand planes (k innermost), with
// elementwise kernels between.  Every operand of the block becomes planes once per
// pass: by rows where it lies along the sum, transposed where it does not.
// dx's two products are one GEMM over [dg | du] and [Wg | Wu], each padded to whole
// k blocks with zeros.

struct Planes {
    FfCall c;
    uint8_t* ws;        // null: only counts
    uint64_t used = 0;
    cudaStream_t s;
    int rc = ZG_OK;

    void* take(uint64_t bytes) {
        void* p = ws ? ws + used : nullptr;
        used += round_up(bytes, 256);
        return p;
    }
    float* matrix(int rows, int cols) {
        return static_cast<float*>(take(static_cast<uint64_t>(rows) * cols * 4));
    }
    // Planes of `rows` rows over k = K, from a [rows, K] matrix or the [K, rows] one
    // whose transpose it is.
    OperandView of(const float* src, int rows, int K, bool transposed) {
        const OperandView v =
            gemm_carve_planes(take(gemm_planes_bytes(c.mode, rows, K)), c.mode, rows, K);
        if (ws && !rc)
            rc = transposed ? gemm_prep_b(c.mode, K, rows, src, rows, v, s)
                            : gemm_prep_rows(c.mode, rows, K, src, K, v, s);
        return v;
    }
    // Two [rows, K] matrices side by side along k.
    OperandView beside(const float* a, const float* b, int rows, int K) {
        OperandView v = gemm_carve_planes(nullptr, c.mode, rows, K), w = v;
        const int64_t one = v.ld;
        v.ld *= 2;
        v.p = take(static_cast<uint64_t>(rows) * v.ld * 4);
        if (ws && !rc) rc = gemm_prep_rows(c.mode, rows, K, a, K, v, s);
        w.ld = v.ld;
        if (ws && !rc) {
            w.p = static_cast<float*>(v.p) + one;
            rc = gemm_prep_rows(c.mode, rows, K, b, K, w, s);
        }
        return v;
    }
    void gemm(const OperandView& a, const OperandView& b, int M, int N, int K, float* out) {
        if (ws && !rc)
            rc = gemm_run({c.mode, a, b}, M, N, K, 1.0f, out, N, nullptr, 0, s);
    }
};

// h = act(g) u; with dh: dg = dh u act'(g) (over dh), du = dh act(g), h.  HBM bound, 12
// and 24 bytes an element (33 and 42 us for 8.4 M).
template <int ACT>
__global__ void __launch_bounds__(256)
    ff_act_kernel(const float* g, const float* u, float* h, int64_t n) {
    const int64_t step = static_cast<int64_t>(gridDim.x) * 256;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += step)
        h[i] = activate<ACT, false>(g[i]).a * u[i];
}
template <int ACT>
__global__ void __launch_bounds__(256)
    ff_slope_kernel(const float* g, const float* u, float* dh_dg, float* du, float* h, int64_t n) {
    const int64_t step = static_cast<int64_t>(gridDim.x) * 256;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += step) {
        const ActValue a = activate<ACT, false>(g[i]);
        const float x = dh_dg[i], y = u[i];
        dh_dg[i] = x * y * a.slope;
        du[i] = x * a.a;
        h[i] = a.a * y;
    }
}

unsigned stream_grid(int64_t n) {
    return static_cast<unsigned>(std::min<int64_t>((n + 255) / 256, 148 * 16));
}

int launch_act(int act, const float* g, const float* u, float* h, int64_t n, cudaStream_t s) {
    const unsigned grid = stream_grid(n);
    switch (act) {
        case ZG_ACT_SILU: ff_act_kernel<ZG_ACT_SILU><<<grid, 256, 0, s>>>(g, u, h, n); break;
        case ZG_ACT_GELU: ff_act_kernel<ZG_ACT_GELU><<<grid, 256, 0, s>>>(g, u, h, n); break;
        case ZG_ACT_GELU_TANH: ff_act_kernel<ZG_ACT_GELU_TANH><<<grid, 256, 0, s>>>(g, u, h, n); break;
        default: ff_act_kernel<ZG_ACT_RELU><<<grid, 256, 0, s>>>(g, u, h, n); break;
    }
    return cuda_status(cudaGetLastError(), "gated_ff activation");
}

int launch_slope(int act, const float* g, const float* u, float* dh, float* du, float* h,
                 int64_t n, cudaStream_t s) {
    const unsigned grid = stream_grid(n);
    switch (act) {
        case ZG_ACT_SILU: ff_slope_kernel<ZG_ACT_SILU><<<grid, 256, 0, s>>>(g, u, dh, du, h, n); break;
        case ZG_ACT_GELU: ff_slope_kernel<ZG_ACT_GELU><<<grid, 256, 0, s>>>(g, u, dh, du, h, n); break;
        case ZG_ACT_GELU_TANH: ff_slope_kernel<ZG_ACT_GELU_TANH><<<grid, 256, 0, s>>>(g, u, dh, du, h, n); break;
        default: ff_slope_kernel<ZG_ACT_RELU><<<grid, 256, 0, s>>>(g, u, dh, du, h, n); break;
    }
    return cuda_status(cudaGetLastError(), "gated_ff activation gradient");
}

struct F32Tensors {
    const float *x, *wg, *wu, *wd, *dy;
    float *pre_g, *pre_u, *y, *dx, *dwg, *dwu, *dwd;
};

// TF32X3 runs on the block's own kernels (gated_ff_f32.cu); the other modes, which
// are chosen for speed over accuracy or for comparison, on sgemm's.
FfOperand operand(const OperandView& v) { return {v.p, v.ld, false}; }

uint64_t tf32x3_forward(const FfCall& c, const F32Tensors& t, uint8_t* ws, cudaStream_t s,
                        int* rc) {
    Planes p{c, ws, 0, s};
    const OperandView x = p.of(t.x, c.m, c.k, false), wg = p.of(t.wg, c.f, c.k, true),
                      wu = p.of(t.wu, c.f, c.k, true), wd = p.of(t.wd, c.d, c.f, true),
                      h = gemm_carve_planes(p.take(gemm_planes_bytes(c.mode, c.m, c.f)), c.mode,
                                            c.m, c.f);
    // counted without pre-activations given: the case that takes more
    float* pre[2] = {ws && t.pre_g ? t.pre_g : p.matrix(c.m, c.f),
                     ws && t.pre_g ? t.pre_u : p.matrix(c.m, c.f)};
    FfProduct gu[2], y;
    for (int i = 0; i < 2; ++i) {
        gu[i].M = c.m, gu[i].N = gu[i].ldc = c.f, gu[i].k[0] = c.k;
        gu[i].a[0] = operand(x), gu[i].b[0] = operand(i ? wu : wg), gu[i].c = pre[i];
    }
    shape_y(c, y);
    y.a[0] = operand(h), y.b[0] = operand(wd), y.c = t.y;
    float* parts = static_cast<float*>(
        p.take(std::max(ff_f32_split_bytes(gu, 2), ff_f32_split_bytes(&y, 1))));
    if (ws && !p.rc) p.rc = ff_f32(gu, 2, parts, s);
    if (ws && !p.rc) p.rc = ff_f32_act(c.act, pre[0], pre[1], c.m, c.f, operand(h), s);
    if (ws && !p.rc) p.rc = ff_f32(&y, 1, parts, s);
    *rc = p.rc;
    return p.used;
}

uint64_t tf32x3_backward(const FfCall& c, const F32Tensors& t, uint8_t* ws, cudaStream_t s,
                         int* rc) {
    Planes p{c, ws, 0, s};
    const OperandView dy = p.of(t.dy, c.m, c.d, false), wd = p.of(t.wd, c.f, c.d, false),
                      w = p.beside(t.wg, t.wu, c.k, c.f), xt = p.of(t.x, c.k, c.m, true),
                      dyt = p.of(t.dy, c.d, c.m, true);
    OperandView dg = gemm_carve_planes(nullptr, c.mode, c.m, c.f), du = dg;
    dg.ld = du.ld = 2 * dg.ld;
    dg.p = p.take(static_cast<uint64_t>(c.m) * dg.ld * 4);
    du.p = static_cast<float*>(dg.p) + (ws ? dg.ld / 2 : 0);
    FfOperand turned[3];  // dg, du, h
    for (FfOperand& o : turned)
        o = operand(gemm_carve_planes(p.take(gemm_planes_bytes(c.mode, c.f, c.m)), c.mode, c.f, c.m));
    float* dh = p.matrix(c.m, c.f);
    FfProduct h, grads[4];
    h.M = c.m, h.N = h.ldc = c.f, h.k[0] = c.d;
    h.a[0] = operand(dy), h.b[0] = operand(wd), h.c = dh;
    shape_grads(c, grads);
    grads[0].k[0] = 2 * gemm_planes_k(c.mode, c.f), grads[0].k[1] = 0;
    grads[0].a[0] = operand(dg), grads[0].b[0] = operand(w), grads[0].c = t.dx;
    grads[1].a[0] = grads[2].a[0] = operand(xt);
    grads[1].b[0] = turned[0], grads[1].c = t.dwg;
    grads[2].b[0] = turned[1], grads[2].c = t.dwu;
    grads[3].a[0] = turned[2], grads[3].b[0] = operand(dyt), grads[3].c = t.dwd;
    float* parts = static_cast<float*>(
        p.take(std::max(ff_f32_split_bytes(&h, 1), ff_f32_split_bytes(grads, 4))));
    if (ws && !p.rc) p.rc = ff_f32(&h, 1, parts, s);
    if (ws && !p.rc)
        p.rc = ff_f32_slope(c.act, t.pre_g, t.pre_u, dh, c.m, c.f, operand(dg), operand(du),
                            turned, s);
    if (ws && !p.rc) p.rc = ff_f32(grads, 4, parts, s);
    *rc = p.rc;
    return p.used;
}

// Runs the pass; with ws null only counts the workspace it takes.
uint64_t f32_forward(const FfCall& c, const F32Tensors& t, uint8_t* ws, cudaStream_t s, int* rc) {
    if (c.mode == ZG_GEMM_TF32X3) return tf32x3_forward(c, t, ws, s, rc);
    Planes p{c, ws, 0, s};
    // counted without pre-activations given: the case that takes more
    float* g = ws && t.pre_g ? t.pre_g : p.matrix(c.m, c.f);
    float* u = ws && t.pre_g ? t.pre_u : p.matrix(c.m, c.f);
    const OperandView x = p.of(t.x, c.m, c.k, false);
    p.gemm(x, p.of(t.wg, c.f, c.k, true), c.m, c.f, c.k, g);
    p.gemm(x, p.of(t.wu, c.f, c.k, true), c.m, c.f, c.k, u);
    float* h = p.matrix(c.m, c.f);
    if (ws && !p.rc) p.rc = launch_act(c.act, g, u, h, static_cast<int64_t>(c.m) * c.f, s);
    const OperandView hp = p.of(h, c.m, c.f, false);
    p.gemm(hp, p.of(t.wd, c.d, c.f, true), c.m, c.d, c.f, t.y);
    *rc = p.rc;
    return p.used;
}

uint64_t f32_backward(const FfCall& c, const F32Tensors& t, uint8_t* ws, cudaStream_t s, int* rc) {
    if (c.mode == ZG_GEMM_TF32X3) return tf32x3_backward(c, t, ws, s, rc);
    Planes p{c, ws, 0, s};
    float *dg = p.matrix(c.m, c.f), *du = p.matrix(c.m, c.f), *h = p.matrix(c.m, c.f);
    p.gemm(p.of(t.dy, c.m, c.d, false), p.of(t.wd, c.f, c.d, false), c.m, c.f, c.d, dg);  // dh
    if (ws && !p.rc)
        p.rc = launch_slope(c.act, t.pre_g, t.pre_u, dg, du, h, static_cast<int64_t>(c.m) * c.f, s);
    const OperandView dgu = p.beside(dg, du, c.m, c.f);
    p.gemm(dgu, p.beside(t.wg, t.wu, c.k, c.f), c.m, c.k, 2 * gemm_planes_k(c.mode, c.f), t.dx);
    const OperandView x = p.of(t.x, c.k, c.m, true);
    p.gemm(x, p.of(dg, c.f, c.m, true), c.k, c.f, c.m, t.dwg);
    p.gemm(x, p.of(du, c.f, c.m, true), c.k, c.f, c.m, t.dwu);
    const OperandView ht = p.of(h, c.f, c.m, true);
    p.gemm(ht, p.of(t.dy, c.d, c.m, true), c.f, c.d, c.m, t.dwd);
    *rc = p.rc;
    return p.used;
}

int check_call(FfCall& c, const char* what) {
    if (c.dtype != ZG_DTYPE_F32 && c.dtype != ZG_DTYPE_F16 && c.dtype != ZG_DTYPE_BF16)
        return set_error(ZG_ERR_DISPATCH, "%s: tensors are f32, bf16 or f16, got dtype %u", what,
                         c.dtype);
    c.size = c.dtype == ZG_DTYPE_F32 ? 4 : 2;
    if (c.act < ZG_ACT_SILU || c.act > ZG_ACT_RELU)
        return set_error(ZG_ERR_DISPATCH, "%s: unknown activation %d", what, c.act);
    if (c.dtype == ZG_DTYPE_F32 && (c.mode < ZG_GEMM_SIMT_FP32 || c.mode > ZG_GEMM_BF16X3))
        return set_error(ZG_ERR_DISPATCH, "%s: unknown mode %d", what, c.mode);
    constexpr int kMost = 1 << 28;  // tiles, planes and box coordinates stay within 32 bits
    if (c.m < 0 || c.k < 1 || c.f < 1 || c.d < 1 || c.m > kMost || c.k > kMost || c.f > kMost ||
        c.d > kMost)
        return set_error(ZG_ERR_DISPATCH, "%s: bad shape: %d rows, sizes %d, %d, %d", what, c.m,
                         c.k, c.f, c.d);
    return ZG_OK;
}

uint64_t ff_workspace(const FfCall& c) {
    if (!f32_tensor(c) || (!c.backward && few_rows(c))) return ff_layout(c).total;
    int rc;
    return c.backward ? f32_backward(c, {}, nullptr, nullptr, &rc)
                      : f32_forward(c, {}, nullptr, nullptr, &rc);
}

int check_workspace(const FfCall& c, const void* ws, uint64_t bytes, const char* what) {
    const uint64_t need = ff_workspace(c);
    if (c.m > 0 && (!ws || bytes < need || (reinterpret_cast<uintptr_t>(ws) & 255u)))
        return set_error(ZG_ERR_DISPATCH,
                         "%s: a 256-byte aligned workspace of %llu bytes is needed, got %llu", what,
                         (unsigned long long)need, (unsigned long long)bytes);
    return ZG_OK;
}

// Inputs start on 16-byte boundaries (the tensor maps' and vector loads' rule),
// outputs on their element's.
int check_pointers(std::initializer_list<const void*> in, std::initializer_list<const void*> out,
                   const FfCall& c, const char* what) {
    for (const void* p : in)
        if (!p || (reinterpret_cast<uintptr_t>(p) & 15u))
            return set_error(ZG_ERR_DISPATCH, "%s: null or not 16-byte aligned input", what);
    for (const void* p : out)
        if (!p || reinterpret_cast<uintptr_t>(p) % c.size)
            return set_error(ZG_ERR_DISPATCH, "%s: null or misaligned output", what);
    return ZG_OK;
}

int products(const FfCall& c, FfEpilogue epi, const FfProduct* p, int count, void* parts,
             cudaStream_t s) {
    if (c.size == 2) return ff_pair(c.dtype, epi, c.act, p, count, static_cast<float*>(parts), s);
    int rc = ZG_OK;
    for (int i = 0; i < count && !rc; ++i) rc = ff_simt(epi, c.act, p[i], s);
    return rc;
}

}  // namespace
}  // namespace zg

using namespace zg;

extern "C" uint64_t zg_gated_ff_workspace_bytes(uint32_t dtype, int mode, int m, int k, int f,
                                                int d, int backward) {
    FfCall c{dtype, mode, ZG_ACT_SILU, m, k, f, d, 0, backward != 0};
    if (check_call(c, "gated_ff") != ZG_OK || m == 0) return 0;
    return ff_workspace(c);
}

extern "C" int zg_gated_ff(uint32_t dtype, int mode, int act, int m, int k, int f, int d,
                           const void* x, const void* w_gate, const void* w_up,
                           const void* w_down, void* y, float* pre_gate, float* pre_up,
                           void* workspace, uint64_t workspace_bytes, void* stream) {
    FfCall c{dtype, mode, act, m, k, f, d, 0, false};
    int rc = check_call(c, "gated_ff");
    if (rc || m == 0) return rc;
    if ((rc = check_pointers({x, w_gate, w_up, w_down}, {y}, c, "gated_ff"))) return rc;
    if ((pre_gate == nullptr) != (pre_up == nullptr) ||
        ((reinterpret_cast<uintptr_t>(pre_gate) | reinterpret_cast<uintptr_t>(pre_up)) & 15u))
        return set_error(ZG_ERR_DISPATCH,
                         "gated_ff: pre_gate and pre_up are both null or both 16-byte aligned");
    if ((rc = check_workspace(c, workspace, workspace_bytes, "gated_ff"))) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (f32_tensor(c) && !few_rows(c)) {
        F32Tensors t{};
        t.x = static_cast<const float*>(x), t.wg = static_cast<const float*>(w_gate);
        t.wu = static_cast<const float*>(w_up), t.wd = static_cast<const float*>(w_down);
        t.pre_g = pre_gate, t.pre_u = pre_up, t.y = static_cast<float*>(y);
        f32_forward(c, t, static_cast<uint8_t*>(workspace), s, &rc);
        return rc;
    }
    const FfLayout l = ff_layout(c);
    const void* src[kInputs] = {x, w_gate, w_up, w_down, nullptr};
    FfInput in[kInputs];
    if ((rc = place_inputs(c, l, static_cast<uint8_t*>(workspace), src, in, s))) return rc;
    FfProduct p;  // h
    p.M = m, p.N = f, p.k[0] = k;
    p.a[0] = {in[kX].p, in[kX].ld, false};
    p.b[0] = {in[kWg].p, in[kWg].ld, true};
    p.b[1] = {in[kWu].p, in[kWu].ld, true};
    p.c = workspace, p.ldc = l.ld_f;
    p.pre_g = pre_gate, p.pre_u = pre_up;
    void* parts = static_cast<uint8_t*>(workspace) + l.parts;
    const bool few = few_rows(c);
    auto rows = [&](bool gated, const FfProduct& f) {
        return c.size == 2 ? ff_rows(dtype, gated, act, f, s) : ff_rows_f32(gated, act, f, s);
    };
    if ((rc = few ? rows(true, p) : products(c, kFfGated, &p, 1, nullptr, s))) return rc;
    FfProduct q;
    shape_y(c, q);
    q.a[0] = {workspace, l.ld_f, false};
    q.b[0] = {in[kWd].p, in[kWd].ld, true};
    q.c = y;
    return few ? rows(false, q) : products(c, kFfStore, &q, 1, parts, s);
}

extern "C" int zg_gated_ff_backward(uint32_t dtype, int mode, int act, int m, int k, int f, int d,
                                    const void* dy, const void* x, const void* w_gate,
                                    const void* w_up, const void* w_down, const float* pre_gate,
                                    const float* pre_up, void* dx, void* dw_gate, void* dw_up,
                                    void* dw_down, void* workspace, uint64_t workspace_bytes,
                                    void* stream) {
    FfCall c{dtype, mode, act, m, k, f, d, 0, true};
    int rc = check_call(c, "gated_ff_backward");
    if (rc) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if ((rc = check_pointers({}, {dw_gate, dw_up, dw_down}, c, "gated_ff_backward"))) return rc;
    if (m == 0) {  // sums over no rows
        const uint64_t up = static_cast<uint64_t>(k) * f * c.size;
        const uint64_t down = static_cast<uint64_t>(f) * d * c.size;
        if ((rc = cuda_status(cudaMemsetAsync(dw_gate, 0, up, s), "gated_ff_backward"))) return rc;
        if ((rc = cuda_status(cudaMemsetAsync(dw_up, 0, up, s), "gated_ff_backward"))) return rc;
        return cuda_status(cudaMemsetAsync(dw_down, 0, down, s), "gated_ff_backward");
    }
    if ((rc = check_pointers({dy, x, w_gate, w_up, w_down, pre_gate, pre_up}, {dx}, c,
                             "gated_ff_backward")))
        return rc;
    if ((rc = check_workspace(c, workspace, workspace_bytes, "gated_ff_backward"))) return rc;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    if (f32_tensor(c)) {
        F32Tensors t{};
        t.x = static_cast<const float*>(x), t.wg = static_cast<const float*>(w_gate);
        t.wu = static_cast<const float*>(w_up), t.wd = static_cast<const float*>(w_down);
        t.dy = static_cast<const float*>(dy);
        t.pre_g = const_cast<float*>(pre_gate), t.pre_u = const_cast<float*>(pre_up);
        t.dx = static_cast<float*>(dx), t.dwg = static_cast<float*>(dw_gate);
        t.dwu = static_cast<float*>(dw_up), t.dwd = static_cast<float*>(dw_down);
        f32_backward(c, t, ws, s, &rc);
        return rc;
    }
    const FfLayout l = ff_layout(c);
    void *h = ws, *dg = ws + l.plane, *du = ws + 2 * l.plane;
    const void* src[kInputs] = {x, w_gate, w_up, w_down, dy};
    FfInput in[kInputs];
    if ((rc = place_inputs(c, l, ws, src, in, s))) return rc;
    FfProduct p;  // dh, and from it dg, du, h
    p.M = m, p.N = f, p.k[0] = d;
    p.a[0] = {in[kDy].p, in[kDy].ld, false};
    p.b[0] = {in[kWd].p, in[kWd].ld, false};
    p.c = dg, p.c2 = du, p.c3 = h, p.ldc = l.ld_f;
    p.pre_g = const_cast<float*>(pre_gate), p.pre_u = const_cast<float*>(pre_up);
    if ((rc = products(c, kFfSlope, &p, 1, nullptr, s))) return rc;
    FfProduct w[4];
    shape_grads(c, w);
    w[0].a[0] = {dg, l.ld_f, false};
    w[0].b[0] = {in[kWg].p, in[kWg].ld, false};
    w[0].a[1] = {du, l.ld_f, false};
    w[0].b[1] = {in[kWu].p, in[kWu].ld, false};
    w[0].c = dx;
    w[1].a[0] = w[2].a[0] = {in[kX].p, in[kX].ld, true};
    w[1].b[0] = {dg, l.ld_f, true}, w[1].c = dw_gate;
    w[2].b[0] = {du, l.ld_f, true}, w[2].c = dw_up;
    w[3].a[0] = {h, l.ld_f, true};
    w[3].b[0] = {in[kDy].p, in[kDy].ld, true}, w[3].c = dw_down;
    return products(c, kFfStore, w, 4, ws + l.parts, s);
}
