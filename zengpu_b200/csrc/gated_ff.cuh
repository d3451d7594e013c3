// gated_ff.cuh - what the kernels of the gated feed-forward block share: the
// activations and their derivatives, the products' operands, the epilogues.
//
//   forward   g = x Wg, u = x Wu, h = act(g) u, y = h Wd
//   backward  dh = dy Wd^T, dg = dh u act'(g), du = dh act(g),
//             dx = dg Wg^T + du Wu^T, dWg = x^T dg, dWu = x^T du, dWd = h^T dy
//
// Sums, g and u are f32.  With 16-bit tensors h, dg and du are rounded once to
// the tensors' type, because the next product reads them as tensor-core operands
// of that type; g and u stay f32 between the passes, so that the backward pass
// adds no rounding of its own to those three.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "zg_common.cuh"

namespace zg {

// Terms of a sum that 16-bit MMAs may add up in TMEM.  The tensor core's f32 additions
// truncate, always toward zero: a sum of n terms of one sign lost 6.4e-9 n of itself
// (n = 300007: 1.9e-3, half a bf16 step), so a run of these 1.05e-4, a fifth of half an f16
// step.  Longer sums are added up from runs by rounded additions.
constexpr int kFfRun = 16384;

template <class T> struct FfElem;
template <> struct FfElem<float> {
    __device__ static float get(float x) { return x; }
    __device__ static float put(float x) { return x; }
};
template <> struct FfElem<__nv_bfloat16> {
    __device__ static float get(__nv_bfloat16 x) { return __bfloat162float(x); }
    __device__ static __nv_bfloat16 put(float x) { return __float2bfloat16_rn(x); }
};
template <> struct FfElem<__half> {
    __device__ static float get(__half x) { return __half2float(x); }
    __device__ static __half put(float x) { return __float2half_rn(x); }
};

// a = act(g) and slope = act'(g).
//   SiLU       s = 1 / (1 + e^-g): g s, s (1 + g (1 - s))
//   GELU       c = Phi(g) = erfc(-g / sqrt 2) / 2: g c, c + g phi(g)
//   GELU_TANH  the same with c = (1 + tanh q) / 2 = 1 / (1 + e^-2q),
//              q = sqrt(2 / pi) (g + 0.044715 g^3): c' = 2 c (1 - c) q'
//   ReLU       relu1: 0 (slope 0) for g <= 0 and NaN
// erfc instead of 1 + erf, and 1 / (1 + e^-2q) instead of 1 + tanh, keep the
// left tails' relative accuracy, where those sums cancel (FAST: a c or s below 2^-126
// becomes zero).
struct ActValue {
    float a, slope;
};

// FAST (16-bit tensors): __expf, whose error grows to 2^-16 relative where the result nears
// 2^-126, and a polynomial for erfc, within 2^-21: together with the rounding of their
// arguments under 2^-14, an eighth of half an f16 step.  f32 tensors take expf, erfcf and
// a true quotient.
// (The correctly rounded reciprocal branches, and took 60 cycles a value one after the
// other; the approximate one is within a unit of the last place.)
__device__ __forceinline__ float rcp_fast(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
template <bool FAST>
__device__ __forceinline__ float logistic(float x) {
    return FAST ? rcp_fast(1.0f + __expf(-x)) : 1.0f / (1.0f + expf(-x));
}

template <int ACT, bool FAST>
__device__ __forceinline__ ActValue activate(float g) {
    if (ACT == ZG_ACT_RELU) return {relu1(g), g > 0.0f ? 1.0f : 0.0f};
    if (ACT == ZG_ACT_SILU) {
        const float s = logistic<FAST>(g);
        return {g * s, s * (1.0f + g * (1.0f - s))};
    }
    if (ACT == ZG_ACT_GELU && FAST) {
        // erfc(z) = (a1 t + ... + a8 t^8) e^(-z^2) for z >= 0, t = 1 / (1 + 0.43 z), the form of
        // Abramowitz and Stegun 7.1.26, whose five coefficients keep the absolute error small
        // (0.4 % of erfc at z = 4).  These are fitted (least squares, reweighted towards the
        // largest deviation) to e^(z^2) erfc(z) from z = 0 to 9.6 in relative terms: within
        // 8.5e-8, and 4e-7 in f32 arithmetic.  z = |g| / sqrt 2 makes the exponential the
        // density's.
        const float e = __expf(-0.5f * g * g);
        const float t = rcp_fast(fmaf(0.43f * 0.70710678118654752f, fabsf(g), 1.0f));
        float p = fmaf(0.073669054f, t, -0.31021592f);
        p = fmaf(p, t, 0.38344166f);
        p = fmaf(p, t, -0.085488908f);
        p = fmaf(p, t, 0.24672212f);
        p = fmaf(p, t, 0.20498736f);
        p = fmaf(p, t, 0.24436975f);
        p = fmaf(p, t, 0.24251497f);
        const float tail = 0.5f * p * t * e;  // Phi(-|g|)
        const float c = g > 0.0f ? 1.0f - tail : tail;
        return {g * c, fmaf(g * 0.39894228040143268f, e, c)};
    }
    if (ACT == ZG_ACT_GELU) {
        const float c = 0.5f * erfcf(-0.70710678118654752f * g);
        return {g * c, c + g * 0.39894228040143268f * expf(-0.5f * g * g)};
    }
    const float k = 0.79788456080286536f;
    const float q = k * (g + 0.044715f * g * g * g);
    const float c = logistic<FAST>(2.0f * q);
    // c (1 - c) is zero long before b differs from g; an infinite b^2 would make that NaN
    const float b = fminf(fmaxf(g, -1e9f), 1e9f);
    return {g * c, c + b * 2.0f * c * (1.0f - c) * k * (1.0f + 3.0f * 0.044715f * b * b)};
}

// One operand of a product over `k`: row r (of M or N), position i of the sum.
//   k-major   p[r * ld + i]
//   mn-major  p[i * ld + r]
struct FfOperand {
    const void* p = nullptr;
    int64_t ld = 0;
    bool mn = false;
};

enum FfEpilogue { kFfStore, kFfGated, kFfSlope };

// D[M x N].  kFfStore: c = a[0] b[0] (+ a[1] b[1] when k[1] > 0).
// kFfGated: g = a[0] b[0], u = a[0] b[1]; c = act(g) u, and g, u to pre_g, pre_u
// unless they are null.  kFfSlope: dh = a[0] b[0] with pre_g and pre_u read:
// c = dg, c2 = du, c3 = h.  c, c2, c3: the tensors' type, pitch ldc; pre_g,
// pre_u: f32, pitch N.
struct FfProduct {
    int M = 0, N = 0;
    int k[2] = {0, 0};
    FfOperand a[2], b[2];
    void* c = nullptr;
    void* c2 = nullptr;
    void* c3 = nullptr;
    int64_t ldc = 0;
    float* pre_g = nullptr;
    float* pre_u = nullptr;
};

// Launches a kernel that may start while the one before it in the stream still runs
// (it calls griddepcontrol.wait before it touches memory).
template <class... Params, class... Args>
int launch_dependent(const char* what, void (*kernel)(Params...), unsigned grid, unsigned threads,
                     size_t smem, cudaStream_t s, const Args&... args) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cuda_status(cudaLaunchKernelEx(&cfg, kernel, args...), what);
}

// Plain CUDA-core product of f32 tensors of any layout (gated_ff.cu).
int ff_simt(FfEpilogue epi, int act, const FfProduct& p, cudaStream_t s);

// 16-bit tensors on the tensor cores (gated_ff_tc.cu): `count` products of one
// epilogue in one launch (at most four).  Operands: 16-byte aligned, pitch a multiple
// of 8.  kFfStore: long sums of few tiles are split, for which `parts` holds
// ff_split_bytes; ldc is N then.
uint64_t ff_split_bytes(const FfProduct* products, int count);
int ff_pair(uint32_t dtype, FfEpilogue epi, int act, const FfProduct* products, int count,
            float* parts, cudaStream_t s);

// f32 tensors in the TF32X3 mode (gated_ff_f32.cu), operands as planes (sgemm_tc.cu,
// k-major, ld in floats), k[0] the sum's length; kFfStore only, parts as ff_pair's.
uint64_t ff_f32_split_bytes(const FfProduct* products, int count);
int ff_f32(const FfProduct* products, int count, float* parts, cudaStream_t s);
// h = act(g) u as planes [m, n]; dg and du as planes, and dg, du and h transposed.
int ff_f32_act(int act, const float* g, const float* u, int m, int n, const FfOperand& h,
               cudaStream_t s);
int ff_f32_slope(int act, const float* g, const float* u, const float* dh, int m, int n,
                 const FfOperand& dg, const FfOperand& du, const FfOperand (&turned)[3],
                 cudaStream_t s);

// The forward products for up to kFfRows rows of 16-bit tensors (gated_ff_rows.cu):
// `gated` as kFfGated, else as kFfStore of one product, launched right behind the
// gated one whose result it reads.  At 4096 x 12288 in bf16 64 rows take 65 us here
// and 65 rows 93 on the CTA pairs (this form took 101 from 65 rows on).
constexpr int kFfRows = 64;
int ff_rows(uint32_t dtype, bool gated, int act, const FfProduct& product, cudaStream_t s);

// The same for f32 tensors, on the CUDA cores (gated_ff_rows_f32.cu).
constexpr int kFfRowsF32 = 32;
int ff_rows_f32(bool gated, int act, const FfProduct& product, cudaStream_t s);

}  // namespace zg
