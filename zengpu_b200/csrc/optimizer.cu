// optimizer.cu - one AdamW step over many tensors at once, and the gradient
// norm that clips it.  Beside Level-1 saxpy / sscal (elementwise.cu), the
// in-place updates of zengpu-blas/src/level1.rs:51-139; the reference has no
// optimiser.
//
// AdamW.  With s = *grad_scale (1 when absent) and step t, per element
//     g' = s g
//     m  = b1 m + (1 - b1) g'
//     v  = b2 v + ((1 - b2) g') g'
//     p  = p (1 - lr wd) - ((lr / (1 - b1^t)) m) / (sqrt(v) / sqrt(1 - b2^t) + eps)
// in f32, every operation rounded on its own in the order written, as the
// other elementwise kernels here do: the result does not depend on which
// vector or scalar path an element takes, nor on the launch.  (The one exception:
// with 8-bit moments the last line's root and quotient are approximate instructions,
// which change the weight's step by up to 2^-21 of itself; m, v and their codes are as
// written.)  Weights are
// f32, or bf16 / f16 either with an f32 master that carries the sum (the
// 16-bit weight is its rounding) or without one (the sum itself is rounded).
//
// Moments in 8 bits: a block of 256 consecutive elements of a tensor stores m
// as e4m3 codes times one f32 scale, and r = sqrt(v) likewise (the root halves
// the exponent range the code has to span).  scale = max|x| / 448, the largest
// code for the largest value.  e4m3 rounds to 2^-4 relative, over 2^17.8 below
// the block's maximum; smaller m becomes zero, but r > 0 is held at the
// smallest code or more, so that no denominator collapses to eps.  The weight
// is updated from m and r before they are rounded.  A block in which m or r is
// not finite gets a NaN scale.
//
// All tensors of a call share one launch: the table of their pointers travels
// in the kernel's parameters (no copy to the device, nothing that a captured
// graph could find overwritten).  A CTA owns a chunk of one tensor, a warp a
// 256-element block of it per turn, as two runs of 128 elements with four
// neighbours per lane (16-byte loads of f32).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <exception>
#include <vector>

#include "zg_common.cuh"

namespace zg {
namespace {

constexpr int kOptThreads = 256;
constexpr int kBlockElems = ZG_ADAMW_BLOCK;  // per warp and turn, and per 8-bit scale
constexpr int kTurnElems = kBlockElems * (kOptThreads / 32);
static_assert(kBlockElems == 32 * 8, "a lane holds eight elements of a block");

template <class T> struct Elem;
template <> struct Elem<float> {
    __device__ static float get(float x) { return x; }
    __device__ static float put(float x) { return x; }
};
template <> struct Elem<__nv_bfloat16> {
    __device__ static float get(__nv_bfloat16 x) { return __bfloat162float(x); }
    __device__ static __nv_bfloat16 put(float x) { return __float2bfloat16_rn(x); }
};
template <> struct Elem<__half> {
    __device__ static float get(__half x) { return __half2float(x); }
    __device__ static __half put(float x) { return __float2half_rn(x); }
};

template <class T> struct alignas(4 * sizeof(T)) Four { T v[4]; };

// Eight elements of the block at `x`: vector form for a whole, aligned block,
// else one element at a time up to `left`.  Element (j, i) of lane l is
// 128 j + 4 l + i in the vector form and 128 j + 32 i + l in the other.
template <class T>
__device__ __forceinline__ void load8(const T* x, bool vec, int lane, int64_t left, T (&out)[8]) {
    if (vec) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const Four<T> f = *reinterpret_cast<const Four<T>*>(x + 128 * j + 4 * lane);
#pragma unroll
            for (int i = 0; i < 4; ++i) out[4 * j + i] = f.v[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int e = 32 * i + lane;
            out[i] = e < left ? x[e] : T(0.0f);
        }
    }
}
template <class T>
__device__ __forceinline__ void store8(T* x, bool vec, int lane, int64_t left, const T (&in)[8]) {
    if (vec) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            Four<T> f;
#pragma unroll
            for (int i = 0; i < 4; ++i) f.v[i] = in[4 * j + i];
            *reinterpret_cast<Four<T>*>(x + 128 * j + 4 * lane) = f;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int e = 32 * i + lane;
            if (e < left) x[e] = in[i];
        }
    }
}

struct Factors {
    float b1, c1, b2, c2;  // beta and 1 - beta, each rounded from 64 bits
    float step_size;       // lr / (1 - b1^t)
    float root;            // 1 / sqrt(1 - b2^t)
    float eps, decay;      // decay: 1 - lr wd
    float one;             // 1
};

struct DeviceHyper {  // values a captured graph reads anew at each replay
    const int64_t* step;
    const float* lr;
    const float* grad_scale;
};

// 1 - b^t without the cancellation that b^t near 1 would bring.
__host__ __device__ inline double bias_correction(double beta, double t) {
    return beta > 0.0 ? -expm1(t * log(beta)) : 1.0;
}
__host__ __device__ inline void schedule(Factors& f, double lr, double beta1, double beta2,
                                         double wd, double t) {
    f.step_size = static_cast<float>(lr / bias_correction(beta1, t));
    f.root = static_cast<float>(1.0 / sqrt(bias_correction(beta2, t)));
    f.decay = static_cast<float>(1.0 - lr * wd);
}

// Tables of two sizes: a launch copies its whole parameter block, so a call of a
// few tensors does not carry the largest one (32764 bytes of parameters at most).
constexpr int kSmallTable = 32;
constexpr int kLargeTable = 440;

template <int CAP, class Tensor>
struct Table {
    Tensor t[CAP];
    uint32_t first[CAP + 1];  // first chunk of tensor i; first[count] is the number of chunks
    int count;
};

// The tensor that chunk c belongs to: the last one whose first chunk is <= c.
template <int CAP, class Tensor>
__device__ __forceinline__ int tensor_of(const Table<CAP, Tensor>& tab, uint32_t c) {
    int lo = 0, hi = tab.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (tab.first[mid] <= c) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Two f32 in a register pair: Blackwell's packed f32 units round each half as the
// scalar operations do, at half the instructions.
using F2 = unsigned long long;
__device__ __forceinline__ F2 pack(float a, float b) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpack(F2 x) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
    return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// a + b as a 1 + b.  The 1 is a value the compiler does not know: it contracts a
// packed product and a packed sum into one rounding, .rn or not.
__device__ __forceinline__ F2 add2(F2 a, F2 b, F2 one) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(one), "l"(b));
    return r;
}
__device__ __forceinline__ F2 both(float a) { return pack(a, a); }

// The larger magnitude; NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(b)));
    return r;
}

template <class T>
__device__ __forceinline__ F2 widen(const T (&x)[8], int i) {
    return pack(Elem<T>::get(x[2 * i]), Elem<T>::get(x[2 * i + 1]));
}
// Copies a whole block's `Bytes` (256 elements) into shared memory, asynchronously.
template <int Bytes>
__device__ __forceinline__ void fetch(uint8_t* to, const void* from, int lane) {
#pragma unroll
    for (int i = 0; i < (Bytes + 511) / 512; ++i)
        if (Bytes >= 512 || lane < Bytes / 16)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                             smem_u32(to) + i * 512 + lane * 16),
                         "l"(static_cast<const uint8_t*>(from) + i * 512 + lane * 16)
                         : "memory");
}

// Eight codes of a lane as two words of four: one load of a word in the vector form.
__device__ __forceinline__ void load_codes(const uint8_t* x, bool vec, int lane, int64_t left,
                                           uint32_t (&w)[2]) {
    if (vec) {
        w[0] = *reinterpret_cast<const uint32_t*>(x + 4 * lane);
        w[1] = *reinterpret_cast<const uint32_t*>(x + 128 + 4 * lane);
    } else {
        w[0] = w[1] = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int e = 32 * i + lane;
            if (e < left) w[i / 4] |= static_cast<uint32_t>(x[e]) << (i % 4 * 8);
        }
    }
}
__device__ __forceinline__ void store_codes(uint8_t* x, bool vec, int lane, int64_t left,
                                            const uint32_t (&w)[2]) {
    if (vec) {
        *reinterpret_cast<uint32_t*>(x + 4 * lane) = w[0];
        *reinterpret_cast<uint32_t*>(x + 128 + 4 * lane) = w[1];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int e = 32 * i + lane;
            if (e < left) x[e] = static_cast<uint8_t>(w[i / 4] >> (i % 4 * 8));
        }
    }
}
// Codes 2 i and 2 i + 1 of the eight.
__device__ __forceinline__ F2 decode(const uint32_t (&w)[2], int i) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(
        static_cast<__nv_fp8x2_storage_t>(w[i / 2] >> (i % 2 * 16)), __NV_E4M3);
    const float2 f = __half22float2(__half2(h));
    return pack(f.x, f.y);
}
__device__ __forceinline__ void encode(uint32_t (&w)[2], int i, float2 y) {
    const uint32_t c = __nv_cvt_float2_to_fp8x2(y, __NV_SATFINITE, __NV_E4M3);
    w[i / 2] = i % 2 ? w[i / 2] | (c << 16) : c;
}

// The scale of a block whose largest magnitude is `top`, and its inverse.
__device__ __forceinline__ float block_scale(float top, float& inv) {
    inv = 0.0f;
    if (!(top > 0.0f)) return top;  // zero, or NaN
    const float s = fmaxf(__fmul_rn(top, 1.0f / 448.0f), 0x1p-126f);
    inv = __frcp_rn(s);
    return top < INFINITY ? s : __int_as_float(0x7fc00000);
}

// The largest over a warp of values that are not negative, or NaN: the order of their
// bits, with NaN last.
__device__ __forceinline__ float warp_top(float top) {
    return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
}

// Eight m of a block as codes, and the block's scale.
__device__ __forceinline__ float encode_m(const F2 (&m)[4], uint32_t (&codes)[2]) {
    float top = 0.0f, inv;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = unpack(m[i]);
        top = max_nan(top, max_nan(f.x, f.y));
    }
    const float s = block_scale(warp_top(top), inv);
#pragma unroll
    for (int i = 0; i < 4; ++i) encode(codes, i, unpack(mul2(m[i], both(inv))));
    return s;
}

// Both flush subnormals: a v below 2^-126 gives root 0, and a denominator below 2^-126
// an infinite reciprocal.  With an eps that this matters to (kTinyEps) neither is called.
__device__ __forceinline__ float sqrt_approx(float x) {
    float r;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float rcp_approx(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// Times 1 / sqrt(1 - b2), the most that a root is scaled up by (at step 1): with an eps
// below that the root of a subnormal v, up to 2^-63 = 1.1e-19 before the scaling, may count
// for 2^-23 of the denominator or more, and where v is zero eps is all of it, subnormal or
// not.  Roots and quotients are exact then.
constexpr double kTinyEps = 1e-12;

// Eight roots of a block as codes, from v and r, the roots to within three units of
// the last place (sqrt.approx: one or two): codes are those of the correctly rounded
// root.  The root of the largest v is taken exactly, and so is that of a value
// whose quotient y by the scale lies within eight units of a point where e4m3's
// rounding turns (the low 20 bits at one half), or among the subnormal codes.
__device__ __forceinline__ float encode_root(const F2 (&v)[4], const F2 (&r)[4],
                                             uint32_t (&codes)[2]) {
    float top = 0.0f, inv;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = unpack(v[i]);
        top = max_nan(top, max_nan(f.x, f.y));
    }
    const float s = block_scale(__fsqrt_rn(warp_top(top)), inv);
    float2 y[4];
    uint32_t close = 0xffffffffu;  // distance to the nearest turn, least of the eight
    float low = 1.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        y[i] = unpack(mul2(r[i], both(inv)));
        low = fminf(low, fminf(y[i].x, y[i].y));
        close = min(close, (__float_as_uint(y[i].x) - 0x7fff8u) << 12);
        close = min(close, (__float_as_uint(y[i].y) - 0x7fff8u) << 12);
    }
    if (low < 0x1p-6f || close <= (16u << 12)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = unpack(v[i]);
            y[i].x = __fmul_rn(__fsqrt_rn(f.x), inv);
            y[i].y = __fmul_rn(__fsqrt_rn(f.y), inv);
            if (f.x > 0.0f) y[i].x = fmaxf(y[i].x, 0x1p-9f);
            if (f.y > 0.0f) y[i].y = fmaxf(y[i].y, 0x1p-9f);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) encode(codes, i, y[i]);
    return s;
}

// What bounds it: HBM.  f32 weights, gradients and moments move 28 bytes per
// element, 16-bit weights with a master and 8-bit moments 16.1; the latter are
// near the issue rate too: roots and quotients are then the approximate
// instructions (a quotient is within 2 units of its last place, on a change of the
// weight that is small beside it; the roots' codes are exact, see encode_root), and
// what a whole call decides is not asked for each pair (exact roots: another kernel; a
// master: a branch a block; 795 -> 713 us).  277 M elements: 1.144 ms (6.8 TB/s) and 0.713 ms (6.2 TB/s).
// EXACT: correctly rounded roots and quotients in the weight's change; always with 32 bits.
template <class P, class G, int BITS, bool EXACT, int CAP>
__global__ void __launch_bounds__(kOptThreads, BITS == 8 ? 3 : 2)
    adamw_kernel(const __grid_constant__ Table<CAP, zg_adamw_tensor> tab, int64_t chunk, Factors f,
                 const zg_adamw_hyper hyper, const DeviceHyper dev) {
    const int i = tensor_of(tab, blockIdx.x);
    const zg_adamw_tensor& t = tab.t[i];
    const int64_t begin = static_cast<int64_t>(blockIdx.x - tab.first[i]) * chunk;
    const int64_t end = min(static_cast<int64_t>(t.n), begin + chunk);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    float gscale = 1.0f;
    if (dev.grad_scale) {
        gscale = *dev.grad_scale;
        if (!isfinite(gscale)) return;  // the step is skipped: nothing changes
    }
    if (dev.step && *dev.step < 1) return;  // steps count from 1
    if (dev.step || dev.lr) {
        __shared__ Factors shared;
        if (threadIdx.x == 0) {
            shared = f;
            schedule(shared, dev.lr ? *dev.lr : hyper.lr, hyper.beta1, hyper.beta2,
                     hyper.weight_decay,
                     static_cast<double>(dev.step ? *dev.step : hyper.step));
        }
        __syncthreads();
        f = shared;
    }

    P* p = static_cast<P*>(t.param);
    const G* g = static_cast<const G*>(t.grad);
    float* master = static_cast<float*>(t.master);
    const bool aligned =
        ((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(g) |
          reinterpret_cast<uintptr_t>(master) | reinterpret_cast<uintptr_t>(t.exp_avg) |
          reinterpret_cast<uintptr_t>(t.exp_avg_sq)) & 15) == 0;

    // Whole blocks of aligned tensors come through shared memory: the next one (with 8-bit
    // moments the next two, 795 us for 277 M elements against 831) is on its way while
    // this one is worked on, at no cost in registers.
    constexpr int kMoment = BITS == 32 ? 4 : 1;
    constexpr int kG = kBlockElems * sizeof(G), kW = kBlockElems * 4, kM = kBlockElems * kMoment;
    constexpr int kDeep = BITS == 8 ? 2 : 1, kPlace = kG + kW + 2 * kM;
    __shared__ __align__(16) uint8_t ring[kOptThreads / 32][kDeep][kPlace];
    auto whole = [&](int64_t b) { return aligned && end - b >= kBlockElems; };
    float asked_ms[kDeep], asked_vs[kDeep];  // the scales, in registers
    auto ask = [&](int64_t b, int place) {
        if (b < end) {
            if (BITS == 8) {
                asked_ms[kDeep - 1] = t.exp_avg_scale[b / kBlockElems];
                asked_vs[kDeep - 1] = t.exp_avg_sq_scale[b / kBlockElems];
            }
            if (whole(b)) {
                uint8_t* to = ring[warp][place];
                fetch<kG>(to, g + b, lane);
                if (master) fetch<kW>(to + kG, master + b, lane);
                else fetch<kBlockElems * sizeof(P)>(to + kG, p + b, lane);
                fetch<kM>(to + kG + kW, static_cast<uint8_t*>(t.exp_avg) + b * kMoment, lane);
                fetch<kM>(to + kG + kW + kM, static_cast<uint8_t*>(t.exp_avg_sq) + b * kMoment, lane);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };

    int64_t b = begin + warp * kBlockElems;
    int place = 0;
    ask(b, 0);
    if (kDeep == 2) {
        asked_ms[0] = asked_ms[1], asked_vs[0] = asked_vs[1];
        ask(b + kTurnElems, 1);
    }
    for (; b < end; b += kTurnElems) {
        const int64_t left = end - b;
        const bool vec = whole(b);
        G gv[8];
        P pv[8];
        float wv[8], mv[8], vv[8];
        uint32_t mc[2], vc[2];
        const float ms = asked_ms[0], vs = asked_vs[0];
        const uint8_t* in_g = ring[warp][place];
        const uint8_t *in_w = in_g + kG, *in_m = in_w + kW, *in_v = in_m + kM;
        auto take = [&](bool v, const G* gb, const float* wb, const P* pb, const uint8_t* mb,
                        const uint8_t* vb) {
            load8<G>(gb, v, lane, left, gv);
            if (master) {
                load8<float>(wb, v, lane, left, wv);
            } else {
                load8<P>(pb, v, lane, left, pv);
#pragma unroll
                for (int e = 0; e < 8; ++e) wv[e] = Elem<P>::get(pv[e]);
            }
            if (BITS == 32) {
                load8<float>(reinterpret_cast<const float*>(mb), v, lane, left, mv);
                load8<float>(reinterpret_cast<const float*>(vb), v, lane, left, vv);
            } else {
                load_codes(mb, v, lane, left, mc);
                load_codes(vb, v, lane, left, vc);
            }
        };
        asm volatile("cp.async.wait_group %0;" ::"n"(kDeep - 1) : "memory");
        __syncwarp();
        if (vec)
            take(true, reinterpret_cast<const G*>(in_g), reinterpret_cast<const float*>(in_w),
                 reinterpret_cast<const P*>(in_w), in_m, in_v);
        else
            take(false, g + b, master + b, p + b,
                 static_cast<uint8_t*>(t.exp_avg) + b * kMoment,
                 static_cast<uint8_t*>(t.exp_avg_sq) + b * kMoment);
        __syncwarp();
        if (kDeep == 2) asked_ms[0] = asked_ms[1], asked_vs[0] = asked_vs[1];
        ask(b + kDeep * kTurnElems, place);
        if (kDeep == 2) place ^= 1;
        F2 m[4], v[4], r[4], w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const F2 ge = mul2(widen(gv, e), both(gscale));
            if (BITS == 32) {
                m[e] = widen(mv, e);
                v[e] = widen(vv, e);
            } else {
                m[e] = mul2(decode(mc, e), both(ms));
                v[e] = mul2(decode(vc, e), both(vs));
                v[e] = mul2(v[e], v[e]);
            }
            m[e] = add2(mul2(m[e], both(f.b1)), mul2(ge, both(f.c1)), both(f.one));
            v[e] = add2(mul2(v[e], both(f.b2)), mul2(mul2(ge, both(f.c2)), ge), both(f.one));
            const float2 v2 = unpack(v[e]);
            r[e] = EXACT ? pack(__fsqrt_rn(v2.x), __fsqrt_rn(v2.y))
                         : pack(sqrt_approx(v2.x), sqrt_approx(v2.y));
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 den = unpack(add2(mul2(r[e], both(f.root)), both(f.eps), both(f.one)));
            const float2 num = unpack(mul2(m[e], both(-f.step_size)));
            const F2 quot = EXACT ? pack(__fdiv_rn(num.x, den.x), __fdiv_rn(num.y, den.y))
                                  : pack(num.x * rcp_approx(den.x), num.y * rcp_approx(den.y));
            w[e] = add2(mul2(widen(wv, e), both(f.decay)), quot, both(f.one));
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 w2 = unpack(w[e]);
            wv[2 * e] = w2.x, wv[2 * e + 1] = w2.y;
            pv[2 * e] = Elem<P>::put(w2.x), pv[2 * e + 1] = Elem<P>::put(w2.y);
        }
        store8<P>(p + b, vec, lane, left, pv);
        if (master) store8<float>(master + b, vec, lane, left, wv);
        if (BITS == 32) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 m2 = unpack(m[e]), v2 = unpack(v[e]);
                mv[2 * e] = m2.x, mv[2 * e + 1] = m2.y;
                vv[2 * e] = v2.x, vv[2 * e + 1] = v2.y;
            }
            store8<float>(static_cast<float*>(t.exp_avg) + b, vec, lane, left, mv);
            store8<float>(static_cast<float*>(t.exp_avg_sq) + b, vec, lane, left, vv);
        } else {
            // elements past a tensor's end are zeros, which change no block's maximum,
            // except that 0 / (0 + eps) may be NaN: only w sees that, and is not stored
            const float new_ms = encode_m(m, mc), new_vs = encode_root(v, r, vc);
            store_codes(static_cast<uint8_t*>(t.exp_avg) + b, vec, lane, left, mc);
            store_codes(static_cast<uint8_t*>(t.exp_avg_sq) + b, vec, lane, left, vc);
            if (lane == 0) {
                t.exp_avg_scale[b / kBlockElems] = new_ms;
                t.exp_avg_sq_scale[b / kBlockElems] = new_vs;
            }
        }
    }
}

// ---- gradient norm ---------------------------------------------------------------
// norm = sqrt(sum g^2) in 64 bits throughout (a square of f32 has at most 48
// bits, so only the sums round, and no f32 gradient overflows), summed in a fixed
// order: per thread over its elements, per CTA by a tree, then one CTA over the
// partial sums.  Reads each gradient once: HBM bound, 87 us for 277 M bf16 (6.3 TB/s).
struct NormTensor {
    const void* g;
    uint64_t n;
};

__device__ __forceinline__ double block_sum(double x) {
    __shared__ double part[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    if (lane == 0) part[warp] = x;
    __syncthreads();
    x = warp == 0 && lane < static_cast<int>(blockDim.x >> 5) ? part[lane] : 0.0;
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;  // complete in warp 0
}

// A thread's share of the sum: the CTA takes every gridDim.x-th chunk.
template <class G, int CAP, int kThreads>
__device__ __forceinline__ double chunk_sums(const Table<CAP, NormTensor>& tab, int64_t chunk) {
    const uint32_t chunks = tab.first[tab.count];
    double sum = 0.0;
    for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
        const int i = tensor_of(tab, c);
        const G* g = static_cast<const G*>(tab.t[i].g);
        const int64_t begin = static_cast<int64_t>(c - tab.first[i]) * chunk;
        const int64_t end = min(static_cast<int64_t>(tab.t[i].n), begin + chunk);
        auto add = [&](G x) {
            const double d = static_cast<double>(Elem<G>::get(x));
            sum = fma(d, d, sum);
        };
        if ((reinterpret_cast<uintptr_t>(g + begin) & 15) == 0) {
            // 16-byte loads, four in flight a thread
            constexpr int kPer = 16 / sizeof(G), kFlight = 4;
            const int n = static_cast<int>(end - begin), pieces = n / kPer;
            const uint4* from = reinterpret_cast<const uint4*>(g + begin);
            for (int at = threadIdx.x; at < pieces; at += kFlight * kThreads) {
                uint4 q[kFlight];
#pragma unroll
                for (int u = 0; u < kFlight; ++u)
                    q[u] = at + u * kThreads < pieces ? __ldcs(from + at + u * kThreads)
                                                         : make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int u = 0; u < kFlight; ++u) {
                    G x[kPer];
                    __builtin_memcpy(x, &q[u], 16);
#pragma unroll
                    for (int e = 0; e < kPer; ++e) add(x[e]);
                }
            }
            if (threadIdx.x < n - pieces * kPer) add(g[begin + pieces * kPer + threadIdx.x]);
        } else {
            for (int64_t at = begin + threadIdx.x; at < end; at += kThreads) add(g[at]);
        }
    }
    return sum;
}

// out[0] = norm, out[1] = min(1, max_norm / norm); NaN when the norm is not finite.
__device__ __forceinline__ void put_norm(double sum, double max_norm, float* out) {
    const double norm = sqrt(sum);
    out[0] = static_cast<float>(norm);
    out[1] = !isfinite(norm) ? __int_as_float(0x7fc00000)
                             : norm > max_norm ? static_cast<float>(max_norm / norm) : 1.0f;
}

template <class G, int CAP>
__global__ void __launch_bounds__(kOptThreads)
    norm_partial_kernel(const __grid_constant__ Table<CAP, NormTensor> tab, int64_t chunk,
                        double* partial) {
    const double sum = block_sum(chunk_sums<G, CAP, kOptThreads>(tab, chunk));
    if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

// Few gradients: one launch, the eight CTAs of one cluster.
constexpr int kNormCluster = 8, kNormThreads = 1024;
template <class G>
__global__ void __cluster_dims__(kNormCluster, 1, 1) __launch_bounds__(kNormThreads)
    norm_cluster_kernel(const __grid_constant__ Table<kSmallTable, NormTensor> tab, int64_t chunk,
                        double max_norm, float* out) {
    __shared__ double mine;
    const double sum = block_sum(chunk_sums<G, kSmallTable, kNormThreads>(tab, chunk));
    if (threadIdx.x == 0) mine = sum;
    cluster_sync();
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        double total = 0.0;
        for (uint32_t r = 0; r < kNormCluster; ++r) {
            double x;
            asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(x) : "r"(mapa_shared(&mine, r)));
            total += x;
        }
        put_norm(total, max_norm, out);
    }
    cluster_sync();  // nobody leaves while its sum is read
}

__global__ void __launch_bounds__(1024)
    norm_final_kernel(const double* partial, int count, double max_norm, float* out) {
    double sum = 0.0;
    for (int i = threadIdx.x; i < count; i += 1024) sum += partial[i];
    sum = block_sum(sum);
    if (threadIdx.x == 0) put_norm(sum, max_norm, out);
}

// ---- host ----------------------------------------------------------------------------
int sm_count() {
    static thread_local int cached_dev = -1, cached = 0;
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev != cached_dev) {
        cudaDeviceGetAttribute(&cached, cudaDevAttrMultiProcessorCount, dev);
        if (cached <= 0) cached = 148;
        cached_dev = dev;
    }
    return cached;
}

// Elements per chunk: whole turns of a CTA, up to eight where that leaves thirty
// chunks for each SM, else as little as one.
int64_t chunk_elems(uint64_t total) {
    const uint64_t want = total / (static_cast<uint64_t>(sm_count()) * 32);
    const uint64_t turns = std::min<uint64_t>(std::max<uint64_t>(want / kTurnElems, 1), 8);
    return static_cast<int64_t>(turns * kTurnElems);
}

template <int CAP, class Tensor>
void fill(Table<CAP, Tensor>& tab, const Tensor* t, int count, int64_t chunk) {
    uint32_t chunks = 0;
    for (int i = 0; i < count; ++i) {
        tab.t[i] = t[i];
        tab.first[i] = chunks;
        chunks += static_cast<uint32_t>((t[i].n + chunk - 1) / chunk);
    }
    tab.first[count] = chunks;
    tab.count = count;
}

struct AdamCall {
    bool exact;
    Factors f;
    zg_adamw_hyper hyper;
    DeviceHyper dev;
    int64_t chunk;
    cudaStream_t stream;
};

template <class P, class G, int BITS, bool EXACT, int CAP>
int launch_adamw_table(const zg_adamw_tensor* t, int count, const AdamCall& c) {
    static_assert(sizeof(Table<CAP, zg_adamw_tensor>) + 256 <= 32764, "kernel parameters");
    Table<CAP, zg_adamw_tensor> tab;
    fill(tab, t, count, c.chunk);
    adamw_kernel<P, G, BITS, EXACT, CAP><<<tab.first[count], kOptThreads, 0, c.stream>>>(
        tab, c.chunk, c.f, c.hyper, c.dev);
    return cuda_status(cudaGetLastError(), "zg_adamw");
}

template <class P, class G, int BITS, bool EXACT>
int launch_adamw(const std::vector<zg_adamw_tensor>& t, const AdamCall& c) {
    for (size_t at = 0; at < t.size(); at += kLargeTable) {
        const int n = static_cast<int>(std::min<size_t>(t.size() - at, kLargeTable));
        const int rc = n <= kSmallTable
                           ? launch_adamw_table<P, G, BITS, EXACT, kSmallTable>(t.data() + at, n, c)
                           : launch_adamw_table<P, G, BITS, EXACT, kLargeTable>(t.data() + at, n, c);
        if (rc) return rc;
    }
    return ZG_OK;
}

template <class P, class G>
int launch_adamw_bits(int bits, const std::vector<zg_adamw_tensor>& t, const AdamCall& c) {
    if (bits == 32) return launch_adamw<P, G, 32, true>(t, c);
    return c.exact ? launch_adamw<P, G, 8, true>(t, c) : launch_adamw<P, G, 8, false>(t, c);
}

template <class P>
int launch_adamw_grad(uint32_t grad, int bits, const std::vector<zg_adamw_tensor>& t,
                      const AdamCall& c) {
    switch (grad) {
        case ZG_DTYPE_F32: return launch_adamw_bits<P, float>(bits, t, c);
        case ZG_DTYPE_BF16: return launch_adamw_bits<P, __nv_bfloat16>(bits, t, c);
        default: return launch_adamw_bits<P, __half>(bits, t, c);
    }
}

bool float_dtype(uint32_t d) {
    return d == ZG_DTYPE_F32 || d == ZG_DTYPE_F16 || d == ZG_DTYPE_BF16;
}

uint64_t elem_bytes(uint32_t d) { return d == ZG_DTYPE_F32 ? 4 : 2; }
bool misaligned(const void* p, uint64_t a) { return reinterpret_cast<uintptr_t>(p) % a != 0; }

template <int CAP, class G>
int launch_norm_table(const NormTensor* t, int count, int64_t chunk, int grid, double* partial,
                      cudaStream_t s) {
    Table<CAP, NormTensor> tab;
    fill(tab, t, count, chunk);
    norm_partial_kernel<G, CAP><<<grid, kOptThreads, 0, s>>>(tab, chunk, partial);
    return cuda_status(cudaGetLastError(), "zg_grad_norm");
}

template <class G>
int launch_norm(const NormTensor* t, int count, int64_t chunk, int grid, double* partial,
                cudaStream_t s) {
    return count <= kSmallTable
               ? launch_norm_table<kSmallTable, G>(t, count, chunk, grid, partial, s)
               : launch_norm_table<kLargeTable, G>(t, count, chunk, grid, partial, s);
}

// Up to this many bytes of gradients one cluster reads them in less than a second
// launch costs: a call takes 7.7 us at 0.9 MB against 10.4 with two launches, and 12.4
// at 2.3 MB against 10.3.
constexpr uint64_t kNormClusterBytes = 1 << 20;

template <class G>
int launch_norm_cluster(const std::vector<NormTensor>& t, int64_t chunk, double max_norm, float* out,
                        cudaStream_t s) {
    Table<kSmallTable, NormTensor> tab;
    fill(tab, t.data(), static_cast<int>(t.size()), chunk);
    norm_cluster_kernel<G><<<kNormCluster, kNormThreads, 0, s>>>(tab, chunk, max_norm, out);
    return cuda_status(cudaGetLastError(), "zg_grad_norm");
}

// CTAs of one partial launch: at most 8 per SM of the largest part sold (so the
// workspace does not depend on the device).
constexpr int kNormGridMax = 8 * 160;

}  // namespace
}  // namespace zg

using namespace zg;

extern "C" int zg_adamw(uint32_t param_dtype, uint32_t grad_dtype, int state_bits,
                        uint32_t count, const zg_adamw_tensor* tensors, const zg_adamw_hyper* h,
                        const int64_t* step_dev, const float* lr_dev, const float* grad_scale_dev,
                        void* stream) try {
    if (!float_dtype(param_dtype) || !float_dtype(grad_dtype))
        return set_error(ZG_ERR_DISPATCH, "adamw: weights and gradients are f32, bf16 or f16, got dtypes %u and %u",
                         param_dtype, grad_dtype);
    if (state_bits != 32 && state_bits != 8)
        return set_error(ZG_ERR_DISPATCH, "adamw: moments have 32 or 8 bits, got %d", state_bits);
    if (!h || (count && !tensors)) return set_error(ZG_ERR_DISPATCH, "adamw: null argument");
    if (!(h->beta1 >= 0.0 && h->beta1 < 1.0 && h->beta2 >= 0.0 && h->beta2 < 1.0))
        return set_error(ZG_ERR_DISPATCH, "adamw: betas must be in [0, 1), got %g and %g", h->beta1,
                         h->beta2);
    if (!(h->eps >= 0.0) || !std::isfinite(h->eps) || !std::isfinite(h->weight_decay) ||
        (!lr_dev && !std::isfinite(h->lr)))
        return set_error(ZG_ERR_DISPATCH, "adamw: lr, eps and weight_decay must be finite, eps >= 0");
    if (!step_dev && h->step < 1)
        return set_error(ZG_ERR_DISPATCH, "adamw: steps count from 1, got %lld", (long long)h->step);
    std::vector<zg_adamw_tensor> used;
    used.reserve(count);
    uint64_t total = 0;
    for (uint32_t i = 0; i < count; ++i) {
        const zg_adamw_tensor& t = tensors[i];
        if (t.n == 0) continue;
        if (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq ||
            (state_bits == 8 && (!t.exp_avg_scale || !t.exp_avg_sq_scale)))
            return set_error(ZG_ERR_DISPATCH, "adamw: null pointer in tensor %u of %llu elements", i,
                             (unsigned long long)t.n);
        if (t.master && param_dtype == ZG_DTYPE_F32)
            return set_error(ZG_ERR_DISPATCH, "adamw: f32 weights take no master (tensor %u)", i);
        if (t.n >= 1ull << 40)
            return set_error(ZG_ERR_DISPATCH, "adamw: tensor %u has %llu elements", i,
                             (unsigned long long)t.n);
        if (misaligned(t.param, elem_bytes(param_dtype)) || misaligned(t.grad, elem_bytes(grad_dtype)) ||
            misaligned(t.master, 4) || misaligned(t.exp_avg_scale, 4) ||
            misaligned(t.exp_avg_sq_scale, 4) ||
            (state_bits == 32 && (misaligned(t.exp_avg, 4) || misaligned(t.exp_avg_sq, 4))))
            return set_error(ZG_ERR_DISPATCH, "adamw: a pointer of tensor %u is not aligned to its type", i);
        used.push_back(t);
        total += t.n;
    }
    if (used.empty()) return ZG_OK;
    AdamCall c;
    c.hyper = *h;
    c.dev = {step_dev, lr_dev, grad_scale_dev};
    c.f.b1 = static_cast<float>(h->beta1);
    c.f.c1 = static_cast<float>(1.0 - h->beta1);
    c.f.b2 = static_cast<float>(h->beta2);
    c.f.c2 = static_cast<float>(1.0 - h->beta2);
    // an eps above zero stays above zero, so that 0 / (0 + eps) is 0
    c.f.eps = h->eps > 0.0 ? std::max(static_cast<float>(h->eps), 0x1p-149f) : 0.0f;
    c.f.one = 1.0f;
    schedule(c.f, lr_dev ? 0.0 : h->lr, h->beta1, h->beta2, h->weight_decay,
             step_dev ? 1.0 : static_cast<double>(h->step));
    c.exact = h->eps < kTinyEps / sqrt(1.0 - h->beta2);
    c.chunk = chunk_elems(total);
    c.stream = static_cast<cudaStream_t>(stream);
    switch (param_dtype) {
        case ZG_DTYPE_F32: return launch_adamw_grad<float>(grad_dtype, state_bits, used, c);
        case ZG_DTYPE_BF16: return launch_adamw_grad<__nv_bfloat16>(grad_dtype, state_bits, used, c);
        default: return launch_adamw_grad<__half>(grad_dtype, state_bits, used, c);
    }
} catch (const std::exception& e) {  // the host ran out of memory for the table
    return set_error(ZG_ERR_BACKEND, "adamw: %s", e.what());
}

extern "C" uint64_t zg_grad_norm_workspace_bytes(uint32_t count) {
    const uint64_t launches = (static_cast<uint64_t>(count) + kLargeTable - 1) / kLargeTable;
    return launches * kNormGridMax * sizeof(double);
}

extern "C" int zg_grad_norm(uint32_t grad_dtype, uint32_t count, const void* const* grads,
                            const uint64_t* sizes, double max_norm, float* out, void* workspace,
                            uint64_t workspace_bytes, void* stream) try {
    if (!float_dtype(grad_dtype))
        return set_error(ZG_ERR_DISPATCH, "grad_norm: gradients are f32, bf16 or f16, got dtype %u",
                         grad_dtype);
    if (!out || (count && (!grads || !sizes)))
        return set_error(ZG_ERR_DISPATCH, "grad_norm: null argument");
    if (!(max_norm > 0.0))
        return set_error(ZG_ERR_DISPATCH, "grad_norm: max_norm must be above zero, got %g", max_norm);
    const uint64_t need = zg_grad_norm_workspace_bytes(count);
    if (need && (!workspace || workspace_bytes < need || misaligned(workspace, 8)))
        return set_error(ZG_ERR_DISPATCH,
                         "grad_norm: an 8-byte aligned workspace of %llu bytes is needed, got %llu",
                         (unsigned long long)need, (unsigned long long)workspace_bytes);
    std::vector<NormTensor> used;
    uint64_t total = 0;
    for (uint32_t i = 0; i < count; ++i) {
        if (sizes[i] == 0) continue;
        if (!grads[i] || misaligned(grads[i], elem_bytes(grad_dtype)) || sizes[i] >= 1ull << 40)
            return set_error(ZG_ERR_DISPATCH, "grad_norm: bad pointer or size in tensor %u", i);
        used.push_back({grads[i], sizes[i]});
        total += sizes[i];
    }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    double* partial = static_cast<double*>(workspace);
    const int64_t chunk = chunk_elems(total);
    if (!used.empty() && used.size() <= kSmallTable &&
        total * elem_bytes(grad_dtype) <= kNormClusterBytes) {
        // a share of the whole for each CTA, in whole turns
        const int64_t chunk = static_cast<int64_t>((total / kNormCluster / kTurnElems + 1) * kTurnElems);
        switch (grad_dtype) {
            case ZG_DTYPE_F32: return launch_norm_cluster<float>(used, chunk, max_norm, out, s);
            case ZG_DTYPE_BF16: return launch_norm_cluster<__nv_bfloat16>(used, chunk, max_norm, out, s);
            default: return launch_norm_cluster<__half>(used, chunk, max_norm, out, s);
        }
    }
    int parts = 0;
    for (size_t at = 0; at < used.size(); at += kLargeTable) {
        const int n = static_cast<int>(std::min<size_t>(used.size() - at, kLargeTable));
        uint64_t chunks = 0;
        for (int i = 0; i < n; ++i) chunks += (used[at + i].n + chunk - 1) / chunk;
        const int grid = static_cast<int>(std::min<uint64_t>(chunks, std::min(8 * sm_count(), kNormGridMax)));
        const NormTensor* t = used.data() + at;
        int rc;
        switch (grad_dtype) {
            case ZG_DTYPE_F32: rc = launch_norm<float>(t, n, chunk, grid, partial + parts, s); break;
            case ZG_DTYPE_BF16: rc = launch_norm<__nv_bfloat16>(t, n, chunk, grid, partial + parts, s); break;
            default: rc = launch_norm<__half>(t, n, chunk, grid, partial + parts, s); break;
        }
        if (rc) return rc;
        parts += grid;
    }
    norm_final_kernel<<<1, 1024, 0, s>>>(partial, parts, max_norm, out);
    return cuda_status(cudaGetLastError(), "zg_grad_norm");
} catch (const std::exception& e) {
    return set_error(ZG_ERR_BACKEND, "grad_norm: %s", e.what());
}
