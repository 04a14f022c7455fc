// gk_act.cuh - activations of the linear operator and their derivatives.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/gk.h"

namespace gk {

// Activations of values that end in 16 bits are evaluated to about 2^-20 of
// themselves (a 16-bit type keeps 2^-9 or 2^-12); those of fp32 with CUDA's
// erff and expf. (Below 2^-126 the quick exponential and reciprocal are 0, and so is silu from -87.4 on, where
// its value is below 2^-119 in size.) The quick gelu has one exponential for both of its parts:
//   Phi(-a) = e^(-a^2/2) t Q(t) / 2,  t = 1 / (1 + 0.45 a / sqrt 2),  a >= 0,
// with Q the degree-7 minimax fit of erfc(x) e^(x^2) / t over x in [0, 9.5]
// (relative error 3e-7), so the far negative side keeps its relative accuracy.
__device__ __forceinline__ float quick_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float quick_rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Phi(z); e = e^(-z^2/2).
__device__ __forceinline__ float quick_cdf(float z, float& e) {
    const float t = quick_rcp(fmaf(fabsf(z), 0.31819805153394639f, 1.0f));
    e = quick_ex2(z * z * -0.72134752044448170f);
    float q = 0.06631925f;
    q = fmaf(q, t, -0.23788772f);
    q = fmaf(q, t, 0.20455141f);
    q = fmaf(q, t, 0.04441312f);
    q = fmaf(q, t, 0.18637764f);
    q = fmaf(q, t, 0.22879136f);
    q = fmaf(q, t, 0.25351842f);
    q = fmaf(q, t, 0.25391682f);
    const float tail = 0.5f * e * t * q;
    return z < 0.0f ? tail : 1.0f - tail;
}

template <bool QUICK>
__device__ __forceinline__ float act_value(float z, int act) {
    switch (act) {
        case GK_ACT_RELU: return z > 0.0f ? z : (z != z ? z : 0.0f);
        case GK_ACT_TANH: return tanhf(z);
        case GK_ACT_GELU:
            if (QUICK) {
                float e;
                return z * quick_cdf(z, e);
            }
            return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
        case GK_ACT_SILU:
            if (QUICK) return z * quick_rcp(1.0f + quick_ex2(z * -1.4426950408889634f));
            return z / (1.0f + expf(-z));
        default: return z;
    }
}

// Two floats in the halves of a register pair; an instruction on both rounds each like one of its own.
__device__ __forceinline__ uint64_t two(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void halves(uint64_t v, float& lo, float& hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float clamped_size(float z) {  // min(|z|, 32), NaN kept
    float r;
    asm("min.NaN.f32 %0, %1, 0f42000000;" : "=f"(r) : "f"(fabsf(z)));
    return r;
}
// e^(-a^2/2) and t Q(t) / 2 (see quick_cdf) for two a = min(|z|, 32), where both have long been 0 beyond.
__device__ __forceinline__ void quick_tails(uint64_t a, uint64_t& e, uint64_t& t, uint64_t& q) {
    float u0, u1, x0, x1;
    halves(fma2(a, two(0.31819805153394639f, 0.31819805153394639f), two(1.0f, 1.0f)), u0, u1);
    halves(mul2(mul2(a, two(-0.72134752044448170f, -0.72134752044448170f)), a), x0, x1);
    t = two(quick_rcp(u0), quick_rcp(u1)), e = two(quick_ex2(x0), quick_ex2(x1));
    q = two(0.5f * 0.06631925f, 0.5f * 0.06631925f);
    q = fma2(q, t, two(0.5f * -0.23788772f, 0.5f * -0.23788772f));
    q = fma2(q, t, two(0.5f * 0.20455141f, 0.5f * 0.20455141f));
    q = fma2(q, t, two(0.5f * 0.04441312f, 0.5f * 0.04441312f));
    q = fma2(q, t, two(0.5f * 0.18637764f, 0.5f * 0.18637764f));
    q = fma2(q, t, two(0.5f * 0.22879136f, 0.5f * 0.22879136f));
    q = fma2(q, t, two(0.5f * 0.25351842f, 0.5f * 0.25351842f));
    q = fma2(q, t, two(0.5f * 0.25391682f, 0.5f * 0.25391682f));
}
// The quick gelu for two values: z Phi(z) = (z + |z|) / 2 - |z| Phi(-|z|), which keeps
// the far negative side's relative accuracy, and NaN for -inf as the product has it.
__device__ __forceinline__ void quick_gelus(float& z0, float& z1) {
    const uint64_t a = two(clamped_size(z0), clamped_size(z1)), half = two(0.5f, 0.5f);
    uint64_t e, t, q;
    quick_tails(a, e, t, q);
    const uint64_t positive = fma2(two(fabsf(z0), fabsf(z1)), half, mul2(two(z0, z1), half));
    const uint64_t h = mul2(mul2(e, t), q);
    halves(fma2(mul2(a, two(-1.0f, -1.0f)), h, positive), z0, z1);
}
// The quick gelu's derivative Phi(z) + z phi(z) for two values. With a = |z| and
// h = e^(-a^2/2) (t Q(t) / 2 - a / sqrt(2 pi)) it is h for z < 0 and 1 - h for
// z > 0, which 1/2 + copysign(1/2 - h, z) is on both sides.
__device__ __forceinline__ void quick_gelu_slopes(float& z0, float& z1) {
    const uint64_t a = two(clamped_size(z0), clamped_size(z1));
    uint64_t e, t, q;
    quick_tails(a, e, t, q);
    const uint64_t h = mul2(e, fma2(q, t, mul2(a, two(-0.39894228040143268f, -0.39894228040143268f))));
    float d0, d1;
    halves(fma2(h, two(-1.0f, -1.0f), two(0.5f, 0.5f)), d0, d1);
    z0 = 0.5f + copysignf(d0, z0);
    z1 = 0.5f + copysignf(d1, z1);
}

// The derivative, from what the forward pass kept: relu takes the output y,
// tanh its value in fp32 (1 - y^2 of a rounded y near one has few right bits),
// gelu and silu the sum z before the activation.
template <bool QUICK>
__device__ __forceinline__ float act_slope(float kept, int act) {
    switch (act) {
        case GK_ACT_RELU: return kept > 0.0f ? 1.0f : 0.0f;
        case GK_ACT_TANH: return 1.0f - kept * kept;
        case GK_ACT_GELU: {
            // Far out z e^(-z^2/2) is 0, but inf * 0 is not; the clamp drops a NaN, which is added again.
            const float z = fminf(fmaxf(kept, -32.0f), 32.0f);
            const float not_a_number = kept != kept ? kept : 0.0f;
            if (QUICK) {
                float e;
                const float cdf = quick_cdf(z, e);
                return fmaf(z * 0.39894228040143268f, e, cdf) + not_a_number;
            }
            return 0.5f * (1.0f + erff(z * 0.70710678118654752f)) + z * expf(-0.5f * z * z) * 0.39894228040143268f +
                   not_a_number;
        }
        case GK_ACT_SILU: {
            const float s = QUICK ? quick_rcp(1.0f + quick_ex2(kept * -1.4426950408889634f))
                                  : 1.0f / (1.0f + expf(-kept));
            // At -inf s is 0 and s * z is not a number; the limit is 0. At +inf z (1 - s) is not one; the limit is 1.
            return s == 0.0f ? 0.0f : (s == 1.0f ? 1.0f : s * (1.0f + kept * (1.0f - s)));
        }
        default: return 1.0f;
    }
}

template <typename T>
__device__ __forceinline__ float as_float(T v);
template <>
__device__ __forceinline__ float as_float<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ float as_float<__half>(__half v) {
    return __half2float(v);
}
template <>
__device__ __forceinline__ float as_float<__nv_bfloat16>(__nv_bfloat16 v) {
    return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T rounded(float v);
template <>
__device__ __forceinline__ float rounded<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ __half rounded<__half>(float v) {
    return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 rounded<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

// 16-bit values whose type is known at run time.
__device__ __forceinline__ float load16(const void* p, int64_t i, bool bf16) {
    return bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i])
                : __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void unpack16(uint32_t v, bool bf16, float& lo, float& hi) {
    if (bf16) {
        lo = __uint_as_float(v << 16);
        hi = __uint_as_float(v & 0xffff0000u);
    } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v));
        lo = f.x, hi = f.y;
    }
}
__device__ __forceinline__ uint32_t pack16(float lo, float hi, bool bf16) {
    uint32_t v;
    if (bf16)
        *reinterpret_cast<__nv_bfloat162*>(&v) = __floats2bfloat162_rn(lo, hi);
    else
        *reinterpret_cast<__half2*>(&v) = __floats2half2_rn(lo, hi);
    return v;
}
__device__ __forceinline__ void store16(void* p, int64_t i, float v, bool bf16) {
    if (bf16)
        static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
    else
        static_cast<__half*>(p)[i] = __float2half_rn(v);
}

}  // namespace gk
