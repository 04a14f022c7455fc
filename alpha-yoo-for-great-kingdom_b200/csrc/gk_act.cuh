// gk_act.cuh - activations of the linear operator and their derivatives.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/gk.h"

namespace gk {

__device__ __forceinline__ float act_value(float z, int act) {
    switch (act) {
        case GK_ACT_RELU: return z > 0.0f ? z : (z != z ? z : 0.0f);
        case GK_ACT_TANH: return tanhf(z);
        case GK_ACT_GELU: return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
        case GK_ACT_SILU: return z / (1.0f + expf(-z));
        default: return z;
    }
}

// The derivative. relu and tanh take the output y, gelu and silu the sum z
// before the activation: the value that the forward pass kept for them.
__device__ __forceinline__ float act_slope(float kept, int act) {
    switch (act) {
        case GK_ACT_RELU: return kept > 0.0f ? 1.0f : 0.0f;
        case GK_ACT_TANH: return 1.0f - kept * kept;
        case GK_ACT_GELU: {
            // Far out z exp(-z^2/2) is 0, but inf * 0 is not.
            const float z = fminf(fmaxf(kept, -32.0f), 32.0f);
            return kept != kept ? kept
                                : 0.5f * (1.0f + erff(z * 0.70710678118654752f)) +
                                      z * expf(-0.5f * z * z) * 0.39894228040143268f;
        }
        case GK_ACT_SILU: {
            const float s = 1.0f / (1.0f + expf(-kept));
            // At -inf s is 0 and s * z is not a number; the limit is 0.
            return s == 0.0f ? 0.0f : s * (1.0f + kept * (1.0f - s));
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
