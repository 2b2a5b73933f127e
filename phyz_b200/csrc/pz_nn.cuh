// Device helpers shared by the recurrent-block operators' kernels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "pz_nn.h"

namespace pz {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }

// Rounding to the array's type, once, to nearest even.
template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) {
    return x;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) {
    return __float2bfloat16_rn(x);
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) {
    return __float2half_rn(x);
}

// The sigmoid by the approximate exp2 and reciprocal (2 ulp and 1 ulp each):
// within 2^-22 of itself near 1 and of e^z near 0; exactly 0 and 1 at the ends.
__device__ __forceinline__ float sigmoid_f32(float z) {
    float e, a;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(z * -1.4426950408889634f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(a) : "f"(1.0f + e));
    return a;
}

// tanh z = 2 sigmoid(2z) - 1; below 1/8, where that cancels, its series to z^7
// (the next term is under 2^-29 of it).
__device__ __forceinline__ float tanh_f32(float z) {
    const float q = z * z;
    const float s = z * fmaf(q, fmaf(q, fmaf(q, -17.0f / 315.0f, 2.0f / 15.0f), -1.0f / 3.0f), 1.0f);
    const float t = fmaf(2.0f, sigmoid_f32(2.0f * z), -1.0f);
    return fabsf(z) < 0.125f ? s : t;
}

constexpr float GELU_C = 0.7978845608028654f;  // sqrt(2 / pi)
constexpr float GELU_K = 0.044715f;

__device__ __forceinline__ float act_f32(float z, int act) {
    switch (act) {
        case PHYZB_ACT_RELU: return z > 0.0f || z != z ? z : 0.0f;
        case PHYZB_ACT_TANH: return tanh_f32(z);
        case PHYZB_ACT_SILU: return z * sigmoid_f32(z);
        // z (1 + tanh u) / 2 = z sigmoid(2u)
        case PHYZB_ACT_GELU: return z * sigmoid_f32(2.0f * GELU_C * (z + GELU_K * z * z * z));
        default: return z;
    }
}

// d act / dz
__device__ __forceinline__ float act_grad_f32(float z, int act) {
    switch (act) {
        case PHYZB_ACT_RELU: return z > 0.0f ? 1.0f : 0.0f;
        case PHYZB_ACT_TANH: {
            const float t = tanh_f32(z);
            return 1.0f - t * t;
        }
        case PHYZB_ACT_SILU: {
            const float s = sigmoid_f32(z);
            return s * (1.0f + z * (1.0f - s));
        }
        case PHYZB_ACT_GELU: {
            const float s = sigmoid_f32(2.0f * GELU_C * (z + GELU_K * z * z * z));
            return s + z * s * (1.0f - s) * 2.0f * GELU_C * (1.0f + 3.0f * GELU_K * z * z);
        }
        default: return 1.0f;
    }
}

}  // namespace pz
