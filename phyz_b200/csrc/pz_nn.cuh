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

// sigmoid(z), right at both ends: exp(-z) overflows to inf, which gives 0.
__device__ __forceinline__ float sigmoid_f32(float z) { return 1.0f / (1.0f + expf(-z)); }

constexpr float GELU_C = 0.7978845608028654f;  // sqrt(2 / pi)
constexpr float GELU_K = 0.044715f;

__device__ __forceinline__ float act_f32(float z, int act) {
    switch (act) {
        case PHYZB_ACT_RELU: return z > 0.0f || z != z ? z : 0.0f;
        case PHYZB_ACT_TANH: return tanhf(z);
        case PHYZB_ACT_SILU: return z * sigmoid_f32(z);
        case PHYZB_ACT_GELU: return 0.5f * z * (1.0f + tanhf(GELU_C * (z + GELU_K * z * z * z)));
        default: return z;
    }
}

// d act / dz
__device__ __forceinline__ float act_grad_f32(float z, int act) {
    switch (act) {
        case PHYZB_ACT_RELU: return z > 0.0f ? 1.0f : 0.0f;
        case PHYZB_ACT_TANH: {
            const float t = tanhf(z);
            return 1.0f - t * t;
        }
        case PHYZB_ACT_SILU: {
            const float s = sigmoid_f32(z);
            return s * (1.0f + z * (1.0f - s));
        }
        case PHYZB_ACT_GELU: {
            const float t = tanhf(GELU_C * (z + GELU_K * z * z * z));
            return 0.5f * (1.0f + t) + 0.5f * z * (1.0f - t * t) * GELU_C * (1.0f + 3.0f * GELU_K * z * z);
        }
        default: return 1.0f;
    }
}

}  // namespace pz
