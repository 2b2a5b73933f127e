// Device helpers shared by the recurrent-block operators' kernels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

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

// 32 neighbours of an array whose elements are `stride` apart, n of them there
// (the others read 0 and are not written): by 32 or 16 bytes a time where they are
// contiguous and aligned.
__device__ __forceinline__ void load32b(const void* p, uint32_t* r) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "l"(p)
                 : "memory");
}
__device__ __forceinline__ void store32b(void* p, const uint32_t* r) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]),
                 "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
template <class T>
__device__ __forceinline__ void load32(const T* p, long long stride, int n, T* v) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    constexpr int W = 8 * sizeof(T);  // words in all
    if (stride == 1 && n == 32 && ((uintptr_t)p & 31) == 0) {
#pragma unroll
        for (int w = 0; w < W; w += 8) load32b((const uint32_t*)p + w, r + w);
    } else if (stride == 1 && n == 32 && ((uintptr_t)p & 15) == 0) {
#pragma unroll
        for (int w = 0; w < W; w += 4) {
            const uint4 q = *reinterpret_cast<const uint4*>((const uint32_t*)p + w);
            r[w] = q.x, r[w + 1] = q.y, r[w + 2] = q.z, r[w + 3] = q.w;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 32; e++) v[e] = e < n ? p[e * stride] : from_f32<T>(0.0f);
    }
}
template <class T>
__device__ __forceinline__ void store32(T* p, long long stride, int n, const T* v) {
    const uint32_t* r = reinterpret_cast<const uint32_t*>(v);
    constexpr int W = 8 * sizeof(T);
    if (stride == 1 && n == 32 && ((uintptr_t)p & 31) == 0) {
#pragma unroll
        for (int w = 0; w < W; w += 8) store32b((uint32_t*)p + w, r + w);
    } else if (stride == 1 && n == 32 && ((uintptr_t)p & 15) == 0) {
#pragma unroll
        for (int w = 0; w < W; w += 4)
            *reinterpret_cast<uint4*>((uint32_t*)p + w) = make_uint4(r[w], r[w + 1], r[w + 2], r[w + 3]);
    } else {
#pragma unroll
        for (int e = 0; e < 32; e++)
            if (e < n) p[e * stride] = v[e];
    }
}

// 32 values as 16 words of pairs, and back
__device__ __forceinline__ void pack32(const float* v, uint32_t* w, __nv_bfloat16) {
#pragma unroll
    for (int k = 0; k < 16; k++) {
        const __nv_bfloat162 p = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]);
        w[k] = *reinterpret_cast<const uint32_t*>(&p);
    }
}
__device__ __forceinline__ void pack32(const float* v, uint32_t* w, __half) {
#pragma unroll
    for (int k = 0; k < 16; k++) {
        const __half2 p = __floats2half2_rn(v[2 * k], v[2 * k + 1]);
        w[k] = *reinterpret_cast<const uint32_t*>(&p);
    }
}
__device__ __forceinline__ void pack32(const float* v, uint32_t* w, float) {
#pragma unroll
    for (int k = 0; k < 32; k++) w[k] = __float_as_uint(v[k]);
}
__device__ __forceinline__ void unpack32(const uint32_t* w, float* v, __half) {
#pragma unroll
    for (int k = 0; k < 16; k++) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
        v[2 * k] = f.x;
        v[2 * k + 1] = f.y;
    }
}
// v += the values
__device__ __forceinline__ void add32(const uint32_t* w, float* v, __nv_bfloat16) {
#pragma unroll
    for (int k = 0; k < 16; k++) {
        v[2 * k] += __uint_as_float(w[k] << 16);
        v[2 * k + 1] += __uint_as_float(w[k] & 0xffff0000u);
    }
}
__device__ __forceinline__ void add32(const uint32_t* w, float* v, __half) {
#pragma unroll
    for (int k = 0; k < 16; k++) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
        v[2 * k] += f.x;
        v[2 * k + 1] += f.y;
    }
}
__device__ __forceinline__ void add32(const uint32_t* w, float* v, float) {
#pragma unroll
    for (int k = 0; k < 32; k++) v[k] += __uint_as_float(w[k]);
}
// 8 neighbours, n of them there
__device__ __forceinline__ void load8(const float* p, int n, float* v) {
    if (n >= 8 && ((uintptr_t)p & 15) == 0) {
        *(float4*)v = *(const float4*)p;
        *(float4*)(v + 4) = *(const float4*)(p + 4);
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = e < n ? p[e] : 0.0f;
    }
}

// f with the activation as a constant
template <class F>
__device__ __forceinline__ void with_act(int act, F f) {
    switch (act) {
        case PHYZB_ACT_RELU: return f(std::integral_constant<int, PHYZB_ACT_RELU>());
        case PHYZB_ACT_TANH: return f(std::integral_constant<int, PHYZB_ACT_TANH>());
        case PHYZB_ACT_SILU: return f(std::integral_constant<int, PHYZB_ACT_SILU>());
        case PHYZB_ACT_GELU: return f(std::integral_constant<int, PHYZB_ACT_GELU>());
        default: return f(std::integral_constant<int, PHYZB_ACT_NONE>());
    }
}

constexpr float LOG2E = 1.4426950408889634f;

// the larger and the smaller one; a NaN stays a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}
__device__ __forceinline__ float min_nan(float a, float b) {
    float m;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}

// a = sigmoid(z) = 1 / (1 + e), e = 2^(-z log2 e), by the approximate exp2 and
// reciprocal (2 ulp and 1 ulp each), and shut = 1 - a = e a: as a difference from the
// rounded a it would be 6 % off at z = 16 and 0 from 17.4 on. e is cut at 2^120, so
// that e a stays 1 there: a is then 2^-120 instead of less, which no f32 sum of
// ordinary values shows. Exactly 1 and 0 for z from 88 on.
__device__ __forceinline__ void gate_f32(float z, float& a, float& shut) {
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(min_nan(z * -LOG2E, 120.0f)));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(a) : "f"(1.0f + e));
    shut = e * a;
}

// sigmoid(z / log2 e) of two values, s = 1 / (1 + e) with e = 2^-z, by one
// reciprocal, 1 / ((1 + e) (1 + f)): exp and reciprocal share a unit of a quarter of
// the lanes, and activations are what an epilogue takes longest over (146 of 478 us at
// 262144 x 1024 values, before it had sixteen warps). Exponents are cut at 60, so that
// the product stays finite: a sigmoid of less than 2^-60 is 2^-60. What multiplies it
// is bounded then (ACT_END).
__device__ __forceinline__ void sigmoid2_pair(float x, float y, float& e, float& f, float& s, float& t) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fminf(-x, 60.0f)));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(f) : "f"(fminf(-y, 60.0f)));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"((1.0f + e) * (1.0f + f)));
    s = r * (1.0f + f);
    t = r * (1.0f + e);
}

// tanh z = 2 sigmoid(2z) - 1 = 2 s - 1; below 1/8, where that cancels, its series to
// z^7 (the next term is under 2^-29 of it).
__device__ __forceinline__ float tanh_of(float z, float s) {
    const float q = z * z;
    const float p = z * fmaf(q, fmaf(q, fmaf(q, -17.0f / 315.0f, 2.0f / 15.0f), -1.0f / 3.0f), 1.0f);
    return fabsf(z) < 0.125f ? p : fmaf(2.0f, s, -1.0f);
}

constexpr float GELU_C = 0.7978845608028654f;  // sqrt(2 / pi)
constexpr float GELU_K = 0.044715f;

// What an activation's sigmoid is of, over log2 e: gelu(z) = z (1 + tanh u) / 2 =
// z sigmoid(2u), u = C (z + K z^3).
template <int ACT>
__device__ __forceinline__ float act_inner(float z) {
    if (ACT == PHYZB_ACT_TANH) return z * (2.0f * LOG2E);
    if (ACT == PHYZB_ACT_SILU) return z * LOG2E;
    return z * fmaf(z * z, 2.0f * LOG2E * GELU_C * GELU_K, 2.0f * LOG2E * GELU_C);
}
// |z| at which the exponent of SiLU's and GELU's sigmoid has come to the cut: from
// there on the activation is 0 or z and its slope 0 or 1, to 2^-54.
template <int ACT>
constexpr float ACT_END = ACT == PHYZB_ACT_GELU ? 7.5f : 42.0f;

// two values through the activation, in place (a NaN stays a NaN)
template <int ACT>
__device__ __forceinline__ void act_pair(float& x, float& y) {
    if (ACT == PHYZB_ACT_NONE) return;
    if (ACT == PHYZB_ACT_RELU) {
        x = x > 0.0f || x != x ? x : 0.0f;
        y = y > 0.0f || y != y ? y : 0.0f;
        return;
    }
    float e, f, s, t;
    sigmoid2_pair(act_inner<ACT>(x), act_inner<ACT>(y), e, f, s, t);
    x = ACT == PHYZB_ACT_TANH ? (x == x ? tanh_of(x, s) : x) : max_nan(x, -ACT_END<ACT>) * s;
    y = ACT == PHYZB_ACT_TANH ? (y == y ? tanh_of(y, t) : y) : max_nan(y, -ACT_END<ACT>) * t;
}
// d act / dz of two values. s (1 - s) is e s s: taken as a difference it is rounding
// alone where s is near 1, and GELU multiplies it by z^3, which is bounded by ACT_END
// (a NaN is not over it, and stays one). tanh's slope is even in z: of |z| its e falls
// to 0 and meets no cut.
template <int ACT>
__device__ __forceinline__ void act_grad_pair(float& x, float& y) {
    if (ACT == PHYZB_ACT_NONE) {
        x = y = 1.0f;
        return;
    }
    if (ACT == PHYZB_ACT_RELU) {
        x = x > 0.0f ? 1.0f : 0.0f;
        y = y > 0.0f ? 1.0f : 0.0f;
        return;
    }
    float e, f, s, t;
    auto inner = [](float z) { return act_inner<ACT>(ACT == PHYZB_ACT_TANH ? fabsf(z) : z); };
    sigmoid2_pair(inner(x), inner(y), e, f, s, t);
    auto slope = [](float z, float e, float s) {
        const float q = e * s * s;
        if (ACT == PHYZB_ACT_TANH) return z == z ? 4.0f * q : z;  // 1 - (2 s - 1)^2
        const float w = ACT == PHYZB_ACT_SILU ? z : z * fmaf(z * z, 6.0f * GELU_C * GELU_K, 2.0f * GELU_C);
        return fabsf(z) >= ACT_END<ACT> ? __saturatef(z) : fmaf(q, w, s);
    };
    x = slope(x, e, s);
    y = slope(y, f, t);
}

}  // namespace pz
