// Element types and activations shared by the kernels of the tensor-core linear.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "sfb_common.cuh"

namespace sfb {

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(float v) { return v; }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }

// an element whose type is known at run time (a bias, a weight's gradient)
__device__ __forceinline__ float load_as(const void *p, int64_t i, int dtype) {
    if (dtype == SFB_F32) return static_cast<const float *>(p)[i];
    if (dtype == SFB_BF16) return to_f(static_cast<const __nv_bfloat16 *>(p)[i]);
    return to_f(static_cast<const __half *>(p)[i]);
}

__device__ __forceinline__ void store_as(void *p, int64_t i, int dtype, float v) {
    if (dtype == SFB_F32) static_cast<float *>(p)[i] = v;
    else if (dtype == SFB_BF16) static_cast<__nv_bfloat16 *>(p)[i] = from_f<__nv_bfloat16>(v);
    else static_cast<__half *>(p)[i] = from_f<__half>(v);
}

template <typename T, int N> struct alignas(N * sizeof(T)) Vec { T v[N]; };

__device__ __forceinline__ float rcp_fast(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// e^x as 2^(x log2 e): relative error about 2^-22 + |x| 2^-24, far below the
// half step of the 16-bit result (2^-9, 2^-12)
__device__ __forceinline__ float exp_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.44269504f));
    return r;
}

__device__ __forceinline__ float sigmoid_fast(float x) { return rcp_fast(1.0f + exp_fast(-x)); }

// Phi(z), the normal distribution's integral, and e^(-z^2/2): the rational
// approximation 7.1.26 of Abramowitz and Stegun's handbook to erf (absolute
// error 1.5e-7), taken on the tail so that Phi of a negative z does not cancel.
__device__ __forceinline__ void normal_parts(float z, float &big, float &e) {
    const float x = fabsf(z) * 0.70710678f;
    const float t = rcp_fast(fmaf(0.3275911f, x, 1.0f));
    e = exp_fast(-0.5f * z * z);
    float q = fmaf(1.061405429f, t, -1.453152027f);
    q = fmaf(q, t, 1.421413741f);
    q = fmaf(q, t, -0.284496736f);
    q = fmaf(q, t, 0.254829592f);
    const float tail = 0.5f * q * t * e;
    big = z < 0.0f ? tail : 1.0f - tail;
}

constexpr float kTanhC = 1.5957691216f;            // 2 sqrt(2 / pi)
constexpr float kTanhB = 0.044715f;

// act(z); gelu_tanh is z sigmoid(2 u) with u the tanh form's argument
template <int ACT>
__device__ __forceinline__ float activate(float z) {
    if constexpr (ACT == SFB_ACT_RELU) {
        return z < 0.0f ? 0.0f : z;                // a NaN stays one
    } else if constexpr (ACT == SFB_ACT_GELU) {
        float big, e;
        normal_parts(z, big, e);
        return z * big;
    } else if constexpr (ACT == SFB_ACT_GELU_TANH) {
        return z * sigmoid_fast(kTanhC * fmaf(kTanhB * z * z, z, z));
    } else if constexpr (ACT == SFB_ACT_SILU) {
        return z * sigmoid_fast(z);
    } else {
        return z;
    }
}

// act'(z)
template <int ACT>
__device__ __forceinline__ float slope(float z) {
    if constexpr (ACT == SFB_ACT_RELU) {
        return z > 0.0f ? 1.0f : 0.0f;
    } else if constexpr (ACT == SFB_ACT_GELU) {
        float big, e;
        normal_parts(z, big, e);
        return fmaf(z * 0.39894228f, e, big);
    } else if constexpr (ACT == SFB_ACT_GELU_TANH) {
        const float s = sigmoid_fast(kTanhC * fmaf(kTanhB * z * z, z, z));
        return fmaf(z * s * (1.0f - s), kTanhC * fmaf(3.0f * kTanhB * z, z, 1.0f), s);
    } else if constexpr (ACT == SFB_ACT_SILU) {
        const float s = sigmoid_fast(z);
        return s * fmaf(z, 1.0f - s, 1.0f);
    } else {
        return 1.0f;
    }
}

// Two pre-activations as the backward pass reads them: fp16 whatever the type of x
// (2^-12 of the value against bf16's 2^-9, at the same two bytes), held within
// fp16's range, where every activation has long reached its asymptote.  For relu a
// positive value must not become 0, which its slope would tell from it.
template <int ACT>
__device__ __forceinline__ uint32_t kept2(float a, float b) {
    if constexpr (ACT == SFB_ACT_RELU) {
        a = a > 0.0f ? fmaxf(a, 0x1p-24f) : a;
        b = b > 0.0f ? fmaxf(b, 0x1p-24f) : b;
    }
    uint32_t r;
    asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}

// runs f with the activation as a compile-time constant
template <typename F>
int with_activation(int act, F f) {
    switch (act) {
        case SFB_ACT_NONE: return f(std::integral_constant<int, SFB_ACT_NONE>{});
        case SFB_ACT_RELU: return f(std::integral_constant<int, SFB_ACT_RELU>{});
        case SFB_ACT_GELU: return f(std::integral_constant<int, SFB_ACT_GELU>{});
        case SFB_ACT_GELU_TANH: return f(std::integral_constant<int, SFB_ACT_GELU_TANH>{});
        case SFB_ACT_SILU: return f(std::integral_constant<int, SFB_ACT_SILU>{});
    }
    return set_error(SFB_EINVAL, "sf tensor linear: activation %d", act);
}

}  // namespace sfb
