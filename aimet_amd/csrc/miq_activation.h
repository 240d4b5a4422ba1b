// The activations of the matrix product's epilogue and their derivatives, in float32.
#ifndef MIQ_ACTIVATION_H
#define MIQ_ACTIVATION_H

#include "miq_common.h"

namespace miq
{
// 1 / (1 + e^-z), by the hardware's exponential and reciprocal (about 1 ulp each); 0 and 1 at the two infinities
__device__ __forceinline__ float sigmoid_fast(float z)
{
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.442695041f));
}

constexpr float kGeluTanhA = 0.7978845608028654f;    // sqrt(2 / pi)
constexpr float kGeluTanhB = 0.044715f;
constexpr float kSqrtHalf  = 0.7071067811865476f;
constexpr float kInvSqrt2Pi = 0.3989422804014327f;

template <int ACT>
__device__ __forceinline__ float act_value(float z)
{
    if (ACT == MIQ_ACT_RELU)
        return z < 0.f ? 0.f : z;   // NaN stays NaN
    if (ACT == MIQ_ACT_SILU)
        return z * sigmoid_fast(z);
    if (ACT == MIQ_ACT_GELU)
        return z * (0.5f + 0.5f * erff(z * kSqrtHalf));
    if (ACT == MIQ_ACT_GELU_TANH)   // (1 + tanh u) / 2 = sigmoid(2 u)
        return z * sigmoid_fast(2.f * kGeluTanhA * (z + kGeluTanhB * z * z * z));
    return z;
}

template <int ACT>
__device__ __forceinline__ float act_slope(float z)
{
    if (ACT == MIQ_ACT_RELU)
        return z <= 0.f ? 0.f : 1.f;
    if (ACT == MIQ_ACT_SILU)
    {
        const float s = sigmoid_fast(z);
        return s * (1.f + z * (1.f - s));
    }
    if (ACT == MIQ_ACT_GELU)
        return 0.5f + 0.5f * erff(z * kSqrtHalf) +
               z * kInvSqrt2Pi * __builtin_amdgcn_exp2f(z * z * (-0.5f * 1.442695041f));
    if (ACT == MIQ_ACT_GELU_TANH)
    {
        const float s = sigmoid_fast(2.f * kGeluTanhA * (z + kGeluTanhB * z * z * z));
        return s + z * s * (1.f - s) * 2.f * kGeluTanhA * (1.f + 3.f * kGeluTanhB * z * z);
    }
    return 1.f;
}
}   // namespace miq

#endif
