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
constexpr float kInvSqrt2Pi = 0.3989422804014327f;

// The normal distribution's Phi(z), and e^(-z^2 / 2) on the way.  For z >= 0, 1 - Phi(z) = e^(-z^2 / 2) t P(t) with
// t = 1 / (1 + z / 4): e^(z^2 / 2) (1 - Phi) is smooth and falls like 1 / z, so a polynomial in t fits it evenly.  P is
// a weighted minimax fit of degree 6 made for this: off by less than 7e-9 in Phi, and by 7e-5 relative in the far
// tail; float32 rounding makes it 2e-7.  erff, for comparison, branches and costs three times as much, which on a
// 256 x 256 tile is as long as a fifth of the product.
__device__ __forceinline__ float normal_cdf(float z, float* gauss)
{
    const float a = fabsf(z), t = __builtin_amdgcn_rcpf(fmaf(a, 0.25f, 1.0f));
    const float e = __builtin_amdgcn_exp2f(z * z * (-0.5f * 1.442695041f));
    float q       = fmaf(t, -0.0933536159454298f, 0.3494622507254152f);
    q             = fmaf(t, q, -0.2813076718914251f);
    q             = fmaf(t, q, 0.2946804801960917f);
    q             = fmaf(t, q, 0.01788529050749215f);
    q             = fmaf(t, q, 0.11399742731721382f);
    q             = fmaf(t, q, 0.09863585623998446f);
    q *= t * e;
    *gauss = e;
    return z > 0.f ? 1.0f - q : q;   // NaN: q is one
}

template <int ACT>
__device__ __forceinline__ float act_value(float z)
{
    if (ACT == MIQ_ACT_RELU)
        return z < 0.f ? 0.f : z;   // NaN stays NaN
    if (ACT == MIQ_ACT_SILU)
        return z * sigmoid_fast(z);
    if (ACT == MIQ_ACT_GELU)
    {
        float e;
        return z * normal_cdf(z, &e);
    }
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
    {
        float e;
        const float phi = normal_cdf(z, &e);
        return fmaf(z * kInvSqrt2Pi, e, phi);
    }
    if (ACT == MIQ_ACT_GELU_TANH)
    {
        const float s = sigmoid_fast(2.f * kGeluTanhA * (z + kGeluTanhB * z * z * z)), d = s * (1.f - s);
        // (far out d is 0, and z^2 may be infinite)
        return d == 0.f ? s : s + z * d * 2.f * kGeluTanhA * (1.f + 3.f * kGeluTanhB * z * z);
    }
    return 1.f;
}
}   // namespace miq

#endif
