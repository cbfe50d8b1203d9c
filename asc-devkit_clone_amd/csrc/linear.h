// linear.h -- the epilogue of the quantised linear (linear.hip):
//   y = cast(act(acc w_scale[n] x_scale[m] + bias[n]) + residual[m, n])
// in fp32, in this order, one rounding at the end (f16 / bf16: nearest even, saturating).
#pragma once

#include "common.h"
#include "launch.h"

namespace ascq {

// GELU, x Phi(x) = x (1 - erfc(x / sqrt 2) / 2).  erfc by Abramowitz and Stegun 7.1.26, a polynomial of degree 5 in
// t = 1 / (1 + p z) times exp(-z^2): 1.5e-7 off at most, so x Phi(x) is within 1e-7 |x|.  The side with the small result is
// a product (-|x| erfc / 2), so it keeps its sign and falls to 0.
__device__ __forceinline__ float gelu_erf(float x)
{
    const float ax = fminf(__builtin_fabsf(x), 20.0f);  // (beyond, erfc is 0)
    const float z = ax * 0.70710678f;
    const float t = __builtin_amdgcn_rcpf(1.0f + 0.3275911f * z);
    const float poly = t * (0.254829592f + t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f))));
    const float tail = 0.5f * ax * poly * __expf(-z * z);
    return x >= 0.0f ? x - tail : (x < 0.0f ? -tail : x);
}
// x / (1 + exp(-x)): -0 as x -> -inf
__device__ __forceinline__ float silu(float x)
{
    return fmaxf(x, -200.0f) * __builtin_amdgcn_rcpf(1.0f + __expf(-x));
}
__device__ __forceinline__ float activate(float v, int act)
{
    switch (act) {
    case ACT_FASTER_GELU: return faster_gelu(v);
    case ACT_RELU: return v > 0.0f || v != v ? v : 0.0f;
    case ACT_GELU: return gelu_erf(v);
    case ACT_SILU: return silu(v);
    default: return v;
    }
}

}  // namespace ascq
