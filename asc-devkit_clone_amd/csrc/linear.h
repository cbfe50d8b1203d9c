// linear.h -- the epilogue of the quantised linear (linear.hip):
//   y = cast(act(acc w_scale[n] x_scale[m] + bias[n]) + residual[m, n])
// in fp32, in this order, one rounding at the end (f16 / bf16: nearest even; a finite value saturates, an infinity stays).
#pragma once

#include "common.h"
#include "launch.h"

namespace ascq {

// Activations of 16-bit outputs: the hardware's exponential and reciprocal, and a polynomial; their errors lie below a
// hundredth of the output's rounding.
// GELU, x Phi(x) = max(x, 0) - |x| Q(|x|), Q the normal tail: exp(-x^2 / 2) times the polynomial of degree 7 in t = 1 / (1 + 0.2
// |x|) that is least off relatively over 0 <= |x| <= 14 (1.2e-6; found by linear programming).  The side with the small result
// is the product alone, so it keeps its sign and its digits, and falls to 0.
__device__ __forceinline__ float gelu_erf(float x)
{
    const float ax = fminf(__builtin_fabsf(x), 20.0f);  // (beyond, the tail is 0)
    const float t = __builtin_amdgcn_rcpf(fmaf(0.2f, ax, 1.0f));
    float q = fmaf(0.27908108f, t, -0.38677869f);
    q = fmaf(q, t, 0.44687112f);
    q = fmaf(q, t, -0.12313594f);
    q = fmaf(q, t, 0.132517f);
    q = fmaf(q, t, 0.07109624f);
    q = fmaf(q, t, 0.08034985f);
    const float tail = ax * (q * t) * __builtin_amdgcn_exp2f(ax * ax * -0.72134752f);
    return (x < 0.0f ? 0.0f : x) - tail;
}
// x / (1 + exp(-b x)): -0 as x -> -inf (SiLU: b = 1, FasterGelu: 1.702).  Both sides times 2^-32, so that the reciprocal of a
// large denominator is a normal number for as long as the result is one.
__device__ __forceinline__ float swish(float x, float b)
{
    const float e = __builtin_amdgcn_exp2f(fmaf(x, -1.44269504f * b, -32.0f));
    return fmaxf(x, -200.0f) * 0x1p-32f * __builtin_amdgcn_rcpf(e + 0x1p-32f);
}
// The same for f32 outputs, to a few units of fp32 where the result is small too.  GELU: the tail as above, the polynomial of
// degree 8 that is least off relatively over 0 <= |x| <= 14 (1.3e-7; found by linear programming), and the square's rounding
// made up for in the exponential.  The others: exp(-|b x|) does not overflow.  (2048 x 8192 x 4096 int8 with SiLU 70 us, by
// the short forms 63, by a division 74.)
__device__ __forceinline__ float reciprocal(float d)  // d within 1 .. 2^100
{
    const float r = __builtin_amdgcn_rcpf(d);
    return fmaf(fmaf(-d, r, 1.0f), r, r);
}
__device__ __forceinline__ float gelu_f32(float x)
{
    const float ax = fminf(__builtin_fabsf(x), 14.5f);  // (beyond, the tail is 0)
    const float t = reciprocal(fmaf(0.3f, ax, 1.0f));
    float q = fmaf(0.035604458f, t, -0.15690421f);
    q = fmaf(q, t, 0.20582908f);
    q = fmaf(q, t, -0.053192466f);
    q = fmaf(q, t, 0.12829745f);
    q = fmaf(q, t, 0.099994525f);
    q = fmaf(q, t, 0.12074095f);
    q = fmaf(q, t, 0.11963014f);
    const float s = ax * ax, rest = fmaf(ax, ax, -s), e = expf(-0.5f * s);
    return (x < 0.0f ? 0.0f : x) - ax * (q * t) * fmaf(e, -0.5f * rest, e);
}
__device__ __forceinline__ float swish_f32(float x, float b)
{
    const float e = expf(-b * __builtin_fabsf(x));
    return fmaxf(x, -200.0f) * (x < 0.0f ? e : 1.0f) * reciprocal(1.0f + e);
}
template <bool F32>
__device__ __forceinline__ float activate(float v, int act)
{
    switch (act) {
    case ACT_FASTER_GELU: return F32 ? swish_f32(v, 1.702f) : swish(v, 1.702f);
    case ACT_RELU: return v > 0.0f || v != v ? v : 0.0f;
    case ACT_GELU: return F32 ? gelu_f32(v) : gelu_erf(v);
    case ACT_SILU: return F32 ? swish_f32(v, 1.0f) : swish(v, 1.0f);
    default: return v;
    }
}

// Eight neighbouring outputs of a row: the scaled sums with their bias, activated, plus the residual's eight, stored.  Rows
// may start at any element; a run that the row ends in goes element by element.
typedef u32x4 u32x4_any __attribute__((aligned(2)));

template <int OUT>
struct OutRun {
    static constexpr int W = OUT == DT_F32 ? 2 : 1, ES = OUT == DT_F32 ? 4 : 2;
    u32x4 w[W];
    __device__ __forceinline__ void load(const void* row, int64_t col, int count)
    {
        const uint8_t* p = (const uint8_t*)row + col * ES;
        if (count >= 8) {
#pragma unroll
            for (int i = 0; i < W; ++i) w[i] = ((const u32x4_any*)p)[i];
            return;
        }
        w[0] = w[W - 1] = (u32x4){0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (e >= count) continue;
            if constexpr (OUT == DT_F32) w[e / 4][e % 4] = ((const uint32_t*)p)[e];
            else w[0][e / 2] |= (uint32_t)((const uint16_t*)p)[e] << (16 * (e & 1));
        }
    }
    __device__ __forceinline__ float get(int e) const
    {
        if constexpr (OUT == DT_F32) return __uint_as_float(w[e / 4][e % 4]);
        const uint16_t b = (uint16_t)(w[0][e / 2] >> (16 * (e & 1)));
        return OUT == DT_F16 ? f16_to_f32(b) : bf16_to_f32(b);
    }
    __device__ __forceinline__ static void store(void* row, int64_t col, int count, const float (&f)[8])
    {
        uint8_t* p = (uint8_t*)row + col * ES;
        uint32_t d[8];
        if constexpr (OUT == DT_F32) {
#pragma unroll
            for (int e = 0; e < 8; ++e) d[e] = __float_as_uint(f[e]);
        } else {
            us2_t top = {0, 0};
#pragma unroll
            for (int e = 0; e < 4; ++e) d[e] = cvt_pair<OUT == DT_BF16>(f[2 * e], f[2 * e + 1], top);
            if (__builtin_expect(cvt_special<OUT == DT_BF16>(top), 0)) {
                auto one = [](float x) { return (uint32_t)f32_to_16_keep_inf<OUT == DT_BF16>(x); };
#pragma unroll
                for (int e = 0; e < 4; ++e) d[e] = one(f[2 * e]) | (one(f[2 * e + 1]) << 16);
            }
        }
        if (count >= 8) {
#pragma unroll
            for (int i = 0; i < W; ++i) ((u32x4_any*)p)[i] = (u32x4){d[4 * i], d[4 * i + 1], d[4 * i + 2], d[4 * i + 3]};
            return;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (e >= count) continue;
            if constexpr (OUT == DT_F32) ((uint32_t*)p)[e] = d[e];
            else ((uint16_t*)p)[e] = (uint16_t)(d[e / 2] >> (16 * (e & 1)));
        }
    }
};

// f(activation) once, whatever the activation: the branch is taken for many elements together
template <bool F32, class F>
__device__ __forceinline__ void activation(int act, F f)
{
    if (act == ACT_NONE) return;
    if (act == ACT_RELU) f([](float x) { return activate<F32>(x, ACT_RELU); });
    else if (act == ACT_GELU) f([](float x) { return activate<F32>(x, ACT_GELU); });
    else {
        const float b = act == ACT_SILU ? 1.0f : 1.702f;
        f([b](float x) { return F32 ? swish_f32(x, b) : swish(x, b); });
    }
}

// sums -> z = sum w_scale x_scale + bias (-0.0f for none: adding it changes nothing) -> act(z), eight at a time
template <bool F32, class A>
__device__ __forceinline__ void activate8(const A (&acc)[8], const float (&ws)[8], float xs, const float (&bias)[8], int act,
                                          float (&v)[8])
{
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)acc[e] * ws[e] * xs + bias[e];
    activation<F32>(act, [&](auto f) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = f(v[e]);
    });
}

}  // namespace ascq
