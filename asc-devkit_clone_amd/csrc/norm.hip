// norm.hip -- residual addition, RMS norm and the 8-bit output with one scale per token, in one pass over the row.
//
//   h_c = rnd(x_c + r_c)        (rounded to x's type: what the residual stream stores is what is normed)
//   rstd = 1 / sqrt(sum_c h_c^2 / n + eps),  t_c = h_c gamma_c,  a = max_c |t_c|
//   q_c = rnd(t_c (Q (1 / a))),  scale = a rstd / Q        Q = 127 (int8), 448 (fp8 e4m3)
//   norm_c = rnd(t_c rstd)      (optional)
// The norm's factor rstd is common to a row, so it drops out of the codes: the sum of squares and the maximum come out of
// the same pass, and the codes need no second reduction.  h, t, the sum and the scale are fp32; the roundings are h's (the
// stored stream's type), the codes' and norm's.
// A row of zeros has codes and scale 0.  A row with a NaN, an infinity, or squares that pass fp32's range has codes 0 and
// scale NaN, so that its products are NaN and not some number.
#include "common.h"
#include "launch.h"

namespace ascq {

namespace {

__device__ __forceinline__ float round_to(float v, int dtype)
{
    if (dtype == DT_F16) return f16_to_f32(f32_to_f16_sat(v));
    if (dtype == DT_BF16) return bf16_to_f32(f32_to_bf16_sat(v));
    return v;
}

struct RowScale {
    float mult, scale, rstd;  // codes = rnd(t * mult); a row without a finite answer: mult 0, scale NaN
};
// top: the largest bits of |t| (a NaN's lie above every number's)
__device__ __forceinline__ RowScale row_scale(float ss, uint32_t top, float inv_n, float eps, float q_max)
{
    RowScale r;
    if (top >= 0x7f800000u || !(ss < __builtin_inff())) {
        r.mult = 0.0f;
        r.scale = r.rstd = __builtin_nanf("");
        return r;
    }
    const float a = __uint_as_float(top);
    r.rstd = top ? 1.0f / sqrtf(ss * inv_n + eps) : 0.0f;
    // (it passes fp32's range below a = 1.3e-36, where t times the largest number still is at most Q)
    r.mult = top ? fminf(q_max * (1.0f / a), 3.402823466e38f) : 0.0f;
    r.scale = a * r.rstd / q_max;
    return r;
}

// sum and bitwise maximum over a workgroup of NW waves
template <int NW>
__device__ __forceinline__ void block_reduce(float& ss, uint32_t& top)
{
    __shared__ float s_sum[NW];
    __shared__ uint32_t s_top[NW];
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        ss += __shfl_xor(ss, o, 64);
        const uint32_t other = (uint32_t)__shfl_xor((int)top, o, 64);
        top = other > top ? other : top;
    }
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
        s_sum[wave] = ss;
        s_top[wave] = top;
    }
    __syncthreads();
    ss = s_sum[0];
    top = s_top[0];
#pragma unroll
    for (int w = 1; w < NW; ++w) {
        ss += s_sum[w];
        top = s_top[w] > top ? s_top[w] : top;
    }
}

// Any n, strides and alignment: one workgroup per row, element by element, the row read twice (the second time from the
// caches).  h is taken from h_out the second time: it may lie where x or the residual lay.
__global__ __launch_bounds__(256) void norm_quant_any_kernel(NormQuantArgs a)
{
    const int64_t row = blockIdx.x;
    const int dt = a.src_type;
    auto first = [&](int64_t c) {
        const float x = load_f32_of(a.x, row * a.ldx + c, dt);
        return a.residual ? round_to(x + load_f32_of(a.residual, row * a.ldr + c, dt), dt) : x;
    };
    float ss = 0.0f;
    uint32_t top = 0;
    for (int64_t c = threadIdx.x; c < a.n; c += 256) {
        const float h = first(c);
        if (a.h_out) store_cast(a.h_out, row * a.ldh + c, h, dt);
        ss += h * h;
        const uint32_t t = __float_as_uint(h * load_f32_of(a.gamma, c, dt)) & 0x7fffffffu;
        top = t > top ? t : top;
    }
    block_reduce<4>(ss, top);
    const RowScale r = row_scale(ss, top, 1.0f / (float)a.n, a.eps, a.dst_type == DT_INT8 ? 127.0f : 448.0f);
    if (threadIdx.x == 0) a.scale_out[row] = r.scale;
    for (int64_t c = threadIdx.x; c < a.n; c += 256) {
        const float h = a.h_out ? load_f32_of(a.h_out, row * a.ldh + c, dt) : first(c);
        const float t = h * load_f32_of(a.gamma, c, dt);
        // (mult 0: a row of zeros, or one without an answer, whose products with 0 may be NaN)
        const float v = r.mult == 0.0f ? 0.0f : t * r.mult;
        if (a.dst_type == DT_INT8) ((int8_t*)a.q)[row * a.n + c] = (int8_t)quant_s8<RM_RINT>(v);
        else ((uint8_t*)a.q)[row * a.n + c] = f32_to_fp8(v, 0);
        if (a.norm_out) store_cast(a.norm_out, row * a.n + c, t * r.rstd, dt);
    }
}

}  // namespace

hipError_t launch_norm_quant(const NormQuantArgs& a, hipStream_t st)
{
    launch_k(norm_quant_any_kernel, dim3((unsigned)a.m), dim3(256), 0u, st, a);
    return hipGetLastError();
}

}  // namespace ascq
