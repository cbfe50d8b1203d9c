// linear.hip -- the quantised linear: 8-bit activations with one scale per token times an 8-bit weight with one scale per
// channel, and bias, activation and residual in the epilogue (linear.h).  int8 sums are exact (int32); fp8 e4m3 sums are
// fp32.
#include "linear.h"

#include "gemm_core.h"

namespace ascq {

namespace {

// 16 bytes of a row that has n of them left (n <= 0: none), zeros behind; src + 16 may lie past the operand
__device__ __forceinline__ u32x4 load16_any(const uint8_t* src, int64_t n, bool aligned)
{
    if (n >= 16 && aligned) return *(const u32x4*)src;
    u32x4 v = {0, 0, 0, 0};
#pragma unroll
    for (int b = 0; b < 16; ++b)
        if (b < n) v[b / 4] |= (uint32_t)src[b] << (8 * (b % 4));
    return v;
}

// Any shape, stride and alignment, 64-bit addresses: 64 x 64 tiles, one stage of 64 K at a time through LDS, a [K, N]
// weight turned on the way.
template <bool F8>
__global__ __launch_bounds__(256) void linear_any_kernel(LinearArgs a)
{
    constexpr int P = 80;  // bytes of a row in LDS: 64, and 16 that spread the rows over the banks
    __shared__ __attribute__((aligned(16))) uint8_t sx[64 * P], sw[64 * P];
    typedef typename std::conditional<F8, v4f, v4i>::type acc_t;
    const int64_t tiles_n = (a.N + 63) / 64;
    const int64_t m0 = (int64_t)blockIdx.x / tiles_n * 64, n0 = (int64_t)blockIdx.x % tiles_n * 64;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, wm = wave >> 1, wn = wave & 1;
    const int r = t >> 2, c = (t & 3) * 16;
    const bool ax = ((uintptr_t)a.x | (uintptr_t)a.ldx) % 16 == 0, aw = ((uintptr_t)a.w | (uintptr_t)a.ldw) % 16 == 0;
    acc_t acc[2][2] = {};
    for (int64_t k0 = 0; k0 < a.K; k0 += 64) {
        const u32x4 vx = load16_any(a.x + (m0 + r) * a.ldx + k0 + c, m0 + r < a.M ? a.K - k0 - c : 0, ax);
        u32x4 vw;
        if (a.w_trans) vw = load16_any(a.w + (n0 + r) * a.ldw + k0 + c, n0 + r < a.N ? a.K - k0 - c : 0, aw);
        else vw = load16_any(a.w + (k0 + r) * a.ldw + n0 + c, k0 + r < a.K ? a.N - n0 - c : 0, aw);
        __syncthreads();
        *(u32x4*)(sx + r * P + c) = vx;
        if (a.w_trans) {
            *(u32x4*)(sw + r * P + c) = vw;
        } else {
#pragma unroll
            for (int b = 0; b < 16; ++b) sw[(c + b) * P + r] = (uint8_t)(vw[b / 4] >> (8 * (b % 4)));
        }
        __syncthreads();
        v4i fx[2], fw[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            fx[i] = *(const v4i*)(sx + (wm * 32 + i * 16 + (lane & 15)) * P + (lane >> 4) * 16);
            fw[i] = *(const v4i*)(sw + (wn * 32 + i * 16 + (lane & 15)) * P + (lane >> 4) * 16);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                if constexpr (F8) {
                    typedef long v2l __attribute__((ext_vector_type(2)));
                    const v2l p = __builtin_bit_cast(v2l, fx[i]), q = __builtin_bit_cast(v2l, fw[j]);
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_fp8_fp8(p[0], q[0], acc[i][j], 0, 0, 0);
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_fp8_fp8(p[1], q[1], acc[i][j], 0, 0, 0);
                } else {
                    acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fx[i], fw[j], acc[i][j], 0, 0, 0);
                }
            }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int64_t m = m0 + wm * 32 + i * 16 + 4 * (lane >> 4) + e, n = n0 + wn * 32 + j * 16 + (lane & 15);
                if (m >= a.M || n >= a.N) continue;
                float v = (float)acc[i][j][e] * a.w_scale[n] * a.x_scale[m];
                if (a.bias) v += a.bias[n];
                v = activate(v, a.act);
                if (a.residual) v += load_f32_of(a.residual, m * a.ldr + n, a.out_type);
                store_cast(a.y, m * a.ldy + n, v, a.out_type);
            }
}

}  // namespace

hipError_t launch_linear(const LinearArgs& a, hipStream_t st)
{
    const dim3 grid((unsigned)(((a.M + 63) / 64) * ((a.N + 63) / 64)));
    if (a.f8) launch_k(linear_any_kernel<true>, grid, dim3(256), 0u, st, a);
    else launch_k(linear_any_kernel<false>, grid, dim3(256), 0u, st, a);
    return hipGetLastError();
}

}  // namespace ascq
