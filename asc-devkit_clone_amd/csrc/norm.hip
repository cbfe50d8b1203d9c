// norm.hip -- residual addition, RMS norm and the 8-bit output with one scale per token, in one pass over the row.
//
//   h_c = rnd(x_c + r_c)        (rounded to x's type: what the residual stream stores is what is normed)
//   rstd = 1 / sqrt(sum_c h_c^2 / n + eps),  t_c = h_c gamma_c,  a = max_c |t_c|
//   q_c = rnd(t_c (Q (1 / a))),  scale = a rstd / Q        Q = 127 (int8), 448 (fp8 e4m3)
//   norm_c = rnd(t_c rstd)      (optional)
// The norm's factor rstd is common to a row, so it drops out of the codes: the sum of squares and the maximum come out of
// the same pass, and the codes need no second reduction.  h, t, the sum and the scale are fp32; the roundings are h's (the
// stored stream's type), the codes' and norm's.
// Bound by memory: 8192 x 8192 bf16 with residual to e4m3 in 77 us, 6.1 TB/s of the bytes it cannot do without; f32 4.9 TB/s
// (4096 x 8192: 88 us); rows that start at any element 4.3 (8192 x 8191: 110 us).  A decode step's 16 x 4096 takes 3.5 us.
// A row of zeros has codes and scale 0.  A row with a NaN, an infinity (which h keeps: only a finite sum saturates), or squares
// that pass fp32's range has codes 0 and scale NaN, so that its products are NaN and not some number.
#include <type_traits>

#include "common.h"
#include "launch.h"

namespace ascq {

namespace {

__device__ __forceinline__ float round_to(float v, int dtype)
{
    if (dtype == DT_F16) return f16_to_f32(f32_to_16_keep_inf<false>(v));
    if (dtype == DT_BF16) return bf16_to_f32(f32_to_16_keep_inf<true>(v));
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
    r.mult = top ? q_max * (1.0f / a) : 0.0f;
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
    __syncthreads();  // (the row before, or this one's first sums, have been read)
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

// Rows whose products t lie below 2^-100 (1 / a and the scale would leave fp32's range), or whose mean square does (squares
// would: only with an eps as small), are done here from memory, with products times 2^100, h times 2^90, or both; the powers go
// back into the scale and the norm.  (A row whose products all are 0 in fp32 is an ordinary row of zeros.)  Each thread has the
// RUN-element pieces threadIdx.x, threadIdx.x + NT, ..., as when it stored h.
enum : int { SMALL_T = 1, SMALL_H = 2 };
__device__ __forceinline__ int small_powers(float ss, uint32_t top, float inv_n, float eps)
{
    const int p = top == 0 ? 0 : (top < 0x0d800000u ? SMALL_T : 0) | (ss * inv_n + eps < 0x1p-100f ? SMALL_H : 0);  // (2^-100)
    return __builtin_amdgcn_readfirstlane(p);
}
template <int NT, int RUN>
__device__ __forceinline__ void finish_small_row(const NormQuantArgs& a, int dt, int64_t row, int small, float inv_n)
{
    const bool small_t = small & SMALL_T, small_h = small & SMALL_H;
    auto each = [&](auto f) {
#pragma unroll 1
        for (int64_t c = threadIdx.x; c * RUN < a.n; c += NT)
#pragma unroll 1
            for (int64_t i = c * RUN; i < c * RUN + RUN && i < a.n; ++i) {
                float h;
                if (a.h_out) h = load_f32_of(a.h_out, row * a.ldh + i, dt);  // (x or the residual may be gone)
                else {
                    h = load_f32_of(a.x, row * a.ldx + i, dt);
                    if (a.residual) h = round_to(h + load_f32_of(a.residual, row * a.ldr + i, dt), dt);
                }
                const float g = load_f32_of(a.gamma, i, dt);
                const float k = small_h ? h * 0x1p90f : h;
                // (no factor overflows: |h g| < 2^-100)
                f(i, k, !small_t ? h * g : __builtin_fabsf(g) < 1.0f ? k * (g * 0x1p100f) : k * 0x1p100f * g);
            }
    };
    float ss = 0.0f;
    uint32_t top = 0;
    each([&](int64_t, float h, float t) {
        ss = fmaf(h, h, ss);
        const uint32_t b = __float_as_uint(t) & 0x7fffffffu;
        top = b > top ? b : top;
    });
    block_reduce<NT / 64>(ss, top);
    const bool int8 = a.dst_type == DT_INT8;
    const float q_max = int8 ? 127.0f : 448.0f;
    const RowScale s = row_scale(ss, top, inv_n, small_h ? a.eps * 0x1p90f * 0x1p90f : a.eps, q_max);
    // t rstd in an order that leaves fp32's range only if the result does
    const float power = small_t ? 0x1p-100f : 0x1p90f;
    auto normed = [&](float t) {
        return (__builtin_fabsf(t) < 1.0f) == (power > 1.0f) ? t * power * s.rstd : t * s.rstd * power;
    };
    const float scale = normed(__uint_as_float(top)) / q_max;
    if (threadIdx.x == 0) a.scale_out[row] = scale;
    each([&](int64_t i, float, float t) {
        const float v = scale > 0.0f ? t * s.mult : 0.0f;
        if (int8) ((int8_t*)a.q)[row * a.n + i] = (int8_t)quant_s8<RM_RINT>(v);
        else ((uint8_t*)a.q)[row * a.n + i] = f32_to_fp8(v, 0);
        if (a.norm_out) store_keep_inf(a.norm_out, row * a.n + i, normed(t), dt);
    });
}

// 16 (8) bytes at any element's (byte's) address: the memory pipeline takes wide accesses of any alignment
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef u32x2 u32x2_any __attribute__((aligned(1)));

// A unit is 8 elements of a row: 16 bytes of a 16-bit type, 32 of f32.
template <int T>
struct Unit {
    static constexpr int W = T == DT_F32 ? 2 : 1;  // 16-byte words
    u32x4 w[W];
    __device__ __forceinline__ float get(int e) const
    {
        if constexpr (T == DT_F32) return __uint_as_float(w[e / 4][e % 4]);
        const uint32_t d = w[0][e / 2];
        const uint16_t b = (uint16_t)(e & 1 ? d >> 16 : d);
        return T == DT_F16 ? f16_to_f32(b) : bf16_to_f32(b);
    }
    // the unit of eight floats, rounded (16-bit types: nearest even; what is finite saturates)
    __device__ __forceinline__ void set(const float (&f)[8])
    {
        if constexpr (T == DT_F32) {
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e / 4][e % 4] = __float_as_uint(f[e]);
        } else {
            us2_t top = {0, 0};
#pragma unroll
            for (int e = 0; e < 4; ++e) w[0][e] = cvt_pair<T == DT_BF16>(f[2 * e], f[2 * e + 1], top);
            if (__builtin_expect(cvt_special<T == DT_BF16>(top), 0)) {
                auto one = [](float x) { return (uint32_t)f32_to_16_keep_inf<T == DT_BF16>(x); };
#pragma unroll
                for (int e = 0; e < 4; ++e) w[0][e] = one(f[2 * e]) | (one(f[2 * e + 1]) << 16);
            }
        }
    }
    template <bool ANY>
    __device__ __forceinline__ void load(const void* row, uint32_t unit)
    {
        typedef typename std::conditional<ANY, u32x4_any, u32x4>::type word_t;
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = __builtin_nontemporal_load((const word_t*)row + unit * W + i);
    }
    template <bool ANY>
    __device__ __forceinline__ void store(void* row, uint32_t unit) const
    {
        typedef typename std::conditional<ANY, u32x4_any, u32x4>::type word_t;
#pragma unroll
        for (int i = 0; i < W; ++i) __builtin_nontemporal_store(w[i], (word_t*)row + unit * W + i);
    }
    // the first `count` elements, zeros behind
    __device__ __forceinline__ void load_part(const void* row, uint32_t unit, int count)
    {
        w[0] = w[W - 1] = (u32x4){0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (e >= count) continue;
            if constexpr (T == DT_F32) w[e / 4][e % 4] = ((const uint32_t*)row)[unit * 8 + e];
            else w[0][e / 2] |= (uint32_t)((const uint16_t*)row)[unit * 8 + e] << (16 * (e & 1));
        }
    }
    __device__ __forceinline__ void store_part(void* row, uint32_t unit, int count) const
    {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (e >= count) continue;
            if constexpr (T == DT_F32) ((uint32_t*)row)[unit * 8 + e] = w[e / 4][e % 4];
            else ((uint16_t*)row)[unit * 8 + e] = (uint16_t)(w[0][e / 2] >> (16 * (e & 1)));
        }
    }
};

// Eight codes of values within the largest code (up to the fp32 roundings in front, which stay below the next one).
// int8: adding 1.5 x 2^23 leaves the nearest integer, ties to even, in the low bits.
__device__ __forceinline__ u32x2 codes8(const float (&v)[8], bool int8)
{
    u32x2 o;
    if (int8) {
        uint32_t b[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) b[e] = __float_as_uint(v[e] + 12582912.0f);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t lo = __builtin_amdgcn_perm(b[4 * h + 1], b[4 * h], 0x0c0c0400u);
            const uint32_t hi = __builtin_amdgcn_perm(b[4 * h + 3], b[4 * h + 2], 0x04000c0cu);
            o[h] = lo | hi;
        }
    } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            int d = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h], v[4 * h + 1], 0, false);
            o[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h + 2], v[4 * h + 3], d, true);
        }
    }
    return o;
}

// One workgroup of NT threads per row, U units per thread, which hold the row (and gamma) in registers between the reduction
// and the codes, so every byte moves once.  All loads of a thread are issued in front of its first wait: units past the
// row read its last whole one and are dropped (in place, another thread may have stored it by then).
// ANY: rows that start at any element, whose last unit may be a part of one.
// waves_per_simd: bf16 and f32, 1024 threads of four 16-byte words, in 64 registers, which are two workgroups per CU (bf16 2048 x
// 32768 with residual 81 us, in the 70 that it takes by itself 88).
template <int T, int NT, int U>
constexpr int waves_per_simd = T != DT_F16 && NT == 1024 && U * Unit<T>::W <= 4 ? 8 : 1;
template <int T, int NT, int U, bool RES, bool ANY>
__global__ __launch_bounds__(NT, (waves_per_simd<T, NT, U>)) void norm_quant_row_kernel(NormQuantArgs a)
{
    const int64_t row = blockIdx.x;
    const uint32_t whole = (uint32_t)(a.n / 8), units = ANY ? (uint32_t)((a.n + 7) / 8) : whole;
    const int part = ANY ? (int)(a.n % 8) : 0;
    constexpr int ES = T == DT_F32 ? 4 : 2;
    const uint8_t* x = (const uint8_t*)a.x + row * a.ldx * ES;
    const uint8_t* r = (const uint8_t*)a.residual + (RES ? row * a.ldr * ES : 0);
    Unit<T> h[U], g[U], add[RES ? U : 1];
    if (!ANY || whole > 0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t c = threadIdx.x + u * NT, k = c < whole ? c : whole - 1;
            h[u].template load<ANY>(x, k);
            if constexpr (RES) add[u].template load<ANY>(r, k);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            typedef typename std::conditional<ANY, u32x4_any, u32x4>::type word_t;
            const uint32_t c = threadIdx.x + u * NT, k = c < whole ? c : whole - 1;
#pragma unroll
            for (int i = 0; i < Unit<T>::W; ++i) g[u].w[i] = ((const word_t*)a.gamma)[k * Unit<T>::W + i];
        }
    }
    float ss = 0.0f;
    uint32_t top = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t c = threadIdx.x + u * NT;
        if (ANY && c == whole && part) {
            h[u].load_part(x, c, part);
            if constexpr (RES) add[u].load_part(r, c, part);
            g[u].load_part(a.gamma, c, part);
        }
        if constexpr (RES) {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = h[u].get(e) + add[u].get(e);
            h[u].set(f);
            if (a.h_out) {
                uint8_t* to = (uint8_t*)a.h_out + row * a.ldh * ES;
                if (c < whole) h[u].template store<ANY>(to, c);
                else if (ANY && c == whole) h[u].store_part(to, c, part);
            }
        }
        float sum = 0.0f;
        uint32_t most = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float v = h[u].get(e);
            sum = fmaf(v, v, sum);
            const uint32_t t = __float_as_uint(v * g[u].get(e)) & 0x7fffffffu;
            most = t > most ? t : most;
        }
        if (c < units) {
            ss += sum;
            top = most > top ? most : top;
        }
    }
    block_reduce<NT / 64>(ss, top);
    const float inv_n = 1.0f / (float)a.n;
    const int small = T == DT_F16 ? 0 : small_powers(ss, top, inv_n, a.eps);
    const bool int8 = a.dst_type == DT_INT8;
    const RowScale s = row_scale(ss, top, inv_n, a.eps, int8 ? 127.0f : 448.0f);
    if (threadIdx.x == 0) a.scale_out[row] = s.scale;
    uint8_t* q = (uint8_t*)a.q + row * a.n;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t c = threadIdx.x + u * NT;
        if (c >= units) break;
        float t[8], v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            t[e] = h[u].get(e) * g[u].get(e);
            // (mult 0: a row of zeros, or one without an answer, whose products with 0 may be NaN)
            v[e] = s.mult == 0.0f ? 0.0f : t[e] * s.mult;
        }
        const u32x2 codes = codes8(v, int8);
        if (!ANY || c < whole) {
            typedef typename std::conditional<ANY, u32x2_any, u32x2>::type codes_t;
            __builtin_nontemporal_store(codes, (codes_t*)q + c);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < part) q[c * 8 + e] = (uint8_t)(codes[e / 4] >> (8 * (e % 4)));
        }
        if (a.norm_out) {
#pragma unroll
            for (int e = 0; e < 8; ++e) t[e] *= s.rstd;
            Unit<T> o;
            o.set(t);
            uint8_t* to = (uint8_t*)a.norm_out + row * a.n * ES;
            if (!ANY || c < whole) o.template store<ANY>(to, c);
            else o.store_part(to, c, part);
        }
    }
    // over what was stored above, and behind it, where the row's registers are free (in front: long rows 9 % to 24 % slower).  f16
    // has no such rows: its smallest number's square is 2^-48.
    if constexpr (T != DT_F16)
        if (__builtin_expect(small, 0)) finish_small_row<NT, 8>(a, T, row, small, inv_n);
}

// Rows too long for registers: one workgroup per row, element by element, the row read twice (the second time from the
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
        if (a.h_out) store_keep_inf(a.h_out, row * a.ldh + c, h, dt);
        ss += h * h;
        const uint32_t t = __float_as_uint(h * load_f32_of(a.gamma, c, dt)) & 0x7fffffffu;
        top = t > top ? t : top;
    }
    block_reduce<4>(ss, top);
    const float inv_n = 1.0f / (float)a.n;
    if (const int small = small_powers(ss, top, inv_n, a.eps)) return finish_small_row<256, 1>(a, dt, row, small, inv_n);
    const RowScale r = row_scale(ss, top, inv_n, a.eps, a.dst_type == DT_INT8 ? 127.0f : 448.0f);
    if (threadIdx.x == 0) a.scale_out[row] = r.scale;
    for (int64_t c = threadIdx.x; c < a.n; c += 256) {
        const float h = a.h_out ? load_f32_of(a.h_out, row * a.ldh + c, dt) : first(c);
        const float t = h * load_f32_of(a.gamma, c, dt);
        // (mult 0: a row of zeros, or one without an answer, whose products with 0 may be NaN)
        const float v = r.mult == 0.0f ? 0.0f : t * r.mult;
        if (a.dst_type == DT_INT8) ((int8_t*)a.q)[row * a.n + c] = (int8_t)quant_s8<RM_RINT>(v);
        else ((uint8_t*)a.q)[row * a.n + c] = f32_to_fp8(v, 0);
        if (a.norm_out) store_keep_inf(a.norm_out, row * a.n + c, t * r.rstd, dt);
    }
}

}  // namespace

// The workgroup of a row: a thread holds up to 8 units (f32: 4)
template <int T, bool RES, bool ANY>
static bool launch_row(const NormQuantArgs& a, hipStream_t st)
{
    const int64_t units = (a.n + 7) / 8;
    const dim3 grid((unsigned)a.m);
#define ASCQ_NORM(NT, U)                                                                   \
    if (units <= NT * U) {                                                                 \
        launch_k((norm_quant_row_kernel<T, NT, U, RES, ANY>), grid, dim3(NT), 0u, st, a);  \
        return true;                                                                       \
    }
    ASCQ_NORM(64, 1)
    ASCQ_NORM(64, 2)
    ASCQ_NORM(256, 1)
    ASCQ_NORM(256, 2)
    if constexpr (T == DT_F32) {
        ASCQ_NORM(512, 2)
        ASCQ_NORM(1024, 2)
        ASCQ_NORM(1024, 4)
    } else {
        ASCQ_NORM(256, 4)
        ASCQ_NORM(256, 8)
        ASCQ_NORM(1024, 4)
        ASCQ_NORM(1024, 8)
    }
#undef ASCQ_NORM
    return false;
}
template <int T>
static bool launch_row_of(const NormQuantArgs& a, bool any, hipStream_t st)
{
    if (any) return a.residual ? launch_row<T, true, true>(a, st) : launch_row<T, false, true>(a, st);
    return a.residual ? launch_row<T, true, false>(a, st) : launch_row<T, false, false>(a, st);
}

static hipError_t launch_rows(const NormQuantArgs& a, hipStream_t st)
{
    const int64_t es = a.src_type == DT_F32 ? 4 : 2;
    const uintptr_t bits = (uintptr_t)a.x | (uintptr_t)a.residual | (uintptr_t)a.h_out | (uintptr_t)a.norm_out |
                           (uintptr_t)a.gamma | (uintptr_t)(a.ldx * es) | (uintptr_t)(a.residual ? a.ldr * es : 0) |
                           (uintptr_t)(a.h_out ? a.ldh * es : 0);
    const bool any = bits % 16 != 0 || (uintptr_t)a.q % 8 != 0 || a.n % 8 != 0;
    const bool done = a.src_type == DT_F16    ? launch_row_of<DT_F16>(a, any, st)
                      : a.src_type == DT_BF16 ? launch_row_of<DT_BF16>(a, any, st)
                                              : launch_row_of<DT_F32>(a, any, st);
    if (!done) {
        log_fallback("norm_quant_any_kernel", "rows too long for a workgroup's registers");
        launch_k(norm_quant_any_kernel, dim3((unsigned)a.m), dim3(256), 0u, st, a);
    }
    return hipGetLastError();
}

hipError_t launch_norm_quant(const NormQuantArgs& a, hipStream_t st)
{
    constexpr int64_t ROWS = 1 << 21;  // of a launch: a grid has fewer than 2^32 threads, a row up to 1024
    const int64_t es = a.src_type == DT_F32 ? 4 : 2;
    for (int64_t r = 0; r < a.m; r += ROWS) {
        NormQuantArgs b = a;
        b.m = a.m - r < ROWS ? a.m - r : ROWS;
        b.q = (uint8_t*)a.q + r * a.n;
        b.scale_out += r;
        b.x = (const uint8_t*)a.x + r * a.ldx * es;
        if (a.residual) b.residual = (const uint8_t*)a.residual + r * a.ldr * es;
        if (a.h_out) b.h_out = (uint8_t*)a.h_out + r * a.ldh * es;
        if (a.norm_out) b.norm_out = (uint8_t*)a.norm_out + r * a.n * es;
        const hipError_t e = launch_rows(b, st);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace ascq
