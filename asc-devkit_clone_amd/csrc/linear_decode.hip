// linear_decode.hip -- the quantised linear (linear.h) of few rows: x [M <= 64, K] and w [N, K] with 16-byte-aligned rows,
// K a multiple of 16, operands below 2^31 bytes.
//
// The weight is read once, so its stream is the bound, and what keeps a stream up is bytes in flight, requested in whole
// lines.  One workgroup per CU stays for all of its blocks of up to 16 channels.  Its KW waves share K: wave v has the units
// (128 K) v, v + KW, ..., U of them, and holds x's fragments of those in registers for good.  Weight units (16 rows x 128
// bytes) come by copies into a ring of D slots in LDS that belongs to the wave alone, so nothing in the loop waits for
// another wave, and the ring runs on from block to block.  At a block's end the waves' sums meet in LDS (int32: exact in
// any order; fp32: in the order of the waves) and go through the epilogue while the next units arrive.
// (Fragments loaded from memory straight into registers, sixteen rows apart: a load serves four lines per cycle's four lanes,
// 14.9 us at 1 x 11008 x 4096 from memory.)
// From memory (weights of 600 MB in turn), int8: 16 x 11008 x 4096 11.8 us, 3.8 TB/s; 16 x 8192 x 8192 15.5, 4.3; 1 x 32000 x 4096
// 26.5, 4.9; 16 x 4096 x 11008 14 to 15; 64 x 4096 x 11008 20.7 (x's fragments leave room for 4 units: K in three; 6 units spill: 26).
// K longer than the registers hold is split over S workgroups, whose sums meet in the workspace in a second launch.
#include "gemm_pipe.h"
#include "linear.h"

namespace ascq {

namespace {

__device__ __forceinline__ float scaled(float v) { return v; }
__device__ __forceinline__ float scaled(int v) { return (float)v; }

constexpr int BLOCKS = 64;  // blocks of 16 channels that a workgroup keeps the scales of

// WIDE: fp8 with the sums of the f16 MFMA, for f32 outputs
template <bool F8, bool WIDE, int MB, int KW, int U, int D>
__global__ __launch_bounds__(64 * KW) void linear_decode_kernel(LinearArgs p)
{
    typedef typename std::conditional<F8, v4f, v4i>::type acc_t;
    typedef typename std::conditional<F8, float, int>::type sum_t;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    acc_t(*red)[KW][MB][64] = (acc_t(*)[KW][MB][64])(smem + KW * D * 2048);  // two buffers
    float* s_ws = (float*)(smem + KW * D * 2048 + 2 * sizeof(acc_t) * KW * MB * 64);
    float* s_b = s_ws + BLOCKS * 16;
    float* s_xs = s_b + BLOCKS * 16;  // [16 MB]
    const int slices = p.splits;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r16 = lane & 15, g = lane >> 4;
    // this workgroup's slice of K, and every step-th block of R <= 16 channels: R shares them out evenly over whole rounds, and
    // the rows of a unit past R are not read (16 x 11008 x 4096: 11.8 us, with whole blocks 12.1).  (Neighbours read neighbouring
    // rows: with an even run of channels each, 8192 x 8192 took 16.6 us against 15.0.  Few workgroups of a split K keep R = 16:
    // more blocks cost them more than rows not read.)
    const int slice = (int)blockIdx.x % slices, b0 = (int)blockIdx.x / slices, step = (int)gridDim.x / slices;
    const int rounds = (int)((p.N + 16 * step - 1) / (16 * step));
    const int R = slices > 1 ? 16 : (int)((p.N + step * rounds - 1) / (step * rounds));
    const int nblocks = (int)((p.N + R - 1) / R);
    // the slice's units: U KW of them each
    const uint32_t K = (uint32_t)p.K, kbase = ((uint32_t)slice * (U * KW) + (uint32_t)wave) * 128u;

    // the epilogue's vectors of this workgroup's blocks
    if (slices == 1)
        for (int i = tid; i < 16 * BLOCKS; i += 64 * KW) {
            const int64_t n = (int64_t)(b0 + i / 16 * step) * R + i % 16;
            if (n >= p.N || i / 16 >= rounds) continue;
            s_ws[i] = p.w_scale[n];
            s_b[i] = p.bias ? p.bias[n] : -0.0f;
        }
    if (tid < 16 * MB) s_xs[tid] = tid < p.M ? p.x_scale[tid] : 0.0f;

    const rsrc4_t rx = make_rsrc4(p.x, (uint32_t)(p.ldx * (p.M - 1) + p.K));
    const rsrc4_t rw = make_rsrc4(p.w, (uint32_t)(p.ldw * (p.N - 1) + p.K));
    const uint32_t ring = lds_addr(smem) + (uint32_t)wave * (D * 2048);
    // copy h of a unit: rows 8 h + lane / 8 of 128 bytes in LDS, 16-byte chunk c of row r at c ^ (r / 2 % 8)
    uint32_t row[2], ch[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        row[h] = 8 * h + (lane >> 3);
        ch[h] = (uint32_t)((lane & 7) ^ ((row[h] >> 1) & 7)) * 16u;
    }
    auto request = [&](const rsrc4_t& r, uint32_t pitch, uint32_t first, uint32_t limit, int u, uint32_t slot) {
        const uint32_t k0 = kbase + (uint32_t)u * (KW * 128u);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const bool in = first + row[h] < limit && k0 + ch[h] < K;  // nothing is read past the rows or K
            dma16(r, ring + slot * 2048u + h * 1024u, in ? (first + row[h]) * pitch + k0 + ch[h] : OOB);
        }
    };
    // the stream: x's units (row block, then u), then the blocks' units; `ask` runs D units ahead of `take`
    uint32_t slot = 0;
    int ask_b = b0, ask_u = 0;
    auto ask_w = [&](uint32_t s) {  // (past the last block nothing is read, but the copies are counted)
        const uint32_t first = ask_b < nblocks ? (uint32_t)(ask_b * R) : 0u, left = ask_b < nblocks ? (uint32_t)p.N - first : 0u;
        request(rw, (uint32_t)p.ldw, first, first + (left < (uint32_t)R ? left : (uint32_t)R), ask_u, s);
        if (++ask_u == U) {
            ask_u = 0;
            ask_b += step;
        }
    };
    // chunks g and 4 + g of the lane's row
    const uint32_t f0 = (uint32_t)(r16 * 128 + ((g ^ ((r16 >> 1) & 7)) * 16)), f1 = (uint32_t)(r16 * 128 + (((4 + g) ^ ((r16 >> 1) & 7)) * 16));
    auto take = [&](v4i& lo, v4i& hi, auto ask) {
        __builtin_amdgcn_sched_barrier(0);
        wait_vmcnt<2 * (D - 1)>();  // the oldest unit is there
        __builtin_amdgcn_sched_barrier(0);
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        const uint8_t* at = smem + wave * (D * 2048) + slot * 2048u;
        lo = *(const v4i*)(at + f0);
        hi = *(const v4i*)(at + f1);
        __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): read, so its slot is free
        __builtin_amdgcn_sched_barrier(0);
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        ask(slot);
        slot = slot + 1 == D ? 0 : slot + 1;
    };
    constexpr int XU = MB * U;
    auto ask_seq = [&](int q, uint32_t s) {  // unit q of the stream, q a constant
        if (q < XU) request(rx, (uint32_t)p.ldx, (uint32_t)(q / U) * 16u, (uint32_t)p.M, q % U, s);
        else ask_w(s);
    };
#pragma unroll
    for (int q = 0; q < D; ++q) ask_seq(q, q);
    v4i x[MB][U][2];
#pragma unroll
    for (int q = 0; q < XU; ++q) take(x[q / U][q % U][0], x[q / U][q % U][1], [&](uint32_t s) { ask_seq(q + D, s); });

    int turn = 0;
    for (int b = b0, i = 0; b < nblocks; b += step, ++i, turn ^= 1) {
        acc_t acc[MB] = {};
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if constexpr (WIDE) {  // (x's codes stay codes: widened once for all blocks they do not fit the registers)
#pragma unroll
                for (int m = 0; m < MB; ++m) asm volatile("" : "+v"(x[m][u][0]), "+v"(x[m][u][1]));
            }
            v4i lo, hi;
            take(lo, hi, ask_w);
#pragma unroll
            for (int m = 0; m < MB; ++m) {
                if constexpr (F8) {
                    const v4i e = x[m][u][0], f = x[m][u][1];
                    const v8i w8 = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                    const v8i x8 = {e[0], e[1], e[2], e[3], f[0], f[1], f[2], f[3]};
                    if constexpr (WIDE) acc[m] = mfma_wide_e4m3(w8, x8, acc[m]);
                    else acc[m] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w8, x8, acc[m], 0, 0, 0, 0, 0, 0);
                } else {
                    acc[m] = __builtin_amdgcn_mfma_i32_16x16x64_i8(lo, x[m][u][0], acc[m], 0, 0, 0);
                    acc[m] = __builtin_amdgcn_mfma_i32_16x16x64_i8(hi, x[m][u][1], acc[m], 0, 0, 0);
                }
            }
        }
#pragma unroll
        for (int m = 0; m < MB; ++m) red[turn][wave][m][lane] = acc[m];
        __builtin_amdgcn_s_waitcnt(0xC07F);
        stage_barrier();  // (the block before was read before this one's second barrier: two buffers take turns)
        for (int id = tid; id < 256 * MB; id += 64 * KW) {
            const int m = id >> 4, n = id & 15;  // lane m % 16 + 16 (n / 4) holds row m, channels 4 (n / 4) .. + 3
            sum_t s = 0;
#pragma unroll
            for (int v = 0; v < KW; ++v) s += ((const sum_t*)&red[turn][v][m >> 4][(m & 15) + 16 * (n >> 2)])[n & 3];
            const int64_t col = (int64_t)b * R + n;
            if (m >= p.M || n >= R || col >= p.N) continue;
            if (slices > 1) {
                ((sum_t*)p.part)[((int64_t)slice * p.M + m) * p.part_pitch + col] = s;
                continue;
            }
            float y = scaled(s) * s_ws[i * 16 + n] * s_xs[m] + s_b[i * 16 + n];
            y = p.out_type == DT_F32 ? activate<true>(y, p.act) : activate<false>(y, p.act);
            if (p.residual) y += load_f32_of(p.residual, m * p.ldr + col, p.out_type);
            store_keep_inf(p.y, m * p.ldy + col, y, p.out_type);
        }
    }
    wait_vmcnt<0>();  // no copy may still target LDS when the wave ends
}

// the sums of a split K, in order, four columns per thread (eight: 1 us more at 64 x 4096, too few threads)
template <bool F8, int OUT>
__global__ __launch_bounds__(256) void linear_slices_kernel(LinearArgs p)
{
    typedef typename std::conditional<F8, v4f, v4i>::type sum4_t;
    typedef u32x2 u32x2_any __attribute__((aligned(2)));
    constexpr int ES = OUT == DT_F32 ? 4 : 2;
    const uint32_t runs = (uint32_t)(p.part_pitch / 4);
    const uint64_t id = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= (uint64_t)p.M * runs) return;
    const int64_t m = (int64_t)(id / runs), n = (int64_t)(id % runs) * 4;
    const int count = p.N - n < 4 ? (int)(p.N - n) : 4;
    if (count <= 0) return;
    const uint8_t* at = (const uint8_t*)p.part + (m * p.part_pitch + n) * 4;
    sum4_t s = *(const sum4_t*)at;
    for (int v = 1; v < p.splits; ++v) s += *(const sum4_t*)(at + v * p.M * p.part_pitch * 4);
    const float xs = p.x_scale[m];
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int64_t c = e < count ? n + e : n;
        y[e] = (float)s[e] * p.w_scale[c] * xs + (p.bias ? p.bias[c] : -0.0f);
    }
    activation<OUT == DT_F32>(p.act, [&](auto f) {
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = f(y[e]);
    });
    if (p.residual) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < count) y[e] += load_f32_of(p.residual, m * p.ldr + n + e, OUT);
    }
    uint8_t* to = (uint8_t*)p.y + (m * p.ldy + n) * ES;
    if (count == 4) {
        if constexpr (OUT == DT_F32) {
            *(u32x4_any*)to = (u32x4){__float_as_uint(y[0]), __float_as_uint(y[1]), __float_as_uint(y[2]), __float_as_uint(y[3])};
        } else {
            uint32_t h[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) h[e] = f32_to_16_keep_inf<OUT == DT_BF16>(y[e]);
            *(u32x2_any*)to = (u32x2){h[0] | (h[1] << 16), h[2] | (h[3] << 16)};
        }
    } else {
        for (int e = 0; e < count; ++e) store_keep_inf(to, e, y[e], OUT);
    }
}

template <bool F8, bool WIDE, int MB, int KW, int U, int D>
hipError_t go(const LinearArgs& a, hipStream_t st)
{
    constexpr auto kern = linear_decode_kernel<F8, WIDE, MB, KW, U, D>;
    constexpr int LDS = KW * D * 2048 + 2 * 16 * KW * MB * 64 + (2 * BLOCKS * 16 + 16 * MB) * 4;
    static_assert(LDS <= 160 * 1024, "LDS");
    static_assert(2 * D < 64, "vmcnt");
    const hipError_t e = ensure_dynamic_lds<kern>(LDS);
    if (e != hipSuccess) return e;
    // workgroups of a slice: one per CU in all, with at least four channels, and at most BLOCKS blocks of 16
    int64_t per = 256 / a.splits;
    if (per * (BLOCKS * 16) < a.N) per = (a.N + BLOCKS * 16 - 1) / (BLOCKS * 16);
    if (per > (a.N + 3) / 4) per = (a.N + 3) / 4;
    launch_k(kern, dim3((unsigned)(per * a.splits)), dim3(64 * KW), (uint32_t)LDS, st, a);
    return hipGetLastError();
}

// waves and, from a table of what the registers hold, units per wave: the first whose waves cover K, else the last
struct DecodePlan {
    int mb, kw, u, slices;
};
DecodePlan decode_plan(int64_t M, int64_t K, bool wide)
{
    DecodePlan d{};
    d.mb = M <= 16 ? 1 : M <= 32 ? 2 : 4;
    d.kw = d.mb == 1 ? 16 : 8;
    const int most = d.mb == 1 ? (wide ? 6 : 8) : d.mb == 2 ? 10 : 4;  // (wide, 8 units: they spill, 16 x 4096 x 14336 23 us)
    const int units = (int)((K + 127) / 128);
    d.slices = (units + d.kw * most - 1) / (d.kw * most);
    const int per = (units + d.slices - 1) / d.slices;
    d.u = (per + d.kw - 1) / d.kw;
    d.u = (d.u + 1) / 2 * 2;  // (2, 4, ...)
    return d;
}

template <bool F8, bool WIDE>
hipError_t launch_plan(const LinearArgs& a, const DecodePlan& d, hipStream_t st)
{
    if (d.mb == 1) {
        if (d.u == 2) return go<F8, WIDE, 1, 16, 2, 3>(a, st);
        if (d.u == 4) return go<F8, WIDE, 1, 16, 4, 3>(a, st);
        if (WIDE || d.u == 6) return go<F8, WIDE, 1, 16, 6, 3>(a, st);
        if constexpr (!WIDE) return go<F8, WIDE, 1, 16, 8, 3>(a, st);
    }
    if (d.mb == 2) {
        if (d.u == 2) return go<F8, WIDE, 2, 8, 2, 6>(a, st);
        if (d.u == 4) return go<F8, WIDE, 2, 8, 4, 6>(a, st);
        if (d.u == 6) return go<F8, WIDE, 2, 8, 6, 6>(a, st);
        if (d.u == 8) return go<F8, WIDE, 2, 8, 8, 6>(a, st);
        return go<F8, WIDE, 2, 8, 10, 6>(a, st);
    }
    if (d.u == 2) return go<F8, WIDE, 4, 8, 2, 5>(a, st);
    return go<F8, WIDE, 4, 8, 4, 5>(a, st);
}

}  // namespace

int linear_decode_splits(int64_t M, int64_t K, bool wide) { return decode_plan(M, K, wide).slices; }

hipError_t launch_linear_decode(const LinearArgs& a, hipStream_t st)
{
    const bool wide = a.f8 && a.out_type == DT_F32;
    const DecodePlan d = decode_plan(a.M, a.K, wide);
    if (!a.f8) return launch_plan<false, false>(a, d, st);
    return wide ? launch_plan<true, true>(a, d, st) : launch_plan<true, false>(a, d, st);
}

hipError_t launch_linear_slices(const LinearArgs& a, hipStream_t st)
{
    const dim3 grid((unsigned)((a.M * (a.part_pitch / 4) + 255) / 256)), block(256);
    auto go_out = [&](auto f8) {
        constexpr bool F8 = decltype(f8)::value;
        if (a.out_type == DT_F16) launch_k((linear_slices_kernel<F8, DT_F16>), grid, block, 0u, st, a);
        else if (a.out_type == DT_BF16) launch_k((linear_slices_kernel<F8, DT_BF16>), grid, block, 0u, st, a);
        else launch_k((linear_slices_kernel<F8, DT_F32>), grid, block, 0u, st, a);
    };
    if (a.f8) go_out(std::true_type{});
    else go_out(std::false_type{});
    return hipGetLastError();
}

}  // namespace ascq
