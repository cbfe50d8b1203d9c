// linear_pipe.h -- the quantised linear (linear.h) on the pipelined MFMA tiles of gemm_pipe.h: x [M, K] with
// 16-byte-aligned rows and w [N, K] the same with K a multiple of 16, or w [K, N] with 4-byte-aligned rows (int8: any K, x's bytes
// past it lying in its pitch); operands below 2^31 bytes.
//
// The epilogue of 16-bit outputs works on the accumulators where they are, a step at a time: R fragment rows of two
// neighbouring fragment columns.  v_permlane16_swap trades halves of the two, after which a lane owns eight columns of a
// row; they are scaled, biased, activated (one branch for the step), joined by the residual, rounded and stored in one
// 16-byte piece.  The residual is requested whole in front of the first step, into the registers that the main loop's operands
// have left (one step ahead instead: 1 % more at 8192^3; a word of each of its lines read in front of the main loop as well: 2 %).
// What it costs is its bytes: all CUs come to their epilogues together and read at memory's rate.
// f32 outputs, and tiles whose columns end inside a piece, go through LDS, which the main loop has left: chunks of fragment
// rows are parked there, then each thread takes runs of eight columns in a rolled loop, so the element-wise code for a row's
// end is there once per chunk and not once per piece.  That form for all (8192^3 int8, bf16 out): 425 us against 418, with
// residual and GELU alike.
//
// 8192^3 int8, w [N, K], from card to card: 409 to 418 us plain, 432 with residual, 436 with GELU, 460 to 472 with both; w [K, N] 421
// and 471 to 487.  2048 x 4096 x 11008 fp8 with residual 73 us (operands cached), 81 from memory.
#pragma once

#include "gemm_pipe.h"
#include "linear.h"

namespace ascq {

template <class T>
struct LinearEpilogue {
    typedef typename T::acc_t acc_t;
    static constexpr bool INT = std::is_same_v<acc_t, v4i>;

    static constexpr int R = T::FM % 2 == 0 ? 2 : 1;
    static constexpr int PAIRS = T::FN / 2, STEPS = PAIRS * (T::FM / R);
    template <bool BF>
    __device__ __forceinline__ static void store16(const LinearArgs& p, const acc_t (&acc)[T::FM][T::FN], const float* s_xs,
                                                   const float* s_ws, const float* s_b, int64_t m0, int64_t n0, int rows,
                                                   int cols, int wm, int wn, int lane)
    {
        const int g = lane >> 4;
        // a lane's first byte of a fragment's rows, from the fragment's first row: 32 bits
        const uint32_t lr = (uint32_t)(lane & 15) * (uint32_t)(p.ldr * 2), ly = (uint32_t)(lane & 15) * (uint32_t)(p.ldy * 2);
        auto col_of = [&](int s) { return T::block_col(wn, s % PAIRS * 2 + (g & 1)) + 8 * (g >> 1); };
        auto base_of = [&](const void* base, int64_t ld, int i) {
            return (uint8_t*)base + ((m0 + T::block_row(wm, i)) * ld + n0) * 2;
        };
        auto inside = [&](int i, int c) { return T::ct_row(wm, i, lane) < rows && c < cols; };
        u32x4 res[STEPS][R];
        const bool has = p.residual != nullptr;
        if (has) {
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                const int c = col_of(s);
#pragma unroll
                for (int q = 0; q < R; ++q) {
                    const int i = s / PAIRS * R + q;
                    if (inside(i, c))
                        res[s][q] = *(const u32x4_any*)(base_of(p.residual, p.ldr, i) + (uint64_t)(lr + (uint32_t)(c * 2)));
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const int c = col_of(s), j = s % PAIRS * 2;
            float v[R][8];
            {
                v4f ws[2], b[2] = {{-0.0f, -0.0f, -0.0f, -0.0f}, {-0.0f, -0.0f, -0.0f, -0.0f}};  // (adding it changes nothing)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    ws[h] = *(const v4f*)(s_ws + c + 4 * h);
                    if (p.bias) b[h] = *(const v4f*)(s_b + c + 4 * h);
                }
#pragma unroll
                for (int q = 0; q < R; ++q) {
                    const int i = s / PAIRS * R + q;
                    const float xs = s_xs[T::ct_row(wm, i, lane)];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const auto x = __builtin_amdgcn_permlane16_swap(acc_bits(acc[i][j][e]), acc_bits(acc[i][j + 1][e]), false, false);
                        v[q][e] = sum(x[0]) * ws[0][e] * xs + b[0][e];
                        v[q][4 + e] = sum(x[1]) * ws[1][e] * xs + b[1][e];
                    }
                }
            }
            activation<false>(p.act, [&](auto f) {
#pragma unroll
                for (int q = 0; q < R; ++q)
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[q][e] = f(v[q][e]);
            });
            if (has) {
#pragma unroll
                for (int q = 0; q < R; ++q)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const uint16_t h = (uint16_t)(res[s][q][e / 2] >> (16 * (e & 1)));
                        v[q][e] += BF ? bf16_to_f32(h) : f16_to_f32(h);
                    }
            }
#pragma unroll
            for (int q = 0; q < R; ++q) {
                const int i = s / PAIRS * R + q;
                us2_t top = {0, 0};
                u32x4 w;
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = cvt_pair<BF>(v[q][2 * e], v[q][2 * e + 1], top);
                if (__builtin_expect(cvt_special<BF>(top), 0)) {
                    auto one = [](float x) { return (uint32_t)f32_to_16_keep_inf<BF>(x); };
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[e] = one(v[q][2 * e]) | (one(v[q][2 * e + 1]) << 16);
                }
                if (inside(i, c)) *(u32x4_any*)(base_of(p.y, p.ldy, i) + (uint64_t)(ly + (uint32_t)(c * 2))) = w;
            }
            __builtin_amdgcn_sched_barrier(0);  // (the temporaries of one step at a time)
        }
    }

    // IPC fragment rows of every wave are a chunk; its rows of fp32 / int32 have 16 bytes of padding, which spread 16 rows over
    // the banks
    static constexpr int PITCH = T::TBN * 4 + 16, WM = T::NW / T::TWN;
    static constexpr int IPC = T::FM % 2 == 0 && WM * 32 * PITCH <= (int)T::LDS_BYTES ? 2 : 1;
    static_assert(WM * 16 * IPC * PITCH <= (int)T::LDS_BYTES, "a chunk fits the ring");
    template <int OUT>
    __device__ __forceinline__ static void through_lds(const LinearArgs& p, uint8_t* smem, const acc_t (&acc)[T::FM][T::FN],
                                                       const float* s_xs, const float* s_ws, const float* s_b, int64_t m0,
                                                       int64_t n0, int rows, int cols, int wm, int wn, int lane)
    {
        constexpr int ES = OUT == DT_F32 ? 4 : 2, SEGS = T::TBN / 8;
        typedef typename std::conditional<INT, int, float>::type sum_t;
#pragma unroll
        for (int ch = 0; ch < T::FM / IPC; ++ch) {
            __syncthreads();  // every wave has left the main loop (the chunk before)
#pragma unroll
            for (int i = 0; i < IPC; ++i)
#pragma unroll
                for (int j = 0; j < T::FN; ++j)
                    *(acc_t*)(smem + (wm * (16 * IPC) + i * 16 + (lane & 15)) * PITCH + T::ct_col(wn, j, lane) * 4) =
                        acc[ch * IPC + i][j];
            __syncthreads();
#pragma unroll 1
            for (int id = threadIdx.x; id < WM * 16 * IPC * SEGS; id += T::NT) {
                const int cr = id / SEGS, col = id % SEGS * 8;
                const int row = T::block_row(cr / (16 * IPC), ch * IPC + cr / 16 % IPC) + cr % 16;
                const int count = cols - col;
                if (row >= rows || count <= 0) continue;
                OutRun<OUT> res;
                if (p.residual) res.load((const uint8_t*)p.residual + (m0 + row) * p.ldr * ES, n0 + col, count);
                sum_t s[8];
                float ws[8], b[8], v[8];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const acc_t q = *(const acc_t*)(smem + cr * PITCH + col * 4 + h * 16);
                    const v4f w = *(const v4f*)(s_ws + col + 4 * h);
                    const v4f bias = *(const v4f*)(s_b + col + 4 * h);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[4 * h + e] = q[e];
                        ws[4 * h + e] = w[e];
                        b[4 * h + e] = p.bias ? bias[e] : -0.0f;
                    }
                }
                activate8<OUT == DT_F32>(s, ws, s_xs[row], b, p.act, v);
                if (p.residual) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] += res.get(e);
                }
                OutRun<OUT>::store((uint8_t*)p.y + (m0 + row) * p.ldy * ES, n0 + col, count, v);
            }
        }
    }

private:
    __device__ __forceinline__ static float sum(uint32_t bits)
    {
        if constexpr (INT) return (float)(int32_t)bits;
        else return __uint_as_float(bits);
    }
};

// SPLIT: few tiles of a long K, each shared by p.splits workgroups, which leave their sums (fp32 / int32) in p.part,
// [split][M][part_pitch]; linear_slices_kernel adds them and runs the epilogue.
// FMT: 0 (e4m3 x e4m3), or 64, whose sums keep all bits.
template <int BM, int BN, int WM, int WN, int OP, bool BTR, bool SPLIT, int FMT>
__global__ __launch_bounds__(WM * WN * 64, 2) void linear_pipe_kernel(LinearArgs p)
{
    using T = GemmPipe<BM, BN, WM, WN, OP, FMT, BTR>;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    int tm, tn;
    const int tiles_m = (int)((p.M + BM - 1) / BM), tiles_n = (int)((p.N + BN - 1) / BN);
    const int split = SPLIT ? (int)blockIdx.x / (tiles_m * tiles_n) : 0;
    pipe_tile(SPLIT ? (int)blockIdx.x % (tiles_m * tiles_n) : (int)blockIdx.x, tiles_m, tiles_n, tm, tn);
    const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
    const int rows = (int)(p.M - m0 < BM ? p.M - m0 : BM), cols = (int)(p.N - n0 < BN ? p.N - n0 : BN);
    PipeArgs c{};
    c.a = make_rsrc4(p.x, (uint32_t)(p.ldx * (p.M - 1) + (p.K + 15) / 16 * 16));  // (whole chunks: within the pitch)
    c.b = make_rsrc4(p.w, (uint32_t)(BTR ? p.ldw * (p.K - 1) + (p.N + 3) / 4 * 4 : p.ldw * (p.N - 1) + p.K));
    c.lda = (uint32_t)p.ldx;
    c.ldb = (uint32_t)p.ldw;
    c.a0 = (uint32_t)(m0 * p.ldx);
    c.b0 = (uint32_t)(BTR ? n0 : n0 * p.ldw);
    c.kbytes = (int32_t)p.K;
    if constexpr (SPLIT) {  // whole stages each, shared out evenly
        const int64_t stages = (p.K + 127) / 128, k0 = stages * split / p.splits * 128, k1 = stages * (split + 1) / p.splits * 128;
        c.a0 += (uint32_t)k0;
        c.b0 += (uint32_t)(BTR ? k0 * p.ldw : k0);
        c.kbytes = (int32_t)((k1 < p.K ? k1 : p.K) - k0);
        typename T::acc_t acc[T::FM][T::FN];
        T::run(c, smem, acc);
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / WN, wn = wave % WN;
        uint8_t* part = (uint8_t*)p.part + ((split * p.M + m0) * p.part_pitch + n0) * 4;
#pragma unroll
        for (int j = 0; j < T::FN; ++j) {
            const int col = T::ct_col(wn, j, lane);  // (the pitch is a multiple of 8)
#pragma unroll
            for (int i = 0; i < T::FM; ++i) {
                const int row = T::ct_row(wm, i, lane);
                if (row < rows && col < cols) *(typename T::acc_t*)(part + (row * p.part_pitch + col) * 4) = acc[i][j];
            }
        }
        return;
    }
    // the epilogue's vectors go to LDS now: older than the main loop's copies, whose first wait covers them.  What lies past
    // the tile's rows and columns reads 0.
    float* s_xs = (float*)(smem + T::LDS_BYTES);
    float* s_ws = s_xs + 256;
    float* s_b = s_ws + 256;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    if (wave == 0) dma16(make_rsrc4(p.x_scale + m0, (uint32_t)rows * 4u), lds_addr(s_xs), (uint32_t)lane * 16u);
    else if (wave == 1) dma16(make_rsrc4(p.w_scale + n0, (uint32_t)cols * 4u), lds_addr(s_ws), (uint32_t)lane * 16u);
    else if (wave == 2 && p.bias) dma16(make_rsrc4(p.bias + n0, (uint32_t)cols * 4u), lds_addr(s_b), (uint32_t)lane * 16u);
    typename T::acc_t acc[T::FM][T::FN];
    T::run(c, smem, acc);

    using E = LinearEpilogue<T>;
    const int wm = wave / WN, wn = wave % WN;
    if (p.out_type == DT_F32) E::template through_lds<DT_F32>(p, smem, acc, s_xs, s_ws, s_b, m0, n0, rows, cols, wm, wn, lane);
    else if (p.out_type == DT_F16) {
        if (cols % 8 == 0) E::template store16<false>(p, acc, s_xs, s_ws, s_b, m0, n0, rows, cols, wm, wn, lane);
        else E::template through_lds<DT_F16>(p, smem, acc, s_xs, s_ws, s_b, m0, n0, rows, cols, wm, wn, lane);
    } else {
        if (cols % 8 == 0) E::template store16<true>(p, acc, s_xs, s_ws, s_b, m0, n0, rows, cols, wm, wn, lane);
        else E::template through_lds<DT_BF16>(p, smem, acc, s_xs, s_ws, s_b, m0, n0, rows, cols, wm, wn, lane);
    }
}

template <int BM, int BN, int WM, int WN, int OP, bool BTR, bool SPLIT = false, int FMT = 0>
static hipError_t launch_linear_tile(const LinearArgs& a, hipStream_t st)
{
    using T = GemmPipe<BM, BN, WM, WN, OP, FMT, BTR>;
    constexpr int LDS = (int)T::LDS_BYTES + (SPLIT ? 0 : 3072);  // the ring, the vectors
    const int tiles = (int)(((a.M + BM - 1) / BM) * ((a.N + BN - 1) / BN)) * (SPLIT ? a.splits : 1);
    const hipError_t e = ensure_dynamic_lds<linear_pipe_kernel<BM, BN, WM, WN, OP, BTR, SPLIT, FMT>>(LDS);
    if (e != hipSuccess) return e;
    launch_k((linear_pipe_kernel<BM, BN, WM, WN, OP, BTR, SPLIT, FMT>), dim3(tiles), dim3(T::NT), (uint32_t)LDS, st, a);
    return hipGetLastError();
}

template <int OP, bool BTR>
static hipError_t launch_linear_layout(const LinearArgs& a, hipStream_t st)
{
    if constexpr (OP == OP_F8)
        if (a.out_type == DT_F32) {
            const bool large = a.tile == PIPE_128x128;  // (linear.hip plans these calls on two shapes)
            if (a.splits > 1)
                return large ? launch_linear_tile<128, 128, 2, 2, OP, BTR, true, 64>(a, st)
                             : launch_linear_tile<64, 128, 2, 2, OP, BTR, true, 64>(a, st);
            return large ? launch_linear_tile<128, 128, 2, 2, OP, BTR, false, 64>(a, st)
                         : launch_linear_tile<64, 128, 2, 2, OP, BTR, false, 64>(a, st);
        }
    if (a.splits > 1)
        return a.tile == PIPE_128x128 ? launch_linear_tile<128, 128, 2, 2, OP, BTR, true>(a, st)
                                      : launch_linear_tile<64, 128, 2, 2, OP, BTR, true>(a, st);
    switch (a.tile) {
    case PIPE_256x256: return launch_linear_tile<256, 256, 2, 4, OP, BTR>(a, st);
    case PIPE_192x256: return launch_linear_tile<192, 256, 2, 4, OP, BTR>(a, st);
    case PIPE_256x192: return launch_linear_tile<256, 192, 4, 2, OP, BTR>(a, st);
    case PIPE_128x256: return launch_linear_tile<128, 256, 2, 4, OP, BTR>(a, st);
    case PIPE_128x192: return launch_linear_tile<128, 192, 4, 2, OP, BTR>(a, st);
    case PIPE_128x128: return launch_linear_tile<128, 128, 2, 2, OP, BTR>(a, st);
    default: return launch_linear_tile<64, 128, 2, 2, OP, BTR>(a, st);
    }
}

}  // namespace ascq
