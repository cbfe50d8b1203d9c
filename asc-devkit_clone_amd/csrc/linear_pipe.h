// linear_pipe.h -- the quantised linear (linear.h) on the pipelined MFMA tiles of gemm_pipe.h: x [M, K] with
// 16-byte-aligned rows and w [N, K] the same with K a multiple of 16, or w [K, N] with 4-byte-aligned rows (int8: any K, x's bytes
// past it lying in its pitch); operands below 2^31 bytes.
//
// The epilogue takes the accumulators through LDS, which the main loop has left: a wave's fragments hold four columns of
// sixteen rows, from which a residual would be read in pieces of 8 bytes.  A chunk of fragment rows (IPC of each wave's) is parked
// as rows of fp32 / int32, then every thread takes runs of eight columns, whose residual it requested before it parked:
// whole lines are read and written, the activation is one branch per run and the code stays small for its five kinds.
// Two buffers take turns, so a chunk costs one barrier.  A row's 16 bytes of padding spread 16 rows over the banks.
#pragma once

#include "gemm_pipe.h"
#include "linear.h"

namespace ascq {

template <int BM, int BN, int WM, int WN, int OP, bool BTR>
struct LinearTile {
    using T = GemmPipe<BM, BN, WM, WN, OP, 0, BTR>;  // (e4m3 x e4m3)
    static constexpr int PITCH = BN * 4 + 16;
    static constexpr int IPC = T::FM % 2 == 0 && 2 * WM * 32 * PITCH <= (int)T::LDS_BYTES + 4096 ? 2 : 1;
    static constexpr int ROWS = WM * 16 * IPC, CHUNKS = T::FM / IPC;
    static constexpr int PARK = 2 * ROWS * PITCH;
    static constexpr int VECTORS = (PARK > (int)T::LDS_BYTES ? PARK : (int)T::LDS_BYTES);  // the scales and bias behind it
    static constexpr int LDS = VECTORS + 3072;
    static_assert(LDS <= 160 * 1024, "LDS");
};

template <int BM, int BN, int WM, int WN, int OP, bool BTR>
__global__ __launch_bounds__(WM * WN * 64, 2) void linear_pipe_kernel(LinearArgs p)
{
    using L = LinearTile<BM, BN, WM, WN, OP, BTR>;
    using T = typename L::T;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    int tm, tn;
    pipe_tile((int)blockIdx.x, (int)((p.M + BM - 1) / BM), (int)((p.N + BN - 1) / BN), tm, tn);
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
    // the epilogue's vectors go to LDS now: older than the main loop's copies, whose first wait covers them.  What lies past
    // the tile's rows and columns reads 0.
    float* s_xs = (float*)(smem + L::VECTORS);
    float* s_ws = s_xs + 256;
    float* s_b = s_ws + 256;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    if (wave == 0) dma16(make_rsrc4(p.x_scale + m0, (uint32_t)rows * 4u), lds_addr(s_xs), (uint32_t)lane * 16u);
    else if (wave == 1) dma16(make_rsrc4(p.w_scale + n0, (uint32_t)cols * 4u), lds_addr(s_ws), (uint32_t)lane * 16u);
    else if (wave == 2 && p.bias) dma16(make_rsrc4(p.bias + n0, (uint32_t)cols * 4u), lds_addr(s_b), (uint32_t)lane * 16u);
    typename T::acc_t acc[T::FM][T::FN];
    T::run(c, smem, acc);

    const int wm = wave / WN, wn = wave % WN;
    constexpr int SEGS = BN / 8, RUNS = L::ROWS * SEGS / T::NT;  // runs of a thread per chunk
    static_assert(L::ROWS * SEGS % T::NT == 0, "runs split evenly");
    typedef typename std::conditional<OP == OP_I8, int, float>::type sum_t;
    typedef typename std::conditional<OP == OP_I8, v4i, v4f>::type sum4_t;
    // (the first chunk's buffer is the ring: every wave has to be out of the main loop)
    __syncthreads();
    auto epilogue = [&](auto out_type) {
        constexpr int OUT = decltype(out_type)::value, ES = OUT == DT_F32 ? 4 : 2;
#pragma unroll
        for (int ch = 0; ch < L::CHUNKS; ++ch) {
            uint8_t* park = smem + (ch & 1) * (L::ROWS * L::PITCH);
            OutRun<OUT> res[RUNS];
            auto run_of = [&](int u, int& cr, int& row, int& col, int& count) {
                const int id = (int)threadIdx.x + u * T::NT;
                cr = id / SEGS;
                col = id % SEGS * 8;
                row = T::block_row(cr / (16 * L::IPC), ch * L::IPC + cr / 16 % L::IPC) + cr % 16;
                count = row < rows ? cols - col : 0;
            };
            if (p.residual) {
#pragma unroll
                for (int u = 0; u < RUNS; ++u) {
                    int cr, row, col, count;
                    run_of(u, cr, row, col, count);
                    if (count > 0) res[u].load((const uint8_t*)p.residual + (m0 + row) * p.ldr * ES, n0 + col, count);
                }
            }
#pragma unroll
            for (int i = 0; i < L::IPC; ++i)
#pragma unroll
                for (int j = 0; j < T::FN; ++j)
                    *(sum4_t*)(park + (wm * (16 * L::IPC) + i * 16 + (lane & 15)) * L::PITCH + T::ct_col(wn, j, lane) * 4) =
                        acc[ch * L::IPC + i][j];
            __syncthreads();
#pragma unroll
            for (int u = 0; u < RUNS; ++u) {
                int cr, row, col, count;
                run_of(u, cr, row, col, count);
                if (count <= 0) continue;
                sum_t s[8];
                float ws[8], b[8], v[8];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const sum4_t q = *(const sum4_t*)(park + cr * L::PITCH + col * 4 + h * 16);
                    const v4f w = *(const v4f*)(s_ws + col + 4 * h);
                    const v4f bias = *(const v4f*)(s_b + col + 4 * h);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[4 * h + e] = q[e];
                        ws[4 * h + e] = w[e];
                        b[4 * h + e] = p.bias ? bias[e] : -0.0f;
                    }
                }
                activate8(s, ws, s_xs[row], b, p.act, v);
                if (p.residual) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] += res[u].get(e);
                }
                OutRun<OUT>::store((uint8_t*)p.y + (m0 + row) * p.ldy * ES, n0 + col, count, v);
            }
        }
    };
    if (p.out_type == DT_F16) epilogue(std::integral_constant<int, DT_F16>{});
    else if (p.out_type == DT_BF16) epilogue(std::integral_constant<int, DT_BF16>{});
    else epilogue(std::integral_constant<int, DT_F32>{});
}

template <int BM, int BN, int WM, int WN, int OP, bool BTR>
static hipError_t launch_linear_tile(const LinearArgs& a, hipStream_t st)
{
    using L = LinearTile<BM, BN, WM, WN, OP, BTR>;
    const int tiles = (int)(((a.M + BM - 1) / BM) * ((a.N + BN - 1) / BN));
    const hipError_t e = ensure_dynamic_lds<linear_pipe_kernel<BM, BN, WM, WN, OP, BTR>>(L::LDS);
    if (e != hipSuccess) return e;
    launch_k((linear_pipe_kernel<BM, BN, WM, WN, OP, BTR>), dim3(tiles), dim3(L::T::NT), (uint32_t)L::LDS, st, a);
    return hipGetLastError();
}

template <int OP, bool BTR>
static hipError_t launch_linear_layout(const LinearArgs& a, hipStream_t st)
{
    switch (pick_pipe_tile(a.M, a.N, a.K)) {
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
