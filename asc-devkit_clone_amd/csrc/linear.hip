// linear.hip -- the quantised linear: 8-bit activations with one scale per token times an 8-bit weight with one scale per
// channel, and bias, activation and residual in the epilogue (linear.h).  int8 sums are exact (int32).  fp8 e4m3 sums are
// held in fp32, but the fp8 MFMA aligns the products of 16 neighbouring k to the largest and drops what lies 2^-13 below it:
// normal data come out 1.5e-5 off (normwise, 16 x 4096 x 4096 to 2048 x 4096 x 11008) where fp32 sums are 7e-8 to 1.5e-7.  That
// is below a 16-bit output's rounding (1.7e-3 in bf16 either way), so those take it; for f32 outputs the codes are widened to
// f16 in registers, for the f16 MFMA, which keeps all bits at half the rate (8192^3 396 -> 811 us; 16 x 32000 x 4096, whose
// weight comes from memory, 27 either way).
// Here: which kernel a call takes -- the weight-streaming one of linear_decode.hip up to 64 rows, the tiles of linear_pipe.h,
// their K shared by several workgroups where tiles are few, or the one below -- and what is copied for it.
#include "linear.h"

#include "gemm_pipe.h"

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
// weight turned on the way.  It takes what nothing else does: K = 0, operands off their alignment without a workspace (1030 x
// 4100 x 4095 int8: 995 us against 38 with one), and a w [K, N] past 2^31 bytes or of few rows that are very far apart.
template <bool F8>
__global__ __launch_bounds__(256) void linear_any_kernel(LinearArgs a, int64_t first)
{
    constexpr int P = 80;  // bytes of a row in LDS: 64, and 16 that spread the rows over the banks
    __shared__ __attribute__((aligned(16))) uint8_t sx[64 * P], sw[64 * P];
    typedef typename std::conditional<F8, v4f, v4i>::type acc_t;
    const int64_t tiles_n = (a.N + 63) / 64;
    const int64_t tile = first + blockIdx.x, m0 = tile / tiles_n * 64, n0 = tile % tiles_n * 64;
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
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const h8 p = widen_e4m3(fx[i][2 * h], fx[i][2 * h + 1]), q = widen_e4m3(fw[j][2 * h], fw[j][2 * h + 1]);
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(p, q, acc[i][j], 0, 0, 0);
                    }
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
                v = a.out_type == DT_F32 ? activate<true>(v, a.act) : activate<false>(v, a.act);
                if (a.residual) v += load_f32_of(a.residual, m * a.ldr + n, a.out_type);
                store_keep_inf(a.y, m * a.ldy + n, v, a.out_type);
            }
}

}  // namespace

namespace {

constexpr int64_t SPAN = (1ll << 31) - 16;  // bytes of an operand that the tiles address

// Which operands of a call the tiles cannot take as they lie, and the pitch of their copies (rows of zero-padded 16-byte
// words).  K-contiguous operands whose K is no multiple of 16 need zeros behind K in one of them -- the smaller, x, as
// long as the other's rows are aligned and what lies behind its K within a 16-byte word cannot be a NaN (int8).
struct PackPlan {
    bool x, w;
    int64_t kp, ldx, ldw;
    size_t x_bytes, w_bytes;
};
PackPlan pack_plan(const LinearArgs& a)
{
    const bool x_ok = ((uintptr_t)a.x | (uintptr_t)a.ldx) % 16 == 0;
    const bool w_ok = ((uintptr_t)a.w | (uintptr_t)a.ldw) % (a.w_trans ? 16 : 4) == 0;
    const bool ragged = a.K % 16 != 0 && (a.w_trans || a.f8);
    PackPlan p{};
    p.x = !x_ok || ragged;
    p.w = !w_ok || (a.w_trans && ragged && a.f8);
    p.kp = (a.K + 15) / 16 * 16;
    p.ldx = p.kp;
    p.ldw = a.w_trans ? p.kp : (a.N + 15) / 16 * 16;
    p.x_bytes = p.x ? (size_t)(a.M * p.ldx) : 0;
    p.w_bytes = p.w ? (size_t)((a.w_trans ? a.N : a.K) * p.ldw) : 0;
    return p;
}
// spans and pitches that the tiles or the copying launch do not take
bool too_large(const LinearArgs& a)
{
    const int64_t kp = (a.K + 15) / 16 * 16;
    // (the epilogue addresses 16 rows with 32-bit offsets)
    if (a.ldy > (1ll << 24) || (a.residual && a.ldr > (1ll << 24))) return true;
    // (rows of a w [K, N] past K are asked for, up to the end of x's last 16-byte word or, fp8, of the stage: their 32-bit offsets
    // must not come round to w again)
    if (!a.w_trans && a.ldw > ((1ll << 32) - a.N - 4096) / (a.f8 ? (a.K + 127) / 128 * 128 : kp)) return true;
    return a.ldx * (a.M - 1) + kp > SPAN || a.M * kp > SPAN || (a.w_trans ? a.ldw * (a.N - 1) + kp : a.ldw * (a.K - 1) + a.N + 3) > SPAN ||
           (a.w_trans ? a.N * kp : a.K * ((a.N + 15) / 16 * 16)) > SPAN;
}

hipError_t launch_any(const LinearArgs& a, const char* why, hipStream_t st)
{
    log_fallback("linear_any_kernel", why);
    constexpr int64_t MOST = 1 << 23;  // tiles of a launch: a grid has fewer than 2^32 threads
    const int64_t tiles = ((a.M + 63) / 64) * ((a.N + 63) / 64);
    for (int64_t at = 0; at < tiles; at += MOST) {
        const dim3 grid((unsigned)(tiles - at < MOST ? tiles - at : MOST));
        if (a.f8) launch_k(linear_any_kernel<true>, grid, dim3(256), 0u, st, a, at);
        else launch_k(linear_any_kernel<false>, grid, dim3(256), 0u, st, a, at);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace

namespace {

bool wide(const LinearArgs& a) { return a.f8 && a.out_type == DT_F32; }
size_t align256(size_t b) { return (b + 255) & ~(size_t)255; }

// How an aligned call runs: the weight-streaming kernel for few rows, or tiles, whose K may be shared by several workgroups
struct Plan {
    bool decode;
    int tile, splits;
};
// wide: fp8 with f32 outputs, on tiles of 128 x 128 or 64 x 128 (their operands as f16 numbers take more registers)
int tile_of(int64_t M, int64_t N, int64_t K, bool wide)
{
    if (!wide) return (int)pick_pipe_tile(M, N, K);
    return pipe_tile_us(PIPE_64x128, M, N, K) < pipe_tile_us(PIPE_128x128, M, N, K) ? PIPE_64x128 : PIPE_128x128;
}
Plan plan_of(int64_t M, int64_t N, int64_t K, bool w_trans, bool wide)
{
    if (w_trans && M <= 64) return {true, 0, linear_decode_splits(M, K, wide)};
    Plan best{false, tile_of(M, N, K, wide), 1};
    // (Up to 256 rows the weight comes from memory, not from a cache that other tiles filled, and few workgroups wait for it, so
    // the table, whose operands were cached, is short of what they take.  Weights of 600 MB in turn, us split and unsplit, with
    // tiles of 64 x 128: 128 x 4096 x 11008, 64 tiles, 22.6 and 42.6, w [K, N] 25.5 and 58.2; 192 x 2048 x 8192, 48, 16.4 and
    // 21.1; 256 x 4096 x 11008, 128, 30.7 and 41.8; at 96 tiles or K = 4096 alike, up to a fifth either way: 192 x 4096 x 4096 15.9
    // and 13.1, w [K, N] 100 x 6144 x 4096 21.2 and 25.1.)
    float least = pipe_tile_us(best.tile, M, N, K);
    if (M <= 256 && ((M + 63) / 64) * ((N + 127) / 128) <= (w_trans ? 96 : 128)) least *= w_trans ? 1.6f : 2.2f;
    for (int tile : {PIPE_128x128, PIPE_64x128})
        for (int s = 2; s <= 16; ++s) {
            const int64_t stages = (K + 127) / 128, per = (stages + s - 1) / s;
            if (per < 4) break;
            // the sums' way through memory and the second launch
            const float extra = 3.0f + (float)(M * N) * (4.0f * s) * 5e-7f;
            const float us = pipe_tile_us(tile, M, N, per * 128, 0, s) + extra;
            if (us < least) {
                best = {false, tile, s};
                least = us;
            }
        }
    return best;
}
int64_t part_pitch(int64_t N) { return (N + 7) / 8 * 8; }
size_t part_bytes(int64_t M, int64_t N, int splits) { return splits > 1 ? (size_t)splits * (size_t)(M * part_pitch(N)) * 4 : 0; }

// Operands past the tiles' 2^31 bytes go in pieces, of rows of x or (w [N, K]) of channels: the rows of a piece, or 0
int64_t row_piece(const LinearArgs& a)
{
    const int64_t kp = (a.K + 15) / 16 * 16, pitch = a.ldx > kp ? a.ldx : kp, most = SPAN / pitch;
    return a.M > most && most >= 512 ? most / 256 * 256 : 0;
}
int64_t channel_piece(const LinearArgs& a)
{
    const int64_t kp = (a.K + 15) / 16 * 16, pitch = a.ldw > kp ? a.ldw : kp, most = SPAN / pitch;
    return a.w_trans && a.N > most && most >= 512 ? most / 256 * 256 : 0;
}
LinearArgs piece_of(const LinearArgs& a, int64_t m0, int64_t m, int64_t n0, int64_t n)
{
    const int64_t es = a.out_type == DT_F32 ? 4 : 2;
    LinearArgs b = a;
    b.x += m0 * a.ldx;
    b.x_scale += m0;
    b.w += n0 * a.ldw;  // (n0 > 0: w [N, K])
    b.w_scale += n0;
    if (a.bias) b.bias += n0;
    if (a.residual) b.residual = (const uint8_t*)a.residual + (m0 * a.ldr + n0) * es;
    b.y = (uint8_t*)a.y + (m0 * a.ldy + n0) * es;
    b.M = m;
    b.N = n;
    return b;
}

}  // namespace

size_t linear_ws_bytes(const LinearArgs& in)
{
    LinearArgs a = in;
    if (a.M == 0 || a.N == 0 || a.K == 0) return 0;
    const int64_t rows = row_piece(a), channels = rows ? 0 : channel_piece(a);
    if (rows || channels) {  // what the whole pieces take or the last one, which may split K where they do not
        int64_t& size = rows ? a.M : a.N;
        const int64_t whole = rows ? rows : channels, last = size % whole;
        size = whole;
        const size_t most = linear_ws_bytes(a);
        size = last;
        const size_t rest = linear_ws_bytes(a);
        return most > rest ? most : rest;
    }
    if (too_large(a)) return 0;
    const PackPlan p = pack_plan(a);
    const size_t pack = p.x_bytes + p.w_bytes;
    const size_t part = part_bytes(a.M, a.N, plan_of(a.M, a.N, a.w_trans ? p.kp : a.K, a.w_trans, wide(a)).splits);
    return part ? align256(pack) + part : pack;
}

hipError_t launch_linear(const LinearArgs& in, uint8_t* ws, size_t ws_bytes, hipStream_t st)
{
    LinearArgs a = in;
    if (a.K == 0) return launch_any(a, "k = 0", st);
    const int64_t rows = row_piece(a), channels = rows ? 0 : channel_piece(a);
    if (rows || channels) {
        const int64_t step = rows ? rows : channels, end = rows ? a.M : a.N;
        for (int64_t at = 0; at < end; at += step) {
            const int64_t n = end - at < step ? end - at : step;
            const hipError_t e = launch_linear(rows ? piece_of(a, at, n, 0, a.N) : piece_of(a, 0, a.M, at, n), ws, ws_bytes, st);
            if (e != hipSuccess) return e;
        }
        return hipSuccess;
    }
    if (too_large(a)) return launch_any(a, "w [k, n] past 2^31 bytes or of few, very long rows, or a pitch past 2^24", st);
    const PackPlan p = pack_plan(a);
    const size_t pack = p.x_bytes + p.w_bytes;
    if (pack) {
        if (pack > ws_bytes) return launch_any(a, "operands off their alignment and no workspace to copy them to", st);
        uint8_t* px = p.x ? ws : nullptr;
        uint8_t* pw = p.w ? ws + p.x_bytes : nullptr;
        const hipError_t e = launch_pack_rows(PackRows{px, a.x, a.M, a.K, a.ldx},
                                              a.w_trans ? PackRows{pw, a.w, a.N, a.K, a.ldw} : PackRows{pw, a.w, a.K, a.N, a.ldw}, st);
        if (e != hipSuccess) return e;
        if (p.x) {
            a.x = px;
            a.ldx = p.ldx;
        }
        if (p.w) {
            a.w = pw;
            a.ldw = p.ldw;
        }
        if (a.w_trans) a.K = p.kp;  // (zeros behind K in one operand at least)
    }
    Plan plan = plan_of(a.M, a.N, a.K, a.w_trans, wide(a));
    if (plan.splits > 1) {
        if (align256(pack) + part_bytes(a.M, a.N, plan.splits) > ws_bytes) plan = {false, tile_of(a.M, a.N, a.K, wide(a)), 1};
        a.part = ws + align256(pack);
        a.part_pitch = part_pitch(a.N);
    }
    a.tile = plan.tile;
    a.splits = plan.splits;
    const hipError_t e = plan.decode ? launch_linear_decode(a, st) : a.f8 ? launch_linear_pipe_f8(a, st) : launch_linear_pipe_i8(a, st);
    return e != hipSuccess || a.splits == 1 ? e : launch_linear_slices(a, st);
}

}  // namespace ascq
