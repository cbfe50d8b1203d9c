// moe.hip -- the router of a mixture of experts (top-k choice, weights, tokens per expert, row order, balance loss and
// gradients) and the movement of rows to the experts' order and back.
//
// Routing of logits l [T, E]:
//   p = softmax(l) over a token's finite logits (-inf and NaN count nothing; +inf counts as the largest finite number),
//   its k choices are the largest logits (equal ones: the lowest expert), never one that counts nothing;
//   w_j = p of choice j, divided by the choices' sum when renormalised;
//   rows are ordered by expert, then by token: slot(t, j) is the row of choice j, row_token its inverse;
//   counts_e = choices of expert e, routed = tokens with at least one choice;
//   loss = E sum_e (counts_e / sum counts) (sum_t p_te / routed).
// Every order is fixed -- no atomic decides a row or the order of a sum -- so equal inputs give equal bits.
//
// A block of ROUTE_TOKENS tokens notes the tokens that chose an expert as one 64-bit mask per expert: the rank of a token
// among them is a population count, and so is the block's count.  Blocks meet through a workspace: their counts and their
// sums of p; a second launch turns the counts before a block into its rows' offsets.
#include "common.h"
#include "group_tile.h"
#include "launch.h"

namespace ascq {

namespace {

constexpr int ROUTE_TOKENS = 64;

__device__ __forceinline__ float load_logit(const void* p, int64_t i, int dtype)
{
    const float v = load_f32_of(p, i, dtype);
    return v != v ? -__builtin_inff() : fminf(v, 3.402823466e38f);
}

// One wave per token, lane l holding experts l, l + 64, ...: the largest remaining logit and its expert (the lowest of
// equals), in every lane; expert -1 when nothing is left that counts
template <int V>
__device__ __forceinline__ void wave_best(const float (&v)[V], int lane, float& best, int& expert)
{
    best = -__builtin_inff();
    expert = -1;
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (v[i] > best) {
            best = v[i];
            expert = lane + 64 * i;
        }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        const float ov = __shfl_xor(best, o, 64);
        const int oe = __shfl_xor(expert, o, 64);
        if (ov > best || (ov == best && (uint32_t)oe < (uint32_t)expert)) {
            best = ov;
            expert = oe;
        }
    }
}
__device__ __forceinline__ float wave_sum(float v)
{
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

__device__ __forceinline__ uint64_t below(int t) { return t >= 64 ? ~0ull : (1ull << t) - 1ull; }

}  // namespace

// one workgroup of 4 waves per ROUTE_TOKENS tokens
template <int V>
__global__ __launch_bounds__(256) void moe_route_kernel(MoeRouteArgs a)
{
    extern __shared__ uint64_t masks[];          // [E] tokens of this block that chose the expert
    float* sums = (float*)(masks + a.E);         // [4][E]
    __shared__ uint64_t live;                    // tokens of this block with a choice
    const int E = (int)a.E, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int e = threadIdx.x; e < E; e += 256) masks[e] = 0;
    if (threadIdx.x == 0) live = 0;
    __syncthreads();
    const int64_t t0 = (int64_t)blockIdx.x * ROUTE_TOKENS;
    float psum[V] = {};
    for (int i = wave; i < ROUTE_TOKENS; i += 4) {
        const int64_t t = t0 + i;
        if (t >= a.T) break;
        float v[V], p[V];
#pragma unroll
        for (int u = 0; u < V; ++u) {
            const int e = lane + 64 * u;
            p[u] = v[u] = e < E ? load_logit(a.logits, t * a.ld + e, a.type) : -__builtin_inff();
        }
        float top = 0.0f, sum = 0.0f, wsum = 0.0f, w = 0.0f;
        int choice = -1;
        for (int j = 0; j < a.k; ++j) {
            float best;
            int e;
            wave_best<V>(v, lane, best, e);
            if (j == 0) {
                top = best;
#pragma unroll
                for (int u = 0; u < V; ++u) p[u] = e >= 0 && p[u] > -__builtin_inff() ? expf(p[u] - top) : 0.0f;
#pragma unroll
                for (int u = 0; u < V; ++u) sum += p[u];
                sum = wave_sum(sum);
                if (e < 0) sum = 1.0f;
                if (lane == 0 && e >= 0) atomicOr((unsigned long long*)&live, 1ull << i);
            }
            const float q = e >= 0 ? expf(best - top) / sum : 0.0f;
            wsum += q;
            if (lane == j) {
                w = q;
                choice = e;
            }
            if (e >= 0) {
                if (lane == (e & 63)) {
#pragma unroll
                    for (int u = 0; u < V; ++u)
                        if (u == e >> 6) v[u] = -__builtin_inff();
                }
                if (lane == 0) atomicOr((unsigned long long*)&masks[e], 1ull << i);
            }
        }
        if (lane < a.k) {
            if (a.renormalize) w = wsum > 0.0f ? w / wsum : 0.0f;
            a.weights[t * a.k + lane] = w;
            a.experts[t * a.k + lane] = choice;
        }
#pragma unroll
        for (int u = 0; u < V; ++u) psum[u] += p[u] / sum;
    }
#pragma unroll
    for (int u = 0; u < V; ++u) {
        const int e = lane + 64 * u;
        if (e < E) sums[wave * E + e] = psum[u];
    }
    __syncthreads();
    // rank of each choice among the block's choices of its expert; the block's counts and sums of p
    for (int i = threadIdx.x; i < ROUTE_TOKENS * a.k; i += 256) {
        const int64_t at = t0 * a.k + i;
        if (at >= a.T * a.k) break;
        const int e = a.experts[at];
        a.slots[at] = e < 0 ? -1 : __popcll(masks[e] & below(i / a.k));
    }
    for (int e = threadIdx.x; e < E; e += 256) {
        a.block_counts[(int64_t)blockIdx.x * E + e] = __popcll(masks[e]);
        a.block_sums[(int64_t)blockIdx.x * E + e] = (sums[e] + sums[E + e]) + (sums[2 * E + e] + sums[3 * E + e]);
    }
    if (threadIdx.x == 0) a.block_live[blockIdx.x] = __popcll(live);
}

// offsets of every block's rows: those of the experts before, then of the blocks before within the expert
__global__ __launch_bounds__(1024) void moe_rows_kernel(MoeRouteArgs a)
{
    extern __shared__ int base[];  // [E]
    __shared__ int64_t wtot[16];
    __shared__ float s_loss[16];
    const int E = (int)a.E, e = threadIdx.x;
    const int64_t blocks = (a.T + ROUTE_TOKENS - 1) / ROUTE_TOKENS;
    int64_t before = 0, all = 0, total;
    float p = 0.0f;
    if (e < E)
        for (int64_t b = 0; b < blocks; ++b) {
            const int c = a.block_counts[b * E + e];
            if (b < (int64_t)blockIdx.x) before += c;
            all += c;
            p += a.block_sums[b * E + e];
        }
    const int64_t first = block_exclusive_scan<1024>(all, wtot, &total);
    if (e < E) base[e] = (int)(first + before);
    __syncthreads();
    const int64_t t0 = (int64_t)blockIdx.x * ROUTE_TOKENS;
    for (int i = threadIdx.x; i < ROUTE_TOKENS * a.k; i += 1024) {
        const int64_t at = t0 * a.k + i;
        if (at >= a.T * a.k) break;
        if (at >= total) a.row_tokens[at] = -1;
        const int x = a.experts[at];
        if (x < 0) continue;
        const int slot = base[x] + a.slots[at];
        a.slots[at] = slot;
        a.row_tokens[slot] = (int)(at / a.k);
    }
    if (blockIdx.x != 0) return;
    int64_t live = 0;
    for (int64_t b = 0; b < blocks; ++b) live += a.block_live[b];
    if (e < E) a.counts[e] = all;
    float part = e < E ? (float)all * p : 0.0f;
    part = wave_sum(part);
    if ((threadIdx.x & 63) == 0) s_loss[threadIdx.x >> 6] = part;
    __syncthreads();
    if (threadIdx.x == 0) {
        float sum = 0.0f;
        for (int w = 0; w < 16; ++w) sum += s_loss[w];
        *a.routed = live;
        *a.loss = total > 0 ? (float)E * (sum / ((float)total * (float)live)) : 0.0f;
    }
}

// d loss / d l and d w / d l: one wave per token
//   g_e = dL E counts_e / (sum counts x routed)  (+ dw_j at choice j without renormalisation),  dl_e = p_e (g_e - sum p g)
//   renormalised: + w_j (dw_j - sum_i dw_i w_i) at choice j
template <int V>
__global__ __launch_bounds__(256) void moe_route_grad_kernel(MoeRouteGradArgs a)
{
    const int E = (int)a.E, lane = threadIdx.x & 63;
    const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t >= a.T) return;
    float p[V], g[V], d[V];
    float top = -__builtin_inff(), cnt = 0.0f;
#pragma unroll
    for (int u = 0; u < V; ++u) {
        const int e = lane + 64 * u;
        p[u] = e < E ? load_logit(a.logits, t * a.ld + e, a.type) : -__builtin_inff();
        g[u] = e < E && a.grad_loss ? (float)a.counts[e] : 0.0f;
        d[u] = 0.0f;
        top = fmaxf(top, p[u]);
        cnt += g[u];
    }
    top = wave_max(top);
    const bool none = !(top > -__builtin_inff());  // nothing counts: no gradient
    float sum = 0.0f;
#pragma unroll
    for (int u = 0; u < V; ++u) {
        p[u] = none ? 0.0f : expf(p[u] - top);
        sum += p[u];
    }
    sum = wave_sum(sum);
    if (a.grad_loss) {
        cnt = wave_sum(cnt);
        const float live = (float)*a.routed;
        const float f = cnt > 0.0f && live > 0.0f ? *a.grad_loss * (float)E / (cnt * live) : 0.0f;
#pragma unroll
        for (int u = 0; u < V; ++u) g[u] *= f;
    }
    if (a.grad_weights) {
        const float dw = lane < a.k ? a.grad_weights[t * a.k + lane] : 0.0f;
        const float w = lane < a.k ? a.weights[t * a.k + lane] : 0.0f;
        const int id = lane < a.k ? a.experts[t * a.k + lane] : -1;
        const float mean = a.renormalize ? wave_sum(id >= 0 ? dw * w : 0.0f) : 0.0f;
        const float add = a.renormalize ? w * (dw - mean) : dw;
        for (int j = 0; j < a.k; ++j) {
            const float x = __shfl(add, j, 64);
            const int e = __shfl(id, j, 64);
#pragma unroll
            for (int u = 0; u < V; ++u)
                if (e == lane + 64 * u) {
                    if (a.renormalize) d[u] += x;
                    else g[u] += x;
                }
        }
    }
    float dot = 0.0f;
    const float inv = none ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int u = 0; u < V; ++u) {
        p[u] *= inv;
        dot += p[u] * g[u];
    }
    dot = wave_sum(dot);
#pragma unroll
    for (int u = 0; u < V; ++u) {
        const int e = lane + 64 * u;
        if (e < E) store_cast(a.grad_logits, t * a.ld_grad + e, none ? 0.0f : p[u] * (g[u] - dot) + d[u], a.type);
    }
}

// Rows to the experts' order: one workgroup per token reads its row once and writes it to its k slots; it also clears the
// rows t k .. t k + k - 1 where no token has them (they lie behind the routed ones).
__global__ __launch_bounds__(256) void moe_dispatch_kernel(MoeRowsArgs a)
{
    const int64_t t = blockIdx.x;
    const uint8_t* src = (const uint8_t*)a.x + t * a.ldx;
    const int64_t rows = a.T * a.k;
    for (int j = 0; j < a.k; ++j) {
        const int64_t slot = a.slots[t * a.k + j];
        if (slot >= 0 && slot < rows) {
            uint8_t* dst = (uint8_t*)a.out + slot * a.row_bytes;
            for (int64_t c = threadIdx.x; c < a.row_bytes; c += 256) dst[c] = src[c];
            if (threadIdx.x == 0 && a.scale_out) a.scale_out[slot] = a.scale[t];
        }
        const int64_t r = t * a.k + j;
        if (a.row_tokens[r] < 0) {
            uint8_t* dst = (uint8_t*)a.out + r * a.row_bytes;
            for (int64_t c = threadIdx.x; c < a.row_bytes; c += 256) dst[c] = 0;
            if (threadIdx.x == 0 && a.scale_out) a.scale_out[r] = 0.0f;
        }
    }
}

// out_t = residual_t + sum_j w_tj y[slot_tj]: fp32, in the order of j, one rounding
__global__ __launch_bounds__(256) void moe_combine_kernel(MoeRowsArgs a)
{
    const int64_t t = blockIdx.x, rows = a.T * a.k;
    for (int64_t c = threadIdx.x; c < a.n; c += 256) {
        float v = 0.0f;
        for (int j = 0; j < a.k; ++j) {
            const int64_t slot = a.slots[t * a.k + j];
            if (slot >= 0 && slot < rows) v += a.weights[t * a.k + j] * load_f32_of(a.y, slot * a.n + c, a.type);
        }
        if (a.residual) v += load_f32_of(a.residual, t * a.n + c, a.type);
        store_cast(a.out, t * a.n + c, v, a.type);
    }
}

// dw_tj = <dout_t, y[slot_tj]>, dy[slot_tj] = w_tj dout_t; rows of no token get 0
__global__ __launch_bounds__(256) void moe_combine_grad_kernel(MoeRowsArgs a)
{
    __shared__ float red[4];
    const int64_t t = blockIdx.x, rows = a.T * a.k;
    for (int j = 0; j < a.k; ++j) {
        const int64_t slot = a.slots[t * a.k + j], r = t * a.k + j;
        const bool ok = slot >= 0 && slot < rows;
        const float w = a.out ? a.weights[r] : 0.0f;
        float dot = 0.0f;
        if (ok)
            for (int64_t c = threadIdx.x; c < a.n; c += 256) {
                const float d = load_f32_of(a.x, t * a.n + c, a.type);
                if (a.grad_weights) dot += d * load_f32_of(a.y, slot * a.n + c, a.type);
                if (a.out) store_cast(a.out, slot * a.n + c, w * d, a.type);
            }
        if (a.grad_weights) {
            dot = wave_sum(dot);
            if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = dot;
            __syncthreads();
            if (threadIdx.x == 0) a.grad_weights[r] = (red[0] + red[1]) + (red[2] + red[3]);
            __syncthreads();
        }
        if (a.out && a.row_tokens[r] < 0)
            for (int64_t c = threadIdx.x; c < a.n; c += 256) store_cast(a.out, r * a.n + c, 0.0f, a.type);
    }
}

namespace {
int64_t route_blocks(int64_t T) { return (T + ROUTE_TOKENS - 1) / ROUTE_TOKENS; }
}  // namespace

size_t moe_route_ws_bytes(int64_t T, int64_t E)
{
    return (size_t)route_blocks(T) * ((size_t)E * 8 + 4);
}

hipError_t launch_moe_route(MoeRouteArgs a, void* ws, hipStream_t st)
{
    const int64_t blocks = route_blocks(a.T);
    a.block_counts = (int*)ws;
    a.block_sums = (float*)(a.block_counts + blocks * a.E);
    a.block_live = (int*)(a.block_sums + blocks * a.E);
    if (blocks > 0) {
        const uint32_t lds = (uint32_t)a.E * 24;
        const dim3 grid((unsigned)blocks), block(256);
        if (a.E <= 64) launch_k(moe_route_kernel<1>, grid, block, lds, st, a);
        else if (a.E <= 128) launch_k(moe_route_kernel<2>, grid, block, lds, st, a);
        else if (a.E <= 256) launch_k(moe_route_kernel<4>, grid, block, lds, st, a);
        else launch_k(moe_route_kernel<16>, grid, block, lds, st, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    launch_k(moe_rows_kernel, dim3((unsigned)(blocks > 0 ? blocks : 1)), dim3(1024), (uint32_t)a.E * 4, st, a);
    return hipGetLastError();
}

hipError_t launch_moe_route_grad(const MoeRouteGradArgs& a, hipStream_t st)
{
    const dim3 grid((unsigned)((a.T + 3) / 4)), block(256);
    if (a.E <= 64) launch_k(moe_route_grad_kernel<1>, grid, block, 0u, st, a);
    else if (a.E <= 128) launch_k(moe_route_grad_kernel<2>, grid, block, 0u, st, a);
    else if (a.E <= 256) launch_k(moe_route_grad_kernel<4>, grid, block, 0u, st, a);
    else launch_k(moe_route_grad_kernel<16>, grid, block, 0u, st, a);
    return hipGetLastError();
}

hipError_t launch_moe_dispatch(const MoeRowsArgs& a, hipStream_t st)
{
    launch_k(moe_dispatch_kernel, dim3((unsigned)a.T), dim3(256), 0u, st, a);
    return hipGetLastError();
}
hipError_t launch_moe_combine(const MoeRowsArgs& a, hipStream_t st)
{
    launch_k(moe_combine_kernel, dim3((unsigned)a.T), dim3(256), 0u, st, a);
    return hipGetLastError();
}
hipError_t launch_moe_combine_grad(const MoeRowsArgs& a, hipStream_t st)
{
    launch_k(moe_combine_grad_kernel, dim3((unsigned)a.T), dim3(256), 0u, st, a);
    return hipGetLastError();
}

}  // namespace ascq
