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
// A chunk of up to 64 tokens notes those that chose an expert as one 64-bit mask per expert: the rank of a token among them
// is a population count, and so is the chunk's count.  Blocks of chunks meet through a workspace: their counts and their
// sums of p; the second launch turns the counts before a block into its rows' offsets.  A few tokens are one block, which
// does it all.
// What bounds it is latency: a chain of k maxima over a token's experts, and two launches, the second of which reads the counts
// of all blocks in each (16384 tokens, 64 experts, k = 6: 7.5 and 7.3 us of kernels; 16384, 256, k = 8: 17.8, of which the
// search's instructions, five per logit and choice, are some 4 at the chip's rate, and 15; 16 tokens, 16 experts, k = 2: 4.8).
#include <type_traits>

#include "common.h"
#include "group_tile.h"
#include "launch.h"

namespace ascq {

namespace {

constexpr int CHUNK = 64;        // tokens of a mask, at most
constexpr int MAX_BLOCKS = 512;  // (each block of the second launch reads the counts of all; fewer, each for a run: slower)
constexpr int MAX_K = 16;

// a gradient, rounded once: past a 16-bit type's range it is infinite, which is what a loss scaler looks for
__device__ __forceinline__ void store_grad(void* p, int64_t i, float v, int dtype)
{
    if (dtype == DT_F16) ((uint16_t*)p)[i] = f32_to_f16(v);
    else if (dtype == DT_BF16) ((__bf16*)p)[i] = (__bf16)v;
    else ((float*)p)[i] = v;
}

__device__ __forceinline__ float wave_sum(float v)
{
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// v of the lane that `ctrl` names among this lane's 16
template <int ctrl>
__device__ __forceinline__ uint32_t moved(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, 0xf, 0xf, true); }
template <int ctrl>
__device__ __forceinline__ float moved(float v) { return __uint_as_float(moved<ctrl>(__float_as_uint(v))); }

// op of v and v of the lane 16 or 32 away
template <int S, class Op>
__device__ __forceinline__ uint32_t far(uint32_t v, Op op)
{
    if constexpr (S == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return op((uint32_t)r[0], (uint32_t)r[1]);
    } else {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return op((uint32_t)r[0], (uint32_t)r[1]);
    }
}
template <int S, class Op>
__device__ __forceinline__ float far(float v, Op op)
{
    return __uint_as_float(far<S>(__float_as_uint(v), [&](uint32_t x, uint32_t y) {
        return __float_as_uint(op(__uint_as_float(x), __uint_as_float(y)));
    }));
}

// op (commutative) over G neighbouring lanes, each of them gets it: within 16 lanes quad permutations, then mirrors, which
// reach the other half because the lanes of a half already agree
template <int G, class T, class Op>
__device__ __forceinline__ T reduce(T v, Op op)
{
    if constexpr (G > 1) v = op(v, moved<0xB1>(v));
    if constexpr (G > 2) v = op(v, moved<0x4E>(v));
    if constexpr (G > 4) v = op(v, moved<0x141>(v));
    if constexpr (G > 8) v = op(v, moved<0x140>(v));
    if constexpr (G > 16) v = far<16>(v, op);
    if constexpr (G > 32) v = far<32>(v, op);
    return v;
}
// the sum over the wave's lanes G, 2 G, ... away: rotations within 16 lanes, then the swaps
template <int G>
__device__ __forceinline__ float sum_across(float v)
{
    auto add = [](float x, float y) { return x + y; };
    if constexpr (G <= 8) v += moved<0x128>(v);
    if constexpr (G <= 4) v += moved<0x124>(v);
    if constexpr (G <= 2) v += moved<0x122>(v);
    if constexpr (G <= 1) v += moved<0x121>(v);
    if constexpr (G <= 16) v = far<16>(v, add);
    if constexpr (G <= 32) v = far<32>(v, add);
    return v;
}
template <int G>
__device__ __forceinline__ float group_sum(float v)
{
    return reduce<G>(v, [](float x, float y) { return x + y; });
}

// a logit as a number whose order is the logit's; NOTHING or less: it counts nothing (-inf, or a choice taken)
constexpr uint32_t NOTHING = 0x007fffffu;
__device__ __forceinline__ uint32_t key_of(float v)
{
    const uint32_t b = __float_as_uint(v + 0.0f);  // (-0 is 0)
    return b ^ ((int)b < 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float((int)k < 0 ? k ^ 0x80000000u : ~k); }

// logits e0 .. e0 + V - 1 of a row (past E: -inf); vec: the row's V are one aligned run
template <int V>
__device__ __forceinline__ void load_logits(const void* row, int type, int e0, int E, bool vec, float (&v)[V])
{
    if (vec && e0 + V <= E) {
        if (type == DT_F32) {
#pragma unroll
            for (int i = 0; i < V / 4; ++i) {
                const u32x4 w = ((const u32x4*)((const float*)row + e0))[i];
#pragma unroll
                for (int j = 0; j < 4; ++j) v[4 * i + j] = __uint_as_float(w[j]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < V / 8; ++i) {
                const u32x4 w = ((const u32x4*)((const uint16_t*)row + e0))[i];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint16_t h = (uint16_t)(w[j / 2] >> (16 * (j & 1)));
                    v[8 * i + j] = type == DT_F16 ? f16_to_f32(h) : bf16_to_f32(h);
                }
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = e0 + i < E ? load_f32_of(row, e0 + i, type) : -__builtin_inff();
    }
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = v[i] != v[i] ? -__builtin_inff() : fminf(v[i], 3.402823466e38f);
}

}  // namespace

// the first chunk of block b of the routing
__device__ __forceinline__ int64_t first_chunk(const MoeRouteArgs& a, int b, int blocks)
{
    return a.chunks <= blocks ? b : (int64_t)a.chunks * b / blocks;
}

// G lanes per token, each with V neighbouring experts; a chunk at a time, all of its tokens at once up to 16 lanes.
// SINGLE: one block has all tokens.
template <int G>
constexpr int route_threads = G < 16 ? 64 * G : 1024;
template <int G, int V, bool SINGLE>
__global__ __launch_bounds__(route_threads<G>) void moe_route_kernel(MoeRouteArgs a)
{
    constexpr int NT = route_threads<G>, NW = NT / 64, TOK = NT / G;  // TOK tokens at once
    extern __shared__ __attribute__((aligned(8))) uint8_t lds[];
    const int E = (int)a.E, k = a.k;
    uint64_t* masks = (uint64_t*)lds;           // [E] tokens of the chunk that chose the expert
    float* sums = (float*)(masks + E);          // [waves][E] sums of p
    int* first = (int*)(sums + NW * E);         // [E] the block's choices of the expert in the chunks before
    __shared__ float s_w[CHUNK * MAX_K], s_f[CHUNK];
    __shared__ int s_e[CHUNK * MAX_K];
    __shared__ int s_live[NW];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, e0 = tid % G * V;
    const int C = a.chunk;
    const int64_t c0 = first_chunk(a, blockIdx.x, gridDim.x), c1 = first_chunk(a, blockIdx.x + 1, gridDim.x);
    const bool vec = ((uintptr_t)a.logits | (uintptr_t)(a.ld * (a.type == DT_F32 ? 4 : 2))) % 16 == 0;
    const int64_t row_bytes = a.ld * (a.type == DT_F32 ? 4 : 2);
    if (tid < E) first[tid] = 0;
    float psum[V] = {};
    int live = 0;
    for (int64_t c = c0; c < c1; ++c) {
        if (tid < E) masks[tid] = 0;
        __syncthreads();
        for (int token = tid / G; token < C; token += TOK) {
            const int64_t t = c * C + token;
            if (c * C + __builtin_amdgcn_readfirstlane(token) >= a.T) break;  // none of the wave's
            float p[V];
            uint32_t key[V];
            if (t < a.T) load_logits<V>((const uint8_t*)a.logits + t * row_bytes, a.type, e0, E, vec, p);
            else {
#pragma unroll
                for (int i = 0; i < V; ++i) p[i] = -__builtin_inff();
            }
#pragma unroll
            for (int i = 0; i < V; ++i) key[i] = key_of(p[i]);
            float top = 0.0f, all = 1.0f, inv = 0.0f;
            for (int j = 0; j < k; ++j) {
                // the largest logit left, then the lowest expert that has it; -1 when nothing is left that counts
                uint32_t best = key[0], at = 0xffffffffu;
#pragma unroll
                for (int i = 1; i < V; ++i) best = best > key[i] ? best : key[i];
                best = reduce<G>(best, [](uint32_t x, uint32_t y) { return x > y ? x : y; });
#pragma unroll
                for (int i = V - 1; i >= 0; --i) at = key[i] == best ? (uint32_t)(e0 + i) : at;
                at = reduce<G>(at, [](uint32_t x, uint32_t y) { return x < y ? x : y; });
                const int e = best > NOTHING ? (int)at : -1;
                if (j == 0) {
                    top = e >= 0 ? of_key(best) : 0.0f;
                    float sum = 0.0f;
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        p[i] = expf(p[i] - top);
                        sum += p[i];
                    }
                    sum = group_sum<G>(sum);
                    all = e >= 0 ? sum : 1.0f;
                    inv = e >= 0 ? 1.0f / sum : 0.0f;  // (of the loss's sums; a weight is divided)
                    live += e >= 0;
                }
#pragma unroll
                for (int i = 0; i < V; ++i) key[i] = e == e0 + i ? 0 : key[i];
                if (e0 == 0) {
                    s_w[token * k + j] = of_key(best);
                    s_e[token * k + j] = e;
                }
            }
            // the choices' weights, a choice per lane of the token's
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            float wsum = 0.0f;
            for (int j = tid % G; j < k; j += G) {
                const int e = s_e[token * k + j];
                const float q = e >= 0 ? expf(s_w[token * k + j] - top) / all : 0.0f;
                wsum += q;
                s_w[token * k + j] = q;
                if (e >= 0) atomicOr((unsigned long long*)&masks[e], 1ull << token);
            }
            wsum = group_sum<G>(wsum);
            if (e0 == 0) s_f[token] = a.renormalize && wsum > 0.0f ? wsum : 1.0f;
#pragma unroll
            for (int i = 0; i < V; ++i) psum[i] += p[i] * inv;
        }
        __syncthreads();
        // the choices leave in order; a choice's rank among those of its expert in this block
        const int64_t left = (a.T - c * C) * k, n = left < C * k ? left : C * k;
        for (int i = tid; i < n; i += NT) {
            const int e = s_e[i], tk = i / k;
            const int64_t at = c * C * k + i;
            a.weights[at] = s_w[i] / s_f[tk];
            a.experts[at] = e;
            const int rank = e < 0 ? -1 : first[e] + __popcll(masks[e] & ((1ull << tk) - 1ull));
            if constexpr (!SINGLE) a.slots[at] = rank;
            else s_w[i] = __int_as_float(rank);
        }
        __syncthreads();
        if (tid < E) first[tid] += __popcll(masks[tid]);
    }
    // sums over the block's tokens: the wave's, then the waves' in order
#pragma unroll
    for (int i = 0; i < V; ++i) psum[i] = sum_across<G>(psum[i]);
    live = (int)sum_across<G>((float)live);  // (exact: fewer than 2^24)
    if (lane < G) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (e0 + i < E) sums[wave * E + e0 + i] = psum[i];
        if (lane == 0) s_live[wave] = live;
    }
    __syncthreads();
    float p = 0.0f;
    int routed = 0;
    for (int w = 0; w < NW; ++w) {
        if (tid < E) p += sums[w * E + tid];
        routed += s_live[w];
    }
    if constexpr (!SINGLE) {
        if (tid < E) {
            a.block_counts[(int64_t)blockIdx.x * E + tid] = first[tid];
            a.block_sums[(int64_t)blockIdx.x * E + tid] = p;
        }
        if (tid == 0) a.block_live[blockIdx.x] = routed;
    } else {
        __shared__ int64_t wtot[NW];
        __shared__ float s_loss[NW];
        int64_t total;
        const int mine = tid < E ? first[tid] : 0;
        const int64_t before = block_exclusive_scan<NT>(mine, wtot, &total);
        if (tid < E) {
            first[tid] = (int)before;
            a.counts[tid] = mine;
        }
        const float part = wave_sum((float)mine * p);
        if (lane == 0) s_loss[wave] = part;
        __syncthreads();
        const int n = (int)a.T * k;
        for (int i = tid; i < n; i += NT) {
            const int rank = __float_as_int(s_w[i]), e = s_e[i];
            const int slot = rank < 0 ? -1 : first[e] + rank;
            a.slots[i] = slot;
            if (slot >= 0) a.row_tokens[slot] = i / k;
            if (i >= total) a.row_tokens[i] = -1;
        }
        if (tid == 0) {
            float sum = 0.0f;
            for (int w = 0; w < NW; ++w) sum += s_loss[w];
            *a.routed = routed;
            *a.loss = total > 0 ? (float)E * (sum / ((float)total * (float)routed)) : 0.0f;
        }
    }
}

// Offsets of a block's rows: those of the experts before, then of the blocks before within the expert.  A thread adds up
// one expert's counts over every P-th block.
__global__ __launch_bounds__(1024) void moe_rows_kernel(MoeRouteArgs a, int blocks)
{
    extern __shared__ int base[];  // [E]
    __shared__ int64_t wtot[16];
    __shared__ float s_loss[16];
    __shared__ int s_all[1024], s_before[1024];
    __shared__ float s_p[1024];
    const int E = (int)a.E, k = a.k, tid = threadIdx.x, b0 = blockIdx.x;
    const int P = 1024 / E, e = tid % E, part = tid / E;
    int before = 0, all = 0;
    float p = 0.0f;
    // what comes after the scan is requested in front of it
    const int64_t c0 = first_chunk(a, b0, blocks), c1 = first_chunk(a, b0 + 1, blocks);
    const int64_t end = c1 * a.chunk < a.T ? c1 * a.chunk * k : a.T * k, at0 = c0 * a.chunk * k + tid;
    const int expert0 = at0 < end ? a.experts[at0] : -1, rank0 = at0 < end ? a.slots[at0] : -1;
    int live = b0 == 0 && tid < blocks ? a.block_live[tid] : 0;  // (blocks <= MAX_BLOCKS)
    static_assert(MAX_BLOCKS <= 1024, "one block per thread");
    if (part < P) {
        for (int b = part; b < blocks; b += 8 * P) {  // eight loads in flight
            int c[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) c[i] = b + i * P < blocks ? a.block_counts[(b + i * P) * E + e] : 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                all += c[i];
                before += b + i * P < b0 ? c[i] : 0;
            }
        }
        if (b0 == 0)
            for (int b = part; b < blocks; b += 8 * P) {
                float c[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) c[i] = b + i * P < blocks ? a.block_sums[(b + i * P) * E + e] : 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) p += c[i];
            }
    }
    s_all[tid] = all;
    s_before[tid] = before;
    s_p[tid] = p;
    __syncthreads();
    all = before = 0;
    p = 0.0f;
    if (tid < E)
        for (int i = 0; i < P; ++i) {
            all += s_all[i * E + tid];
            before += s_before[i * E + tid];
            p += s_p[i * E + tid];
        }
    int64_t total;
    const int64_t start = block_exclusive_scan<1024>(all, wtot, &total);
    if (tid < E) base[tid] = (int)start + before;
    __syncthreads();
    for (int64_t at = at0; at < end; at += 1024) {
        if (at >= total) a.row_tokens[at] = -1;
        const int x = at == at0 ? expert0 : a.experts[at];
        if (x < 0) continue;
        const int slot = base[x] + (at == at0 ? rank0 : a.slots[at]);
        a.slots[at] = slot;
        a.row_tokens[slot] = (int)(at / k);
    }
    if (b0 != 0) return;
    if (tid < E) a.counts[tid] = all;
    const float loss = wave_sum(tid < E ? (float)all * p : 0.0f);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) live += __shfl_xor(live, o, 64);
    if ((tid & 63) == 0) {
        s_loss[tid >> 6] = loss;
        s_all[tid >> 6] = live;
    }
    __syncthreads();
    if (tid == 0) {
        float sum = 0.0f;
        live = 0;
        for (int w = 0; w < 16; ++w) {
            sum += s_loss[w];
            live += s_all[w];
        }
        *a.routed = live;
        *a.loss = total > 0 ? (float)E * (sum / ((float)total * (float)live)) : 0.0f;
    }
}

// d loss / d l and d w / d l: G lanes per token, each with V neighbouring experts
//   g_e = dL E counts_e / (sum counts x routed)  (+ dw_j at choice j without renormalisation),  dl_e = p_e (g_e - sum p g)
//   renormalised: + w_j (dw_j - sum_i dw_i w_i) at choice j
// Bound by latency (64 experts, k = 6: 16384 tokens 8 to 9 us, 100000 32 us, 1.8 TB/s of what it has to move).
template <int G, int V>
__global__ __launch_bounds__(256) void moe_route_grad_kernel(MoeRouteGradArgs a)
{
    const int E = (int)a.E, e0 = (int)threadIdx.x % G * V;
    const int64_t t = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
    const bool here = t < a.T;  // (the lanes of a wave go through the butterflies together)
    const int64_t es = a.type == DT_F32 ? 4 : 2;
    const bool vec = ((uintptr_t)a.logits | (uintptr_t)(a.ld * es)) % 16 == 0;
    float p[V], g[V], d[V];
    // a token's choices, all of them requested in front of the first use
    int choice[MAX_K];
    float dw[MAX_K], add[MAX_K];
    if (a.grad_weights && here) {
#pragma unroll
        for (int j = 0; j < MAX_K; ++j) {
            if (j >= a.k) continue;
            const int x = a.experts[t * a.k + j];
            choice[j] = x < E ? x : -1;  // (no expert: no choice)
            dw[j] = a.grad_weights[t * a.k + j];
            add[j] = a.weights[t * a.k + j];
        }
    }
    if (here) load_logits<V>((const uint8_t*)a.logits + t * a.ld * es, a.type, e0, E, vec, p);
    float top = -__builtin_inff(), cnt = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        if (!here) p[i] = -__builtin_inff();
        g[i] = e0 + i < E && a.grad_loss ? (float)a.counts[e0 + i] : 0.0f;
        d[i] = 0.0f;
        top = fmaxf(top, p[i]);
        cnt += g[i];
    }
    top = reduce<G>(top, [](float x, float y) { return fmaxf(x, y); });
    const bool none = !(top > -__builtin_inff());  // nothing counts: no gradient
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        p[i] = none ? 0.0f : expf(p[i] - top);
        sum += p[i];
    }
    sum = group_sum<G>(sum);
    if (a.grad_loss) {
        cnt = group_sum<G>(cnt);
        const float live = (float)*a.routed;
        const float f = cnt > 0.0f && live > 0.0f ? *a.grad_loss * ((float)E / (cnt * live)) : 0.0f;  // (no product larger than f)
#pragma unroll
        for (int i = 0; i < V; ++i) g[i] *= f;
    }
    if (a.grad_weights && here) {
        float mean = 0.0f;
#pragma unroll
        for (int j = 0; j < MAX_K; ++j) {
            if (j >= a.k) continue;
            if (!a.renormalize) add[j] = 1.0f;
            mean += choice[j] >= 0 ? dw[j] * add[j] : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < MAX_K; ++j) {
            if (j >= a.k) continue;
            const float x = a.renormalize ? add[j] * (dw[j] - mean) : dw[j];
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (choice[j] == e0 + i) {
                    if (a.renormalize) d[i] += x;
                    else g[i] += x;
                }
        }
    }
    float dot = 0.0f;
    const float inv = none ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        p[i] *= inv;
        dot += p[i] * g[i];
    }
    dot = group_sum<G>(dot);
    if (!here) return;
#pragma unroll
    for (int i = 0; i < V; ++i) d[i] = none ? 0.0f : p[i] * (g[i] - dot) + d[i];
    uint8_t* out = (uint8_t*)a.grad_logits + t * a.ld_grad * es;
    const bool vec_out = ((uintptr_t)a.grad_logits | (uintptr_t)(a.ld_grad * es)) % 16 == 0;
    if (vec_out && e0 + V <= E && a.type == DT_F32) {
#pragma unroll
        for (int i = 0; i < V / 4; ++i)
            ((u32x4*)((float*)out + e0))[i] = (u32x4){__float_as_uint(d[4 * i]), __float_as_uint(d[4 * i + 1]),
                                                      __float_as_uint(d[4 * i + 2]), __float_as_uint(d[4 * i + 3])};
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (e0 + i < E) store_grad(out, e0 + i, d[i], a.type);
    }
}

namespace {

// 16 bytes at an address of any alignment
typedef u32x4 u32x4_any __attribute__((aligned(1)));
template <bool ANY>
using row_word = typename std::conditional<ANY, u32x4_any, u32x4>::type;

// 8 elements of a row of T, at element 8 u; `count` of them where the row ends inside
template <int T, bool ANY>
struct Eight {
    static constexpr int W = T == DT_F32 ? 2 : 1;
    u32x4 w[W];
    __device__ __forceinline__ float get(int e) const
    {
        if constexpr (T == DT_F32) return __uint_as_float(w[e / 4][e % 4]);
        const uint16_t b = (uint16_t)(w[0][e / 2] >> (16 * (e & 1)));
        return T == DT_F16 ? f16_to_f32(b) : bf16_to_f32(b);
    }
    __device__ __forceinline__ void load(const void* row, int64_t u, int count)
    {
        if (!ANY || count >= 8) {
#pragma unroll
            for (int i = 0; i < W; ++i) w[i] = __builtin_nontemporal_load((const row_word<ANY>*)row + u * W + i);
            return;
        }
        w[0] = w[W - 1] = (u32x4){0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (e >= count) continue;
            if constexpr (T == DT_F32) w[e / 4][e % 4] = ((const uint32_t*)row)[u * 8 + e];
            else w[0][e / 2] |= (uint32_t)((const uint16_t*)row)[u * 8 + e] << (16 * (e & 1));
        }
    }
    // SAT: what is finite saturates in 16-bit types, else it overflows to infinity
    template <bool SAT>
    __device__ __forceinline__ static void store(void* row, int64_t u, int count, const float (&f)[8])
    {
        uint32_t d[8];
        if constexpr (T == DT_F32) {
#pragma unroll
            for (int e = 0; e < 8; ++e) d[e] = __float_as_uint(f[e]);
        } else {
            us2_t top = {0, 0};
#pragma unroll
            for (int e = 0; e < 4; ++e) d[e] = cvt_pair<T == DT_BF16>(f[2 * e], f[2 * e + 1], top);
            if (SAT && __builtin_expect(cvt_special<T == DT_BF16>(top), 0)) {
                auto one = [](float x) { return (uint32_t)f32_to_16_keep_inf<T == DT_BF16>(x); };
#pragma unroll
                for (int e = 0; e < 4; ++e) d[e] = one(f[2 * e]) | (one(f[2 * e + 1]) << 16);
            }
        }
        if (!ANY || count >= 8) {
#pragma unroll
            for (int i = 0; i < W; ++i)
                __builtin_nontemporal_store((u32x4){d[4 * i], d[4 * i + 1], d[4 * i + 2], d[4 * i + 3]},
                                            (row_word<ANY>*)row + u * W + i);
            return;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (e >= count) continue;
            if constexpr (T == DT_F32) ((uint32_t*)row)[u * 8 + e] = d[e];
            else ((uint16_t*)row)[u * 8 + e] = (uint16_t)(d[e / 2] >> (16 * (e & 1)));
        }
    }
};

// a token's slot j, or -1 when it is none of the rows
__device__ __forceinline__ int64_t row_of(const MoeRowsArgs& a, int64_t t, int j)
{
    const int64_t slot = a.slots[t * a.k + j];
    return slot >= 0 && slot < a.T * a.k ? slot : -1;
}

// four waves per workgroup: the wave's number among all (a scalar, so that what a wave shares is loaded once)
__device__ __forceinline__ int64_t wave_of() { return (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

}  // namespace

// Rows to the experts' order: `waves` waves per token, interleaved by 1 KB, read its row once and write it to its k slots, so
// nothing is read twice; they also clear the rows t k .. t k + k - 1 where no token has them (they lie behind the routed
// ones).  Bound by memory: 4096 tokens x 2 of 4096 bytes in 9.8 us, 5.2 TB/s; 512 x 6 of 2048 in 4.7.
template <bool ANY>
__global__ __launch_bounds__(256) void moe_dispatch_kernel(MoeRowsArgs a, int waves)
{
    const int64_t w = wave_of(), t = a.first + w / waves, words = a.row_bytes / 16;
    if (t >= a.T) return;
    const int c0 = (int)(w % waves) * 64, lane = threadIdx.x & 63;
    const int rest = ANY ? (int)(a.row_bytes % 16) : 0;
    const uint8_t* src = (const uint8_t*)a.x + t * a.ldx;
    uint8_t* out = (uint8_t*)a.out;
    // f(the token's row of choice j or -1, row t k + j where no token has it, else -1)
    auto each = [&](auto f) {
        for (int j0 = 0; j0 < a.k; j0 += 4) {
            int64_t slot[4], clear[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int at = j0 + j < a.k ? j0 + j : 0;
                slot[j] = row_of(a, t, at);
                clear[j] = a.row_tokens[t * a.k + at] < 0 ? t * a.k + at : -1;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j0 + j < a.k) f(slot[j], clear[j]);
        }
    };
    const float scale = a.scale_out ? a.scale[t] : 0.0f;
    for (int64_t c = c0 + lane; c < words; c += waves * 64) {
        const u32x4 v = ((const row_word<ANY>*)src)[c];
        each([&](int64_t slot, int64_t clear) {
            if (slot >= 0) __builtin_nontemporal_store(v, (row_word<ANY>*)(out + slot * a.row_bytes) + c);
            if (clear >= 0) __builtin_nontemporal_store((u32x4){0, 0, 0, 0}, (row_word<ANY>*)(out + clear * a.row_bytes) + c);
        });
    }
    // the bytes behind the last whole word, and the scales
    if (c0 == 0 && (lane < rest || (lane == 16 && a.scale_out))) {
        const int64_t at = words * 16 + lane;
        const uint8_t byte = lane < rest ? src[at] : 0;
        each([&](int64_t slot, int64_t clear) {
            if (lane == 16) {
                if (slot >= 0) a.scale_out[slot] = scale;
                if (clear >= 0) a.scale_out[clear] = 0.0f;
            } else {
                if (slot >= 0) out[slot * a.row_bytes + at] = byte;
                if (clear >= 0) out[clear * a.row_bytes + at] = 0;
            }
        });
    }
}

// out_t = sum_j w_tj y[slot_tj] + residual_t: fp32, in the order of j, one rounding (a finite sum saturates).  `waves` waves per token, interleaved by
// 512 elements; four rows' loads of a thread are in flight together (a choice of no row reads row 0 and is dropped).  Bound by
// memory: 4096 x 2 rows of 4096 bf16 with residual in 26 us, 5.2 TB/s; x 8 rows of 2048 in 33 us.
template <int T, bool ANY>
__global__ __launch_bounds__(256) void moe_combine_kernel(MoeRowsArgs a, int waves)
{
    constexpr int ES = T == DT_F32 ? 4 : 2;
    const int64_t w = wave_of(), t = a.first + w / waves, pitch = a.n * ES;
    if (t >= a.T) return;
    for (int64_t u = w % waves * 64 + (threadIdx.x & 63); u * 8 < a.n; u += waves * 64) {
        const int count = ANY && a.n - u * 8 < 8 ? (int)(a.n - u * 8) : 8;
        float v[8] = {};
        Eight<T, ANY> r;
        if (a.residual) r.load((const uint8_t*)a.residual + t * pitch, u, count);
        for (int j0 = 0; j0 < a.k; j0 += 4) {
            Eight<T, ANY> y[4];
            bool ok[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (j0 + j >= a.k) continue;
                const int64_t slot = row_of(a, t, j0 + j);
                ok[j] = slot >= 0;
                y[j].load((const uint8_t*)a.y + (ok[j] ? slot : 0) * pitch, u, count);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (j0 + j >= a.k) continue;
                const float weight = a.weights[t * a.k + j0 + j];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] += ok[j] ? weight * y[j].get(e) : 0.0f;
            }
        }
        if (a.residual) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += r.get(e);
        }
        Eight<T, ANY>::template store<true>((uint8_t*)a.out + t * pitch, u, count, v);
    }
}

// dw_tj = <dout_t, y[slot_tj]>, dy[slot_tj] = w_tj dout_t (past its type's range infinite); rows of no token get 0.  An item is a token and up to `per` <= 4 of its
// choices, whose gradient it reads once; W waves do it: four, or one for rows of fewer than 2048 (13370 tokens x 2 of 512:
// 17 us, with four waves 43; 8192 x 2 of 2048: 34, with one wave 42).  Few items take a choice each (14 tokens x 8 of 3904: 4.5
// us, four choices 7.0; 512 x 6 of 2048: 14, four 10).  Bound by memory: 4096 x 2 rows of 4096 bf16 in 35 us, 4.8 TB/s.
template <int T, bool ANY, int W>
__global__ __launch_bounds__(256) void moe_combine_grad_kernel(MoeRowsArgs a, int per)
{
    constexpr int ES = T == DT_F32 ? 4 : 2;
    __shared__ float red[4][4];
    const int groups = (a.k + per - 1) / per, lane = (int)threadIdx.x % (64 * W);
    const int64_t item = a.first + wave_of() / W, pitch = a.n * ES;
    const bool here = item < a.T * groups;  // (an item past the last does nothing, but meets the others)
    const int64_t t = here ? item / groups : 0;
    const int j0 = (int)(here ? item % groups : 0) * per, jn = here ? (a.k - j0 < per ? a.k - j0 : per) : 0;
    float dot[4] = {};
    if (here) {
        int64_t slot[4];
        float w[4];
        bool clear[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t r = t * a.k + j0 + j;
            slot[j] = j < jn ? row_of(a, t, j0 + j) : -1;
            w[j] = j < jn && a.out ? a.weights[r] : 0.0f;
            clear[j] = j < jn && a.out && a.row_tokens[r] < 0;
        }
        for (int64_t u = lane; u * 8 < a.n; u += 64 * W) {
            const int count = ANY && a.n - u * 8 < 8 ? (int)(a.n - u * 8) : 8;
            Eight<T, ANY> d, y[4];
            d.load((const uint8_t*)a.x + t * pitch, u, count);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j < jn && a.grad_weights) y[j].load((const uint8_t*)a.y + (slot[j] >= 0 ? slot[j] : 0) * pitch, u, count);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (j >= jn) continue;
                if (a.grad_weights && slot[j] >= 0) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) dot[j] = fmaf(d.get(e), y[j].get(e), dot[j]);
                }
                float f[8];
                if (a.out && slot[j] >= 0) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[e] = w[j] * d.get(e);
                    Eight<T, ANY>::template store<false>((uint8_t*)a.out + slot[j] * pitch, u, count, f);
                }
                if (clear[j]) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[e] = 0.0f;
                    Eight<T, ANY>::template store<false>((uint8_t*)a.out + (t * a.k + j0 + j) * pitch, u, count, f);
                }
            }
        }
    }
    if (!a.grad_weights) return;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (j >= jn) continue;
        dot[j] = wave_sum(dot[j]);
        if constexpr (W == 1) {
            if (lane == 0) a.grad_weights[t * a.k + j0 + j] = dot[j];
        } else {
            if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6][j] = dot[j];
        }
    }
    if constexpr (W > 1) {
        __syncthreads();
        const int j = lane, first = (int)threadIdx.x / (64 * W) * W;
        if (j < jn) {
            float sum = red[first][j];
#pragma unroll
            for (int v = 1; v < W; ++v) sum += red[first + v][j];
            a.grad_weights[t * a.k + j0 + j] = sum;
        }
    }
}

namespace {
// tokens of a chunk: 64, or 16 where experts are many and tokens few, so that more CUs share the k searches through the logits
// (512 tokens, 256 experts, k = 8: both launches 13.7 us, with 64 21.4)
int route_chunk(int64_t T, int64_t E) { return E > 64 && T <= 2048 ? 16 : CHUNK; }
int64_t route_blocks(int64_t T, int64_t E)
{
    const int64_t chunk = route_chunk(T, E), chunks = (T + chunk - 1) / chunk;
    return chunks < MAX_BLOCKS ? chunks : MAX_BLOCKS;
}
// one block for all tokens (64 tokens, 256 experts, k = 8: alone 17 us, by chunks 13.2; 6 tokens 8.7)
bool route_alone(int64_t T, int64_t E) { return T <= 1 || (T <= MOE_ROUTE_ALONE && T * E <= 8192); }

template <int G, int V, bool SINGLE>
hipError_t launch_route(const MoeRouteArgs& a, int blocks, hipStream_t st)
{
    constexpr auto kern = moe_route_kernel<G, V, SINGLE>;
    constexpr uint32_t per = 8 + 4 * (route_threads<G> / 64) + 4;  // bytes of LDS per expert
    const hipError_t e = ensure_dynamic_lds<kern>(G * V * per);
    if (e != hipSuccess) return e;
    launch_k(kern, dim3((unsigned)blocks), dim3(route_threads<G>), (uint32_t)a.E * per, st, a);
    return hipGetLastError();
}
template <bool SINGLE>
hipError_t launch_route_experts(const MoeRouteArgs& a, int blocks, hipStream_t st)
{
    if (a.E <= 8) return launch_route<1, 8, SINGLE>(a, blocks, st);
    if (a.E <= 16) return launch_route<2, 8, SINGLE>(a, blocks, st);
    if (a.E <= 32) return launch_route<4, 8, SINGLE>(a, blocks, st);
    if (a.E <= 64) return launch_route<8, 8, SINGLE>(a, blocks, st);
    if (a.E <= 128) return launch_route<16, 8, SINGLE>(a, blocks, st);
    if (a.E <= 256) return launch_route<32, 8, SINGLE>(a, blocks, st);
    if (a.E <= 512) return launch_route<64, 8, SINGLE>(a, blocks, st);
    return launch_route<64, 16, SINGLE>(a, blocks, st);
}
}  // namespace

size_t moe_route_ws_bytes(int64_t T, int64_t E)
{
    const int64_t blocks = route_blocks(T, E);
    return route_alone(T, E) ? 0 : (size_t)blocks * ((size_t)E * 8 + 4);
}

hipError_t launch_moe_route(MoeRouteArgs a, void* ws, hipStream_t st)
{
    if (route_alone(a.T, a.E) || !ws) {
        a.chunk = CHUNK;
        a.chunks = (int)((a.T + CHUNK - 1) / CHUNK);
        return a.T <= MOE_ROUTE_ALONE ? launch_route_experts<true>(a, 1, st) : hipErrorInvalidValue;
    }
    const int blocks = (int)route_blocks(a.T, a.E);
    a.chunk = route_chunk(a.T, a.E);
    a.chunks = (int)((a.T + a.chunk - 1) / a.chunk);
    a.block_counts = (int*)ws;
    a.block_sums = (float*)(a.block_counts + (int64_t)blocks * a.E);
    a.block_live = (int*)(a.block_sums + (int64_t)blocks * a.E);
    const hipError_t e = launch_route_experts<false>(a, blocks, st);
    if (e != hipSuccess) return e;
    launch_k(moe_rows_kernel, dim3((unsigned)blocks), dim3(1024), (uint32_t)a.E * 4, st, a, blocks);
    return hipGetLastError();
}

namespace {
template <int G, int V>
hipError_t launch_grad(const MoeRouteGradArgs& a, hipStream_t st)
{
    constexpr int64_t TOKENS = (1ll << 31) / G;  // of a launch: a grid has fewer than 2^32 threads
    const int64_t es = a.type == DT_F32 ? 4 : 2;
    for (int64_t t = 0; t < a.T; t += TOKENS) {
        MoeRouteGradArgs b = a;
        b.T = a.T - t < TOKENS ? a.T - t : TOKENS;
        b.grad_logits = (uint8_t*)a.grad_logits + t * a.ld_grad * es;
        b.logits = (const uint8_t*)a.logits + t * a.ld * es;
        if (a.weights) b.weights += t * a.k;
        if (a.experts) b.experts += t * a.k;
        if (a.grad_weights) b.grad_weights += t * a.k;
        launch_k((moe_route_grad_kernel<G, V>), dim3((unsigned)((b.T + 256 / G - 1) / (256 / G))), dim3(256), 0u, st, b);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}
}  // namespace

hipError_t launch_moe_route_grad(const MoeRouteGradArgs& a, hipStream_t st)
{
    if (a.E <= 8) return launch_grad<1, 8>(a, st);
    if (a.E <= 16) return launch_grad<2, 8>(a, st);
    if (a.E <= 32) return launch_grad<4, 8>(a, st);
    if (a.E <= 64) return launch_grad<8, 8>(a, st);
    if (a.E <= 128) return launch_grad<16, 8>(a, st);
    if (a.E <= 256) return launch_grad<32, 8>(a, st);
    if (a.E <= 512) return launch_grad<64, 8>(a, st);
    return launch_grad<64, 16>(a, st);
}

namespace {
// waves that share a token's row of `units` 16-byte (or 8-element) words: one word per thread, which is what is fastest from a
// handful of tokens (14 x 8 rows of 3904: combine 6.9 us, with half as many waves 13) to 16384, within a grid's bound
int row_waves(int64_t T, int64_t units)
{
    const int64_t all = (units + 63) / 64, most = (1 << 20) / T;
    return (int)(all < 1 ? 1 : all < most ? all : most > 1 ? most : 1);
}

// A grid has fewer than 2^32 threads: launches of up to 2^25 items (tokens; as many have a wave each).  f(args, how many)
template <class F>
hipError_t in_pieces(const MoeRowsArgs& a, int64_t items, F f)
{
    constexpr int64_t MOST = 1 << 25;
    MoeRowsArgs b = a;
    for (b.first = 0; b.first < items; b.first += MOST) {
        const hipError_t e = f(b, items - b.first < MOST ? items - b.first : MOST);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

// rows of whole 16-byte words (f32: of 8 elements), all of them aligned
bool rows_aligned(const MoeRowsArgs& a)
{
    const uintptr_t bits = (uintptr_t)a.x | (uintptr_t)a.out | (uintptr_t)a.y | (uintptr_t)a.residual;
    return bits % 16 == 0 && a.n % 8 == 0;
}
// f(type, any alignment)
template <class F>
hipError_t with_row_kernel(const MoeRowsArgs& a, F f)
{
    auto types = [&](auto any) {
        if (a.type == DT_F16) f(std::integral_constant<int, DT_F16>{}, any);
        else if (a.type == DT_BF16) f(std::integral_constant<int, DT_BF16>{}, any);
        else f(std::integral_constant<int, DT_F32>{}, any);
    };
    if (rows_aligned(a)) types(std::false_type{});
    else types(std::true_type{});
    return hipGetLastError();
}
}  // namespace

hipError_t launch_moe_dispatch(const MoeRowsArgs& in, hipStream_t st)
{
    const uintptr_t bits = (uintptr_t)in.x | (uintptr_t)in.out | (uintptr_t)in.ldx | (uintptr_t)in.row_bytes;
    const int waves = row_waves(in.T, in.row_bytes / 16);  // (T > 2^20: 1)
    return in_pieces(in, in.T, [&](const MoeRowsArgs& a, int64_t tokens) {
        const dim3 grid((unsigned)((tokens * waves + 3) / 4)), block(256);
        if (bits % 16 == 0) launch_k(moe_dispatch_kernel<false>, grid, block, 0u, st, a, waves);
        else launch_k(moe_dispatch_kernel<true>, grid, block, 0u, st, a, waves);
        return hipGetLastError();
    });
}

hipError_t launch_moe_combine(const MoeRowsArgs& in, hipStream_t st)
{
    const int waves = row_waves(in.T, (in.n + 7) / 8);
    return in_pieces(in, in.T, [&](const MoeRowsArgs& a, int64_t tokens) {
        return with_row_kernel(a, [&](auto type, auto any) {
            launch_k((moe_combine_kernel<decltype(type)::value, decltype(any)::value>), dim3((unsigned)((tokens * waves + 3) / 4)),
                     dim3(256), 0u, st, a, waves);
        });
    });
}

hipError_t launch_moe_combine_grad(const MoeRowsArgs& in, hipStream_t st)
{
    const int per = in.T * in.k <= 1024 ? 1 : 4;  // (808 rows: alike)
    const int64_t all = in.T * ((in.k + per - 1) / per);
    return in_pieces(in, all, [&](const MoeRowsArgs& a, int64_t items) {
        return with_row_kernel(a, [&](auto type, auto any) {
            constexpr int T = decltype(type)::value;
            constexpr bool ANY = decltype(any)::value;
            if (a.n < 2048 || all >= 1 << 24)  // (four waves each: within a grid)
                launch_k((moe_combine_grad_kernel<T, ANY, 1>), dim3((unsigned)((items + 3) / 4)), dim3(256), 0u, st, a, per);
            else
                launch_k((moe_combine_grad_kernel<T, ANY, 4>), dim3((unsigned)items), dim3(256), 0u, st, a, per);
        });
    });
}

}  // namespace ascq
