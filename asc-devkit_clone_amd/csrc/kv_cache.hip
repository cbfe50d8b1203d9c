// kv_cache.hip -- writing the paged int4 key / value cache, and cutting it to the tokens that matter.
//
// A cached row of d channels (one token, one key head) is d / 2 bytes of int4 codes and one (scale, offset) pair of f16 per
// `group` channels; it stands for value(c) = f16(c scale + offset).  Pages are [key head][token][channel], so that the tokens
// of a head lie side by side.
#include "common.h"

namespace ascq {

namespace {

typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef v4f v4f_any __attribute__((aligned(4)));

// 8 channels of a row as fp32: NaN counts as 0, magnitudes end at 61440 -- beyond it a code's value could round past f16
template <int TYPE>
__device__ __forceinline__ void load8(float (&x)[8], const void* p)
{
    if constexpr (TYPE == DT_F32) {
        const v4f a = ((const v4f_any*)p)[0], b = ((const v4f_any*)p)[1];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = a[i], x[i + 4] = b[i];
    } else {
        const u32x4 w = *(const u32x4_any*)p;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint16_t lo = (uint16_t)w[i], hi = (uint16_t)(w[i] >> 16);
            x[2 * i] = TYPE == DT_BF16 ? bf16_to_f32(lo) : f16_to_f32(lo);
            x[2 * i + 1] = TYPE == DT_BF16 ? bf16_to_f32(hi) : f16_to_f32(hi);
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        x[i] = x[i] != x[i] ? 0.0f : x[i];
        x[i] = __builtin_fminf(__builtin_fmaxf(x[i], -61440.0f), 61440.0f);
    }
}

// A lane takes 8 channels of a row (one word of codes), the group / 8 lanes of a group find its range by exchanges.  fp32 in
// the order that the header states, every operation IEEE: the same bits as that order anywhere.
template <int TYPE>
__global__ __launch_bounds__(256) void kv_append_kernel(KvAppendArgs a)
{
    const int words = a.c.d / 8;  // lanes of a row: 8, 16, 32
    const int64_t lane = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int w = (int)(lane % words);
    const int64_t row = lane / words;  // token, keys or values, head
    const int h = (int)(row % a.c.kv_heads);
    const int64_t rest = row / a.c.kv_heads;
    const bool value = rest & 1;
    const int64_t t = a.first + (rest >> 1);
    const int64_t slot = t < a.T ? a.slots[t] : -1;
    const int64_t page = slot >> a.c.page_shift;
    const bool live = slot >= 0 && page < a.c.pages;
    float x[8] = {};
    if (live) {
        const int64_t at = t * (value ? a.ld_v : a.ld_k) + h * (value ? a.hd_v : a.hd_k) + 8 * w;
        load8<TYPE>(x, (const uint8_t*)(value ? a.v : a.k) + at * (TYPE == DT_F32 ? 4 : 2));
    }
    float lo = x[0], hi = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) lo = __builtin_fminf(lo, x[i]), hi = __builtin_fmaxf(hi, x[i]);
    const int lanes = a.c.group / 8;
    for (int off = 1; off < lanes; off <<= 1) {
        lo = __builtin_fminf(lo, __shfl_xor(lo, off, 64));
        hi = __builtin_fmaxf(hi, __shfl_xor(hi, off, 64));
    }
    if (!live) return;
    const _Float16 s = (_Float16)((hi - lo) / 15.0f);
    const _Float16 o = (_Float16)(lo + 8.0f * (float)s);
    const float inv = (float)s > 0.0f ? 1.0f / (float)s : 0.0f;
    uint32_t code = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float c = __builtin_rintf((x[i] - (float)o) * inv);
        code |= ((uint32_t)(int)__builtin_fminf(__builtin_fmaxf(c, -8.0f), 7.0f) & 15u) << (4 * i);
    }
    const int64_t place = ((int64_t)h << a.c.page_shift) + (slot & (((int64_t)1 << a.c.page_shift) - 1));
    uint8_t* codes = (value ? a.c.v : a.c.k) + page * a.c.ld_code + place * (a.c.d / 2);
    ((uint32_t*)codes)[w] = code;
    if (w % lanes == 0) {
        uint32_t* scales = (value ? a.c.v_scale : a.c.k_scale) + page * a.c.ld_scale + place * (a.c.d / a.c.group);
        scales[w / lanes] = (uint32_t)h_bits(s) | ((uint32_t)h_bits(o) << 16);
    }
}

}  // namespace

hipError_t launch_kv_append(KvAppendArgs a, hipStream_t st)
{
    // tokens of a launch: fewer than 2^31 lanes
    const int64_t per = (int64_t)a.c.kv_heads * 2 * (a.c.d / 8);
    const int64_t most = ((int64_t)1 << 31) / per;
    for (a.first = 0; a.first < a.T; a.first += most) {
        const int64_t n = a.T - a.first < most ? a.T - a.first : most;
        KvAppendArgs part = a;
        part.T = a.first + n;
        const dim3 grid((uint32_t)((n * per + 255) / 256));
        if (a.type == DT_F32) launch_k(kv_append_kernel<DT_F32>, grid, dim3(256), 0, st, part);
        else if (a.type == DT_BF16) launch_k(kv_append_kernel<DT_BF16>, grid, dim3(256), 0, st, part);
        else launch_k(kv_append_kernel<DT_F16>, grid, dim3(256), 0, st, part);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

namespace {

// a weight as an integer of the same order: NaN lowest, -0 equal to 0
__device__ __forceinline__ uint32_t order_key(float w)
{
    if (w != w) return 0u;
    const uint32_t u = __float_as_uint(w + 0.0f);
    return (u >> 31) ? ~u : u | 0x80000000u;
}

constexpr int SEL = 1024;  // threads of a selection

// Which tokens of a (sequence, head) stay.  The threshold -- the need-th largest weight among the tokens before the last
// `recent` -- is found digit by digit (11, 11 and 10 bits of the ordered key) by counting; then every wave takes a run of
// positions, counts what stays, and writes the positions in order: of weights equal to the threshold the first ones stay.
__global__ __launch_bounds__(SEL) void kv_select_kernel(KvEvictArgs a)
{
    __shared__ uint32_t hist[2048];
    __shared__ uint32_t pick[2];  // digit, how many are still needed of it
    __shared__ uint32_t above[SEL / 64], equal[SEL / 64];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int h = (int)(blockIdx.x % a.c.kv_heads);
    const int64_t b = a.first + blockIdx.x / a.c.kv_heads;
    const int64_t most = (int64_t)a.s.table_pages << a.c.page_shift;
    int64_t len64 = a.s.lengths[b];
    len64 = len64 < 0 ? 0 : len64 > most ? most : len64;
    const int len = (int)len64;
    const int n = len < a.keep ? len : a.keep;
    int* kept = a.kept + (b * a.c.kv_heads + h) * (int64_t)a.keep;
    const float* w = a.weights + (b * a.c.kv_heads + h) * a.cap;
    if (h == 0 && tid == 0) a.lengths_out[b] = n;
    for (int i = n + tid; i < a.keep; i += SEL) kept[i] = -1;
    if (len <= a.keep) {
        for (int i = tid; i < n; i += SEL) kept[i] = i;
        return;
    }
    const int old = len - a.recent;                 // (recent <= keep < len)
    uint32_t need = (uint32_t)(a.keep - a.recent);  // to be chosen among the first `old`
    for (int i = tid; i < a.recent; i += SEL) kept[need + i] = old + i;
    if (need == 0) return;
    uint32_t prefix = 0, mask = 0;
#pragma unroll 1
    for (int digit = 0; digit < 3; ++digit) {
        const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0;
        const uint32_t bins = digit == 2 ? 1024 : 2048;
        for (uint32_t i = tid; i < 2048; i += SEL) hist[i] = 0;
        __syncthreads();
        for (int i = tid; i < old; i += SEL) {
            const uint32_t key = order_key(w[i]);
            if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & (bins - 1)], 1u);
        }
        __syncthreads();
        // from the top bin down: a wave sums 64 lanes' runs of bins
        if (wave == 0) {
            const uint32_t run = bins / 64;
            uint32_t mine = 0;
            for (uint32_t i = 0; i < run; ++i) mine += hist[bins - 1 - (lane * run + i)];
            uint32_t before = mine;  // inclusive prefix over lanes
            for (int off = 1; off < 64; off <<= 1) {
                const uint32_t up = __shfl_up(before, off, 64);
                if (lane >= off) before += up;
            }
            before -= mine;
            if (before < need && need <= before + mine) {
                uint32_t left = need - before, i = 0;
                while (i + 1 < run && hist[bins - 1 - (lane * run + i)] < left) left -= hist[bins - 1 - (lane * run + i)], ++i;
                pick[0] = bins - 1 - (lane * run + i);
                pick[1] = left;
            }
        }
        __syncthreads();
        prefix |= pick[0] << shift;
        mask |= (bins - 1) << shift;
        need = pick[1];
        __syncthreads();
    }
    // `need` tokens of weight equal to the threshold stay, and all above it
    const int per = (((old + SEL / 64 - 1) / (SEL / 64)) + 63) & ~63;
    const int from = wave * per < old ? wave * per : old, to = from + per < old ? from + per : old;
    uint32_t more = 0, same = 0;
    for (int i = from; i < to; i += 64) {
        const uint32_t key = i + lane < to ? order_key(w[i + lane]) : 0u;
        more += __popcll(__ballot(i + lane < to && key > prefix));
        same += __popcll(__ballot(i + lane < to && key == prefix));
    }
    if (lane == 0) above[wave] = more, equal[wave] = same;
    __syncthreads();
    uint32_t at = 0, ties = 0;
    for (int i = 0; i < wave; ++i) at += above[i], ties += equal[i];
    at += ties < need ? ties : need;
    const uint64_t lower = ((uint64_t)1 << lane) - 1;
    for (int i = from; i < to; i += 64) {
        const bool in = i + lane < to;
        const uint32_t key = in ? order_key(w[i + lane]) : 0u;
        const uint64_t eq = __ballot(in && key == prefix);
        const bool stay = in && (key > prefix || (key == prefix && ties + __popcll(eq & lower) < need));
        const uint64_t all = __ballot(stay);
        if (stay) kept[at + __popcll(all & lower)] = i + lane;
        at += __popcll(all);
        ties += __popcll(eq);
    }
}

// where token t of a sequence lies: its page, or -1
__device__ __forceinline__ int64_t page_of(const int* table, int pages_of_row, int t, const KvCacheArgs& c)
{
    const int col = t >> c.page_shift;
    if (col >= pages_of_row) return -1;
    const int64_t p = table[col];
    return p >= 0 && p < c.pages ? p : -1;
}

constexpr int MOVE = 1024;  // threads of a move

// every thread's loads have returned before any thread goes on
__device__ __forceinline__ void reads_done()
{
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

// Moves the kept tokens of a (sequence, head) to its first places, in order.  Four planes: keys, values, and their scales; a
// fifth moves the weights.  A piece is WORDS 32-bit words of a row.  To other pages (gridDim.x runs of tokens) nothing is in
// the way.  In place, one workgroup takes the tokens of a plane in order, all reads of a run before its writes: the token of
// place i comes from a position >= i, so that later reads lie behind all earlier writes.
template <int WORDS>
__device__ __forceinline__ void move_rows(const KvEvictArgs& a, uint32_t* pool, int64_t ld, int words, int64_t b, int h, int n)
{
    typedef uint32_t piece __attribute__((ext_vector_type(WORDS)));
    const int* kept = a.kept + (b * a.c.kv_heads + h) * (int64_t)a.keep;
    const int* src = a.s.table + b * a.s.ld_table;
    const bool away = a.into != nullptr;
    const int* dst = away ? a.into + b * a.ld_into : src;
    const int dst_pages = away ? a.into_pages : a.s.table_pages;
    const int pieces = words / WORDS, tokens = MOVE / pieces;  // tokens of a run
    const int p = threadIdx.x % pieces, mine = threadIdx.x / pieces;
    const int mask = (1 << a.c.page_shift) - 1;
    constexpr int DEEP = 4;
    for (int64_t base = (int64_t)blockIdx.x * tokens * DEEP; base < n; base += (int64_t)gridDim.x * tokens * DEEP) {
        piece x[DEEP];
        int to[DEEP];
#pragma unroll
        for (int u = 0; u < DEEP; ++u) {
            const int64_t i = base + u * tokens + mine;
            to[u] = -1;
            if (mine < tokens && i < n) {
                const int t = kept[i];
                to[u] = !away && t == i ? -1 : (int)i;
                const int64_t page = page_of(src, a.s.table_pages, t, a.c);
                const uint32_t* row = pool + (page < 0 ? 0 : page) * ld + (((int64_t)h << a.c.page_shift) + (t & mask)) * words;
                x[u] = page < 0 ? piece{} : ((const piece*)row)[p];  // (a token on no page holds nothing)
            }
        }
        if (!away) reads_done();
#pragma unroll
        for (int u = 0; u < DEEP; ++u) {
            if (to[u] < 0) continue;
            const int64_t page = page_of(dst, dst_pages, to[u], a.c);
            if (page < 0) continue;
            uint32_t* row = pool + page * ld + (((int64_t)h << a.c.page_shift) + (to[u] & mask)) * words;
            ((piece*)row)[p] = x[u];
        }
    }
}

__global__ __launch_bounds__(MOVE) void kv_move_kernel(KvEvictArgs a)
{
    const int h = (int)(blockIdx.y % a.c.kv_heads);
    const int64_t b = a.first + blockIdx.y / a.c.kv_heads;
    const int n = a.lengths_out[b];
    const int plane = blockIdx.z;
    const int words = a.c.d / 8, groups = a.c.d / a.c.group;
    if (plane == 4) {
        // the weights: gathered to the front, zeros behind; a run's reads end before its writes
        const float* w = a.weights + (b * a.c.kv_heads + h) * a.cap;
        float* out = a.weights_out + (b * a.c.kv_heads + h) * a.cap_out;
        const int* kept = a.kept + (b * a.c.kv_heads + h) * (int64_t)a.keep;
        const bool apart = a.weights != a.weights_out;
        if (!apart && blockIdx.x > 0) return;
        const int64_t step = (apart ? (int64_t)gridDim.x : 1) * MOVE;
        for (int64_t base = (int64_t)blockIdx.x * MOVE; base < a.cap_out; base += step) {
            const int64_t i = base + threadIdx.x;
            const float x = i < n ? w[kept[i]] : 0.0f;
            if (!apart) reads_done();
            if (i < a.cap_out) out[i] = x;
        }
        return;
    }
    if (plane < 2) move_rows<4>(a, (uint32_t*)(plane ? a.c.v : a.c.k), a.c.ld_code / 4, words, b, h, n);
    else if (groups % 4 == 0) move_rows<4>(a, plane == 3 ? a.c.v_scale : a.c.k_scale, a.c.ld_scale, groups, b, h, n);
    else if (groups % 2 == 0) move_rows<2>(a, plane == 3 ? a.c.v_scale : a.c.k_scale, a.c.ld_scale, groups, b, h, n);
    else move_rows<1>(a, plane == 3 ? a.c.v_scale : a.c.k_scale, a.c.ld_scale, groups, b, h, n);
}

}  // namespace

hipError_t launch_kv_evict(KvEvictArgs a, hipStream_t st)
{
    const int64_t runs = ((int64_t)a.keep + 1023) / 1024;
    const uint32_t x = a.into ? (uint32_t)(runs < 64 ? runs : 64) : 1;
    // sequences of a launch: fewer than 2^16 rows of workgroups, and than 2^32 threads
    const int64_t rows = ((int64_t)1 << 32) / (5 * MOVE * (int64_t)x) - 1;
    const int64_t most = (rows < 65535 ? rows : 65535) / a.c.kv_heads;
    for (a.first = 0; a.first < a.s.batch; a.first += most) {
        const int64_t n = a.s.batch - a.first < most ? a.s.batch - a.first : most;
        launch_k(kv_select_kernel, dim3((uint32_t)(n * a.c.kv_heads)), dim3(SEL), 0, st, a);
        hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        hipLaunchKernelGGL(kv_move_kernel, dim3(x, (uint32_t)(n * a.c.kv_heads), 5), dim3(MOVE), 0, st, a);
        e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace ascq
