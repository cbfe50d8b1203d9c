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

// 8 channels of a row as fp32
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
}

// the smallest (HIGH 0) or largest x of 4, 8 or 16 neighbouring lanes, in all of them: exchanges inside a row of 16 lanes, by quads
// and by mirrors (whose halves agree already)
template <int HIGH, int CTRL>
__device__ __forceinline__ float with_lane(float x)
{
    const float y = __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xF, 0xF, true));
    return HIGH ? __builtin_fmaxf(x, y) : __builtin_fminf(x, y);
}
template <int HIGH>
__device__ __forceinline__ float of_group(float x, int lanes)
{
    x = with_lane<HIGH, 0xB1>(x);  // lanes 1 0 3 2 of a quad
    x = with_lane<HIGH, 0x4E>(x);  // 2 3 0 1
    if (lanes > 4) x = with_lane<HIGH, 0x141>(x);  // the mirror of 8
    if (lanes > 8) x = with_lane<HIGH, 0x140>(x);  // of 16
    return x;
}

// A lane takes 8 channels (one word of codes) of a token's keys and values in a head, the group / 8 lanes of a group find its range
// by exchanges.  fp32 in the order that the header states, every operation IEEE: the same bits as that order anywhere.
// The two rows' loads are in flight together, and no index needs a division.  8192 tokens x 8 heads of 128, f16, a group a row, to
// slots in no order: 14.6 us for 42 MB (2.9 TB/s), the vector units busy 55 % of it (two IEEE divisions a group, by each of its lanes),
// and every row's codes and pair are pieces of 64 and 4 bytes at a place of their own.  16 tokens: 3.6 us, launch and latency.
template <int TYPE>
__global__ __launch_bounds__(256) void kv_append_kernel(KvAppendArgs a, int word_bits, FastDiv heads)
{
    const uint32_t lane = blockIdx.x * 256 + threadIdx.x;
    const int w = (int)(lane & ((1u << word_bits) - 1));
    const uint32_t row = lane >> word_bits, token = fdiv(row, heads);
    const int h = (int)(row - token * a.c.kv_heads);
    const int64_t t = a.first + token;
    const int64_t slot = t < a.T ? a.slots[t] : -1;
    const int64_t page = slot >> a.c.page_shift;
    const bool live = slot >= 0 && page < a.c.pages;
    float x[2][8] = {};
    if (t < a.T) {  // (whether they are written or not: the loads do not wait for the slot)
        load8<TYPE>(x[0], (const uint8_t*)a.k + (t * a.ld_k + h * a.hd_k + 8 * w) * (TYPE == DT_F32 ? 4 : 2));
        load8<TYPE>(x[1], (const uint8_t*)a.v + (t * a.ld_v + h * a.hd_v + 8 * w) * (TYPE == DT_F32 ? 4 : 2));
    }
    const int lanes = a.c.group / 8;
    const int64_t place = ((int64_t)h << a.c.page_shift) + (slot & (((int64_t)1 << a.c.page_shift) - 1));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float lo = x[i][0], hi = x[i][0];
        uint32_t big = __float_as_uint(x[i][0]) & 0x7fffffffu;  // (NaN above all)
#pragma unroll
        for (int e = 1; e < 8; ++e) {
            lo = __builtin_fminf(lo, x[i][e]), hi = __builtin_fmaxf(hi, x[i][e]);
            const uint32_t bits = __float_as_uint(x[i][e]) & 0x7fffffffu;
            big = big > bits ? big : bits;
        }
        if (__ballot(big > __float_as_uint(61440.0f))) {
            // NaN counts as 0, magnitudes end at 61440: beyond it a code's value could round past f16
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[i][e] = x[i][e] != x[i][e] ? 0.0f : x[i][e];
                x[i][e] = __builtin_fminf(__builtin_fmaxf(x[i][e], -61440.0f), 61440.0f);
            }
            lo = hi = x[i][0];
#pragma unroll
            for (int e = 1; e < 8; ++e) lo = __builtin_fminf(lo, x[i][e]), hi = __builtin_fmaxf(hi, x[i][e]);
        }
        lo = of_group<0>(lo, lanes);
        hi = of_group<1>(hi, lanes);
        const _Float16 s = (_Float16)((hi - lo) / 15.0f);
        const _Float16 o = (_Float16)(lo + 8.0f * (float)s);
        const float inv = (float)s > 0.0f ? 1.0f / (float)s : 0.0f;
        uint32_t code = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            // clamp(rint(t)) = rint(clamp(t)) for these bounds; added to 1.5 2^23 a number rounds to an integer, its low bits
            const float t = __builtin_amdgcn_fmed3f((x[i][e] - (float)o) * inv, -8.0f, 7.0f) + 12582912.0f;
            code |= (__float_as_uint(t) & 15u) << (4 * e);
        }
        if (!live) continue;
        ((uint32_t*)((i ? a.c.v : a.c.k) + page * a.c.ld_code + place * (a.c.d / 2)))[w] = code;
        if ((w & (lanes - 1)) == 0) {
            uint32_t* scales = (i ? a.c.v_scale : a.c.k_scale) + page * a.c.ld_scale + place * (a.c.d / a.c.group);
            scales[w / lanes] = (uint32_t)h_bits(s) | ((uint32_t)h_bits(o) << 16);
        }
    }
}

}  // namespace

hipError_t launch_kv_append(KvAppendArgs a, hipStream_t st)
{
    // tokens of a launch: 2^30 lanes at most (the division's range is 2^31)
    const int64_t per = (int64_t)a.c.kv_heads * (a.c.d / 8);
    const int64_t most = ((int64_t)1 << 30) / per;
    const int bits = a.c.d == 64 ? 3 : a.c.d == 128 ? 4 : 5;
    const FastDiv heads = fast_div((uint32_t)a.c.kv_heads);
    for (a.first = 0; a.first < a.T; a.first += most) {
        const int64_t n = a.T - a.first < most ? a.T - a.first : most;
        KvAppendArgs part = a;
        part.T = a.first + n;
        const dim3 grid((uint32_t)((n * per + 255) / 256));
        if (a.type == DT_F32) launch_k(kv_append_kernel<DT_F32>, grid, dim3(256), 0, st, part, bits, heads);
        else if (a.type == DT_BF16) launch_k(kv_append_kernel<DT_BF16>, grid, dim3(256), 0, st, part, bits, heads);
        else launch_k(kv_append_kernel<DT_F16>, grid, dim3(256), 0, st, part, bits, heads);
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

constexpr int SEL = 1024, WAVES = SEL / 64;  // threads of a selection

// Which tokens of a (sequence, head) stay.  The threshold -- the need-th largest weight among the tokens before the last `recent` --
// is found digit by digit (11, 11 and 10 bits of the ordered key) by counting; then positions are written in order, those above the
// threshold and, of those equal to it, the first.  Each wave has a run of neighbouring positions, in registers (HELD a thread) unless
// the sequence has more than SEL HELD, and then SEL HELD at a time.  Zeros, which many tokens of a long context have, are counted a
// wave at a time, as counting them one by one in LDS would be one after the other.  Bound by the chain of scans and barriers, not by
// its bytes (16 x 8 rows of up to 4096 weights: 10.9 us, 0.8 MB).
// From the top bin down, a thread two of them (c0 the higher): where the need-th is.  pick: the bin, how many are needed of it.
__device__ __forceinline__ void pick_bin(uint32_t c0, uint32_t c1, uint32_t bins, uint32_t need, uint32_t (&sums)[WAVES],
                                         uint32_t (&pick)[2])
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t sum = c0 + c1;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint32_t up = __shfl_up(sum, off, 64);
        sum += lane >= off ? up : 0;
    }
    if (lane == 63) sums[wave] = sum;
    __syncthreads();
    uint32_t before = sum - c0 - c1;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) before += i < wave ? sums[i] : 0;
    if (before < need && need <= before + c0 + c1) {
        const uint32_t top = bins - 1 - 2 * threadIdx.x;
        const bool first = need <= before + c0;
        pick[0] = first ? top : top - 1;
        pick[1] = first ? need - before : need - before - c0;
    }
    __syncthreads();
}
__device__ __forceinline__ constexpr int shift_of(int digit) { return digit == 0 ? 21 : digit == 1 ? 10 : 0; }
__device__ __forceinline__ constexpr uint32_t bins_of(int digit) { return digit == 2 ? 1024 : 2048; }

template <int HELD>
__global__ __launch_bounds__(SEL) void kv_select_kernel(KvEvictArgs a)
{
    __shared__ uint32_t hist[2048];
    __shared__ uint32_t sums[WAVES], pick[2];  // digit, how many are still needed of it
    __shared__ uint32_t above[WAVES], equal[WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
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

    // pieces of SEL HELD positions at most; a wave's positions of a piece: from + 64 k + lane, k < rows
    const int pieces = (old + SEL * HELD - 1) / (SEL * HELD);
    const int rows = pieces > 1 ? HELD : (old + SEL - 1) / SEL;
    uint32_t key[HELD];
    auto from_of = [&](int piece) { return piece * SEL * HELD + wave * rows * 64; };
    auto load = [&](int piece) {
        const int from = from_of(piece);
        float x[HELD];  // (loaded together; the last one again past the end)
#pragma unroll
        for (int k = 0; k < HELD; ++k) {
            const int i = from + 64 * k + lane;
            x[k] = w[k < rows && i < old ? i : old - 1];
        }
#pragma unroll
        for (int k = 0; k < HELD; ++k) key[k] = order_key(x[k]);
    };
    if (pieces == 1) load(0);
    constexpr uint32_t ZERO = 0x80000000u;
    uint32_t prefix = 0, mask = 0;
#pragma unroll 1
    for (int digit = 0; digit < 3; ++digit) {
        const int shift = shift_of(digit);
        const uint32_t bins = bins_of(digit);
        hist[tid] = hist[tid + SEL] = 0;
        __syncthreads();
        uint32_t zeros = 0;
#pragma unroll 1
        for (int piece = 0; piece < pieces; ++piece) {
            if (pieces > 1) load(piece);
            const int from = from_of(piece);
#pragma unroll
            for (int k = 0; k < HELD; ++k) {
                if (k >= rows || from + 64 * k >= old) break;
                const bool in = from + 64 * k + lane < old && (key[k] & mask) == prefix;
                zeros += __popcll(__ballot(in && key[k] == ZERO));
                if (in && key[k] != ZERO) atomicAdd(&hist[(key[k] >> shift) & (bins - 1)], 1u);
            }
        }
        if (lane == 0 && zeros) atomicAdd(&hist[(ZERO >> shift) & (bins - 1)], zeros);
        __syncthreads();
        const uint32_t top = bins - 1 - 2 * tid;
        const bool counts = 2 * tid < (int)bins;
        pick_bin(counts ? hist[top] : 0, counts ? hist[top - 1] : 0, bins, need, sums, pick);
        prefix |= pick[0] << shift;
        mask |= (bins - 1) << shift;
        need = pick[1];
    }
    // `need` tokens of weight equal to the threshold stay, and all above it
    uint32_t at = 0, ties = 0;  // places and equal ones before this piece
    const uint64_t lower = ((uint64_t)1 << lane) - 1;
#pragma unroll 1
    for (int piece = 0; piece < pieces; ++piece) {
        if (pieces > 1) load(piece);
        const int from = from_of(piece);
        uint32_t more = 0, same = 0;
#pragma unroll
        for (int k = 0; k < HELD; ++k) {
            if (k >= rows || from + 64 * k >= old) break;
            const bool in = from + 64 * k + lane < old;
            more += __popcll(__ballot(in && key[k] > prefix));
            same += __popcll(__ballot(in && key[k] == prefix));
        }
        if (piece > 0) __syncthreads();
        if (lane == 0) above[wave] = more, equal[wave] = same;
        __syncthreads();
        uint32_t here = at, tied = ties;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) {
            if (i < wave) here += above[i], tied += equal[i];
            at += above[i], ties += equal[i];
        }
        uint32_t place = here + (tied < need ? tied : need);
#pragma unroll
        for (int k = 0; k < HELD; ++k) {
            if (k >= rows || from + 64 * k >= old) break;
            const bool in = from + 64 * k + lane < old;
            const uint64_t eq = __ballot(in && key[k] == prefix);
            const bool stay = in && (key[k] > prefix || (key[k] == prefix && tied + __popcll(eq & lower) < need));
            const uint64_t all = __ballot(stay);
            if (stay) kept[place + __popcll(all & lower)] = from + 64 * k + lane;
            place += __popcll(all);
            tied += __popcll(eq);
        }
    }
}

// The same for long sequences, a part of PART positions to a workgroup and a launch to a digit.  A launch first finds the digit
// before it from all parts' counts (each workgroup for itself: they lie in L2), then counts its own part; the last one writes the
// positions, behind those of the parts before.  Of a (sequence, head), in `counts`: per part the counts of the three digits and
// how many of it lie above the first two, and what was found.  2 x 8 rows of 131072: 4.2, 7.4, 7.5 and 7.8 us, of which a launch
// is about 3 and the sums over the parts' counts 3 (24 MB from L2); by one workgroup a row 182.
constexpr int PART = 8 * SEL;
constexpr int COUNTS = 2048 + 2048 + 1024 + 2;
struct Found {
    uint32_t prefix, need;
};
__host__ __device__ __forceinline__ constexpr int64_t counts_of_pair(int parts) { return (int64_t)parts * COUNTS + 4; }

template <int DIGIT>  // 0, 1, 2; 3: write the positions
__global__ __launch_bounds__(SEL) void kv_select_part_kernel(KvEvictArgs a)
{
    __shared__ uint32_t hist[2048];
    __shared__ uint32_t sums[WAVES], pick[2], sides[2][WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int part = (int)(blockIdx.x % a.parts);
    const int64_t pair = blockIdx.x / a.parts;  // of this launch
    const int h = (int)(pair % a.c.kv_heads);
    const int64_t b = a.first + pair / a.c.kv_heads;
    const int64_t most = (int64_t)a.s.table_pages << a.c.page_shift;
    int64_t len64 = a.s.lengths[b];
    len64 = len64 < 0 ? 0 : len64 > most ? most : len64;
    const int len = (int)len64;
    const int n = len < a.keep ? len : a.keep;
    int* kept = a.kept + (b * a.c.kv_heads + h) * (int64_t)a.keep;
    const int old = len - a.recent;  // (recent <= keep)
    if (DIGIT == 0) {
        // what needs no choice
        if (h == 0 && tid == 0 && part == 0) a.lengths_out[b] = n;
        const int chosen = len <= a.keep ? 0 : a.keep - a.recent;
        for (int i = chosen + part * SEL + tid; i < a.keep; i += a.parts * SEL)
            kept[i] = i >= n ? -1 : len <= a.keep ? i : old + (i - chosen);
    }
    if (len <= a.keep || a.keep == a.recent) return;
    const int parts = (old + PART - 1) / PART;  // (at most a.parts)
    if (part >= parts) return;
    uint32_t* const all = a.counts + pair * counts_of_pair(a.parts);
    uint32_t* const own = all + (int64_t)part * COUNTS;
    Found* const found = (Found*)(all + (int64_t)a.parts * COUNTS);  // after digit 0 and 1

    // the part's keys: wave by wave 512 neighbouring positions
    const float* w = a.weights + (b * a.c.kv_heads + h) * a.cap;
    const int from = part * PART + wave * 512;
    float x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const int i = from + 64 * k + lane;
        x[k] = w[i < old ? i : old - 1];
    }
    Found f{0, (uint32_t)(a.keep - a.recent)};
    uint32_t mask = 0;
    // of a thread's two bins, this part's counts (the last launch: those of the parts before), and its share of what lies above
    uint32_t m0 = 0, m1 = 0, more = 0, same = 0;
    if constexpr (DIGIT > 0) {
        constexpr int LAST = DIGIT - 1;
        constexpr uint32_t bins = bins_of(LAST);
        if (DIGIT > 1) f = found[LAST - 1];
        const uint32_t top = bins - 1 - 2 * tid;
        const bool counts = 2 * tid < (int)bins;
        uint32_t c0 = 0, c1 = 0;
        if (counts) {
#pragma unroll 16
            for (int p = 0; p < parts; ++p) {
                const u32x2 c = *(const u32x2*)(all + (int64_t)p * COUNTS + 2048 * LAST + top - 1);
                c0 += c[1], c1 += c[0];
                const bool of_part = DIGIT < 3 ? p == part : p < part;
                m0 += of_part ? c[1] : 0, m1 += of_part ? c[0] : 0;
            }
        } else if (DIGIT == 3 && wave == WAVES - 1) {  // (above the first two digits; this wave has no bins of the third)
            for (int p = lane >> 1; p < part; p += 32) more += all[(int64_t)p * COUNTS + 5120 + (lane & 1)];
        }
        pick_bin(c0, c1, bins, f.need, sums, pick);
        f.prefix |= pick[0] << shift_of(LAST);
        f.need = pick[1];
        mask = ~((1u << shift_of(LAST)) - 1);
        if constexpr (DIGIT < 3) {
            // how many of this part lie above
            more = (top > pick[0] ? m0 : 0) + (top - 1 > pick[0] ? m1 : 0);
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) more += __shfl_xor(more, off, 64);
            if (lane == 0) sides[0][wave] = more;
            __syncthreads();
            if (tid == 0) {
                uint32_t sum = 0;
#pragma unroll
                for (int i = 0; i < WAVES; ++i) sum += sides[0][i];
                own[5120 + LAST] = sum;
                if (part == 0) found[LAST] = f;
            }
        }
    }
    uint32_t key[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) key[k] = order_key(x[k]);
    if constexpr (DIGIT < 3) {
        constexpr int shift = shift_of(DIGIT);
        constexpr uint32_t bins = bins_of(DIGIT), ZERO = 0x80000000u;
        hist[tid] = hist[tid + SEL] = 0;
        __syncthreads();
        uint32_t zeros = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const bool in = from + 64 * k + lane < old && (key[k] & mask) == f.prefix;
            zeros += __popcll(__ballot(in && key[k] == ZERO));
            if (in && key[k] != ZERO) atomicAdd(&hist[(key[k] >> shift) & (bins - 1)], 1u);
        }
        if (lane == 0 && zeros) atomicAdd(&hist[(ZERO >> shift) & (bins - 1)], zeros);
        __syncthreads();
        if (2 * tid < (int)bins) *(u32x2*)(own + 2048 * DIGIT + 2 * tid) = (u32x2){hist[2 * tid], hist[2 * tid + 1]};
    } else {
        // places before this part: above the threshold, and equal to it
        const uint32_t top = bins_of(2) - 1 - 2 * tid;
        more += (top > pick[0] ? m0 : 0) + (top - 1 > pick[0] ? m1 : 0);
        same = top == pick[0] ? m0 : top - 1 == pick[0] ? m1 : 0;
        uint32_t here = 0, equal = 0;  // of this wave
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const bool in = from + 64 * k + lane < old;
            here += __popcll(__ballot(in && key[k] > f.prefix));
            equal += __popcll(__ballot(in && key[k] == f.prefix));
        }
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            more += __shfl_xor(more, off, 64);
            same += __shfl_xor(same, off, 64);
        }
        __shared__ uint32_t before[2][WAVES];
        if (lane == 0) before[0][wave] = more, before[1][wave] = same, sides[0][wave] = here, sides[1][wave] = equal;
        __syncthreads();
        uint32_t place = 0, tied = 0;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) {
            place += before[0][i], tied += before[1][i];
            if (i < wave) place += sides[0][i], tied += sides[1][i];
        }
        place += tied < f.need ? tied : f.need;
        const uint64_t lower = ((uint64_t)1 << lane) - 1;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const bool in = from + 64 * k + lane < old;
            const uint64_t eq = __ballot(in && key[k] == f.prefix);
            const bool stay = in && (key[k] > f.prefix || (key[k] == f.prefix && tied + __popcll(eq & lower) < f.need));
            const uint64_t set = __ballot(stay);
            if (stay) kept[place + __popcll(set & lower)] = from + 64 * k + lane;
            place += __popcll(set);
            tied += __popcll(eq);
        }
    }
}

// the page of token t of a sequence, or -1
__device__ __forceinline__ int page_of(const int* table, int pages_of_row, int t, const KvCacheArgs& c)
{
    const int col = t >> c.page_shift;
    if (col >= pages_of_row) return -1;
    const int p = table[col];
    return p >= 0 && p < c.pages ? p : -1;
}

// every thread's loads have returned before any thread goes on
__device__ __forceinline__ void reads_done()
{
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

// N words of W-word pieces of `TOKENS` tokens' rows: read all, then write all
template <int W, int N>
struct Rows {
    typedef uint32_t piece __attribute__((ext_vector_type(W)));
    piece x[N];
    template <int THREADS>
    __device__ __forceinline__ void read(const uint32_t* pool, int64_t ld, int words, int h, const KvCacheArgs& c, const int2* src)
    {
        const int per = words / W;  // pieces of a row
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int i = u * THREADS + threadIdx.x, token = i / per, p = i % per;
            const int2 at = src[token];
            x[u] = at.x < 0 ? piece{}
                            : ((const piece*)(pool + at.x * ld + (((int64_t)h << c.page_shift) + at.y) * words))[p];
        }
    }
    template <int THREADS>
    __device__ __forceinline__ void write(uint32_t* pool, int64_t ld, int words, int h, const KvCacheArgs& c, const int2* dst) const
    {
        const int per = words / W;
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int i = u * THREADS + threadIdx.x, token = i / per, p = i % per;
            const int2 at = dst[token];
            if (at.x >= 0) ((piece*)(pool + at.x * ld + (((int64_t)h << c.page_shift) + at.y) * words))[p] = x[u];
        }
    }
};

// Moves the kept tokens of a (sequence, head) to its first places, in order, THREADS tokens at a time: their pages are looked up once,
// then all their rows are read before any is written.  To other pages nothing is in the way, and the runs of tokens are shared by
// gridDim.x workgroups.  In place one workgroup takes the tokens of a plane (keys, values, scales, weights: gridDim.z) in order: the
// token of place i comes from a position >= i, so that a run's reads lie behind all earlier runs' writes.
// Bound by rows of 64 and 16 bytes read from anywhere: 2 sequences x 8 heads, 16384 kept of 131072, d 128: 28 us for 42 MB kept
// (108 MB read in whole lines, 48 written: 5.6 TB/s); 16 sequences of up to 4096 cut to 2048 15 us (40 MB read, 33 written).  In place
// the first takes 52 us (16 runs of 1024 tokens one behind the other, on 64 workgroups), the second 12: what keeps its place is not
// written.
template <int D, int G, int THREADS>
__global__ __launch_bounds__(THREADS) void kv_move_kernel(KvEvictArgs a)
{
    constexpr int WORDS = D / 8, GROUPS = D / G, SW = GROUPS < 4 ? GROUPS : 4;
    __shared__ int2 src[THREADS], dst[THREADS];  // page and row there; -1: none
    const int h = (int)(blockIdx.y % a.c.kv_heads);
    const int64_t b = a.first + blockIdx.y / a.c.kv_heads;
    const int n = a.lengths_out[b];
    const int plane = gridDim.z == 1 ? -1 : (int)blockIdx.z;  // (-1: all)
    const int* kept = a.kept + (b * a.c.kv_heads + h) * (int64_t)a.keep;
    const int* from = a.s.table + b * a.s.ld_table;
    const bool away = a.into != nullptr;
    const int* to = away ? a.into + b * a.ld_into : from;
    const int to_pages = away ? a.into_pages : a.s.table_pages, mask = (1 << a.c.page_shift) - 1;
    const int tid = threadIdx.x;
    const float* w = a.weights + (b * a.c.kv_heads + h) * a.cap;
    float* out = a.weights_out + (b * a.c.kv_heads + h) * a.cap_out;
    const bool apart = a.weights != a.weights_out;  // (weights in place go in one run of workgroups, by a plane of their own)
    if (plane == 3 || (plane < 0 && apart)) {
        // the weights: gathered to the front, zeros behind
        for (int64_t base = (int64_t)blockIdx.x * THREADS; base < a.cap_out; base += (int64_t)gridDim.x * THREADS) {
            const int64_t i = base + tid;
            const float x = i < n ? w[kept[i]] : 0.0f;
            if (!apart) reads_done();
            if (i < a.cap_out) out[i] = x;
        }
        if (plane == 3) return;
    }
    for (int base = blockIdx.x * THREADS; base < n; base += gridDim.x * THREADS) {
        const int i = base + tid;
        int2 s = {-1, 0}, d = {-1, 0};
        if (i < n) {
            const int t = kept[i];
            s = {page_of(from, a.s.table_pages, t, a.c), t & mask};
            if (away || t != i) d = {page_of(to, to_pages, i, a.c), i & mask};
        }
        src[tid] = s;
        dst[tid] = d;
        __syncthreads();
        Rows<4, WORDS / 4> k, v;
        Rows<SW, GROUPS / SW> ks, vs;
        if (plane < 0 || plane == 0) k.template read<THREADS>((uint32_t*)a.c.k, a.c.ld_code / 4, WORDS, h, a.c, src);
        if (plane < 0 || plane == 1) v.template read<THREADS>((uint32_t*)a.c.v, a.c.ld_code / 4, WORDS, h, a.c, src);
        if (plane < 0 || plane == 2) {
            ks.template read<THREADS>(a.c.k_scale, a.c.ld_scale, GROUPS, h, a.c, src);
            vs.template read<THREADS>(a.c.v_scale, a.c.ld_scale, GROUPS, h, a.c, src);
        }
        if (!away) reads_done();
        if (plane < 0 || plane == 0) k.template write<THREADS>((uint32_t*)a.c.k, a.c.ld_code / 4, WORDS, h, a.c, dst);
        if (plane < 0 || plane == 1) v.template write<THREADS>((uint32_t*)a.c.v, a.c.ld_code / 4, WORDS, h, a.c, dst);
        if (plane < 0 || plane == 2) {
            ks.template write<THREADS>(a.c.k_scale, a.c.ld_scale, GROUPS, h, a.c, dst);
            vs.template write<THREADS>(a.c.v_scale, a.c.ld_scale, GROUPS, h, a.c, dst);
        }
        __syncthreads();
    }
}

// the weights alone, in place, while the rows went elsewhere
__global__ __launch_bounds__(SEL) void kv_move_weights_kernel(KvEvictArgs a)
{
    const int64_t row = a.first * a.c.kv_heads + blockIdx.x;
    const int n = a.lengths_out[row / a.c.kv_heads];
    const int* kept = a.kept + row * (int64_t)a.keep;
    float* w = a.weights_out + row * a.cap_out;
    for (int64_t base = 0; base < a.cap_out; base += SEL) {
        const int64_t i = base + threadIdx.x;
        const float x = i < n ? w[kept[i]] : 0.0f;
        reads_done();
        if (i < a.cap_out) w[i] = x;
    }
}

template <int D, int G>
void move(const KvEvictArgs& a, int64_t n, hipStream_t st)
{
    const uint32_t rows = (uint32_t)(n * a.c.kv_heads);
    if (!a.into) {
        hipLaunchKernelGGL(HIP_KERNEL_NAME(kv_move_kernel<D, G, 1024>), dim3(1, rows, 4), dim3(1024), 0, st, a);
        return;
    }
    const int64_t runs = ((int64_t)a.keep + 255) / 256;
    hipLaunchKernelGGL(HIP_KERNEL_NAME(kv_move_kernel<D, G, 256>), dim3((uint32_t)(runs < 64 ? runs : 64), rows), dim3(256), 0, st, a);
    if (a.weights == a.weights_out) hipLaunchKernelGGL(kv_move_weights_kernel, dim3(rows), dim3(SEL), 0, st, a);
}

}  // namespace

namespace {
// parts of a selection: one up to 16 SEL positions (us a launch, 128 rows of 4096 12, and 16 of 131072 by one workgroup each 182), and
// where the parts of one sequence are more than a launch has room for (2^34 tokens over all key heads)
constexpr int64_t PARTS = (int64_t)1 << 21;
int parts_of(const KvEvictArgs& a)
{
    const int64_t cap = (int64_t)a.s.table_pages << a.c.page_shift, parts = (cap + PART - 1) / PART;
    return cap <= 16 * SEL || parts * a.c.kv_heads > PARTS ? 1 : (int)parts;
}
// sequences of a launch: fewer than 2^16 rows of workgroups, and than 2^32 threads (64 x 256 or 4 x 1024 a row, SEL a part)
int64_t sequences_of(const KvEvictArgs& a, int parts)
{
    const int64_t most = 65535 / a.c.kv_heads, rows = PARTS / parts / a.c.kv_heads;
    return most < rows ? most : rows;
}
}  // namespace

size_t kv_evict_ws_bytes(const KvEvictArgs& a)
{
    const int parts = parts_of(a);
    const int64_t most = sequences_of(a, parts);
    return parts < 2 ? 0 : (size_t)((a.s.batch < most ? a.s.batch : most) * a.c.kv_heads * counts_of_pair(parts)) * sizeof(uint32_t);
}

hipError_t launch_kv_evict(KvEvictArgs a, void* ws, size_t ws_bytes, hipStream_t st)
{
    a.parts = ws && ws_bytes >= kv_evict_ws_bytes(a) ? parts_of(a) : 1;
    a.counts = (uint32_t*)ws;
    const int64_t most = sequences_of(a, a.parts);
    for (a.first = 0; a.first < a.s.batch; a.first += most) {
        const int64_t n = a.s.batch - a.first < most ? a.s.batch - a.first : most;
        const dim3 grid((uint32_t)(n * a.c.kv_heads * a.parts));
        if (a.parts > 1) {
            launch_k(kv_select_part_kernel<0>, grid, dim3(SEL), 0, st, a);
            hipLaunchKernelGGL(kv_select_part_kernel<1>, grid, dim3(SEL), 0, st, a);
            hipLaunchKernelGGL(kv_select_part_kernel<2>, grid, dim3(SEL), 0, st, a);
            hipLaunchKernelGGL(kv_select_part_kernel<3>, grid, dim3(SEL), 0, st, a);
        } else if ((int64_t)a.s.table_pages << a.c.page_shift <= 4 * SEL) {
            launch_k(kv_select_kernel<4>, grid, dim3(SEL), 0, st, a);
        } else {
            launch_k(kv_select_kernel<16>, grid, dim3(SEL), 0, st, a);
        }
        hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        switch (a.c.d * 256 + a.c.group) {
        case 64 * 256 + 32: move<64, 32>(a, n, st); break;
        case 64 * 256 + 64: move<64, 64>(a, n, st); break;
        case 128 * 256 + 32: move<128, 32>(a, n, st); break;
        case 128 * 256 + 64: move<128, 64>(a, n, st); break;
        case 128 * 256 + 128: move<128, 128>(a, n, st); break;
        case 256 * 256 + 32: move<256, 32>(a, n, st); break;
        case 256 * 256 + 64: move<256, 64>(a, n, st); break;
        default: move<256, 128>(a, n, st); break;
        }
        e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace ascq
