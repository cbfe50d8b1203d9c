// kv_attention.hip -- attention over the paged int4 key / value cache, and the weight each cached token received.
//
// A tile is 16 rows -- (query, head of a key head's group) pairs -- against tokens in steps of 32.  A wave computes
// S^T = K Q^T with v_mfma_f32_16x16x32_f16, so that a lane's scores belong to one row (its column l & 15) and to the tokens
// 4 (l >> 4) .. + 3 of both halves of the step.  That is the layout in which O^T = V^T P^T takes P as it is: the token order
// inside a step is free as long as V's fragments follow it.  No score crosses lanes but the running maximum, and the maximum
// moves (and O is rescaled) only when a score passes it by 2^15.
//
// Codes become f16 values in registers, value(c) = fma(c, scale, offset) rounded once: exactly what the cache stands for.
// Nibbles are masked under the exponent of 1024 -- bits 0-3 give 1024 + u, bits 4-7 1024 + 16 u, u = c + 8 -- and one exact
// operation takes them to c.  K's words hold 8 channels of a token, whose order inside a product is free again (Q follows).
// V's hold 8 channels of a token where a fragment wants 8 tokens of a channel: one v_perm_b32 pairs the halves of two tokens'
// words, and the same masks then give pairs of tokens.
//
// Scores are fp32 sums of exact f16 products.  Queries are scaled by a power of two per row, the largest into [2^14, 2^15): exact for
// what lies within 2^31 (bf16) or 2^28 (f16) of it, off by 2^-39 of it at most below.  P is rounded to f16 after exp2, as the matrix
// instruction takes it: by 2^-11 of a weight at most, or, where f16 has no smaller step, 2^-33 of the row's largest.  Sums and
// statistics are fp32, of the unrounded weights.
#include "gemm_core.h"

#include <type_traits>

namespace ascq {

namespace {

typedef u32x4 u32x4_any __attribute__((aligned(2)));

// Tables that a kernel reads and nobody writes meanwhile, so that their uniform loads go through the scalar cache whatever is
// stored in between: as vector loads they would wait for all loads before them.
typedef const int __attribute__((address_space(4))) * Table;
__device__ __forceinline__ Table table_of(const int* p) { return (Table)(uintptr_t)p; }

struct View {
    int start, rows, n, len;  // first row of q; queries computed; queries there are; tokens
};
__device__ __forceinline__ View view_of(const KvAttentionArgs& a, int64_t b)
{
    View v;
    int64_t start = b, n = 1;
    if (a.s.starts) {
        start = table_of(a.s.starts)[b];
        n = (int64_t)table_of(a.s.starts)[b + 1] - start;
    }
    if (start < 0 || start > a.T || n < 0) start = 0, n = 0;
    int64_t rows = n < a.max_q ? n : a.max_q;
    if (rows > (int64_t)a.T - start) rows = (int64_t)a.T - start;
    v.start = (int)start;
    v.rows = (int)rows;
    v.n = (int)n;
    const int64_t most = (int64_t)a.s.table_pages << a.c.page_shift;
    const int64_t len = table_of(a.s.lengths)[b];
    v.len = (int)(len < 0 ? 0 : len > most ? most : len);
    return v;
}

// the tokens [low, hi) that the rows of a tile see together, and where their first step begins (at most 31 tokens before); a row's own
// limits follow from its query
struct Range {
    int lo, hi, low;
};
__device__ __forceinline__ Range range_of(const KvAttentionArgs& a, const View& v, int tile)
{
    const int first = tile * a.tile_rows / a.ratio;
    int last = (tile * a.tile_rows + a.tile_rows - 1) / a.ratio;
    last = last < v.rows ? last : v.rows - 1;
    Range r{0, v.len, 0};
    const int64_t at = (int64_t)v.len - v.n;  // the first query's token
    if (a.causal) {
        const int64_t hi = at + last + 1;
        r.hi = hi < 0 ? 0 : hi < v.len ? (int)hi : v.len;
    }
    if (a.window) {
        const int64_t lo = at + first - a.window + 1;
        r.low = lo < 0 ? 0 : lo < v.len ? (int)lo : v.len;
        r.lo = r.low < v.len ? r.low & ~31 : v.len;
    }
    return r;
}

// where 16 tokens of a sequence lie: their rows in the pools of one key head, and whether there is such a page
struct Half {
    int64_t code, scale;  // bytes, words
    bool ok;
};
__device__ __forceinline__ int page_at(const KvAttentionArgs& a, Table table, int token)
{
    // (called for sequences of tokens alone, whose table has columns; a load without a branch around it)
    const int col = token >> a.c.page_shift, last = a.s.table_pages - 1;
    const int page = table[col < last ? col : last];
    return col <= last ? page : -1;
}
__device__ __forceinline__ Half half_at(const KvAttentionArgs& a, int page, int h, int token)
{
    Half r;
    r.ok = page >= 0 && page < a.c.pages;
    const int64_t p = r.ok ? page : 0;
    const int row = (h << a.c.page_shift) + (token & ((1 << a.c.page_shift) - 1));
    r.code = p * a.c.ld_code + (int64_t)row * (a.c.d / 2);
    r.scale = p * a.c.ld_scale + (int64_t)row * (a.c.d / a.c.group);
    return r;
}

constexpr uint32_t NIB0 = 0x000F000Fu, NIB1 = 0x00F000F0u, MAGIC0 = 0x64086408u, MAGIC1 = 0x64806480u;
// the codes c of the nibbles at bits 0-3 (HIGH 0) or 4-7 (HIGH 1) of both halves of x, as two f16
template <int HIGH>
__device__ __forceinline__ h2 codes_of(uint32_t x)
{
    if constexpr (HIGH) {
        const h2 u = __builtin_bit_cast(h2, (x & NIB1) ^ MAGIC1);  // 1024 + 16 (c + 8)
        return __builtin_elementwise_fma(u, (h2){(_Float16)0.0625f, (_Float16)0.0625f},
                                         (h2){(_Float16)-72.0f, (_Float16)-72.0f});
    } else {
        const h2 u = __builtin_bit_cast(h2, (x & NIB0) ^ MAGIC0);  // 1024 + (c + 8)
        return u - (h2){(_Float16)1032.0f, (_Float16)1032.0f};
    }
}
__device__ __forceinline__ h2 low_pair(uint32_t a, uint32_t b)  // the low halves of a and b
{
    return __builtin_bit_cast(h2, __builtin_amdgcn_perm(b, a, 0x05040100u));
}
__device__ __forceinline__ h2 high_pair(uint32_t a, uint32_t b)
{
    return __builtin_bit_cast(h2, __builtin_amdgcn_perm(b, a, 0x07060302u));
}

// a word of K (8 channels of a token) as a fragment; channels in the order 0 4 1 5 2 6 3 7
__device__ __forceinline__ h8 key_fragment(uint32_t w, h2 s, h2 o)
{
    const uint32_t w8 = w >> 8;
    h8 f;
    f.s01 = __builtin_elementwise_fma(codes_of<0>(w), s, o);
    f.s23 = __builtin_elementwise_fma(codes_of<1>(w), s, o);
    f.s45 = __builtin_elementwise_fma(codes_of<0>(w8), s, o);
    f.s67 = __builtin_elementwise_fma(codes_of<1>(w8), s, o);
    return f;
}

template <int D>
struct Shape {
    static constexpr int STEPS = D / 32;           // products of 32 channels
    static constexpr int TILES = D / 16;           // tiles of 16 channels of O
    static constexpr int KW = D / 32;              // words of K of a lane per token
    static constexpr int VW = D == 256 ? 2 : 1;    // words of V of a lane per token (D = 64: half of one)
    static constexpr int MD = D < 128 ? D : 128;   // channels merged at a time
};

// the codes and scales of a step of 32 tokens, as the lanes of a wave need them
template <int D, int G>
struct Step {
    static constexpr int KS = D / 4 > G ? D / 4 / G : 1;  // groups of K of a lane
    uint32_t k[2][Shape<D>::KW], ks[2][KS], v[8][Shape<D>::VW], vs[8];
};

// Where a lane's parts begin, in bytes behind the row of 16 tokens that a scalar address gives
struct Lane {
    uint32_t k, ks, v, vs;
};
template <class T>
__device__ __forceinline__ T read(const void* row, uint32_t lane, int words = 0)
{
    return *(const T*)((const uint8_t*)row + lane + 4 * words);
}

template <int D, int G>
__device__ __forceinline__ void load_keys(Step<D, G>& x, const KvAttentionArgs& a, const Half (&half)[2], const Lane& at)
{
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint8_t* k = a.c.k + half[h].code;
        const uint32_t* ks = a.c.k_scale + half[h].scale;
        if constexpr (Shape<D>::KW == 2) {
            const u32x2 t = read<u32x2>(k, at.k);
            x.k[h][0] = t[0], x.k[h][1] = t[1];
        } else {
#pragma unroll
            for (int i = 0; i < Shape<D>::KW; i += 4) {
                const u32x4 t = read<u32x4>(k, at.k, i);
#pragma unroll
                for (int e = 0; e < 4; ++e) x.k[h][i + e] = t[e];
            }
        }
#pragma unroll
        for (int i = 0; i < Step<D, G>::KS; ++i) x.ks[h][i] = read<uint32_t>(ks, at.ks, i);
    }
}
template <int D, int G>
__device__ __forceinline__ void load_values(Step<D, G>& x, const KvAttentionArgs& a, const Half (&half)[2], const Lane& at)
{
    constexpr int W = D / 8, GR = D / G;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint8_t* v = a.c.v + half[h].code;
        const uint32_t* vs = a.c.v_scale + half[h].scale;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (Shape<D>::VW == 2) {
                const u32x2 t = read<u32x2>(v, at.v, i * W);
                x.v[4 * h + i][0] = t[0], x.v[4 * h + i][1] = t[1];
            } else {
                x.v[4 * h + i][0] = read<uint32_t>(v, at.v, i * W);
            }
            x.vs[4 * h + i] = read<uint32_t>(vs, at.vs, i * GR);
        }
    }
}
template <int D, int G>
__device__ __forceinline__ Lane lane_of_step(int r, int j)
{
    constexpr int W = D / 8, GR = D / G;
    return Lane{4u * (r * W + j * (W / 4)), 4u * (r * GR + j * (D / 4) / G),
                4u * (4 * j * W + (D == 64 ? r >> 1 : r * Shape<D>::VW)), 4u * (4 * j * GR + r * (D / 16) / G)};
}

// the scores of NQ times 16 rows against 32 tokens: s[c][h][i] is row 16 c + r, token 16 h + 4 j + i
template <int D, int G, int NQ>
__device__ __forceinline__ void scores(v4f (&s)[NQ][2], const uint32_t (&k)[2][Shape<D>::KW],
                                       const uint32_t (&ks)[2][Step<D, G>::KS], const h8 (&q)[NQ][Shape<D>::STEPS])
{
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int c = 0; c < NQ; ++c) s[c][h] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < Shape<D>::STEPS; ++i) {
            const uint32_t w = ks[h][i * Step<D, G>::KS / Shape<D>::STEPS];
            const h8 f = key_fragment(k[h][i], low_pair(w, w), high_pair(w, w));
#pragma unroll
            for (int c = 0; c < NQ; ++c) s[c][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, q[c][i], s[c][h], 0, 0, 0);
        }
    }
}

// O^T += V^T P^T of 32 tokens: tile n's rows are the channels r (D / 16) + n
template <int D, int G, int NQ>
__device__ __forceinline__ void add_values(v4f (&acc)[NQ][Shape<D>::TILES], const Step<D, G>& x, const h8 (&p)[NQ], int r)
{
    h2 s[4], o[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        s[u] = low_pair(x.vs[2 * u], x.vs[2 * u + 1]);
        o[u] = high_pair(x.vs[2 * u], x.vs[2 * u + 1]);
    }
#pragma unroll
    for (int w = 0; w < Shape<D>::VW; ++w) {
        constexpr int HALVES = D == 64 ? 1 : 2;
#pragma unroll
        for (int half = 0; half < HALVES; ++half) {
            h8 f[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const uint32_t sel = D == 64 ? (r & 1 ? 0x07060302u : 0x05040100u) : half ? 0x07060302u : 0x05040100u;
                const uint32_t y = __builtin_amdgcn_perm(x.v[2 * u + 1][w], x.v[2 * u][w], sel);  // a pair of tokens: 4 channels each
                const uint32_t y8 = y >> 8;
                const h2 c0 = __builtin_elementwise_fma(codes_of<0>(y), s[u], o[u]);
                const h2 c1 = __builtin_elementwise_fma(codes_of<1>(y), s[u], o[u]);
                const h2 c2 = __builtin_elementwise_fma(codes_of<0>(y8), s[u], o[u]);
                const h2 c3 = __builtin_elementwise_fma(codes_of<1>(y8), s[u], o[u]);
                f[0][2 * u] = c0[0], f[0][2 * u + 1] = c0[1];
                f[1][2 * u] = c1[0], f[1][2 * u + 1] = c1[1];
                f[2][2 * u] = c2[0], f[2][2 * u + 1] = c2[1];
                f[3][2 * u] = c3[0], f[3][2 * u + 1] = c3[1];
            }
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int c = 0; c < NQ; ++c) {
                    v4f& t = acc[c][w * 8 + half * 4 + n];
                    t = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[n], p[c], t, 0, 0, 0);
                }
        }
    }
}

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// Row r of a tile as fragments (8 channels of lane j's quarter a step, in K's order), scaled by a power of two that brings its
// largest magnitude to [2^14, 2^15): f16's rounding is then off by 2^-39 of it at most, and by nothing in what is not far below.  The scale's
// sign goes into the row too, so that what is returned -- a score to base 2 is that times the product -- is positive, never 0
// or infinite, and masked products of -inf stay that.  Rows that are not there are zeros.
template <int D>
__device__ __forceinline__ float load_row(h8 (&q)[Shape<D>::STEPS], const uint16_t* row, bool there, bool bf16, int j, float scale)
{
    u32x4 raw[Shape<D>::STEPS];
    us2_t most = {0, 0};  // magnitudes order as their bits do, NaN above all
#pragma unroll
    for (int i = 0; i < Shape<D>::STEPS; ++i) {
        raw[i] = there ? *(const u32x4_any*)(row + j * (D / 4) + 8 * i) : (u32x4){0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 4; ++e) most = __builtin_elementwise_max(most, __builtin_bit_cast(us2_t, raw[i][e] & 0x7fff7fffu));
    }
    uint32_t bits = most[0] > most[1] ? most[0] : most[1];
    const uint32_t b16 = __shfl_xor(bits, 16, 64);
    bits = bits > b16 ? bits : b16;
    const uint32_t b32 = __shfl_xor(bits, 32, 64);
    bits = bits > b32 ? bits : b32;
    const float top = bf16 ? bf16_to_f32((uint16_t)bits) : f16_to_f32((uint16_t)bits);
    int e = (int)(__float_as_uint(top) >> 23) - 127;
    e = e < -100 ? -100 : e > 127 ? 14 : e;  // (0 and tiny rows; infinite ones pass as they are)
    float up = __uint_as_float((uint32_t)(127 + 14 - e) << 23);
    up = scale > 0.0f ? up : scale < 0.0f ? -up : 0.0f;
#pragma unroll
    for (int i = 0; i < Shape<D>::STEPS; ++i) {
        float x[8];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const uint16_t lo = (uint16_t)raw[i][c], hi = (uint16_t)(raw[i][c] >> 16);
            x[2 * c] = (bf16 ? bf16_to_f32(lo) : f16_to_f32(lo)) * up;
            x[2 * c + 1] = (bf16 ? bf16_to_f32(hi) : f16_to_f32(hi)) * up;
        }
        const h8 f = {(_Float16)x[0], (_Float16)x[4], (_Float16)x[1], (_Float16)x[5],
                      (_Float16)x[2], (_Float16)x[6], (_Float16)x[3], (_Float16)x[7]};
        q[i] = f;
    }
    const float undo = __uint_as_float((uint32_t)(127 - 14 + e) << 23) * (__builtin_fabsf(scale) * LOG2E);
    return __builtin_fminf(__builtin_fmaxf(undo, 0x1p-126f), 0x1p127f);
}

constexpr float MARGIN = 15.0f, BELOW = 8.0f;  // a weight is exp2(score - reference), 2^8 at the maximum, 2^15 at most

// where the splits of a row leave their sums: d of O, the reference, the sum of weights, for each
template <int D>
__device__ __forceinline__ float* part_of(const KvAttentionArgs& a, int64_t b, int tile, int h, int row)
{
    const int64_t all = (int64_t)a.max_q * a.ratio;
    const int rows = (int)(all < a.tile_rows ? all : a.tile_rows);
    return a.part + ((((b - a.first) * a.tiles + tile) * a.c.kv_heads + h) * (int64_t)rows + row) * a.splits * (D + 2);
}

__device__ __forceinline__ void store8(uint16_t* to, const float (&o)[8], float by, bool bf16)
{
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float lo = o[2 * e] * by, hi = o[2 * e + 1] * by;
        if (bf16) w[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f2_t){lo, hi}, bf2_t));
        else w[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f2_t){lo, hi}, h2_t));
    }
    *(u32x4_any*)to = w;
}

// What a lane knows of the row it scores: its tokens [low, limit), what undoes the scaling of its query, the softmax's reference
// (none yet: -inf), what is subtracted for it, and the sum of its weights.
struct Row {
    int low, limit;
    float undo, ref, base, sum;
};

// the tokens that query `query` of a sequence sees
__device__ __forceinline__ void sees(const KvAttentionArgs& a, const View& v, int query, int& low, int& limit)
{
    const int64_t at = (int64_t)v.len - v.n + query;
    limit = a.causal ? (at + 1 < 0 ? 0 : at + 1 < v.len ? (int)(at + 1) : v.len) : v.len;
    low = a.window ? (at - a.window + 1 < 0 ? 0 : at - a.window + 1 < v.len ? (int)(at - a.window + 1) : v.len) : 0;
}

// scores -> weights (f16) of the tokens t .. t + 31 below `end`; `edge`: some row does not see some of them;
// `meanwhile` is work that the weights do not depend on
template <int NQ, int TILES, class F>
__device__ __forceinline__ void weigh(h8 (&p)[NQ], v4f (&s)[NQ][2], Row (&row)[NQ], v4f (&acc)[NQ][TILES], bool edge, int t, int end,
                                      bool ok0, bool ok1, int j, F meanwhile)
{
    if (edge) {
#pragma unroll
        for (int c = 0; c < NQ; ++c)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int token = t + (e >> 2) * 16 + 4 * j + (e & 3);
                const bool seen = token >= row[c].low && token < row[c].limit && token < end && (e < 4 ? ok0 : ok1);
                s[c][e >> 2][e & 3] = seen ? s[c][e >> 2][e & 3] : -__builtin_inff();
            }
    }
    float top[NQ];
    bool moves = false;
#pragma unroll
    for (int c = 0; c < NQ; ++c) {
        top[c] = s[c][0][0];
#pragma unroll
        for (int e = 1; e < 8; ++e) top[c] = __builtin_fmaxf(top[c], s[c][e >> 2][e & 3]);
        top[c] *= row[c].undo;
        moves |= top[c] > row[c].ref + MARGIN;
    }
    if (__ballot(moves)) {
#pragma unroll
        for (int c = 0; c < NQ; ++c) {
            top[c] = __builtin_fmaxf(top[c], __shfl_xor(top[c], 16, 64));
            top[c] = __builtin_fmaxf(top[c], __shfl_xor(top[c], 32, 64));
            const float to = __builtin_fmaxf(row[c].ref, top[c] - BELOW);
            const float f = to == row[c].ref ? 1.0f : __builtin_amdgcn_exp2f(row[c].ref - to);
            row[c].sum *= f;
#pragma unroll
            for (int n = 0; n < TILES; ++n) acc[c][n] *= f;
            row[c].ref = to;
            row[c].base = to == -__builtin_inff() ? 0.0f : to;
        }
    }
    meanwhile();
#pragma unroll
    for (int c = 0; c < NQ; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[c][e >> 2][e & 3], row[c].undo, -row[c].base));
            row[c].sum += w;
            p[c][e] = (_Float16)w;
        }
}

// Four waves share a range of a sequence's tokens, a wave every fourth step of 32; their sums meet in LDS.  One range: the
// result.  Several: each leaves its sums, and kv_join_kernel adds them.  Workgroups go through the first ranges of all tiles and
// heads, then the second ones (those behind short sequences come last and end at once), a place further each time: workgroups
// are dealt to the eight XCDs in turn, and neither a sequence nor the first ranges, which all sequences have, fall to one of them
// (32 sequences of 1 to 8192 tokens: 56 us without that, 41 with it).
// Bound by vector arithmetic on its way to HBM's rate: codes to values, the exponentials, and what the matrix instructions leave.
// One set of registers a step, at four waves a SIMD, is faster than two sets at three: the other waves cover the loads.  One query
// each of 32 heads, 8 key heads of 128: 8 sequences of 131072 tokens 205 us, 1090 MB at 5.3 TB/s, the vector units busy 70 %; 32
// ragged ones up to 8192 40.6 us, 4.0 TB/s, busy 43 %: they end unevenly; 16 x 5 queries (NQ 2) over up to 4099 tokens 26.8 us for
// 39 MB: some 500 vector instructions a step, at most eight steps a wave and uneven (a second set of registers, which 32 rows have room
// for: 27.5), vector units busy 22 % and waiting 36 % of the time: two waves a SIMD do not cover a step's way, and 12 of 32 rows are
// empty.  One query over 4096 tokens 7.0 us: the way of a step or two, from table over codes to merge, rather than any rate.
template <int D, int G, int NQ>
__global__ __launch_bounds__(256, D == 256 ? 3 - NQ : NQ > 1 ? 2 : 4) void kv_attention_kernel(KvAttentionArgs a, uint32_t groups)
{
    constexpr int TILES = Shape<D>::TILES, MD = Shape<D>::MD;
    __shared__ float merge[4][16][MD + 4];
    __shared__ float stat[2][4][NQ * 16];
    const int split = (int)(blockIdx.x / groups);
    uint32_t id = blockIdx.x % groups + split;
    while (id >= groups) id -= groups;
    const int h = (int)(id % a.c.kv_heads);
    id /= a.c.kv_heads;
    const int tile = (int)(id % a.tiles);
    const int64_t b = a.first + id / a.tiles;
    const View v = view_of(a, b);
    if (tile * a.tile_rows >= v.rows * a.ratio) return;
    const Range range = range_of(a, v, tile);
    const int64_t begin64 = range.lo + (int64_t)split * a.chunk;
    if (split > 0 && begin64 >= range.hi) return;
    const int begin = (int)(begin64 < range.hi ? begin64 : range.hi);
    const int end = range.hi - begin > a.chunk ? begin + a.chunk : range.hi;
    const int lane = threadIdx.x & 63, r = lane & 15, j = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Table table = table_of(a.s.table + b * a.s.ld_table);

    // The first step is on its way before the queries.  Keys of the next step are loaded when this one's have become scores, values
    // when they have been added: a set of registers each, a step's arithmetic of the other waves to arrive in.  Behind the last
    // step it is loaded again, so that no branch hides how many loads are on their way.
    const Lane at = lane_of_step<D, G>(r, j);
    Step<D, G> x;
    Half here[2];
    int pages[2], t = begin + 32 * wave;
    auto look = [&](int token) {
        pages[0] = page_at(a, table, token);
        pages[1] = page_at(a, table, token + 16);
    };
    if (t < end) {
        look(t);
        here[0] = half_at(a, pages[0], h, t);
        here[1] = half_at(a, pages[1], h, t + 16);
        load_keys<D, G>(x, a, here, at);
        load_values<D, G>(x, a, here, at);
        look(t + 128 < end ? t + 128 : t);
    }

    h8 q[NQ][Shape<D>::STEPS];
    Row row[NQ];
    int all_limit = v.len, all_low = 0;  // what every row sees
#pragma unroll
    for (int c = 0; c < NQ; ++c) {
        const int at = tile * a.tile_rows + c * 16 + r, query = at / a.ratio;
        const bool there = query < v.rows;
        const uint16_t* from = (const uint16_t*)a.q + (int64_t)(v.start + (there ? query : 0)) * a.ld_q +
                               (int64_t)(h * a.ratio + at % a.ratio) * a.hd_q;
        row[c].undo = load_row<D>(q[c], from, there, a.type == DT_BF16, j, a.scale);
        sees(a, v, there ? query : v.rows - 1, row[c].low, row[c].limit);  // (rows that are not there: as the last query)
        row[c].ref = -__builtin_inff();
        row[c].base = row[c].sum = 0.0f;
        all_limit = all_limit < row[c].limit ? all_limit : row[c].limit;
        all_low = all_low > row[c].low ? all_low : row[c].low;
    }
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) {
        const int x = __shfl_xor(all_limit, off, 64), y = __shfl_xor(all_low, off, 64);
        all_limit = all_limit < x ? all_limit : x;
        all_low = all_low > y ? all_low : y;
    }
    all_limit = __builtin_amdgcn_readfirstlane(all_limit);
    all_low = __builtin_amdgcn_readfirstlane(all_low);
    all_limit = all_limit < end ? all_limit : end;

    v4f acc[NQ][TILES];
#pragma unroll
    for (int c = 0; c < NQ; ++c)
#pragma unroll
        for (int n = 0; n < TILES; ++n) acc[c][n] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};

    for (; t < end; t += 128) {
        const int then = t + 128 < end ? t + 128 : t;
        v4f s[NQ][2];
        scores<D, G, NQ>(s, x.k, x.ks, q);
        const Half next[2] = {half_at(a, pages[0], h, then), half_at(a, pages[1], h, then + 16)};
        load_keys<D, G>(x, a, next, at);
        look(then + 128 < end ? then + 128 : then);
        const bool edge = t < all_low || t + 32 > all_limit || !here[0].ok || !here[1].ok;
        if (edge) {
            // what no row sees -- behind the sequence, or before all windows -- may be anything: its values become 0 (a weight of 0
            // would not: 0 times NaN)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int token = t + (e >> 2) * 16 + 4 * j + (e & 3);
                x.vs[e] = token >= range.low && token < end && here[e >> 2].ok ? x.vs[e] : 0u;
            }
        }
        h8 p[NQ];
        weigh<NQ, TILES>(p, s, row, acc, edge, t, end, here[0].ok, here[1].ok, j, [] {});
        add_values<D, G, NQ>(acc, x, p, r);
        load_values<D, G>(x, a, next, at);
        here[0] = next[0];
        here[1] = next[1];
    }

    // the waves' sums
#pragma unroll
    for (int c = 0; c < NQ; ++c) {
        row[c].sum += __shfl_xor(row[c].sum, 16, 64);
        row[c].sum += __shfl_xor(row[c].sum, 32, 64);
        if (j == 0) stat[0][wave][c * 16 + r] = row[c].ref, stat[1][wave][c * 16 + r] = row[c].sum;
    }
    __syncthreads();
    constexpr int EACH = 8, PER = MD / EACH;  // channels of a thread, threads of a row
    const int orow = threadIdx.x / PER, och = threadIdx.x % PER * EACH;
#pragma unroll
    for (int c = 0; c < NQ; ++c) {
        float top = -__builtin_inff();
#pragma unroll
        for (int w = 0; w < 4; ++w) top = __builtin_fmaxf(top, stat[0][w][c * 16 + r]);
        const float f = row[c].ref == -__builtin_inff() && row[c].sum == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(row[c].base - top);
        float total = 0.0f, most = -__builtin_inff();
        if (orow < 16) {
#pragma unroll
            for (int w = 0; w < 4; ++w) most = __builtin_fmaxf(most, stat[0][w][c * 16 + orow]);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float ref = stat[0][w][c * 16 + orow], l = stat[1][w][c * 16 + orow];
                total += l == 0.0f ? 0.0f : l * __builtin_amdgcn_exp2f((ref == -__builtin_inff() ? 0.0f : ref) - most);
            }
        }
        const int out_row = tile * a.tile_rows + c * 16 + orow, out_query = out_row / a.ratio;
        const bool writes = orow < 16 && out_query < v.rows;
        const int head = h * a.ratio + out_row % a.ratio;
        const int64_t token = v.start + out_query;
        float* part = nullptr;
        if (a.splits > 1 && writes) part = part_of<D>(a, b, tile, h, c * 16 + orow) + (int64_t)split * (D + 2);
#pragma unroll
        for (int piece = 0; piece < D / MD; ++piece) {
            if (c + piece > 0) __syncthreads();
            // lane (r, j) has channels j (D / 4) .. of row r: 4 runs of TILES
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c0 = j * (D / 4) + i * TILES - piece * MD;
                if (c0 >= 0 && c0 < MD) {
#pragma unroll
                    for (int n = 0; n < TILES; ++n) merge[wave][r][c0 + n] = acc[c][n][i] * f;
                }
            }
            __syncthreads();
            if (writes) {
                float o[EACH];
#pragma unroll
                for (int e = 0; e < EACH; ++e)
                    o[e] = merge[0][orow][och + e] + merge[1][orow][och + e] + merge[2][orow][och + e] + merge[3][orow][och + e];
                if (a.splits > 1) {
#pragma unroll
                    for (int e = 0; e < EACH; ++e) part[piece * MD + och + e] = o[e];
                } else {
                    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
                    store8((uint16_t*)a.out + token * a.ld_out + head * a.hd_out + piece * MD + och, o, inv, a.type == DT_BF16);
                }
            }
        }
        if (writes && och == 0) {
            if (a.splits > 1) part[D] = most, part[D + 1] = total;
            else if (a.lse) a.lse[token * a.heads + head] = total == 0.0f ? -__builtin_inff() : LN2 * (most + log2f(total));
        }
    }
}

// Many rows: WAVES waves of 16 NQ rows each go through the tokens together, and codes become fragments once for all of them.  A step
// is 32 tokens for every four waves: each converts a quarter of 32 tokens into a ring of three steps in LDS, laid out lane by
// lane as the matrix instruction reads them.  While a wave weighs the scores of 32 tokens, its products of the next 32's keys
// run, and the values' products follow.  A quarter: in K half the words of one of the two halves, in V 2 (d = 256: 4) of the D /
// 16 tiles.
// Bound by the waves' arithmetic beside the matrix products, and the meeting at each step: 2 x 1024 queries of 32 heads over 8192
// tokens, 258 GFLOP below the diagonal: 292 us (880 TFLOP/s; a plain product of large matrices 1355), matrix cores busy 35 %, vector
// units 47 %, waiting 28 % of the waves' time, no bank conflicts.  Four waves of 32 rows in 32-token
// steps: 538; 64 rows a wave do not fit the registers (990).  Causal tiles start in ascending order, the longest last: a prompt's first
// 8192 queries of 32 heads, 550 GFLOP below the diagonal, 721 us (762 TFLOP/s), 2 x 1024 51 us.  A wave without rows (33 to 64 rows for
// eight waves) still reads keys and multiplies them.
template <int D, int G>
struct Quarter {
    static constexpr int KN = Shape<D>::KW / 2, VN = D == 256 ? 4 : 2;
    uint32_t k[KN], ks, v[8], vs[8];
    bool ok0, ok1;
};

template <int D, int G>
__device__ __forceinline__ void load_quarter(Quarter<D, G>& x, const KvAttentionArgs& a, const int (&pages)[2], int h, int t, int wave,
                                             const Lane& at)
{
    constexpr int W = D / 8, GR = D / G, KN = Quarter<D, G>::KN;
    const Half half[2] = {half_at(a, pages[0], h, t), half_at(a, pages[1], h, t + 16)};
    x.ok0 = half[0].ok, x.ok1 = half[1].ok;
    const Half& mine = wave >> 1 ? half[1] : half[0];
    const uint8_t* k = a.c.k + mine.code;
    if constexpr (KN == 4) {
        const u32x4 w = read<u32x4>(k, at.k);
#pragma unroll
        for (int i = 0; i < 4; ++i) x.k[i] = w[i];
    } else if constexpr (KN == 2) {
        const u32x2 w = read<u32x2>(k, at.k);
        x.k[0] = w[0], x.k[1] = w[1];
    } else {
        x.k[0] = read<uint32_t>(k, at.k);
    }
    x.ks = read<uint32_t>(a.c.k_scale + mine.scale, at.ks);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        x.v[e] = read<uint32_t>(a.c.v + half[e >> 2].code, at.v, (e & 3) * W);
        x.vs[e] = read<uint32_t>(a.c.v_scale + half[e >> 2].scale, at.vs, (e & 3) * GR);
    }
}
template <int D, int G>
__device__ __forceinline__ Lane lane_of_quarter(int wave, int r, int j)
{
    constexpr int W = D / 8, GR = D / G, KN = Quarter<D, G>::KN;
    const int part = wave & 1;
    return Lane{4u * (r * W + j * (W / 4) + part * KN), 4u * (r * GR + (j * (D / 4) + part * (D / 8)) / G),
                4u * (4 * j * W + (D == 64 ? r >> 1 : D == 128 ? r : 2 * r + (wave >> 1))),
                4u * (4 * j * GR + r * (D / 16) / G)};
}

template <int D, int G>
__device__ __forceinline__ void convert_quarter(h8* slot, Quarter<D, G>& x, int t, int low, int end, int wave, int r, int j, int lane)
{
    constexpr int STEPS = Shape<D>::STEPS, KN = Quarter<D, G>::KN;
    const int part = wave & 1, half = wave >> 1;
    const h2 ks = low_pair(x.ks, x.ks), ko = high_pair(x.ks, x.ks);
#pragma unroll
    for (int i = 0; i < KN; ++i) slot[(half * STEPS + part * KN + i) * 64 + lane] = key_fragment(x.k[i], ks, ko);
    if (D == 64 && half) return;  // (four tiles: two waves have them)
    if (t < low || t + 32 > end || !x.ok0 || !x.ok1) {
        // what no row of the tile sees may be anything: its values become 0
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int token = t + (e >> 2) * 16 + 4 * j + (e & 3);
            x.vs[e] = token >= low && token < end && (e < 4 ? x.ok0 : x.ok1) ? x.vs[e] : 0u;
        }
    }
    // this wave's channels of a word: of the half `high`, those of `odd` (or all four)
    const uint32_t high = D == 64 ? r & 1 : D == 128 ? half : part;
    const uint32_t sel = high ? 0x07060302u : 0x05040100u;
    h8 f[Quarter<D, G>::VN];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const h2 s = low_pair(x.vs[2 * u], x.vs[2 * u + 1]), o = high_pair(x.vs[2 * u], x.vs[2 * u + 1]);
        uint32_t y = __builtin_amdgcn_perm(x.v[2 * u + 1], x.v[2 * u], sel);
        if constexpr (D == 256) {
            const h2 c0 = __builtin_elementwise_fma(codes_of<0>(y), s, o), c1 = __builtin_elementwise_fma(codes_of<1>(y), s, o);
            f[0][2 * u] = c0[0], f[0][2 * u + 1] = c0[1];
            f[1][2 * u] = c1[0], f[1][2 * u + 1] = c1[1];
            y >>= 8;
            const h2 c2 = __builtin_elementwise_fma(codes_of<0>(y), s, o), c3 = __builtin_elementwise_fma(codes_of<1>(y), s, o);
            f[2][2 * u] = c2[0], f[2][2 * u + 1] = c2[1];
            f[3][2 * u] = c3[0], f[3][2 * u + 1] = c3[1];
        } else {
            y >>= 8 * part;
            const h2 c0 = __builtin_elementwise_fma(codes_of<0>(y), s, o), c1 = __builtin_elementwise_fma(codes_of<1>(y), s, o);
            f[0][2 * u] = c0[0], f[0][2 * u + 1] = c0[1];
            f[1][2 * u] = c1[0], f[1][2 * u + 1] = c1[1];
        }
    }
    const int first = D == 256 ? half * 8 + part * 4 : D == 128 ? half * 4 + part * 2 : part * 2;
#pragma unroll
    for (int n = 0; n < Quarter<D, G>::VN; ++n) slot[(2 * STEPS + first + n) * 64 + lane] = f[n];
}

template <int D, int G, int NQ, int WAVES>
__global__ __launch_bounds__(64 * WAVES, NQ * D > 256 ? 1 : 2) void kv_chunk_kernel(KvAttentionArgs a, uint32_t groups)
{
    constexpr int STEPS = Shape<D>::STEPS, TILES = Shape<D>::TILES, SET = (2 * STEPS + TILES) * 64;
    constexpr int SETS = WAVES / 4, TOKENS = 32 * SETS, SLOT = SETS * SET;
    extern __shared__ h8 ring[];  // three steps
    const int split = (int)(blockIdx.x / groups);
    uint32_t id = blockIdx.x % groups;
    const int h = (int)(id % a.c.kv_heads);
    id /= a.c.kv_heads;
    const int tile = (int)(id % a.tiles);
    const int64_t b = a.first + id / a.tiles;
    const View v = view_of(a, b);
    if (tile * a.tile_rows >= v.rows * a.ratio) return;
    const Range range = range_of(a, v, tile);
    const int64_t begin64 = range.lo + (int64_t)split * a.chunk;
    if (split > 0 && begin64 >= range.hi) return;
    const int begin = (int)(begin64 < range.hi ? begin64 : range.hi);
    const int end = range.hi - begin > a.chunk ? begin + a.chunk : range.hi;
    const int lane = threadIdx.x & 63, r = lane & 15, j = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), quarter = wave & 3, mine = 32 * (wave >> 2);
    const Table table = table_of(a.s.table + b * a.s.ld_table);

    // codes of step t: looked up two steps ahead, loaded one ahead (of the conversion, which is one ahead of their use)
    const Lane place = lane_of_quarter<D, G>(quarter, r, j);
    Quarter<D, G> x{};
    int pages[2];
    auto look = [&](int t) {
        pages[0] = page_at(a, table, t + mine);
        pages[1] = page_at(a, table, t + mine + 16);
    };
    auto load = [&](int t) {
        load_quarter<D, G>(x, a, pages, h, t + mine, quarter, place);
        look(t + TOKENS);
    };
    // which pages of a set exist, for every wave
    __shared__ uint32_t good[3][2];
    auto convert = [&](int at, h8* slot, int t) {
        if (quarter == 0 && lane == 0) good[at][wave >> 2] = (x.ok0 ? 1u : 0u) | (x.ok1 ? 2u : 0u);
        convert_quarter<D, G>(slot + (wave >> 2) * SET, x, t + mine, range.low, end, quarter, r, j, lane);
    };
    if (begin < end) {
        look(begin);
        load(begin);
    }

    h8 q[NQ][STEPS];
    Row row[NQ];
    int all_limit = v.len, all_low = 0, any_limit = 0, any_low = v.len;
#pragma unroll
    for (int c = 0; c < NQ; ++c) {
        const int at = tile * a.tile_rows + (wave * NQ + c) * 16 + r, query = at / a.ratio;
        const bool there = query < v.rows;
        const uint16_t* from = (const uint16_t*)a.q + (int64_t)(v.start + (there ? query : 0)) * a.ld_q +
                               (int64_t)(h * a.ratio + at % a.ratio) * a.hd_q;
        row[c].undo = load_row<D>(q[c], from, there, a.type == DT_BF16, j, a.scale);
        sees(a, v, there ? query : v.rows - 1, row[c].low, row[c].limit);
        row[c].ref = -__builtin_inff();
        row[c].base = row[c].sum = 0.0f;
        all_limit = all_limit < row[c].limit ? all_limit : row[c].limit;
        all_low = all_low > row[c].low ? all_low : row[c].low;
        any_limit = any_limit > row[c].limit ? any_limit : row[c].limit;
        any_low = any_low < row[c].low ? any_low : row[c].low;
    }
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) {
        const int y0 = __shfl_xor(all_limit, off, 64), y1 = __shfl_xor(all_low, off, 64);
        const int y2 = __shfl_xor(any_limit, off, 64), y3 = __shfl_xor(any_low, off, 64);
        all_limit = all_limit < y0 ? all_limit : y0;
        all_low = all_low > y1 ? all_low : y1;
        any_limit = any_limit > y2 ? any_limit : y2;
        any_low = any_low < y3 ? any_low : y3;
    }
    all_limit = __builtin_amdgcn_readfirstlane(all_limit);
    all_low = __builtin_amdgcn_readfirstlane(all_low);
    any_limit = __builtin_amdgcn_readfirstlane(any_limit);
    any_low = __builtin_amdgcn_readfirstlane(any_low);
    all_limit = all_limit < end ? all_limit : end;
    any_limit = any_limit < end ? any_limit : end;
    if ((tile * a.tile_rows + wave * NQ * 16) / a.ratio >= v.rows) any_limit = 0;  // (no rows of its own)

    v4f acc[NQ][TILES];
#pragma unroll
    for (int c = 0; c < NQ; ++c)
#pragma unroll
        for (int n = 0; n < TILES; ++n) acc[c][n] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};

    auto products = [&](v4f(&s)[NQ][2], const h8(&k)[2 * STEPS]) {
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
#pragma unroll
            for (int c = 0; c < NQ; ++c) s[c][hh] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < STEPS; ++i)
#pragma unroll
                for (int c = 0; c < NQ; ++c)
                    s[c][hh] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[hh * STEPS + i], q[c][i], s[c][hh], 0, 0, 0);
        }
    };
    auto keys = [&](h8(&k)[2 * STEPS], const h8* set) {
#pragma unroll
        for (int i = 0; i < 2 * STEPS; ++i) k[i] = set[i * 64 + lane];
    };
    // 32 tokens from t on, whose scores are in `s` and values in `set`; the scores of the next 32, in `other`, go to `n`
    auto attend = [&](int t, v4f(&s)[NQ][2], const h8* set, uint32_t ok, v4f(&n)[NQ][2], const h8* other) {
        h8 k[2 * STEPS];
        keys(k, other);
        if (t < any_limit && t + 32 > any_low) {
            const bool edge = t < all_low || t + 32 > all_limit || ok != 3u;
            h8 p[NQ], vals[TILES];
            weigh<NQ, TILES>(p, s, row, acc, edge, t, end, ok & 1u, ok & 2u, j, [&] {
#pragma unroll
                for (int m = 0; m < TILES; ++m) vals[m] = set[(2 * STEPS + m) * 64 + lane];
                products(n, k);
            });
#pragma unroll
            for (int m = 0; m < TILES; ++m)
#pragma unroll
                for (int c = 0; c < NQ; ++c) acc[c][m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vals[m], p[c], acc[c][m], 0, 0, 0);
        } else {
            products(n, k);
        }
    };

    v4f s0[NQ][2], s1[NQ][2];
    int now = 0, next = 1, spare = 2;
    if (begin < end) convert(0, ring, begin);
    if (begin + TOKENS < end) {
        load(begin + TOKENS);
        convert(1, ring + SLOT, begin + TOKENS);
    }
    if (begin + 2 * TOKENS < end) load(begin + 2 * TOKENS);
    __syncthreads();
    {
        h8 k[2 * STEPS];
        keys(k, ring);
        products(s0, k);
    }
    for (int t = begin; t < end; t += TOKENS) {
        const h8 *set = ring + now * SLOT, *following = ring + next * SLOT;
        const uint32_t ok0 = __builtin_amdgcn_readfirstlane(good[now][0]), ok1 = __builtin_amdgcn_readfirstlane(good[now][SETS - 1]);
        auto feed = [&] {
            if (t + 2 * TOKENS < end) {
                convert(spare, ring + spare * SLOT, t + 2 * TOKENS);
                if (t + 3 * TOKENS < end) load(t + 3 * TOKENS);
            }
        };
        if constexpr (SETS == 2) {
            // (waves w and w + 4 share a SIMD: one converts while the other multiplies)
            if (wave < 4) feed();
            attend(t, s0, set, ok0, s1, set + SET);
            if (wave >= 4) feed();
            attend(t + 32, s1, set + SET, ok1, s0, following);
        } else {
            feed();
            attend(t, s0, set, ok0, s1, following);
#pragma unroll
            for (int c = 0; c < NQ; ++c) s0[c][0] = s1[c][0], s0[c][1] = s1[c][1];
        }
        __syncthreads();  // the step after next is written, this one is read
        const int old = now;
        now = next;
        next = spare;
        spare = old;
    }

    // each wave has its rows' sums: lane (r, j) the channels j (D / 4) .. of row r
#pragma unroll
    for (int c = 0; c < NQ; ++c) {
        float sum = row[c].sum;
        sum += __shfl_xor(sum, 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        const int in_tile = (wave * NQ + c) * 16 + r, at = tile * a.tile_rows + in_tile, query = at / a.ratio;
        if (query >= v.rows) continue;
        const int head = h * a.ratio + at % a.ratio;
        const int64_t token = v.start + query;
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        float* part = a.splits > 1 ? part_of<D>(a, b, tile, h, in_tile) + (int64_t)split * (D + 2) : nullptr;
        uint16_t* out = (uint16_t*)a.out + token * a.ld_out + head * a.hd_out;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c0 = j * (D / 4) + i * TILES;
            if (a.splits > 1) {
#pragma unroll
                for (int n = 0; n < TILES; ++n) part[c0 + n] = acc[c][n][i];
            } else if constexpr (TILES >= 8) {
#pragma unroll
                for (int n = 0; n < TILES; n += 8) {
                    float o[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) o[e] = acc[c][n + e][i];
                    store8(out + c0 + n, o, inv, a.type == DT_BF16);
                }
            } else {
#pragma unroll
                for (int n = 0; n < TILES; ++n) {
                    const float o = acc[c][n][i] * inv;
                    out[c0 + n] = a.type == DT_BF16 ? __builtin_bit_cast(uint16_t, (__bf16)o) : f32_to_f16(o);
                }
            }
        }
        if (j == 0) {
            if (a.splits > 1) part[D] = row[c].ref, part[D + 1] = sum;
            else if (a.lse) a.lse[token * a.heads + head] = sum == 0.0f ? -__builtin_inff() : LN2 * (row[c].base + log2f(sum));
        }
    }
}

// Adds what the ranges of a row left, eight at a time so that their loads are in flight together: WAVES waves a row, each taking
// every WAVES-th range, their sums added in order.  A launch of its own: 4 to 5 us for 2 MB, latency.
template <int D, int WAVES>
__global__ __launch_bounds__(256) void kv_join_kernel(KvAttentionArgs a, uint32_t all_rows)
{
    constexpr int E = D / 64, ROWS = 4 / WAVES;
    __shared__ float o_of[WAVES][D], l_of[WAVES];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t all = (int64_t)a.max_q * a.ratio;
    const int rows = (int)(all < a.tile_rows ? all : a.tile_rows);
    uint32_t id = blockIdx.x * ROWS + (WAVES == 1 ? wave : 0);
    if (id >= all_rows) return;
    const int orow = (int)(id % rows);
    id /= rows;
    const int h = (int)(id % a.c.kv_heads);
    id /= a.c.kv_heads;
    const int tile = (int)(id % a.tiles);
    const int64_t b = a.first + id / a.tiles;
    const View v = view_of(a, b);
    const int row = tile * a.tile_rows + orow, query = row / a.ratio;
    if (query >= v.rows) return;
    const Range range = range_of(a, v, tile);
    const int64_t span = (int64_t)range.hi - range.lo;
    const int n = span <= a.chunk ? 1 : (int)((span + a.chunk - 1) / a.chunk);
    const float* part = part_of<D>(a, b, tile, h, orow);
    float most = -__builtin_inff();
    for (int s = lane; s < n; s += 64) most = __builtin_fmaxf(most, part[(int64_t)s * (D + 2) + D]);
    most = wave_max(most);
    float total = 0.0f, o[E] = {};
    for (int s0 = WAVES == 1 ? 0 : wave; s0 < n; s0 += 8 * WAVES) {
        float x[8][E], c[8], l[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int s = s0 + WAVES * u < n ? s0 + WAVES * u : n - 1;
            const float* from = part + (int64_t)s * (D + 2);
            c[u] = from[D], l[u] = from[D + 1];
#pragma unroll
            for (int e = 0; e < E; ++e) x[u][e] = from[lane * E + e];
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const float f = s0 + WAVES * u >= n || l[u] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(c[u] - most);
            total += f == 0.0f ? 0.0f : l[u] * f;
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] += f == 0.0f ? 0.0f : x[u][e] * f;
        }
    }
    if constexpr (WAVES > 1) {
#pragma unroll
        for (int e = 0; e < E; ++e) o_of[wave][lane * E + e] = o[e];
        if (lane == 0) l_of[wave] = total;
        __syncthreads();
        if (wave > 0) return;
#pragma unroll
        for (int w = 1; w < WAVES; ++w) {
            total += l_of[w];
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] += o_of[w][lane * E + e];
        }
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    const int head = h * a.ratio + row % a.ratio;
    const int64_t token = v.start + query;
    uint16_t* out = (uint16_t*)a.out + token * a.ld_out + head * a.hd_out + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const float y = o[e] * inv;
        out[e] = a.type == DT_BF16 ? __builtin_bit_cast(uint16_t, (__bf16)y) : f32_to_f16(y);
    }
    if (a.lse && lane == 0) a.lse[token * a.heads + head] = total == 0.0f ? -__builtin_inff() : LN2 * (most + log2f(total));
}

// The weight that cached tokens received: the scores again, exp(score - lse) summed over a tile's rows, tile after tile.  Here S = Q
// K^T, the operands the other way round, so that a lane's scores belong to one token (its column) and to the rows 4 j .. 4 j + 3: the
// sum over rows stays in the lane until the end.  A wave takes 64 tokens at a time (d = 256: 32), whose keys stay in registers while
// the rows, converted once per workgroup, come from LDS, eight tiles at a time (sixteen for eight waves and d below 256); more tiles
// take another turn over the tokens, adding to what the turn before left in the output.  One query each of 16 ragged sequences up to
// 8192 (32 heads, 8 key heads of 128): 25 us for 56 MB read and written, no unit busy (vector 16 %) and waves waiting 44 % of their time:
// a range is three steps a wave at most, behind the rows' way through LDS and a barrier.  64 queries of 2 sequences over 16384:
// 33 us, 17 GFLOP of products, matrix cores busy 17 %, vector units 36 %, waiting 37 %: a tile's rows are read from LDS when they are used.
template <int D, int WAVES>
constexpr int TURN = WAVES == 8 && D < 256 ? 16 : 8;  // tiles of rows in LDS
struct TileRows {
    float undo[16], lse[16];
    int low[16], limit[16];
    v4i span;  // what any row sees begins and ends there; what all do
};

template <int D, int G, int WAVES>
__global__ __launch_bounds__(64 * WAVES, WAVES == 8 ? 2 : 3) void kv_weights_kernel(KvAttentionArgs a, uint32_t groups)
{
    constexpr int TURN = ascq::TURN<D, WAVES>;
    constexpr int STEPS = Shape<D>::STEPS, KW = Shape<D>::KW, NT = D == 256 ? 2 : 4, TOKENS = 16 * NT;
    constexpr int W = D / 8, GR = D / G, KS = Step<D, G>::KS;
    extern __shared__ h8 rows_of[];
    __shared__ TileRows info[TURN];
    const int part = (int)(blockIdx.x / groups);
    uint32_t id = blockIdx.x % groups + part;
    while (id >= groups) id -= groups;
    const int h = (int)(id % a.c.kv_heads);
    const int64_t b = a.first + id / a.c.kv_heads;
    const int lane = threadIdx.x & 63, r = lane & 15, j = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const View v = view_of(a, b);
    float* out = a.w_out + (b * a.c.kv_heads + h) * (int64_t)a.cap;
    const float* in = a.w_in ? a.w_in + (b * a.c.kv_heads + h) * (int64_t)a.cap : nullptr;
    const int64_t begin64 = (int64_t)part * a.chunk;
    const int begin = (int)begin64, stop = a.cap - begin > a.chunk ? begin + a.chunk : a.cap;  // (begin < cap)
    const int end = stop < v.len ? stop : v.len;
    const Table table = table_of(a.s.table + b * a.s.ld_table);
    if (!in)
        for (int i = (begin > v.len ? begin : v.len) + (int)threadIdx.x; i < stop; i += 64 * WAVES) out[i] = 0.0f;
    if (begin >= end) return;

    const uint32_t at_k = 4u * (r * W + j * (W / 4)), at_s = 4u * (r * GR + j * (D / 4) / G);
    uint32_t k[NT][KW], ks[NT][KS], ok = 0;
    int pages[NT];  // (looked up a step ahead of the loads)
    auto look = [&](int t) {
#pragma unroll
        for (int n = 0; n < NT; ++n) pages[n] = page_at(a, table, t + 16 * n);
    };
    // What a lane's token has, before the call or from earlier turns: loaded whether it counts or not, as its store is issued
    // whether it has a token or not (one behind the range is dropped), so that no branch hides how many are on their way.
    float had = 0.0f;
    const rsrc_t results = make_rsrc(out + begin, 4u * (uint32_t)(end - begin));
    auto load = [&](int t, int turn) {
        ok = 0;
        had = (in && turn == 0 ? in : out)[t + lane < end ? t + lane : end - 1];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const Half half = half_at(a, pages[n], h, t + 16 * n);
            ok |= half.ok ? 1u << n : 0u;
            const uint8_t* from = a.c.k + half.code;
            if constexpr (KW == 2) {
                const u32x2 w = read<u32x2>(from, at_k);
                k[n][0] = w[0], k[n][1] = w[1];
            } else {
#pragma unroll
                for (int i = 0; i < KW; i += 4) {
                    const u32x4 w = read<u32x4>(from, at_k, i);
#pragma unroll
                    for (int e = 0; e < 4; ++e) k[n][i + e] = w[e];
                }
            }
#pragma unroll
            for (int i = 0; i < KS; ++i) ks[n][i] = read<uint32_t>(a.c.k_scale + half.scale, at_s, i);
        }
        look(t + WAVES * TOKENS);
    };

    const int tiles = (v.rows * a.ratio + 15) / 16;
    for (int turn = 0; turn == 0 || turn < tiles; turn += TURN) {
        int t = begin + TOKENS * wave;
        if (t < end) {
            look(t);
            load(t, turn);
        }
        if (turn > 0) __syncthreads();
        for (int tile = turn + wave; tile < tiles && tile < turn + TURN; tile += WAVES) {
            const int row = tile * 16 + r, query = row / a.ratio;
            const bool there = query < v.rows;
            const int64_t token = v.start + (there ? query : 0);
            const int head = h * a.ratio + row % a.ratio;
            h8 q[STEPS];
            const float undo = load_row<D>(q, (const uint16_t*)a.q + token * a.ld_q + (int64_t)head * a.hd_q, there,
                                           a.type == DT_BF16, j, a.scale);
            float lse = there ? a.lse[token * a.heads + head] : __builtin_inff();
            lse = lse == -__builtin_inff() ? __builtin_inff() : lse * LOG2E;  // (a row that saw nothing gives nothing)
            int low = 0, limit = v.len;
            if (there) sees(a, v, query, low, limit);
            TileRows& x = info[tile - turn];
#pragma unroll
            for (int i = 0; i < STEPS; ++i) rows_of[((tile - turn) * STEPS + i) * 64 + lane] = q[i];
            // (a row that is not there sees nothing; it does not make a step one of an edge, though)
            int any_low = there ? low : v.len, any_limit = there ? limit : 0, all_low = low, all_limit = limit;
            if (j == 0) x.undo[r] = undo, x.lse[r] = lse, x.low[r] = low, x.limit[r] = any_limit;
#pragma unroll
            for (int off = 1; off < 16; off <<= 1) {
                const int y0 = __shfl_xor(any_low, off, 64), y1 = __shfl_xor(any_limit, off, 64);
                const int y2 = __shfl_xor(all_low, off, 64), y3 = __shfl_xor(all_limit, off, 64);
                any_low = any_low < y0 ? any_low : y0;
                any_limit = any_limit > y1 ? any_limit : y1;
                all_low = all_low > y2 ? all_low : y2;
                all_limit = all_limit < y3 ? all_limit : y3;
            }
            if (lane == 0) x.span = (v4i){any_low, any_limit, all_low, all_limit};
        }
        __syncthreads();
        const int here = tiles - turn < TURN ? tiles - turn : TURN;
        for (; t < end; t += WAVES * TOKENS) {
            h8 f[NT][STEPS];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < STEPS; ++i) {
                    const uint32_t w = ks[n][i * KS / STEPS];
                    f[n][i] = key_fragment(k[n][i], low_pair(w, w), high_pair(w, w));
                }
            const uint32_t good = ok;
            const float before = turn > 0 ? had : in ? a.decay * had : 0.0f;
            if (t + WAVES * TOKENS < end) load(t + WAVES * TOKENS, turn);
            float got[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) got[n] = 0.0f;
            for (int tile = 0; tile < here; ++tile) {
                // (a tile's reads together: they take longer than its products)
                const TileRows& x = info[tile];
                const v4i span = x.span;
                const v4f undo = *(const v4f*)(x.undo + 4 * j), lse = *(const v4f*)(x.lse + 4 * j);
                h8 q[STEPS];
                if constexpr (WAVES == 8)
#pragma unroll
                    for (int i = 0; i < STEPS; ++i) q[i] = rows_of[(tile * STEPS + i) * 64 + lane];
                if (t >= __builtin_amdgcn_readfirstlane(span[1]) || t + TOKENS <= __builtin_amdgcn_readfirstlane(span[0])) continue;
                const bool edge = t < __builtin_amdgcn_readfirstlane(span[2]) ||
                                  t + TOKENS > __builtin_amdgcn_readfirstlane(span[3]) || good != (1u << NT) - 1;
                v4f s[NT];
#pragma unroll
                for (int n = 0; n < NT; ++n) s[n] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < STEPS; ++i) {
                    if constexpr (WAVES < 8) q[i] = rows_of[(tile * STEPS + i) * 64 + lane];  // (registers for more waves)
#pragma unroll
                    for (int n = 0; n < NT; ++n) s[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(q[i], f[n][i], s[n], 0, 0, 0);
                }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[n][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][i], undo[i], -lse[i]));
                if (edge) {
                    const v4i low = *(const v4i*)(x.low + 4 * j), limit = *(const v4i*)(x.limit + 4 * j);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const int token = t + 16 * n + r;
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            s[n][i] = token >= low[i] && token < limit[i] && (good >> n & 1u) ? s[n][i] : 0.0f;
                    }
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) got[n] += (s[n][0] + s[n][1]) + (s[n][2] + s[n][3]);
            }
            float mine = 0.0f;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                got[n] += __shfl_xor(got[n], 16, 64);
                got[n] += __shfl_xor(got[n], 32, 64);
                mine = j == n ? got[n] : mine;
            }
            // (lane 16 n + r: token r of tile n)
            __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(before + mine), results,
                                                  lane < TOKENS ? 4u * (uint32_t)(t - begin + lane) : OOB, 0, 0);
        }
    }
}

constexpr int UNIT = 128;  // tokens of a range: a step of each of four waves, or two steps of eight

// tokens that a tile can see at most
int64_t widest(const KvAttentionArgs& a)
{
    const int64_t all = (int64_t)a.s.table_pages << a.c.page_shift;
    const int64_t seen = a.window && a.causal ? (int64_t)a.window + a.tile_rows / a.ratio + 1 + 31 : all;
    return seen < all ? seen : all;
}

int rows_in_use(const KvAttentionArgs& a)
{
    const int64_t rows = (int64_t)a.max_q * a.ratio;
    return (int)(rows < a.tile_rows ? rows : a.tile_rows);
}

// bytes that one split of every row takes in the workspace
size_t split_bytes(const KvAttentionArgs& a)
{
    return (size_t)a.s.batch * a.tiles * a.c.kv_heads * rows_in_use(a) * (a.c.d + 2) * sizeof(float);
}

// tiles of rows, and ranges of tokens as far as `room` bytes go
void plan(KvAttentionArgs& a, size_t room)
{
    a.ratio = a.heads / a.c.kv_heads;
    const int64_t rows = (int64_t)a.max_q * a.ratio;
    a.tile_rows = rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 && a.c.d == 256 ? 64 : rows <= 128 || a.c.d == 256 ? 128 : 256;
    a.tiles = (int)((rows + a.tile_rows - 1) / a.tile_rows);
    const int64_t span = widest(a);
    const int64_t groups = (int64_t)a.s.batch * a.tiles * a.c.kv_heads;
    // Ranges: one workgroup per CU where a step of each of its waves (UNIT tokens) is left to it, and more of them while three steps
    // are: up to six per CU of few rows (four fit at a time), two of 32 rows, one of more rows, whose sums of further ranges are many.
    // (up to 16 rows, us: 32 ragged sequences up to 8192 / 8 of 131072: 1024 ranges 53 / 205, 1536 41 / 206, 2048 43 / 207;
    // 32 rows, 2 x 8 queries over 65536 / 32 ragged ones: 256 48 / 78, 512 44 / 76 with the join, 1024 51 / 74; more rows, 64
    // queries over 16384 / 4 x 256 over ragged ones: 256 42 / 299, 512 62 / 265)
    const int64_t wanted = a.tile_rows == 16 ? 1536 : a.tile_rows == 32 ? 512 : 256;
    const int64_t short_ones = (span + UNIT - 1) / UNIT, long_ones = (span + 3 * UNIT - 1) / (3 * UNIT);
    int64_t splits = wanted / groups, few = 256 / groups;
    few = few < short_ones ? few : short_ones;
    const int64_t most = few > long_ones ? few : long_ones, fit = (int64_t)(room / split_bytes(a));
    splits = splits < most ? splits : most;
    splits = splits < fit ? splits : fit;
    splits = splits < 1 ? 1 : splits;
    const int64_t chunk = ((span + splits - 1) / splits + UNIT - 1) / UNIT * UNIT;
    a.chunk = (int)(chunk < UNIT ? UNIT : chunk);
    a.splits = (int)((span + a.chunk - 1) / a.chunk);
    if (a.splits < 1) a.splits = 1;
}

template <int D, int G>
hipError_t run_attention(KvAttentionArgs a, hipStream_t st)
{
    const int64_t per = (int64_t)a.tiles * a.c.kv_heads;         // tiles and heads of a sequence
    const int64_t most = ((int64_t)1 << 22) / (per * a.splits);  // sequences of a launch: at most 2^31 threads
    float* part = a.part;
    for (int64_t at = 0; at < a.s.batch; at += most) {
        const int64_t n = a.s.batch - at < most ? a.s.batch - at : most;
        a.first = (int)at;
        KvAttentionArgs now = a;
        now.s.batch = (int)(at + n);
        const int64_t rows = per * rows_in_use(a);
        now.part = part + at * rows * a.splits * (a.c.d + 2);
        const uint32_t groups = (uint32_t)(n * per);
        const dim3 grid(groups * a.splits);
        hipError_t e = hipSuccess;
        auto chunk = [&](auto nq, auto waves) {
            constexpr int NQ = decltype(nq)::value, WAVES = decltype(waves)::value;
            constexpr int LDS = 3 * (WAVES / 4) * (2 * Shape<D>::STEPS + Shape<D>::TILES) * 1024;
            e = ensure_dynamic_lds<kv_chunk_kernel<D, G, NQ, WAVES>>(LDS);
            if (e == hipSuccess) launch_k(kv_chunk_kernel<D, G, NQ, WAVES>, grid, dim3(64 * WAVES), LDS, st, now, groups);
        };
        using one = std::integral_constant<int, 1>;
        using two = std::integral_constant<int, 2>;
        using waves = std::integral_constant<int, D == 256 ? 4 : 8>;
        if (a.tile_rows == 16) launch_k(kv_attention_kernel<D, G, 1>, grid, dim3(256), 0, st, now, groups);
        else if (a.tile_rows == 32) launch_k(kv_attention_kernel<D, G, 2>, grid, dim3(256), 0, st, now, groups);
        else if (a.tile_rows == 16 * waves::value) chunk(one{}, waves{});
        else chunk(two{}, waves{});
        if (e == hipSuccess) e = hipGetLastError();
        if (e != hipSuccess) return e;
        if (a.splits > 1) {
            const uint32_t all = (uint32_t)(n * rows);
            if (a.splits > 16) hipLaunchKernelGGL(HIP_KERNEL_NAME(kv_join_kernel<D, 4>), dim3(all), dim3(256), 0, st, now, all);
            else hipLaunchKernelGGL(HIP_KERNEL_NAME(kv_join_kernel<D, 1>), dim3((all + 3) / 4), dim3(256), 0, st, now, all);
            e = hipGetLastError();
            if (e != hipSuccess) return e;
        }
    }
    return hipSuccess;
}

template <int D, int G, int WAVES>
hipError_t run_weights_by(KvAttentionArgs a, int64_t tiles, int64_t wanted, hipStream_t st)
{
    constexpr int TILE = Shape<D>::STEPS * 1024, MOST = ascq::TURN<D, WAVES>;
    hipError_t e = ensure_dynamic_lds<kv_weights_kernel<D, G, WAVES>>(MOST * TILE);
    if (e != hipSuccess) return e;
    const int64_t groups = (int64_t)a.s.batch * a.c.kv_heads;
    constexpr int unit = (D == 256 ? 32 : 64) * WAVES;
    int64_t parts = wanted / groups;
    parts = parts < 4 ? 4 : parts;  // (a range is below 2^30 bytes)
    a.chunk = (int)(((a.cap + parts - 1) / parts + unit - 1) / unit * unit);
    parts = (a.cap + (int64_t)a.chunk - 1) / a.chunk;
    const int64_t per = parts * a.c.kv_heads, most = ((int64_t)1 << 22) / per;  // sequences of a launch: at most 2^31 threads
    for (int64_t at = 0; at < a.s.batch; at += most) {
        const int64_t n = a.s.batch - at < most ? a.s.batch - at : most;
        a.first = (int)at;
        launch_k(kv_weights_kernel<D, G, WAVES>, dim3((uint32_t)(n * per)), dim3(64 * WAVES),
                 (uint32_t)((tiles < MOST ? tiles : MOST) * TILE), st, a, (uint32_t)(n * a.c.kv_heads));
        e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

template <int D, int G>
hipError_t run_weights(KvAttentionArgs a, hipStream_t st)
{
    a.ratio = a.heads / a.c.kv_heads;
    const int64_t tiles = ((int64_t)a.max_q * a.ratio + 15) / 16;
    // Up to 4 tiles of rows ranges as in the attention; more rows: eight waves share the conversion of the rows, a workgroup per CU
    // (us, 64 queries of 2 x 32 heads over 16384 tokens: 4 waves 50, 8 37; ranges of up to 4 tiles, one query of 64 ragged sequences
    // up to 4096 / 8 queries of 8 up to 8192 / one of 2 x 65536: 768 33 / 18 / 25, 1024 34 / 15 / 27, 1536 33 / 15 / 28, 2304 35 / 17 / 29)
    return tiles > 4 ? run_weights_by<D, G, 8>(a, tiles, 256, st) : run_weights_by<D, G, 4>(a, tiles, 1536, st);
}

#define KV_SHAPES(RUN)                                              \
    switch (a.c.d * 256 + a.c.group) {                              \
    case 64 * 256 + 32: return RUN<64, 32>(a, st);                  \
    case 64 * 256 + 64: return RUN<64, 64>(a, st);                  \
    case 128 * 256 + 32: return RUN<128, 32>(a, st);                \
    case 128 * 256 + 64: return RUN<128, 64>(a, st);                \
    case 128 * 256 + 128: return RUN<128, 128>(a, st);              \
    case 256 * 256 + 32: return RUN<256, 32>(a, st);                \
    case 256 * 256 + 64: return RUN<256, 64>(a, st);                \
    case 256 * 256 + 128: return RUN<256, 128>(a, st);              \
    default: return hipErrorInvalidValue;                           \
    }

}  // namespace

size_t kv_attention_ws_bytes(KvAttentionArgs a)
{
    plan(a, SIZE_MAX);
    return a.splits < 2 ? 0 : split_bytes(a) * a.splits;
}

hipError_t launch_kv_attention(KvAttentionArgs a, void* ws, size_t ws_bytes, hipStream_t st)
{
    plan(a, ws ? ws_bytes : 0);
    a.part = (float*)ws;
    KV_SHAPES(run_attention)
}

hipError_t launch_kv_weights(KvAttentionArgs a, hipStream_t st)
{
    KV_SHAPES(run_weights)
}

}  // namespace ascq
