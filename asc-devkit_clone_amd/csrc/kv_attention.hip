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
// Scores are fp32 sums of exact f16 products (bf16 queries are scaled by a power of two per row into f16's range, which
// keeps all their bits); P is rounded to f16 after exp2 (2^-12 a weight at most, and independent), sums and statistics are
// fp32.
#include "common.h"

namespace ascq {

namespace {

typedef u32x4 u32x4_any __attribute__((aligned(2)));

struct View {
    int start, rows, n, len;  // first row of q; queries computed; queries there are; tokens
};
__device__ __forceinline__ View view_of(const KvAttentionArgs& a, int64_t b)
{
    View v;
    int64_t start = b, n = 1;
    if (a.s.starts) {
        start = a.s.starts[b];
        n = (int64_t)a.s.starts[b + 1] - start;
    }
    if (start < 0 || start > a.T || n < 0) start = 0, n = 0;
    int64_t rows = n < a.max_q ? n : a.max_q;
    if (rows > (int64_t)a.T - start) rows = (int64_t)a.T - start;
    v.start = (int)start;
    v.rows = (int)rows;
    v.n = (int)n;
    const int64_t most = (int64_t)a.s.table_pages << a.c.page_shift;
    const int64_t len = a.s.lengths[b];
    v.len = (int)(len < 0 ? 0 : len > most ? most : len);
    return v;
}

// the tokens [lo, hi) that the rows of tile `t` see together; a row's own limits follow from its query
struct Range {
    int lo, hi;
};
__device__ __forceinline__ Range range_of(const KvAttentionArgs& a, const View& v, int tile)
{
    const int first = tile * 16 / a.ratio;
    int last = (tile * 16 + 15) / a.ratio;
    last = last < v.rows ? last : v.rows - 1;
    Range r{0, v.len};
    const int64_t at = (int64_t)v.len - v.n;  // the first query's token
    if (a.causal) {
        const int64_t hi = at + last + 1;
        r.hi = hi < 0 ? 0 : hi < v.len ? (int)hi : v.len;
    }
    if (a.window) {
        const int64_t lo = at + first - a.window + 1;
        r.lo = lo < 0 ? 0 : lo < v.len ? (int)lo & ~31 : v.len;
    }
    return r;
}

// where 16 tokens of a sequence lie: their rows in the pools of one key head, and whether there is such a page
struct Half {
    int64_t code, scale;  // bytes, words
    bool ok;
};
__device__ __forceinline__ Half half_at(const KvAttentionArgs& a, const int* table, int h, int token)
{
    const int col = token >> a.c.page_shift;
    const int page = col < a.s.table_pages ? table[col] : -1;
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

template <int D, int G>
__device__ __forceinline__ void load_step(Step<D, G>& x, const KvAttentionArgs& a, const Half (&half)[2], int r, int j)
{
    constexpr int W = D / 8, GR = D / G;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t* k = (const uint32_t*)(a.c.k + half[h].code) + r * W + j * (W / 4);
        if constexpr (Shape<D>::KW == 2) {
            const u32x2 t = *(const u32x2*)k;
            x.k[h][0] = t[0], x.k[h][1] = t[1];
        } else {
#pragma unroll
            for (int i = 0; i < Shape<D>::KW; i += 4) {
                const u32x4 t = *(const u32x4*)(k + i);
#pragma unroll
                for (int e = 0; e < 4; ++e) x.k[h][i + e] = t[e];
            }
        }
        const uint32_t* ks = a.c.k_scale + half[h].scale + r * GR + j * (D / 4) / G;
#pragma unroll
        for (int i = 0; i < Step<D, G>::KS; ++i) x.ks[h][i] = ks[i];
        const uint32_t* v = (const uint32_t*)(a.c.v + half[h].code) + 4 * j * W + (D == 64 ? r >> 1 : r * Shape<D>::VW);
        const uint32_t* vs = a.c.v_scale + half[h].scale + 4 * j * GR + r * (D / 16) / G;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (Shape<D>::VW == 2) {
                const u32x2 t = *(const u32x2*)(v + i * W);
                x.v[4 * h + i][0] = t[0], x.v[4 * h + i][1] = t[1];
            } else {
                x.v[4 * h + i][0] = v[i * W];
            }
            x.vs[4 * h + i] = vs[i * GR];
        }
    }
}

// the scores of 16 rows against 32 tokens: s[h][i] is row r, token 16 h + 4 j + i
template <int D, int G>
__device__ __forceinline__ void scores(v4f (&s)[2], const uint32_t (&k)[2][Shape<D>::KW],
                                       const uint32_t (&ks)[2][Step<D, G>::KS], const h8 (&q)[Shape<D>::STEPS])
{
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        s[h] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < Shape<D>::STEPS; ++i) {
            const uint32_t w = ks[h][i * Step<D, G>::KS / Shape<D>::STEPS];
            const h8 f = key_fragment(k[h][i], low_pair(w, w), high_pair(w, w));
            s[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, q[i], s[h], 0, 0, 0);
        }
    }
}

// O^T += V^T P^T of 32 tokens: tile n's rows are the channels r (D / 16) + n
template <int D, int G>
__device__ __forceinline__ void add_values(v4f (&acc)[Shape<D>::TILES], const Step<D, G>& x, h8 p, int r)
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
            uint32_t y[4];  // a pair of tokens: 4 channels each
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const uint32_t sel = D == 64 ? (r & 1 ? 0x07060302u : 0x05040100u) : half ? 0x07060302u : 0x05040100u;
                y[u] = __builtin_amdgcn_perm(x.v[2 * u + 1][w], x.v[2 * u][w], sel);
            }
            h8 f[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const uint32_t y8 = y[u] >> 8;
                const h2 c0 = __builtin_elementwise_fma(codes_of<0>(y[u]), s[u], o[u]);
                const h2 c1 = __builtin_elementwise_fma(codes_of<1>(y[u]), s[u], o[u]);
                const h2 c2 = __builtin_elementwise_fma(codes_of<0>(y8), s[u], o[u]);
                const h2 c3 = __builtin_elementwise_fma(codes_of<1>(y8), s[u], o[u]);
                f[0][2 * u] = c0[0], f[0][2 * u + 1] = c0[1];
                f[1][2 * u] = c1[0], f[1][2 * u + 1] = c1[1];
                f[2][2 * u] = c2[0], f[2][2 * u + 1] = c2[1];
                f[3][2 * u] = c3[0], f[3][2 * u + 1] = c3[1];
            }
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                v4f& t = acc[w * 8 + half * 4 + n];
                t = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[n], p, t, 0, 0, 0);
            }
        }
    }
}

// Row r of a tile as fragments (8 channels of lane j's quarter a step, in K's order), scaled by a power of two that brings its
// largest magnitude to [2^14, 2^15): f16 then keeps every bit that matters (39 powers of two below the largest).  Returns what
// a score is multiplied by to undo that; rows that are not there are zeros.
template <int D>
__device__ __forceinline__ float load_row(h8 (&q)[Shape<D>::STEPS], const uint16_t* row, bool there, bool bf16, int j)
{
    u32x4 raw[Shape<D>::STEPS];
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < Shape<D>::STEPS; ++i) {
        raw[i] = there ? *(const u32x4_any*)(row + j * (D / 4) + 8 * i) : (u32x4){0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint16_t lo = (uint16_t)raw[i][e], hi = (uint16_t)(raw[i][e] >> 16);
            top = __builtin_fmaxf(top, __builtin_fabsf(bf16 ? bf16_to_f32(lo) : f16_to_f32(lo)));
            top = __builtin_fmaxf(top, __builtin_fabsf(bf16 ? bf16_to_f32(hi) : f16_to_f32(hi)));
        }
    }
    top = __builtin_fmaxf(top, __shfl_xor(top, 16, 64));
    top = __builtin_fmaxf(top, __shfl_xor(top, 32, 64));
    int e = (int)(__float_as_uint(top) >> 23) - 127;
    e = e < -100 ? -100 : e > 127 ? 14 : e;  // (0 and tiny rows; infinite ones pass as they are)
    const float up = __uint_as_float((uint32_t)(127 + 14 - e) << 23);
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
    return __uint_as_float((uint32_t)(127 - 14 + e) << 23);
}

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float MARGIN = 15.0f, BELOW = 8.0f;  // a weight is exp2(score - reference), 2^8 at the maximum, 2^15 at most

// Four waves share a range of a sequence's tokens, a wave every fourth step of 32; their sums meet in LDS.  One range: the
// result.  Several: each leaves its sums, and kv_join_kernel adds them.
template <int D, int G>
__global__ __launch_bounds__(256) void kv_attention_kernel(KvAttentionArgs a)
{
    constexpr int TILES = Shape<D>::TILES, MD = Shape<D>::MD;
    __shared__ float merge[4][16][MD + 4];
    __shared__ float stat[2][4][16];
    uint32_t id = blockIdx.x;
    const int split = (int)(id % a.splits);
    id /= a.splits;
    const int h = (int)(id % a.c.kv_heads);
    id /= a.c.kv_heads;
    const int tile = (int)(id % a.tiles);
    const int64_t b = a.first + id / a.tiles;
    const View v = view_of(a, b);
    if (tile * 16 >= v.rows * a.ratio) return;
    const Range range = range_of(a, v, tile);
    const int64_t begin64 = range.lo + (int64_t)split * a.chunk;
    if (split > 0 && begin64 >= range.hi) return;
    const int begin = (int)(begin64 < range.hi ? begin64 : range.hi);
    const int end = range.hi - begin > a.chunk ? begin + a.chunk : range.hi;
    const int lane = threadIdx.x & 63, r = lane & 15, j = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int* table = a.s.table + b * a.s.ld_table;

    const int row = tile * 16 + r, query = row / a.ratio;
    const bool there = query < v.rows;
    h8 q[Shape<D>::STEPS];
    const uint16_t* from = (const uint16_t*)a.q + (int64_t)(v.start + (there ? query : 0)) * a.ld_q +
                           (int64_t)(h * a.ratio + row % a.ratio) * a.hd_q;
    const float undo = load_row<D>(q, from, there, a.type == DT_BF16, j) * (a.scale * LOG2E);
    // the row's tokens [low, limit); rows that are not there take those of the last query
    const int mine = there ? query : v.rows - 1;
    const int64_t at = (int64_t)v.len - v.n + mine;
    const int limit = a.causal ? (at + 1 < 0 ? 0 : at + 1 < v.len ? (int)(at + 1) : v.len) : v.len;
    const int low = a.window ? (at - a.window + 1 < 0 ? 0 : at - a.window + 1 < v.len ? (int)(at - a.window + 1) : v.len) : 0;
    int all_limit = limit, all_low = low;  // what every row sees
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) {
        const int x = __shfl_xor(all_limit, off, 64), y = __shfl_xor(all_low, off, 64);
        all_limit = all_limit < x ? all_limit : x;
        all_low = all_low > y ? all_low : y;
    }
    all_limit = __builtin_amdgcn_readfirstlane(all_limit);
    all_low = __builtin_amdgcn_readfirstlane(all_low);

    v4f acc[TILES];
#pragma unroll
    for (int n = 0; n < TILES; ++n) acc[n] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
    float ref = -__builtin_inff(), base = 0.0f, sum = 0.0f;  // reference (none yet) and what is subtracted; sum of weights

    Step<D, G> now, next;
    Half here[2], there_half[2];
    int t = begin + 32 * wave;
    if (t < end) {
        here[0] = half_at(a, table, h, t);
        here[1] = half_at(a, table, h, t + 16);
        load_step<D, G>(now, a, here, r, j);
    }
    for (; t < end; t += 128) {
        if (t + 128 < end) {
            there_half[0] = half_at(a, table, h, t + 128);
            there_half[1] = half_at(a, table, h, t + 144);
            load_step<D, G>(next, a, there_half, r, j);
        }
        v4f s[2];
        scores<D, G>(s, now.k, now.ks, q);
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = s[e >> 2][e & 3] * undo;
        if (t < all_low || t + 32 > all_limit || t + 32 > end || !here[0].ok || !here[1].ok) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int token = t + (e >> 2) * 16 + 4 * j + (e & 3);
                const bool seen = token >= low && token < limit && token < end && here[e >> 2].ok;
                x[e] = seen ? x[e] : -__builtin_inff();
                // (what lies behind the sequence may be anything: its values become 0)
                now.vs[e] = token < end && here[e >> 2].ok ? now.vs[e] : 0u;
            }
        }
        float top = x[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) top = __builtin_fmaxf(top, x[e]);
        if (__ballot(top > ref + MARGIN)) {
            top = __builtin_fmaxf(top, __shfl_xor(top, 16, 64));
            top = __builtin_fmaxf(top, __shfl_xor(top, 32, 64));
            const float to = __builtin_fmaxf(ref, top - BELOW);
            const float f = to == ref ? 1.0f : __builtin_amdgcn_exp2f(ref - to);
            sum *= f;
#pragma unroll
            for (int n = 0; n < TILES; ++n) acc[n] *= f;
            ref = to;
            base = to == -__builtin_inff() ? 0.0f : to;
        }
        h8 p;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float w = __builtin_amdgcn_exp2f(x[e] - base);
            sum += w;
            p[e] = (_Float16)w;
        }
        add_values<D, G>(acc, now, p, r);
        now = next;
        here[0] = there_half[0];
        here[1] = there_half[1];
    }
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);

    // the waves' sums
    if (j == 0) stat[0][wave][r] = ref, stat[1][wave][r] = sum;
    __syncthreads();
    float top = -__builtin_inff();
#pragma unroll
    for (int w = 0; w < 4; ++w) top = __builtin_fmaxf(top, stat[0][w][r]);
    const float f = ref == -__builtin_inff() && sum == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(base - top);
    constexpr int EACH = 8, PER = MD / EACH;  // channels of a thread, threads of a row
    const int orow = threadIdx.x / PER, och = threadIdx.x % PER * EACH;
    float total = 0.0f, most = -__builtin_inff();
    if (orow < 16) {
#pragma unroll
        for (int w = 0; w < 4; ++w) most = __builtin_fmaxf(most, stat[0][w][orow]);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float c = stat[0][w][orow], l = stat[1][w][orow];
            total += l == 0.0f ? 0.0f : l * __builtin_amdgcn_exp2f((c == -__builtin_inff() ? 0.0f : c) - most);
        }
    }
    const int out_row = tile * 16 + orow, out_query = out_row / a.ratio;
    const bool writes = orow < 16 && out_query < v.rows;
    const int head = h * a.ratio + out_row % a.ratio;
    const int64_t token = v.start + out_query;
    float* part = a.part;
    if (a.splits > 1 && writes)
        part += ((((b - a.first) * a.tiles + tile) * a.c.kv_heads + h) * (int64_t)a.rows + orow) * a.splits * (D + 2) +
                (int64_t)split * (D + 2);
#pragma unroll
    for (int piece = 0; piece < D / MD; ++piece) {
        // lane (r, j) has channels j (D / 4) .. of row r: 4 runs of TILES
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c0 = j * (D / 4) + i * TILES - piece * MD;
            if (c0 >= 0 && c0 < MD) {
#pragma unroll
                for (int n = 0; n < TILES; ++n) merge[wave][r][c0 + n] = acc[n][i] * f;
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
                u32x4 w;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float lo = o[2 * e] * inv, hi = o[2 * e + 1] * inv;
                    if (a.type == DT_BF16) w[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f2_t){lo, hi}, bf2_t));
                    else w[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f2_t){lo, hi}, h2_t));
                }
                *(u32x4_any*)((uint16_t*)a.out + token * a.ld_out + head * a.hd_out + piece * MD + och) = w;
            }
        }
        if (piece + 1 < D / MD) __syncthreads();
    }
    if (writes && och == 0) {
        if (a.splits > 1) part[D] = most, part[D + 1] = total;
        else if (a.lse) a.lse[token * a.heads + head] = total == 0.0f ? -__builtin_inff() : LN2 * (most + log2f(total));
    }
}

// adds what the ranges of a row left, in their order: a wave per row
template <int D>
__global__ __launch_bounds__(256) void kv_join_kernel(KvAttentionArgs a)
{
    const int lane = threadIdx.x & 63;
    int64_t id = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int orow = (int)(id % a.rows);
    id /= a.rows;
    const int h = (int)(id % a.c.kv_heads);
    id /= a.c.kv_heads;
    const int tile = (int)(id % a.tiles);
    const int64_t b = a.first + id / a.tiles;
    if (b >= a.s.batch) return;
    const View v = view_of(a, b);
    const int row = tile * 16 + orow, query = row / a.ratio;
    if (query >= v.rows) return;
    const Range range = range_of(a, v, tile);
    const int64_t span = (int64_t)range.hi - range.lo;
    const int n = span <= a.chunk ? 1 : (int)((span + a.chunk - 1) / a.chunk);
    const float* part = a.part + ((((b - a.first) * a.tiles + tile) * a.c.kv_heads + h) * (int64_t)a.rows + orow) * a.splits * (D + 2);
    float most = -__builtin_inff();
    for (int s = lane; s < n; s += 64) most = __builtin_fmaxf(most, part[(int64_t)s * (D + 2) + D]);
    most = wave_max(most);
    float total = 0.0f, o[D / 64];
#pragma unroll
    for (int e = 0; e < D / 64; ++e) o[e] = 0.0f;
    for (int s = 0; s < n; ++s) {
        const float* from = part + (int64_t)s * (D + 2);
        const float c = from[D], l = from[D + 1];
        const float f = l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(c - most);
        total += l * f;
#pragma unroll
        for (int e = 0; e < D / 64; ++e) o[e] += from[e * 64 + lane] * f;
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    const int head = h * a.ratio + row % a.ratio;
    const int64_t token = v.start + query;
    uint16_t* out = (uint16_t*)a.out + token * a.ld_out + head * a.hd_out;
#pragma unroll
    for (int e = 0; e < D / 64; ++e) {
        const float x = o[e] * inv;
        out[e * 64 + lane] = a.type == DT_BF16 ? __builtin_bit_cast(uint16_t, (__bf16)x) : f32_to_f16(x);
    }
    if (a.lse && lane == 0) a.lse[token * a.heads + head] = total == 0.0f ? -__builtin_inff() : LN2 * (most + log2f(total));
}

// The weight that 32 tokens per wave received: the scores again, exp(score - lse) summed over the rows of every tile, in order.
template <int D, int G>
__global__ __launch_bounds__(256) void kv_weights_kernel(KvAttentionArgs a, int blocks)
{
    uint32_t id = blockIdx.x;
    const int block = (int)(id % blocks);
    id /= blocks;
    const int h = (int)(id % a.c.kv_heads);
    const int64_t b = a.first + id / a.c.kv_heads;
    const int lane = threadIdx.x & 63, r = lane & 15, j = lane >> 4;
    const int64_t first = ((int64_t)block * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * 32;
    const View v = view_of(a, b);
    float* out = a.w_out + (b * a.c.kv_heads + h) * (int64_t)a.cap;
    const float* in = a.w_in ? a.w_in + (b * a.c.kv_heads + h) * (int64_t)a.cap : nullptr;
    if (first >= v.len) {
        // no tokens here: a row without earlier weights is written to its end
        if (!in && lane < 32 && first + lane < a.cap) out[first + lane] = 0.0f;
        return;
    }
    const int t = (int)first;
    const int* table = a.s.table + b * a.s.ld_table;
    const Half half[2] = {half_at(a, table, h, t), half_at(a, table, h, t + 16)};
    Step<D, G> x;
    load_step<D, G>(x, a, half, r, j);
    float got[8] = {};
    const int tiles = (v.rows * a.ratio + 15) / 16;
    for (int tile = 0; tile < tiles; ++tile) {
        const Range range = range_of(a, v, tile);
        if (t >= range.hi || t + 32 <= range.lo) continue;
        const int row = tile * 16 + r, query = row / a.ratio;
        const bool there = query < v.rows;
        const int64_t token = v.start + (there ? query : 0);
        const int head = h * a.ratio + row % a.ratio;
        h8 q[Shape<D>::STEPS];
        const float undo = load_row<D>(q, (const uint16_t*)a.q + token * a.ld_q + (int64_t)head * a.hd_q, there,
                                       a.type == DT_BF16, j) * (a.scale * LOG2E);
        float lse = there ? a.lse[token * a.heads + head] : __builtin_inff();
        lse = lse == -__builtin_inff() ? __builtin_inff() : lse * LOG2E;  // (a row that saw nothing gives nothing)
        const int64_t at = (int64_t)v.len - v.n + query;
        v4f s[2];
        scores<D, G>(s, x.k, x.ks, q);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int64_t pos = t + (e >> 2) * 16 + 4 * j + (e & 3);
            const bool seen = there && pos < v.len && (!a.causal || pos <= at) && (!a.window || pos > at - a.window) && half[e >> 2].ok;
            const float w = __builtin_amdgcn_exp2f(s[e >> 2][e & 3] * undo - lse);
            got[e] += seen ? w : 0.0f;
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
#pragma unroll
        for (int off = 1; off < 16; off <<= 1) got[e] += __shfl_xor(got[e], off, 64);
        const int64_t pos = first + (e >> 2) * 16 + 4 * j + (e & 3);
        if (r == e && pos < a.cap) {
            if (pos < v.len) out[pos] = in ? __builtin_fmaf(a.decay, in[pos], got[e]) : got[e];
            else if (!in) out[pos] = 0.0f;
        }
    }
}

// tokens that a tile of 16 rows can see at most
int64_t widest(const KvAttentionArgs& a)
{
    const int64_t all = (int64_t)a.s.table_pages << a.c.page_shift;
    const int64_t seen = a.window && a.causal ? (int64_t)a.window + 16 / a.ratio + 1 + 31 : all;
    return seen < all ? seen : all;
}

void plan(KvAttentionArgs& a, bool room)
{
    a.ratio = a.heads / a.c.kv_heads;
    const int64_t rows = (int64_t)a.max_q * a.ratio;
    a.tiles = (int)((rows + 15) / 16);
    a.rows = (int)(rows < 16 ? rows : 16);
    const int64_t span = widest(a);
    const int64_t groups = (int64_t)a.s.batch * a.tiles * a.c.kv_heads;
    int64_t splits = 1;
    if (room && groups < 1024) {
        splits = 1024 / groups;
        const int64_t most = (span + 255) / 256;
        splits = splits < most ? splits : most;
    }
    if (splits < 1) splits = 1;
    const int64_t chunk = ((span + splits - 1) / splits + 127) / 128 * 128;
    a.chunk = (int)(chunk < 128 ? 128 : chunk);
    a.splits = (int)((span + a.chunk - 1) / a.chunk);
    if (a.splits < 1) a.splits = 1;
}

size_t part_bytes(const KvAttentionArgs& a)
{
    if (a.splits < 2) return 0;
    return (size_t)a.s.batch * a.tiles * a.c.kv_heads * a.rows * a.splits * (a.c.d + 2) * sizeof(float);
}

template <int D, int G>
hipError_t run_attention(KvAttentionArgs a, hipStream_t st)
{
    const int64_t per = (int64_t)a.tiles * a.c.kv_heads * a.splits;  // workgroups of a sequence
    const int64_t most = ((int64_t)1 << 23) / per;                   // sequences of a launch: below 2^31 threads
    float* part = a.part;
    for (int64_t at = 0; at < a.s.batch; at += most) {
        const int64_t n = a.s.batch - at < most ? a.s.batch - at : most;
        a.first = (int)at;
        KvAttentionArgs now = a;
        now.s.batch = (int)(at + n);
        now.part = part + at * a.tiles * a.c.kv_heads * a.rows * a.splits * (a.c.d + 2);
        launch_k(kv_attention_kernel<D, G>, dim3((uint32_t)(n * per)), dim3(256), 0, st, now);
        hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        if (a.splits > 1) {
            const int64_t rows = n * a.tiles * a.c.kv_heads * a.rows;
            hipLaunchKernelGGL(kv_join_kernel<D>, dim3((uint32_t)((rows + 3) / 4)), dim3(256), 0, st, now);
            e = hipGetLastError();
            if (e != hipSuccess) return e;
        }
    }
    return hipSuccess;
}

template <int D, int G>
hipError_t run_weights(KvAttentionArgs a, hipStream_t st)
{
    const int64_t blocks = ((int64_t)a.cap + 127) / 128, per = blocks * a.c.kv_heads;
    const int64_t most = ((int64_t)1 << 23) / per;
    for (int64_t at = 0; at < a.s.batch; at += most) {
        const int64_t n = a.s.batch - at < most ? a.s.batch - at : most;
        a.first = (int)at;
        launch_k(kv_weights_kernel<D, G>, dim3((uint32_t)(n * per)), dim3(256), 0, st, a, (int)blocks);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
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
    plan(a, true);
    return part_bytes(a);
}

hipError_t launch_kv_attention(KvAttentionArgs a, void* ws, size_t ws_bytes, hipStream_t st)
{
    plan(a, ws != nullptr);
    if (part_bytes(a) > ws_bytes) plan(a, false);
    a.part = (float*)ws;
    KV_SHAPES(run_attention)
}

hipError_t launch_kv_weights(KvAttentionArgs a, hipStream_t st)
{
    plan(a, false);
    KV_SHAPES(run_weights)
}

}  // namespace ascq
