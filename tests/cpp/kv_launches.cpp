// The launches of the paged cache's operators cover the tokens, sequences and rows of a call once each, in grids of fewer than 2^32
// threads and less than 65536 rows of blocks, and the workspace covers what the launches write.  Exit status 0 = they do.
#include <cstdio>

#include "launches.h"

static int failures = 0;

static void expect(bool good, const char* what, long a, long b, long c)
{
    if (good) return;
    std::printf("%s: %ld %ld %ld\n", what, a, b, c);
    ++failures;
}

static bool fits(const Launch& l)
{
    return l.threads() < 1ull << 32 && l.grid.x > 0 && l.grid.y > 0 && l.grid.y < 65536 && l.grid.z > 0 && l.grid.z < 65536;
}

int main()
{
    void* p = (void*)0x100000000000;
    for (int64_t t : {(int64_t)1, (int64_t)777, (int64_t)1 << 20, ((int64_t)1 << 24) + 1, (int64_t)INT32_MAX})
        for (int kv : {1, 8, 1024}) {
            const ascq_kv_cache c{p, p, p, p, 1 << 20, 0, 0, kv, 64, 128, 32};
            const ascq_kv_append_param ap{t, 0, 0, 0, 0, ASCQ_DT_F16};
            first_argument() = sizeof(ascq::KvAppendArgs);
            launches().clear();
            bool good = ascq_kv_append(&c, p, p, (int64_t*)p, &ap, nullptr) == ASCQ_OK;
            int64_t at = 0;
            for (const Launch& l : launches()) {
                const auto a = l.args<ascq::KvAppendArgs>();
                good &= fits(l) && a.first == at && l.threads() >= (uint64_t)(a.T - a.first) * kv * 16;
                at = a.T;
            }
            expect(good && at == t, "append", t, kv, at);
        }
    first_argument() = sizeof(ascq::KvAttentionArgs);
    for (int batch : {1, 3, 64, 5000, 1 << 20, INT32_MAX})
        for (int64_t queries : {(int64_t)1, (int64_t)5, (int64_t)1000, (int64_t)300000})
            for (int kv : {1, 8, 96})
                for (int ratio : {1, 4, 20})
                    for (int pages : {0, 1, 100, 1 << 20}) {
                        const ascq_kv_cache c{p, p, p, p, 1 << 20, 0, 0, kv, 64, 128, 32};
                        const ascq_kv_sequences s{(int32_t*)p, (int32_t*)p, (int32_t*)p, 0, batch, pages};
                        const ascq_kv_attention_param ap{INT32_MAX, queries, 0, 0, 0, 0, 0, ASCQ_DT_F16, kv * ratio, 1, 1.0f};
                        const int64_t most_tiles = (queries * ratio + 15) / 16;
                        if (most_tiles * kv > 1 << 23 || (double)batch * most_tiles * kv > 1e10) continue;  // (refused; thousands of launches)
                        size_t bytes = 0;
                        expect(ascq_kv_attention_workspace_size(&c, &s, &ap, &bytes) == ASCQ_OK, "size", batch, queries, kv);
                        for (int room = 0; room < 2; ++room) {
                            launches().clear();
                            bool good = ascq_kv_attention(p, nullptr, p, &c, &s, &ap, room ? p : nullptr, room ? bytes : 0, nullptr) == ASCQ_OK;
                            int64_t at = 0, joined = 0;
                            for (const Launch& l : launches()) {
                                const auto a = l.args<ascq::KvAttentionArgs>();
                                const int64_t all = queries * ratio, tiles = a.tiles, rows = all < a.tile_rows ? all : a.tile_rows;
                                good &= fits(l) && a.ratio == ratio && tiles * a.tile_rows >= all && (tiles - 1) * a.tile_rows < all;
                                const int64_t groups = (int64_t)(a.s.batch - a.first) * tiles * kv;
                                if (l.is("kv_join")) {
                                    good &= a.first == joined && l.grid.x * (l.is("Li1EEE") ? 4ull : 1ull) >= (uint64_t)groups * rows;
                                    joined = a.s.batch;
                                } else {
                                    good &= a.first == at && l.grid.x == (uint64_t)groups * a.splits;
                                    good &= (int64_t)a.splits * a.chunk >= (int64_t)pages * 64;
                                    at = a.s.batch;
                                }
                                if (a.splits > 1) {
                                    const uint64_t end = ((uint8_t*)a.part - (uint8_t*)p) + (uint64_t)groups * rows * a.splits * 130 * 4;
                                    good &= room && end <= bytes;
                                }
                            }
                            expect(good && at == batch && (joined == 0 || joined == batch), "attention", batch, queries, at);
                        }
                        if ((double)batch * kv > 1e9) continue;
                        launches().clear();
                        const int64_t cap = pages * 64 + 1;
                        bool good = ascq_kv_weights((float*)p, nullptr, cap, 1.0f, p, (float*)p, &c, &s, &ap, nullptr) == ASCQ_OK;
                        int64_t at = 0;
                        for (const Launch& l : launches()) {
                            const auto a = l.args<ascq::KvAttentionArgs>();
                            good &= fits(l) && a.first == at;
                            const int64_t blocks = (cap + a.chunk - 1) / a.chunk;
                            good &= l.grid.x % (blocks * kv) == 0 && a.chunk > 0 && (int64_t)a.chunk * 4 < 1ll << 31;
                            at += l.grid.x / (blocks * kv);
                        }
                        expect(good && at == batch, "weights", batch, cap, at);
                    }
    first_argument() = sizeof(ascq::KvEvictArgs);
    for (int batch : {1, 100, 70000, 1 << 20})
        for (int kv : {1, 8, 1024})
            for (int keep : {1, 1000, 1 << 20}) {
                const ascq_kv_cache c{p, p, p, p, 1 << 20, 0, 0, kv, 64, 128, 32};
                const ascq_kv_sequences s{(int32_t*)p, (int32_t*)p, nullptr, 0, batch, 1 << 15};
                const ascq_kv_evict_param ep{1 << 21, 1 << 21, 0, keep, 0, 1 << 15};
                size_t bytes = 0;
                expect(ascq_kv_evict_workspace_size(&c, &s, &bytes) == ASCQ_OK && bytes > 0, "evict size", batch, kv, keep);
                for (int room = 0; room < 2; ++room)
                    for (void* into : {(void*)nullptr, (void*)0x300000000000}) {
                        launches().clear();
                        bool good = ascq_kv_evict((int32_t*)p, (int32_t*)p + 1, (float*)p, (float*)p, (int32_t*)into, &c, &s, &ep,
                                                  room ? p : nullptr, room ? bytes : 0, nullptr) == ASCQ_OK;
                        int64_t selected[5] = {}, moved = 0;
                        for (const Launch& l : launches()) {
                            const auto a = l.args<ascq::KvEvictArgs>();
                            good &= fits(l);
                            if (l.is("select")) {
                                const int digit = l.is("part_kernelILi0") ? 1 : l.is("part_kernelILi1") ? 2 : l.is("part_kernelILi2") ? 3
                                                  : l.is("part_kernelILi3") ? 4 : 0;
                                good &= a.first == selected[digit] && l.grid.x % (kv * a.parts) == 0 && (a.parts > 1) == (digit > 0);
                                good &= digit == 0 || (room && l.grid.x * (size_t)(5122 * a.parts + 4) / a.parts * 4 <= bytes &&
                                                       (int64_t)a.parts * 8192 >= (int64_t)s.table_pages * 64);
                                selected[digit] += l.grid.x / (kv * a.parts);
                            } else if (!l.is("weights")) {
                                good &= a.first == moved && l.grid.y % kv == 0 && (into || l.grid.x == 1);
                                moved += l.grid.y / kv;
                            }
                        }
                        for (int i = 0; i < 5; ++i) good &= selected[i] == ((i > 0) == (room > 0) ? batch : 0);
                        expect(good && moved == batch, "evict", batch, selected[room], moved);
                    }
            }
    std::printf("%d failure(s)\n", failures);
    return failures != 0;
}
