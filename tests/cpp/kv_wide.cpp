// Evictions whose page tables have room for as many tokens as a call takes, over few and many key heads: grids of fewer than 2^32
// threads and 65536 rows of blocks, every sequence once, counts inside the workspace.  Exit status 0 = they are.
#include <cstdio>

#include "launches.h"

int main()
{
    int failures = 0;
    void* p = (void*)0x100000000000;
    first_argument() = sizeof(ascq::KvEvictArgs);
    for (int pages : {1 << 16, 1 << 18, 1 << 20})
        for (int kv : {1, 15, 16, 31, 32, 33, 200, 1024})
            for (int batch : {1, 2, 9})
                for (int room = 0; room < 2; ++room) {
                    const ascq_kv_cache c{p, p, p, p, 1 << 20, 0, 0, kv, 1024, 64, 64};
                    const ascq_kv_sequences s{(int32_t*)p, (int32_t*)p, nullptr, 0, batch, pages};
                    const ascq_kv_evict_param ep{(int64_t)pages << 10, 1000, 0, 1000, 16, 1};
                    size_t bytes = 0;
                    bool good = ascq_kv_evict_workspace_size(&c, &s, &bytes) == ASCQ_OK;
                    launches().clear();
                    good &= ascq_kv_evict((int32_t*)p, (int32_t*)p + 1, (float*)p, (float*)p + 8, (int32_t*)0x300000000000, &c, &s, &ep,
                                          room ? p : nullptr, room ? bytes : 0, nullptr) == ASCQ_OK;
                    int64_t selected = 0, moved = 0;
                    for (const Launch& l : launches()) {
                        const auto a = l.args<ascq::KvEvictArgs>();
                        good &= l.threads() < 1ull << 32 && l.grid.x > 0 && l.grid.y > 0 && l.grid.y < 65536;
                        if (l.is("part_kernel")) good &= room && l.grid.x / a.parts * (5122 * (size_t)a.parts + 4) * 4 <= bytes;
                        if (l.is("select_kernel") || l.is("part_kernelILi3")) {
                            good &= a.first == selected;
                            selected += l.grid.x / (kv * a.parts);
                        } else if (l.is("move_kernel")) {
                            good &= a.first == moved;
                            moved += l.grid.y / kv;
                        }
                    }
                    if (good && selected == batch && moved == batch) continue;
                    std::printf("pages %d heads %d batch %d room %d\n", pages, kv, batch, room);
                    ++failures;
                }
    std::printf("%d failure(s)\n", failures);
    return failures != 0;
}
