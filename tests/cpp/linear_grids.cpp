// The linear's launches stay below 2^32 threads, and those of its general kernel cover the output's tiles once each.
// Exit status 0 = they do.
#include <cstdio>

#include "launches.h"

int main()
{
    first_argument() = sizeof(ascq::LinearArgs);
    second_argument() = 8;
    int failures = 0, several = 0;
    struct {
        int64_t m, n, k;
    } sizes[] = {{1, 1, 0},        {1000, 1000, 0}, {(1ll << 30) + 70, 1, 0}, {INT32_MAX, 64, 0}, {1, INT32_MAX, 0}, {1 << 17, 1 << 19, 0},
                 {INT32_MAX, 3, 5}, {64, INT32_MAX, 1}};
    for (const auto& z : sizes)
        for (int fp8 = 0; fp8 < 2; ++fp8)
            for (int trans = 0; trans < 2; ++trans) {
                ascq_linear_param p{};
                p.m = z.m, p.n = z.n, p.k = z.k, p.w_trans = trans;
                p.operand_type = fp8 ? ASCQ_DT_FP8_E4M3 : ASCQ_DT_INT8;
                p.out_type = ASCQ_DT_F16;
                void* v = (void*)0x40000000;
                launches().clear();
                const ascq_status s = ascq_quant_linear((void*)0x100000000000, (void*)0x200000000000, (float*)v,
                                                        (void*)0x300000000000, (float*)v, nullptr, nullptr, &p, nullptr, 0, nullptr);
                bool bad = s != ASCQ_OK || launches().empty();
                int64_t at = 0, all = 0;
                uint8_t* y = nullptr;
                for (const Launch& l : launches()) {
                    bad |= l.threads() >= 1ull << 32;
                    if (!l.is("linear_any_kernel")) continue;
                    const auto a = l.args<ascq::LinearArgs>();
                    if (a.y != y) {  // (the next piece of the rows or channels)
                        bad |= at != all;
                        y = (uint8_t*)a.y;
                        at = 0;
                        all = (a.M + 63) / 64 * ((a.N + 63) / 64);
                    }
                    bad |= l.second != at;
                    several += at > 0;
                    at += l.grid.x;
                }
                if (bad || at != all) {
                    std::printf("m %ld n %ld k %ld fp8 %d w_trans %d: status %d, %zu launches\n", (long)z.m, (long)z.n, (long)z.k,
                                fp8, trans, s, launches().size());
                    ++failures;
                }
            }
    std::printf("%d failure(s), %d further launches\n", failures, several);
    return failures != 0 || several == 0;
}
