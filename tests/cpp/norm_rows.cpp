// The norm's launches cover the rows of a call once each, in grids of fewer than 2^32 threads.  Exit status 0 = they do.
#include <cstdio>

#include "launches.h"

int main()
{
    first_argument() = sizeof(ascq::NormQuantArgs);
    int failures = 0;
    for (int type : {ASCQ_DT_F16, ASCQ_DT_F32})
        for (int64_t n : {1, 8, 600, 1032, 5000, 16000, 40000, 100000})
            for (int64_t m : {(int64_t)1, (int64_t)1 << 21, ((int64_t)1 << 21) + 1, (int64_t)1 << 24, ((int64_t)1 << 26) + 3,
                              (int64_t)INT32_MAX})
                for (int full = 0; full < 2; ++full) {
                    const int64_t es = type == ASCQ_DT_F32 ? 4 : 2, ldx = n + 8, ldr = n + 16, ldh = n + 24;
                    ascq_norm_quant_param p{m, n, ldx, full ? ldr : 0, full ? ldh : 0, type, ASCQ_DT_INT8, 1e-6f};
                    uint8_t *q = (uint8_t*)0x100000000000, *x = (uint8_t*)0x200000000000, *r = (uint8_t*)0x400000000000,
                            *h = (uint8_t*)0x800000000000, *o = (uint8_t*)0x1000000000000, *s = (uint8_t*)0x10000000;
                    if (!full) r = h = o = nullptr;
                    launches().clear();
                    const ascq_status got = ascq_add_rms_norm_quant(q, (float*)s, h, o, x, r, (void*)0x1000, &p, nullptr);
                    int64_t at = 0;
                    bool bad = got != ASCQ_OK;
                    for (const Launch& l : launches()) {
                        const auto a = l.args<ascq::NormQuantArgs>();
                        bad |= l.threads() >= 1ull << 32 || l.grid.x != a.m || a.n != n || a.ldx != ldx;
                        bad |= a.q != q + at * n || (uint8_t*)a.scale_out != s + at * 4 || a.x != x + at * ldx * es;
                        bad |= a.residual != (full ? r + at * ldr * es : nullptr) || a.h_out != (full ? h + at * ldh * es : nullptr);
                        bad |= a.norm_out != (full ? o + at * n * es : nullptr);
                        at += a.m;
                    }
                    if (bad || at != m) {
                        std::printf("type %d n %ld m %ld: status %d, %zu launches, %ld rows\n", type, (long)n, (long)m, got,
                                    launches().size(), (long)at);
                        ++failures;
                    }
                }
    std::printf("%d failure(s)\n", failures);
    return failures != 0;
}
