// The linear's tiles address a w [K, N] with 32-bit offsets and rely on the rows past K lying past its range: they read 0 there.
// For every call that takes them that has to hold -- a product of 32 bits that comes round would reach w again -- and calls of
// ordinary pitches have to take them.  Exit status 0 = it holds.
#include <cstdio>

#include "launches.h"

int main()
{
    first_argument() = sizeof(ascq::LinearArgs);
    int failures = 0, tiles = 0, others = 0;
    for (int fp8 = 0; fp8 < 2; ++fp8)
        for (int64_t k : {1, 2, 3, 7, 14, 15, 16, 17, 33, 100, 128, 500, 4096})
            for (int64_t n : {64, 4096})
                for (int64_t ld : {(int64_t)0, (int64_t)1 << 14, (int64_t)1 << 20, ((int64_t)1 << 24) + 16, ((int64_t)1 << 25) + 64,
                                   (int64_t)1 << 26, (int64_t)1 << 27, (int64_t)1 << 28, ((int64_t)1 << 29) - 4,
                                   ((int64_t)1 << 31) - 8192, (int64_t)1 << 32, ((int64_t)1 << 36) + 16}) {
                    ascq_linear_param p{};
                    p.m = 200, p.n = n, p.k = k, p.ld_x = 8192, p.ld_w = ld;
                    p.operand_type = fp8 ? ASCQ_DT_FP8_E4M3 : ASCQ_DT_INT8;
                    p.out_type = ASCQ_DT_F16;
                    void *x = (void*)0x10000000, *w = (void*)0x200000000, *v = (void*)0x40000000;
                    size_t bytes = 0;
                    if (ascq_quant_linear_workspace_size(x, w, &p, &bytes) != ASCQ_OK) return 1;
                    launches().clear();
                    if (ascq_quant_linear((void*)0x30000000, x, (float*)v, w, (float*)v, nullptr, nullptr, &p,
                                          (void*)0x50000000, bytes, nullptr) != ASCQ_OK)
                        return 1;
                    for (const Launch& l : launches()) {
                        if (!l.is("linear_pipe_kernel")) {
                            others += l.is("linear_any_kernel");
                            continue;
                        }
                        ++tiles;
                        const auto a = l.args<ascq::LinearArgs>();
                        const uint64_t range = (uint64_t)(a.ldw * (a.K - 1) + (a.N + 3) / 4 * 4);
                        // (int8: x's chunks of 16 bytes past K are zeros; fp8: 0 times a NaN would be one)
                        const int64_t end = fp8 ? (a.K + 127) / 128 * 128 : (a.K + 15) / 16 * 16;
                        bool bad = range >= 1ull << 31 || (a.K > 1 && a.ldw >= 1ll << 32);
                        for (int64_t row = a.K; row < end; ++row)
                            for (int64_t col : {(int64_t)0, a.N + 255})
                                bad |= (uint32_t)((uint32_t)row * (uint32_t)a.ldw + (uint32_t)col) < range;
                        if (bad) {
                            std::printf("fp8 %d k %ld n %ld pitch %ld: rows past K come round\n", fp8, (long)k, (long)n, (long)ld);
                            ++failures;
                        }
                    }
                    const bool ordinary = (ld ? ld : n) * ((k + 127) / 128 * 128) < 1ll << 31;
                    if (ordinary && (launches().empty() || launches().back().is("linear_any_kernel"))) {
                        std::printf("fp8 %d k %ld n %ld pitch %ld: not on the tiles\n", fp8, (long)k, (long)n, (long)ld);
                        ++failures;
                    }
                }
    std::printf("%d on tiles, %d on the general kernel, %d failure(s)\n", tiles, others, failures);
    return failures != 0 || tiles == 0 || others == 0;
}
