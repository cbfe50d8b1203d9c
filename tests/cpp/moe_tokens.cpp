// The launches of the routing's gradient and of the rows' movement cover the tokens of a call once each, in grids of fewer than
// 2^32 threads.  Exit status 0 = they do.
#include <cstdio>

#include "launches.h"

static int failures = 0;

// `unit` threads per token (or item) and `all` of them; f: the first and the last + 1 that a launch covers
template <class F>
static void covered(const char* what, int64_t n, int64_t all, ascq_status status, F f)
{
    int64_t at = 0;
    bool bad = status != ASCQ_OK;
    for (const Launch& l : launches()) {
        int64_t first = 0, end = 0;
        f(l, first, end);
        bad |= l.threads() >= 1ull << 32 || first != at || end < first;
        at = end;
    }
    if (bad || at < all) {
        std::printf("%s n %ld of %ld: status %d, %zu launches, %ld covered\n", what, (long)n, (long)all, status, launches().size(),
                    (long)at);
        ++failures;
    }
}

int main()
{
    void *p = (void*)0x100000000000, *q = (void*)0x200000000000, *r = (void*)0x10000000;
    for (int64_t t : {(int64_t)1, (int64_t)5, (int64_t)1 << 20, ((int64_t)1 << 24) + 1, (int64_t)1 << 25, ((int64_t)1 << 26) + 3,
                      (int64_t)1 << 30, (int64_t)INT32_MAX}) {
        for (int64_t n : {1, 8, 600, 4096, 100000}) {
            const int k = t > 1 << 27 ? 1 : 2;
            ascq_rows_param rp{t, n, 0, ASCQ_DT_F16, k};
            first_argument() = sizeof(ascq::MoeRowsArgs);
            second_argument() = 4;
            auto tokens = [&](const Launch& l, int64_t& first, int64_t& end) {
                const auto a = l.args<ascq::MoeRowsArgs>();
                first = a.first;
                end = first + (int64_t)l.grid.x * 4 / l.second;  // (waves of a token)
                if (end > t) end = t;
                if (a.T != t || a.out != p) end = -1;
            };
            launches().clear();
            ascq_status s = ascq_moe_dispatch(p, nullptr, q, nullptr, (int32_t*)r, (int32_t*)r, &rp, nullptr);
            covered("dispatch", n, t, s, tokens);
            launches().clear();
            s = ascq_moe_combine(p, q, (int32_t*)r, (float*)r, nullptr, &rp, nullptr);
            covered("combine", n, t, s, tokens);
            launches().clear();
            s = ascq_moe_combine_grad((float*)r, p, q, q, (int32_t*)r, (int32_t*)r, (float*)r, &rp, nullptr);
            const int64_t groups = (k + (t * k <= 1024 ? 1 : 4) - 1) / (t * k <= 1024 ? 1 : 4), items = t * groups;
            covered("combine_grad", n, items, s, [&](const Launch& l, int64_t& first, int64_t& end) {
                const auto a = l.args<ascq::MoeRowsArgs>();
                first = a.first;
                end = first + (l.is("Li1EEEv") ? (int64_t)l.grid.x * 4 : (int64_t)l.grid.x);
                if (end > items) end = items;
                if (a.T != t || a.out != p || (!l.is("Li1EEEv") && !l.is("Li4EEEv"))) end = -1;
            });
        }
        first_argument() = sizeof(ascq::MoeRouteGradArgs);
        second_argument() = 0;
        for (int64_t e : {8, 16, 64, 256, 257, 1024}) {
            const int k = 1;
            ascq_route_param gp{t, e, e + 1, ASCQ_DT_F16, k, 1};
            launches().clear();
            const ascq_status s = ascq_moe_route_grad(p, e + 3, q, (float*)r, (int32_t*)r, (int64_t*)r, (int64_t*)r, (float*)r,
                                                      (float*)r, &gp, nullptr);
            int lanes = 1;
            while (lanes * 8 < e && lanes < 64) lanes *= 2;
            covered("route_grad", e, t, s, [&](const Launch& l, int64_t& first, int64_t& end) {
                const auto a = l.args<ascq::MoeRouteGradArgs>();
                first = ((uint8_t*)a.grad_logits - (uint8_t*)p) / (2 * (e + 3));
                end = first + a.T;
                const bool whole = (int64_t)l.grid.x * (256 / lanes) >= a.T;
                if (!whole || a.logits != (uint8_t*)q + first * 2 * (e + 1) || a.weights != (float*)r + first * k ||
                    a.experts != (int*)r + first * k || a.grad_weights != (float*)r + first * k || a.counts != (int64_t*)r)
                    end = -1;
            });
        }
    }
    std::printf("%d failure(s)\n", failures);
    return failures != 0;
}
