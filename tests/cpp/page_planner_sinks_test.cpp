// CPU unit test of the page bookkeeping of windowed models (PagePlanner with
// n_sink >= 0).  Built and run by tests/test_window.py with g++; prints "ok <n>".
//
// At every step, for every token of it, each position that the token sees
// (the window up to its own, and the sinks) has a device page; no page is held
// twice; pages that nothing will see again are released at the latest one step
// later; a step that runs out of pages changes nothing.
#include <cstdio>
#include <cstdlib>
#include <set>
#include <vector>

#include "page_planner.h"

static int g_checks = 0;
#define CHECK(c)                                                              \
    do {                                                                      \
        ++g_checks;                                                           \
        if (!(c)) {                                                           \
            std::fprintf(stderr, "%s:%d: CHECK(%s) failed\n", __FILE__, __LINE__, #c); \
            std::exit(1);                                                     \
        }                                                                     \
    } while (0)

using sfa::PageAction;
using sfa::PagePlanner;

static void walk(int P, int n_ctx, int W, int n_sink, unsigned seed) {
    const int n_seq = 3, win = W < n_ctx ? W : n_ctx;
    const int max_pages = (n_ctx + P - 1) / P;
    const int kept = (win + P - 2) / P + 2 + (n_sink + P - 1) / P;
    const int n_pages = n_seq * (kept < max_pages ? kept : max_pages);
    PagePlanner pl(n_seq, P, n_ctx, W, n_pages, 0, false, seed, true, n_sink);
    std::vector<int> used(n_seq, 0);
    unsigned r = seed * 2654435761u + 1;
    for (int step = 0; step < 400; ++step) {
        int32_t n_tok[3];
        for (int b = 0; b < n_seq; ++b) {
            r = r * 1664525u + 1013904223u;
            const int kind = r >> 29;
            n_tok[b] = kind < 3 ? 1 : kind < 4 ? 0 : (int)((r >> 8) % (unsigned)P) + 1;
            if (used[b] + n_tok[b] > n_ctx) {
                std::vector<PageAction> acts;
                pl.reset(b, &acts);
                used[b] = 0;
            }
        }
        std::vector<PageAction> acts;
        CHECK(pl.plan_step(n_tok, &acts) == 0);  // the pool is large enough for every step
        for (const PageAction &a : acts) CHECK(a.kind == PageAction::kAlloc || a.kind == PageAction::kDrop);
        std::set<int32_t> held;
        int n_held = 0;
        for (int b = 0; b < n_seq; ++b) {
            const int32_t *row = &pl.table()[(size_t)b * max_pages];
            for (int t = used[b]; t < used[b] + n_tok[b]; ++t)
                for (int p = 0; p <= t; ++p)
                    if (p > t - win || p < n_sink) CHECK(row[p / P] >= 0);
            for (int lp = 0; lp < max_pages; ++lp) {
                if (row[lp] < 0) continue;
                CHECK(row[lp] < n_pages && held.insert(row[lp]).second);
                ++n_held;
                // some token of this step may see it, or it holds a sink
                CHECK(lp * P < n_sink || (lp + 1) * P - 1 > used[b] - win);
            }
            used[b] += n_tok[b];
            CHECK((int)pl.store(b).used() == used[b]);
        }
        CHECK(pl.stats().dev_in_use == n_held);
    }
}

int main() {
    for (unsigned s = 1; s <= 4; ++s) {
        walk(64, 1000, 100, 5, s);
        walk(64, 1000, 64, 0, s);
        walk(64, 1000, 1, 1, s);
        walk(64, 1000, 200, 129, s);
        walk(128, 640, 5000, 7, s);
        walk(64, 1000, 63, 5000, s);
    }
    // out of pages: nothing changes
    PagePlanner pl(1, 64, 1000, 128, 2, 0, false, 1, true, 4);
    std::vector<PageAction> acts;
    int32_t n = 64;
    CHECK(pl.plan_step(&n, &acts) == 0 && pl.plan_step(&n, &acts) == 0);
    const auto table = pl.table();
    const size_t had = acts.size();
    CHECK(pl.plan_step(&n, &acts) == 4);
    CHECK(pl.table() == table && acts.size() == had && pl.store(0).used() == 128);
    n = 65;
    CHECK(pl.plan_step(&n, &acts) == 1);
    std::printf("ok %d\n", g_checks);
    return 0;
}
