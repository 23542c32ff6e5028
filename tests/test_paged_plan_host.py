"""How attention over a paged cache is dealt to the SMs, and what of a workspace belongs to whom."""
from conftest import compile_and_run

CHECK = r"""
#include "paged_plan.h"
#include <cstdio>
#include <cstdlib>
#include <random>
using namespace tb;

#define CHECK(c) do { if (!(c)) { printf("line %d: %s (seqs %d heads %d group %d hd %d e4m3 %d rows %d max_q %d max_kv %d sms %d)\n", __LINE__, #c, \
    seqs, heads, group, hd, (int)e4m3, rows, max_q, max_kv, sms); return 1; } } while (0)

int main() {
    std::mt19937 rng(7);
    auto log_int = [&](int lo, int hi) {
        const double f = (double)rng() / 4294967296.0;
        int x = lo;
        while (x < hi && (double)rng() / 4294967296.0 < 0.85) x = x * 2 + (int)(rng() % 2);
        return x > hi ? lo + (int)(f * (hi - lo)) : x;
    };
    for (int t = 0; t < 20000; ++t) {
        const int seqs = log_int(1, 65535), heads = log_int(1, 64), group = 1 + (int)(rng() % 128), sms = t % 3 ? 148 : log_int(1, 200);
        const bool e4m3 = rng() % 2;
        const int hd = e4m3 ? 16 * (1 + (int)(rng() % 8)) : 8 * (1 + (int)(rng() % 16));
        const int rows = log_int(1, 1 << 20), max_q = 1 + (int)(rng() % (unsigned)log_int(1, rows)), max_kv = log_int(1, 1 << 22);
        const PagedPlan p = paged_plan(seqs, heads, group, hd, e4m3, rows, max_q, max_kv, sms);
        const int wide = hd > 64 ? 2 : 1;
        CHECK(p.grid >= 1 && p.grid <= paged_per_sm(wide, e4m3) * sms && p.grid <= paged_counters(sms));
        CHECK(p.rows_bytes % 16 == 0 && p.workspace >= 0 && p.workspace <= p.room);
        CHECK(p.workspace == 0 || p.rows_bytes >= paged_counters(sms) * 4);
        CHECK(p.whole == (max_kv <= PA_WHOLE) && (!p.whole || p.grid <= (long long)seqs * heads));
        if (!p.whole) CHECK(p.rows_bytes >= paged_counters(sms) * 4 + 2LL * p.grid * PA_ROWS * (hd + 2) * 4);
        // a batch within the bounds has no more tiles than there is room for units
        if (p.most_units > 0) {
            CHECK(p.most_units % 4 == 0 && p.most_pieces > 0 && p.most_pieces <= p.most_units && p.most_units <= (long long)heads * PL_TILES + 1024);
            for (int k = 0; k < 4; ++k) {
                long long left = rows, tiles = 0;
                const int tokens = PT_ROWS / group, least = PA_ROWS / group + 1;
                for (int s = 0; s < seqs && left > 0; ++s) {
                    const int n = (int)std::min<long long>(left, k == 0 ? least : k == 1 ? max_q : 1 + (int)(rng() % (unsigned)max_q));
                    if (n > max_q) break;
                    left -= n;
                    if (n * group > PA_ROWS) tiles += (n + tokens - 1) / tokens;
                }
                CHECK(tiles * heads <= p.most_units);
            }
        }
        // smaller bounds need no more than the room
        for (int k = 0; k < 8; ++k) {
            const int r = 1 + (int)(rng() % (unsigned)rows), q = 1 + (int)(rng() % (unsigned)std::min(r, max_q)), v = 1 + (int)(rng() % (unsigned)(k % 2 ? max_kv : std::min(max_kv, 700)));
            const PagedPlan x = paged_plan(1 + (int)(rng() % (unsigned)seqs), heads, group, hd, e4m3, r, q, v, sms);
            CHECK(x.workspace <= p.room && x.room <= p.room);
        }
    }
    puts("ok");
    return 0;
}
"""


def test_plans_fit_their_workspace_and_smaller_batches_need_no_more(tmp_path):
    assert compile_and_run(tmp_path, CHECK).strip() == "ok"
