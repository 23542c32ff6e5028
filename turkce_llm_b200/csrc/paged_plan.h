// How attention over a paged cache is dealt to the SMs: host arithmetic only, no CUDA headers (tests/test_paged_plan_host.py).
#pragma once
#include <algorithm>
#include <cstdint>

namespace tb {

constexpr int PA_ROWS = 16;          // query rows (token, head of the group) of an item: one tensor-core fragment
constexpr int PA_WHOLE = 512;        // up to so many keys an item is one CTA's
constexpr int PA_LEAST = 512;        // keys of a CTA's run, at least

// keys per block of the kernel for few rows (wide: head dimensions in 64s)
constexpr int paged_keys(int wide, bool e4m3) { return wide == 1 && e4m3 ? 128 : 64; }

// CTAs of the kernel for few rows that an SM holds: by their shared memory, a ring of blocks of which 48 KB and more are on their way
constexpr int paged_per_sm(int wide, bool e4m3) { return wide == 1 && e4m3 ? 3 : 2; }

constexpr int PT_ROWS = 128, PT_KEYS = 128;      // query rows and keys of the kernel for longer chunks
// CTAs of that kernel that an SM holds
constexpr int paged_tiles_per_sm(int wide, bool e4m3) { return wide == 1 && !e4m3 ? 2 : 1; }

struct PagedPlan {
    bool whole;                      // few rows: every item is one CTA's
    int grid;                        // few rows: CTAs
    int most_units;                  // longer chunks: room for pieces of tiles; 0: a CTA per tile
    int64_t rows_bytes, workspace;   // bytes of the kernel for few rows (a counter and two results per CTA); of both
};

inline PagedPlan paged_plan(int seqs, int heads, int group, int hd, bool e4m3, int rows, int max_q, int max_kv, int sms) {
    PagedPlan p;
    const int wide = hd > 64 ? 2 : 1;
    const int64_t items = (int64_t)seqs * heads, most = (int64_t)paged_per_sm(wide, e4m3) * sms;
    p.whole = max_kv <= PA_WHOLE;
    const int64_t keys = paged_keys(wide, e4m3), blocks = items * (((int64_t)max_kv + keys - 1) / keys), least = PA_LEAST / keys;
    p.grid = (int)std::max<int64_t>(1, std::min(most, p.whole ? items : (blocks + least - 1) / least));
    // a word per CTA (to a multiple of 16 bytes), then its two results
    p.rows_bytes = p.whole ? 0 : (int64_t)(p.grid + 3) / 4 * 16 + 2LL * p.grid * PA_ROWS * (hd + 2) * 4;
    p.most_units = 0;
    p.workspace = p.rows_bytes;
    if ((int64_t)max_q * group > PA_ROWS) {
        // No more tiles than this many: every sequence that has tiles at all has more than PA_ROWS rows per key head.  Where that is
        // less than two for every CTA that the chip holds, tiles are cut into pieces (up to three for every CTA).
        const int64_t tokens = PT_ROWS / group, least_rows = PA_ROWS / group + 1;
        const int64_t tiles = heads * (rows / tokens + std::min<int64_t>(seqs, rows / least_rows)), slots = (int64_t)paged_tiles_per_sm(wide, e4m3) * sms;
        if (tiles < 2 * slots && max_kv > PT_KEYS) {
            p.most_units = (int)(std::max(slots, tiles) + 3) / 4 * 4;
            // header, then for every unit: a counter, a flag, what it is, and [128] (maximum, sum) and [128][64 wide] float32
            p.workspace += 16 + (int64_t)p.most_units * (4 + 4 + 32 + PT_ROWS * (8 + 64 * wide * 4));
        }
    }
    return p;
}

}  // namespace tb
