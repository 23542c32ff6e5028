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

constexpr int PL_TILES = 1024;                   // tiles of a head that the plan on the device can hold
constexpr int PT_ROWS = 128, PT_KEYS = 128;      // query rows and keys of the kernel for longer chunks
// CTAs of that kernel that an SM holds
constexpr int paged_tiles_per_sm(int wide, bool e4m3) { return wide == 1 && !e4m3 ? 2 : 1; }

// A workspace begins with a counter for every CTA of the kernel for few rows that the chip can hold, whatever the call: what a call leaves
// there (zeros) is where the next one, of another size or type, looks for it.  Nothing else outlives a call.
constexpr int PA_MOST_PER_SM = 3;
constexpr int64_t paged_counters(int sms) { return ((int64_t)PA_MOST_PER_SM * sms + 3) / 4 * 4; }

struct PagedPlan {
    bool whole;                      // few rows: every item is one CTA's
    int grid;                        // few rows: CTAs
    int most_units, most_pieces;     // longer chunks: room for tiles or pieces of them, and for pieces' results; 0: a CTA per tile
    int64_t rows_bytes, workspace;   // bytes of the counters and the kernel for few rows (two results per CTA); of both (0: none needed)
    int64_t room;                    // bytes that no batch within these bounds needs more than
};

inline PagedPlan paged_plan(int seqs, int heads, int group, int hd, bool e4m3, int rows, int max_q, int max_kv, int sms) {
    PagedPlan p;
    const int wide = hd > 64 ? 2 : 1;
    const int64_t items = (int64_t)seqs * heads, most = (int64_t)paged_per_sm(wide, e4m3) * sms, counters = paged_counters(sms) * 4;
    p.whole = max_kv <= PA_WHOLE;
    const int64_t keys = paged_keys(wide, e4m3), blocks = items * (((int64_t)max_kv + keys - 1) / keys), least = PA_LEAST / keys;
    p.grid = (int)std::max<int64_t>(1, std::min(most, p.whole ? items : (blocks + least - 1) / least));
    const int64_t results = p.whole ? 0 : 2LL * p.grid * PA_ROWS * (hd + 2) * 4;
    p.rows_bytes = counters + (results + 15) / 16 * 16;
    p.most_units = p.most_pieces = 0;
    p.workspace = p.room = p.whole ? 0 : p.rows_bytes;
    if ((int64_t)max_q * group > PA_ROWS) {
        // No more tiles than this many: every sequence that has tiles at all has more than PA_ROWS rows per key head.  Where that is
        // less than two for every CTA that the chip holds, tiles are cut into pieces (no more of them than CTAs).  Where it is less than
        // half of a CTA for every tile that a sequence may have, they are dealt out all the same: 4,096 single tokens and a chunk of 60
        // rows, 6 heads of 64, take 175 us so, and 322 us with 24,582 CTAs of which 6 have a tile.
        const int64_t tokens = PT_ROWS / group, least_rows = PA_ROWS / group + 1;
        const int64_t per_head = rows / tokens + std::min<int64_t>(seqs, rows / least_rows), tiles = heads * per_head;
        const int64_t slots = (int64_t)paged_tiles_per_sm(wide, e4m3) * sms;
        // header, then for every unit: a counter, a flag, what it is; for every piece [128] (maximum, sum) and [128][64 wide] float32
        auto bytes = [&](int64_t units) { return 16 + (units + 3) / 4 * 4 * (4 + 4 + 32) + (slots + 3) / 4 * 4 * PT_ROWS * (8 + 64 * wide * 4); };
        if (per_head <= PL_TILES && ((max_kv > PT_KEYS && tiles < 2 * slots) || 2 * tiles <= items * ((max_q + tokens - 1) / tokens))) {
            p.most_units = (int)(std::max(slots, tiles) + 3) / 4 * 4;
            p.most_pieces = (int)(slots + 3) / 4 * 4;
            p.workspace = p.rows_bytes + bytes(p.most_units);
        }
        p.room = p.rows_bytes + bytes(std::max(slots, std::min(tiles, (int64_t)heads * PL_TILES)));
    }
    return p;
}

}  // namespace tb
