// How attention over a paged cache is cut into work for the SMs: host arithmetic only, no CUDA headers
// (tests/test_paged_plan_host.py).
#pragma once
#include <algorithm>
#include <cstdint>

namespace tb {

constexpr int PA_ROWS = 16;          // query rows (token, head of the group) of a tile: one tensor-core fragment
constexpr int PA_KEYS = 64;          // keys per stage of the ring, 16 for each of four warps

struct PagedPlan {
    int tiles;                       // row tiles of the longest chunk
    int split_keys, splits;          // keys per CTA along the cache (a multiple of PA_KEYS) and how many such pieces max_kv has
    int64_t workspace;               // bytes for the pieces' results: 0 for one piece
};

inline PagedPlan paged_plan(int seqs, int heads, int group, int hd, int rows, int max_q, int max_kv, int sms) {
    PagedPlan p;
    p.tiles = (int)(((int64_t)max_q * group + PA_ROWS - 1) / PA_ROWS);
    // pieces so that there are about three CTAs for every SM, but none shorter than two stages
    const int64_t items = (int64_t)seqs * heads * p.tiles;
    const int64_t want = std::max<int64_t>(1, 3LL * sms / std::max<int64_t>(items, 1));
    const int64_t blocks = ((int64_t)max_kv + PA_KEYS - 1) / PA_KEYS;
    const int64_t per = std::max<int64_t>(std::min<int64_t>(2, blocks), (blocks + want - 1) / want);
    p.split_keys = (int)(std::max<int64_t>(per, 1) * PA_KEYS);
    p.splits = (int)std::max<int64_t>(1, ((int64_t)max_kv + p.split_keys - 1) / p.split_keys);
    p.workspace = p.splits > 1 ? (int64_t)p.splits * rows * heads * group * (hd + 2) * 4 : 0;
    return p;
}

}  // namespace tb
