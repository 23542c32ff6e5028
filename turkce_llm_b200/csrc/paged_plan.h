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

struct PagedPlan {
    bool whole;                      // every item is one CTA's
    int grid;                        // CTAs of the kernel for few rows
    int64_t workspace;               // bytes: a counter and two results per CTA
};

inline PagedPlan paged_plan(int seqs, int heads, int hd, bool e4m3, int max_kv, int sms) {
    PagedPlan p;
    const int64_t items = (int64_t)seqs * heads, most = (int64_t)paged_per_sm(hd > 64 ? 2 : 1, e4m3) * sms;
    p.whole = max_kv <= PA_WHOLE;
    const int64_t keys = paged_keys(hd > 64 ? 2 : 1, e4m3), blocks = items * (((int64_t)max_kv + keys - 1) / keys), least = PA_LEAST / keys;
    p.grid = (int)std::max<int64_t>(1, std::min(most, p.whole ? items : (blocks + least - 1) / least));
    // a word per CTA (to a multiple of 16 bytes), then its two results
    p.workspace = p.whole ? 0 : (int64_t)(p.grid + 3) / 4 * 16 + 2LL * p.grid * PA_ROWS * (hd + 2) * 4;
    return p;
}

}  // namespace tb
