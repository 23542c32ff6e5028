// Whether two matrices in memory share a byte: host arithmetic for the refusals (tests/test_overlap_host.py).
#pragma once
#include <algorithm>
#include <cstdint>

namespace tb {

// `rows` rows of `bytes` bytes, the next one `pitch` bytes behind
struct RowSpan {
    const void* at;
    long long rows, bytes, pitch;
};

inline bool spans_overlap(RowSpan a, RowSpan b) {
    if (!a.at || !b.at || a.rows <= 0 || b.rows <= 0 || a.bytes <= 0 || b.bytes <= 0) return false;
    const long long a0 = (long long)reinterpret_cast<uintptr_t>(a.at), b0 = (long long)reinterpret_cast<uintptr_t>(b.at);
    if (a0 + (a.rows - 1) * a.pitch + a.bytes <= b0 || b0 + (b.rows - 1) * b.pitch + b.bytes <= a0) return false;
    auto floor_div = [](long long x, long long y) { return x / y - (x % y != 0 && (x < 0) != (y < 0)); };
    if (a.rows == 1) a.pitch = b.pitch;
    if (b.rows == 1) b.pitch = a.pitch;
    if (a.pitch <= 0) return true;                               // (two single rows that meet)
    if (a.pitch == b.pitch) {
        // row i of a and row i - k of b meet where d - a.bytes < k pitch < d + b.bytes
        const long long d = b0 - a0, k = std::max(floor_div(d - a.bytes, a.pitch) + 1, -(b.rows - 1));
        return k <= a.rows - 1 && k * a.pitch < d + b.bytes;
    }
    if (a.rows > b.rows) return spans_overlap(b, a);
    if (b.pitch <= 0) return true;
    for (long long i = 0; i < a.rows; ++i) {
        // the first row of b that ends behind the beginning of this row
        const long long x = a0 + i * a.pitch, j = std::max(0LL, floor_div(x - b0 - b.bytes, b.pitch) + 1);
        if (j < b.rows && b0 + j * b.pitch < x + a.bytes) return true;
    }
    return false;
}

// `heads` pieces of `bytes` per row, `head_pitch` bytes from one to the next: two such matrices of one shape
inline bool heads_overlap(const void* a, const void* b, long long rows, long long pitch, long long heads, long long head_pitch, long long bytes) {
    for (long long h = 1 - heads; h < heads; ++h)
        if (spans_overlap({a, rows, bytes, pitch}, {static_cast<const char*>(b) + h * head_pitch, rows, bytes, pitch})) return true;
    return false;
}

}  // namespace tb
