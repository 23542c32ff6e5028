// What kernels leave on the device for the host to find: two words in front of the tickets and packed maxima that kernels share.  Which of the
// two is told, and what goes back to zero with it, is host arithmetic without CUDA types (tests/test_error_words_host.py).
#pragma once
#include <cstddef>

namespace tb {

constexpr size_t kErrorBytes = 1024;      // the words, and everything behind them
constexpr size_t kErrorTickets = 128;     // where the tickets begin

struct ErrorWords {
    int wait;                             // a kernel gave up on a bounded wait: its output is invalid
    int argument;                         // an argument that only the device sees was outside its array: the kernel has gone on without it
};

// code 0: nothing to tell.  What to clear: the word itself (at `word` bytes), and behind a failed wait the tickets and maxima, which the kernel
// may have left half-way.  An argument's code clears nothing but itself: other kernels may be at work with the tickets.
struct ErrorReport {
    int code;
    bool wait;
    size_t word;
    bool tickets;
};

// arguments: whether the caller tells of arguments (a call of its own that waits for something else leaves them for the one that does)
inline ErrorReport error_report(const ErrorWords& w, bool arguments) {
    if (w.wait != 0) return {w.wait, true, offsetof(ErrorWords, wait), true};
    if (arguments && w.argument != 0) return {w.argument, false, offsetof(ErrorWords, argument), false};
    return {0, false, 0, false};
}

inline const char* argument_error(int code) {
    return code == 71                 ? "a page table names a page outside the pool; its rows were left out"
           : code == 75               ? "a page table names a page outside the pool; rows that see it are NaN"
           : code == 72 || code == 76 ? "a length or position of a batch is outside what its call allows; its rows were left out"
           : code == 81               ? "a length, index or penalty of the rules on logits is outside its range; what it concerns was left out"
                                      : "an argument on the device is outside its array";
}

}  // namespace tb
