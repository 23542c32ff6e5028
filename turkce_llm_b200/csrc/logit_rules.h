// The rules on logits as their kernel has them (the entry point's arrays), and how rows are cut into slices.  The slices are host arithmetic
// without CUDA types.
#pragma once
#include <cstdint>

namespace tb {

constexpr int kLogitSlice = 4096;         // most columns per CTA: four per thread in two rounds

// Columns of the vocabulary per CTA: a multiple of 32 up to 4096, a few words of a mask.  (Where slices begin in front of it, at a whole
// 16-byte piece of the logits, two CTAs read the word between them.)  As many as give every SM
// four CTAs, so that few rows spread over the chip and many rows do not read their ids more often than needed.
inline int logit_rules_slice(int rows, int V, int sms) {
    const long long want = 4LL * sms;
    long long slices = (want + rows - 1) / rows;
    long long s = (V + slices - 1) / slices;
    s = (s + 31) / 32 * 32;
    return (int)(s < 512 ? 512 : s > kLogitSlice ? kLogitSlice : s);
}

struct LogitRuleArgs {
    const uint32_t* prompt = nullptr; const int* prompt_len = nullptr; int prompt_ld = 0;
    const uint32_t* output = nullptr; const int* output_len = nullptr; int output_ld = 0;
    const float *repetition = nullptr, *frequency = nullptr, *presence = nullptr;
    const int* bias_start = nullptr; const uint32_t* bias_id = nullptr; const float* bias_value = nullptr; int bias_entries = 0;
    const uint32_t* mask = nullptr; const int* mask_row = nullptr; int masks = 0, mask_ld = 0;
};

}  // namespace tb
