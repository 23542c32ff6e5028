// Penalties for repeated tokens, biases and masks on the logits of a batch, in one pass over them.
//
// A CTA owns a slice of the vocabulary of one row.  It counts the row's ids that fall into its slice in shared memory (whole
// numbers: the order of the atomic additions does not show), gathers the slice's bias entries there, and then reads, changes and
// writes its logits once.  Bound: the logits, 8 bytes each; every CTA of a row reads the row's ids again, from L2.
#include "../../include/turkce_b200.h"
#include "common.h"
#include "logit_rules.h"

#include <algorithm>

namespace tb {

namespace {

constexpr int LR_THREADS = 256;
constexpr uint32_t LR_PROMPT = 0x80000000u;      // bits of a token's word: among the prompt's ids
constexpr uint32_t LR_TWICE = 0x40000000u;       // more than one bias entry; the rest counts the output ids
constexpr uint32_t LR_COUNT = 0x3fffffffu;

struct LogitParams {
    LogitRuleArgs r;
    const float* in; long long ld_in;
    float* out; long long ld_out;
    int V, slice;
    int* err;
};

template <bool WIDE>
__global__ void __launch_bounds__(LR_THREADS)
logit_rules_kernel(const LogitParams p) {
    extern __shared__ uint32_t lr_smem[];
    uint32_t* seen = lr_smem;                                    // [slice]
    uint32_t* owner = lr_smem + p.slice;                         // [slice]: the token's first bias entry, then the sum's bits
    __shared__ int twice;
    pdl_wait();
    pdl_launch_dependents();
    const int row = blockIdx.y, tid = threadIdx.x;
    const int v0 = blockIdx.x * p.slice, n = min(p.slice, p.V - v0);
    const LogitRuleArgs& r = p.r;
    const float rep = r.repetition ? r.repetition[row] : 1.0f, freq = r.frequency ? r.frequency[row] : 0.0f,
                pres = r.presence ? r.presence[row] : 0.0f;
    const bool counts = rep != 1.0f || freq != 0.0f || pres != 0.0f;
    int b0 = 0, b1 = 0;
    if (r.bias_start) {
        b0 = r.bias_start[row]; b1 = r.bias_start[row + 1];
        if (b0 < 0 || b1 < b0 || b1 > r.bias_entries) {
            if (tid == 0) atomicExch(p.err, 81);
            b0 = b1 = 0;
        }
    }
    const bool biased = b1 > b0;
    if (counts || biased) {
        for (int i = tid; i < n; i += LR_THREADS) {
            seen[i] = 0u;
            if (biased) owner[i] = 0xffffffffu;
        }
        if (tid == 0) twice = 0;
        __syncthreads();
        if (counts) {
            auto look = [&](const uint32_t* ids, const int* lens, int len_stride, int ld, bool prompt) {
                if (!ids) return;
                int len = lens[row * len_stride];
                if (len < 0 || len > ld) {
                    if (tid == 0) atomicExch(p.err, 81);
                    len = min(max(len, 0), ld);
                }
                const uint32_t* at = ids + (long long)row * ld;
                for (int i = tid; i < len; i += LR_THREADS) {
                    const uint32_t t = at[i] - (uint32_t)v0;
                    if (at[i] >= (uint32_t)v0 && t < (uint32_t)n) {
                        if (prompt) atomicOr(&seen[t], LR_PROMPT);
                        else atomicAdd(&seen[t], 1u);
                    }
                }
            };
            if (rep != 1.0f) look(r.prompt, r.prompt_len, r.prompt_len_stride, r.prompt_ld, true);
            look(r.output, r.output_len, r.output_len_stride, r.output_ld, false);
        }
        if (biased) {
            for (int i = b0 + tid; i < b1; i += LR_THREADS) {
                const uint32_t id = r.bias_id[i], t = id - (uint32_t)v0;
                if (id >= (uint32_t)v0 && t < (uint32_t)n) atomicMin(&owner[t], (uint32_t)i);
            }
            __syncthreads();
            // entries that are not their token's first one
            for (int i = b0 + tid; i < b1; i += LR_THREADS) {
                const uint32_t id = r.bias_id[i], t = id - (uint32_t)v0;
                if (id >= (uint32_t)v0 && t < (uint32_t)n && owner[t] != (uint32_t)i) { atomicOr(&seen[t], LR_TWICE); twice = 1; }
            }
            __syncthreads();
            // a token's sum in the order of the list.  (Its word turns from an index into a sum: every thread that still looks for
            // an index owns it.)
            const bool any = twice != 0;
            for (int t = tid; t < n; t += LR_THREADS) {
                const uint32_t i = owner[t];
                float sum = 0.0f;
                if (i != 0xffffffffu) {
                    sum = r.bias_value[i];
                    if (any && (seen[t] & LR_TWICE))
                        for (int j = (int)i + 1; j < b1; ++j)
                            if (r.bias_id[j] == (uint32_t)(v0 + t)) sum += r.bias_value[j];
                }
                owner[t] = __float_as_uint(sum);
            }
        }
        __syncthreads();
    }
    const uint32_t* mask = nullptr;
    if (r.mask) {
        const int m = r.mask_row ? r.mask_row[row] : row;
        if (m >= r.masks || m < -1) {
            if (tid == 0) atomicExch(p.err, 81);
        } else if (m >= 0) {
            mask = r.mask + (long long)m * r.mask_ld;
        }
    }
    auto rule = [&](float z, int t) -> float {
        if (counts) {
            const uint32_t w = seen[t], c = w & LR_COUNT;
            if (c != 0u || (w & LR_PROMPT)) {
                if (rep != 1.0f) z = z > 0.0f ? __fdiv_rn(z, rep) : z * rep;
                if (c != 0u) {
                    z = __fsub_rn(z, __fmul_rn(freq, (float)c));
                    z = __fsub_rn(z, pres);
                }
            }
        }
        if (biased) z += __uint_as_float(owner[t]);
        return z;
    };
    const float* in = p.in + (long long)row * p.ld_in + v0;
    float* out = p.out + (long long)row * p.ld_out + v0;
    if (WIDE) {
        // four columns per thread: slices start at multiples of 32, so that four columns share a mask word
        for (int t = tid * 4; t < n; t += LR_THREADS * 4) {
            const uint32_t bits = mask ? mask[(v0 + t) >> 5] >> (t & 31) : 0xfu;
            if (t + 4 <= n) {
                const float4 z = *reinterpret_cast<const float4*>(in + t);
                float4 o;
                o.x = bits & 1u ? rule(z.x, t) : -INFINITY;
                o.y = bits & 2u ? rule(z.y, t + 1) : -INFINITY;
                o.z = bits & 4u ? rule(z.z, t + 2) : -INFINITY;
                o.w = bits & 8u ? rule(z.w, t + 3) : -INFINITY;
                *reinterpret_cast<float4*>(out + t) = o;
            } else {
                for (int i = 0; t + i < n; ++i) out[t + i] = bits >> i & 1u ? rule(in[t + i], t + i) : -INFINITY;
            }
        }
    } else {
        for (int t = tid; t < n; t += LR_THREADS) {
            const bool allowed = !mask || (mask[(v0 + t) >> 5] >> (t & 31) & 1u);
            out[t] = allowed ? rule(in[t], t) : -INFINITY;
        }
    }
}

}  // namespace

int launch_logit_rules(DeviceCtx* ctx, const LogitRuleArgs& r, const float* in, long long ld_in, float* out, long long ld_out, int rows,
                       int V, cudaStream_t st) {
    LogitParams p;
    p.r = r; p.in = in; p.ld_in = ld_in; p.out = out; p.ld_out = ld_out; p.V = V; p.err = ctx->d_err;
    p.slice = logit_rules_slice(rows, V, ctx->sm_count);
    const bool wide = ((reinterpret_cast<uintptr_t>(in) | reinterpret_cast<uintptr_t>(out)) & 15u) == 0 && ld_in % 4 == 0 && ld_out % 4 == 0;
    const size_t smem = (size_t)p.slice * 8;
    prof_mark(ctx, "logit_rules", 0.0, 8.0 * rows * V, st);
    TB_CUDA(launch_kernel(wide ? logit_rules_kernel<true> : logit_rules_kernel<false>, dim3((V + p.slice - 1) / p.slice, rows), dim3(LR_THREADS),
                          smem, st, p));
    ctx->launches++;
    prof_close(ctx, st);
    return 0;
}

}  // namespace tb

using namespace tb;

extern "C" int tb_logits_adjust(const TbLogitRules* rules, const float* d_logits, int64_t ld_logits, float* d_out, int64_t ld_out, int rows,
                                int vocab, void* stream) {
    TB_CHECK(rules != nullptr, "tb_logits_adjust: NULL rules");
    TB_CHECK(rows >= 0 && rows <= 65535 && vocab > 0 && vocab < (1 << 30), "tb_logits_adjust: rows must be in [0, 65535] and vocab in [1, 2^30)");
    if (rows == 0) return 0;
    TB_CHECK(d_logits && d_out, "tb_logits_adjust: NULL logits");
    TB_CHECK(ld_logits >= vocab && ld_out >= vocab, "tb_logits_adjust: leading dimensions must be at least vocab");
    TB_CHECK(d_out != d_logits || ld_out == ld_logits, "tb_logits_adjust: in place, both leading dimensions must be the same");
    if (d_out != d_logits) {
        const uintptr_t a0 = reinterpret_cast<uintptr_t>(d_logits), a1 = a0 + ((rows - 1) * ld_logits + vocab) * 4;
        const uintptr_t b0 = reinterpret_cast<uintptr_t>(d_out), b1 = b0 + ((rows - 1) * ld_out + vocab) * 4;
        TB_CHECK(a1 <= b0 || b1 <= a0, "tb_logits_adjust: the output overlaps the logits");
    }
    const TbLogitRules& r = *rules;
    TB_CHECK(!r.prompt || (r.prompt_len && r.prompt_ld > 0 && r.prompt_ld < (1 << 30)), "tb_logits_adjust: prompt ids need lengths and a leading dimension below 2^30");
    TB_CHECK(!r.output || (r.output_len && r.output_ld > 0 && r.output_ld < (1 << 30)), "tb_logits_adjust: output ids need lengths and a leading dimension below 2^30");
    TB_CHECK(!r.bias_start || r.bias_entries == 0 || (r.bias_id && r.bias_value), "tb_logits_adjust: bias entries need ids and values");
    TB_CHECK(r.bias_entries >= 0, "tb_logits_adjust: bias_entries must not be negative");
    TB_CHECK(!r.mask || (r.masks > 0 && r.mask_ld >= (vocab + 31) / 32), "tb_logits_adjust: masks need %d words each", (vocab + 31) / 32);
    TB_CHECK(!r.mask || r.mask_row || r.masks >= rows, "tb_logits_adjust: %d masks for %d rows need mask_row", r.masks, rows);
    LogitRuleArgs a;
    a.prompt = r.prompt; a.prompt_len = r.prompt_len; a.prompt_ld = r.prompt_ld; a.prompt_len_stride = 1;
    a.output = r.output; a.output_len = r.output_len; a.output_ld = r.output_ld; a.output_len_stride = 1;
    a.repetition = r.repetition; a.frequency = r.frequency; a.presence = r.presence;
    a.bias_start = r.bias_entries > 0 ? r.bias_start : nullptr; a.bias_id = r.bias_id; a.bias_value = r.bias_value; a.bias_entries = r.bias_entries;
    a.mask = r.mask; a.mask_row = r.mask_row; a.masks = r.masks; a.mask_ld = r.mask_ld;
    DeviceCtx* ctx;
    TB_TRY(get_ctx(&ctx));
    return launch_logit_rules(ctx, a, d_logits, ld_logits, d_out, ld_out, rows, vocab, static_cast<cudaStream_t>(stream));
}
