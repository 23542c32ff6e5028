// Penalties for repeated tokens, biases and masks on the logits of a batch, in one pass over them.
//
// A CTA owns a slice of the vocabulary of one row.  It counts the row's ids that fall into its slice in shared memory (whole
// numbers: the order of the atomic additions does not show), gathers the slice's bias entries there, and then reads, changes and
// writes its logits once.  Bound: the logits, 8 bytes each; every CTA of a row reads the row's ids again, from L2.
#include "../../include/turkce_b200.h"
#include "common.h"
#include "logit_rules.h"
#include "overlap.h"

#include <algorithm>

namespace tb {

namespace {

constexpr int LR_THREADS = 512;
constexpr uint32_t LR_PROMPT = 0x80000000u;      // bits of a token's word: among the prompt's ids
constexpr uint32_t LR_BIAS = 0x40000000u;        // a bias entry
constexpr uint32_t LR_TWICE = 0x20000000u;       // more than one; the rest counts the output ids
constexpr uint32_t LR_COUNT = 0x1fffffffu;
constexpr int LR_IDS = 2;                        // ids of the prompt and of the output that a thread asks for at once
constexpr uint32_t LR_NONE = 0xffffffffu;
constexpr int LR_AGAIN = 64;
constexpr float LR_LEAST = 0x1p-32f, LR_MOST = 0x1p32f;          // repetition penalties
constexpr int LR_ROUNDS = kLogitSlice / (LR_THREADS * 4);

struct LogitParams {
    LogitRuleArgs r;
    const float* in; long long ld_in;
    float* out; long long ld_out;
    int V, slice;
    int* err;
};

// The logits of a slice are asked for first and held in registers while the ids are counted: the two share the time of one trip
// to memory.  (Counting first and reading then: 49 us for 256 rows of 31,769 with 750 ids and 150 biases each.)
// WIDE: rows of logits and result that begin at the same place of a 16-byte piece, whatever it is: a CTA's slice begins at a whole piece, up
// to three columns in front of a multiple of the slice, and a thread has four neighbours.  Else a thread has every 512th column.  (Rows of
// 31,769 begin at another place each: four neighbours in single accesses took 31.6 us.)
template <bool WIDE>
__global__ void __launch_bounds__(LR_THREADS)
logit_rules_kernel(const LogitParams p) {
    extern __shared__ uint32_t lr_smem[];
    uint32_t* seen = lr_smem;                                    // [slice]
    float* bias = reinterpret_cast<float*>(lr_smem + p.slice);   // [slice], where LR_BIAS is set
    __shared__ int again, again_at[LR_AGAIN];                    // tokens with more than one bias entry
    pdl_wait();
    pdl_launch_dependents();
    const int row = blockIdx.y, tid = threadIdx.x;
    const LogitRuleArgs& r = p.r;
    const float* in = p.in + (long long)row * p.ld_in;
    float* out = p.out + (long long)row * p.ld_out;
    // columns v0 .. v0 + slice - 1, those that exist
    const int v0 = (int)blockIdx.x * p.slice - (WIDE ? (int)(reinterpret_cast<uintptr_t>(in) >> 2 & 3u) : 0);
    const int lo = max(-v0, 0), n = min(p.slice, p.V - v0);
    if (n <= 0) return;
    in += v0; out += v0;
    auto column = [&](int g, int i) { return WIDE ? (g * LR_THREADS + tid) * 4 + i : (g * 4 + i) * LR_THREADS + tid; };
    auto whole = [&](int t) { return WIDE && t >= lo && t + 4 <= n; };       // four columns that all exist
    float z[LR_ROUNDS][4];
#pragma unroll
    for (int g = 0; g < LR_ROUNDS; ++g) {
        if (whole(column(g, 0))) {
            const float4 w = *reinterpret_cast<const float4*>(in + column(g, 0));
            z[g][0] = w.x; z[g][1] = w.y; z[g][2] = w.z; z[g][3] = w.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) z[g][i] = column(g, i) >= lo && column(g, i) < n ? in[column(g, i)] : 0.0f;
        }
    }
    // The first ids of the row as well, before it is known how many count: lengths, ids and logits come in the same time.
    uint32_t ids[2][LR_IDS];
    auto early = [&](const uint32_t* at, int ld, uint32_t (&to)[LR_IDS]) {
#pragma unroll
        for (int i = 0; i < LR_IDS; ++i) to[i] = at && i * LR_THREADS + tid < ld ? at[(long long)row * ld + i * LR_THREADS + tid] : LR_NONE;
    };
    early(r.prompt, r.prompt_ld, ids[0]);
    early(r.output, r.output_ld, ids[1]);
    int lens[2] = {r.prompt ? r.prompt_len[row] : 0, r.output ? r.output_len[row] : 0};
    float rep = r.repetition ? r.repetition[row] : 1.0f;
    rep = rep >= LR_LEAST && rep <= LR_MOST ? rep : 1.0f;        // (its inverse or a remainder may be outside float32; or it is none)
    const float freq = r.frequency ? r.frequency[row] : 0.0f,
                pres = r.presence ? r.presence[row] : 0.0f;
    int b0 = 0, b1 = 0;
    if (r.bias_start) {
        b0 = r.bias_start[row]; b1 = r.bias_start[row + 1];
        if (b0 < 0 || b1 < b0 || b1 > r.bias_entries) {
            if (tid == 0) report_argument(p.err, 81);
            b0 = b1 = 0;
        }
    }
    // this thread's first bias entry
    const int my_bias = b0 + tid;
    const uint32_t bias_id = my_bias < b1 ? r.bias_id[my_bias] : LR_NONE;
    const float bias_value = my_bias < b1 ? r.bias_value[my_bias] : 0.0f;
    const bool counts = rep != 1.0f || freq != 0.0f || pres != 0.0f, biased = b1 > b0;
    const uint32_t* mask = nullptr;
    if (r.mask) {
        const int m = r.mask_row ? r.mask_row[row] : row;
        if (m >= r.masks || m < -1) {
            if (tid == 0) report_argument(p.err, 81);
        } else if (m >= 0) {
            mask = r.mask + (long long)m * r.mask_ld;
        }
    }
    uint32_t allowed = 0xffffffffu;                              // bit 4 g + i
    if (mask) {
        allowed = 0u;
#pragma unroll
        for (int g = 0; g < LR_ROUNDS; ++g) {
            if (whole(column(g, 0))) {
                const int v = v0 + column(g, 0), bit = v & 31;
                const uint32_t a = mask[v >> 5], b = bit > 28 ? mask[(v >> 5) + 1] : 0u;
                allowed |= (__funnelshift_r(a, b, bit) & 0xfu) << (4 * g);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int t = column(g, i);
                    if (t >= lo && t < n) allowed |= (mask[(v0 + t) >> 5] >> ((v0 + t) & 31) & 1u) << (4 * g + i);
                }
            }
        }
    }
    if (counts || biased) {
        for (int i = tid * 4; i < p.slice; i += LR_THREADS * 4) *reinterpret_cast<uint4*>(seen + i) = make_uint4(0u, 0u, 0u, 0u);
        if (tid == 0) again = 0;
        __syncthreads();
        auto place = [&](uint32_t id) -> uint32_t { return id < (uint32_t)p.V ? id - (uint32_t)v0 : LR_NONE; };       // (of this slice where below n)
        if (counts) {
            auto look = [&](int which, const uint32_t* at, int ld) {
                if (!at || (which == 0 && rep == 1.0f)) return;
                int len = lens[which];
                if (len < 0 || len > ld) {
                    if (tid == 0) report_argument(p.err, 81);
                    len = min(max(len, 0), ld);
                }
                auto one = [&](uint32_t id) {
                    const uint32_t t = place(id);
                    if (t >= (uint32_t)n) return;
                    if (which == 0) atomicOr(&seen[t], LR_PROMPT);
                    else atomicAdd(&seen[t], 1u);
                };
#pragma unroll
                for (int i = 0; i < LR_IDS; ++i)
                    if (i * LR_THREADS + tid < len) one(ids[which][i]);
#pragma unroll 4
                for (int i = LR_IDS * LR_THREADS + tid; i < len; i += LR_THREADS) one(at[(long long)row * ld + i]);
            };
            look(0, r.prompt, r.prompt_ld);
            look(1, r.output, r.output_ld);
        }
        // a token's only entry leaves its value; who finds that there is one already makes a note
        for (int i = my_bias; i < b1; i += LR_THREADS) {
            const uint32_t t = place(i == my_bias ? bias_id : r.bias_id[i]);
            if (t >= (uint32_t)n) continue;
            const uint32_t before = atomicOr(&seen[t], LR_BIAS);
            if (!(before & LR_BIAS)) {
                bias[t] = i == my_bias ? bias_value : r.bias_value[i];
            } else if (!(atomicOr(&seen[t], LR_TWICE) & LR_TWICE)) {
                const int k = atomicAdd(&again, 1);
                if (k < LR_AGAIN) again_at[k] = (int)t;
            }
        }
        __syncthreads();
        if (again > 0) {
            // those tokens' entries in the order of the list, a warp per token.  (More of them than there is room for: every token is looked at.)
            const int lane = tid & 31, count = again <= LR_AGAIN ? again : p.slice;
            for (int k = tid >> 5; k < count; k += LR_THREADS / 32) {
                const int t = again <= LR_AGAIN ? again_at[k] : k;
                if (t >= n || !(seen[t] & LR_TWICE)) continue;
                float sum = 0.0f;
                for (int j0 = b0; j0 < b1; j0 += 32) {
                    const bool same = j0 + lane < b1 && r.bias_id[j0 + lane] == (uint32_t)(v0 + t);
                    const float value = same ? r.bias_value[j0 + lane] : 0.0f;
                    for (uint32_t left = __ballot_sync(0xffffffffu, same); left != 0u; left &= left - 1u)
                        sum += __shfl_sync(0xffffffffu, value, __ffs(left) - 1);
                }
                if (lane == 0) bias[t] = sum;
            }
            __syncthreads();
        }
    }
    const float inverse = __frcp_rn(rep);
    if (tid == 0 && r.repetition && rep == 1.0f && r.repetition[row] != 1.0f) report_argument(p.err, 81);       // (read again: not to be held)
    auto rule = [&](float x, uint32_t w, int t) -> float {
        if (counts && (w & (LR_COUNT | LR_PROMPT)) != 0u) {
            // x / rep by Markstein's correction (a quotient by the correctly rounded reciprocal, and what its remainder adds, both fused):
            // the nearest number while the remainder is one that float32 has, else two units in the last place from it at most; x * rep of
            // what is not positive
            const float q = x * inverse, y = __fmaf_rn(__fmaf_rn(-q, rep, x), inverse, q);
            x = x > 0.0f ? (q < INFINITY ? y : q) : x * rep;
            if ((w & LR_COUNT) != 0u) x = __fsub_rn(__fsub_rn(x, __fmul_rn(freq, (float)(w & LR_COUNT))), pres);
        }
        if (w & LR_BIAS) x += bias[t];
        return x;
    };
#pragma unroll
    for (int g = 0; g < LR_ROUNDS; ++g) {
        const int t = column(g, 0);
        if (counts || biased) {
            uint32_t w[4] = {0u, 0u, 0u, 0u};
            if (WIDE) {
                if (t < n) {
                    const uint4 w4 = *reinterpret_cast<const uint4*>(seen + t);
                    w[0] = w4.x; w[1] = w4.y; w[2] = w4.z; w[3] = w4.w;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) if (column(g, i) < n) w[i] = seen[column(g, i)];
            }
            // (most columns are touched by no rule)
            if ((w[0] | w[1] | w[2] | w[3]) != 0u) {
#pragma unroll
                for (int i = 0; i < 4; ++i) z[g][i] = rule(z[g][i], w[i], column(g, i));
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (!(allowed >> (4 * g + i) & 1u)) z[g][i] = -INFINITY;
        if (whole(t)) {
            *reinterpret_cast<float4*>(out + t) = make_float4(z[g][0], z[g][1], z[g][2], z[g][3]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (column(g, i) >= lo && column(g, i) < n) out[column(g, i)] = z[g][i];
        }
    }
}

}  // namespace

int launch_logit_rules(DeviceCtx* ctx, const LogitRuleArgs& r, const float* in, long long ld_in, float* out, long long ld_out, int rows,
                       int V, cudaStream_t st) {
    LogitParams p;
    p.r = r; p.in = in; p.ld_in = ld_in; p.out = out; p.ld_out = ld_out; p.V = V; p.err = ctx->d_err;
    p.slice = logit_rules_slice(rows, V, ctx->sm_count);
    const bool wide = ((reinterpret_cast<uintptr_t>(in) ^ reinterpret_cast<uintptr_t>(out)) & 15u) == 0 && (rows == 1 || (ld_in - ld_out) % 4 == 0);
    const size_t smem = (size_t)p.slice * 8;
    prof_mark(ctx, "logit_rules", 0.0, 8.0 * rows * V, st);
    TB_CUDA(launch_kernel(wide ? logit_rules_kernel<true> : logit_rules_kernel<false>, dim3((V + (wide ? 3 : 0) + p.slice - 1) / p.slice, rows), dim3(LR_THREADS),
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
    TB_CHECK(d_out == d_logits || !spans_overlap({d_logits, rows, vocab * 4LL, ld_logits * 4}, {d_out, rows, vocab * 4LL, ld_out * 4}),
             "tb_logits_adjust: the output overlaps the logits");
    const TbLogitRules& r = *rules;
    TB_CHECK(!r.prompt || (r.prompt_len && r.prompt_ld > 0 && r.prompt_ld < (1 << 29)), "tb_logits_adjust: prompt ids need lengths and a leading dimension below 2^29");
    TB_CHECK(!r.output || (r.output_len && r.output_ld > 0 && r.output_ld < (1 << 29)), "tb_logits_adjust: output ids need lengths and a leading dimension below 2^29");
    TB_CHECK(!r.bias_start || r.bias_entries == 0 || (r.bias_id && r.bias_value), "tb_logits_adjust: bias entries need ids and values");
    TB_CHECK(r.bias_entries >= 0, "tb_logits_adjust: bias_entries must not be negative");
    TB_CHECK(!r.mask || (r.masks > 0 && r.mask_ld >= (vocab + 31) / 32), "tb_logits_adjust: masks need %d words each", (vocab + 31) / 32);
    TB_CHECK(!r.mask || r.mask_row || r.masks >= rows, "tb_logits_adjust: %d masks for %d rows need mask_row", r.masks, rows);
    LogitRuleArgs a;
    a.prompt = r.prompt; a.prompt_len = r.prompt_len; a.prompt_ld = r.prompt_ld;
    a.output = r.output; a.output_len = r.output_len; a.output_ld = r.output_ld;
    a.repetition = r.repetition; a.frequency = r.frequency; a.presence = r.presence;
    a.bias_start = r.bias_start; a.bias_id = r.bias_id; a.bias_value = r.bias_value; a.bias_entries = r.bias_entries;
    a.mask = r.mask; a.mask_row = r.mask_row; a.masks = r.masks; a.mask_ld = r.mask_ld;
    DeviceCtx* ctx;
    TB_TRY(get_ctx(&ctx));
    return launch_logit_rules(ctx, a, d_logits, ld_logits, d_out, ld_out, rows, vocab, static_cast<cudaStream_t>(stream));
}
