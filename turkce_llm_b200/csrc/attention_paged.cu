// Causal attention of new tokens over a paged cache of keys and values (bf16, or 8-bit codes with a scale per row).
//
// For query row (token i, head h) of a sequence, with positions up to its own visible:
//   o = sum_t p_t v_t / sum_t p_t,   p_t = 2^(s_t - m),   s_t = scale log2(e) <q, k_t>,   m = max s_t,
// in one pass over the keys: a running maximum m, the sum l and the accumulator rescaled where m grows.  Pieces of the cache
// are taken by different CTAs where there are few sequences; each leaves (o, m, l), and the CTA that is last with its piece adds them
// in the order of the pieces.
//
// Sequences with at most 16 query rows per key head (new tokens times the heads that share it) are paged_rows_kernel's, the others
// paged_chunk_kernel's.  Where tiles are few, paged_plan_kernel deals them out: tiles start first, single tokens beside them.
//
// 8-bit rows: a key's scale multiplies its score, a value's its probability (few rows) or its tile (chunks).  Probabilities are f16.
#include "paged.cuh"
#include "paged_plan.h"
#include "ptx.cuh"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace tb {

namespace {

struct PagedAttParams {
    PagedView v;
    const int *q_start, *kv_len;
    const bf16* Q; long long ld_q;
    const void* K;
    const float *ks, *vs;
    bf16* att; long long ld_att;
    float* lse;                      // [rows, H] or NULL
    float* part_o; float2* part_ml;  // [2 grid][16][hd], [2 grid][16]: results of items that a CTA shares with its neighbours
    unsigned int* arrived;           // [grid], zero between launches: pieces written of the item that begins in a CTA's run and goes on
    int rows, H, group, max_q, max_kv, grid, whole;
    const int* runs;                 // few rows: CTAs that share the work, as the plan says; nullptr: all
    int behind_chunks;               // few rows: the kernel in front is paged_chunk_kernel, which writes other rows
    uint32_t group_magic;            // x / group = x * group_magic >> 16 for x < 128
    float scale_log2;
    int* err;
};

// the sequence's first row, number of new rows and number of keys; false where they are outside what the call allows
__device__ __forceinline__ bool batch_ok(const PagedAttParams& p, int q0, int q1, int kv) {
    const int n = q1 - q0;
    return q0 >= 0 && q1 >= q0 && q1 <= p.rows && n <= p.max_q && kv >= 0 && kv <= p.max_kv &&
           kv <= (long long)p.v.table_ld << p.v.page_shift;
}
__device__ __forceinline__ bool batch_of(const PagedAttParams& p, int s, int& q0, int& n, int& kv) {
    q0 = p.q_start[s];
    const int q1 = p.q_start[s + 1];
    kv = p.kv_len[s];
    n = q1 - q0;
    return batch_ok(p, q0, q1, kv);
}

// ------------------------------------------------------------------------------- few rows: mma fragments
// Sequences whose new rows, times the heads that share a key head, are at most 16: single tokens, and a few of them.  What counts
// here is bytes: an item is one (sequence, key head), its rows are padded to the 16 of a fragment, and the tensor work is still
// small beside the keys and values that come in.  A CTA of four warps, each with a quarter of the keys of every block, and a fifth one
// that fills a ring of blocks.  A warp keeps maximum, sum and accumulator of its own keys; they are put together at the item's end.
//
// The grid is as many CTAs as the chip holds, and the blocks of all items, laid end to end, are dealt to them in equal runs: the
// ring goes on from item to item without a pause, and sequences of any lengths keep every SM equally long.  An item that
// lies in several runs is added up by the CTA that is last with its piece, in the order of the runs.  (One CTA per item and piece of
// 1024 keys: 47 us for 64 sequences of 400 .. 4096 keys and 6 heads of 64, 35 % of it a tail; pieces of 256 keys: 65 us, a start for
// each.)  Where no sequence has more than PA_WHOLE keys, an item is one CTA's and there is nothing to add.
//
// Fragments without a shuffle: the contraction over the head dimension may take the elements in any order, so lane (r, c) of a
// key's fragment (r = lane / 4, c = lane % 4) holds elements 16 c .. 16 c + 15 of key r, two 16-byte reads, and the queries lie
// the same way.  Of a value's rows 2c, 2c + 1, 2c + 8, 2c + 9 it takes elements 8 r .. 8 r + 7, and pairs of two keys are made
// with byte permutes; accumulator tile i then holds elements 8 (2c) + i and 8 (2c + 1) + i of rows r and r + 8.
//
// 8-bit rows of up to 64: as many bytes are twice the keys, and a step of a warp is 32 of them.
// Codes become f16, which holds each of them, against queries in f16 (a row scaled by a power of two).  The exponent e of a value's scale is
// added to the score before the maximum is taken, so that probabilities, which become f16, carry it: p' = 2^(s + e - m), against 2^-13 of
// the largest: at most 2^15 with what is left of the scale, and products of probability and scale down to 2^-38 of the largest count.  The sum
// takes the exponent back, l = sum of p' 2^(B - e) with B the largest exponent of the item's first 32 keys, of those that all its rows see.  That
// holds while every e lies within NEAR of B; behind it p' may be no number that float32 has, and the sum would lose a key whose value is
// small beside another.  Rows that have seen such a key get their sum at the item's end, from the keys once more (64 sequences of 16,000
// keys: 820 us).  Rows of zeros, which have the smallest scale there is (SCALE_LEAST), count as B - NEAR: what is lost is below 2^-117.
//
// Bound: memory; 64 sequences of 16,000 keys, 6 heads of 64: bf16 6.7 TB/s, 8 bits 5.1 TB/s, there by the instructions around the
// conversions (42 % of the issue slots of 12 warps that wait for one another's loads; 120 bytes of registers spilled).  A call of 40 us loses 4 us before its first block is
// there and 2 to 4 us to the spread of its CTAs' ends.
constexpr float PA_UP = 13.f;
// The reference of a row that has seen no key yet, or keys that score minus infinity alone: no score is lower, but it is a number, so that minus
// infinity is below it and not beside it.
constexpr float PA_LOW = -3.402823466e38f;
constexpr int PA_WARPS = 4;
constexpr int PA_THREADS = (PA_WARPS + 1) * 32;
constexpr int PA_SCAN = 4;               // sequences per lane of one look at the batch
enum { PA_FIRST = 1, PA_LAST = 2, PA_FINAL = 4, PA_END = 8 };

template <int NH, bool E4M3>
struct RowsShape {
    static constexpr int KEYS = paged_keys(NH, E4M3), KW = KEYS / PA_WARPS;      // keys per block and per warp
    static constexpr int ROW_BYTES = E4M3 ? 64 * NH : 128;                   // of one 64-element (8 bits: all) column block
    static constexpr int BLOCK = KEYS * ROW_BYTES;                           // one column block of a block's keys
    static constexpr int TILE = E4M3 ? BLOCK : NH * BLOCK;
    static constexpr int STAGES = NH == 2 ? (E4M3 ? 3 : 2) : (E4M3 ? 2 : 4);
    static constexpr int Q_BYTES = PA_ROWS * 128 * NH, WHAT = 32, SCALES = E4M3 ? 2 * KEYS * 4 : 0;
    static constexpr int LD = 64 * NH + 4;                                   // floats per row of a warp's result
    // ring of keys and values | scales | queries of an item's first block | what a block is | scale parts of a warp | results | barriers
    static constexpr int STAGE = 2 * TILE;
    static constexpr int O_SCALE = STAGES * STAGE, O_Q = O_SCALE + STAGES * SCALES, O_WHAT = O_Q + STAGES * Q_BYTES;
    static constexpr int O_PARTS = O_WHAT + STAGES * WHAT;
    static constexpr int O_OUT = O_PARTS + (E4M3 ? KEYS * 16 : 0);
    static constexpr int O_BARS = O_OUT + PA_WARPS * PA_ROWS * (LD + 2) * 4;
    static constexpr int SMEM = 1024 + O_BARS + 2 * STAGES * 8 + 16;
    static constexpr int PER_SM = SMEM <= 75 * 1024 ? 3 : SMEM <= 113 * 1024 ? 2 : 1;
};

__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, std::false_type) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, std::true_type) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// two 8-bit codes (low half of the word) -> a pair of f16, exact
__device__ __forceinline__ uint32_t e4m3_f16(uint32_t two) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)two));
    return h;
}
__device__ __forceinline__ uint32_t e5m2_pair(float lo, float hi) {
    uint16_t h;
    asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(h) : "f"(hi), "f"(lo));
    return h;
}
__device__ __forceinline__ float2 f16_floats(uint32_t two) { return __half22float2(*reinterpret_cast<const __half2*>(&two)); }
__device__ __forceinline__ uint32_t f16_pair(float lo, float hi) {
    uint32_t h;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(h) : "f"(hi), "f"(lo));
    return h;
}
// 2^n for n from -126 to 127
__device__ __forceinline__ float power_of_two(int n) { return __uint_as_float((uint32_t)(127 + n) << 23); }
// The exponent of a value's scale as float32 keeps it: a scale is 2^(exponent - 127) * part with |part| < 2, below 4 where it is above 2^126.
// 0: infinity or NaN, their own part with any exponent.
constexpr int NEAR = 40;
constexpr float SCALE_LEAST = 0x1p-126f;
__device__ __forceinline__ int scale_exponent(float s) {
    const int e = (int)(__float_as_uint(s) >> 23) & 255;
    return e == 255 ? 0 : min(max(e, 1), 253);
}
// a sum of 2^x and the largest x, put together with another one
__device__ __forceinline__ void add_sums(float2& to, float2 x) {
    const float top = fmaxf(to.x, x.x), base = top == -INFINITY ? 0.f : top;
    to = make_float2(top, to.y * ex2_approx(to.x - base) + x.y * ex2_approx(x.x - base));
}

// an arrival when this thread's copies so far are there (the barrier's count has room for it)
__device__ __forceinline__ void copy_async_arrive(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// A named barrier for the warps that wait for one another: whether all of them say so.  (A warp whose wait ran out comes here too and says
// no, so that nobody waits for it.)
__device__ __forceinline__ bool all_of(bool mine, int barrier, int threads) {
    int whole;
    asm volatile("{\n\t.reg .pred P, Q;\n\tsetp.ne.s32 P, %1, 0;\n\tbar.red.and.pred Q, %2, %3, P;\n\tselp.s32 %0, 1, 0, Q;\n\t}"
                 : "=r"(whole) : "r"(mine ? 1 : 0), "r"(barrier), "r"(threads) : "memory");
    return whole != 0;
}

// blocks of one head of a sequence that the kernel for few rows takes
template <int KEYS>
__device__ __forceinline__ int row_blocks(const PagedAttParams& p, bool ok, int n, int kv) {
    return ok && n > 0 && n * p.group <= PA_ROWS ? max(1, (kv + KEYS - 1) / KEYS) : 0;
}

// A page outside the pool: what takes the place of its keys is NaN (as bf16 and as 8-bit codes), of its values zeros.  Rows that see such a key are
// NaN, and no other sequence's values are in them.  By a whole warp; `bad` has a bit for each of the block's pieces; the fence is for the
// tensor cores, and for the copies that overwrite this next.  (A call: inside its loop it cost single tokens in pages of 16 keys 5 %.)
constexpr uint32_t PA_NAN = 0x7fff7fffu;
__device__ __noinline__ void fill_pieces(uint8_t* tile, unsigned bad, int piece_bytes, uint32_t word) {
    const int lane = threadIdx.x & 31;
    for (; bad != 0u; bad &= bad - 1u)
        for (int x = lane * 16; x < piece_bytes; x += 32 * 16)
            *reinterpret_cast<uint4*>(tile + (__ffs(bad) - 1) * piece_bytes + x) = make_uint4(word, word, word, word);
    fence_proxy_async();
    __syncwarp();
}

template <int NH, bool E4M3>
__global__ void __launch_bounds__(PA_THREADS, (RowsShape<NH, E4M3>::PER_SM))
paged_rows_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const PagedAttParams p) {
    typedef RowsShape<NH, E4M3> Sh;
    typedef std::integral_constant<bool, E4M3> Kind;
    constexpr int STAGES = Sh::STAGES, KEYS = Sh::KEYS, KW = Sh::KW, NT = KW / 8;
    constexpr int KEYS_LOG2 = KEYS == 128 ? 7 : 6;
    static_assert(KEYS == 1 << KEYS_LOG2, "");
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + Sh::O_BARS);
    uint64_t* empty = full + STAGES;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(empty + STAGES);
    volatile int* is_last = abort_flag + 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        // (8 bits: the scales come by the lanes' own copies, each with an arrival of its own)
        for (int i = 0; i < STAGES; ++i) { mbar_init(&full[i], E4M3 ? 33 : 1); mbar_init(&empty[i], PA_WARPS); }
        *abort_flag = 0;
        fence_mbar_init();
    }
    __syncthreads();
    if (!p.behind_chunks) pdl_wait();    // (the tiles' kernel has waited itself before it let this one start)

    if (warp == PA_WARPS) {
        // ---- producer: finds this CTA's items, and fills the ring with their blocks.  A lane per piece of a page.
        const int heads = p.v.heads, seqs = p.v.seqs;
        const int piece_shift = min(p.v.page_shift, KEYS_LOG2), pieces = KEYS >> piece_shift;   // keys per copy, copies per block
        const int piece_keys = 1 << piece_shift, per_page_shift = p.v.page_shift - piece_shift;
        int s = 0, h = 0, b = 0;              // the next block: of sequence s, head h
        long long left = 0, at_block = 0, per = 1;      // blocks of this CTA's run that are still to come; the next one's number; a run
        if (p.whole) {
            s = (int)(blockIdx.x / (unsigned)heads);
            h = (int)(blockIdx.x % (unsigned)heads);
        } else {
            // all sequences' blocks: lane i looks at PA_SCAN sequences in a row
            int nb[PA_SCAN];
            auto look = [&](int s0, long long& mine) {
                int q[PA_SCAN + 1], kv[PA_SCAN];
                const int a = s0 + lane * PA_SCAN;
#pragma unroll
                for (int i = 0; i <= PA_SCAN; ++i) q[i] = p.q_start[min(a + i, seqs)];
#pragma unroll
                for (int i = 0; i < PA_SCAN; ++i) kv[i] = p.kv_len[min(a + i, seqs - 1)];
                mine = 0;
#pragma unroll
                for (int i = 0; i < PA_SCAN; ++i) {
                    const bool ok = batch_ok(p, q[i], q[i + 1], kv[i]);
                    if (!ok && a + i < seqs) report_argument(p.err, 76);
                    nb[i] = a + i < seqs ? row_blocks<KEYS>(p, ok, q[i + 1] - q[i], kv[i]) : 0;
                    mine += nb[i];
                }
                long long incl = mine;
                for (int o = 1; o < 32; o <<= 1) {
                    const long long x = __shfl_up_sync(0xffffffffu, incl, o);
                    if (lane >= o) incl += x;
                }
                return incl;
            };
            long long total = 0, mine, incl = 0;
            for (int s0 = 0; s0 < seqs; s0 += 32 * PA_SCAN) {
                incl = look(s0, mine);
                total += __shfl_sync(0xffffffffu, incl, 31);
            }
            total *= heads;
            const int runs = p.runs ? min(max(__ldcg(p.runs), 1), p.grid) : p.grid;
            per = max((total + runs - 1) / runs, (long long)(PA_LEAST >> KEYS_LOG2));
            at_block = per * blockIdx.x;
            left = min(per, total - at_block);
            if (left > 0) {
                long long before = 0;
                for (int s0 = 0; s0 < seqs; s0 += 32 * PA_SCAN) {
                    if (seqs > 32 * PA_SCAN) incl = look(s0, mine);
                    const unsigned ends_behind = __ballot_sync(0xffffffffu, (before + incl) * heads > at_block);
                    if (ends_behind) {
                        const int who = __ffs(ends_behind) - 1;
                        long long rest = at_block - (before + incl - mine) * heads;      // (of the lane that has it)
                        int i = 0;
#pragma unroll
                        for (int x = 0; x < PA_SCAN - 1; ++x)
                            if (i == x && rest >= (long long)nb[x] * heads) { rest -= (long long)nb[x] * heads; ++i; }
                        int blocks = nb[0];
#pragma unroll
                        for (int x = 1; x < PA_SCAN; ++x) blocks = i == x ? nb[x] : blocks;
                        blocks = max(blocks, 1);
                        h = (int)(rest / blocks); b = (int)(rest - (long long)h * blocks); s = s0 + lane * PA_SCAN + i;
                        s = __shfl_sync(0xffffffffu, s, who); h = __shfl_sync(0xffffffffu, h, who); b = __shfl_sync(0xffffffffu, b, who);
                        break;
                    }
                    before += __shfl_sync(0xffffffffu, incl, 31);
                }
            }
        }
        int i = 0;                            // blocks put into the ring
        bool ok = true;
        auto slot_free = [&]() {
            if (i >= STAGES) ok = mbar_wait(&empty[i % STAGES], (uint32_t)((i / STAGES) & 1) ^ 1u, abort_flag);
            ok = __all_sync(0xffffffffu, ok);
            return ok;
        };
        while (ok && s < seqs && (p.whole || left > 0)) {
            int q0, n, kv;
            const bool fine = batch_of(p, s, q0, n, kv);
            if (!fine && p.whole && lane == 0) report_argument(p.err, 76);
            const int blocks = row_blocks<KEYS>(p, fine, n, kv);
            const int b_end = p.whole ? blocks : (int)min((long long)blocks, b + left);
            const int* table = p.v.table + (long long)s * p.v.table_ld;
            const int last_piece = (kv + piece_keys - 1) >> piece_shift;
            auto page_at = [&](int piece) -> int {
                if (piece >= last_piece) return 0;
                const int pg = table[piece >> per_page_shift];
                if ((unsigned)pg < (unsigned)p.v.pages) return pg;
                report_argument(p.err, 75);
                return -1;
            };
            // the table is read 32 pieces at a time, one round ahead
            int held = b * pieces, now = 0, next = 0;
            if (b < b_end) { now = page_at(held + lane); next = page_at(held + 32 + lane); }
            int c0 = 0, runs = 1;             // the run that the item begins in, and how many it lies in
            if (!p.whole && b < b_end) {
                c0 = (int)((at_block - b) / per);
                runs = (int)((at_block - b + blocks - 1) / per) - c0 + 1;
            }
            const int b_begin = b;
            bool any_bad = __any_sync(0xffffffffu, now < 0);
            for (; b < b_end; ++b) {
                const int at = b * pieces;
                if (at >= held + 32) { held += 32; now = next; next = page_at(held + 32 + lane); any_bad = __any_sync(0xffffffffu, now < 0); }
                const int pg = __shfl_sync(0xffffffffu, now, (at - held + lane) & 31);
                const int count = max(0, min(pieces, last_piece - at));      // copies of this block
                if (!slot_free()) break;
                const int st = i % STAGES;
                uint8_t* tile = smem + st * Sh::STAGE;
                uint64_t* bar = &full[st];
                const bool first = b == b_begin;
                int copies = count;
                if (any_bad) {
                    const unsigned bad = __ballot_sync(0xffffffffu, lane < count && pg < 0);
                    copies -= __popc(bad);
                    for (int c = 0; c < (E4M3 ? 1 : NH); ++c) {
                        fill_pieces(tile + c * Sh::BLOCK, bad, piece_keys * Sh::ROW_BYTES, PA_NAN);
                        fill_pieces(tile + Sh::TILE + c * Sh::BLOCK, bad, piece_keys * Sh::ROW_BYTES, 0u);
                    }
                }
                if (lane == 0) {
                    int4* what = reinterpret_cast<int4*>(smem + Sh::O_WHAT + st * Sh::WHAT);
                    what[0] = make_int4((first ? PA_FIRST : 0) | (b == b_end - 1 ? PA_LAST : 0) | (runs == 1 ? PA_FINAL : 0) | s << 16, b * KEYS, q0, n);
                    what[1] = make_int4(kv, h, c0, runs);
                    mbar_expect_tx(bar, (uint32_t)(copies * piece_keys * (2 * Sh::TILE / KEYS) + (first ? n * p.group * p.v.hd * 2 : 0)));
                }
                __syncwarp();
                if (first && lane < n)
                    bulk_load(smem + Sh::O_Q + st * Sh::Q_BYTES + lane * p.group * p.v.hd * 2,
                              p.Q + (long long)(q0 + lane) * p.ld_q + (long long)h * p.group * p.v.hd, (uint32_t)(p.group * p.v.hd * 2), bar);
                if (lane < count && pg >= 0) {
                    const int block = pg * heads + h, r0 = ((at + lane) & ((1 << per_page_shift) - 1)) << piece_shift;
                    const int o = lane << piece_shift;
#pragma unroll
                    for (int c = 0; c < (E4M3 ? 1 : NH); ++c) {
                        tma_load_3d(tile + c * Sh::BLOCK + o * Sh::ROW_BYTES, &tmK, bar, c * 64, r0, block);
                        tma_load_3d(tile + Sh::TILE + c * Sh::BLOCK + o * Sh::ROW_BYTES, &tmV, bar, c * 64, r0, block);
                    }
                }
                if (E4M3) {
                    // four scales per copy: of keys, then of values.  (A bulk copy per piece of a page and array: 225 us instead of 192 for
                    // 64 sequences of 16,000 keys in pages of 16, 6 heads of 64; as fast in pages of 64.)
                    float* sc = reinterpret_cast<float*>(smem + Sh::O_SCALE + st * Sh::SCALES);
#pragma unroll
                    for (int x = 0; x < KEYS / 64; ++x) {
                        const int four = x * 32 + lane, key = (four & (KEYS / 4 - 1)) * 4, piece = key >> piece_shift;
                        const int block = max(__shfl_sync(0xffffffffu, pg, piece), 0) * heads + h;       // (no matter which, beside codes of NaN and 0)
                        const int r0 = (((at + piece) & ((1 << per_page_shift) - 1)) << piece_shift) + (key & (piece_keys - 1));
                        if (piece < count) copy_async16(sc + four * 4, (four < KEYS / 4 ? p.ks : p.vs) + ((long long)block << p.v.page_shift) + r0);
                    }
                    copy_async_arrive(bar);
                }
                __syncwarp();
                ++i;
            }
            if (p.whole) {
                b = 0;
                h += (int)(gridDim.x % (unsigned)heads);
                s += (int)(gridDim.x / (unsigned)heads);
                if (h >= heads) { h -= heads; ++s; }
            } else {
                left -= b - b_begin;
                at_block += b - b_begin;
                if (b >= blocks) {
                    b = 0;
                    if (blocks == 0 || ++h == heads) { h = 0; ++s; }
                }
            }
        }
        if (ok && slot_free() && (lane == 0 || E4M3)) {
            if (E4M3) mbar_arrive(&full[i % STAGES]);
            if (lane == 0) *reinterpret_cast<int*>(smem + Sh::O_WHAT + (i % STAGES) * Sh::WHAT) = PA_END;
            if (lane == 0) mbar_arrive(&full[i % STAGES]);
        }
        if (p.behind_chunks) pdl_wait();     // what follows finds the tiles' rows as well
        pdl_launch_dependents_now();
        if (!ok && lane == 0) { *abort_flag = 1; atomicExch(p.err, 73); }
        // (the consumers wait for everything that has been asked for)
        return;
    }

    const int r = lane >> 2, c = lane & 3;
    float* so = reinterpret_cast<float*>(smem + Sh::O_OUT);
    float2* sml = reinterpret_cast<float2*>(so + PA_WARPS * PA_ROWS * Sh::LD);
    float4* parts = reinterpret_cast<float4*>(smem + Sh::O_PARTS) + warp * KW;     // (8 bits) of this warp's keys
    // query fragments: elements 16 c .. of rows r and r + 8, head-dimension block by block
    uint32_t qf[NH][4][4];
    float row_factor[2] = {p.scale_log2, p.scale_log2};
    int pos[2] = {0, 0}, first_pos = 0, last_pos = 0, nrows = 0;
    float o[8 * NH][4], m[2], l[2];
    bool ok = true;
    int st = 0;
    uint32_t phase = 0;
    // (8 bits) what a warp knows of its item lies where the item's result goes at its end: B, the first key, the first one with a value's scale
    // far from B (which concerns the rows that see it)
    int* known = reinterpret_cast<int*>(so + warp * PA_ROWS * Sh::LD);
    enum { K_BASE, K_FIRST, K_FAR };
    for (;;) {
        if (!mbar_wait(&full[st], phase, abort_flag)) {
            if (lane == 0) *abort_flag = 1;
            all_of(false, 1, 128);
            ok = false;
            break;
        }
        const uint8_t* sK = smem + st * Sh::STAGE;
        const uint8_t* sV = sK + Sh::TILE;
        const int4 what = *reinterpret_cast<const int4*>(smem + Sh::O_WHAT + st * Sh::WHAT);           // flags and sequence, first key, first row, new rows
        if (what.x & PA_END) { all_of(true, 1, 128); break; }
        const int4 more = *reinterpret_cast<const int4*>(smem + Sh::O_WHAT + st * Sh::WHAT + 16);      // keys, head, first run, runs
        const int kv = more.x, n = what.w;
        if (what.x & PA_FIRST) {
            nrows = n * p.group;
            first_pos = kv - n; last_pos = kv - 1;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int rr = r + 8 * x;
                pos[x] = kv - n + (int)((uint32_t)min(rr, nrows - 1) * p.group_magic >> 16);
                const uint8_t* q = smem + Sh::O_Q + st * Sh::Q_BYTES + rr * p.v.hd * 2;
                uint32_t big = 0u;
#pragma unroll
                for (int b = 0; b < NH; ++b)
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        const int e = 64 * b + 16 * c + 8 * g;
                        uint4 w = make_uint4(0u, 0u, 0u, 0u);
                        if (e < p.v.hd && rr < nrows) w = *reinterpret_cast<const uint4*>(q + e * 2);
                        qf[b][2 * g][x] = w.x; qf[b][2 * g][2 + x] = w.y; qf[b][2 * g + 1][x] = w.z; qf[b][2 * g + 1][2 + x] = w.w;
                        if (E4M3) {
                            const uint32_t a = __vmaxu2(__vmaxu2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu), __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu));
                            big = max(big, max(a & 0xffffu, a >> 16));
                        }
                    }
                if (E4M3) {
                    // as f16, the row scaled by a power of two so that its largest magnitude lies in [1, 2), or below 4: exact but for
                    // what is less than 2^-24 of it
                    big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
                    big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
                    const bool odd = big >> 7 == 255u;                                 // (an infinity or NaN)
                    const int e = min(max((int)(big >> 7), 1), 253);                   // (2^(127 - e) and its inverse are normal numbers)
                    const float down = power_of_two(127 - e), up = power_of_two(e - 127);
                    row_factor[x] = odd ? p.scale_log2 : p.scale_log2 * up;
#pragma unroll
                    for (int b = 0; b < NH; ++b)
#pragma unroll
                        for (int g = 0; g < 4; ++g)
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                const float2 f = bf16_floats(qf[b][g][x + 2 * j]);
                                qf[b][g][x + 2 * j] = odd ? f16_pair(f.x, f.y) : f16_pair(f.x * down, f.y * down);
                            }
                }
                m[x] = PA_LOW; l[x] = 0.f;
            }
            if (E4M3) {
                const float vs = reinterpret_cast<const float*>(smem + Sh::O_SCALE + st * Sh::SCALES)[KEYS + lane];
                const int base = __reduce_max_sync(0xffffffffu, (lane == 0 || what.y + lane <= first_pos) && vs > SCALE_LEAST ? scale_exponent(vs) : 0);
                if (lane <= K_FAR) known[lane] = lane == K_BASE ? max(base, 1) : lane == K_FIRST ? what.y : 0x7fffffff;
                __syncwarp();
            }
#pragma unroll
            for (int e = 0; e < 8 * NH; ++e) { o[e][0] = 0.f; o[e][1] = 0.f; o[e][2] = 0.f; o[e][3] = 0.f; }
        }
        const int kk = KW * warp, k0 = what.y + kk;                        // this warp's keys
        // One step: this warp's keys of the block.  at_edge: some row does not see all of them.
        auto step = [&](auto at_edge) {
            constexpr bool edge = decltype(at_edge)::value;
            if (E4M3) {
                // a lane per key: what the scales do to scores, probabilities and sums
                const float* sc = reinterpret_cast<const float*>(smem + Sh::O_SCALE + st * Sh::SCALES) + kk;
                if (lane < KW) {
                    const float vs = sc[KEYS + lane];
                    const int B = known[K_BASE];
                    int e = scale_exponent(vs);
                    e = e == 0 ? B : vs == SCALE_LEAST ? max(B - NEAR, 1) : e;
                    const int off = e - B, near = min(max(off, -NEAR), NEAR);
                    parts[lane] = make_float4(sc[lane], __uint_as_float(0x4b000000u | (uint32_t)e) - 8388735.0f /* e - 127 */, vs * power_of_two(127 - e),
                                              power_of_two(-near));
                    if (off != near) atomicMin(known + K_FAR, k0 + lane);
                }
                __syncwarp();
            }
            float z[NT][4];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                z[t][0] = z[t][1] = z[t][2] = z[t][3] = 0.f;
                const int key = kk + 8 * t + r;
#pragma unroll
                for (int b = 0; b < NH; ++b) {
                    uint32_t w[8];
                    if (E4M3) {
                        const uint4 x = *reinterpret_cast<const uint4*>(sK + key * Sh::ROW_BYTES + 64 * b + 16 * c);
                        const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) { w[2 * e] = e4m3_f16(u[e]); w[2 * e + 1] = e4m3_f16(u[e] >> 16); }
                    } else {
                        // (128-byte swizzle: the 16-byte pieces of a row lie at piece ^ (row & 7))
                        const uint8_t* row = sK + b * Sh::BLOCK + key * 128;
                        const uint4 x = *reinterpret_cast<const uint4*>(row + (((2 * c) ^ (key & 7)) << 4));
                        const uint4 y = *reinterpret_cast<const uint4*>(row + (((2 * c + 1) ^ (key & 7)) << 4));
                        w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w; w[4] = y.x; w[5] = y.y; w[6] = y.z; w[7] = y.w;
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) mma_16816(z[t], qf[b][e], w[2 * e], w[2 * e + 1], Kind());
                }
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                if (E4M3) {
                    // the key's scale on the score; the value's scale, but for a factor below 2, in the exponent of the probability
                    const float4 f = parts[8 * t + 2 * c], g = parts[8 * t + 2 * c + 1];
                    z[t][0] = fmaf(z[t][0], f.x * row_factor[0], f.y); z[t][1] = fmaf(z[t][1], g.x * row_factor[0], g.y);
                    z[t][2] = fmaf(z[t][2], f.x * row_factor[1], f.y); z[t][3] = fmaf(z[t][3], g.x * row_factor[1], g.y);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) z[t][e] *= p.scale_log2;
                }
                if (edge) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (k0 + 8 * t + 2 * c + (e & 1) > pos[e >> 1]) z[t][e] = -INFINITY;
                }
            }
            // ---- running maximum and sum
            bool moved = false;
            float alpha[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float mx = fmaxf(z[0][2 * h], z[0][2 * h + 1]);
#pragma unroll
                for (int t = 1; t < NT; ++t) mx = fmaxf(mx, fmaxf(z[t][2 * h], z[t][2 * h + 1]));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const float mn = fmaxf(m[h], E4M3 ? mx - PA_UP : mx);
                alpha[h] = mn > m[h] ? ex2_approx(m[h] - mn) : 1.0f;
                moved |= mn > m[h];
                m[h] = mn;
            }
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                for (int h = 0; h < 2; ++h) l[h] *= alpha[h];
#pragma unroll
                for (int t = 0; t < 8 * NH; ++t) { o[t][0] *= alpha[0]; o[t][1] *= alpha[0]; o[t][2] *= alpha[1]; o[t][3] *= alpha[1]; }
            }
            uint32_t pa[NT / 2][4];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                float4 f = make_float4(0.f, 0.f, 1.f, 1.f), g = f;
                if (E4M3) { f = parts[8 * t + 2 * c]; g = parts[8 * t + 2 * c + 1]; }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float p0 = ex2_approx(z[t][2 * h] - m[h]), p1 = ex2_approx(z[t][2 * h + 1] - m[h]);
                    if (E4M3) {
                        // (a key that the row does not see may have any scale)
                        const bool no0 = edge && z[t][2 * h] == -INFINITY, no1 = edge && z[t][2 * h + 1] == -INFINITY;
                        l[h] += (no0 ? 0.f : p0 * f.w) + (no1 ? 0.f : p1 * g.w);
                        p0 = no0 ? 0.f : p0 * f.z;
                        p1 = no1 ? 0.f : p1 * g.z;
                        pa[t / 2][2 * (t & 1) + h] = f16_pair(p0, p1);
                    } else {
                        l[h] += p0 + p1;
                        pa[t / 2][2 * (t & 1) + h] = bf16_pair(p0, p1);
                    }
                }
            }
            // ---- values
            // at an edge: keys behind position `last` count as zeros, and only the rows of that position take the product
            auto values = [&](int last) {
#pragma unroll
                for (int half = 0; half < NT / 2; ++half) {
                    uint32_t a[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) a[j] = !edge || pos[j & 1] == last ? pa[half][j] : 0u;
#pragma unroll
                    for (int b = 0; b < NH; ++b) {
                        uint32_t w[4][4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int key = kk + 16 * half + 2 * c + (j & 1) + 8 * (j >> 1);
                            const bool seen = !edge || what.y + key <= last;
                            if (E4M3) {
                                uint2 x = *reinterpret_cast<const uint2*>(sV + key * Sh::ROW_BYTES + 64 * b + 8 * r);
                                if (!seen) x = make_uint2(0u, 0u);
                                w[j][0] = x.x; w[j][1] = x.y;
                            } else {
                                uint4 x = *reinterpret_cast<const uint4*>(sV + b * Sh::BLOCK + key * 128 + ((r ^ (key & 7)) << 4));
                                if (!seen) x = make_uint4(0u, 0u, 0u, 0u);
                                w[j][0] = x.x; w[j][1] = x.y; w[j][2] = x.z; w[j][3] = x.w;
                            }
                        }
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            uint32_t b0, b1;
                            if (E4M3) {
                                // byte e of two keys side by side
                                const uint32_t sel = 0x0040u + 0x0011u * (e & 3);
                                b0 = e4m3_f16(__byte_perm(w[0][e >> 2], w[1][e >> 2], sel));
                                b1 = e4m3_f16(__byte_perm(w[2][e >> 2], w[3][e >> 2], sel));
                            } else {
                                const uint32_t sel = e & 1 ? 0x7632u : 0x5410u;
                                b0 = __byte_perm(w[0][e >> 1], w[1][e >> 1], sel);
                                b1 = __byte_perm(w[2][e >> 1], w[3][e >> 1], sel);
                            }
                            if (!edge) {
                                mma_16816(o[8 * b + e], a, b0, b1, Kind());
                            } else {
                                float d[4] = {0.f, 0.f, 0.f, 0.f};
                                mma_16816(d, a, b0, b1, Kind());
                                if (pos[0] == last) { o[8 * b + e][0] += d[0]; o[8 * b + e][1] += d[1]; }
                                if (pos[1] == last) { o[8 * b + e][2] += d[2]; o[8 * b + e][3] += d[3]; }
                            }
                        }
                    }
                }
            };
            if (!edge) values(0);
            else       // token by token: what a token does not see must not reach it, not even as 0 * infinity
#pragma unroll 1
                for (int last = max(first_pos, 0); last <= last_pos; ++last) values(last);
        };
        if (k0 <= last_pos) {
            if (k0 + KW - 1 > first_pos) step(std::true_type());
            else step(std::false_type());
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[st]);
        if (++st == STAGES) { st = 0; phase ^= 1u; }
        if (!(what.x & PA_LAST)) continue;

        // ---- the item's end: the four warps' results, [warp][16 rows][LD] floats, maxima and sums behind.  (8 bits: what leaves the CTA, or the
        // kernel, are means of values and sums in units of scores alone: other parts of the item have other B.)
        int B = 0;
        bool far[2] = {false, false};
        float2 sum[2];                                                     // of rows that have seen a key far from B: the largest score and the sum
        if (E4M3) {
            B = known[K_BASE];
#pragma unroll
            for (int h = 0; h < 2; ++h) { far[h] = pos[h] >= known[K_FAR]; sum[h] = make_float2(-INFINITY, 0.f); }
            if (__any_sync(0xffffffffu, far[0] || far[1])) {
                const int first_key = known[K_FIRST];
                const int* table = p.v.table + (long long)((uint32_t)what.x >> 16) * p.v.table_ld;
#pragma unroll 1
                for (int t0 = first_key + kk; t0 <= min(k0, last_pos); t0 += KEYS) {
#pragma unroll 1
                    for (int t = 0; t < KW; t += 8) {
                        // (lane (r, c): elements 16 c .. of key t0 + t + r; products with keys t0 + t + 2 c and the next)
                        __syncwarp();
                        auto row_of = [&](int key) -> long long {
                            const int page = key <= last_pos ? table[key >> p.v.page_shift] : -1;
                            if ((unsigned)page >= (unsigned)p.v.pages) return -1;
                            return (((long long)page * p.v.heads + more.y) << p.v.page_shift) + (key & ((1 << p.v.page_shift) - 1));
                        };
                        const long long row = row_of(t0 + t + r);
                        float z[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int b = 0; b < NH; ++b) {
                            uint4 x = make_uint4(0u, 0u, 0u, 0u);
                            if (row >= 0 && 64 * b + 16 * c < p.v.hd) x = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p.K) + row * p.v.hd + 64 * b + 16 * c);
                            const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                            for (int e = 0; e < 4; ++e) mma_16816(z, qf[b][e], e4m3_f16(u[e]), e4m3_f16(u[e] >> 16), Kind());
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int key = t0 + t + 2 * c + (e & 1);
                            if (key > pos[e >> 1]) continue;
                            const long long at = row_of(key);
                            const float scale = at < 0 ? __uint_as_float(0x7fffffffu) : p.ks[at];        // (a page outside the pool: NaN)
                            add_sums(sum[e >> 1], make_float2(z[e] * (scale * row_factor[e >> 1]), 1.f));
                        }
                    }
                }
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int x = 1; x < 4; x <<= 1) add_sums(sum[h], make_float2(__shfl_xor_sync(0xffffffffu, sum[h].x, x), __shfl_xor_sync(0xffffffffu, sum[h].y, x)));
                __syncwarp();
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
            float* dst = so + (warp * PA_ROWS + r + 8 * h) * Sh::LD + 16 * c;
#pragma unroll
            for (int b = 0; b < NH; ++b)
#pragma unroll
                for (int e = 0; e < 8; e += 4) {
                    *reinterpret_cast<float4*>(dst + 64 * b + e) =
                        make_float4(o[8 * b + e][2 * h], o[8 * b + e + 1][2 * h], o[8 * b + e + 2][2 * h], o[8 * b + e + 3][2 * h]);
                    *reinterpret_cast<float4*>(dst + 64 * b + 8 + e) =
                        make_float4(o[8 * b + e][2 * h + 1], o[8 * b + e + 1][2 * h + 1], o[8 * b + e + 2][2 * h + 1], o[8 * b + e + 3][2 * h + 1]);
                }
            if (c == 0) {
                float2 ml = make_float2(m[h], l[h]);
                if (E4M3 && far[h]) {
                    // behind the row, what makes a mean of its values where the sum is against another reference, in two factors; the sum's sign says so
                    const float half = ex2_approx(0.5f * (m[h] - sum[h].x));
                    *reinterpret_cast<float2*>(so + (warp * PA_ROWS + r + 8 * h) * Sh::LD + 64 * NH) = make_float2(half / sum[h].y, half);
                    ml = make_float2(sum[h].x, -sum[h].y);
                }
                sml[warp * PA_ROWS + r + 8 * h] = ml;
            }
        }
        if (!all_of(true, 1, 128)) { ok = false; break; }
        const int chunks = p.v.hd >> 3, points = nrows * chunks;           // eight elements per thread
        auto finish = [&](int rr, int e, float M, float L, const float (&acc)[8]) {
            const int tok = rr / p.group, hq = more.y * p.group + (rr - tok * p.group), row = what.z + tok;
            const bool none = kv - n + tok < 0;                            // a row without a key
            const float inv = none ? 0.f : E4M3 ? (L == 0.f ? __uint_as_float(0x7fffffffu) : 1.0f) : 1.0f / L;        // (8 bits: means already)
            *reinterpret_cast<uint4*>(p.att + (long long)row * p.ld_att + (long long)hq * p.v.hd + e) =
                make_uint4(bf16_pair(acc[0] * inv, acc[1] * inv), bf16_pair(acc[2] * inv, acc[3] * inv),
                           bf16_pair(acc[4] * inv, acc[5] * inv), bf16_pair(acc[6] * inv, acc[7] * inv));
            if (p.lse && e == 0) p.lse[(long long)row * p.H + hq] = none ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
        };
        auto add = [](auto means, float& M, float& L, float (&acc)[8], float2 ml, const float4& a, const float4& d) {
            if (ml.y == 0.f) return;                                       // (no key of this part was visible)
            const float mn = L == 0.f ? ml.x : fmaxf(M, ml.x);
            float f = L == 0.f ? 0.f : ex2_approx(M - mn), g = ex2_approx(ml.x - mn);
            if (decltype(means)::value) {
                f *= L; g *= ml.y;
                L = f + g;
                const float inv = __fdividef(1.0f, L);
                f *= inv; g *= inv;
            } else {
                L = L * f + ml.y * g;
            }
            M = mn;
            const float x[8] = {a.x, a.y, a.z, a.w, d.x, d.y, d.z, d.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i] = (f == 0.f ? 0.f : acc[i] * f) + x[i] * g;
        };
        for (int x = threadIdx.x; x < points; x += PA_WARPS * 32) {
            const int rr = x / chunks, e = (x - rr * chunks) * 8;
            float M = -INFINITY, L = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            float2 ml[PA_WARPS];
            bool any_far = false;
#pragma unroll
            for (int w = 0; w < PA_WARPS; ++w) { ml[w] = sml[w * PA_ROWS + rr]; any_far |= E4M3 && ml[w].y < 0.f; }
            if (!any_far) {
#pragma unroll
                for (int w = 0; w < PA_WARPS; ++w) {
                    const float4* src = reinterpret_cast<const float4*>(so + (w * PA_ROWS + rr) * Sh::LD + e);
                    add(std::false_type(), M, L, acc, ml[w], src[0], src[1]);
                }
                if (E4M3) {
                    const float a = L == 0.f ? 0.f : __fdividef(1.0f, L), b = power_of_two(B - 127);
#pragma unroll
                    for (int i = 0; i < 8; ++i) acc[i] = acc[i] * a * b;
                    M -= (float)(B - 127);
                }
            } else {
#pragma unroll 1
                for (int w = 0; w < PA_WARPS; ++w) {
                    const float4* src = reinterpret_cast<const float4*>(so + (w * PA_ROWS + rr) * Sh::LD + e);
                    float2 its = sml[w * PA_ROWS + rr], f;
                    if (its.y < 0.f) {
                        f = *reinterpret_cast<const float2*>(so + (w * PA_ROWS + rr) * Sh::LD + 64 * NH);
                        its.y = -its.y;
                    } else {
                        f = make_float2(1.0f / its.y, power_of_two(B - 127));
                        its.x -= (float)(B - 127);
                    }
                    const float4 x = src[0], y = src[1];
                    add(std::true_type(), M, L, acc, its, make_float4(x.x * f.x * f.y, x.y * f.x * f.y, x.z * f.x * f.y, x.w * f.x * f.y),
                        make_float4(y.x * f.x * f.y, y.y * f.x * f.y, y.z * f.x * f.y, y.w * f.x * f.y));
                }
            }
            if (what.x & PA_FINAL) {
                finish(rr, e, M, L, acc);
            } else {
                const int slot = (2 * blockIdx.x + ((int)blockIdx.x == more.z ? 1 : 0)) * PA_ROWS + rr;
                float4* dst = reinterpret_cast<float4*>(p.part_o + (long long)slot * p.v.hd + e);
                __stcg(dst, make_float4(acc[0], acc[1], acc[2], acc[3]));
                __stcg(dst + 1, make_float4(acc[4], acc[5], acc[6], acc[7]));
                if (e == 0) __stcg(p.part_ml + slot, make_float2(M, L));
            }
        }
        if (what.x & PA_FINAL) {
            asm volatile("bar.sync 1, 128;" ::: "memory");                 // the buffer is read
            continue;
        }
        // ---- an item of several runs: whoever is last with its piece adds them, in the order of the runs.  The run that the item begins
        // in has it in slot 1 of its CTA, the others in slot 0.
        asm volatile("bar.sync 1, 128;" ::: "memory");
        if (threadIdx.x == 0) {
            __threadfence();                                               // (everyone's piece, before the count)
            const unsigned int before = atomicAdd(p.arrived + more.z, 1u);
            *is_last = before == (unsigned int)more.w - 1u ? 1 : 0;
            if (*is_last) p.arrived[more.z] = 0u;                          // ready for the next launch
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
        if (!*is_last) continue;
        __threadfence();
        // threads in groups, each with every groups-th piece; then the groups' results
        const int groups = points <= 128 ? 128 / points : 1;
        for (int x0 = threadIdx.x; x0 < (points <= 128 ? groups * points : points); x0 += PA_WARPS * 32) {
            const int g = points <= 128 ? x0 / points : 0, x = x0 - g * points, rr = x / chunks, e = (x - rr * chunks) * 8;
            float M = -INFINITY, L = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
            for (int i = g; i < more.w; i += groups) {
                const int slot = (2 * (more.z + i) + (i == 0 ? 1 : 0)) * PA_ROWS + rr;
                const float4* src = reinterpret_cast<const float4*>(p.part_o + (long long)slot * p.v.hd + e);
                add(Kind(), M, L, acc, __ldcg(p.part_ml + slot), __ldcg(src), __ldcg(src + 1));
            }
            if (groups == 1) {
                finish(rr, e, M, L, acc);
            } else {
                float* to = so + x0 * 10;
                to[0] = M; to[1] = L;
#pragma unroll
                for (int i = 0; i < 8; ++i) to[2 + i] = acc[i];
            }
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
        if (groups > 1) {
            for (int x = threadIdx.x; x < points; x += PA_WARPS * 32) {
                const int rr = x / chunks, e = (x - rr * chunks) * 8;
                float M = -INFINITY, L = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                for (int g = 0; g < groups; ++g) {
                    const float* from = so + (g * points + x) * 10;
                    add(Kind(), M, L, acc, make_float2(from[0], from[1]), make_float4(from[2], from[3], from[4], from[5]),
                        make_float4(from[6], from[7], from[8], from[9]));
                }
                finish(rr, e, M, L, acc);
            }
            asm volatile("bar.sync 1, 128;" ::: "memory");
        }
    }
    if (!ok) {
        // (what was asked for may still arrive: the block keeps its memory a little longer)
        if (lane == 0) { *abort_flag = 1; atomicExch(p.err, 74); }
        for (int i = 0; i < 64; ++i) __nanosleep(1000);
    }
}

// ------------------------------------------------------------------------------- chunks: tcgen05
// (constants of the tiles: paged_plan.h)
// CTA = one tile of 128 query rows of a sequence: 128 / group tokens with the heads that share a key head side by side, so that
// every key and value that comes in is used by all of them.  The roles are those of attention_fwd_kernel: a producer warp, one that
// issues the products, and two groups of four softmax warps (thread = query row) that take the half blocks of 64 keys in turn,
// with a score buffer, a probability buffer, a maximum, a sum and an accumulator in tensor memory each.  What is different:
//  * keys and values come by one copy per piece of a page;
//  * where a block holds keys that some row does not see (the chunk's own tokens, the rest of the last page), what is not finite
//    among its values is set to zero before the product, because 0 * infinity would reach the rows that do not see it; a row that does
//    see it gets it added at the end (add_what_is_not_finite);
//  * heads of 128 and 8-bit rows (TS): queries and probabilities lie in tensor memory, so that the tensor cores read nothing but keys
//    and values from shared memory (8-bit chunks of 128 behind 16,000 keys: 94.6 -> 84.9 us; heads of 64 have no room for it beside two
//    CTAs per SM);
//  * 8-bit rows: keys stay codes.  A query row becomes two 8-bit terms (below), and the products of both with the same codes are one
//    sum (111 -> 102 us, where keys were turned into f16 before).  Four more warps turn values into f16 tiles, a key per thread.  A value's
//    scale goes into its tile against the largest scale so far (a power of two, which the accumulators follow as they follow the
//    maximum): 11 bits of every value whose scale is within 2^-21 of the largest, and an absolute error below 2^-31 of the largest
//    value behind that.  Where a block holds keys that some row does not see, a value is against the largest scale up to its own key (a
//    row that sees it sees those too), and what that is below the largest that the row sees goes into the row's probability: what a row
//    does not see, however large, costs it nothing.
//
// Bound: a group's way through a block.  Clocks per block of 64 keys, bf16 heads of 64 (two CTAs per SM) / of 128 / 8 bits of 128: scores to
// come 510 / 570 / 630, from tensor memory 250 / 150 / 290, maximum 300, product before to end 270 / 190 / 290, exponentials and their way
// back 1,680 / 1,140 / 1,250.  Neither fewer loads, nor a quarter of the products, nor no exponentials at all change the total by more than
// 10 %.  2 x 512 rows of 8 heads of 128 behind 32,000 keys: bf16 159 us (851 TFLOP/s), 8 bits 200 us (675 TFLOP/s; 196 before every row had
// its own largest scale at the edge).
//
// A row's reference m follows its largest score only when that lies more than PT_SLACK above it (log2): every sum and product is against
// the same m, so the result is the same, probabilities reach 2^8 at most, and the accumulators are seldom scaled (104 -> 94.6 us).
// 8 bits: probabilities are f16 there, against 2^-PT_UP of that score: 2^15 at most, and those down to 2^-32 of the largest count.
constexpr float PT_SLACK = 8.f, PT_UP = 7.f;
constexpr int PT_TILE = 128 * 128;                      // bytes of a [128][64] 16-bit tile

template <int NH, bool E4M3>
struct ChunkShape {
    static constexpr int THREADS = E4M3 ? 448 : 320;
    static constexpr int KST = NH == 2 || E4M3 ? 3 : 2, VST = E4M3 ? 2 : KST;        // stages of keys and of values
    // Query rows and probabilities in tensor memory, where it has room for them: what the tensor cores read of shared memory is then keys and
    // values alone.
    static constexpr bool TS = NH == 2 || E4M3;
    static constexpr int K_TILE = E4M3 ? PT_TILE : NH * PT_TILE;         // bytes of a stage of keys: bf16, or codes (rows of 128 bytes)
    static constexpr int RAW = PT_KEYS * 64 * NH;                        // bytes of a block's codes of values
    static constexpr int O_K = NH * PT_TILE, O_V = O_K + KST * K_TILE, O_P = O_V + VST * NH * PT_TILE, O_RAW = O_P + (TS ? 0 : 2 * PT_TILE);
    // (8 bits) stages of codes of values as they come in
    static constexpr int RST = 2;
    static constexpr int O_KS = O_RAW + (E4M3 ? RST * RAW : 0);          // [8][128] key scales * scale_log2
    static constexpr int O_RF = O_KS + (E4M3 ? 8 * PT_KEYS * 4 : 0);     // [128] row factors
    static constexpr int O_EX = O_RF + (E4M3 ? PT_ROWS * 4 : 0);         // [2][128] exponents of values in blocks at the edge
    static constexpr int O_SEEN = O_EX + (E4M3 ? 2 * PT_KEYS * 4 : 0);   // [2][128] the largest that a row has seen there
    static constexpr int O_BARS = O_SEEN + (E4M3 ? 2 * PT_ROWS * 4 : 0);
    // (bf16 heads of 64: exactly what lets two CTAs share an SM; 256 bytes of barriers behind the tiles or in the alignment's pad)
    static constexpr int SMEM = 1024 + O_BARS + (TS ? 640 : 0);
    static constexpr int PER_SM = TS ? 1 : 2;
    static_assert(SMEM <= (TS ? 227 : 113) * 1024, "shared memory of an SM");
    static constexpr int TMEM = TS ? 512 : 256;
};

// A piece of a tile's keys, [blocks from, to): what one CTA does.  first, pieces: the tile's pieces are units first .. first + pieces - 1.
struct alignas(16) ChunkUnit { int s, head, tile, from, to, first, pieces; };

struct PagedChunkParams {
    PagedAttParams a;
    int tokens, tiles;                // tokens per tile; tiles of max_q
    int planned;                      // units come from paged_plan_kernel; else a CTA per tile
    int most_units, most_pieces, slots;       // room for units, for pieces' results; CTAs that the chip holds
    int* count;                       // units there are; CTAs of paged_rows_kernel that have work
    int rows_keys_log2, rows_cost;    // keys of its blocks; what one costs, in quarters of a tile's block
    int rows_slots, rows_lost;        // CTAs of it that the chip holds; how many fewer for a CTA with a tile
    unsigned int* arrived;            // [most_units]: pieces written, by the tile's first unit
    int* bad;                         // [most_units]: a piece has left out a value that is not finite
    ChunkUnit* units;
    float2* part_ml;                  // [most_pieces][128]
    float4* part_o;                   // [most_pieces][NH 64 / 4][128]: a row per thread side by side
};

// blocks of keys that a tile's last token sees (at least one: a tile of rows without a key)
__device__ __forceinline__ int tile_blocks(int n, int kv, int tile, int tokens) {
    const int last = kv - n + min(n, (tile + 1) * tokens) - 1;
    return last >= 0 ? last / PT_KEYS + 1 : 1;
}

// How few tiles are cut into pieces: by the number of pieces of the longest one for which (rounds of CTAs) * (blocks of a piece and what a
// piece costs beside them) is least.  One block of threads, some microseconds; where there are tiles enough (the host's bound), they are
// not cut and this does not run.
static_assert(sizeof(ChunkUnit) == 32, "room for units: paged_plan.h");
constexpr int PL_THREADS = 512;
__global__ void __launch_bounds__(PL_THREADS)
paged_plan_kernel(const PagedChunkParams pp) {
    __shared__ int seq[PL_TILES], idx[PL_TILES], nb[PL_TILES], off[PL_TILES];
    __shared__ int count, longest, best_cap, cost[PL_THREADS / 32], caps[PL_THREADS / 32], runs[PL_THREADS / 32], total;
    __shared__ unsigned long long few;                       // blocks of paged_rows_kernel
    __shared__ int of_warp[PL_THREADS / 32];
    const PagedAttParams& p = pp.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) { count = 0; longest = 1; total = 0; few = 0; }
    __syncthreads();
    pdl_wait();
    pdl_launch_dependents();
    // ---- the tiles of one head, in the order of the sequences; a thread per sequence
    for (int s0 = 0; s0 < p.v.seqs; s0 += PL_THREADS) {
        int q0, n = 0, kv = 0, tiles = 0, blocks = 0;
        if (s0 + tid < p.v.seqs && batch_of(p, s0 + tid, q0, n, kv)) {
            if (n * p.group > PA_ROWS) tiles = (n + pp.tokens - 1) / pp.tokens;
            else if (n > 0) blocks = max(1, (kv + (1 << pp.rows_keys_log2) - 1) >> pp.rows_keys_log2);
        }
        int incl = tiles;
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += x;
        }
        if (lane == 31) of_warp[warp] = incl;
        for (int o = 16; o > 0; o >>= 1) blocks += __shfl_xor_sync(0xffffffffu, blocks, o);      // (32 times 2^26 at most)
        if (lane == 0 && blocks > 0) atomicAdd(&few, (unsigned long long)blocks);
        __syncthreads();
        int at = count + incl - tiles, all = 0;
#pragma unroll
        for (int w = 0; w < PL_THREADS / 32; ++w) {
            if (w < warp) at += of_warp[w];
            all += of_warp[w];
        }
        for (int t = 0; t < tiles && at + t < PL_TILES; ++t) { seq[at + t] = s0 + tid; idx[at + t] = t; nb[at + t] = tile_blocks(n, kv, t, pp.tokens); }
        if (tiles > 0) atomicMax(&longest, tile_blocks(n, kv, tiles - 1, pp.tokens));
        __syncthreads();
        if (tid == 0) count += all;
        __syncthreads();
    }
    const int tiles = min(count, PL_TILES);                  // (no more than the host's bound, which is below)
    // ---- a warp per number of pieces
    {
        const int pieces = warp < 8 ? warp + 1 : (warp - 5) * 4;      // 1 .. 8, 12, 16, .. 40
        const int cap = (longest + pieces - 1) / pieces;
        int units = 0;
        for (int t = lane; t < tiles; t += 32) units += (nb[t] + cap - 1) / cap;
        units = __reduce_add_sync(0xffffffffu, units) * p.v.heads;
        if (lane == 0) {
            caps[warp] = cap;
            // (in quarters of a block: three blocks for the start of a piece and its result to memory, one for a piece's result on its way
            // back, four for the start of the few rows' kernel.)  Both kernels side by side, or one after the other.
            const long long tile_cost = 4 * ((long long)(units + pp.slots - 1) / pp.slots * (cap + 3) + pieces), blocks = (long long)few * p.v.heads;
            const int beside = pp.rows_slots - pp.rows_lost * units;
            long long best = tile_cost;
            runs[warp] = pp.rows_slots;
            if (blocks > 0) {
                best += pp.rows_cost * blocks / pp.rows_slots + 16;
                if (beside > 0) {
                    const long long both = max(tile_cost, pp.rows_cost * blocks / beside + 16);
                    if (both < best) { best = both; runs[warp] = beside; }
                }
            }
            cost[warp] = (pieces == 1 || units <= pp.most_pieces) ? (int)min(best, 0x7ffffffeLL) : 0x7fffffff;
        }
    }
    __syncthreads();
    if (tid == 0) {
        int w = 0;
        for (int i = 1; i < PL_THREADS / 32; ++i) if (cost[i] < cost[w]) w = i;
        best_cap = caps[w];
        pp.count[1] = runs[w];
    }
    __syncthreads();
    const int cap = best_cap;
    if (warp == 0) {
        int before = 0;
        for (int t0 = 0; t0 < tiles; t0 += 32) {
            const int pieces = t0 + lane < tiles ? (nb[t0 + lane] + cap - 1) / cap * p.v.heads : 0;
            int incl = pieces;
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += x;
            }
            if (t0 + lane < tiles) off[t0 + lane] = before + incl - pieces;
            before += __shfl_sync(0xffffffffu, incl, 31);
        }
        if (lane == 0) { total = min(before, pp.most_units); *pp.count = total; }
    }
    __syncthreads();
    for (int t = warp; t < tiles; t += PL_THREADS / 32) {
        const int pieces = (nb[t] + cap - 1) / cap, per = (nb[t] + pieces - 1) / pieces;
        for (int x = lane; x < pieces * p.v.heads; x += 32) {
            const int head = x / pieces, i = x - head * pieces, u = off[t] + x;
            if (u >= pp.most_units) continue;
            ChunkUnit c;
            c.s = seq[t]; c.head = head; c.tile = idx[t]; c.from = min(i * per, nb[t]); c.to = min((i + 1) * per, nb[t]);
            c.first = u - i; c.pieces = pieces;
            pp.units[u] = c;
            pp.arrived[u] = 0u;
        }
    }
}

__device__ __forceinline__ bool not_finite_16(uint32_t two) {            // either bf16 of a pair
    return (two & 0x7f80u) == 0x7f80u || (two & 0x7f800000u) == 0x7f800000u;
}

__device__ __forceinline__ uint32_t finite_16(uint32_t two) {             // zeros for what is not
    if ((two & 0x7f80u) == 0x7f80u) two &= 0xffff0000u;
    if ((two & 0x7f800000u) == 0x7f800000u) two &= 0xffffu;
    return two;
}

// What the product left out: values that are not finite, of the keys from k0 on that the row sees, added to the row's columns 32 b ..
// of every 64 in the staged result (bf16, 128-byte swizzle).  Rare; straight from the pool.
template <int NH, bool E4M3>
__device__ __forceinline__ void add_what_is_not_finite(const PagedAttParams& p, const uint8_t* V, int s, int head, int k0, int pos, int b, int r, uint8_t* row) {
#pragma unroll 1
    for (int k = k0; k <= pos; ++k) {
        const int page = p.v.table[(long long)s * p.v.table_ld + (k >> p.v.page_shift)];
        if ((unsigned)page >= (unsigned)p.v.pages) continue;
        const long long at = (((long long)page * p.v.heads + head) << p.v.page_shift) + (k & ((1 << p.v.page_shift) - 1));
        const float scale = E4M3 ? p.vs[at] : 1.f;
#pragma unroll 1
        for (int d = 0; d < p.v.hd; ++d) {
            if (((d >> 5) & 1) != b) continue;
            // (8 bits: a code and a scale that are numbers are in the product, even if theirs is more than float32 has)
            const float value = E4M3 ? e4m3_floats(V[at * p.v.hd + d]).x : __bfloat162float(reinterpret_cast<const bf16*>(V)[at * p.v.hd + d]);
            if (fabsf(value) < INFINITY && fabsf(scale) < INFINITY) continue;
            const float x = value * scale;
            bf16* o = reinterpret_cast<bf16*>(row + (d >> 6) * PT_TILE + ((((d & 63) >> 3) ^ (r & 7)) << 4)) + (d & 7);
            *o = __float2bfloat16_rn(__bfloat162float(*o) + x);
        }
    }
}

template <int NH, bool E4M3>
__global__ void __launch_bounds__((ChunkShape<NH, E4M3>::THREADS), (ChunkShape<NH, E4M3>::PER_SM))
paged_chunk_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                   const uint8_t* __restrict__ pool_v, const PagedChunkParams pp) {
    typedef ChunkShape<NH, E4M3> Sh;
    const PagedAttParams& p = pp.a;
    constexpr int KST = Sh::KST, VST = Sh::VST;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t pad = (1024u - (smem_u32(smem_raw) & 1023u)) & 1023u;
    uint8_t* smem = smem_raw + pad;
    uint8_t *sQ = smem, *sK = smem + Sh::O_K, *sV = smem + Sh::O_V, *sP = smem + Sh::O_P;
    uint64_t* bars = reinterpret_cast<uint64_t*>(pad <= 768u ? smem + Sh::O_BARS : smem_raw);
    uint64_t* q_full = bars;          // 1: the query tile has come
    uint64_t* q_ready = bars + 1;     // and is in tensor memory (8 bits: as two terms of 8 bits)
    uint64_t* k_full = bars + (Sh::TS ? 44 : 2);       // KST
    uint64_t* k_empty = bars + (Sh::TS ? 48 : 4);      // KST: the scores of both halves have been formed
    uint64_t* v_full = bars + (Sh::TS ? 52 : 6);     // VST
    uint64_t* v_empty = bars + (Sh::TS ? 56 : 8);    // VST
    uint64_t* v_land = bars + 10;     // 1: values of a block that is looked through first
    uint64_t* s_full = bars + 11;     // 2
    uint64_t* s_free = bars + 13;     // 2
    uint64_t* p_full = bars + 15;     // 2
    uint64_t* o_full = bars + 17;     // 2
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 19);
    uint64_t* raw_full = bars + 32;   // (8 bits) RST: codes of values; behind the 256 bytes of the rest
    uint64_t* raw_empty = bars + 36;  // RST
    uint64_t* ks_full = bars + 60;    // 8: what the softmax warps read of a block's scales.  (Not k_full, which may be a whole round ahead of them.)
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* bad_value = abort_flag + 1;                              // a value that is not finite has been set to zero
    volatile int* v_exponent = abort_flag + 2;                             // (8 bits) the reference of the last block that all rows see
    volatile int* is_last = abort_flag + 3;                                // this CTA was the last with its piece of a tile
    float* v_moved = reinterpret_cast<float*>(tmem_slot + 6);              // (8 bits) [8]: 2^(reference before - reference) of a block
    uint32_t* warp_most = tmem_slot + 14;                                  // (8 bits) [2][4]

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_wait();
    pdl_launch_dependents_now();         // paged_rows_kernel reads nothing of this kernel's: it starts where there is room
    int s, head, tile, from = 0, to = 0x7fffffff, pieces = 1, first_unit = 0;
    if (pp.planned) {
        if ((int)blockIdx.x >= *pp.count) return;
        const int4* u = reinterpret_cast<const int4*>(pp.units + blockIdx.x);
        const int4 a = u[0], b = u[1];
        s = a.x; head = a.y; tile = a.z; from = a.w; to = b.x; first_unit = b.y; pieces = b.z;
    } else {
        // the heaviest tiles of all sequences first
        s = (int)(blockIdx.x / (unsigned)p.v.heads); head = (int)(blockIdx.x % (unsigned)p.v.heads);
        tile = pp.tiles - 1 - (int)(blockIdx.z * gridDim.y + blockIdx.y);
        if (tile < 0) return;
    }
    int q0, n, kv;
    const bool fine = batch_of(p, s, q0, n, kv);                           // (paged_rows_kernel reports it)
    const int tok0 = tile * pp.tokens;
    if (!fine || n * p.group <= PA_ROWS || tok0 >= n) return;
    const int tokens = min(pp.tokens, n - tok0);
    const int first_pos = kv - n + tok0, last_pos = first_pos + tokens - 1;
    const int nkv = min(to, last_pos >= 0 ? last_pos / PT_KEYS + 1 : 0) - from;      // blocks of keys, from block `from` on
    const int edge0 = max(0, first_pos + 1) / PT_KEYS;                     // the first block with a key that some row does not see
    // the producer's first pages, on their way while the block sets itself up
    const int piece_shift = min(p.v.page_shift, 7), page_pieces = PT_KEYS >> piece_shift, piece_keys = 1 << piece_shift;
    const int per_page_shift = p.v.page_shift - piece_shift, last_piece = (last_pos + piece_keys) >> piece_shift, piece0 = from * page_pieces;
    const int* table = p.v.table + (long long)s * p.v.table_ld;
    auto page_at = [&](int piece) -> int {
        if (piece >= last_piece) return 0;
        const int pg = table[piece >> per_page_shift];
        if ((unsigned)pg < (unsigned)p.v.pages) return pg;
        report_argument(p.err, 75);
        return -1;
    };
    int held = piece0, now = 0, next = 0;
    if (warp == 0 && nkv > 0) { now = page_at(piece0 + lane); next = page_at(piece0 + 32 + lane); }

    if (threadIdx.x == 32 * 2) {
        mbar_init(q_full, 1); mbar_init(q_ready, 4); mbar_init(v_land, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1); mbar_init(&s_free[i], 4); mbar_init(&p_full[i], 4); mbar_init(&o_full[i], 1);
        }
        if (E4M3)
            for (int i = 0; i < Sh::RST; ++i) { mbar_init(&raw_full[i], 1); mbar_init(&raw_empty[i], 4); }
        for (int i = 0; i < KST; ++i) { mbar_init(&k_full[i], 1); mbar_init(&k_empty[i], 1); }
        for (int i = 0; i < VST; ++i) { mbar_init(&v_full[i], E4M3 ? 4 : 1); mbar_init(&v_empty[i], 1); }
        if (E4M3)
            for (int i = 0; i < 8; ++i) mbar_init(&ks_full[i], 4);
        *abort_flag = 0; *bad_value = 0; *v_exponent = 0;
        fence_mbar_init();
    }
    if (warp == 1) { tmem_alloc(tmem_slot, Sh::TMEM); tmem_relinquish(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const uint32_t tS = tmem_base, tO = tmem_base + 128;                   // two score buffers of 64, two accumulators of 64 NH columns,
    const uint32_t tP = tO + 128 * NH, tQ = tP + 64;                       // two of probabilities, 64 16-bit values each, the rows

    if (warp == 0) {
        // ---- producer: a lane per piece of a page
        bool ok = true, any_bad = __any_sync(0xffffffffu, now < 0);
        if (lane == 0 && nkv > 0) {
            mbar_expect_tx(q_full, (uint32_t)(NH * pp.tokens * p.group * 128));
            for (int c = 0; c < NH; ++c) tma_load_3d(sQ + c * PT_TILE, &tmQ, q_full, c * 64, head * p.group, q0 + tok0);
        }
        int landed = 0;
        if (E4M3) {
            for (int j = 0; j < nkv; ++j) {
                const int at = piece0 + j * page_pieces, st = j % KST, rs = j % Sh::RST, o = lane << piece_shift;
                if (at >= held + 32) { held += 32; now = next; next = page_at(held + 32 + lane); any_bad = __any_sync(0xffffffffu, now < 0); }
                const int pg = __shfl_sync(0xffffffffu, now, (at - held + lane) & 31);
                const int count = min(page_pieces, last_piece - at);
                const unsigned bad = any_bad ? __ballot_sync(0xffffffffu, lane < count && pg < 0) : 0u;
                const int copies = count - __popc(bad);
                const bool copied = lane < count && pg >= 0;
                const int block = pg * p.v.heads + head, r0 = ((at + lane) & ((1 << per_page_shift) - 1)) << piece_shift;
                ok = __all_sync(0xffffffffu, mbar_wait(&k_empty[st], (uint32_t)((j / KST) & 1) ^ 1u, abort_flag));
                if (!ok) break;
                if (bad != 0u) fill_pieces(sK + st * Sh::K_TILE, bad, piece_keys * 128, PA_NAN);
                if (lane == 0) mbar_expect_tx(&k_full[st], (uint32_t)(copies * piece_keys * 128));
                __syncwarp();
                if (copied) tma_load_3d(sK + st * Sh::K_TILE + o * 128, &tmK, &k_full[st], 0, r0, block);
                __syncwarp();
                ok = __all_sync(0xffffffffu, mbar_wait(&raw_empty[rs], (uint32_t)((j / Sh::RST) & 1) ^ 1u, abort_flag));
                if (!ok) break;
                if (bad != 0u) fill_pieces(smem + Sh::O_RAW + rs * Sh::RAW, bad, piece_keys * 64 * NH, 0u);
                if (lane == 0) mbar_expect_tx(&raw_full[rs], (uint32_t)(copies * piece_keys * 64 * NH));
                __syncwarp();
                if (copied) tma_load_3d(smem + Sh::O_RAW + rs * Sh::RAW + o * 64 * NH, &tmV, &raw_full[rs], 0, r0, block);
                __syncwarp();
            }
        }
        for (int j = 0; j < nkv && ok && !E4M3; ++j) {
            const int at = piece0 + j * page_pieces;
            if (at >= held + 32) { held += 32; now = next; next = page_at(held + 32 + lane); any_bad = __any_sync(0xffffffffu, now < 0); }
            const int pg = __shfl_sync(0xffffffffu, now, (at - held + lane) & 31);
            const int count = min(page_pieces, last_piece - at);
            const unsigned bad = any_bad ? __ballot_sync(0xffffffffu, lane < count && pg < 0) : 0u;
            const int copies = count - __popc(bad);
            const bool copied = lane < count && pg >= 0;
            const int block = pg * p.v.heads + head, r0 = ((at + lane) & ((1 << per_page_shift) - 1)) << piece_shift;
            const int o = lane << piece_shift;
            const int st = j % KST;
            {
                const int vst = j % VST;
                ok = mbar_wait(&k_empty[st], (uint32_t)((j / KST) & 1) ^ 1u, abort_flag);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                if (bad != 0u)
                    for (int c = 0; c < NH; ++c) fill_pieces(sK + (st * NH + c) * PT_TILE, bad, piece_keys * 128, PA_NAN);
                if (lane == 0) mbar_expect_tx(&k_full[st], (uint32_t)(copies * piece_keys * 128 * NH));
                __syncwarp();
                if (copied)
                    for (int c = 0; c < NH; ++c) tma_load_3d(sK + (st * NH + c) * PT_TILE + o * 128, &tmK, &k_full[st], c * 64, r0, block);
                ok = mbar_wait(&v_empty[vst], (uint32_t)((j / VST) & 1) ^ 1u, abort_flag);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                const bool edge = from + j >= edge0;
                uint64_t* bar = edge ? v_land : &v_full[vst];
                uint8_t* tile_v = sV + vst * NH * PT_TILE;
                if (bad != 0u)
                    for (int c = 0; c < NH; ++c) fill_pieces(tile_v + c * PT_TILE, bad, piece_keys * 128, 0u);
                if (lane == 0) mbar_expect_tx(bar, (uint32_t)(copies * piece_keys * 128 * NH));
                __syncwarp();
                if (copied)
                    for (int c = 0; c < NH; ++c) tma_load_3d(tile_v + c * PT_TILE + o * 128, &tmV, bar, c * 64, r0, block);
                if (edge) {
                    ok = mbar_wait(v_land, (uint32_t)(landed & 1), abort_flag);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    ++landed;
                    const int seen = last_pos + 1 - (from + j) * PT_KEYS;           // rows of the tile that some query sees
                    bool bad = false;
#pragma unroll 1
                    for (int x0 = 0; x0 < PT_KEYS * 8 * NH; x0 += 32 * 8) {             // eight 16-byte pieces per lane side by side
                        uint4 w[8];
                        bool any = false;
#pragma unroll
                        for (int i = 0; i < 8; ++i) w[i] = *reinterpret_cast<const uint4*>(tile_v + (x0 + i * 32 + lane) * 16);
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            any |= not_finite_16(w[i].x) || not_finite_16(w[i].y) || not_finite_16(w[i].z) || not_finite_16(w[i].w);
                        if (!any) continue;
#pragma unroll 1
                        for (int i = 0; i < 8; ++i) {
                            uint4* at16 = reinterpret_cast<uint4*>(tile_v + (x0 + i * 32 + lane) * 16);
                            uint4 y = *at16;
                            // (behind the last row that some query sees: whatever a page holds, or an earlier block)
                            if (((x0 + i * 32 + lane) >> 3) % PT_KEYS < seen &&
                                (not_finite_16(y.x) || not_finite_16(y.y) || not_finite_16(y.z) || not_finite_16(y.w))) bad = true;
                            *at16 = make_uint4(finite_16(y.x), finite_16(y.y), finite_16(y.z), finite_16(y.w));
                        }
                    }
                    if (bad) *bad_value = 1;
                    fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&v_full[vst]);
                }
            }
            __syncwarp();
        }
        if (!ok && lane == 0) { *abort_flag = 1; atomicExch(p.err, 77); }
    } else if (warp == 1) {
        if (elect_one() && nkv > 0) {
            const uint32_t fmt = E4M3 ? 0u : 1u;
            // (8 bits: the row's first term is e5m2)
            const uint32_t idesc_s = umma_idesc(fmt, 0u, 0u, PT_ROWS, 64), idesc_s1 = idesc_s | 1u << 7, idesc_o = umma_idesc(fmt, 0u, 1u, PT_ROWS, 64 * NH);
            const uint64_t dQ = umma_desc_sw128(smem_u32(sQ), 16, 1024), dK0 = umma_desc_sw128(smem_u32(sK), 16, 1024);
            const uint64_t dP0 = umma_desc_sw128(smem_u32(sP), 16, 1024), dV0 = umma_desc_sw128(smem_u32(sV), PT_TILE, 1024);
            constexpr uint64_t TILE = PT_TILE >> 4, KSTEP = 32 >> 4, MNSTEP = 2048 >> 4;
            const int nsub = 2 * nkv;
            bool ok = mbar_wait(Sh::TS ? q_ready : q_full, 0, abort_flag);
            auto issue_scores = [&](int i) -> bool {
                const int j = i >> 1, st = j % KST, b = i & 1;
                if (b == 0 && !mbar_wait(&k_full[st], (uint32_t)((j / KST) & 1), abort_flag)) return false;
                if (!mbar_wait(&s_free[b], (uint32_t)((i >> 1) & 1) ^ 1u, abort_flag)) return false;
                tc_fence_after();
                const uint64_t dK = dK0 + (uint64_t)st * (Sh::K_TILE >> 4) + (uint64_t)b * (TILE / 2);
#pragma unroll
                for (int k = 0; k < 4 * NH; ++k) {
                    if (E4M3) {                                             // both terms of the rows with the same codes
                        umma_f8_ts(tS + (uint32_t)(b * 64), tQ + (uint32_t)(8 * k), dK + (k % (2 * NH)) * KSTEP, k < 2 * NH ? idesc_s1 : idesc_s, k > 0 ? 1u : 0u);
                    } else if (Sh::TS) {
                        umma_bf16_ts(tS + (uint32_t)(b * 64), tQ + (uint32_t)(8 * k), dK + (k >> 2) * TILE + (k & 3) * KSTEP, idesc_s, k > 0 ? 1u : 0u);
                    } else {
                        umma_bf16(tS + (uint32_t)(b * 64), dQ + (k >> 2) * TILE + (k & 3) * KSTEP, dK + (k >> 2) * TILE + (k & 3) * KSTEP, idesc_s,
                                  k > 0 ? 1u : 0u);
                    }
                }
                umma_commit(&s_full[b]);
                if (b == 1) umma_commit(&k_empty[st]);
                return true;
            };
            if (ok) ok = issue_scores(0) && issue_scores(1);
            for (int i = 0; i < nsub && ok; ++i) {
                const int j = i >> 1, b = i & 1, vst = j % VST;
                if (i + 2 < nsub && !issue_scores(i + 2)) { ok = false; break; }
                if (!mbar_wait(&p_full[b], (uint32_t)(j & 1), abort_flag)) { ok = false; break; }
                if (b == 0 && !mbar_wait(&v_full[vst], (uint32_t)((j / VST) & 1), abort_flag)) { ok = false; break; }
                tc_fence_after();
                const uint64_t dP = dP0 + (uint64_t)b * TILE, dV = dV0 + (uint64_t)(vst * NH) * TILE + (uint64_t)b * (4 * MNSTEP);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if (Sh::TS)
                        umma_bf16_ts(tO + (uint32_t)(b * 64 * NH), tP + (uint32_t)(b * 32 + 8 * k), dV + k * MNSTEP, idesc_o, (i > 1 || k > 0) ? 1u : 0u);
                    else
                        umma_bf16(tO + (uint32_t)(b * 64 * NH), dP + k * KSTEP, dV + k * MNSTEP, idesc_o, (i > 1 || k > 0) ? 1u : 0u);
                }
                umma_commit(&o_full[b]);
                if (b == 1) umma_commit(&v_empty[vst]);
            }
            if (!ok) { *abort_flag = 1; atomicExch(p.err, 78); }
        }
    } else if (warp < 10) {
        // ---- softmax
        const int q = warp & 3, b = (warp - 2) >> 2, r = q * 32 + lane;
        const int tok = min((int)((uint32_t)r * p.group_magic >> 16), tokens - 1);
        const int pos = first_pos + tok;
        const bool mine = r < tokens * p.group;
        const uint32_t lane_base = (uint32_t)(q * 32) << 16;
        const uint32_t ts = tS + lane_base + (uint32_t)(b * 64), to = tO + lane_base + (uint32_t)(b * 64 * NH);
        float m = PA_LOW, l = 0.f, c1 = p.scale_log2;
        bool ok = true;
        // (8 bits) this row's reference of value scales, once there is one of its own: the others have v_exponent
        int* seen_exponent = reinterpret_cast<int*>(smem + Sh::O_SEEN) + b * PT_ROWS + r;
        if (E4M3) *seen_exponent = -1;
        uint32_t v[2][32];
        if (Sh::TS && !E4M3 && nkv > 0 && b == 0) {                         // the rows to tensor memory
            ok = __all_sync(0xffffffffu, mbar_wait(q_full, 0, abort_flag));
#pragma unroll
            for (int c = 0; c < NH; ++c) {
#pragma unroll
                for (int d = 0; d < 8; ++d) {
                    const uint4 w = *reinterpret_cast<const uint4*>(sQ + c * PT_TILE + r * 128 + ((d ^ (r & 7)) << 4));
                    v[0][4 * d] = w.x; v[0][4 * d + 1] = w.y; v[0][4 * d + 2] = w.z; v[0][4 * d + 3] = w.w;
                }
                tmem_st32(tQ + lane_base + (uint32_t)(c * 32), v[0]);
            }
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0 && ok) mbar_arrive(q_ready);
        }
        if (E4M3 && nkv > 0) {
            ok = mbar_wait(q_ready, 0, abort_flag);
            c1 = reinterpret_cast<const float*>(smem + Sh::O_RF)[r];
        }
        for (int j = 0; j < nkv && ok; ++j) {
            if (E4M3 && !mbar_wait(&ks_full[j & 7], (uint32_t)((j >> 3) & 1), abort_flag)) { ok = false; break; }
            if (!mbar_wait(&s_full[b], (uint32_t)(j & 1), abort_flag)) { ok = false; break; }
            tc_fence_after();
            tmem_ld32(ts, v[0]);
            tmem_ld32(ts + 32, v[1]);
            tmem_ld_wait();
            float moved = 1.f;
            if (E4M3) {
                const float4* ks = reinterpret_cast<const float4*>(smem + Sh::O_KS) + (j & 7) * (PT_KEYS / 4) + b * 16;
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        const float4 f = ks[c * 8 + e / 4];
                        const float2 x = __fmul2_rn(make_float2(__uint_as_float(v[c][e]), __uint_as_float(v[c][e + 1])), make_float2(f.x, f.y));
                        const float2 y = __fmul2_rn(make_float2(__uint_as_float(v[c][e + 2]), __uint_as_float(v[c][e + 3])), make_float2(f.z, f.w));
                        v[c][e] = __float_as_uint(x.x); v[c][e + 1] = __float_as_uint(x.y);
                        v[c][e + 2] = __float_as_uint(y.x); v[c][e + 3] = __float_as_uint(y.y);
                    }
                moved = v_moved[j & 7];
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s_free[b]);
            const bool edge = from + j >= edge0;
            const int lim = edge ? pos - (from + j) * PT_KEYS - b * 64 : 64;         // columns e <= lim are allowed
            float mx = -INFINITY;
            if (edge) {
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    if (e > lim) v[0][e] = 0xff800000u;                     // -infinity: no probability
                    if (e + 32 > lim) v[1][e] = 0xff800000u;
                    mx = fmaxf(mx, fmaxf(__uint_as_float(v[0][e]), __uint_as_float(v[1][e])));
                }
            } else {
                float m0 = -INFINITY, m1 = -INFINITY, m2 = -INFINITY, m3 = -INFINITY;
#pragma unroll
                for (int e = 0; e < 32; e += 4) {
                    m0 = fmaxf(m0, fmaxf(__uint_as_float(v[0][e]), __uint_as_float(v[1][e])));
                    m1 = fmaxf(m1, fmaxf(__uint_as_float(v[0][e + 1]), __uint_as_float(v[1][e + 1])));
                    m2 = fmaxf(m2, fmaxf(__uint_as_float(v[0][e + 2]), __uint_as_float(v[1][e + 2])));
                    m3 = fmaxf(m3, fmaxf(__uint_as_float(v[0][e + 3]), __uint_as_float(v[1][e + 3])));
                }
                mx = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3));
            }
            float m_new = fmaxf(m, mx * c1);
            float alpha = 1.0f;
            if (m_new > m + (E4M3 ? PT_SLACK + PT_UP : PT_SLACK)) {
                if (E4M3) m_new -= PT_UP;
                alpha = ex2_approx(m - m_new);
                l *= alpha;
                m = m_new;
            }
            if (E4M3) alpha *= moved;
            const int* exponents = reinterpret_cast<const int*>(smem + Sh::O_EX) + ((from + j - edge0) & 1) * PT_KEYS + b * 64;
            if (E4M3 && edge) {
                const int before = *seen_exponent < 0 ? *v_exponent : *seen_exponent;
                const int its_exponent = lim < 0 ? before : max(before, exponents[min(lim, 63)]);
                *seen_exponent = its_exponent;
                alpha *= power_of_two(max(before - its_exponent, -126));
            }
            const bool move = __any_sync(0xffffffffu, alpha != 1.0f);
            if (j > 0 && !mbar_wait(&o_full[b], (uint32_t)((j - 1) & 1), abort_flag)) { ok = false; break; }
            // (a row that sees no key of this half: minus infinity against anything.  Against m as well is as right, and costs a spilled register.)
            const float nm = lim < 0 ? 0.f : -m;
            const float2 c2 = make_float2(c1, c1), nm2 = make_float2(nm, nm);
            float2 ls[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
            uint8_t* prow = sP + b * PT_TILE + r * 128;
            uint32_t all[32];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    uint32_t w[4];
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
                        const int e = 8 * g + 2 * h;
                        const float2 x = __ffma2_rn(make_float2(__uint_as_float(v[c][e]), __uint_as_float(v[c][e + 1])), c2, nm2);
                        const float2 pr = make_float2(ex2_approx(x.x), ex2_approx(x.y));
                        ls[h & 1] = __fadd2_rn(ls[h & 1], pr);
                        w[h] = E4M3 ? f16_pair(pr.x, pr.y) : bf16_pair(pr.x, pr.y);
                    }
                    if (Sh::TS) {
#pragma unroll
                        for (int h = 0; h < 4; ++h) all[16 * c + 4 * g + h] = w[h];
                    } else {
                        *reinterpret_cast<uint4*>(prow + (((4 * c + g) ^ (r & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            }
            if (Sh::TS) tmem_st32(tP + lane_base + (uint32_t)(b * 32), all);
            if (E4M3 && edge && __any_sync(0xffffffffu, exponents[0] < *seen_exponent)) {
                const int its_exponent = *seen_exponent;
                tmem_st_wait();
                tmem_ld32(tP + lane_base + (uint32_t)(b * 32), v[0]);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const int2 x = *reinterpret_cast<const int2*>(exponents + 2 * i);
                    const float2 pr = f16_floats(v[0][i]);
                    v[0][i] = f16_pair(pr.x * power_of_two(min(max(x.x - its_exponent, -127), 0)), pr.y * power_of_two(min(max(x.y - its_exponent, -127), 0)));
                }
                tmem_st32(tP + lane_base + (uint32_t)(b * 32), v[0]);
            }
            l += (ls[0].x + ls[0].y) + (ls[1].x + ls[1].y);
            if (move && j > 0) {
                tc_fence_after();
#pragma unroll 1
                for (int h2 = 0; h2 < 2 * NH; ++h2) {                       // (unrolled, it costs registers that the loop around it needs)
                    tmem_ld32(to + (uint32_t)(h2 * 32), v[0]);
                    tmem_ld_wait();
#pragma unroll
                    for (int e = 0; e < 32; ++e) v[0][e] = __float_as_uint(__uint_as_float(v[0][e]) * alpha);
                    tmem_st32(to + (uint32_t)(h2 * 32), v[0]);
                }
            }
            if (Sh::TS || (move && j > 0)) tmem_st_wait();
            tc_fence_before();
            if (!Sh::TS) fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[b]);
        }
        // ---- the two groups' results together
        if (ok && nkv > 0)
            ok = mbar_wait(&o_full[0], (uint32_t)((nkv - 1) & 1), abort_flag) && mbar_wait(&o_full[1], (uint32_t)((nkv - 1) & 1), abort_flag) &&
                 mbar_wait(&v_full[(nkv - 1) % VST], (uint32_t)(((nkv - 1) / VST) & 1), abort_flag);        // (for bad_value)
        float2* stat = reinterpret_cast<float2*>(Sh::TS ? sK : sP);        // (nothing reads keys any more)
        if (ok) stat[b * PT_ROWS + r] = make_float2(m, l);
        asm volatile("bar.sync 1, 256;" ::: "memory");
        const bool none = pos < 0;                                          // a row without a key
        float M = -INFINITY, L = 0.f, w0 = 0.f, w1 = 0.f, unit = 1.f;
        int last = 1;                                                       // this CTA has the tile's result
        if (ok) {
            const float2 s0 = stat[r], s1 = stat[PT_ROWS + r];
            M = fmaxf(s0.x, s1.x) + (E4M3 ? PT_SLACK + PT_UP : 0.f);         // (products and their scale within float32)
            const float e0 = s0.y == 0.f ? 0.f : ex2_approx(s0.x - M), e1 = s1.y == 0.f ? 0.f : ex2_approx(s1.x - M);
            L = s0.y * e0 + s1.y * e1;
            w0 = e0; w1 = e1;
            if (E4M3) {                                                     // (by itself: a product with w may be no number that float32 has)
                const int* x = reinterpret_cast<const int*>(smem + Sh::O_SEEN) + r;
                const int x0 = x[0] < 0 ? *v_exponent : x[0], x1 = x[PT_ROWS] < 0 ? *v_exponent : x[PT_ROWS], most = max(x0, x1);
                w0 *= power_of_two(max(x0 - most, -127)); w1 *= power_of_two(max(x1 - most, -127));
                unit = exp2f((float)(most - 127 - 6));
            }
        }
        tc_fence_after();
        // columns 64 c + 32 b .. of this row, against M
        auto own = [&](int c) {
            if (nkv > 0) {
                tmem_ld32(tO + lane_base + (uint32_t)(64 * c + 32 * b), v[0]);
                tmem_ld32(tO + lane_base + (uint32_t)(64 * NH + 64 * c + 32 * b), v[1]);
                tmem_ld_wait();
            }
#pragma unroll
            for (int e = 0; e < 32; ++e)
                v[0][e] = __float_as_uint((w0 == 0.f ? 0.f : __uint_as_float(v[0][e]) * w0) + (w1 == 0.f ? 0.f : __uint_as_float(v[1][e]) * w1));
        };
        if (pieces > 1) {
            // this piece's result to memory, a float4 of every row side by side; whoever is last adds them in their order
            if (ok) {
                float4* to16 = pp.part_o + ((long long)blockIdx.x * (16 * NH)) * PT_ROWS + r;
#pragma unroll 1
                for (int c = 0; c < NH; ++c) {
                    own(c);
#pragma unroll
                    for (int d = 0; d < 8; ++d)
                        __stcg(to16 + (16 * c + 8 * b + d) * PT_ROWS, make_float4(__uint_as_float(v[0][4 * d]) * unit, __uint_as_float(v[0][4 * d + 1]) * unit,
                                                                                  __uint_as_float(v[0][4 * d + 2]) * unit, __uint_as_float(v[0][4 * d + 3]) * unit));
                }
                if (b == 0) __stcg(pp.part_ml + (long long)blockIdx.x * PT_ROWS + r, make_float2(M, L));
                if (warp == 2 && lane == 0) pp.bad[blockIdx.x] = *bad_value;
            }
            if (all_of(ok, 1, 256)) {
                if (warp == 2 && lane == 0) __threadfence();                // (everyone's piece, before the count)
                if (warp == 2 && lane == 0) *is_last = atomicAdd(pp.arrived + first_unit, 1u) == (unsigned int)pieces - 1u ? 1 : 0;
                asm volatile("bar.sync 1, 256;" ::: "memory");
                last = *is_last;
            } else {
                ok = false;
            }
            if (ok && last) {
                __threadfence();
                M = -INFINITY;
                L = 0.f;
                bool any = false;
                for (int i = 0; i < pieces; ++i) {
                    const float2 ml = __ldcg(pp.part_ml + (long long)(first_unit + i) * PT_ROWS + r);
                    if (__ldcg(pp.bad + first_unit + i)) any = true;
                    if (ml.y == 0.f) continue;
                    const float mn = L == 0.f ? ml.x : fmaxf(M, ml.x);
                    L = (L == 0.f ? 0.f : L * ex2_approx(M - mn)) + ml.y * ex2_approx(ml.x - mn);
                    M = mn;
                }
                if (any) *bad_value = 1;
            }
        }
        if (ok && last) {
            const float inv = none ? 0.f : 1.0f / L;
            // as bf16 through the query tile, so that whole rows leave side by side
            uint8_t* row = sQ + r * 128;
#pragma unroll 1
            for (int c = 0; c < NH; ++c) {
                if (pieces == 1) {
                    own(c);
                } else {
#pragma unroll
                    for (int e = 0; e < 32; ++e) v[0][e] = 0u;
#pragma unroll 2
                    for (int i = 0; i < pieces; ++i) {
                        const float2 ml = __ldcg(pp.part_ml + (long long)(first_unit + i) * PT_ROWS + r);
                        const float f = ml.y == 0.f ? 0.f : ex2_approx(ml.x - M);        // (a piece without a key for this row holds zeros)
                        const float4* from16 = pp.part_o + ((long long)(first_unit + i) * (16 * NH) + 16 * c + 8 * b) * PT_ROWS + r;
#pragma unroll
                        for (int d = 0; d < 8; ++d) {
                            const float4 x = __ldcg(from16 + d * PT_ROWS);
                            v[0][4 * d] = __float_as_uint(fmaf(x.x, f, __uint_as_float(v[0][4 * d])));
                            v[0][4 * d + 1] = __float_as_uint(fmaf(x.y, f, __uint_as_float(v[0][4 * d + 1])));
                            v[0][4 * d + 2] = __float_as_uint(fmaf(x.z, f, __uint_as_float(v[0][4 * d + 2])));
                            v[0][4 * d + 3] = __float_as_uint(fmaf(x.w, f, __uint_as_float(v[0][4 * d + 3])));
                        }
                    }
                }
                auto out = [&](int e) { return none ? 0.f : __uint_as_float(v[0][e]) * inv * (pieces == 1 ? unit : 1.f); };
#pragma unroll
                for (int d = 0; d < 4; ++d)
                    *reinterpret_cast<uint4*>(row + c * PT_TILE + (((4 * b + d) ^ (r & 7)) << 4)) =
                        make_uint4(bf16_pair(out(8 * d), out(8 * d + 1)), bf16_pair(out(8 * d + 2), out(8 * d + 3)),
                                   bf16_pair(out(8 * d + 4), out(8 * d + 5)), bf16_pair(out(8 * d + 6), out(8 * d + 7)));
            }
            if (*bad_value && mine && !none) add_what_is_not_finite<NH, E4M3>(p, pool_v, s, head, edge0 * PT_KEYS, pos, b, r, row);
            if (p.lse && b == 0 && mine)
                p.lse[(long long)(q0 + tok0 + tok) * p.H + head * p.group + r - tok * p.group] =
                    none ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
        }
        if (all_of(ok, 1, 256) && last) {
            // 8 NH lanes per row, each with 16 bytes
            const int e = lane & (8 * NH - 1), rows_of_tile = tokens * p.group;
            const uint8_t* src = sQ + (e >> 3) * PT_TILE;
#pragma unroll
            for (int i = 0; i < 4 * NH; ++i) {
                const int rr = (warp - 2) * 16 + i * (4 / NH) + (lane >> (NH == 1 ? 3 : 4));
                const int t = (int)((uint32_t)rr * p.group_magic >> 16), g = rr - t * p.group;
                if (rr < rows_of_tile && e * 8 < p.v.hd)
                    *reinterpret_cast<uint4*>(p.att + (long long)(q0 + tok0 + t) * p.ld_att + (long long)(head * p.group + g) * p.v.hd + e * 8) =
                        *reinterpret_cast<const uint4*>(src + rr * 128 + (((e & 7) ^ (rr & 7)) << 4));
            }
        }
        if (!ok && lane == 0) { *abort_flag = 1; atomicExch(p.err, 79); }
    } else if (E4M3) {
        // ---- thread = query row once, which becomes two terms of 8 bits; then a key of every block, whose value becomes f16
        const int t = threadIdx.x - 320, q = warp - 10;
        bool ok = true;
        if (nkv > 0) ok = __all_sync(0xffffffffu, mbar_wait(q_full, 0, abort_flag));
        if (nkv > 0 && ok) {
            const int r = (warp & 3) * 32 + lane;                           // (the lanes of tensor memory that this warp reaches)
            uint32_t most = 0u;
            const uint8_t* row = sQ + r * 128;
            auto eight = [&](int d) { return *reinterpret_cast<const uint4*>(row + (d >> 3) * PT_TILE + (((d & 7) ^ (r & 7)) << 4)); };
#pragma unroll
            for (int d = 0; d < 8 * NH; ++d) {
                const uint4 w = eight(d);
                const uint32_t a = __vmaxu2(__vmaxu2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu), __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu));
                most = max(most, max(a & 0xffffu, a >> 16));
            }
            // Scaled by a power of two so that the row's largest magnitude lies in [2^11, 2^12).  Three bits of an element are its e5m2
            // term, and what is left of its eight fits four bits, an e4m3 term of at most 2^8: exact but for what lies below 2^-10, which
            // is 2^-21 of the row's largest.  (Both with the same codes of the keys, as they lie in the cache: no key is converted.)
            const int e = max((int)(most >> 7), 12);
            const bool odd = e == 255;                                      // (an infinity or NaN: no score of this row is a number)
            const float down = odd ? 1.f : __uint_as_float((uint32_t)(265 - e) << 23), up = odd ? 1.f : __uint_as_float((uint32_t)(e - 11) << 23);
            reinterpret_cast<float*>(smem + Sh::O_RF)[r] = up;
            const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
#pragma unroll 1
            for (int c = 0; c < NH; ++c) {                                  // 64 elements: 16 columns of first terms, 16 of second ones
                uint32_t hi[16], lo[16];
#pragma unroll
                for (int d = 0; d < 8; ++d) {
                    const uint4 w = eight(8 * c + d);
                    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        uint32_t a[2], b[2];
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            float2 f = bf16_floats(u[2 * i + x]);
                            f.x *= down; f.y *= down;
                            a[x] = e5m2_pair(f.x, f.y);
                            const float2 g = f16_floats((a[x] & 0xffu) << 8 | (a[x] & 0xff00u) << 16);
                            b[x] = e4m3_pair(f.x - g.x, f.y - g.y);
                        }
                        hi[2 * d + i] = odd ? 0x7f7f7f7fu : a[0] | a[1] << 16;
                        lo[2 * d + i] = odd ? 0x7f7f7f7fu : b[0] | b[1] << 16;
                    }
                }
                tmem_st16(tQ + lane_base + (uint32_t)(16 * c), hi);
                tmem_st16(tQ + lane_base + (uint32_t)(16 * (NH + c)), lo);
            }
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_ready);
        }
        // Scales by plain loads, a block ahead, and the pages they are found by another one.  (Bulk copies beside the codes are as fast, but
        // cost a copy per piece of a page.)
        auto page_of = [&](int j) -> int {                                  // of this thread's key of a block; -1: none
            const int key = (from + j) * PT_KEYS + t;
            if (j >= nkv || key > last_pos) return -1;
            const int pg = table[key >> p.v.page_shift];
            return (unsigned)pg < (unsigned)p.v.pages ? pg : 0;             // (the producer reports it; codes of NaN and 0 have any scale)
        };
        float ks_new = 0.f, vs_new = 0.f;
        auto load_scales = [&](int j, int pg) {
            const long long row = (((long long)pg * p.v.heads + head) << p.v.page_shift) + (((from + j) * PT_KEYS + t) & ((1 << p.v.page_shift) - 1));
            ks_new = pg < 0 ? 0.f : p.ks[row];
            vs_new = pg < 0 ? 0.f : p.vs[row];
        };
        int reference = 0;
        float f = 0.f, f_next = 0.f;                                        // the factor of this key's value, in this block and the next
        bool fin = true, fin_next = true;                                   // its scale is finite
        // What the softmax warps need of a block's scales, a block ahead of the values and so four blocks ahead of those that are still
        // read at most: a ring of eight.
        auto scales = [&](int j) -> bool {
            const float vs = vs_new;
            const uint32_t ve = (__float_as_uint(vs) >> 23) & 255u;
            fin_next = ve != 255u;
            // the block's reference: the largest exponent of a value's scale so far
            const uint32_t most = __reduce_max_sync(0xffffffffu, fin_next ? ve : 0u);
            uint32_t* w4 = warp_most + (j & 1) * 4;
            if (lane == 0) w4[q] = most;
            if (!all_of(ok, 2, 128)) return false;
            const int now = max(reference, (int)max(max(w4[0], w4[1]), max(w4[2], w4[3])));
            int its = now;
            reinterpret_cast<float*>(smem + Sh::O_KS)[(j & 7) * PT_KEYS + t] = ks_new * p.scale_log2;
            const bool at_edge = from + j >= edge0;
            if (at_edge) {
                // so far up to this key
                its = fin_next ? (int)ve : 0;
#pragma unroll 1
                for (int o = 1; o < 32; o <<= 1) {
                    const int x = __shfl_up_sync(0xffffffffu, its, o);
                    if (lane >= o) its = max(its, x);
                }
                its = max(its, reference);
                for (int w = 0; w < 3; ++w) if (w < q) its = max(its, (int)w4[w]);
                reinterpret_cast<int*>(smem + Sh::O_EX)[((from + j - edge0) & 1) * PT_KEYS + t] = its;       // (there are two such blocks at most)
            }
            if (t == 0) {
                v_moved[j & 7] = at_edge ? 1.f : power_of_two(max(reference - now, -126));                   // (at the edge: a row's own)
                if (!at_edge) *v_exponent = now;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&ks_full[j & 7]);
            reference = now;
            // code * scale * 2^(6 - reference), in two steps: 2^(127 - reference) alone may be no normal number
            const int half_way = (127 - its) / 2;
            f_next = fin_next ? vs * power_of_two(half_way) * power_of_two(133 - its - half_way) : vs;
            return true;
        };
        // a row's 16-byte pieces in an order that differs from thread to thread: eight of them read 128 different bytes of banks
        auto piece = [&](int x) { return NH == 2 ? (x + t) & 7 : (x + (t >> 1)) & 3; };
        auto nan_codes = [](uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; };
        load_scales(0, page_of(0));
        if (nkv > 0) ok = scales(0);
        load_scales(1, page_of(1));
        int page = page_of(2);
        for (int j = 0; j < nkv && ok; ++j) {
            const int vst = j % VST, rs = j % Sh::RST;
            const uint8_t* rv = smem + Sh::O_RAW + rs * Sh::RAW + t * 64 * NH;
            f = f_next; fin = fin_next;
            if (j + 1 < nkv && !scales(j + 1)) { ok = false; break; }
            load_scales(j + 2, page);
            page = page_of(j + 3);
            ok = mbar_wait(&raw_full[rs], (uint32_t)((j / Sh::RST) & 1), abort_flag) && mbar_wait(&v_empty[vst], (uint32_t)((j / VST) & 1) ^ 1u, abort_flag);
            if (!ok) {
                if (lane == 0) *abort_flag = 1;
                if (j + 2 < nkv) all_of(false, 2, 128);                     // (where the others meet in scales(j + 2))
                break;
            }
            const bool seen = (from + j) * PT_KEYS + t <= last_pos, looked = from + j >= edge0 && seen;
            bool bad = looked && !fin;
            if (looked && fin) {
                uint32_t has = 0u;
#pragma unroll
                for (int d = 0; d < 4 * NH; ++d) {
                    const uint4 w = *reinterpret_cast<const uint4*>(rv + 16 * d);
                    has |= nan_codes(w.x) | nan_codes(w.y) | nan_codes(w.z) | nan_codes(w.w);
                }
                bad = has != 0u;
            }
            if (bad) *bad_value = 1;
            const bool zero = !seen || (bad && !fin);
            const uint32_t f2 = zero ? 0u : f16_pair(f, f);
            uint8_t* row = sV + vst * NH * PT_TILE + t * 128;
#pragma unroll
            for (int c = 0; c < NH; ++c)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int y = piece(4 * c + x), d = y & 3;
                    uint8_t* to = row + (y >> 2) * PT_TILE;
                    uint4 w = *reinterpret_cast<const uint4*>(rv + 16 * y);
                    if (zero) w = make_uint4(0u, 0u, 0u, 0u);
                    if (bad) {                                              // NaN codes to zero
                        w.x &= ~((nan_codes(w.x) >> 7) * 255u); w.y &= ~((nan_codes(w.y) >> 7) * 255u);
                        w.z &= ~((nan_codes(w.z) >> 7) * 255u); w.w &= ~((nan_codes(w.w) >> 7) * 255u);
                    }
                    uint32_t u[8] = {w.x, w.x >> 16, w.y, w.y >> 16, w.z, w.z >> 16, w.w, w.w >> 16};
#pragma unroll
                    for (int i = 0; i < 8; ++i) asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(u[i]) : "r"(e4m3_f16(u[i])), "r"(f2));
                    *reinterpret_cast<uint4*>(to + (((2 * d) ^ (t & 7)) << 4)) = make_uint4(u[0], u[1], u[2], u[3]);
                    *reinterpret_cast<uint4*>(to + (((2 * d + 1) ^ (t & 7)) << 4)) = make_uint4(u[4], u[5], u[6], u[7]);
                }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) { mbar_arrive(&v_full[vst]); mbar_arrive(&raw_empty[rs]); }
        }
        if (!ok && lane == 0) { *abort_flag = 1; atomicExch(p.err, 80); }
    }

    __syncwarp();
    if (*abort_flag) for (int i = 0; i < 64; ++i) __nanosleep(1000);
    tc_fence_before();
    __syncthreads();
    if (warp == 1) { tc_fence_after(); tmem_dealloc(tmem_base, Sh::TMEM); }
}

template <int NH, bool E4M3>
int launch_rows(DeviceCtx* ctx, const TbKvCache* c, const PagedAttParams& p, cudaStream_t st) {
    typedef RowsShape<NH, E4M3> Sh;
    static_assert(Sh::PER_SM == paged_per_sm(NH, E4M3) && Sh::PER_SM <= PA_MOST_PER_SM, "the plan counts on as many CTAs per SM");
    CUtensorMap tmK, tmV;
    const int box_rows = std::min(c->page_size, Sh::KEYS);
    TB_TRY(make_cache_map(&tmK, c->K, E4M3 ? 1 : 2, c->head_dim, c->page_size, (long long)c->pages * c->heads, 64 * (E4M3 ? NH : 1), box_rows, !E4M3));
    TB_TRY(make_cache_map(&tmV, c->V, E4M3 ? 1 : 2, c->head_dim, c->page_size, (long long)c->pages * c->heads, 64 * (E4M3 ? NH : 1), box_rows, !E4M3));
    static bool attr_set[64] = {false};
    if (!attr_set[ctx->device & 63]) {
        TB_CUDA(cudaFuncSetAttribute(paged_rows_kernel<NH, E4M3>, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::SMEM));
        attr_set[ctx->device & 63] = true;
    }
    prof_mark(ctx, "paged_rows", 0.0, 0.0, st);          // (how much of the batch is whose, and how long it is, only the device knows)
    TB_CUDA(launch_kernel_early(paged_rows_kernel<NH, E4M3>, dim3(p.grid), dim3(PA_THREADS), Sh::SMEM, st, tmK, tmV, p));
    ctx->launches++;
    prof_close(ctx, st);
    return 0;
}

template <int NH, bool E4M3>
int plan_chunks(DeviceCtx* ctx, const PagedAttParams& p, const PagedPlan& pl, uint8_t* ws, PagedChunkParams* pp, cudaStream_t st) {
    typedef ChunkShape<NH, E4M3> Sh;
    static_assert(Sh::PER_SM == paged_tiles_per_sm(NH, E4M3), "the plan counts on as many CTAs per SM");
    pp->a = p;
    pp->tokens = PT_ROWS / p.group;
    pp->tiles = (p.max_q + pp->tokens - 1) / pp->tokens;
    pp->planned = pl.most_units > 0 ? 1 : 0; pp->most_units = pl.most_units; pp->most_pieces = pl.most_pieces; pp->slots = Sh::PER_SM * ctx->sm_count;
    // a CTA with a tile takes the place of one of the two that an SM holds for few rows, or of all
    pp->rows_keys_log2 = paged_keys(NH, E4M3) == 128 ? 7 : 6; pp->rows_cost = NH == 2 && !E4M3 ? 6 : 3;
    pp->rows_slots = paged_per_sm(NH, E4M3) * ctx->sm_count; pp->rows_lost = Sh::TS ? paged_per_sm(NH, E4M3) : 1;
    // (see paged_plan.h for the room)
    pp->count = reinterpret_cast<int*>(ws);
    pp->arrived = reinterpret_cast<unsigned int*>(ws + 16);
    pp->bad = reinterpret_cast<int*>(pp->arrived + pl.most_units);
    pp->units = reinterpret_cast<ChunkUnit*>(pp->bad + pl.most_units);
    pp->part_ml = reinterpret_cast<float2*>(pp->units + pl.most_units);
    pp->part_o = reinterpret_cast<float4*>(pp->part_ml + (size_t)pl.most_pieces * PT_ROWS);
    if (!pp->planned) return 0;
    prof_mark(ctx, "paged_plan", 0.0, 0.0, st);
    TB_CUDA(launch_kernel(paged_plan_kernel, dim3(1), dim3(PL_THREADS), 0, st, *pp));
    ctx->launches++;
    prof_close(ctx, st);
    return 0;
}

template <int NH, bool E4M3>
int launch_chunks(DeviceCtx* ctx, const TbKvCache* c, const PagedChunkParams& pp, cudaStream_t st) {
    typedef ChunkShape<NH, E4M3> Sh;
    const PagedAttParams& p = pp.a;
    CUtensorMap tmQ, tmK, tmV;
    TB_TRY(make_query_map(&tmQ, p.Q, c->head_dim, p.H, p.rows, p.ld_q, p.group, pp.tokens));
    const int box_rows = std::min(c->page_size, PT_KEYS);
    TB_TRY(make_cache_map(&tmK, c->K, E4M3 ? 1 : 2, c->head_dim, c->page_size, (long long)c->pages * c->heads, E4M3 ? 128 : 64, box_rows, true));
    TB_TRY(make_cache_map(&tmV, c->V, E4M3 ? 1 : 2, c->head_dim, c->page_size, (long long)c->pages * c->heads, 64 * (E4M3 ? NH : 1), box_rows, !E4M3));
    static bool attr_set[64] = {false};
    if (!attr_set[ctx->device & 63]) {
        TB_CUDA(cudaFuncSetAttribute(paged_chunk_kernel<NH, E4M3>, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::SMEM));
        attr_set[ctx->device & 63] = true;
    }
    prof_mark(ctx, "paged_chunk", 0.0, 0.0, st);
    // (rows * q_heads is below 2^31, so that there are no more than 2^24 tiles)
    const unsigned layer = std::min(pp.tiles, 65535);
    const dim3 grid = pp.planned ? dim3(pp.most_units) : dim3((unsigned)c->heads * (unsigned)c->seqs, layer, ((unsigned)pp.tiles + layer - 1) / layer);
    TB_CUDA(launch_kernel_early(paged_chunk_kernel<NH, E4M3>, grid, dim3(Sh::THREADS), Sh::SMEM, st, tmQ, tmK, tmV, static_cast<const uint8_t*>(c->V), pp));
    ctx->launches++;
    prof_close(ctx, st);
    return 0;
}

template <int NH, bool E4M3>
int launch_both(DeviceCtx* ctx, const TbKvCache* c, PagedAttParams& p, const PagedPlan& pl, uint8_t* more, cudaStream_t st) {
    if (p.behind_chunks) {
        PagedChunkParams pp;
        TB_TRY((plan_chunks<NH, E4M3>(ctx, p, pl, more, &pp, st)));
        TB_TRY((launch_chunks<NH, E4M3>(ctx, c, pp, st)));
        if (pp.planned) p.runs = pp.count + 1;
    }
    return launch_rows<NH, E4M3>(ctx, c, p, st);
}

}  // namespace

int launch_attention_paged(DeviceCtx* ctx, const TbKvCache* c, const int* q_start, const int* kv_len, const bf16* Q, long long ld_q, int rows,
                           int H, int max_q, int max_kv, float scale, bf16* att, long long ld_att, float* lse, void* ws, int64_t ws_bytes,
                           cudaStream_t st) {
    const int group = H / c->heads;
    const PagedPlan pl = paged_plan(c->seqs, c->heads, group, c->head_dim, c->type == TB_KV_E4M3, rows, max_q, max_kv, ctx->sm_count);
    TB_CHECK(pl.workspace == 0 || (ws != nullptr && ws_bytes >= pl.workspace), "tb_attention_paged: the workspace has %lld bytes, %lld are needed",
             (long long)(ws ? ws_bytes : 0), (long long)pl.workspace);
    PagedAttParams p;
    p.v = paged_view(c);
    p.q_start = q_start; p.kv_len = kv_len; p.Q = Q; p.ld_q = ld_q; p.K = c->K; p.ks = c->k_scale; p.vs = c->v_scale;
    p.att = att; p.ld_att = ld_att; p.lse = lse;
    p.part_o = static_cast<float*>(ws) + paged_counters(ctx->sm_count);
    p.part_ml = reinterpret_cast<float2*>(p.part_o + 2LL * pl.grid * PA_ROWS * c->head_dim);
    p.arrived = static_cast<unsigned int*>(ws);
    p.rows = rows; p.H = H; p.group = group; p.max_q = max_q; p.max_kv = max_kv; p.grid = pl.grid; p.whole = pl.whole ? 1 : 0;
    p.scale_log2 = scale * 1.4426950408889634f; p.err = ctx->d_err;
    p.group_magic = (65536u + group - 1) / group; p.behind_chunks = max_q * (long long)group > PA_ROWS ? 1 : 0;
    p.runs = nullptr;
    const bool wide = c->head_dim > 64, e4m3 = c->type == TB_KV_E4M3;
    uint8_t* more = static_cast<uint8_t*>(ws) + pl.rows_bytes;
    return e4m3 ? (wide ? launch_both<2, true>(ctx, c, p, pl, more, st) : launch_both<1, true>(ctx, c, p, pl, more, st))
                : (wide ? launch_both<2, false>(ctx, c, p, pl, more, st) : launch_both<1, false>(ctx, c, p, pl, more, st));
}

}  // namespace tb

using namespace tb;

static int check_attention(const TbKvCache* cache, int rows, int q_heads, int max_q, int max_kv) {
    TB_TRY(check_cache(cache, "tb_attention_paged"));
    TB_CHECK(rows >= 0 && max_q >= 0 && max_kv >= 0, "tb_attention_paged: rows, max_q and max_kv must not be negative");
    TB_CHECK(q_heads > 0 && q_heads % cache->heads == 0, "tb_attention_paged: %d query heads cannot share %d key heads", q_heads, cache->heads);
    TB_CHECK(q_heads / cache->heads <= PT_ROWS, "tb_attention_paged: at most %d query heads share a key head (got %d)", PT_ROWS, q_heads / cache->heads);
    TB_CHECK((long long)rows * q_heads < (1LL << 31), "tb_attention_paged: rows * q_heads must be below 2^31");
    return 0;
}

extern "C" {

int64_t tb_attention_paged_workspace(const TbKvCache* cache, int rows, int q_heads, int max_q, int max_kv) {
    DeviceCtx* ctx;
    if (check_attention(cache, rows, q_heads, max_q, max_kv) != 0 || get_ctx(&ctx) != 0) return -1;
    return paged_plan(cache->seqs, cache->heads, q_heads / cache->heads, cache->head_dim, cache->type == TB_KV_E4M3, rows, std::min(max_q, rows),
                      max_kv, ctx->sm_count).room;
}

int tb_attention_paged(const TbKvCache* cache, const int32_t* d_q_start, const int32_t* d_kv_len, const void* d_Q, int64_t ld_q, int rows,
                       int q_heads, int max_q, int max_kv, float scale, void* d_att, int64_t ld_att, float* d_lse, void* d_workspace,
                       int64_t workspace_bytes, void* stream) {
    TB_TRY(check_attention(cache, rows, q_heads, max_q, max_kv));
    if (rows == 0 || max_q == 0) return 0;
    TB_CHECK(d_q_start && d_kv_len && d_Q && d_att, "tb_attention_paged: NULL operand");
    const long long width = (long long)q_heads * cache->head_dim;
    TB_CHECK(ld_q >= width && ld_q % 8 == 0 && ld_att >= width && ld_att % 8 == 0,
             "tb_attention_paged: leading dimensions must be multiples of 8 and at least %lld (got %lld, %lld)", width, (long long)ld_q,
             (long long)ld_att);
    TB_CHECK(((reinterpret_cast<uintptr_t>(d_Q) | reinterpret_cast<uintptr_t>(d_att) | reinterpret_cast<uintptr_t>(d_workspace)) & 15u) == 0,
             "tb_attention_paged: rows and workspace must be 16-byte aligned");
    TB_CHECK(scale > 0.f && scale < INFINITY, "tb_attention_paged: scale must be positive and finite");
    const RowSpan q = {d_Q, rows, width * 2, ld_q * 2}, att = {d_att, rows, width * 2, ld_att * 2}, lse = {d_lse, 1, (long long)rows * q_heads * 4, 0};
    const RowSpan room = {workspace_bytes > 0 ? d_workspace : nullptr, 1, workspace_bytes, 0};
    TB_CHECK(!spans_overlap(q, att), "tb_attention_paged: the result must not lie over the queries");
    TB_CHECK(!spans_overlap(lse, q) && !spans_overlap(lse, att), "tb_attention_paged: the sums must not lie over the queries or the result");
    TB_CHECK(!spans_overlap(room, q) && !spans_overlap(room, att) && !spans_overlap(room, lse),
             "tb_attention_paged: the workspace must not lie over the queries, the result or the sums");
    TB_CHECK(!over_pools(cache, att) && !over_pools(cache, lse) && !over_pools(cache, room),
             "tb_attention_paged: the result, the sums and the workspace must not lie over the pools");
    DeviceCtx* ctx;
    TB_TRY(get_ctx(&ctx));
    return launch_attention_paged(ctx, cache, d_q_start, d_kv_len, static_cast<const bf16*>(d_Q), ld_q, rows, q_heads, std::min(max_q, rows),
                                  max_kv, scale, static_cast<bf16*>(d_att), ld_att, d_lse, d_workspace, workspace_bytes,
                                  static_cast<cudaStream_t>(stream));
}

}  // extern "C"
