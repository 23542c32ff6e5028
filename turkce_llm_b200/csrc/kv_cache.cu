// Writing new tokens' keys and values into a paged cache, position rotation included, and reading rows of it back.
//
// Both kernels move bytes and do little else: eight elements of one head per thread, so that a head of 64 is one 256-byte
// (float32), 128-byte (bf16) or 64-byte (8-bit) piece of consecutive threads on either side.  A warp belongs to one row
// (token), and finds the row's sequence, position and page once for all its heads.
#include "paged.cuh"

#include <algorithm>

namespace tb {

int check_cache(const TbKvCache* c, const char* who) {
    TB_CHECK(c != nullptr, "%s: NULL cache", who);
    TB_CHECK(c->K && c->V && c->table, "%s: the cache has a NULL pool or table", who);
    TB_CHECK(c->type == TB_KV_BF16 || c->type == TB_KV_E4M3, "%s: unknown cache type %d", who, c->type);
    const int step = c->type == TB_KV_E4M3 ? 16 : 8;
    TB_CHECK(c->head_dim >= step && c->head_dim <= 128 && c->head_dim % step == 0, "%s: head_dim must be a multiple of %d up to 128 (got %d)",
             who, step, c->head_dim);
    TB_CHECK(c->page_size == 16 || c->page_size == 32 || c->page_size == 64 || c->page_size == 128 || c->page_size == 256,
             "%s: page_size must be 16, 32, 64, 128 or 256 (got %d)", who, c->page_size);
    TB_CHECK(c->pages > 0 && c->heads > 0 && c->seqs > 0 && c->table_ld > 0, "%s: cache dims must be positive", who);
    TB_CHECK((long long)c->pages * c->heads < (1LL << 31), "%s: pages * heads must be below 2^31", who);
    TB_CHECK((long long)c->table_ld * c->page_size < (1LL << 31), "%s: table_ld * page_size must be below 2^31", who);
    TB_CHECK(c->seqs <= 65535, "%s: at most 65535 sequences (got %d)", who, c->seqs);
    const uintptr_t at = reinterpret_cast<uintptr_t>(c->K) | reinterpret_cast<uintptr_t>(c->V);
    TB_CHECK((at & 15u) == 0, "%s: the pools must be 16-byte aligned", who);
    if (c->type == TB_KV_E4M3) {
        TB_CHECK(c->k_scale && c->v_scale, "%s: an 8-bit cache needs both scale arrays", who);
        TB_CHECK(((reinterpret_cast<uintptr_t>(c->k_scale) | reinterpret_cast<uintptr_t>(c->v_scale)) & 15u) == 0,
                 "%s: the scale arrays must be 16-byte aligned", who);
    } else {
        TB_CHECK(!c->k_scale && !c->v_scale, "%s: a bf16 cache has no scales", who);
    }
    return 0;
}

namespace {

constexpr int KV_THREADS = 256;
constexpr int KV_WARPS = KV_THREADS / 32;
constexpr int KV_ROUND = 4;          // (read) groups of heads that a warp asks for at a time
constexpr int KV_AHEAD = 3;          // (append) groups of heads on their way to a warp

struct AppendParams {
    PagedView v;
    const int *q_start, *kv_len;
    const void* x; long long ld_x;
    int rows, H, per_warp, parts, threads_log2;       // rows per warp, or warps per row; threads per head: 1 << threads_log2
    const float *cos_t, *sin_t;
    int positions, half, aligned;                     // rot_dim / 2; both tables begin on 16 bytes
    bf16* Q; long long ld_q;
    void *K, *V;
    float *ks, *vs;
    int* err;
};

// eight elements as they lie in memory, and as float32
template <bool BF16_IN> struct Raw8 { uint4 w[BF16_IN ? 1 : 2]; };
__device__ __forceinline__ void copy_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
template <bool BF16_IN>
__device__ __forceinline__ void widen8(const Raw8<BF16_IN>& r, float (&f)[8]) {
    if (BF16_IN) {
        const uint32_t u[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 p = bf16_floats(u[i]);
            f[2 * i] = p.x; f[2 * i + 1] = p.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint4 w = r.w[BF16_IN ? 0 : i];
            f[4 * i] = __uint_as_float(w.x); f[4 * i + 1] = __uint_as_float(w.y);
            f[4 * i + 2] = __uint_as_float(w.z); f[4 * i + 3] = __uint_as_float(w.w);
        }
    }
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
    return make_uint4(bf16_pair(f[0], f[1]), bf16_pair(f[2], f[3]), bf16_pair(f[4], f[5]), bf16_pair(f[6], f[7]));
}

// Where the rows row0 .. row0 + count - 1 (count <= 32) of a warp belong: lane i has row row0 + i's sequence (-1: none), the end of that
// sequence's rows and a number of it (lens[s]).  Rows of one sequence, the usual case, take one look at the starts.
struct RowsOf { int s, end, len; };
__device__ __forceinline__ RowsOf rows_of(const int* __restrict__ start, const int* __restrict__ lens, int seqs, int row0, int count) {
    const int lane = threadIdx.x & 31, row = row0 + min(lane, count - 1);
    RowsOf r;
    r.s = sequence_of(start, seqs, row0);
    r.end = r.s >= 0 ? start[r.s + 1] : row0;
    if (row0 + count > r.end) {                                  // (the same for all lanes)
        int lo = 0, hi = seqs;                                   // the last start at or before this lane's row is in [lo, hi)
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (start[mid] <= row) lo = mid;
            else hi = mid;
        }
        r.s = start[lo] <= row ? lo : -1;
        r.end = r.s >= 0 ? start[r.s + 1] : row;
        if (row >= r.end) r.s = -1;                              // behind the last sequence
    }
    r.len = r.s >= 0 && lens ? lens[r.s] : 0;
    return r;
}
__device__ __forceinline__ long long shfl64(long long x, int lane) {
    return (long long)__shfl_sync(0xffffffffu, (unsigned long long)x, lane);
}

// Rotated elements are a cos - b sin and a sin + b cos with every product rounded, the same sums whichever thread forms them.
// A warp has p.per_warp rows, or a row's every `parts`-th group of heads.  The groups come through a ring in shared memory, KV_AHEAD of them
// on their way while it works on one, a thread reading what it asked for itself: with the next group alone on its way, in registers, an SM
// had 12 KB in flight, and 12,600 rows of 12 + 8 heads of 64 into an 8-bit cache took 31 us.
template <bool BF16_IN, bool HALVES, bool E4M3>
__global__ void __launch_bounds__(KV_THREADS, 3)
kv_append_kernel(const AppendParams p) {
    __shared__ Raw8<BF16_IN> ring[KV_WARPS][KV_AHEAD + 1][32];
    __shared__ float4 angles[KV_WARPS][2][32];                   // cosines, then sines, of this row and the next
    pdl_wait();
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned w = blockIdx.x * KV_WARPS + warp;
    const int part = (int)(w % (unsigned)p.parts), row0 = (int)(w / (unsigned)p.parts) * p.per_warp;
    if (row0 >= p.rows) return;                                  // (whole warps)
    const int count = min(p.per_warp, p.rows - row0);
    const int hd = p.v.hd, G = p.v.heads, all = p.H + 2 * G;
    const int heads_of_warp = 32 >> p.threads_log2, step = heads_of_warp * p.parts;
    const int e0 = (lane & ((1 << p.threads_log2) - 1)) * 8;     // first of this thread's elements
    const int first_head = part * heads_of_warp + (lane >> p.threads_log2);
    const int groups = (all - part * heads_of_warp + step - 1) / step, total = count * groups;
    const bool lane_in = e0 < hd;
    // the next (row, group of heads) to be asked for, and its place in the ring
    constexpr int SIZE = BF16_IN ? 2 : 4;
    const char* next = static_cast<const char*>(p.x) + ((long long)row0 * p.ld_x + (first_head * hd + e0)) * SIZE;
    const int to_next_group = step * hd * SIZE;
    const long long to_next_row = p.ld_x * SIZE - (long long)(groups - 1) * to_next_group;
    int next_group = 0, left = total, place = 0;
    const int last_group = lane_in ? groups - (first_head + (groups - 1) * step < all ? 0 : 1) : 0;      // groups that have this lane's head
    auto ask = [&]() {
        if (left > 0) {
            if (next_group < last_group) {
                Raw8<BF16_IN>& to = ring[warp][place][lane];
                copy_async16(&to, next);
                if (!BF16_IN) copy_async16(reinterpret_cast<uint4*>(&to) + 1, next + 16);
            }
            --left;
            const bool wrap = ++next_group == groups;
            next += wrap ? to_next_row : (long long)to_next_group;
            next_group = wrap ? 0 : next_group;
            place = place == KV_AHEAD ? 0 : place + 1;
        }
        copy_async_commit();
    };
#pragma unroll
    for (int j = 0; j < KV_AHEAD; ++j) ask();                    // (needs nothing of the batch)
    // ---- lane i: position and place in the cache of row row0 + i
    const RowsOf mine_of = rows_of(p.q_start, p.kv_len, p.v.seqs, row0, count);
    long long my_pos = (long long)mine_of.len - mine_of.end + row0 + lane, my_slot = -1;
    if (mine_of.s < 0 || lane >= count) {
        my_pos = -1;
    } else if (my_pos < 0 || my_pos >= (long long)p.v.table_ld << p.v.page_shift || (p.half > 0 && my_pos >= p.positions)) {
        report_argument(p.err, 72);
        my_pos = -1;
    } else {
        const int page = p.v.table[(long long)mine_of.s * p.v.table_ld + (my_pos >> p.v.page_shift)];
        if ((unsigned)page < (unsigned)p.v.pages) my_slot = ((long long)page * G << p.v.page_shift) + (my_pos & ((1 << p.v.page_shift) - 1));
        else report_argument(p.err, 71);
    }
    // (halves) partners are read from the other thread's place in the ring, all eight at once where they are a whole number of threads apart
    const bool by_lane = HALVES && (p.half & 7) == 0;
    const int other_lane = !by_lane || e0 >= 2 * p.half ? lane : e0 < p.half ? lane + (p.half >> 3) : lane - (p.half >> 3);
    // A row's angles: with the groups of the row before it, where these are enough for them to have arrived.
    const bool wide_angles = p.aligned && (p.half & 3) == 0, angles_ahead = wide_angles && groups >= KV_AHEAD && p.half > 0;
    auto ask_angles = [&](int i) {
        const long long next_pos = shfl64(my_pos, i);
        const int quads = p.half >> 2;
        if (next_pos >= 0 && lane < 2 * quads)
            copy_async16(&angles[warp][i & 1][lane], (lane < quads ? p.cos_t : p.sin_t) + next_pos * p.half + (lane < quads ? lane : lane - quads) * 4);
    };
    // this thread's angles of the row at hand; they are the same in every head
    float c[HALVES ? 8 : 4], d[HALVES ? 8 : 4];
    long long pos = -1, slot = -1;
    int i = -1, group = groups - 1, at_ring = KV_AHEAD;
#pragma unroll 1
    for (int k0 = 0; k0 < total; ++k0) {
        __syncwarp();                                            // (other lanes' elements and angles are read)
        if (group == groups - 1 && angles_ahead && i + 2 < count) ask_angles(i + 2);
        ask();
        copy_async_wait<KV_AHEAD>();
        __syncwarp();
        at_ring = at_ring == KV_AHEAD ? 0 : at_ring + 1;
        if (++group == groups) {
            group = 0;
            ++i;
            pos = shfl64(my_pos, i); slot = shfl64(my_slot, i);
            if (p.half > 0 && pos >= 0) {
                // (the same angles in memory and in the ring: generic addresses)
                const float* ct = angles_ahead && i > 0 ? reinterpret_cast<const float*>(angles[warp][i & 1]) : p.cos_t + pos * p.half;
                const float* st = angles_ahead && i > 0 ? ct + p.half : p.sin_t + pos * p.half;
                if (HALVES ? by_lane && wide_angles : wide_angles) {
                    const int e = HALVES ? e0 : e0 >> 1, at = HALVES && e >= p.half ? e - p.half : e;
                    const bool turns = HALVES ? e < 2 * p.half : e < p.half;
                    const float flip = HALVES && e < p.half ? -1.f : 1.f;        // a cos - b sin as a cos + b (-sin): the same rounding
#pragma unroll
                    for (int k = 0; k < (HALVES ? 8 : 4); k += 4) {
                        const float4 x = turns ? *reinterpret_cast<const float4*>(ct + at + k) : make_float4(1.f, 1.f, 1.f, 1.f);
                        const float4 y = turns ? *reinterpret_cast<const float4*>(st + at + k) : make_float4(0.f, 0.f, 0.f, 0.f);
                        c[k] = x.x; c[k + 1] = x.y; c[k + 2] = x.z; c[k + 3] = x.w;
                        d[k] = y.x * flip; d[k + 1] = y.y * flip; d[k + 2] = y.z * flip; d[k + 3] = y.w * flip;
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < (HALVES ? 8 : 4); ++k) {
                        const int e = HALVES ? e0 + k : (e0 >> 1) + k, at = HALVES && e >= p.half ? e - p.half : e;
                        const bool turns = HALVES ? e < 2 * p.half : e < p.half;
                        c[k] = turns ? ct[at] : 1.f;
                        d[k] = turns ? (HALVES && e < p.half ? -st[at] : st[at]) : 0.f;
                    }
                }
            }
        }
        if (pos < 0) continue;                                   // not of the batch, or out of range
        {
            const int head = first_head + group * step, row = row0 + i;
            const bool mine = lane_in && head < all;
            const int warp_head = head - (lane >> p.threads_log2);   // the warp's first head
            float x[8];
            if (mine) {
                widen8<BF16_IN>(ring[warp][at_ring][lane], x);
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k) x[k] = 0.f;
            }
            if (p.half > 0 && warp_head < p.H + G) {             // (a group of values alone has nothing to rotate)
                const bool turns = head < p.H + G;
                if (!HALVES) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        if (turns && (e0 >> 1) + k < p.half) {
                            const float a = x[2 * k], b = x[2 * k + 1];
                            x[2 * k] = __fsub_rn(__fmul_rn(a, c[k]), __fmul_rn(b, d[k]));
                            x[2 * k + 1] = __fadd_rn(__fmul_rn(a, d[k]), __fmul_rn(b, c[k]));
                        }
                    }
                } else if (by_lane) {
                    if (mine && turns && e0 < 2 * p.half) {
                        float other[8];
                        widen8<BF16_IN>(ring[warp][at_ring][other_lane], other);
#pragma unroll
                        for (int k = 0; k < 8; ++k) x[k] = __fadd_rn(__fmul_rn(x[k], c[k]), __fmul_rn(other[k], d[k]));
                    }
                } else {
                    const int first_lane = lane >> p.threads_log2 << p.threads_log2;
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int e = e0 + k;
                        if (mine && turns && e < 2 * p.half) {
                            const int o = e < p.half ? e + p.half : e - p.half;
                            const Raw8<BF16_IN>* from = &ring[warp][at_ring][first_lane + (o >> 3)];
                            const float other = BF16_IN ? __bfloat162float(reinterpret_cast<const bf16*>(from)[o & 7]) : reinterpret_cast<const float*>(from)[o & 7];
                            x[k] = __fadd_rn(__fmul_rn(x[k], c[k]), __fmul_rn(other, d[k]));
                        }
                    }
                }
            }
            if (warp_head < p.H && mine && head < p.H) *reinterpret_cast<uint4*>(p.Q + (long long)row * p.ld_q + (head * hd + e0)) = pack8(x);
            if (warp_head + heads_of_warp <= p.H) continue;      // (queries alone)
            // largest magnitude of the row: as integers, so that NaN is larger than infinity and infinity than the rest
            uint32_t big = 0u;
            if (E4M3) {
#pragma unroll
                for (int k = 0; k < 8; ++k) big = max(big, __float_as_uint(x[k]) & 0x7fffffffu);
                for (int o = (1 << p.threads_log2) >> 1; o > 0; o >>= 1) big = max(big, __shfl_xor_sync(0xffffffffu, big, o));
            }
            if (!mine || head < p.H || slot < 0) continue;
            const bool key = head < p.H + G;
            const long long at = slot + ((head - p.H - (key ? 0 : G)) << p.v.page_shift);
            if (!E4M3) {
                *reinterpret_cast<uint4*>(static_cast<bf16*>(key ? p.K : p.V) + at * hd + e0) = pack8(x);
            } else {
                float inverse;
                const float scale = e4m3_scale(__uint_as_float(big), &inverse);
                float by = scale;
                if (scale < E4M3_SMALL) {                        // (remainders would be below what float32 has: all of it 2^64 times as large)
                    by *= 0x1p64f; inverse *= 0x1p-64f;
#pragma unroll
                    for (int k = 0; k < 8; ++k) x[k] *= 0x1p64f;
                }
                uint32_t q[4];
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    q[k] = e4m3_pair(quotient_to_odd(x[2 * k], by, inverse), quotient_to_odd(x[2 * k + 1], by, inverse));
                *reinterpret_cast<uint2*>(static_cast<uint8_t*>(key ? p.K : p.V) + at * hd + e0) = make_uint2(q[0] | q[1] << 16, q[2] | q[3] << 16);
                if (e0 == 0) (key ? p.ks : p.vs)[at] = scale;
            }
        }
    }
}

struct ReadParams {
    PagedView v;
    const int *start, *first;
    int rows, per_warp, parts, threads_log2, kinds;   // rows per warp, or warps per row; threads per head; 1 or 2 of K and V
    const void *A, *B;                                // the pools read (B: the second one)
    const float *as, *bs;
    bf16 *oA, *oB;
    long long ld_row, ld_head;
    int* err;
};

template <bool E4M3>
__global__ void __launch_bounds__(KV_THREADS)
kv_read_kernel(const ReadParams p) {
    pdl_wait();
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned w = blockIdx.x * KV_WARPS + warp;
    const int part = (int)(w % (unsigned)p.parts), row0 = (int)(w / (unsigned)p.parts) * p.per_warp;
    if (row0 >= p.rows) return;
    const int count = min(p.per_warp, p.rows - row0);
    const int hd = p.v.hd, G = p.v.heads, all = p.kinds * G;
    const int heads_of_warp = 32 >> p.threads_log2, step = heads_of_warp * p.parts;
    constexpr int EPT = E4M3 ? 16 : 8;                           // elements per thread: 16 bytes of the cache
    const int e0 = (lane & ((1 << p.threads_log2) - 1)) * EPT;
    // ---- lane i: the place in the cache of row row0 + i
    const RowsOf mine_of = rows_of(p.start, p.first, p.v.seqs, row0, count);
    long long my_slot = -1;
    if (mine_of.s >= 0 && lane < count) {
        const long long t = (long long)row0 + lane - p.start[mine_of.s] + mine_of.len;
        if (t < 0 || t >= (long long)p.v.table_ld << p.v.page_shift) {
            report_argument(p.err, 72);
        } else {
            const int page = p.v.table[(long long)mine_of.s * p.v.table_ld + (t >> p.v.page_shift)];
            if ((unsigned)page < (unsigned)p.v.pages) my_slot = ((long long)page * G << p.v.page_shift) + (t & ((1 << p.v.page_shift) - 1));
            else report_argument(p.err, 71);
        }
    }
    // All (row, group of heads) pairs of the warp, four of them on their way at a time
    const int groups = (all - part * heads_of_warp + step - 1) / step, total = count * groups;
#pragma unroll 1
    for (int k0 = 0; k0 < total; k0 += KV_ROUND) {
        uint4 in[KV_ROUND];
        float scale[KV_ROUND];
        long long to[KV_ROUND];
        bool second[KV_ROUND];
#pragma unroll
        for (int j = 0; j < KV_ROUND; ++j) {
            const int k = min(k0 + j, total - 1), i = k / groups, head = part * heads_of_warp + (k - i * groups) * step + (lane >> p.threads_log2);
            const long long slot = shfl64(my_slot, i);
            second[j] = head >= G;
            const int h = second[j] ? head - G : head;
            to[j] = -1;
            if (slot >= 0 && k0 + j < total && head < all && e0 < hd) {
                to[j] = (long long)(row0 + i) * p.ld_row + h * p.ld_head + e0;
                const long long at = slot + ((long long)h << p.v.page_shift);
                in[j] = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(second[j] ? p.B : p.A) + (at * hd + e0) * (E4M3 ? 1 : 2)));
                if (E4M3) scale[j] = __ldg((second[j] ? p.bs : p.as) + at);
            }
        }
#pragma unroll
        for (int j = 0; j < KV_ROUND; ++j) {
            if (to[j] < 0) continue;
            uint4* o16 = reinterpret_cast<uint4*>((second[j] ? p.oB : p.oA) + to[j]);
            if (E4M3) {
                const uint32_t u[4] = {in[j].x, in[j].y, in[j].z, in[j].w};
                uint32_t o[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float2 f = e4m3_floats(i & 1 ? u[i >> 1] >> 16 : u[i >> 1] & 0xffffu);
                    o[i] = bf16_pair(f.x * scale[j], f.y * scale[j]);
                }
                o16[0] = make_uint4(o[0], o[1], o[2], o[3]);
                o16[1] = make_uint4(o[4], o[5], o[6], o[7]);
            } else {
                o16[0] = in[j];
            }
        }
    }
}

// threads per head (a power of two that divides a warp), and how rows are dealt to warps: what a warp finds out about a sequence
// serves up to four rows, where that leaves sixteen warps for every SM; where there are fewer rows than eight for every SM, a row's
// groups of heads go to different warps.
void shape_of(const DeviceCtx* ctx, int hd, int elements, int heads, int rows, int* threads_log2, int* per_warp, int* parts, long long* blocks) {
    int t = 0;
    while ((elements << t) < hd) ++t;
    *threads_log2 = t;
    const int in_warp = 32 >> t, groups = (heads + in_warp - 1) / in_warp;
    *parts = (int)std::max<long long>(1, std::min<long long>(groups, 8LL * ctx->sm_count / rows));
    *per_warp = (int)std::max<long long>(1, std::min<long long>(4, rows / (16LL * ctx->sm_count)));
    *blocks = (((long long)rows + *per_warp - 1) / *per_warp * *parts + KV_WARPS - 1) / KV_WARPS;
}

}  // namespace

int launch_kv_append(DeviceCtx* ctx, const TbKvCache* c, const int* q_start, const int* kv_len, const void* x, bool x_bf16, long long ld_x,
                     int rows, int H, const float* cos_t, const float* sin_t, int positions, int rot_dim, int form, bf16* Q,
                     long long ld_q, cudaStream_t st) {
    AppendParams p;
    p.v = paged_view(c);
    p.q_start = q_start; p.kv_len = kv_len; p.x = x; p.ld_x = ld_x; p.rows = rows; p.H = H;
    p.cos_t = cos_t; p.sin_t = sin_t; p.positions = positions; p.half = rot_dim / 2;
    p.aligned = ((reinterpret_cast<uintptr_t>(cos_t) | reinterpret_cast<uintptr_t>(sin_t)) & 15u) == 0;
    p.Q = Q; p.ld_q = ld_q; p.K = c->K; p.V = c->V; p.ks = c->k_scale; p.vs = c->v_scale; p.err = ctx->d_err;
    long long blocks;
    shape_of(ctx, c->head_dim, 8, H + 2 * c->heads, rows, &p.threads_log2, &p.per_warp, &p.parts, &blocks);
    TB_CHECK(blocks < (1LL << 31) / KV_WARPS, "tb_kv_append: too many rows");
    typedef void (*Kernel)(AppendParams);
    const bool halves = form == TB_ROPE_HALVES && rot_dim > 0, e4m3 = c->type == TB_KV_E4M3;
    static const Kernel kernels[8] = {
        kv_append_kernel<false, false, false>, kv_append_kernel<false, false, true>, kv_append_kernel<false, true, false>,
        kv_append_kernel<false, true, true>, kv_append_kernel<true, false, false>, kv_append_kernel<true, false, true>,
        kv_append_kernel<true, true, false>, kv_append_kernel<true, true, true>};
    const double n = (double)rows * c->head_dim;
    prof_mark(ctx, "kv_append", 0.0, n * ((H + 2.0 * c->heads) * (x_bf16 ? 2 : 4) + 2.0 * H + 2.0 * c->heads * (e4m3 ? 1 : 2)), st);
    TB_CUDA(launch_kernel(kernels[(x_bf16 ? 4 : 0) + (halves ? 2 : 0) + (e4m3 ? 1 : 0)], dim3((unsigned)blocks), dim3(KV_THREADS), 0, st, p));
    ctx->launches++;
    prof_close(ctx, st);
    return 0;
}

int launch_kv_read(DeviceCtx* ctx, const TbKvCache* c, const int* start, const int* first, int rows, bf16* K, bf16* V, long long ld_row,
                   long long ld_head, cudaStream_t st) {
    ReadParams p;
    p.v = paged_view(c);
    p.start = start; p.first = first; p.rows = rows; p.kinds = K && V ? 2 : 1;
    p.A = K ? c->K : c->V; p.as = K ? c->k_scale : c->v_scale; p.oA = K ? K : V;
    p.B = c->V; p.bs = c->v_scale; p.oB = V;
    p.ld_row = ld_row; p.ld_head = ld_head; p.err = ctx->d_err;
    long long blocks;
    shape_of(ctx, c->head_dim, c->type == TB_KV_E4M3 ? 16 : 8, p.kinds * c->heads, rows, &p.threads_log2, &p.per_warp, &p.parts, &blocks);
    TB_CHECK(blocks < (1LL << 31) / KV_WARPS, "tb_kv_read: too many rows");
    const bool e4m3 = c->type == TB_KV_E4M3;
    prof_mark(ctx, "kv_read", 0.0, (double)rows * p.kinds * c->heads * c->head_dim * (e4m3 ? 3 : 4), st);
    TB_CUDA(launch_kernel(e4m3 ? kv_read_kernel<true> : kv_read_kernel<false>, dim3((unsigned)blocks), dim3(KV_THREADS), 0, st, p));
    ctx->launches++;
    prof_close(ctx, st);
    return 0;
}

}  // namespace tb

using namespace tb;

extern "C" {

int tb_kv_append(const TbKvCache* cache, const int32_t* d_q_start, const int32_t* d_kv_len, const void* d_qkv, int qkv_bf16,
                 int64_t ld_qkv, int rows, int q_heads, const float* d_cos, const float* d_sin, int positions, int rot_dim,
                 int rope_form, void* d_Q, int64_t ld_q, void* stream) {
    TB_TRY(check_cache(cache, "tb_kv_append"));
    TB_CHECK(rows >= 0, "tb_kv_append: rows must not be negative");
    TB_CHECK(d_q_start && d_kv_len, "tb_kv_append: NULL batch array");
    TB_CHECK(rows == 0 || (d_qkv && d_Q), "tb_kv_append: NULL operand");
    TB_CHECK(q_heads > 0 && q_heads % cache->heads == 0, "tb_kv_append: %d query heads cannot share %d key heads", q_heads, cache->heads);
    const int per16 = qkv_bf16 ? 8 : 4;
    const long long width = ((long long)q_heads + 2LL * cache->heads) * cache->head_dim;
    TB_CHECK(ld_qkv >= width && ld_qkv % per16 == 0, "tb_kv_append: ld_qkv must be a multiple of %d and at least %lld (got %lld)", per16, width,
             (long long)ld_qkv);
    TB_CHECK(ld_q >= (long long)q_heads * cache->head_dim && ld_q % 8 == 0, "tb_kv_append: ld_q must be a multiple of 8 and at least %lld (got %lld)",
             (long long)q_heads * cache->head_dim, (long long)ld_q);
    TB_CHECK(((reinterpret_cast<uintptr_t>(d_qkv) | reinterpret_cast<uintptr_t>(d_Q)) & 15u) == 0, "tb_kv_append: rows must be 16-byte aligned");
    const RowSpan from = {d_qkv, rows, width * (qkv_bf16 ? 2 : 4), ld_qkv * (qkv_bf16 ? 2 : 4)};
    const RowSpan to = {d_Q, rows, (long long)q_heads * cache->head_dim * 2, ld_q * 2};
    TB_CHECK(!spans_overlap(from, to), "tb_kv_append: the queries must not lie over the rows they come from");
    TB_CHECK(rot_dim >= 0 && rot_dim <= cache->head_dim && rot_dim % 2 == 0, "tb_kv_append: rot_dim must be even and at most head_dim (got %d)", rot_dim);
    TB_CHECK(rope_form == TB_ROPE_PAIRS || rope_form == TB_ROPE_HALVES, "tb_kv_append: unknown rotation form %d", rope_form);
    TB_CHECK(rot_dim == 0 || (d_cos && d_sin && positions > 0), "tb_kv_append: a rotation needs both tables");
    TB_CHECK(!over_pools(cache, from) && !over_pools(cache, to), "tb_kv_append: the rows must not lie over the pools");
    if (rows == 0) return 0;
    DeviceCtx* ctx;
    TB_TRY(get_ctx(&ctx));
    return launch_kv_append(ctx, cache, d_q_start, d_kv_len, d_qkv, qkv_bf16 != 0, ld_qkv, rows, q_heads, d_cos, d_sin, positions, rot_dim,
                            rope_form, static_cast<bf16*>(d_Q), ld_q, static_cast<cudaStream_t>(stream));
}

int tb_kv_read(const TbKvCache* cache, const int32_t* d_start, const int32_t* d_first, int rows, void* d_K, void* d_V, int64_t ld_row,
               int64_t ld_head, void* stream) {
    TB_TRY(check_cache(cache, "tb_kv_read"));
    TB_CHECK(rows >= 0, "tb_kv_read: rows must not be negative");
    TB_CHECK(d_start, "tb_kv_read: NULL row starts");
    TB_CHECK(d_K || d_V, "tb_kv_read: both outputs are NULL");
    TB_CHECK(ld_row >= cache->head_dim && ld_row % 8 == 0 && ld_head >= cache->head_dim && ld_head % 8 == 0,
             "tb_kv_read: ld_row and ld_head must be multiples of 8 and at least head_dim (got %lld, %lld)", (long long)ld_row,
             (long long)ld_head);
    TB_CHECK(ld_row >= (cache->heads - 1) * ld_head + cache->head_dim || ld_head >= (rows - 1LL) * ld_row + cache->head_dim,
             "tb_kv_read: rows of ld_row %lld and heads of ld_head %lld lie over one another", (long long)ld_row, (long long)ld_head);
    TB_CHECK(((reinterpret_cast<uintptr_t>(d_K) | reinterpret_cast<uintptr_t>(d_V)) & 15u) == 0, "tb_kv_read: outputs must be 16-byte aligned");
    TB_CHECK(!d_K || !d_V || !heads_overlap(d_K, d_V, rows, ld_row * 2, cache->heads, ld_head * 2, cache->head_dim * 2LL),
             "tb_kv_read: the two outputs lie over one another");
    for (void* out : {d_K, d_V})
        for (int h = 0; h < cache->heads; ++h)
            TB_CHECK(!out || !over_pools(cache, {static_cast<const char*>(out) + h * ld_head * 2, rows, cache->head_dim * 2LL, ld_row * 2}),
                     "tb_kv_read: the outputs must not lie over the pools");
    if (rows == 0) return 0;
    DeviceCtx* ctx;
    TB_TRY(get_ctx(&ctx));
    return launch_kv_read(ctx, cache, d_start, d_first, rows, static_cast<bf16*>(d_K), static_cast<bf16*>(d_V), ld_row, ld_head,
                          static_cast<cudaStream_t>(stream));
}

}  // extern "C"
