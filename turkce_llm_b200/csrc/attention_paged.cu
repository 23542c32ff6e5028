// Causal attention of new tokens over a paged cache of keys and values (bf16, or 8-bit codes with a scale per row).
//
// For query row (token i, head h) of a sequence, with positions up to its own visible:
//   o = sum_t p_t v_t / sum_t p_t,   p_t = 2^(s_t - m),   s_t = scale log2(e) <q, k_t>,   m = max s_t,
// in one pass over the keys: a running maximum m, the sum l and the accumulator rescaled where m grows.  Pieces of the cache
// are taken by different CTAs where there are few sequences; each leaves (o, m, l) and paged_combine_kernel adds them in the order
// of the pieces.
//
// An 8-bit key's scale multiplies its score, an 8-bit value's scale its probability before that is rounded to bf16, so the codes
// enter the tensor cores as they are (exact in bf16) and nothing is rounded more often than with a bf16 cache.
#include "paged.cuh"
#include "paged_plan.h"
#include "ptx.cuh"

#include <algorithm>
#include <type_traits>

namespace tb {

namespace {

struct PagedAttParams {
    PagedView v;
    const int *q_start, *kv_len;
    const bf16* Q; long long ld_q;
    const float *ks, *vs;
    bf16* att; long long ld_att;
    float* lse;                      // [rows, H] or NULL
    float* part_o; float2* part_ml;  // [splits][rows * H][hd], [splits][rows * H]
    int rows, H, group, max_q, max_kv, split_keys;
    float scale_log2;
    int* err;
};

// the sequence's first row, number of new rows and number of keys; false where they are outside what the call allows
__device__ __forceinline__ bool batch_of(const PagedAttParams& p, int s, int& q0, int& n, int& kv) {
    q0 = p.q_start[s];
    const int q1 = p.q_start[s + 1];
    kv = p.kv_len[s];
    n = q1 - q0;
    return q0 >= 0 && q1 >= q0 && q1 <= p.rows && n <= p.max_q && kv >= 0 && kv <= p.max_kv &&
           kv <= (long long)p.v.table_ld << p.v.page_shift;
}

// ------------------------------------------------------------------------------- few rows: mma fragments
// CTA = 16 query rows of one key head and one piece of the cache; four warps with 16 keys of every stage of 64 each, a fifth one
// that fills the ring.  What counts here is bytes: the rows are padded to 16 and the tensor work is still small beside the keys
// and values that come in.  A warp keeps maximum, sum and accumulator of its own keys; they are put together at the end.
//
// Fragments without a shuffle: the contraction over the head dimension may take the elements in any order, so lane (r, c) of a
// key's fragment (r = lane / 4, c = lane % 4) holds elements 16 c .. 16 c + 15 of key r, two 16-byte reads, and the queries lie
// the same way.  Of a value's rows 2c, 2c + 1, 2c + 8, 2c + 9 it takes elements 8 r .. 8 r + 7, and pairs of two keys are made
// with byte permutes; accumulator tile i then holds elements 8 (2c) + i and 8 (2c + 1) + i of rows r and r + 8.
constexpr int PA_WARPS = 4;
constexpr int PA_THREADS = (PA_WARPS + 1) * 32;
constexpr int PA_STAGES = 4;

template <int NH, bool E4M3>
struct RowsShape {
    static constexpr int ROW_BYTES = E4M3 ? 64 * NH : 128;                   // of one 64-element (8 bits: all) column block
    static constexpr int BLOCK = PA_KEYS * ROW_BYTES;                        // one column block of 64 keys
    static constexpr int TILE = E4M3 ? BLOCK : NH * BLOCK;
    static constexpr int STAGE = 2 * TILE + (E4M3 ? 2 * PA_KEYS * 4 : 0);
    static constexpr int SMEM = 1024 + PA_STAGES * STAGE + 256;
};

__device__ __forceinline__ void mma_bf16_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// two 8-bit codes -> a pair of bf16
__device__ __forceinline__ uint32_t e4m3_bf16(uint32_t two) {
    const float2 f = e4m3_floats(two);
    return bf16_pair(f.x, f.y);
}

template <int NH, bool E4M3>
__global__ void __launch_bounds__(PA_THREADS)
paged_rows_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const PagedAttParams p) {
    typedef RowsShape<NH, E4M3> Sh;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + PA_STAGES * Sh::STAGE);
    uint64_t* empty = full + PA_STAGES;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(empty + PA_STAGES);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < PA_STAGES; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], PA_WARPS); }
        *abort_flag = 0;
        fence_mbar_init();
    }
    __syncthreads();
    pdl_wait();
    const int split = blockIdx.x, s = blockIdx.z;
    const int head = blockIdx.y % p.v.heads, tile = blockIdx.y / p.v.heads;
    int q0, n, kv;
    if (!batch_of(p, s, q0, n, kv)) {
        if (threadIdx.x == 0) atomicExch(p.err, 76);
        return;
    }
    const int row0 = tile * PA_ROWS, nrows = min(PA_ROWS, n * p.group - row0);
    if (nrows <= 0) return;
    const int first_pos = kv - n + row0 / p.group, last_pos = kv - n + (row0 + nrows - 1) / p.group;
    const int kv_end = last_pos + 1;                              // (no more than kv; negative for rows without a key)
    const bool whole = kv <= p.split_keys;                        // one piece: the result is final
    const int k_begin = split * p.split_keys, k_end = min(k_begin + p.split_keys, kv_end);
    if (k_begin > 0 && k_begin >= kv_end) return;                 // (piece 0 of a row without keys writes its zeros)
    const int stages = k_end > k_begin ? (k_end - k_begin + PA_KEYS - 1) / PA_KEYS : 0;

    if (warp == PA_WARPS) {
        // ---- producer: a lane per piece of a page; the table is read 32 entries at a time, one round ahead
        const int piece_shift = min(p.v.page_shift, 6), pieces = PA_KEYS >> piece_shift;      // keys per copy, copies per stage
        const int piece_keys = 1 << piece_shift, per_page_shift = p.v.page_shift - piece_shift;
        const int* table = p.v.table + (long long)s * p.v.table_ld;
        const int first_piece = k_begin >> piece_shift, last_piece = (k_end + piece_keys - 1) >> piece_shift;
        auto page_at = [&](int piece) -> int {
            if (piece >= last_piece) return 0;
            const int pg = table[piece >> per_page_shift];
            if ((unsigned)pg < (unsigned)p.v.pages) return pg;
            atomicExch(p.err, 75);
            return 0;
        };
        int held = first_piece, pages_now = page_at(first_piece + lane), pages_next = page_at(first_piece + 32 + lane);
        bool ok = true;
        for (int i = 0; i < stages && ok; ++i) {
            const int st = i % PA_STAGES;
            const int at = first_piece + i * pieces;
            if (at >= held + 32) { held += 32; pages_now = pages_next; pages_next = page_at(held + 32 + lane); }
            const int piece = at + lane;
            const int pg = __shfl_sync(0xffffffffu, pages_now, (at - held + lane) & 31);
            const int count = min(pieces, last_piece - at);       // copies of this stage
            if (i >= PA_STAGES) ok = mbar_wait(&empty[st], (uint32_t)((i / PA_STAGES) & 1) ^ 1u, abort_flag);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            uint8_t* sK = smem + st * Sh::STAGE;
            uint8_t* sV = sK + Sh::TILE;
            if (lane == 0) mbar_expect_tx(&full[st], (uint32_t)(count * piece_keys * (2 * Sh::TILE / PA_KEYS + (E4M3 ? 8 : 0))));
            __syncwarp();
            if (lane < count) {
                const int block = pg * p.v.heads + head, r0 = (piece & ((1 << per_page_shift) - 1)) << piece_shift;
                const int o = lane << piece_shift;
#pragma unroll
                for (int b = 0; b < (E4M3 ? 1 : NH); ++b) {
                    tma_load_3d(sK + b * Sh::BLOCK + o * Sh::ROW_BYTES, &tmK, &full[st], b * 64, r0, block);
                    tma_load_3d(sV + b * Sh::BLOCK + o * Sh::ROW_BYTES, &tmV, &full[st], b * 64, r0, block);
                }
                if (E4M3) {
                    float* sc = reinterpret_cast<float*>(sK + 2 * Sh::TILE);
                    const long long row = ((long long)block << p.v.page_shift) + r0;
                    bulk_load(sc + o, p.ks + row, (uint32_t)piece_keys * 4u, &full[st]);
                    bulk_load(sc + PA_KEYS + o, p.vs + row, (uint32_t)piece_keys * 4u, &full[st]);
                }
            }
            __syncwarp();
        }
        pdl_launch_dependents_now();
        if (!ok && lane == 0) { *abort_flag = 1; atomicExch(p.err, 73); }
        // (the CTA stays until what was asked for has arrived: the consumers wait for every stage)
        return;
    }

    const int r = lane >> 2, c = lane & 3;
    // query fragments: elements 16 c .. of rows r and r + 8, head-dimension block by block
    uint32_t qf[NH][4][4];
    int pos[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int rr = r + 8 * i;
        const int tok = (row0 + min(rr, nrows - 1)) / p.group, g = (row0 + min(rr, nrows - 1)) % p.group;
        pos[i] = kv - n + tok;
        const bf16* q = p.Q + (long long)(q0 + tok) * p.ld_q + (long long)(head * p.group + g) * p.v.hd;
#pragma unroll
        for (int b = 0; b < NH; ++b)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int e = 64 * b + 16 * c + 8 * h;
                uint4 w = make_uint4(0u, 0u, 0u, 0u);
                if (e < p.v.hd && rr < nrows) w = *reinterpret_cast<const uint4*>(q + e);
                qf[b][2 * h][i] = w.x; qf[b][2 * h][2 + i] = w.y; qf[b][2 * h + 1][i] = w.z; qf[b][2 * h + 1][2 + i] = w.w;
            }
    }
    float o[8 * NH][4];
#pragma unroll
    for (int i = 0; i < 8 * NH; ++i) { o[i][0] = 0.f; o[i][1] = 0.f; o[i][2] = 0.f; o[i][3] = 0.f; }
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    bool ok = true;
    for (int i = 0; i < stages; ++i) {
        const int st = i % PA_STAGES;
        if (!mbar_wait(&full[st], (uint32_t)((i / PA_STAGES) & 1), abort_flag)) { ok = false; break; }
        const uint8_t* sK = smem + st * Sh::STAGE;
        const uint8_t* sV = sK + Sh::TILE;
        const float* sc = reinterpret_cast<const float*>(sK + 2 * Sh::TILE);
        const int kk = 16 * warp, k0 = k_begin + i * PA_KEYS + kk;         // this warp's 16 keys
        if (k0 < k_end) {
            // ---- scores of two tiles of 8 keys
            float z[2][4];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                z[t][0] = z[t][1] = z[t][2] = z[t][3] = 0.f;
                const int key = kk + 8 * t + r;
#pragma unroll
                for (int b = 0; b < NH; ++b) {
                    uint32_t w[8];
                    if (E4M3) {
                        const uint4 x = *reinterpret_cast<const uint4*>(sK + key * Sh::ROW_BYTES + 64 * b + 16 * c);
                        const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) { w[2 * e] = e4m3_bf16(u[e] & 0xffffu); w[2 * e + 1] = e4m3_bf16(u[e] >> 16); }
                    } else {
                        // (128-byte swizzle: the 16-byte pieces of a row lie at piece ^ (row & 7))
                        const uint8_t* row = sK + b * Sh::BLOCK + key * 128;
                        const uint4 x = *reinterpret_cast<const uint4*>(row + (((2 * c) ^ (key & 7)) << 4));
                        const uint4 y = *reinterpret_cast<const uint4*>(row + (((2 * c + 1) ^ (key & 7)) << 4));
                        w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w; w[4] = y.x; w[5] = y.y; w[6] = y.z; w[7] = y.w;
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) mma_bf16_16816(z[t], qf[b][e], w[2 * e], w[2 * e + 1]);
                }
                float f0 = p.scale_log2, f1 = p.scale_log2;
                if (E4M3) {
                    const float2 f = *reinterpret_cast<const float2*>(sc + kk + 8 * t + 2 * c);
                    f0 *= f.x; f1 *= f.y;
                }
                z[t][0] *= f0; z[t][1] *= f1; z[t][2] *= f0; z[t][3] *= f1;
            }
            const bool edge = k0 + 15 > first_pos;                         // some row does not see all of these keys
            if (edge) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (k0 + 8 * t + 2 * c + (e & 1) > pos[e >> 1]) z[t][e] = -INFINITY;
            }
            // ---- running maximum and sum
            bool moved = false;
            float alpha[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float mx = fmaxf(fmaxf(z[0][2 * h], z[0][2 * h + 1]), fmaxf(z[1][2 * h], z[1][2 * h + 1]));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const float mn = fmaxf(m[h], mx);
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
            uint32_t pa[4];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                float f0 = 1.f, f1 = 1.f;
                if (E4M3) {
                    const float2 f = *reinterpret_cast<const float2*>(sc + PA_KEYS + kk + 8 * t + 2 * c);
                    f0 = f.x; f1 = f.y;
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    // (a row that has seen no key yet: its maximum is -infinity, and so are its scores)
                    const float base = m[h] == -INFINITY ? 0.f : m[h];
                    float p0 = ex2_approx(z[t][2 * h] - base), p1 = ex2_approx(z[t][2 * h + 1] - base);
                    l[h] += p0 + p1;
                    if (E4M3) {
                        // (a masked key's scale may be anything)
                        p0 = z[t][2 * h] == -INFINITY ? 0.f : p0 * f0;
                        p1 = z[t][2 * h + 1] == -INFINITY ? 0.f : p1 * f1;
                    }
                    pa[2 * t + h] = bf16_pair(p0, p1);
                }
            }
            // ---- values
            // keys behind position `last` count as zeros; at an edge, only the rows of that position take the product
            auto values = [&](const uint32_t (&a)[4], int last, auto at_edge) {
#pragma unroll
                for (int b = 0; b < NH; ++b) {
                    uint32_t w[4][4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int key = kk + 2 * c + (j & 1) + 8 * (j >> 1);
                        const bool seen = k0 - kk + key <= last;
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
                            b0 = e4m3_bf16(__byte_perm(w[0][e >> 2], w[1][e >> 2], sel) & 0xffffu);
                            b1 = e4m3_bf16(__byte_perm(w[2][e >> 2], w[3][e >> 2], sel) & 0xffffu);
                        } else {
                            const uint32_t sel = e & 1 ? 0x7632u : 0x5410u;
                            b0 = __byte_perm(w[0][e >> 1], w[1][e >> 1], sel);
                            b1 = __byte_perm(w[2][e >> 1], w[3][e >> 1], sel);
                        }
                        if (!at_edge.value) {
                            mma_bf16_16816(o[8 * b + e], a, b0, b1);
                        } else {
                            float d[4] = {0.f, 0.f, 0.f, 0.f};
                            mma_bf16_16816(d, a, b0, b1);
                            if (pos[0] == last) { o[8 * b + e][0] += d[0]; o[8 * b + e][1] += d[1]; }
                            if (pos[1] == last) { o[8 * b + e][2] += d[2]; o[8 * b + e][3] += d[3]; }
                        }
                    }
                }
            };
            if (!edge) values(pa, 0x7fffffff, std::false_type());
            else       // token by token: what a token does not see must not reach it, not even as 0 * infinity
                for (int last = first_pos; last <= last_pos; ++last) values(pa, last, std::true_type());
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[st]);
    }
    if (!ok) {
        // (what was asked for may still arrive: the block keeps its memory a little longer)
        if (lane == 0) { *abort_flag = 1; atomicExch(p.err, 74); }
        for (int i = 0; i < 64; ++i) __nanosleep(1000);
    }

    // ---- the four warps' results: [warp][16 rows][64 NH + 4] floats over the ring, maxima and sums behind
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    }
    asm volatile("bar.sync 1, 128;" ::: "memory");                         // every stage has been read
    constexpr int LD = 64 * NH + 4;
    float* so = reinterpret_cast<float*>(smem);
    float2* sml = reinterpret_cast<float2*>(so + PA_WARPS * PA_ROWS * LD);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float* dst = so + (warp * PA_ROWS + r + 8 * h) * LD + 16 * c;
#pragma unroll
        for (int b = 0; b < NH; ++b)
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                *reinterpret_cast<float4*>(dst + 64 * b + e) =
                    make_float4(o[8 * b + e][2 * h], o[8 * b + e + 1][2 * h], o[8 * b + e + 2][2 * h], o[8 * b + e + 3][2 * h]);
                *reinterpret_cast<float4*>(dst + 64 * b + 8 + e) =
                    make_float4(o[8 * b + e][2 * h + 1], o[8 * b + e + 1][2 * h + 1], o[8 * b + e + 2][2 * h + 1], o[8 * b + e + 3][2 * h + 1]);
            }
        if (c == 0) sml[warp * PA_ROWS + r + 8 * h] = make_float2(m[h], l[h]);
    }
    asm volatile("bar.sync 1, 128;" ::: "memory");
    const int chunks = p.v.hd >> 3;                                        // eight elements per thread
    for (int x = threadIdx.x; x < nrows * chunks; x += PA_WARPS * 32) {
        const int rr = x / chunks, e = (x - rr * chunks) * 8;
        float M = -INFINITY, L = 0.f, f[PA_WARPS];
#pragma unroll
        for (int w = 0; w < PA_WARPS; ++w) M = fmaxf(M, sml[w * PA_ROWS + rr].x);
        float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < PA_WARPS; ++w) {
            const float2 ml = sml[w * PA_ROWS + rr];
            f[w] = ml.y == 0.f ? 0.f : ex2_approx(ml.x - M);              // (a sum of 0: no key of this warp's was visible)
            L += ml.y * f[w];
            if (f[w] != 0.f) {
                const float4* src = reinterpret_cast<const float4*>(so + (w * PA_ROWS + rr) * LD + e);
                const float4 a = src[0], b = src[1];
                acc[0] += a.x * f[w]; acc[1] += a.y * f[w]; acc[2] += a.z * f[w]; acc[3] += a.w * f[w];
                acc[4] += b.x * f[w]; acc[5] += b.y * f[w]; acc[6] += b.z * f[w]; acc[7] += b.w * f[w];
            }
        }
        const int tok = (row0 + rr) / p.group, hq = head * p.group + (row0 + rr) % p.group;
        const long long at = (long long)(q0 + tok) * p.H + hq;
        if (whole) {
            const bool none = kv - n + tok < 0;                            // a row without a key
            const float inv = none ? 0.f : 1.0f / L;
            *reinterpret_cast<uint4*>(p.att + (long long)(q0 + tok) * p.ld_att + (long long)hq * p.v.hd + e) =
                make_uint4(bf16_pair(acc[0] * inv, acc[1] * inv), bf16_pair(acc[2] * inv, acc[3] * inv),
                           bf16_pair(acc[4] * inv, acc[5] * inv), bf16_pair(acc[6] * inv, acc[7] * inv));
            if (p.lse && e == 0) p.lse[at] = none ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
        } else {
            const long long slot = (long long)split * p.rows * p.H + at;
            float4* dst = reinterpret_cast<float4*>(p.part_o + slot * p.v.hd + e);
            dst[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
            dst[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
            if (e == 0) p.part_ml[slot] = make_float2(M, L);
        }
    }
}

// ------------------------------------------------------------------------------- pieces of a row, in their order
// A warp per (row, head); rows of sequences that took one piece are final already.
constexpr int PC_WARPS = 8;
__global__ void __launch_bounds__(PC_WARPS * 32)
paged_combine_kernel(const PagedAttParams p) {
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const long long at = (long long)blockIdx.x * PC_WARPS + (threadIdx.x >> 5);
    if (at >= (long long)p.rows * p.H) return;
    const int row = (int)(at / p.H), hq = (int)(at - (long long)row * p.H);
    const int s = sequence_of(p.q_start, p.v.seqs, row);
    if (s < 0) return;
    int q0, n, kv;
    if (!batch_of(p, s, q0, n, kv) || row >= q0 + n || kv <= p.split_keys) return;
    const int pos = kv - n + row - q0;
    const int pieces = pos < 0 ? 0 : pos / p.split_keys + 1;
    const long long step = (long long)p.rows * p.H;
    float M = -INFINITY, L = 0.f;
    for (int i = 0; i < pieces; ++i) M = fmaxf(M, p.part_ml[i * step + at].x);
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    const int e = lane * 4;
    for (int i = 0; i < pieces; ++i) {
        const float2 ml = p.part_ml[i * step + at];
        if (ml.y == 0.f) continue;
        const float f = ex2_approx(ml.x - M);
        L += ml.y * f;
        if (e < p.v.hd) {
            const float4 a = *reinterpret_cast<const float4*>(p.part_o + (i * step + at) * p.v.hd + e);
            acc[0] += a.x * f; acc[1] += a.y * f; acc[2] += a.z * f; acc[3] += a.w * f;
        }
    }
    const float inv = pos < 0 ? 0.f : 1.0f / L;
    if (e < p.v.hd)
        *reinterpret_cast<uint2*>(p.att + (long long)row * p.ld_att + (long long)hq * p.v.hd + e) =
            make_uint2(bf16_pair(acc[0] * inv, acc[1] * inv), bf16_pair(acc[2] * inv, acc[3] * inv));
    if (p.lse && lane == 0) p.lse[at] = pos < 0 ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
}

template <int NH, bool E4M3>
int launch_rows(DeviceCtx* ctx, const TbKvCache* c, const PagedAttParams& p, const PagedPlan& pl, cudaStream_t st) {
    typedef RowsShape<NH, E4M3> Sh;
    CUtensorMap tmK, tmV;
    const int box_rows = std::min(c->page_size, PA_KEYS);
    TB_TRY(make_cache_map(&tmK, c->K, E4M3 ? 1 : 2, c->head_dim, c->page_size, (long long)c->pages * c->heads, 64 * (E4M3 ? NH : 1), box_rows));
    TB_TRY(make_cache_map(&tmV, c->V, E4M3 ? 1 : 2, c->head_dim, c->page_size, (long long)c->pages * c->heads, 64 * (E4M3 ? NH : 1), box_rows));
    static bool attr_set[64] = {false};
    if (!attr_set[ctx->device & 63]) {
        TB_CUDA(cudaFuncSetAttribute(paged_rows_kernel<NH, E4M3>, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::SMEM));
        attr_set[ctx->device & 63] = true;
    }
    prof_mark(ctx, "paged_rows", 4.0 * p.rows * p.H * (double)p.max_kv * c->head_dim, 0.0, st);
    TB_CUDA(launch_kernel(paged_rows_kernel<NH, E4M3>, dim3(pl.splits, c->heads * pl.tiles, c->seqs), dim3(PA_THREADS), Sh::SMEM, st, tmK, tmV, p));
    ctx->launches++;
    prof_close(ctx, st);
    return 0;
}

}  // namespace

int launch_attention_paged(DeviceCtx* ctx, const TbKvCache* c, const int* q_start, const int* kv_len, const bf16* Q, long long ld_q, int rows,
                           int H, int max_q, int max_kv, float scale, bf16* att, long long ld_att, float* lse, void* ws, int64_t ws_bytes,
                           cudaStream_t st) {
    const int group = H / c->heads;
    const PagedPlan pl = paged_plan(c->seqs, c->heads, group, c->head_dim, rows, max_q, max_kv, ctx->sm_count);
    TB_CHECK(pl.workspace == 0 || (ws != nullptr && ws_bytes >= pl.workspace), "tb_attention_paged: the workspace has %lld bytes, %lld are needed",
             (long long)(ws ? ws_bytes : 0), (long long)pl.workspace);
    TB_CHECK((long long)c->heads * pl.tiles <= 65535, "tb_attention_paged: max_q %d with %d heads is too much for one launch", max_q, H);
    PagedAttParams p;
    p.v = paged_view(c);
    p.q_start = q_start; p.kv_len = kv_len; p.Q = Q; p.ld_q = ld_q; p.ks = c->k_scale; p.vs = c->v_scale;
    p.att = att; p.ld_att = ld_att; p.lse = lse;
    p.part_o = static_cast<float*>(ws);
    p.part_ml = reinterpret_cast<float2*>(p.part_o + (long long)pl.splits * rows * H * c->head_dim);
    p.rows = rows; p.H = H; p.group = group; p.max_q = max_q; p.max_kv = max_kv; p.split_keys = pl.split_keys;
    p.scale_log2 = scale * 1.4426950408889634f; p.err = ctx->d_err;
    const bool wide = c->head_dim > 64;
    if (c->type == TB_KV_E4M3) TB_TRY(wide ? (launch_rows<2, true>(ctx, c, p, pl, st)) : (launch_rows<1, true>(ctx, c, p, pl, st)));
    else TB_TRY(wide ? (launch_rows<2, false>(ctx, c, p, pl, st)) : (launch_rows<1, false>(ctx, c, p, pl, st)));
    if (pl.splits > 1) {
        const long long blocks = ((long long)rows * H + PC_WARPS - 1) / PC_WARPS;
        TB_CHECK(blocks < (1LL << 31), "tb_attention_paged: too many rows");
        prof_mark(ctx, "paged_combine", 0.0, (double)pl.workspace, st);
        TB_CUDA(launch_kernel(paged_combine_kernel, dim3((unsigned)blocks), dim3(PC_WARPS * 32), 0, st, p));
        ctx->launches++;
        prof_close(ctx, st);
    }
    return 0;
}

}  // namespace tb

using namespace tb;

static int check_attention(const TbKvCache* cache, int rows, int q_heads, int max_q, int max_kv) {
    TB_TRY(check_cache(cache, "tb_attention_paged"));
    TB_CHECK(rows >= 0 && max_q >= 0 && max_kv >= 0, "tb_attention_paged: rows, max_q and max_kv must not be negative");
    TB_CHECK(q_heads > 0 && q_heads % cache->heads == 0, "tb_attention_paged: %d query heads cannot share %d key heads", q_heads, cache->heads);
    TB_CHECK((long long)rows * q_heads < (1LL << 31), "tb_attention_paged: rows * q_heads must be below 2^31");
    return 0;
}

extern "C" {

int64_t tb_attention_paged_workspace(const TbKvCache* cache, int rows, int q_heads, int max_q, int max_kv) {
    DeviceCtx* ctx;
    if (check_attention(cache, rows, q_heads, max_q, max_kv) != 0 || get_ctx(&ctx) != 0) return -1;
    return paged_plan(cache->seqs, cache->heads, q_heads / cache->heads, cache->head_dim, rows, std::min(max_q, rows), max_kv, ctx->sm_count).workspace;
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
    TB_CHECK(d_Q != d_att, "tb_attention_paged: the result must not lie over the queries");
    DeviceCtx* ctx;
    TB_TRY(get_ctx(&ctx));
    return launch_attention_paged(ctx, cache, d_q_start, d_kv_len, static_cast<const bf16*>(d_Q), ld_q, rows, q_heads, std::min(max_q, rows),
                                  max_kv, scale, static_cast<bf16*>(d_att), ld_att, d_lse, d_workspace, workspace_bytes,
                                  static_cast<cudaStream_t>(stream));
}

}  // extern "C"
