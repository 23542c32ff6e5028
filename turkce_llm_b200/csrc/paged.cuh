// What the kernels over a paged cache share: the view of the pool, which sequence a row belongs to, and 8-bit codes.
#pragma once
#include "../../include/turkce_b200.h"
#include "common.h"
#include "overlap.h"

namespace tb {

struct PagedView {
    const int* table;
    int pages, page_shift, heads, hd, seqs, table_ld;
};

// host: the checks that every entry point makes of a cache
int check_cache(const TbKvCache* c, const char* who);
// host: whether rows lie over one of the cache's pools
inline bool over_pools(const TbKvCache* c, RowSpan rows) {
    const long long n = (long long)c->pages * c->heads * c->page_size, bytes = n * c->head_dim * (c->type == TB_KV_E4M3 ? 1 : 2);
    for (const void* pool : {c->K, c->V})
        if (spans_overlap({pool, 1, bytes, bytes}, rows)) return true;
    for (const void* scales : {c->k_scale, c->v_scale})
        if (spans_overlap({scales, 1, n * 4, n * 4}, rows)) return true;
    return false;
}
inline int page_shift_of(int page_size) {
    int s = 0;
    while ((1 << s) < page_size) ++s;
    return s;
}
inline PagedView paged_view(const TbKvCache* c) {
    PagedView v;
    v.table = c->table;
    v.pages = c->pages; v.page_shift = page_shift_of(c->page_size); v.heads = c->heads; v.hd = c->head_dim;
    v.seqs = c->seqs; v.table_ld = c->table_ld;
    return v;
}

#ifdef __CUDACC__

// The sequence whose rows hold `row`: the last one that starts at or before it; -1 where none does.  A warp looks at 32
// starts per step, so that up to 32 sequences take one read and up to 1024 take two.  All lanes of the warp call it with the
// same row.
__device__ __forceinline__ int sequence_of(const int* __restrict__ start, int seqs, int row) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = seqs;
    while (true) {
        const int step = (hi - lo + 31) >> 5;
        const int i = lo + lane * step;
        const unsigned below = __ballot_sync(0xffffffffu, i < hi && start[i] <= row);
        const int n = __popc(below);
        if (n == 0) return -1;
        lo += (n - 1) * step;
        hi = min(lo + step, hi);
        if (hi - lo <= 1) return lo;
    }
}

// x / scale on its way to the nearest 8-bit float (4 exponent bits, 3 of significand; halves to the even one): a float32 that lies on the
// same side of every middle of two codes as the true quotient.  By Markstein's correction of a quotient from its remainder, q is within a unit of its last place of that, its remainder tells on which
// side, and a number strictly between two floats becomes the one of them whose last bit is set, which no middle has.  Where q is a middle, its
// remainder has to be exact: with a scale of 2^-100 and more (E4M3_SMALL) it is a multiple of 2^-133, which float32 has.
constexpr float E4M3_SMALL = 0x1p-100f;
__device__ __forceinline__ float quotient_to_odd(float x, float scale, float inverse) {
    const float q0 = x * inverse;
    const float q = __fmaf_rn(__fmaf_rn(-q0, scale, x), inverse, q0);
    const float rest = __fmaf_rn(-q, scale, x);
    // (|q| too large: the remainder has the other sign.  Where q is 0 the remainder is x.)
    const uint32_t b = __float_as_uint(q), too_large = (__float_as_uint(rest) ^ __float_as_uint(x)) >> 31;
    const uint32_t odd = rest != 0.0f ? (b - too_large) | 1u : b;
    return __uint_as_float((odd & 0x7fffffffu) | (__float_as_uint(x) & 0x80000000u));      // (zeros keep their sign)
}
// the scale of an 8-bit row from its largest magnitude: the nearest float32 to big / 448, at least the smallest normal number, and about its
// inverse (quotient_to_odd corrects what that is off)
__device__ __forceinline__ float e4m3_scale(float big, float* inverse) {
    const float one = 1.0f / 448.0f;                             // rounded; a quotient by it corrected by its remainder is the nearest
    const float q = big * one;
    float scale = __fmaf_rn(__fmaf_rn(-q, 448.0f, big), one, q);
    if (scale < 1.17549435e-38f) scale = 1.17549435e-38f;        // (stays NaN where it is)
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(scale));
    *inverse = r;
    return scale;
}
__device__ __forceinline__ uint32_t e4m3_pair(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
// two codes -> two float32 / a pair of bf16 (exact)
__device__ __forceinline__ float2 e4m3_floats(uint32_t two) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)two));
    float2 f;
    asm("{\n\t.reg .f16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}" : "=f"(f.x), "=f"(f.y) : "r"(h));
    return f;
}
// 16 bytes on their way to shared memory, by this thread
__device__ __forceinline__ void copy_async16(void* to_shared, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to_shared)), "l"(from) : "memory");
}
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 bf16_floats(uint32_t two) {
    return make_float2(__uint_as_float(two << 16), __uint_as_float(two & 0xffff0000u));
}

#endif
}  // namespace tb
