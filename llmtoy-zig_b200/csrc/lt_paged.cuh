// lt_paged.cuh — what the paged-cache kernels share: the cache descriptor and
// its addressing, the descriptors of an attention call, warp-level matrix
// products on two-term operands, and small numeric helpers.
//
// A paged cache is one pool of pages for K and one for V.  Page p holds
// page_size slots; position j of sequence s lives in slot j % page_size of page
// table[s][j / page_size].  Strides are in bytes here and 64-bit throughout:
// a pool of long contexts passes 4 GiB.
#pragma once

#include "lt_launch.cuh"

namespace lt {

// Page of a position and its slot there; a shift for the usual page sizes.
LT_DEVINL uint32_t page_of(const PagedKvDev &kv, uint32_t j) {
    return kv.page_shift != kNoShift ? j >> kv.page_shift : j / kv.page_size;
}
LT_DEVINL uint32_t slot_of(const PagedKvDev &kv, uint32_t j) {
    return kv.page_shift != kNoShift ? j & (kv.page_size - 1) : j % kv.page_size;
}

// Byte offset of position j of a sequence (its page-table row `row`) for head
// h, or ~0 when the page id lies outside the pool (the caller reports it).
LT_DEVINL uint64_t paged_offset(const PagedKvDev &kv, uint32_t page, uint32_t j, uint32_t h) {
    return (uint64_t)page * kv.page_stride + (uint64_t)slot_of(kv, j) * kv.slot_stride +
           (uint64_t)h * kv.head_stride;
}

LT_DEVINL void prefetch_l2(const void *p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

LT_DEVINL float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 16-byte asynchronous copy to shared memory; zero-fills when !take (the
// source is then not read).
LT_DEVINL void cp_async16(uint32_t dst, const void *src, bool take) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}
LT_DEVINL void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
LT_DEVINL void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Four 8x8 b16 matrices; lane l gives the address of row l % 8 of matrix l / 8.
LT_DEVINL void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
LT_DEVINL void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
LT_DEVINL float4 lds128(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}

// C[16x8] += A[16x16] B[16x8], f16 operands, f32 sums.
LT_DEVINL void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// C[16x8] += A[16x8] B[8x8], tf32 operands, f32 sums.
LT_DEVINL void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
LT_DEVINL uint32_t to_tf32(float x) {
    uint32_t y;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(y) : "f"(x));
    return y;
}
// x = hi + lo with hi and lo in tf32 (11 significant bits each).
LT_DEVINL void split_tf32(float x, uint32_t &hi, uint32_t &lo) {
    hi = to_tf32(x);
    lo = to_tf32(x - __uint_as_float(hi));
}
// Two values as packed f16 pairs: hi the nearest f16, lo the rest's nearest.
LT_DEVINL void split_f16x2(float x, float y, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&l);
}

// tanh in two ranges, parted at ln(3) / 2, where tanh is 1/2, as Cody and Waite do
// ("Software Manual for the Elementary Functions", 1980): above, 1 - 2 / (1 + e^(2x))
// takes at most 1/2 from 1 and loses no digits; below, x + x^3 P(x^2) with P the least
// squares fit of degree 4 on 400 Chebyshev points in x^2, weighted for the relative
// error of tanh (6.1e-8 in f32).  Capped scores seldom leave the lower range.
constexpr float kTanhSmall = 0.549306f;
LT_DEVINL float tanh_small(float x) {
    const float y = x * x;
    float r = -0.006269626785069704f;
    r = fmaf(r, y, 0.021067650988698006f);
    r = fmaf(r, y, -0.05385109782218933f);
    r = fmaf(r, y, 0.1333257108926773f);
    r = fmaf(r, y, -0.33333316445350647f);
    return fmaf(r * y, x, x);
}

LT_DEVINL float2 fmul2(float2 a, float2 b) {
    f2u A, B, D;
    A.f = a;
    B.f = b;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(D.u) : "l"(A.u), "l"(B.u));
    return D.f;
}
// tanh_small of two values.
LT_DEVINL float2 tanh_small2(float2 x) {
    const float2 y = fmul2(x, x);
    auto both = [](float c) { return make_float2(c, c); };
    float2 r = both(-0.006269626785069704f);
    r = ffma2(r, y, both(0.021067650988698006f));
    r = ffma2(r, y, both(-0.05385109782218933f));
    r = ffma2(r, y, both(0.1333257108926773f));
    r = ffma2(r, y, both(-0.33333316445350647f));
    return ffma2(fmul2(r, y), x, x);
}

// tanh over the whole range, absolute error about 1.5e-7 above kTanhSmall.  No branch:
// it stands in unrolled loops.  The quotient's limit, 0, is put in where 1 + e^(2|x|)
// leaves __fdividef's range.
LT_DEVINL float tanh_any(float x) {
    const float a = fabsf(x), d = 1.0f + ex2(a * 2.885390081777927f);
    const float t = copysignf(1.0f - (d < 1e30f ? __fdividef(2.0f, d) : 0.0f), x);
    return a <= kTanhSmall ? tanh_small(x) : (x != x ? x : t);
}

// Score of one (query, key) pair in units of log2: the scaled product, capped
// by cap * tanh(s / cap), minus slope * |distance|.  f is the row's factor on
// the raw product: scale * log2(e) without a cap, scale / cap with one.
LT_DEVINL float score_log2(float dot, float f, float cap, float slope, float dist) {
    constexpr float kLog2e = 1.4426950408889634f;
    float s = dot * f;
    if (cap != 0.0f) s = tanh_any(s) * (cap * kLog2e);
    return fmaf(-slope * kLog2e, dist, s);
}

// Row R of (sequence s, KV head kh) by itself, key by key, masked keys never
// touched: for rows whose tile result is not finite, which a value outside the
// row's own keys may have caused.  Output dims [d0, d0 + nd), nd a multiple of 16.
static __noinline__ __device__ void slow_row(const PagedAttnArgs &a, uint32_t s, uint32_t kh, uint32_t R, uint32_t d0,
                                         uint32_t nd) {
    const uint32_t hd = a.kv.hd, cap = (uint32_t)min((uint64_t)a.kv.max_pages * a.kv.page_size, (uint64_t)a.max_len);
    const uint32_t len = min(a.lens[s], cap), nq = a.cu[s + 1] - a.cu[s], q_row = a.cu[s] + R / a.group;
    const uint32_t head = kh * a.group + R % a.group;
    const float *q = a.q + (uint64_t)q_row * a.q_stride + (uint64_t)head * hd;
    float *out = a.out + (uint64_t)q_row * a.out_stride + (uint64_t)head * hd;
    const uint32_t *table = a.table + (uint64_t)s * a.kv.max_pages;
    const uint32_t *docs = a.docs ? a.docs + (uint64_t)s * a.doc_stride : nullptr;
    const int64_t i = (int64_t)len - nq + R / a.group;
    int64_t lo = 0, hi = len;
    if (a.window) lo = max((int64_t)0, i - (int64_t)a.window + 1);
    if (a.causal) hi = min(hi, max(i + 1, a.prefix ? (int64_t)a.prefix[s] : (int64_t)0));
    if (docs && i < 0) hi = 0;
    const float slope = a.slopes ? a.slopes[head] : 0.0f;
    const float f = a.softcap != 0.0f ? a.scale / a.softcap : a.scale * 1.4426950408889634f;
    float m = -INFINITY;
    for (uint32_t d = d0; d < d0 + nd; d += 16) {
        float o[16], l = 0.0f;
        for (int e = 0; e < 16; e++) o[e] = 0.0f;
        for (int pass = d == d0 ? 0 : 1; pass < 2; pass++) {
            for (int64_t j = lo; j < hi; j++) {
                if (docs && docs[j] != docs[i]) continue;
                const uint32_t page = table[j / a.kv.page_size];
                if (page >= a.kv.n_pages) continue;
                const uint64_t off = paged_offset(a.kv, page, (uint32_t)j, kh);
                float dot = 0.0f;
                for (uint32_t e = 0; e < hd; e++) dot = fmaf(q[e], kv_ld(a.kv.k + off, e, a.kv.f16), dot);
                const float t = score_log2(dot, f, a.softcap, slope, fabsf((float)(i - j)));
                if (pass == 0) {
                    m = t != t || m != m ? NAN : fmaxf(m, t);
                } else {
                    const float p = ex2(t - m);
                    l += p;
                    for (int e = 0; e < 16; e++) o[e] = fmaf(p, kv_ld(a.kv.v + off, d + e, a.kv.f16), o[e]);
                }
            }
        }
        for (int e = 0; e < 16; e++) out[d + e] = l == 0.0f ? 0.0f : o[e] / l;
    }
}

}  // namespace lt
