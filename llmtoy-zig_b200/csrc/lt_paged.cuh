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

// Byte offset in a pool of position j of a sequence, on page `page` of it (which
// the caller has looked up and checked), for head h.
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

// N consecutive cache elements from element i, a multiple of N: 4 bytes or a multiple of 8.
template <int N>
LT_DEVINL void kv_ld_row(const uint8_t *p, uint32_t i, uint32_t f16, float (&v)[N]) {
    if (f16) {
        uint32_t w[N / 2];
        const uint8_t *at = p + 2 * i;
        if constexpr (N == 2) {
            w[0] = *reinterpret_cast<const uint32_t *>(at);
        } else {
#pragma unroll
            for (int e = 0; e < N / 2; e += 2) {
                const uint2 t = *reinterpret_cast<const uint2 *>(at + 4 * e);
                w[e] = t.x, w[e + 1] = t.y;
            }
        }
#pragma unroll
        for (int e = 0; e < N; e += 2) {
            const float2 t = __half22float2(*reinterpret_cast<const __half2 *>(&w[e / 2]));
            v[e] = t.x, v[e + 1] = t.y;
        }
    } else {
#pragma unroll
        for (int e = 0; e < N; e += 2) {
            const float2 t = *reinterpret_cast<const float2 *>(p + 4 * (i + e));
            v[e] = t.x, v[e + 1] = t.y;
        }
    }
}

// Row R of (sequence s, KV head kh) by itself, by one warp, key by key, masked keys never touched: for rows
// whose tile result is not finite, which a value outside the row's own keys may have caused.  Lane l holds
// elements l HD / 32 on; output dims [d0, d0 + nd).  A sum that is NaN makes every dim NaN: the rest of the
// keys is then left alone.  Several keys at a time, so that their loads and sums overlap.
template <int HD>
static __noinline__ __device__ void slow_row(const PagedAttnArgs &a, uint32_t s, uint32_t kh, uint32_t R, uint32_t d0,
                                             uint32_t nd) {
    constexpr int N = HD / 32, U = 4;
    const uint32_t e0 = (threadIdx.x & 31) * N;
    const uint32_t cap = (uint32_t)min((uint64_t)a.kv.max_pages * a.kv.page_size, (uint64_t)a.max_len);
    const uint32_t len = min(a.lens[s], cap), nq = a.cu[s + 1] - a.cu[s], q_row = a.cu[s] + R / a.group;
    const uint32_t head = kh * a.group + R % a.group;
    const float *q = a.q + (uint64_t)q_row * a.q_stride + (uint64_t)head * HD;
    const uint32_t *table = a.table + (uint64_t)s * a.kv.max_pages;
    const uint32_t *docs = a.docs ? a.docs + (uint64_t)s * a.doc_stride : nullptr;
    const int64_t i = (int64_t)len - nq + R / a.group;
    int64_t lo = 0, hi = len;
    if (a.window) lo = max((int64_t)0, i - (int64_t)a.window + 1);
    if (a.causal) hi = min(hi, max(i + 1, a.prefix ? (int64_t)a.prefix[s] : (int64_t)0));
    if (docs && i < 0) hi = 0;
    const float slope = a.slopes ? a.slopes[head] : 0.0f;
    const float f = a.softcap != 0.0f ? a.scale / a.softcap : a.scale * 1.4426950408889634f;
    float x[N], o[N], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < N; e++) {
        x[e] = q[e0 + e];
        o[e] = 0.0f;
    }
    for (int64_t j0 = lo; j0 < hi && l == l; j0 += U) {
        uint64_t off[U];
        bool seen[U];
        float dot[U];
#pragma unroll
        for (int u = 0; u < U; u++) {  // alike in all lanes
            const int64_t j = j0 + u;
            seen[u] = j < hi && (!docs || docs[j] == docs[i]);
            const uint32_t page = seen[u] ? table[page_of(a.kv, (uint32_t)j)] : 0;
            seen[u] = seen[u] && page < a.kv.n_pages;
            off[u] = seen[u] ? paged_offset(a.kv, page, (uint32_t)j, kh) : 0;
            dot[u] = 0.0f;
            if (seen[u]) {
                float k[N];
                kv_ld_row(a.kv.k + off[u], e0, a.kv.f16, k);
#pragma unroll
                for (int e = 0; e < N; e++) dot[u] = fmaf(x[e], k[e], dot[u]);
            }
        }
#pragma unroll
        for (int w = 16; w > 0; w >>= 1) {
#pragma unroll
            for (int u = 0; u < U; u++) dot[u] += __shfl_xor_sync(0xffffffffu, dot[u], w);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (!seen[u]) continue;
            float v[N];
            kv_ld_row(a.kv.v + off[u], e0, a.kv.f16, v);
            const float t = score_log2(dot[u], f, a.softcap, slope, fabsf((float)(i - j0 - u)));
            const float mn = t == t ? fmaxf(m, t) : t, base = mn == -INFINITY ? 0.0f : mn;
            const float al = ex2(m - base), p = ex2(t - base);
            m = mn;
            l = fmaf(l, al, p);
#pragma unroll
            for (int e = 0; e < N; e++) o[e] = fmaf(o[e], al, p * v[e]);
        }
    }
    if (e0 < d0 || e0 >= d0 + nd) return;
    float *out = a.out + (uint64_t)q_row * a.out_stride + (uint64_t)head * HD;
#pragma unroll
    for (int e = 0; e < N; e++) out[e0 + e] = l == 0.0f ? 0.0f : (l == l ? o[e] / l : l);
}

}  // namespace lt
