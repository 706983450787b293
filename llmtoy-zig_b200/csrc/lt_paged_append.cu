// lt_paged_append.cu — queries, keys and values of a batch of tokens on their
// way into a paged cache.
//
// Per head vector x of a token at position p (src/model/forward.zig:281-292,
// the per-head norms of src/model/gemma4/forward.zig:267-269, src/ops/rope.zig:
// 14-75, as lt_attn_prep does for one token):
//   x <- x / sqrt(mean(x^2) + eps) * w           (Q and K when weights are given)
//   (a, b) <- (a cos t - b sin t, a sin t + b cos t),  t = p / theta^(2i / hd)
//   V heads optionally x / sqrt(mean(x^2) + eps), no rotation.
// Q goes to its own buffer, K and V to the token's slot of the cache.
//
// Bound: memory (each value is read and written once).  A warp holds one head
// vector in registers, so the norm is one warp sum and a pair never leaves its
// lane; the angles of a token are the same for all its heads, so a CTA computes
// them once into shared memory (powf and sincosf cost more than the rotation).
#include "lt_paged.cuh"

namespace lt {

constexpr int kAppThreads = 256;

// rope.zig:21-24: 1 / theta^(2i / len), each step rounded in f32.
LT_DEVINL float append_freq(float theta, uint32_t i, uint32_t len) {
    const float e = __fdiv_rn((float)(2 * i), (float)len);
    return __fdiv_rn(1.0f, powf(theta, e));
}

template <int N>
LT_DEVINL void load_vec(const float *p, float (&v)[N]) {
    if constexpr (N == 4) {
        const float4 t = *reinterpret_cast<const float4 *>(p);
        v[0] = t.x, v[1] = t.y, v[2] = t.z, v[3] = t.w;
    } else if constexpr (N == 2) {
        const float2 t = *reinterpret_cast<const float2 *>(p);
        v[0] = t.x, v[1] = t.y;
    } else {
        v[0] = p[0];
    }
}
template <int N>
LT_DEVINL void store_vec(float *p, const float (&v)[N]) {
    if constexpr (N == 4)
        *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
    else if constexpr (N == 2)
        *reinterpret_cast<float2 *>(p) = make_float2(v[0], v[1]);
    else
        p[0] = v[0];
}
// f16 elements are rounded to nearest even, as the one-token caches store them.
template <int N>
LT_DEVINL void store_kv(uint8_t *p, uint32_t i, const float (&v)[N], uint32_t f16) {
    if (!f16) {
        store_vec<N>(reinterpret_cast<float *>(p) + i, v);
    } else if constexpr (N == 1) {
        reinterpret_cast<__half *>(p)[i] = __float2half_rn(v[0]);
    } else {
        __half2 h[N / 2];
#pragma unroll
        for (int e = 0; e < N / 2; e++) h[e] = __floats2half2_rn(v[2 * e], v[2 * e + 1]);
        if constexpr (N == 2)
            *reinterpret_cast<__half2 *>(reinterpret_cast<__half *>(p) + i) = h[0];
        else
            *reinterpret_cast<uint2 *>(reinterpret_cast<__half *>(p) + i) =
                make_uint2(*reinterpret_cast<uint32_t *>(&h[0]), *reinterpret_cast<uint32_t *>(&h[1]));
    }
}

// Lane l holds N = HD / 64 rotation pairs, as elements l N .. and HD / 2 + l N ..,
// so that a warp's accesses are contiguous: pair by pair across the two (NeoX), or
// each half of them consecutive pairs.  Consecutive pairs of head_dim 64 (N = 1)
// would straddle lanes: there elements 2 l and 2 l + 1.
// Grid (ntok, ceil(vectors / heads_per_cta)).
template <int HD>
__global__ void __launch_bounds__(kAppThreads) k_paged_append(PagedAppendArgs a) {
    constexpr int N = HD / 64, HALF = HD / 2;
    __shared__ float2 s_cs[HALF];
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t t = blockIdx.x;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t H = a.n_heads, KV = a.kv.n_kv, vecs = H + 2 * KV;
    const uint32_t first = blockIdx.y * a.heads_per_cta, last = min(vecs, first + a.heads_per_cta);
    const uint32_t pos = a.pos[t], seq = a.seq[t], at = a.slot ? a.slot[t] : pos;
    for (uint32_t i = threadIdx.x; i < HALF; i += kAppThreads) {
        float s, c;
        sincosf(__fmul_rn((float)pos, append_freq(a.theta, i, HD)), &s, &c);
        s_cs[i] = make_float2(c, s);
    }
    // the token's slot; a bad sequence, position or page id is reported and nothing is stored
    bool ok = seq < a.n_seq && at / a.kv.page_size < a.kv.max_pages;
    uint32_t page = 0;
    if (ok) {
        page = a.table[(uint64_t)seq * a.kv.max_pages + at / a.kv.page_size];
        ok = page < a.kv.n_pages;
    }
    if (!ok && threadIdx.x == 0) atomicExch(a.err, DEV_ERR_BAD_INDEX);
    const uint64_t base = ok ? paged_offset(a.kv, page, at, 0) : 0;
    __syncthreads();

    const bool neox = a.rope_neox;
    const bool split = neox || N > 1;
    const uint32_t e0 = split ? lane * N : 2 * lane, e1 = split ? HALF + lane * N : 2 * lane + 1;
    for (uint32_t h = first + warp; h < last; h += kAppThreads / 32) {
        const float *src = a.qkv + ((uint64_t)t * vecs + h) * HD;
        float x[N], y[N];
        load_vec<N>(src + e0, x);
        load_vec<N>(src + e1, y);
        const bool is_q = h < H, is_v = h >= H + KV;
        const float *w = is_q ? a.q_norm : is_v ? nullptr : a.k_norm;
        if (w || (is_v && a.v_norm)) {
            float ss = 0.0f;
#pragma unroll
            for (int e = 0; e < N; e++) ss = fmaf(x[e], x[e], fmaf(y[e], y[e], ss));
            ss = warp_sum(ss);
            const float inv = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(ss, (float)HD), a.eps)));
#pragma unroll
            for (int e = 0; e < N; e++) {
                x[e] *= inv;
                y[e] *= inv;
                if (w) {
                    x[e] *= w[e0 + e];
                    y[e] *= w[e1 + e];
                }
            }
        }
        if (!is_v) {
            if (neox) {
#pragma unroll
                for (int e = 0; e < N; e++) {
                    const float2 cs = s_cs[lane * N + e];
                    const float p = x[e], q = y[e];
                    x[e] = __fsub_rn(__fmul_rn(p, cs.x), __fmul_rn(q, cs.y));
                    y[e] = __fadd_rn(__fmul_rn(p, cs.y), __fmul_rn(q, cs.x));
                }
            } else if constexpr (N > 1) {  // x and y hold N / 2 consecutive pairs each
#pragma unroll
                for (int e = 0; e < N; e += 2) {
                    const float2 cx = s_cs[(lane * N + e) / 2], cy = s_cs[(HALF + lane * N + e) / 2];
                    const float p = x[e], q = x[e + 1], t = y[e], u = y[e + 1];
                    x[e] = __fsub_rn(__fmul_rn(p, cx.x), __fmul_rn(q, cx.y));
                    x[e + 1] = __fadd_rn(__fmul_rn(p, cx.y), __fmul_rn(q, cx.x));
                    y[e] = __fsub_rn(__fmul_rn(t, cy.x), __fmul_rn(u, cy.y));
                    y[e + 1] = __fadd_rn(__fmul_rn(t, cy.y), __fmul_rn(u, cy.x));
                }
            } else {
                const float2 cs = s_cs[lane];
                const float p = x[0], q = y[0];
                x[0] = __fsub_rn(__fmul_rn(p, cs.x), __fmul_rn(q, cs.y));
                y[0] = __fadd_rn(__fmul_rn(p, cs.y), __fmul_rn(q, cs.x));
            }
        }
        if (is_q) {
            float *dst = a.q + ((uint64_t)t * H + h) * HD;
            store_vec<N>(dst + e0, x);
            store_vec<N>(dst + e1, y);
        } else if (ok) {
            uint8_t *dst = (is_v ? a.kv.v : a.kv.k) + base + (uint64_t)(h - H - (is_v ? KV : 0)) * a.kv.head_stride;
            store_kv<N>(dst, e0, x, a.kv.f16);
            store_kv<N>(dst, e1, y, a.kv.f16);
        }
    }
}

cudaError_t launch_paged_append(const LaunchCfg &c, PagedAppendArgs a) {
    const uint32_t vecs = a.n_heads + 2 * a.kv.n_kv, warps = kAppThreads / 32;
    // Few tokens: one head vector per warp, so that the SMs share a token's
    // heads; many: one CTA per token, which computes the angles once.  Up to 148
    // tokens both take 5.5 us; 296 tokens, 16/8 heads of 256: 5.6 and 6.7 us, 592:
    // 9.7 and 9.9; 32/4 heads of 128: 8.5 and 7.5 us; 1184 tokens: 16.9 and 13.8 us,
    // 16.9 and 11.5.
    const bool few = a.ntok < 4u * (uint32_t)c.num_sms;
    a.heads_per_cta = few ? warps : vecs;
    a.err = c.dev_err;
    const dim3 grid(a.ntok, (vecs + a.heads_per_cta - 1) / a.heads_per_cta);
    switch (a.kv.hd) {
    case 64: return launch_k(c, "paged_append", k_paged_append<64>, grid, dim3(kAppThreads), 0, a);
    case 128: return launch_k(c, "paged_append", k_paged_append<128>, grid, dim3(kAppThreads), 0, a);
    case 256: return launch_k(c, "paged_append", k_paged_append<256>, grid, dim3(kAppThreads), 0, a);
    default: return cudaErrorInvalidValue;
    }
}

}  // namespace lt
