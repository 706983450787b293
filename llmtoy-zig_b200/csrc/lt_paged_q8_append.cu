// lt_paged_q8_append.cu — queries, keys and values of a batch of tokens on their
// way into a paged cache of 8-bit codes.
//
// Per head vector what lt_paged_append.cu does (norm, rotation); then, for K and V of
// one KV head and one block of slots that the call writes to,
//   top = max |x| over the new rows' elements,  scale = max(top / 127, scale of the codes that stay),
//   code = x / scale to nearest,  a code that stays: code * (old scale / scale) to nearest.
// A maximum does not depend on order, so neither do scales and codes.
//
// Angles: p / theta^(2i/hd) in units of pi, reduced to [-1, 1] in f64, before the f32
// sine and cosine: an angle in f32 alone is off by up to half a unit in its last place, 2e-4 at
// position 4000.
//
// Bound: memory.  A CTA takes one block of one sequence; a warp one head vector of all of
// the block's tokens, 16 at a time, so that a block of 16 stays in registers between its
// maximum and its codes.  Longer blocks are read again (from L2).
#include "lt_paged_q8.cuh"

namespace lt {

constexpr int kQaThreads = 256, kQaWarps = kQaThreads / 32, kQaChunk = 16;

template <int N>
struct QaInt {
    static constexpr int value = N;
};

// A sequence's share of the call: n new rows from row c0 on, its first new position, and the blocks they lie in.
struct QaSeq {
    uint32_t c0, n, first, b0, blocks;
};
LT_DEVINL QaSeq qa_seq(const PagedQ8AppendArgs &a, uint32_t s, bool report) {
    QaSeq q = {0, 0, 0, 0, 0};
    const uint32_t c0 = a.cu[s], c1 = a.cu[s + 1], len = a.lens[s];
    const uint64_t cap = min((uint64_t)a.kv.max_pages * a.kv.page_size, (uint64_t)1 << 30);
    if (c0 > c1 || c1 > a.total_q || c1 - c0 > a.max_q || c1 - c0 > len || len > cap) {
        if (report) atomicExch(a.err, DEV_ERR_BAD_INDEX);
        return q;
    }
    if (c0 == c1) return q;
    q.c0 = c0;
    q.n = c1 - c0;
    q.first = len - q.n;
    q.b0 = q.first >> a.kv.block_shift;
    q.blocks = ((len - 1) >> a.kv.block_shift) - q.b0 + 1;
    return q;
}

template <int N>
LT_DEVINL void qa_load(const float *p, float (&v)[N]) {
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
LT_DEVINL void qa_store(float *p, const float (&v)[N]) {
    if constexpr (N == 4)
        *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
    else if constexpr (N == 2)
        *reinterpret_cast<float2 *>(p) = make_float2(v[0], v[1]);
    else
        p[0] = v[0];
}
LT_DEVINL uint32_t qa_code(float x, float scale) {  // scale > 0
    return (uint32_t)(int)fminf(fmaxf(rintf(__fdiv_rn(x, scale)), -127.0f), 127.0f) & 0xffu;
}
template <int N>
LT_DEVINL void qa_store_codes(uint8_t *p, const float (&v)[N], float scale) {
    uint32_t w = 0;
    if (scale > 0.0f) {
#pragma unroll
        for (int e = 0; e < N; e++) w |= qa_code(v[e], scale) << (8 * e);
    }
    if constexpr (N == 4)
        *reinterpret_cast<uint32_t *>(p) = w;
    else if constexpr (N == 2)
        *reinterpret_cast<uint16_t *>(p) = (uint16_t)w;
    else
        *p = (uint8_t)w;
}

// Lane l holds N = HD / 64 rotation pairs as k_paged_append does: elements l N .. and HD / 2 + l N .. (consecutive
// pairs of head_dim 64: 2 l and 2 l + 1).  Grid (blocks of all sequences at most, ceil(vectors / heads_per_cta)).
template <int HD>
__global__ void __launch_bounds__(kQaThreads) k_paged_q8_append(const __grid_constant__ PagedQ8AppendArgs a) {
    constexpr int N = HD / 64, HALF = HD / 2;
    __shared__ double s_turn[HALF];  // turns of pi per position
    __shared__ float2 s_cs[kQaChunk][HALF];
    __shared__ uint64_t s_scan[kQaWarps];
    __shared__ QaSeq s_q;
    __shared__ uint32_t s_seq, s_block;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_launch_dependents();
    for (int i = tid; i < HALF; i += kQaThreads) s_turn[i] = exp2(-a.log2_theta * (double)(2 * i) / HD) * 0.31830988618379067;
    pdl_wait();

    // the sequence and block of this CTA: blocks of all sequences, counted through
    const uint32_t per = (a.n_seq + kQaThreads - 1) / kQaThreads;
    const uint32_t sa = min(a.n_seq, tid * per), sb = min(a.n_seq, sa + per);
    uint64_t mine = 0;
    for (uint32_t s = sa; s < sb; s++) mine += qa_seq(a, s, blockIdx.x == 0 && blockIdx.y == 0).blocks;
    uint64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
    }
    if (lane == 31) s_scan[warp] = incl;
    __syncthreads();
    uint64_t before = incl - mine, all = 0;
#pragma unroll
    for (int w = 0; w < kQaWarps; w++) {
        if (w < warp) before += s_scan[w];
        all += s_scan[w];
    }
    if (blockIdx.x >= all) return;
    if (blockIdx.x >= before && blockIdx.x < before + mine) {
        uint64_t rem = blockIdx.x - before;
        for (uint32_t s = sa; s < sb; s++) {
            const QaSeq q = qa_seq(a, s, false);
            if (rem < q.blocks) {
                s_q = q;
                s_seq = s;
                s_block = (uint32_t)rem;
                break;
            }
            rem -= q.blocks;
        }
    }
    __syncthreads();
    const QaSeq q = s_q;
    const uint32_t size = 1u << a.kv.block_shift;
    const uint32_t start = (q.b0 + s_block) << a.kv.block_shift;                // the block's first position
    const uint32_t p0 = max(start, q.first), p1 = min(start + size, q.first + q.n);  // positions p0 .. p1 - 1 are new
    const uint32_t ntok = p1 - p0, old = p0 - start, row0 = q.c0 + (p0 - q.first);
    const uint32_t page = a.table[(uint64_t)s_seq * a.kv.max_pages + page_of(a.kv, start)];
    const bool there = page < a.kv.n_pages;
    if (!there && tid == 0) atomicExch(a.err, DEV_ERR_BAD_INDEX);

    const uint32_t H = a.n_heads, KV = a.kv.n_kv, vecs = H + 2 * KV;
    const uint32_t first = blockIdx.y * a.heads_per_cta, last = min(vecs, first + a.heads_per_cta);
    const bool neox = a.rope_neox;
    const bool split = neox || N > 1;
    const uint32_t e0 = split ? lane * N : 2 * lane, e1 = split ? HALF + lane * N : 2 * lane + 1;

    // angles of tokens t0 .. of the block
    auto angles = [&](uint32_t t0) {
        __syncthreads();
        const uint32_t n = min(ntok - t0, (uint32_t)kQaChunk);
        for (uint32_t i = tid; i < n * HALF; i += kQaThreads) {
            const uint32_t t = i / HALF, e = i % HALF;
            const uint32_t pos = a.pos ? a.pos[row0 + t0 + t] : p0 + t0 + t;
            const double turn = (double)pos * s_turn[e];
            float s, c;
            sincospif((float)(turn - 2.0 * rint(turn * 0.5)), &s, &c);
            s_cs[t][e] = make_float2(c, s);
        }
        __syncthreads();
    };
    // head vector h of NT tokens from t0 on, of which n are there, normalised and rotated
    auto fetch = [&](auto &x, auto &y, uint32_t h, uint32_t t0, uint32_t n) {
        constexpr int NT = sizeof(x) / sizeof(x[0]);
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const float *src = a.qkv + ((uint64_t)(row0 + t0 + t) * vecs + h) * HD;
            if ((uint32_t)t < n) {
                qa_load<N>(src + e0, x[t]);
                qa_load<N>(src + e1, y[t]);
            } else {
#pragma unroll
                for (int e = 0; e < N; e++) x[t][e] = y[t][e] = 0.0f;
            }
        }
        const bool is_q = h < H, is_v = h >= H + KV;
        const float *w = is_q ? a.q_norm : is_v ? nullptr : a.k_norm;
        if (w || (is_v && a.v_norm)) {
            float wx[N], wy[N];
#pragma unroll
            for (int e = 0; e < N; e++) {
                wx[e] = w ? w[e0 + e] : 1.0f;
                wy[e] = w ? w[e1 + e] : 1.0f;
            }
#pragma unroll
            for (int t = 0; t < NT; t++) {
                float ss = 0.0f;
#pragma unroll
                for (int e = 0; e < N; e++) ss = fmaf(x[t][e], x[t][e], fmaf(y[t][e], y[t][e], ss));
                ss = warp_sum(ss);
                const float inv = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(ss, (float)HD), a.eps)));
#pragma unroll
                for (int e = 0; e < N; e++) {
                    x[t][e] = x[t][e] * inv * wx[e];
                    y[t][e] = y[t][e] * inv * wy[e];
                }
            }
        }
        if (is_v) return;
#pragma unroll
        for (int t = 0; t < NT; t++) {
            if ((uint32_t)t >= n) break;
            if (neox) {
#pragma unroll
                for (int e = 0; e < N; e++) {
                    const float2 cs = s_cs[t][lane * N + e];
                    const float p = x[t][e], r = y[t][e];
                    x[t][e] = fmaf(p, cs.x, -r * cs.y);
                    y[t][e] = fmaf(p, cs.y, r * cs.x);
                }
            } else if constexpr (N > 1) {
#pragma unroll
                for (int e = 0; e < N; e += 2) {
                    const float2 cx = s_cs[t][(lane * N + e) / 2], cy = s_cs[t][(HALF + lane * N + e) / 2];
                    const float p = x[t][e], r = x[t][e + 1], u = y[t][e], v = y[t][e + 1];
                    x[t][e] = fmaf(p, cx.x, -r * cx.y);
                    x[t][e + 1] = fmaf(p, cx.y, r * cx.x);
                    y[t][e] = fmaf(u, cy.x, -v * cy.y);
                    y[t][e + 1] = fmaf(u, cy.y, v * cy.x);
                }
            } else {
                const float2 cs = s_cs[t][lane];
                const float p = x[t][0], r = y[t][0];
                x[t][0] = fmaf(p, cs.x, -r * cs.y);
                y[t][0] = fmaf(p, cs.y, r * cs.x);
            }
        }
    };
    // the largest magnitude, as bits: NaN is above infinity, infinity above every number
    auto top_of = [&](const auto &x, const auto &y) {
        constexpr int NT = sizeof(x) / sizeof(x[0]);
        uint32_t top = 0;
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int e = 0; e < N; e++)
                top = max(top, max(__float_as_uint(x[t][e]) & 0x7fffffffu, __float_as_uint(y[t][e]) & 0x7fffffffu));
        return __reduce_max_sync(0xffffffffu, top);
    };
    // the block's scale for head vector h; codes that stay go onto it
    auto rescale = [&](uint32_t h, uint32_t top) {
        const bool is_v = h >= H + KV;
        const uint32_t kh = h - H - (is_v ? KV : 0);
        float *at = (is_v ? a.kv.v_scale : a.kv.k_scale) + q8_scale_at(a.kv, page, start, kh);
        float scale = top > __float_as_uint(kQ8Most) ? __int_as_float(0x7fffffff) : __fdiv_rn(__uint_as_float(top), 127.0f);
        if (old) {
            const float was = *at;
            __syncwarp();
            if (!(was >= 0.0f && was <= 3.402823466e38f)) scale = __int_as_float(0x7fffffff);
            if (scale > was) {
                const float f = __fdiv_rn(was, scale);
                uint8_t *codes = (is_v ? a.kv.v : a.kv.k) + paged_offset(a.kv, page, start, kh);
                for (uint32_t i = lane; i < old * (HD / 4); i += 32) {
                    uint32_t *p = reinterpret_cast<uint32_t *>(codes + (uint64_t)(i / (HD / 4)) * a.kv.slot_stride) + i % (HD / 4);
                    const uint32_t c = *p;
                    uint32_t w = 0;
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        w |= ((uint32_t)__float2int_rn((float)(int8_t)(c >> (8 * e)) * f) & 0xffu) << (8 * e);
                    *p = w;
                }
            }
            if (scale <= was) scale = was;
        }
        if (lane == 0) *at = scale;
        return scale;
    };
    auto put = [&](const auto &x, const auto &y, uint32_t h, uint32_t t0, uint32_t n, float scale) {
        constexpr int NT = sizeof(x) / sizeof(x[0]);
        const bool is_v = h >= H + KV;
        uint8_t *dst = (is_v ? a.kv.v : a.kv.k) + paged_offset(a.kv, page, p0 + t0, h - H - (is_v ? KV : 0));
#pragma unroll
        for (int t = 0; t < NT; t++) {
            if ((uint32_t)t >= n) break;
            qa_store_codes<N>(dst + t * a.kv.slot_stride + e0, x[t], scale);
            qa_store_codes<N>(dst + t * a.kv.slot_stride + e1, y[t], scale);
        }
    };
    __shared__ uint32_t s_top[2048];  // of K and V heads of this CTA (n_kv <= 1024)
    auto work = [&](auto nt) {
        constexpr int NT = decltype(nt)::value;
        float x[NT][N], y[NT][N];
        if (ntok <= NT) {
            angles(0);
            for (uint32_t h = first + warp; h < last; h += kQaWarps) {
                fetch(x, y, h, 0, ntok);
                if (h < H) {
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        if ((uint32_t)t >= ntok) break;
                        float *dst = a.q + ((uint64_t)(row0 + t) * H + h) * HD;
                        qa_store<N>(dst + e0, x[t]);
                        qa_store<N>(dst + e1, y[t]);
                    }
                } else if (there) {
                    const float scale = rescale(h, top_of(x, y));
                    put(x, y, h, 0, ntok, scale);
                }
            }
            return;
        }
        // more tokens than the registers hold: the maxima first, then everything again for the codes
        for (uint32_t i = tid; i < 2 * KV; i += kQaThreads) s_top[i] = 0;
        for (int pass = 0; pass < 2; pass++) {
            for (uint32_t t0 = 0; t0 < ntok; t0 += NT) {
                const uint32_t n = min(ntok - t0, (uint32_t)NT);
                angles(t0);
                for (uint32_t h = first + warp; h < last; h += kQaWarps) {
                    if (pass && h < H) continue;
                    fetch(x, y, h, t0, n);
                    if (h < H) {
#pragma unroll
                        for (int t = 0; t < NT; t++) {
                            if ((uint32_t)t >= n) break;
                            float *dst = a.q + ((uint64_t)(row0 + t0 + t) * H + h) * HD;
                            qa_store<N>(dst + e0, x[t]);
                            qa_store<N>(dst + e1, y[t]);
                        }
                    } else if (!there) {
                        continue;
                    } else if (pass == 0) {
                        const uint32_t top = max(s_top[h - H], top_of(x, y));
                        __syncwarp();
                        if (lane == 0) s_top[h - H] = top;
                        __syncwarp();
                    } else {
                        const uint32_t top = s_top[h - H];
                        __syncwarp();
                        // s_top holds the scale's bits from the first chunk on
                        float scale = __uint_as_float(top);
                        if (t0 == 0) {
                            scale = rescale(h, top);
                            if (lane == 0) s_top[h - H] = __float_as_uint(scale);
                        }
                        __syncwarp();
                        put(x, y, h, t0, n, scale);
                    }
                }
            }
        }
    };
    if (ntok == 1)
        work(QaInt<1>());
    else
        work(QaInt<kQaChunk>());
}

cudaError_t launch_paged_q8_append(const LaunchCfg &c, PagedQ8AppendArgs a) {
    const uint32_t vecs = a.n_heads + 2 * a.kv.n_kv;
    a.err = c.dev_err;
    // blocks that the rows of all sequences can lie in: n rows touch at most n / size + 2, and n
    const uint64_t blocks = min((uint64_t)a.total_q, (uint64_t)(a.total_q >> a.kv.block_shift) + 2 * (uint64_t)a.n_seq);
    const bool few = blocks < 4u * (uint32_t)c.num_sms;
    a.heads_per_cta = few ? kQaWarps : vecs;
    const dim3 grid((uint32_t)blocks, (vecs + a.heads_per_cta - 1) / a.heads_per_cta);
    switch (a.kv.hd) {
    case 64: return launch_k(c, "paged_q8_append", k_paged_q8_append<64>, grid, dim3(kQaThreads), 0, a);
    case 128: return launch_k(c, "paged_q8_append", k_paged_q8_append<128>, grid, dim3(kQaThreads), 0, a);
    case 256: return launch_k(c, "paged_q8_append", k_paged_q8_append<256>, grid, dim3(kQaThreads), 0, a);
    default: return cudaErrorInvalidValue;
    }
}

}  // namespace lt
