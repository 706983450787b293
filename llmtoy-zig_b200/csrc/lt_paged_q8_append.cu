// lt_paged_q8_append.cu — queries, keys and values of a batch of tokens on their
// way into a paged cache of 8-bit codes.
//
// Per head vector what lt_paged_append.cu does (norm, rotation); then, for K and V of
// one KV head and one block of slots that the call writes to,
//   top = max |x| over the new rows' elements,  scale = max(top / 127, scale of the codes that stay),
//   code = x / scale to nearest,  a code that stays: code * (old scale / scale) to nearest,
// where the quotient is a product with a rounded inverse or quotient, off by 127 * 2^-23 = 1.5e-5 at most: nearer than
// that to the middle between two codes it may go to either.
// A maximum does not depend on order, so neither do scales and codes.
//
// Angles: p / theta^(2i/hd) in units of pi, reduced to [-1, 1] in f64, before the f32
// sine and cosine: an angle in f32 alone is off by up to half a unit in its last place, 2e-4 at
// position 4000.
//
// Bound: memory (each value is read once, and written once or as a quarter of its size).  One B200, calls by
// themselves in a row (three sets of inputs larger than L2): 7003 prompt tokens (16/8 heads of 256,
// normalised values) 75.2 us, 5.0 TB/s, with a warp per row and no teams 214; 8192 tokens of 32/4 heads
// of 128 62 us, 5.0 TB/s (blocks of 128: 73); one token of each of 64 sequences 3.8 us from a graph and 5.1
// launched by the host, where launch and the lengths' scan count.  Spills: 100 bytes at head_dim 256 with
// blocks of 128 (255 registers), 84 at 128, 28 at 256 with smaller blocks.  A CTA takes one block of one
// sequence; teams of its warps go through the head vectors, each warp with CHUNK of the block's
// tokens in registers from the load to the codes, the team's maximum through shared
// memory.  What costs instructions otherwise is shared among tokens: the sums of squares
// of a chunk are reduced together (16 rows: 16 shuffles instead of 80, one square root per
// lane instead of 16), and a code is the low byte of x / scale + 1.5 * 2^23, one operation.
#include "lt_paged_q8.cuh"

namespace lt {

constexpr int kQaThreads = 256, kQaWarps = kQaThreads / 32;

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
// Codes of N values times r: the low bytes of x r + 1.5 * 2^23, whose unit is 1 (|x r| is at most 127 and a bit).
template <int N>
LT_DEVINL void qa_store_codes(uint8_t *p, const float (&v)[N], float r) {
    uint32_t w[N];
#pragma unroll
    for (int e = 0; e < N; e++) w[e] = __float_as_uint(fmaf(v[e], r, 12582912.0f));
    if constexpr (N == 4)
        *reinterpret_cast<uint32_t *>(p) = __byte_perm(__byte_perm(w[0], w[1], 0x0040), __byte_perm(w[2], w[3], 0x0040), 0x5410);
    else if constexpr (N == 2)
        *reinterpret_cast<uint16_t *>(p) = (uint16_t)__byte_perm(w[0], w[1], 0x0040);
    else
        *p = (uint8_t)w[0];
}

// Sums over the warp of NT values per lane (NT 1, 8 or 16): lane l returns that of value l % NT.
template <int NT>
LT_DEVINL float warp_sums(float (&v)[NT], int lane) {
#pragma unroll
    for (int n = NT / 2; n >= 1; n /= 2) {  // halves of the values change places between lanes n apart
        const bool up = lane & n;
#pragma unroll
        for (int i = 0; i < n; i++) {
            const float give = up ? v[i] : v[i + n], keep = up ? v[i + n] : v[i];
            v[i] = keep + __shfl_xor_sync(0xffffffffu, give, n);
        }
    }
    float x = v[0];
#pragma unroll
    for (int n = NT; n < 32; n *= 2) x += __shfl_xor_sync(0xffffffffu, x, n);
    return x;
}

// Lane l holds N = HD / 64 rotation pairs as k_paged_append does: elements l N .. and HD / 2 + l N .. (consecutive
// pairs of head_dim 64: 2 l and 2 l + 1).  Grid (blocks of all sequences at most, ceil(vectors / heads_per_cta)).
// CHUNK: tokens of a warp; 1: calls whose sequences have one row each.
template <int HD, int CHUNK>
__global__ void __launch_bounds__(kQaThreads, CHUNK == 1 ? 4 : HD * CHUNK >= 4096 ? 1 : 2) k_paged_q8_append(const __grid_constant__ PagedQ8AppendArgs a) {
    constexpr int N = HD / 64, HALF = HD / 2;
    extern __shared__ __align__(16) float2 s_cs[];  // [tokens of the block][HALF]
    __shared__ double s_turn[HALF];  // turns of pi per position
    __shared__ uint32_t s_top[2][kQaWarps];
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

    // angles of the block's new tokens
    for (uint32_t i = tid; i < ntok * HALF; i += kQaThreads) {
        const uint32_t t = i / HALF, e = i % HALF;
        const uint32_t pos = a.pos ? a.pos[row0 + t] : p0 + t;
        const double turn = (double)pos * s_turn[e];
        float s, c;
        sincospif((float)(turn - 2.0 * rint(turn * 0.5)), &s, &c);
        s_cs[i] = make_float2(c, s);
    }
    __syncthreads();

    // this warp's team and its tokens t0 .. t0 + n - 1
    const uint32_t team_warps = CHUNK == 1 ? 1 : max(1u, size / CHUNK), teams = kQaWarps / team_warps;
    const uint32_t team = warp / team_warps, t0 = warp % team_warps * CHUNK;
    const uint32_t n = t0 < ntok ? min(ntok - t0, (uint32_t)CHUNK) : 0;
    auto team_sync = [&]() {
        __syncwarp();
        if (team_warps > 1) asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(team_warps * 32) : "memory");
    };
    uint32_t turn = 0;
    for (uint32_t h = first + team; h < last; h += teams, turn ^= 1) {
        const bool is_q = h < H, is_v = h >= H + KV;
        float x[CHUNK][N], y[CHUNK][N];
#pragma unroll
        for (int t = 0; t < CHUNK; t++) {
            const float *src = a.qkv + ((uint64_t)(row0 + t0 + t) * vecs + h) * HD;
            if ((uint32_t)t < n) {
                qa_load<N>(src + e0, x[t]);
                qa_load<N>(src + e1, y[t]);
            } else {
#pragma unroll
                for (int e = 0; e < N; e++) x[t][e] = y[t][e] = 0.0f;
            }
        }
        // The next head's rows towards L2 meanwhile.  head_dim 256, whose chunks are the fewest tokens: 77.9 -> 74.9 us; 128 loses
        // more to the registers that the addresses take (62.2 -> 64.6).
        if (HD == 256 && CHUNK > 1 && h + teams < last) {
            constexpr uint32_t LINES = HD / 32;
#pragma unroll
            for (uint32_t i = lane; i < CHUNK * LINES; i += 32)
                if (i / LINES < n) prefetch_l2(a.qkv + ((uint64_t)(row0 + t0 + i / LINES) * vecs + h + teams) * HD + i % LINES * 32);
        }
        const float *w = is_q ? a.q_norm : is_v ? nullptr : a.k_norm;
        if (w || (is_v && a.v_norm)) {
            float ss[CHUNK], wx[N], wy[N];
#pragma unroll
            for (int e = 0; e < N; e++) {
                wx[e] = w ? w[e0 + e] : 1.0f;
                wy[e] = w ? w[e1 + e] : 1.0f;
            }
#pragma unroll
            for (int t = 0; t < CHUNK; t++) {
                ss[t] = 0.0f;
#pragma unroll
                for (int e = 0; e < N; e++) ss[t] = fmaf(x[t][e], x[t][e], fmaf(y[t][e], y[t][e], ss[t]));
            }
            // 0 for rows that are not there, which stay 0 and out of the block's maximum: with eps = 0 their own inverse
            // would be infinite
            const float mean = fmaf(warp_sums<CHUNK>(ss, lane), 1.0f / HD, a.eps);
            const float inv = (uint32_t)lane % CHUNK < n ? __fdiv_rn(1.0f, __fsqrt_rn(mean)) : 0.0f;
#pragma unroll
            for (int t = 0; t < CHUNK; t++) {
                const float f = __shfl_sync(0xffffffffu, inv, t);
#pragma unroll
                for (int e = 0; e < N; e++) {
                    x[t][e] *= f * wx[e];
                    y[t][e] *= f * wy[e];
                }
            }
        }
        if (!is_v) {
#pragma unroll
            for (int t = 0; t < CHUNK; t++) {
                const float2 *cs = s_cs + ((uint32_t)t < n ? t0 + t : 0) * HALF;
                if (neox) {
#pragma unroll
                    for (int e = 0; e < N; e++) {
                        const float2 z = cs[lane * N + e];
                        const float p = x[t][e], r = y[t][e];
                        x[t][e] = fmaf(p, z.x, -r * z.y);
                        y[t][e] = fmaf(p, z.y, r * z.x);
                    }
                } else if constexpr (N > 1) {
#pragma unroll
                    for (int e = 0; e < N; e += 2) {
                        const float2 zx = cs[(lane * N + e) / 2], zy = cs[(HALF + lane * N + e) / 2];
                        const float p = x[t][e], r = x[t][e + 1], u = y[t][e], v = y[t][e + 1];
                        x[t][e] = fmaf(p, zx.x, -r * zx.y);
                        x[t][e + 1] = fmaf(p, zx.y, r * zx.x);
                        y[t][e] = fmaf(u, zy.x, -v * zy.y);
                        y[t][e + 1] = fmaf(u, zy.y, v * zy.x);
                    }
                } else {
                    const float2 z = cs[lane];
                    const float p = x[t][0], r = y[t][0];
                    x[t][0] = fmaf(p, z.x, -r * z.y);
                    y[t][0] = fmaf(p, z.y, r * z.x);
                }
            }
        }
        if (is_q) {
#pragma unroll
            for (int t = 0; t < CHUNK; t++) {
                if ((uint32_t)t >= n) break;
                float *dst = a.q + ((uint64_t)(row0 + t0 + t) * H + h) * HD;
                qa_store<N>(dst + e0, x[t]);
                qa_store<N>(dst + e1, y[t]);
            }
            continue;
        }
        if (!there) continue;
        // the largest magnitude, as bits: NaN is above infinity, infinity above every number
        uint32_t top = 0;
#pragma unroll
        for (int t = 0; t < CHUNK; t++)
#pragma unroll
            for (int e = 0; e < N; e++)
                top = max(top, max(__float_as_uint(x[t][e]) & 0x7fffffffu, __float_as_uint(y[t][e]) & 0x7fffffffu));
        top = __reduce_max_sync(0xffffffffu, top);
        if (team_warps > 1) {  // of the team; the two places take turns, so that one barrier does
            if (lane == 0) s_top[turn][warp] = top;
            team_sync();
            for (uint32_t i = team * team_warps; i < (team + 1) * team_warps; i++) top = max(top, s_top[turn][i]);
        }
        // The block's scale.  Every warp of the team works it out; the first writes it, after all have read the old one,
        // and puts the codes that stay onto it.
        const uint32_t kh = h - H - (is_v ? KV : 0);
        float *at = (is_v ? a.kv.v_scale : a.kv.k_scale) + q8_scale_at(a.kv, page, start, kh);
        uint8_t *codes = (is_v ? a.kv.v : a.kv.k) + paged_offset(a.kv, page, start, kh);
        float scale = top > __float_as_uint(kQ8Most) ? __int_as_float(0x7fffffff) : __fdiv_rn(__uint_as_float(top), 127.0f);
        if (old) {
            const float was = *at;
            if (!(was >= 0.0f && was <= 3.402823466e38f)) scale = __int_as_float(0x7fffffff);
            team_sync();
            if (scale > was && t0 == 0) {
                const float f = __fdiv_rn(was, scale);
                for (uint32_t i = lane; i < old * (HD / 4); i += 32) {
                    uint32_t *p = reinterpret_cast<uint32_t *>(codes + (uint64_t)(i / (HD / 4)) * a.kv.slot_stride) + i % (HD / 4);
                    const uint32_t c = *p;
                    uint32_t b = 0;
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        b |= ((uint32_t)__float2int_rn((float)(int8_t)(c >> (8 * e)) * f) & 0xffu) << (8 * e);
                    *p = b;
                }
            }
            if (scale <= was) scale = was;
        }
        if (lane == 0 && t0 == 0) *at = scale;
        // Codes: x / scale by its inverse (0: no codes).  Where that is not a normal number everything is scaled up first,
        // and the values held to the codes' range: a scale of few bits may be far from top / 127.
        const bool tiny = scale < 0x1p-100f;
        const float r = scale > 0.0f ? __fdiv_rn(1.0f, tiny ? scale * 0x1p100f : scale) : 0.0f;
        if (tiny) {
#pragma unroll
            for (int t = 0; t < CHUNK; t++)
#pragma unroll
                for (int e = 0; e < N; e++) {
                    const float most = 127.0f * (scale * 0x1p100f);
                    x[t][e] = fminf(fmaxf(x[t][e] * 0x1p100f, -most), most);
                    y[t][e] = fminf(fmaxf(y[t][e] * 0x1p100f, -most), most);
                }
        }
        const bool none = !(scale > 0.0f);  // zeros, or no numbers: codes of 0
        codes += (uint64_t)(p0 - start + t0) * a.kv.slot_stride;
#pragma unroll
        for (int t = 0; t < CHUNK; t++) {
            if ((uint32_t)t >= n) break;
            if (none) {
#pragma unroll
                for (int e = 0; e < N; e++) x[t][e] = y[t][e] = 0.0f;
            }
            qa_store_codes<N>(codes + t * a.kv.slot_stride + e0, x[t], r);
            qa_store_codes<N>(codes + t * a.kv.slot_stride + e1, y[t], r);
        }
    }
}

namespace {

// Tokens of a warp: what its registers hold, and a block's tokens fill at most the CTA's warps.
template <int HD>
cudaError_t qa_launch(const LaunchCfg &c, PagedQ8AppendArgs a) {
    const uint32_t vecs = a.n_heads + 2 * a.kv.n_kv, size = 1u << a.kv.block_shift;
    // blocks that the rows of all sequences can lie in: n rows touch at most n / size + 2, and n
    const uint64_t blocks = min((uint64_t)a.total_q, (uint64_t)(a.total_q >> a.kv.block_shift) + 2 * (uint64_t)a.n_seq);
    const uint32_t chunk = a.max_q == 1 ? 1 : HD == 256 && size < 128 ? 8 : 16;
    const uint32_t teams = chunk == 1 ? kQaWarps : kQaWarps / max(1u, size / chunk);
    // few blocks: several CTAs share one's heads, so that there are some six CTAs to an SM
    const uint64_t want = max((uint64_t)1, (uint64_t)c.num_sms * 6 / blocks);
    const uint32_t rounds = (uint32_t)max((uint64_t)1, (vecs + teams * want - 1) / (teams * want));
    a.heads_per_cta = rounds * teams;
    const dim3 grid((uint32_t)blocks, (vecs + a.heads_per_cta - 1) / a.heads_per_cta);
    const size_t smem = (size_t)min(a.max_q, size) * HD / 2 * sizeof(float2);
    if (chunk == 1) return launch_k(c, "paged_q8_append", k_paged_q8_append<HD, 1>, grid, dim3(kQaThreads), smem, a);
    if constexpr (HD == 256)
        if (chunk == 8) return launch_k(c, "paged_q8_append", k_paged_q8_append<HD, 8>, grid, dim3(kQaThreads), smem, a);
    return launch_k(c, "paged_q8_append", k_paged_q8_append<HD, 16>, grid, dim3(kQaThreads), smem, a);
}

}  // namespace

cudaError_t launch_paged_q8_append(const LaunchCfg &c, PagedQ8AppendArgs a) {
    a.err = c.dev_err;
    switch (a.kv.hd) {
    case 64: return qa_launch<64>(c, a);
    case 128: return qa_launch<128>(c, a);
    case 256: return qa_launch<256>(c, a);
    default: return cudaErrorInvalidValue;
    }
}

}  // namespace lt
