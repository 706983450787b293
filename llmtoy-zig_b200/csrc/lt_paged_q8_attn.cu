// lt_paged_q8_attn.cu — attention over a paged cache of 8-bit codes.
//
// The formulas are lt_paged_attn.cu's, with the blocks' scales as lt_paged_q8.cuh puts
// them.  One warp per query row and head: it goes through the keys with the running
// maximum m and sum l, lane i on dims i hd / 32 on.
#include "lt_paged_q8.cuh"

namespace lt {

constexpr int kQrWarps = 4;

template <int N>
LT_DEVINL void q8_ld_row(const uint8_t *p, float (&v)[N]) {
#pragma unroll
    for (int e = 0; e < N; e++) v[e] = (float)(int8_t)p[e];
}

template <int HD>
__global__ void __launch_bounds__(kQrWarps * 32) k_paged_q8_rows(const __grid_constant__ PagedAttnArgs a, uint64_t rows) {
    constexpr int N = HD / 32, U = 4;
    pdl_launch_dependents();
    pdl_wait();
    const uint64_t r = (uint64_t)blockIdx.x * kQrWarps + threadIdx.x / 32;
    if (r >= rows) return;
    const uint32_t lane = threadIdx.x & 31, head = (uint32_t)(r % a.n_heads), kh = head / a.group;
    const uint64_t rest = r / a.n_heads;
    const uint32_t s = (uint32_t)(rest / a.max_q), t = (uint32_t)(rest % a.max_q);
    const uint32_t cap = (uint32_t)min((uint64_t)a.kv.max_pages * a.kv.page_size, (uint64_t)a.max_len);
    const uint32_t given = a.lens[s], len = min(given, cap);
    uint32_t q0 = s, nq = 1;
    bool bad = given > cap;
    if (a.cu) {
        const uint32_t c0 = a.cu[s], c1 = a.cu[s + 1];
        const bool ok = c0 <= c1 && c1 <= a.total_q && c1 - c0 <= a.max_q;
        bad |= !ok;
        q0 = c0;
        nq = ok ? c1 - c0 : 0;
    }
    if (bad && lane == 0 && t == 0) atomicExch(a.err, DEV_ERR_BAD_INDEX);
    if (t >= nq) return;
    const uint32_t row = q0 + t, *table = a.table + (uint64_t)s * a.kv.max_pages;
    const uint32_t *docs = a.docs ? a.docs + (uint64_t)s * a.doc_stride : nullptr;
    const int64_t i = (int64_t)len - nq + t;
    int64_t lo = 0, hi = len;
    if (a.window) lo = max((int64_t)0, i - (int64_t)a.window + 1);
    if (a.cu && a.causal) hi = min(hi, max(i + 1, a.prefix ? (int64_t)a.prefix[s] : (int64_t)0));
    if (docs && i < 0) hi = 0;
    const float slope = a.slopes ? a.slopes[head] : 0.0f;
    const float f = a.softcap != 0.0f ? a.scale / a.softcap : a.scale * 1.4426950408889634f;
    const float *q = a.q + (uint64_t)row * a.q_stride + (uint64_t)head * HD + lane * N;
    float x[N], o[N], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < N; e++) {
        x[e] = q[e];
        o[e] = 0.0f;
    }
    for (int64_t j0 = lo; j0 < hi; j0 += U) {
        uint32_t page[U];
        bool seen[U];
        float dot[U];
#pragma unroll
        for (int u = 0; u < U; u++) {  // alike in all lanes
            const int64_t j = j0 + u;
            seen[u] = j < hi && (!docs || docs[j] == docs[i]);
            page[u] = seen[u] ? table[page_of(a.kv, (uint32_t)j)] : 0;
            if (page[u] >= a.kv.n_pages) {
                if (lane == 0) atomicExch(a.err, DEV_ERR_BAD_INDEX);
                seen[u] = false;
            }
            dot[u] = 0.0f;
            if (seen[u]) {
                float k[N];
                q8_ld_row(a.kv.k + paged_offset(a.kv, page[u], (uint32_t)j, kh) + lane * N, k);
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
            const uint32_t j = (uint32_t)(j0 + u);
            const uint64_t at = q8_scale_at(a.kv, page[u], j, kh);
            const Q8Scale sc = q8_scale(a.kv.k_scale[at], a.kv.v_scale[at]);
            float v[N];
            q8_ld_row(a.kv.v + paged_offset(a.kv, page[u], j, kh) + lane * N, v);
            const float y = score_log2(dot[u] * sc.k, f, a.softcap, slope, fabsf((float)(i - (int64_t)j))) + sc.v_log2;
            const float mn = fmaxf(m, y), base = mn == -INFINITY ? 0.0f : mn;
            const float al = ex2(m - base), p = ex2(y - base);
            m = mn;
            l = fmaf(l, al, p * sc.v_inv);
#pragma unroll
            for (int e = 0; e < N; e++) o[e] = fmaf(o[e], al, p * v[e]);
        }
    }
    float *out = a.out + (uint64_t)row * a.out_stride + (uint64_t)head * HD + lane * N;
#pragma unroll
    for (int e = 0; e < N; e++) out[e] = l == 0.0f ? 0.0f : (l == l ? o[e] / l : l);
}

size_t paged_q8_attn_scratch(const PagedAttnArgs &, int) { return 0; }

cudaError_t launch_paged_q8_attn(const LaunchCfg &c, PagedAttnArgs a, uint8_t *) {
    a.err = c.dev_err;
    const uint64_t rows = (uint64_t)a.n_seq * a.max_q * a.n_heads, ctas = (rows + kQrWarps - 1) / kQrWarps;
    if (ctas > 0x7fffffffull) return cudaErrorInvalidValue;
    const dim3 grid((uint32_t)ctas), block(kQrWarps * 32);
    switch (a.kv.hd) {
    case 64: return launch_k(c, "paged_q8_attn", k_paged_q8_rows<64>, grid, block, 0, a, rows);
    case 128: return launch_k(c, "paged_q8_attn", k_paged_q8_rows<128>, grid, block, 0, a, rows);
    case 256: return launch_k(c, "paged_q8_attn", k_paged_q8_rows<256>, grid, block, 0, a, rows);
    default: return cudaErrorInvalidValue;
    }
}

}  // namespace lt
