// lt_paged_walk.cuh — how the kernels for single tokens and few rows share the
// tiles of all sequences among their CTAs, and join what several of them left.
//
// A unit is (sequence, KV head, 8 rows); its tiles are counted through, unit after
// unit, and every CTA takes an equal stretch of the count.  A unit that several
// CTAs share leaves a record (m, l, sum) of each, which are added up in CTA order.
#pragma once

#include "lt_paged.cuh"

namespace lt {

constexpr int kPaWarps = 4, kPaThreads = kPaWarps * 32, kPaRows = 8;

// What a unit costs beyond its tiles, in tiles.  64 sequences of 200 to 8192: 66 us without, 62 with 1,
// 58 with 2 to 4 (a CTA of many short units was the last to end).
constexpr uint32_t kUnitCost = 3;

// A sequence's share of the work.
struct PaSeq {
    uint32_t len, nq, q0;   // cached positions, query tokens, first query row
    uint32_t lo;            // first position any query sees
    uint32_t base;          // where its tiles start: lo, or the block of 16 it lies in
    uint32_t blocks, tiles; // 8-row blocks per KV head, tiles per unit
    LT_DEVINL uint32_t cost() const { return tiles + kUnitCost; }
};

template <bool PROMPT>
LT_DEVINL PaSeq pa_seq(const PagedAttnArgs &a, uint32_t s, uint32_t tile, bool report) {
    PaSeq q;
    uint32_t n = a.lens[s];
    const uint64_t cap = min((uint64_t)a.kv.max_pages * a.kv.page_size, (uint64_t)a.max_len);
    bool bad = n > cap;
    if (bad) n = (uint32_t)cap;
    q.len = n;
    if (PROMPT) {
        const uint32_t c0 = a.cu[s], c1 = a.cu[s + 1];
        const bool ok = c0 <= c1 && c1 <= a.total_q && c1 - c0 <= a.max_q;
        bad |= !ok;
        q.q0 = ok ? c0 : 0;
        q.nq = ok ? c1 - c0 : 0;
        const int64_t lo = (int64_t)n - q.nq - a.window + 1;
        q.lo = a.window && lo > 0 ? (uint32_t)min(lo, (int64_t)n) : 0;
        q.blocks = (uint32_t)(((uint64_t)q.nq * a.group + kPaRows - 1) / kPaRows);
    } else {
        q.q0 = s;
        q.nq = 1;
        q.lo = a.window && n > a.window ? n - a.window : 0;
        q.blocks = (a.group + kPaRows - 1) / kPaRows;
    }
    q.base = q.lo & ~15u;  // blocks then lie within pages whose size is a multiple of theirs
    q.tiles = max(1u, (n - q.base + tile - 1) / tile);
    if (bad && report) atomicExch(a.err, DEV_ERR_BAD_INDEX);
    return q;
}

// Where a walk through the tiles stands.
template <bool PROMPT>
struct PaWalk {
    uint32_t s, unit, tile;  // unit within the sequence: kv head * blocks + row block
    PaSeq q;
    uint32_t kh, rb;
    uint32_t lo, hi;         // positions that this unit's rows can see
    uint32_t base;

    LT_DEVINL void set_unit(const PagedAttnArgs &a) {
        kh = q.blocks ? unit / q.blocks : 0;
        rb = q.blocks ? unit % q.blocks : 0;
        lo = q.lo;
        hi = q.len;
        base = q.base;
        if (PROMPT) {
            const uint32_t rows = q.nq * a.group;  // nq <= max_q: checked on the host not to overflow
            const uint32_t t0 = rb * kPaRows / a.group, t1 = (min(rows, rb * kPaRows + kPaRows) - 1) / a.group;
            const int64_t i0 = (int64_t)q.len - q.nq + t0, i1 = (int64_t)q.len - q.nq + t1;
            if (a.causal) {
                int64_t e = i1 + 1;
                if (a.prefix) e = max(e, (int64_t)a.prefix[s]);
                hi = (uint32_t)max((int64_t)0, min(e, (int64_t)q.len));
            }
            if (a.window) lo = (uint32_t)max((int64_t)q.lo, i0 - (int64_t)a.window + 1);
        }
    }
    // The next unit's first tile; past the last sequence s == n_seq.
    template <int TILE>
    LT_DEVINL void next_unit(const PagedAttnArgs &a) {
        tile = 0;
        if (++unit >= q.blocks * a.kv.n_kv) {
            unit = 0;
            do {
                if (++s >= a.n_seq) return;
                q = pa_seq<PROMPT>(a, s, TILE, false);
            } while (q.blocks == 0);
        }
        set_unit(a);
    }
};

LT_DEVINL uint64_t div_small(uint64_t a, uint64_t b) {  // 32-bit division where it will do
    return (a | b) >> 32 ? a / b : (uint32_t)a / (uint32_t)b;
}

// T tiles over G <= T CTAs: the first `more` get each + 1, the others each.
struct PaShare {
    uint64_t each, more;
    LT_DEVINL PaShare(uint64_t T, uint32_t G) : each(div_small(T, G)), more(T - each * G) {}
    LT_DEVINL uint64_t start(uint32_t c) const { return each * c + min((uint64_t)c, more); }
    LT_DEVINL uint32_t owner(uint64_t f) const {
        const uint64_t big = more * (each + 1);
        return (uint32_t)(f < big ? div_small(f, each + 1) : more + div_small(f - big, each));
    }
};

// The number of a unit: its place in unit_info and unit_ml.
LT_DEVINL uint64_t pa_unit(const PagedAttnArgs &a, uint32_t s, uint32_t kh, uint32_t rb) {
    return ((uint64_t)s * a.kv.n_kv + kh) * a.row_blocks + rb;
}

// Partial p of a unit whose first CTA is `first`: that CTA's second record,
// the later ones' first.
LT_DEVINL uint64_t pa_part(uint32_t first, uint32_t p) { return 2 * (uint64_t)(first + p) + (p == 0 ? 1 : 0); }

constexpr uint32_t kPaMaxParts = 512;  // CTAs of a launch at most (pa_grid), and so records of a unit

// Row r of a unit that several CTAs share: out = sum_p 2^(m_p - m) o_p / sum_p 2^(m_p - m) l_p over
// its records in CTA order.  The first records' sums are on their way while the weights are found.
template <int HD, bool PROMPT>
LT_DEVINL void pa_join_row(const PagedAttnArgs &a, uint64_t u, uint32_t r) {
    constexpr int LANES = HD / 4, GROUPS = 128 / LANES, EARLY = 8;
    __shared__ float s_w[kPaMaxParts], s_red[4], s_red2[4];
    __shared__ float4 s_o[128];
    __shared__ uint32_t s_off;
    const uint32_t rb = (uint32_t)(u % a.row_blocks);
    const uint32_t kh = (uint32_t)(u / a.row_blocks % a.kv.n_kv), s = (uint32_t)(u / a.row_blocks / a.kv.n_kv);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint32_t nq = 1, q0 = s;
    if (PROMPT) {
        const uint32_t c0 = a.cu[s], c1 = a.cu[s + 1];
        if (!(c0 <= c1 && c1 <= a.total_q && c1 - c0 <= a.max_q)) return;
        q0 = c0;
        nq = c1 - c0;
    }
    const uint32_t R = rb * kPaRows + r;
    if (R >= nq * a.group) return;
    const uint32_t first = a.unit_info[2 * u], n = a.unit_info[2 * u + 1];
    if (n < 2 || n > kPaMaxParts) return;
    const int grp = tid / LANES, x = tid % LANES;
    const auto sums = [&](uint32_t p) {
        return *reinterpret_cast<const float4 *>(a.part_o + (pa_part(first, p) * kPaRows + r) * HD + 4 * x);
    };
    float4 v[EARLY];
#pragma unroll
    for (int i = 0; i < EARLY; i++)
        if (grp + i * GROUPS < n) v[i] = sums(grp + i * GROUPS);
    constexpr int PER = kPaMaxParts / 128;
    float pm[PER], pl[PER], m = -INFINITY;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        pm[i] = -INFINITY;
        pl[i] = 0.0f;
        if (tid + 128 * i < n) {
            const float *ml = a.part_ml + pa_part(first, tid + 128 * i) * 16 + r;
            pm[i] = ml[0];
            pl[i] = ml[8];
        }
    }
#pragma unroll
    for (int i = 0; i < PER; i++) m = fmaxf(m, pm[i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) s_red[warp] = m;
    if (tid == 0) s_off = 0;
    __syncthreads();
    m = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
    const float ms = m == -INFINITY ? 0.0f : m;
    float l = 0.0f;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const float w = ex2(pm[i] - ms);
        if (tid + 128 * i < n) s_w[tid + 128 * i] = w;
        l = fmaf(pl[i], w, l);
    }
    l = warp_sum(l);
    if (lane == 0) s_red2[warp] = l;
    __syncthreads();
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto add = [&](const float4 &t, float w) {
        acc.x = fmaf(t.x, w, acc.x);
        acc.y = fmaf(t.y, w, acc.y);
        acc.z = fmaf(t.z, w, acc.z);
        acc.w = fmaf(t.w, w, acc.w);
    };
#pragma unroll
    for (int i = 0; i < EARLY; i++)
        if (grp + i * GROUPS < n) add(v[i], s_w[grp + i * GROUPS]);
#pragma unroll 8
    for (uint32_t p = grp + EARLY * GROUPS; p < n; p += GROUPS) add(sums(p), s_w[p]);
    s_o[tid] = acc;
    __syncthreads();
    if (grp == 0) {
        l = (s_red2[0] + s_red2[1]) + (s_red2[2] + s_red2[3]);
#pragma unroll
        for (int i = 1; i < GROUPS; i++) add(s_o[i * LANES + x], 1.0f);
        const float inv = l > 0.0f ? __fdiv_rn(1.0f, l) : (l == 0.0f ? 0.0f : l);
        float *dst = a.out + (uint64_t)(q0 + R / a.group) * a.out_stride + (uint64_t)(kh * a.group + R % a.group) * HD + 4 * x;
        *reinterpret_cast<float4 *>(dst) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
        if (PROMPT && (acc.x - acc.x) + (acc.y - acc.y) + (acc.z - acc.z) + (acc.w - acc.w) + (l - l) != 0.0f) s_off = 1;
    }
    if (PROMPT) {
        __syncthreads();
        if (s_off && warp == 0) slow_row<HD>(a, s, kh, R, 0, HD);
    }
}

}  // namespace lt
