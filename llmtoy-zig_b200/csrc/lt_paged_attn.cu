// lt_paged_attn.cu — attention over a paged cache: one new token per sequence,
// and (prompts over f32 caches, a few tokens) several.
//
// For query row r = (token, head) at position i and the visible keys j:
//   s_j = score(q_r . k_j)  (scale, cap, distance bias: score_log2)
//   out_r = sum_j 2^(s_j - m) v_j / sum_j 2^(s_j - m),  m = max_j s_j
// in one pass over the keys with the running maximum m and sum l; rows that see
// no key give zero.  With `mass`, sum_r of the normalised weights is added to
// mass[kv head][j].
//
// Bound: memory (K and V are read once per 8 query heads of a KV head).
// - Work is (sequence, KV head, 8 rows) x tiles of the sequence's keys, counted
//   through one after the other (a unit's start counts as kUnitCost tiles more:
//   its queries, its merge, its output); every CTA takes an equal share of the count,
//   wherever it begins and ends, so lengths may differ as they like.  A unit
//   that several CTAs share leaves partial (m, l, sum) records, which
//   k_paged_finish adds up in CTA order: the result does not depend on timing.
// - Each warp owns 16 keys of a tile (8 for f32 caches) and a ring of kStages
//   such blocks in shared memory, filled by 16-byte asynchronous copies; rows sit
//   at padded pitches so that matrix loads meet no bank conflict.
// - The products run on the tensor cores without losing the f32 queries: a row
//   goes in as two f16 terms (22 bits) in rows r and r + 8 of a 16-row
//   operand, and so do the softmax weights; the two halves of the accumulator
//   add up to the f32 product.  f32 caches use tf32 the same way, with K and V
//   split into two terms as well.  A query row is scaled by a power of two so
//   that its f16 terms neither overflow nor vanish.
//
// One B200: 64 sequences of 200 to 8192 positions, 32/4 heads of 128, f16 (289
// MB): 57 to 61 us, 5.0 TB/s; one sequence of 130001 with weights accumulated (270 MB):
// 67 us, the main kernel about 55 of it, the second about 11; one window of 1024
// over an f32 cache, 16/8 heads of 256: 15 us, three dependent round trips to memory
// and two launches.  Two stages with 12 warps per SM instead of three with 8: 89 us
// for the 64 sequences.
#include "lt_paged_walk.cuh"

namespace lt {

constexpr uint32_t kMassKeys = 512;

template <int HD, bool F16>
struct PaShape {
    static constexpr int KB = F16 ? 16 : 8;                 // keys per warp and tile
    static constexpr int TILE = KB * kPaWarps;
    static constexpr int ROW = HD * (F16 ? 2 : 4);          // bytes
    static constexpr int KP = ROW + (F16 ? 16 : 64), VP = ROW + 16;
    static constexpr int BLOCK = KB * (KP + VP);
    static constexpr int STAGES = 3;
    static constexpr int QSTEPS = F16 ? HD / 16 : HD / 8;   // k-steps of 512-byte operand fragments
    static constexpr int RING = BLOCK * STAGES * kPaWarps;
    static constexpr int QBYTES = QSTEPS * 512;
    static constexpr int MERGE = 2 * kPaRows * (HD + 2) * 4;
    static constexpr int UNION = QBYTES > MERGE ? QBYTES : MERGE;
    static constexpr int SMEM = RING + UNION + 16 * 8 * kPaWarps + 64;
    static constexpr int CTAS = HD == 256 ? 1 : HD == 128 ? 2 : 3;
};

// PLAIN: neither cap nor distance bias.
template <int HD, bool F16, bool PROMPT, bool PLAIN>
__global__ void __launch_bounds__(kPaThreads, PaShape<HD, F16>::CTAS) k_paged_attn(const __grid_constant__ PagedAttnArgs a) {
    using S = PaShape<HD, F16>;
    constexpr int KB = S::KB, TILE = S::TILE, NB = HD / 8;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t s_scan[kPaWarps];
    __shared__ uint64_t s_rem;
    __shared__ uint32_t s_seq;
    __shared__ PaSeq s_q;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, j4 = lane & 3;
    uint8_t *ring = smem + warp * (S::BLOCK * S::STAGES);
    uint8_t *qm = smem + S::RING;  // query fragments, then the merge records
    uint64_t *offs = reinterpret_cast<uint64_t *>(smem + S::RING + S::UNION) + warp * 16;
    float *rowf = reinterpret_cast<float *>(smem + S::RING + S::UNION + 16 * 8 * kPaWarps);
    const uint32_t ring_u = smem_u32(ring), qm_u = smem_u32(qm);
    const uint32_t c = blockIdx.x;
    pdl_launch_dependents();
    // Lengths, page table and queries towards L2, and their translations towards this SM, while the
    // kernel before still runs (only hints: the values are read after the wait).
    {
        const uint64_t line = ((uint64_t)c * kPaThreads + tid) * 32, entries = (uint64_t)a.n_seq * a.kv.max_pages;
        if (line < entries) prefetch_l2(a.table + line);
        if (tid == 0) prefetch_l2(a.table + (c < entries ? c : 0));
        if (tid < 32 && tid * 32 < a.n_seq) prefetch_l2(a.lens + tid * 32);
        if (tid == 32) prefetch_l2(a.q);
        if (tid == 64) prefetch_l2(a.kv.k);
        if (tid == 96) prefetch_l2(a.kv.v);
    }
    pdl_wait();

    // the tiles of all sequences, and where this CTA's share begins
    const uint32_t per = (a.n_seq + kPaThreads - 1) / kPaThreads;
    const uint32_t sa = min(a.n_seq, tid * per), sb = min(a.n_seq, sa + per);
    uint64_t mine = 0;
#pragma unroll 4
    for (uint32_t s = sa; s < sb; s++) {
        const PaSeq q = pa_seq<PROMPT>(a, s, TILE, c == 0);
        mine += (uint64_t)q.blocks * a.kv.n_kv * q.cost();
    }
    uint64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
    }
    if (lane == 31) s_scan[warp] = incl;
    __syncthreads();
    uint64_t T = 0, before = incl - mine;
#pragma unroll
    for (int w = 0; w < kPaWarps; w++) {
        if (w < warp) before += s_scan[w];
        T += s_scan[w];
    }
    // no more CTAs than tiles, so that every CTA of a unit leaves a record
    const uint32_t G = (uint32_t)min((uint64_t)gridDim.x, T);
    if (c >= G) return;
    const PaShare share(T, G);
    uint64_t f0 = share.start(c);
    const uint64_t f1 = share.start(c + 1);
    if (f0 >= before && f0 < before + mine) {
        uint64_t rem = f0 - before;
        for (uint32_t s = sa; s < sb; s++) {
            const PaSeq q = pa_seq<PROMPT>(a, s, TILE, false);
            const uint64_t w = (uint64_t)q.blocks * a.kv.n_kv * q.cost();
            if (rem < w) {
                s_seq = s;
                s_rem = rem;
                s_q = q;
                break;
            }
            rem -= w;
        }
    }
    __syncthreads();
    PaWalk<PROMPT> cw, lw;  // the compute walk and the copies ahead of it
    cw.s = s_seq;
    cw.q = s_q;
    cw.unit = (uint32_t)div_small(s_rem, cw.q.cost());
    cw.tile = (uint32_t)(s_rem - (uint64_t)cw.unit * cw.q.cost());
    if (cw.tile >= cw.q.tiles) {  // in what the unit before costs beyond its tiles
        f0 += cw.q.cost() - cw.tile;
        if (f0 >= f1) return;
        cw.template next_unit<TILE>(a);
    } else {
        cw.set_unit(a);
    }
    lw = cw;
    uint64_t lf = f0;  // lw's place in the count

    // a unit's queries: warp w takes rows 2 w and 2 w + 1; the first unit's come while K and V are looked up
    float qv[2][HD / 32];
    auto load_q = [&]() {
        const uint32_t rows = min((uint32_t)kPaRows, cw.q.nq * a.group - cw.rb * kPaRows);
#pragma unroll
        for (int rr = 0; rr < 2; rr++) {
            const uint32_t r = warp * 2 + rr, R = cw.rb * kPaRows + r;
            const float *src = a.q + (uint64_t)(cw.q.q0 + R / a.group) * a.q_stride + (uint64_t)(cw.kh * a.group + R % a.group) * HD;
#pragma unroll
            for (int e = 0; e < HD / 64; e++) {
                const float2 t = r < rows ? *reinterpret_cast<const float2 *>(src + 64 * e + 2 * lane) : make_float2(0.0f, 0.0f);
                qv[rr][2 * e] = t.x;
                qv[rr][2 * e + 1] = t.y;
            }
        }
    };
    load_q();

    // The block to copy next: where whole blocks lie within pages, its page is looked up
    // once and its rows are a stride apart; else lane r < KB looks up row r.
    constexpr int CH = S::ROW / 16, STEP = 32 / (CH < 32 ? CH : 32);
    const bool in_page = a.kv.page_size % KB == 0;
    const int row0 = CH < 32 ? lane / CH : 0, col0 = CH < 32 ? lane % CH : lane;
    const uint64_t lane_off = (uint64_t)row0 * a.kv.slot_stride + col0 * 16, step_off = STEP * a.kv.slot_stride;
    struct Job {
        uint32_t page, key, kh, lo, hi;  // key 0xffffffff: only zeros
        bool there;
    };
    auto look = [&]() {
        Job j = {a.kv.n_pages, lw.base + lw.tile * TILE + warp * KB + (in_page ? 0 : lane), lw.kh, lw.lo, lw.hi, true};
        if (in_page ? j.key < j.hi && j.key + KB > j.lo : lane < KB && j.key < j.hi && j.key >= j.lo)
            j.page = a.table[(uint64_t)lw.s * a.kv.max_pages + page_of(a.kv, j.key)];
        else
            j.key = 0xffffffffu;
        return j;
    };
    auto copy = [&](const Job &j, int stage) {
        const uint32_t key = j.key;
        bool take = key != 0xffffffffu;
        if (take && j.page >= a.kv.n_pages) {
            take = false;
            atomicExch(a.err, DEV_ERR_BAD_INDEX);
        }
        const uint32_t kdst = ring_u + stage * S::BLOCK + row0 * S::KP + col0 * 16;
        const uint32_t vdst = ring_u + stage * S::BLOCK + KB * S::KP + row0 * S::VP + col0 * 16;
        // (one short body for whole and partial blocks: this code runs few times, and its fetching shows)
        if (in_page) {
            const uint64_t o = take ? paged_offset(a.kv, j.page, key, j.kh) + lane_off : 0;
            const uint8_t *pk = a.kv.k + o, *pv = a.kv.v + o;
            const uint32_t from = take ? max(j.lo, key) - key : 0, to = take ? min(j.hi - key, (uint32_t)KB) : 0;
#pragma unroll
            for (int r = 0; r < KB; r += STEP) {
                const bool t = r + row0 >= from && r + row0 < to;
#pragma unroll
                for (int x = 0; x < CH; x += 32) {
                    cp_async16(kdst + r * S::KP + x * 16, pk + x * 16, t);
                    cp_async16(vdst + r * S::VP + x * 16, pv + x * 16, t);
                }
                pk += step_off;
                pv += step_off;
            }
            return;
        }
        __syncwarp();
        if (lane < KB) offs[lane] = take ? paged_offset(a.kv, j.page, key, j.kh) : ~0ull;
        __syncwarp();
#pragma unroll 1
        for (int r = 0; r < KB; r += STEP) {
            const uint64_t o = offs[r + row0];
            const bool t = o != ~0ull;
#pragma unroll
            for (int x = 0; x < CH; x += 32) {
                const uint64_t src = t ? o + (x + col0) * 16 : 0;
                cp_async16(kdst + r * S::KP + x * 16, a.kv.k + src, t);
                cp_async16(vdst + r * S::VP + x * 16, a.kv.v + src, t);
            }
        }
    };
    // all pages of the first blocks are looked up before the first copy waits for its own
    Job jobs[S::STAGES];
    auto look_next = [&](Job &j) {
        j.there = lf < f1;
        if (!j.there) return;
        j = look();
        if (++lw.tile < lw.q.tiles) {
            lf++;
        } else {
            lf += 1 + kUnitCost;
            if (lf < f1) lw.template next_unit<TILE>(a);
        }
    };
#pragma unroll
    for (int st = 0; st < S::STAGES; st++) look_next(jobs[st]);
#pragma unroll
    for (int st = 0; st < S::STAGES - 1; st++) {
        if (jobs[st].there) copy(jobs[st], st);
        cp_async_commit();
    }
    Job job = jobs[S::STAGES - 1];

    uint64_t f = f0;
    int stage = 0;
    while (f < f1) {
        // ── one segment: this CTA's tiles of one unit ──
        const uint32_t seg = (uint32_t)min((uint64_t)(cw.q.tiles - cw.tile), f1 - f);
        const uint64_t unit_f0 = f - cw.tile;
        const uint32_t rows = min((uint32_t)kPaRows, cw.q.nq * a.group - cw.rb * kPaRows);
        // queries to operand fragments
#pragma unroll
        for (int rr = 0; rr < 2; rr++) {
            const uint32_t r = warp * 2 + rr;
            float(&v)[HD / 32] = qv[rr];
            float top = 0.0f;
#pragma unroll
            for (int e = 0; e < HD / 32; e++) top = fmaxf(top, fabsf(v[e]));
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            // the largest element lands in [2^8, 2^9)
            float up = 1.0f;
            if (F16 && top > 0.0f && top < INFINITY) {
                const int ex = min(max(8 - (int)(__float_as_uint(top) >> 23) + 127, -126), 126);
                up = __uint_as_float((uint32_t)(ex + 127) << 23);
            }
            if (lane == 0) rowf[r] = (a.softcap != 0.0f ? a.scale / a.softcap : a.scale * 1.4426950408889634f) / up;
#pragma unroll
            for (int e = 0; e < HD / 64; e++) {
                const uint32_t k = 64 * e + 2 * lane;
                if (F16) {
                    uint32_t hi, lo;
                    split_f16x2(v[2 * e] * up, v[2 * e + 1] * up, hi, lo);
                    const uint32_t at = (k / 16) * 512 + (r * 4 + (k % 8) / 2) * 16 + ((k % 16) / 8) * 8;
                    *reinterpret_cast<uint2 *>(qm + at) = make_uint2(hi, lo);
                } else {
                    // element 16 i + 4 j + c: fragment 2 i + c / 2, lane 4 r + j, registers 2 (c % 2) and + 1
#pragma unroll
                    for (int d = 0; d < 2; d++) {
                        uint32_t hi, lo;
                        split_tf32(v[2 * e + d], hi, lo);
                        const uint32_t kk = k + d, cc = kk % 4;
                        const uint32_t at = (2 * (kk / 16) + cc / 2) * 512 + (r * 4 + (kk % 16) / 4) * 16 + (cc & 1) * 8;
                        *reinterpret_cast<uint2 *>(qm + at) = make_uint2(hi, lo);
                    }
                }
            }
        }
        __syncthreads();
        constexpr bool QREG = F16 && HD <= 128;
        uint32_t qf[QREG ? S::QSTEPS : 1][4];
        if constexpr (QREG) {
#pragma unroll
            for (int i = 0; i < S::QSTEPS; i++) {
                const float4 t = lds128(qm_u + i * 512 + lane * 16);
                qf[i][0] = __float_as_uint(t.x), qf[i][1] = __float_as_uint(t.y);
                qf[i][2] = __float_as_uint(t.z), qf[i][3] = __float_as_uint(t.w);
            }
        }
        // this thread's row g: factor, bias slope, what it sees
        const uint32_t R = cw.rb * kPaRows + g;
        const float rf = rowf[g];
        const uint32_t head = cw.kh * a.group + R % a.group;
        const float slope = a.slopes && (uint32_t)g < rows ? a.slopes[head] : 0.0f;
        // positions are 32 bits wide here, and so are their differences: a length is at most 2^30, and a query that
        // far before position 0 is clamped
        const int row_i = (int)max((int64_t)cw.q.len - cw.q.nq + R / a.group, -((int64_t)1 << 30));
        int row_lo = cw.q.lo, row_hi = cw.q.len;
        uint32_t my_doc = 0;
        const uint32_t *docs = nullptr;
        if (PROMPT) {
            if (a.causal) {
                row_hi = min(row_i + 1, (int)cw.q.len);
                if (a.prefix) row_hi = max(row_hi, (int)min(a.prefix[cw.s], cw.q.len));  // any prefix up to 2^32 - 1
            }
            row_lo = a.window ? (int)max((int64_t)0, (int64_t)row_i - a.window + 1) : 0;
            if (a.docs) {
                docs = a.docs + (uint64_t)cw.s * a.doc_stride;
                if ((uint32_t)g < rows && row_i >= 0)
                    my_doc = docs[row_i];
                else
                    row_hi = 0;
            }
        }
        // Sums in registers; each block's product is computed from zero and added here: the tensor
        // core truncates where it accumulates, and so do long chains of products (hence C chains below).
        float o[NB][2];
#pragma unroll
        for (int n = 0; n < NB; n++) o[n][0] = o[n][1] = 0.0f;
        float m = -INFINITY, l = 0.0f;

        for (uint32_t it = 0; it < seg; it++) {
            cp_async_wait<S::STAGES - 2>();
            __syncwarp();
            const uint32_t k0 = cw.base + cw.tile * TILE + warp * KB;  // the block's first position
            if (k0 < cw.hi && k0 + KB > cw.lo) {
                const uint32_t kb = ring_u + stage * S::BLOCK, vb = kb + KB * S::KP;
                constexpr int NS = KB / 4;  // scores per thread: keys k0 + 8 (n / 2) + 2 j4 + n % 2
                float sc[NS];
                if constexpr (F16) {
                    constexpr int C = HD == 256 ? 4 : 2;
                    float s0[C][4] = {}, s1[C][4] = {};
                    const uint32_t ka = kb + ((lane >> 4) * 8 + (lane & 7)) * S::KP + ((lane >> 3) & 1) * 16;
#pragma unroll
                    for (int i = 0; i < S::QSTEPS; i++) {
                        uint32_t b[4];
                        ldsm4(b, ka + i * 32);
                        uint32_t qa[4];
                        if constexpr (QREG) {
                            qa[0] = qf[i][0], qa[1] = qf[i][1], qa[2] = qf[i][2], qa[3] = qf[i][3];
                        } else {
                            const float4 t = lds128(qm_u + i * 512 + lane * 16);
                            qa[0] = __float_as_uint(t.x), qa[1] = __float_as_uint(t.y);
                            qa[2] = __float_as_uint(t.z), qa[3] = __float_as_uint(t.w);
                        }
                        mma_f16(s0[i % C], qa, b[0], b[1]);
                        mma_f16(s1[i % C], qa, b[2], b[3]);
                    }
#pragma unroll
                    for (int n = 0; n < NS; n++) {
                        const float(&x)[C][4] = n < 2 ? s0 : s1;
                        sc[n] = x[0][n & 1] + x[1][n & 1];
                        float lo = x[0][2 + (n & 1)] + x[1][2 + (n & 1)];
                        if (C == 4) {
                            sc[n] += x[C - 2][n & 1] + x[C - 1][n & 1];
                            lo += x[C - 2][2 + (n & 1)] + x[C - 1][2 + (n & 1)];
                        }
                        sc[n] += lo;
                    }
                } else {
                    constexpr int C = 2;  // chains: 4 of the high terms of K, 2 of the low ones
                    float s0[2 * C][4] = {}, s1[C][4] = {};
                    const uint32_t ka = kb + g * S::KP + j4 * 16;
#pragma unroll 4
                    for (int i = 0; i < HD / 16; i++) {
                        const float4 t = lds128(ka + i * 64);
                        const float kv4[4] = {t.x, t.y, t.z, t.w};
                        uint32_t bh[4], bl[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) split_tf32(kv4[e], bh[e], bl[e]);
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const float4 u = lds128(qm_u + (2 * i + e) * 512 + lane * 16);
                            const uint32_t qa[4] = {__float_as_uint(u.x), __float_as_uint(u.y), __float_as_uint(u.z),
                                                    __float_as_uint(u.w)};
                            mma_tf32(s0[i % (2 * C)], qa, bh[2 * e], bh[2 * e + 1]);
                            mma_tf32(s1[i % C], qa, bl[2 * e], bl[2 * e + 1]);
                        }
                    }
#pragma unroll
                    for (int n = 0; n < 2; n++) {
                        float hi = 0.0f, lo = 0.0f;
#pragma unroll
                        for (int c = 0; c < 2 * C; c++) hi += s0[c][n], lo += s0[c][2 + n];
#pragma unroll
                        for (int c = 0; c < C; c++) lo += s1[c][n] + s1[c][2 + n];
                        sc[n] = hi + lo;
                    }
                }
                float top = -INFINITY;
                const bool whole = !PROMPT && k0 >= cw.lo && k0 + KB <= cw.hi;
                // distance to this thread's first key; the positions alone may need more than a float's 24 bits
                const float dist = (float)(row_i - (int)(k0 + 2 * j4));
#pragma unroll
                for (int n = 0; n < NS; n++) {
                    const int j = (int)k0 + 8 * (n / 2) + 2 * j4 + (n & 1);
                    sc[n] = PLAIN ? sc[n] * rf : score_log2(sc[n], rf, a.softcap, slope, fabsf(dist - (float)(8 * (n / 2) + (n & 1))));
                    if (PROMPT) {
                        bool seen = j >= row_lo && j < row_hi;
                        if (docs && seen) seen = docs[j] == my_doc;
                        if (!seen) sc[n] = -INFINITY;
                    } else {
                        const bool seen = whole || (j >= row_lo && j < row_hi);
                        if (a.mass && seen && (uint32_t)g < rows)
                            a.scores[((uint64_t)cw.s * a.n_heads + head) * a.score_stride + j] = sc[n];
                        if (!seen) sc[n] = -INFINITY;
                    }
                    top = fmaxf(top, sc[n]);
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float mn = fmaxf(m, top);
                const float al = mn > m ? ex2(m - mn) : 1.0f;  // m = -inf: 0
                l *= al;
                m = mn;
                // weights scaled by 2^10 so that small ones keep their f16 bits; l carries the same factor
                const float base = m == -INFINITY ? 0.0f : m - (F16 ? 10.0f : 0.0f);
#pragma unroll
                for (int n = 0; n < NS; n++) {
                    sc[n] = ex2(sc[n] - base);
                    l += sc[n];
                }
                if constexpr (F16) {
                    uint32_t pa[4];
                    split_f16x2(sc[0], sc[1], pa[0], pa[1]);
                    split_f16x2(sc[2], sc[3], pa[2], pa[3]);
                    const uint32_t va = vb + (((lane >> 3) & 1) * 8 + (lane & 7)) * S::VP + (lane >> 4) * 16;
#pragma unroll
                    for (int n = 0; n < NB; n += 2) {
                        uint32_t b[4];
                        ldsm4_t(b, va + n * 16);
                        float c0[4] = {}, c1[4] = {};
                        mma_f16(c0, pa, b[0], b[1]);
                        mma_f16(c1, pa, b[2], b[3]);
                        o[n][0] = fmaf(o[n][0], al, c0[0] + c0[2]);
                        o[n][1] = fmaf(o[n][1], al, c0[1] + c0[3]);
                        o[n + 1][0] = fmaf(o[n + 1][0], al, c1[0] + c1[2]);
                        o[n + 1][1] = fmaf(o[n + 1][1], al, c1[1] + c1[3]);
                    }
                } else {
                    // operand index j4 is key 2 j4, index j4 + 4 key 2 j4 + 1; column g of product c is dim 32 i + 4 g + c
                    uint32_t pa[4];
                    split_tf32(sc[0], pa[0], pa[1]);
                    split_tf32(sc[1], pa[2], pa[3]);
                    const uint32_t va = vb + 2 * j4 * S::VP + g * 16;
#pragma unroll
                    for (int i = 0; i < HD / 32; i++) {
                        const float4 t0 = lds128(va + i * 128), t1 = lds128(va + S::VP + i * 128);
                        const float x0[4] = {t0.x, t0.y, t0.z, t0.w}, x1[4] = {t1.x, t1.y, t1.z, t1.w};
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            uint32_t h0, l0, h1, l1;
                            split_tf32(x0[e], h0, l0);
                            split_tf32(x1[e], h1, l1);
                            float c0[4] = {};
                            mma_tf32(c0, pa, l0, l1);
                            mma_tf32(c0, pa, h0, h1);
                            o[4 * i + e][0] = fmaf(o[4 * i + e][0], al, c0[0] + c0[2]);
                            o[4 * i + e][1] = fmaf(o[4 * i + e][1], al, c0[1] + c0[3]);
                        }
                    }
                }
            }
            __syncwarp();
            int fill = stage + S::STAGES - 1;
            if (fill >= S::STAGES) fill -= S::STAGES;
            if (job.there) {
                copy(job, fill);
                look_next(job);
            }
            cp_async_commit();
            if (++stage == S::STAGES) stage = 0;
            if (it + 1 < seg) cw.tile++;
        }

        // ── merge the warps: 2 and 3 into 0 and 1, then 1 into 0 ──
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        auto dim = [&](int n, int e) { return F16 ? 8 * n + 2 * j4 + e : 32 * (n / 4) + 8 * j4 + 4 * e + n % 4; };
        __syncthreads();  // every warp is done with the query fragments
#pragma unroll
        for (int half = kPaWarps / 2; half >= 1; half /= 2) {
            float *rec = reinterpret_cast<float *>(qm) + (warp % half) * kPaRows * (HD + 2) + g * (HD + 2);
            if (warp >= half && warp < 2 * half) {
#pragma unroll
                for (int n = 0; n < NB; n++) {
                    rec[dim(n, 0)] = o[n][0];
                    rec[dim(n, 1)] = o[n][1];
                }
                if (j4 == 0) {
                    rec[HD] = m;
                    rec[HD + 1] = l;
                }
            }
            __syncthreads();
            if (warp < half) {
                const float m2 = rec[HD], mn = fmaxf(m, m2);
                const float w1 = m == -INFINITY ? 0.0f : ex2(m - mn), w2 = m2 == -INFINITY ? 0.0f : ex2(m2 - mn);
                l = l * w1 + rec[HD + 1] * w2;
#pragma unroll
                for (int n = 0; n < NB; n++) {
                    o[n][0] = o[n][0] * w1 + rec[dim(n, 0)] * w2;
                    o[n][1] = o[n][1] * w1 + rec[dim(n, 1)] * w2;
                }
                m = mn;
            }
            __syncthreads();
        }
        if (warp == 0) {
            const uint32_t first = share.owner(unit_f0), last = share.owner(unit_f0 + cw.q.tiles - 1);
            const uint64_t u = pa_unit(a, cw.s, cw.kh, cw.rb);
            if (unit_f0 == f && lane == 0) {
                a.unit_info[2 * u] = first;
                a.unit_info[2 * u + 1] = last - first + 1;
            }
            if (first == last) {
                const float inv = l > 0.0f ? __fdiv_rn(1.0f, l) : (l == 0.0f ? 0.0f : l);
                float off = l - l;  // not 0 where the row is not finite
#pragma unroll
                for (int n = 0; n < NB; n++) off += (o[n][0] - o[n][0]) + (o[n][1] - o[n][1]);
                off += __shfl_xor_sync(0xffffffffu, off, 1);
                off += __shfl_xor_sync(0xffffffffu, off, 2);
                if ((uint32_t)g < rows && (!PROMPT || off == 0.0f)) {
                    float *dst = a.out + (uint64_t)(cw.q.q0 + R / a.group) * a.out_stride + (uint64_t)head * HD;
#pragma unroll
                    for (int n = 0; n < NB; n++) {
                        dst[dim(n, 0)] = o[n][0] * inv;
                        dst[dim(n, 1)] = o[n][1] * inv;
                    }
                }
                if (PROMPT) {
                    uint32_t again = __ballot_sync(0xffffffffu, (uint32_t)g < rows && off != 0.0f) & 0x11111111u;
                    for (; again; again &= again - 1)
                        slow_row<HD>(a, cw.s, cw.kh, cw.rb * kPaRows + (__ffs(again) - 1) / 4, 0, HD);
                }
                if (!PROMPT && a.mass && j4 == 0) {
                    a.unit_ml[u * 16 + g] = m;
                    a.unit_ml[u * 16 + 8 + g] = l;
                }
            } else {
                const uint64_t p = 2 * (uint64_t)c + (unit_f0 == f ? 1 : 0);
                float *dst = a.part_o + (p * kPaRows + g) * HD;
#pragma unroll
                for (int n = 0; n < NB; n++) {
                    dst[dim(n, 0)] = o[n][0];
                    dst[dim(n, 1)] = o[n][1];
                }
                if (j4 == 0) {
                    a.part_ml[p * 16 + g] = m;
                    a.part_ml[p * 16 + 8 + g] = l;
                }
            }
        }
        __syncthreads();  // the merge records are read before the next queries overwrite them
        f = unit_f0 + cw.q.cost();  // the next unit, unless this one goes on elsewhere
        if (f < f1) {
            cw.template next_unit<TILE>(a);
            load_q();  // (fetched before the merge they cost registers: 59.5 us for the 64 sequences, 57.6 without)
        }
    }
    cp_async_wait<0>();
}

// mass[s][kv head][j] += sum over the KV head's query heads of 2^(score - m) / l, for
// kMassKeys positions from j0 on; a thread's cells are its own.  m and l are those of the
// whole row, which no CTA knows before all of the unit's are done: the scores wait in
// scratch (33 MB next to 270 MB of K and V for the long sequence; K again would be 135).  The scores are on
// their way while the heads' m and l are put together, 16 threads to a head.
LT_DEVINL void pa_mass(const PagedAttnArgs &a, uint32_t s, uint32_t kh, uint32_t j0) {
    extern __shared__ float s_ml[];  // [group] maxima, [group] 1 / sum
    const PaSeq q = pa_seq<false>(a, s, 1, false);
    if (j0 >= q.len || j0 + kMassKeys <= q.lo) return;
    const int tid = threadIdx.x;
    constexpr int H = 8;
    const uint32_t j = j0 + 4 * tid;
    const float *sc = a.scores + ((uint64_t)s * a.n_heads + kh * a.group) * a.score_stride + j;
    float4 v[H];
    auto load = [&](uint32_t h0) {
#pragma unroll
        for (int h = 0; h < H; h++)
            if (j < q.len && h0 + h < a.group) v[h] = *reinterpret_cast<const float4 *>(sc + (h0 + h) * a.score_stride);
    };
    load(0);
    float *mass = a.mass + ((uint64_t)s * a.kv.n_kv + kh) * a.mass_stride + j;
    float old[4];
#pragma unroll
    for (int e = 0; e < 4; e++) old[e] = j + e >= q.lo && j + e < q.len ? mass[e] : 0.0f;
    for (uint32_t h0 = 0; h0 < a.group; h0 += 8) {  // 8 heads at once: the rows of one unit
        const uint32_t h = h0 + tid / 16, t = tid % 16;
        const uint64_t u = pa_unit(a, s, kh, h0 / kPaRows);
        const uint32_t r = tid / 16, first = a.unit_info[2 * u], n = a.unit_info[2 * u + 1];
        float m = -INFINITY, l = 0.0f;
        if (h < a.group) {
            if (n < 2) {
                if (t == 0) {
                    m = a.unit_ml[u * 16 + r];
                    l = a.unit_ml[u * 16 + 8 + r];
                }
            } else {
                for (uint32_t p0 = t; p0 < n; p0 += 16 * 8) {
                    float pm[8], pl[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const bool there = p0 + 16 * i < n;
                        const float *ml = a.part_ml + pa_part(first, there ? p0 + 16 * i : 0) * 16 + r;
                        pm[i] = there ? ml[0] : -INFINITY;
                        pl[i] = there ? ml[8] : 0.0f;
                    }
                    float mn = m;
#pragma unroll
                    for (int i = 0; i < 8; i++) mn = fmaxf(mn, pm[i]);
                    const float ms = mn == -INFINITY ? 0.0f : mn;
                    l *= ex2(m - ms);
#pragma unroll
                    for (int i = 0; i < 8; i++) l = fmaf(pl[i], ex2(pm[i] - ms), l);
                    m = mn;
                }
            }
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) {
            const float m2 = __shfl_xor_sync(0xffffffffu, m, o), l2 = __shfl_xor_sync(0xffffffffu, l, o);
            const float mn = fmaxf(m, m2), ms = mn == -INFINITY ? 0.0f : mn;
            const float x = l * ex2(m - ms), y = l2 * ex2(m2 - ms);
            l = x + y;
            m = mn;
        }
        if (t == 0 && h < a.group) {
            // the sums carry the weights' factor 2^10 on f16 caches
            s_ml[h] = m == -INFINITY ? 0.0f : m - (a.kv.f16 ? 10.0f : 0.0f);
            s_ml[a.group + h] = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);  // NaN stays, as in the output
        }
    }
    __syncthreads();
    if (j >= q.len) return;
    float w[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t h0 = 0; h0 < a.group; h0 += H) {
        if (h0) load(h0);
#pragma unroll
        for (int h = 0; h < H; h++) {
            if (h0 + h >= a.group) break;
            const float m = s_ml[h0 + h], f = s_ml[a.group + h0 + h];
            w[0] = fmaf(ex2(v[h].x - m), f, w[0]);
            w[1] = fmaf(ex2(v[h].y - m), f, w[1]);
            w[2] = fmaf(ex2(v[h].z - m), f, w[2]);
            w[3] = fmaf(ex2(v[h].w - m), f, w[3]);
        }
    }
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (j + e >= q.lo && j + e < q.len) mass[e] = old[e] + w[e];
}

// What is left when the tiles are done: rows to join, then weights to add up.
template <int HD, bool PROMPT>
__global__ void __launch_bounds__(128) k_paged_finish(const __grid_constant__ PagedAttnArgs a, uint32_t n_join) {
    pdl_launch_dependents();
    pdl_wait();
    if constexpr (PROMPT) {  // many units, few of them shared: a CTA looks at one unit
        if (a.unit_info[2 * (uint64_t)blockIdx.x + 1] < 2) return;
        for (uint32_t r = 0; r < kPaRows; r++) {
            pa_join_row<HD, PROMPT>(a, blockIdx.x, r);
            __syncthreads();
        }
    } else if (blockIdx.x < n_join) {  // few units: a CTA does one row
        pa_join_row<HD, PROMPT>(a, blockIdx.x / kPaRows, blockIdx.x % kPaRows);
    } else {
        const uint32_t b = blockIdx.x - n_join, steps = (a.max_len + kMassKeys - 1) / kMassKeys;
        pa_mass(a, b / steps / a.kv.n_kv, b / steps % a.kv.n_kv, b % steps * kMassKeys);
    }
}

namespace {

size_t up256(size_t v) { return (v + 255) & ~(size_t)255; }

struct PaScratch {
    size_t part_o, part_ml, unit_ml, unit_info, scores, total;
};
PaScratch pa_layout(const PagedAttnArgs &a, uint32_t G) {
    const uint64_t rows = (uint64_t)(a.cu ? a.max_q : 1) * a.group;
    const uint64_t units = (uint64_t)a.n_seq * a.kv.n_kv * ((rows + kPaRows - 1) / kPaRows);
    PaScratch s;
    size_t off = 0;
    auto take = [&](size_t b) {
        const size_t at = off;
        off += up256(b);
        return at;
    };
    s.part_o = take((size_t)2 * G * kPaRows * a.kv.hd * 4);
    s.part_ml = take((size_t)2 * G * 16 * 4);
    s.unit_info = take(units * 8);
    s.unit_ml = take(a.mass ? units * 64 : 0);
    s.scores = take(a.mass ? (size_t)a.n_seq * a.n_heads * ((a.max_len + 3) & ~3u) * 4 : 0);
    s.total = off;
    return s;
}

uint32_t pa_grid(uint32_t hd, int num_sms) {
    return min((uint32_t)num_sms * (hd == 256 ? 1 : hd == 128 ? 2 : 3), kPaMaxParts);
}

template <int HD, bool F16, bool PROMPT>
cudaError_t pa_launch(const LaunchCfg &c, const PagedAttnArgs &a, uint64_t units) {
    const char *label = PROMPT ? "paged_attn_rows" : "paged_attn";
    const dim3 grid(pa_grid(HD, c.num_sms));
    cudaError_t e;
    if (a.softcap == 0.0f && !a.slopes)
        e = launch_k(c, label, k_paged_attn<HD, F16, PROMPT, true>, grid, dim3(kPaThreads), PaShape<HD, F16>::SMEM, a);
    else
        e = launch_k(c, label, k_paged_attn<HD, F16, PROMPT, false>, grid, dim3(kPaThreads), PaShape<HD, F16>::SMEM, a);
    if (e != cudaSuccess) return e;
    const uint64_t join = PROMPT ? units : units * kPaRows;
    const uint64_t mass = a.mass ? (uint64_t)((a.max_len + kMassKeys - 1) / kMassKeys) * a.kv.n_kv * a.n_seq : 0;
    if (join + mass > 0x7fffffffull) return cudaErrorInvalidValue;
    return launch_k(c, "paged_finish", k_paged_finish<HD, PROMPT>, dim3((uint32_t)(join + mass)), dim3(128),
                    a.mass ? 2 * a.group * sizeof(float) : 0, a, (uint32_t)join);
}

template <bool F16, bool PROMPT>
cudaError_t pa_launch_hd(const LaunchCfg &c, const PagedAttnArgs &a, uint64_t units) {
    switch (a.kv.hd) {
    case 64: return pa_launch<64, F16, PROMPT>(c, a, units);
    case 128: return pa_launch<128, F16, PROMPT>(c, a, units);
    case 256: return pa_launch<256, F16, PROMPT>(c, a, units);
    default: return cudaErrorInvalidValue;
    }
}

}  // namespace

size_t paged_attn_scratch(const PagedAttnArgs &a, int num_sms) { return pa_layout(a, pa_grid(a.kv.hd, num_sms)).total; }

cudaError_t launch_paged_attn(const LaunchCfg &c, PagedAttnArgs a, uint8_t *scratch) {
    const PaScratch s = pa_layout(a, pa_grid(a.kv.hd, c.num_sms));
    a.part_o = (float *)(scratch + s.part_o);
    a.part_ml = (float *)(scratch + s.part_ml);
    a.unit_info = (uint32_t *)(scratch + s.unit_info);
    a.unit_ml = (float *)(scratch + s.unit_ml);
    a.scores = (float *)(scratch + s.scores);
    a.score_stride = (a.max_len + 3) & ~3u;
    a.err = c.dev_err;
    const uint64_t rows = (uint64_t)(a.cu ? a.max_q : 1) * a.group;
    a.row_blocks = (uint32_t)((rows + kPaRows - 1) / kPaRows);
    const uint64_t units = (uint64_t)a.n_seq * a.kv.n_kv * a.row_blocks;
    if (a.cu) return a.kv.f16 ? pa_launch_hd<true, true>(c, a, units) : pa_launch_hd<false, true>(c, a, units);
    return a.kv.f16 ? pa_launch_hd<true, false>(c, a, units) : pa_launch_hd<false, false>(c, a, units);
}

}  // namespace lt
