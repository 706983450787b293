// lt_paged_prompt.cu — attention of many queries per sequence over a paged f16
// cache, on the 5th-generation tensor cores.
//
// Same formula as lt_paged_attn.cu.  Rows are (token, head of the KV head's
// group) pairs, so all the heads that read a KV head share its tiles.  The f32
// queries enter as two f16 planes (scaled per row by a power of two), the
// softmax weights too: S = Qlo K^T + Qhi K^T and O = Plo V + Phi V, 22 bits of
// each, twice the multiply-adds of a 16-bit product.  O of each tile is added up
// in registers: the tensor core's accumulator truncates, and over thousands of
// keys that would show.
//
// A CTA (one per SM) works on 256 rows (128 for head_dim 256):
//   warps 0-3, 4-7   softmax of row tile 0 and 1, a thread per row.  head_dim 256:
//                    both on the one row tile, each half of the keys and of O.
//   warp 8           issues the MMAs
//   warps 9-11       bring K and V tiles from their pages (16-byte asynchronous
//                    copies into 128-byte-swizzled rows) into a ring of stages
// While one tile's softmax runs, the tensor cores work for the other: per tile
// of keys the MMA order is PV0 QK0' PV1 QK1' (' the next keys).  S and P share
// their columns of tensor memory; P lies as it is read: per 32 keys 16 columns
// of high terms, then 16 of low ones, over the 32 columns of S they come from.
#include "lt_paged.cuh"
#include "lt_umma.cuh"

namespace lt {

constexpr int kPpThreads = 384, kPpProducers = 96;
constexpr int kPpSkipTiles = 4096;  // tiles whose documents are looked at beforehand

template <int HD>
struct PpShape {
    static constexpr int TILES = HD == 256 ? 1 : 2;       // row tiles of 128
    static constexpr int ROWS = TILES * 128;
    static constexpr int KT = HD == 256 ? 64 : 128;       // keys per tile
    static constexpr int NBLK = HD / 64;                  // 128-byte-wide column blocks
    static constexpr int STAGE = KT * HD * 2;
    static constexpr int STAGES = HD == 64 ? 6 : 3;
    static constexpr int DOCS = HD == 64 ? 4 : 2;         // document-number buffers
    static constexpr int QPLANE = 128 * HD * 2;
    static constexpr int Q_BYTES = TILES * 2 * QPLANE;
    static constexpr int OFF_RING = Q_BYTES;
    static constexpr int OFF_OFFS = OFF_RING + STAGES * STAGE;
    static constexpr int OFF_DOCS = OFF_OFFS + KT * 8;
    static constexpr int OFF_SKIP = OFF_DOCS + DOCS * KT * 4;
    static constexpr int OFF_BARS = OFF_SKIP + kPpSkipTiles / 8;
    static constexpr int SMEM = OFF_BARS + 256;
    static constexpr uint32_t S_COL(int i) { return (HD == 256 ? 64 : 128) * i; }
    static constexpr uint32_t O_COL(int i) { return 256 + (HD == 256 ? 0 : 128 * i); }
    static constexpr uint32_t X_COL = 128;                // head_dim 256: the halves' row maxima and sums
};

// 32 consecutive TMEM columns of this thread's lane.
LT_DEVINL void tmem_st32(uint32_t taddr, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
        "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
        "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}
LT_DEVINL void tmem_st1(uint32_t taddr, float v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(taddr), "r"(__float_as_uint(v)) : "memory");
}
LT_DEVINL float tmem_ld1(uint32_t taddr) {
    uint32_t v;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(v) : "r"(taddr));
    return __uint_as_float(v);
}
LT_DEVINL void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// D[tmem] (+)= A[tmem] * B, issued by one thread; A: 128 lanes, two f16 of K per column.
LT_DEVINL void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate));
}
// Operand whose rows run along K (V: one row of 64 N values per key): 64-wide
// blocks of N lie `block` bytes apart, groups of 8 keys 1024 bytes.
LT_DEVINL uint64_t umma_desc_sw128_mn(uint32_t saddr, uint32_t block) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(block >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
constexpr uint32_t kUmmaBTransposed = 1u << 16;  // instruction descriptor: B along N

LT_DEVINL void mbar_arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
template <int N>
LT_DEVINL void regs_inc() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
LT_DEVINL void regs_dec() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int ID, int N>
LT_DEVINL void named_sync() {
    asm volatile("bar.sync %0, %1;" ::"n"(ID), "n"(N) : "memory");
}

// What one row sees and how it scores.
struct PpRow {
    const float *q;      // nullptr: no such row
    int64_t i;           // position
    int64_t lo, hi;      // keys [lo, hi), document aside
    uint32_t doc;
    float slope;
};

LT_DEVINL float pp_kv(const uint8_t *p, uint32_t d) { return __half2float(reinterpret_cast<const __half *>(p)[d]); }

// The row by itself, key by key, masked keys never touched: for rows whose tile
// result is not finite, which a value outside the row's own keys may have caused.
__noinline__ __device__ void pp_slow_row(const PagedAttnArgs &a, const PpRow &r, const uint32_t *table,
                                         const uint32_t *docs, uint32_t kh, float rf, uint32_t d0, uint32_t nd,
                                         float *out) {
    const uint32_t hd = a.kv.hd;
    float m = -INFINITY;
    for (uint32_t d = d0; d < d0 + nd; d += 16) {
        float o[16], l = 0.0f;
        for (int e = 0; e < 16; e++) o[e] = 0.0f;
        for (int pass = d == d0 ? 0 : 1; pass < 2; pass++) {
            for (int64_t j = r.lo < 0 ? 0 : r.lo; j < r.hi; j++) {
                if (docs && docs[j] != r.doc) continue;
                const uint32_t page = table[j / a.kv.page_size];
                if (page >= a.kv.n_pages) continue;
                const uint64_t off = paged_offset(a.kv, page, (uint32_t)j, kh);
                float dot = 0.0f;
                for (uint32_t e = 0; e < hd; e++) dot = fmaf(r.q[e], pp_kv(a.kv.k + off, e), dot);
                const float t = score_log2(dot, rf, a.softcap, r.slope, fabsf((float)(r.i - j)));
                if (pass == 0) {
                    m = t != t ? t : fmaxf(m, t);
                } else {
                    const float p = ex2(t - m);
                    l += p;
                    for (int e = 0; e < 16; e++) o[e] = fmaf(p, pp_kv(a.kv.v + off, d + e), o[e]);
                }
            }
        }
        for (int e = 0; e < 16; e++) out[d + e] = l == 0.0f ? 0.0f : o[e] / l;
    }
}

template <int HD, bool EXTRA>
__global__ void __launch_bounds__(kPpThreads, 1) k_paged_prompt(PagedAttnArgs a) {
    using S = PpShape<HD>;
    constexpr int KT = S::KT, NS = S::STAGES;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint64_t *offs = reinterpret_cast<uint64_t *>(smem + S::OFF_OFFS);
    uint32_t *docs_s = reinterpret_cast<uint32_t *>(smem + S::OFF_DOCS);
    uint32_t *skip = reinterpret_cast<uint32_t *>(smem + S::OFF_SKIP);  // bit set: some row may see the tile
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + S::OFF_BARS), *empty = full + NS;
    uint64_t *s_full = empty + NS, *p_full = s_full + 2, *o_full = p_full + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(o_full + 2);
    volatile uint32_t *dead = tmem_slot + 1;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_launch_dependents();
    pdl_wait();

    // this CTA's rows; the longest (last) row blocks of a causal prompt come first
    const uint32_t s = blockIdx.z, kh = blockIdx.y, rb = gridDim.x - 1 - blockIdx.x;
    const uint32_t cap = (uint32_t)min((uint64_t)a.kv.max_pages * a.kv.page_size, (uint64_t)a.max_len);
    uint32_t len = a.lens[s];
    const uint32_t c0 = a.cu[s], c1 = a.cu[s + 1];
    const bool ok = c0 <= c1 && c1 <= a.total_q && c1 - c0 <= a.max_q;
    if ((len > cap || !ok) && rb == 0 && kh == 0 && tid == 0) atomicExch(a.err, DEV_ERR_BAD_INDEX);
    len = min(len, cap);
    if (!ok) return;
    const uint32_t nq = c1 - c0, rows = nq * a.group, R0 = rb * S::ROWS;
    if (R0 >= rows) return;
    const uint32_t t0 = R0 / a.group, t1 = (min(rows, R0 + S::ROWS) - 1) / a.group;
    const int64_t i0 = (int64_t)len - nq + t0, i1 = (int64_t)len - nq + t1;
    const uint32_t prefix = a.causal && a.prefix ? a.prefix[s] : 0;
    int64_t hi64 = len, lo64 = 0;
    if (a.causal) hi64 = min(hi64, max(i1 + 1, (int64_t)prefix));
    if (a.window) lo64 = max((int64_t)0, i0 - (int64_t)a.window + 1);
    const uint32_t hi = (uint32_t)max((int64_t)0, hi64), lo = (uint32_t)min(lo64, (int64_t)hi);
    const uint32_t tiles = (hi - lo + KT - 1) / KT;
    const uint32_t *table = a.table + (uint64_t)s * a.kv.max_pages;
    const uint32_t *docs = a.docs ? a.docs + (uint64_t)s * a.doc_stride : nullptr;
    const bool skipping = docs && tiles <= kPpSkipTiles;

    if (tid == 0) {
        for (int i = 0; i < NS; i++) {
            mbar_init(full + i, kPpProducers);
            mbar_init(empty + i, 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(s_full + i, 1);
            mbar_init(p_full + i, HD == 256 ? 256 : 128);
            mbar_init(o_full + i, 1);
        }
        *dead = 0;
        fence_barrier_init();
    }
    if (warp == 8) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    if (skipping) {
        // a tile is left out when the ranges of document numbers do not meet
        for (int i = tid; i < kPpSkipTiles / 32; i += kPpThreads) skip[i] = 0;
        uint32_t dmin = 0xffffffffu, dmax = 0;
        for (int64_t i = max((int64_t)0, i0) + lane; i <= i1; i += 32) {
            dmin = min(dmin, docs[i]);
            dmax = max(dmax, docs[i]);
        }
        dmin = __reduce_min_sync(0xffffffffu, dmin);
        dmax = __reduce_max_sync(0xffffffffu, dmax);
        __syncthreads();
        for (uint32_t t = warp; t < tiles; t += kPpThreads / 32) {
            uint32_t kmin = 0xffffffffu, kmax = 0;
#pragma unroll
            for (int e = 0; e < KT / 32; e++) {
                const uint32_t j = lo + t * KT + e * 32 + lane;
                if (j < hi) {
                    kmin = min(kmin, docs[j]);
                    kmax = max(kmax, docs[j]);
                }
            }
            kmin = __reduce_min_sync(0xffffffffu, kmin);
            kmax = __reduce_max_sync(0xffffffffu, kmax);
            if (lane == 0 && kmin <= dmax && dmin <= kmax) atomicOr(skip + t / 32, 1u << (t % 32));
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    auto wait = [&](uint64_t *bar, uint32_t phase) {
        if (*dead) return;
        if (!mbar_wait_bounded(bar, phase, kWaitLimitNs)) {
            *dead = 1;
            atomicExch(a.err, DEV_ERR_TMA_TIMEOUT);
        }
    };
    // the first tile at or after t that is worked on
    auto next_tile = [&](uint32_t t) {
        if (skipping)
            while (t < tiles && !(skip[t / 32] >> (t % 32) & 1u)) t++;
        return t;
    };

    if (warp >= 8) {
        regs_dec<56>();
        if (warp > 8) {
            // ── K and V tiles into the ring ──
            const int pt = tid - 288, pw = warp - 9;
            constexpr int CH = HD / 8, RPI = 32 / CH;  // 16-byte chunks per row, rows per warp and step
            const int col = lane % CH;
            uint32_t n = 0, jj = 0;
            for (uint32_t t = next_tile(0); t < tiles; t = next_tile(t + 1), jj++) {
                uint64_t mine[(KT + kPpProducers - 1) / kPpProducers];
#pragma unroll
                for (int u = 0; u < (KT + kPpProducers - 1) / kPpProducers; u++) {
                    const uint32_t r = pt + u * kPpProducers, j = lo + t * KT + r;
                    mine[u] = ~0ull;
                    if (r < KT && j < hi) {
                        const uint32_t page = table[j / a.kv.page_size];
                        if (page < a.kv.n_pages)
                            mine[u] = paged_offset(a.kv, page, j, kh);
                        else
                            atomicExch(a.err, DEV_ERR_BAD_INDEX);
                    }
                }
                named_sync<1, kPpProducers>();  // the last tile's offsets are read
#pragma unroll
                for (int u = 0; u < (KT + kPpProducers - 1) / kPpProducers; u++)
                    if (pt + u * kPpProducers < KT) offs[pt + u * kPpProducers] = mine[u];
                named_sync<1, kPpProducers>();
                for (int kv = 0; kv < 2; kv++, n++) {
                    const uint32_t st = n % NS;
                    wait(empty + st, ((n / NS) & 1) ^ 1);
                    if (docs && kv == 0)
                        for (int r = pt; r < KT; r += kPpProducers)
                            docs_s[(jj % S::DOCS) * KT + r] = lo + t * KT + r < hi ? docs[lo + t * KT + r] : 0;
                    const uint8_t *src = kv ? a.kv.v : a.kv.k;
                    const uint32_t dst = smem_u32(smem) + S::OFF_RING + st * S::STAGE + (col / 8) * (KT * 128);
#pragma unroll 4
                    for (int r = pw * RPI + lane / CH; r < KT; r += 3 * RPI) {
                        const uint64_t o = offs[r];
                        const bool take = o != ~0ull;
                        cp_async16(dst + r * 128 + (((col & 7) ^ (r & 7)) << 4), src + (take ? o : 0) + col * 16, take);
                    }
                    cp_async_commit();
                    if (n) {  // the copies before these have landed: hand their stage to the tensor cores
                        cp_async_wait<1>();
                        fence_async_smem();
                        mbar_arrive(full + (n - 1) % NS);
                    }
                }
            }
            if (n) {
                cp_async_wait<0>();
                fence_async_smem();
                mbar_arrive(full + (n - 1) % NS);
            }
        } else if (lane == 0) {
            // ── MMAs ──
            constexpr uint32_t IQK = umma_idesc_f16_f32(128, KT);
            constexpr uint32_t IPV = umma_idesc_f16_f32(128, HD) | kUmmaBTransposed;
            const uint32_t q_u = smem_u32(smem), ring = q_u + S::OFF_RING;
            auto qk = [&](int tile, uint32_t stage, uint32_t d) {
#pragma unroll 1
                for (int pl = 1; pl >= 0; pl--) {  // low plane first: small terms while the sum is small
                    const uint32_t qa = q_u + (tile * 2 + pl) * S::QPLANE;
#pragma unroll
                    for (int i = 0; i < HD / 16; i++)
                        umma_f16(d, umma_desc_sw128(qa + (i / 4) * 16384 + (i % 4) * 32),
                                 umma_desc_sw128(ring + stage * S::STAGE + (i / 4) * (KT * 128) + (i % 4) * 32), IQK,
                                 pl == 0 || i > 0);
                }
            };
            auto pv = [&](uint32_t p, uint32_t stage, uint32_t d) {
#pragma unroll 1
                for (int pl = 1; pl >= 0; pl--) {
#pragma unroll
                    for (int i = 0; i < KT / 16; i++)
                        umma_f16_ts(d, p + 32 * (i / 2) + 16 * pl + 8 * (i % 2),
                                    umma_desc_sw128_mn(ring + stage * S::STAGE + i * 2048, KT * 128), IPV, pl == 0 || i > 0);
                }
            };
            uint32_t t = next_tile(0), jj = 0;
            if (t < tiles) {
                // the queries are in place once both softmax groups have arrived on p_full the first time
                wait(p_full + 0, 0);
                if (HD != 256) wait(p_full + 1, 0);
                wait(full + 0, 0);
                tc_fence_after();
                if constexpr (HD == 256) {
                    qk(0, 0, tmem + S::S_COL(0));
                    umma_commit(s_full + 0);
                    umma_commit(empty + 0);
                } else {
                    qk(0, 0, tmem + S::S_COL(0));
                    umma_commit(s_full + 0);
                    qk(1, 0, tmem + S::S_COL(1));
                    umma_commit(s_full + 1);
                    umma_commit(empty + 0);
                }
                while (t < tiles) {
                    const uint32_t tn = next_tile(t + 1);
                    const uint32_t nv = 2 * jj + 1, nk = 2 * jj + 2;
                    if constexpr (HD == 256) {
                        if (tn < tiles) {
                            wait(full + nk % NS, (nk / NS) & 1);
                            tc_fence_after();
                            qk(0, nk % NS, tmem + S::S_COL((jj + 1) & 1));
                            umma_commit(s_full + ((jj + 1) & 1));
                            umma_commit(empty + nk % NS);
                        }
                        wait(full + nv % NS, (nv / NS) & 1);
                        wait(p_full + 0, (jj + 1) & 1);
                        tc_fence_after();
                        pv(tmem + S::S_COL(jj & 1), nv % NS, tmem + S::O_COL(0));
                        umma_commit(o_full + 0);
                        umma_commit(empty + nv % NS);
                    } else {
#pragma unroll 1
                        for (int w = 0; w < 2; w++) {
                            if (w == 0) wait(full + nv % NS, (nv / NS) & 1);
                            wait(p_full + w, (jj + 1) & 1);
                            tc_fence_after();
                            pv(tmem + S::S_COL(w), nv % NS, tmem + S::O_COL(w));
                            umma_commit(o_full + w);
                            if (w == 1) umma_commit(empty + nv % NS);
                            if (tn < tiles) {
                                if (w == 0) {
                                    wait(full + nk % NS, (nk / NS) & 1);
                                    tc_fence_after();
                                }
                                qk(w, nk % NS, tmem + S::S_COL(w));
                                umma_commit(s_full + w);
                                if (w == 1) umma_commit(empty + nk % NS);
                            }
                        }
                    }
                    t = tn;
                    jj++;
                }
            }
        }
        __syncwarp();
    } else {
        // ── softmax: one row per thread ──
        regs_inc<224>();
        const int wg = warp >> 2, r = tid & 127, tile = HD == 256 ? 0 : wg;
        constexpr int CW = HD == 256 ? 32 : KT;          // score columns of this thread
        constexpr int OW = HD == 256 ? 128 : HD;         // output columns
        const int half = HD == 256 ? wg : 0;
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t R = R0 + tile * 128 + r;
        const bool real = R < rows;
        PpRow row;
        const uint32_t token = real ? R / a.group : 0, head = kh * a.group + (real ? R % a.group : 0);
        row.q = a.q + (uint64_t)(c0 + token) * a.q_stride + (uint64_t)head * HD;
        row.i = (int64_t)len - nq + token;
        row.lo = a.window ? row.i - (int64_t)a.window + 1 : 0;
        row.hi = a.causal ? min((int64_t)len, max(row.i + 1, (int64_t)prefix)) : (int64_t)len;
        row.doc = 0;
        row.slope = EXTRA && a.slopes ? a.slopes[head] : 0.0f;
        if (docs) {
            if (row.i >= 0)
                row.doc = docs[row.i];
            else
                row.hi = 0;
        }
        if (!real) row.hi = 0;
        // queries to two f16 planes: the warp takes its 32 rows one by one
        const float f0 = EXTRA && a.softcap != 0.0f ? a.scale / a.softcap : a.scale * 1.4426950408889634f;
        float rf = 0.0f;
        if (HD != 256 || wg == 0) {
#pragma unroll 4
            for (int x = 0; x < 32; x++) {
                const uint32_t rr = (warp & 3) * 32 + x, RR = R0 + tile * 128 + rr;
                constexpr int PER = HD / 32;
                float v[PER];
#pragma unroll
                for (int e = 0; e < PER; e++) v[e] = 0.0f;
                if (RR < rows) {
                    const float *src = a.q + (uint64_t)(c0 + RR / a.group) * a.q_stride + (uint64_t)(kh * a.group + RR % a.group) * HD;
#pragma unroll
                    for (int e = 0; e < PER; e += 2) {
                        const float2 y = *reinterpret_cast<const float2 *>(src + 64 * (e / 2) + 2 * lane);
                        v[e] = y.x;
                        v[e + 1] = y.y;
                    }
                }
                float top = 0.0f;
#pragma unroll
                for (int e = 0; e < PER; e++) top = fmaxf(top, fabsf(v[e]));
                top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
                float up = 1.0f;
                if (top > 0.0f && top < INFINITY) {
                    const int ex = min(max(8 - (int)(__float_as_uint(top) >> 23) + 127, -126), 126);
                    up = __uint_as_float((uint32_t)(ex + 127) << 23);
                }
                if (lane == x) rf = f0 / up;
                const float sg = f0 < 0.0f ? -up : up;  // the factor on the scores stays positive
#pragma unroll
                for (int e = 0; e < PER; e += 2) {
                    uint32_t h, l;
                    split_f16x2(v[e] * sg, v[e + 1] * sg, h, l);
                    const uint32_t at = tile * 2 * S::QPLANE + (e / 2) * 16384 + sw128_offset(rr, 2 * lane);
                    *reinterpret_cast<uint32_t *>(smem + at) = h;
                    *reinterpret_cast<uint32_t *>(smem + at + S::QPLANE) = l;
                }
            }
            fence_async_smem();
        }
        if constexpr (HD == 256) {  // the second group works on the same rows
            if (wg == 0) {
                tmem_st1(tmem + lane_base + S::X_COL, rf);
                tmem_wait_st();
            }
            tc_fence_before();
            named_sync<2, 256>();
            tc_fence_after();
            rf = tmem_ld1(tmem + lane_base + S::X_COL);
            tmem_wait_ld();
            tc_fence_before();
            named_sync<2, 256>();
            tc_fence_after();
        }
        rf = fabsf(rf);
        mbar_arrive(p_full + tile);

        float o[OW];
#pragma unroll
        for (int e = 0; e < OW; e++) o[e] = 0.0f;
        float m = -INFINITY, l = 0.0f, alpha = 1.0f;
        const uint32_t o_addr = tmem + lane_base + S::O_COL(tile) + half * 128;
        auto add_o = [&]() {  // o = o * alpha + this tile's product
#pragma unroll
            for (int c = 0; c < OW; c += 32) {
                uint32_t v[32];
                tmem_ld32(o_addr + c, v);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; e++) o[c + e] = fmaf(o[c + e], alpha, __uint_as_float(v[e]));
            }
        };
        uint32_t jj = 0;
        for (uint32_t t = next_tile(0); t < tiles; t = next_tile(t + 1), jj++) {
            const int sb = HD == 256 ? (jj & 1) : tile;
            const uint32_t s_addr = tmem + lane_base + S::S_COL(sb) + half * 32;
            const int64_t k0 = (int64_t)lo + t * KT + half * 32;
            wait(s_full + sb, HD == 256 ? (jj / 2) & 1 : jj & 1);
            __syncwarp();
            tc_fence_after();
            const bool whole = !docs && row.lo <= k0 && k0 + CW <= row.hi;
            const bool plain = __all_sync(0xffffffffu, whole || !real);
            // pass 1: the row's maximum; capped, biased or masked scores go back to tensor memory
            float top = -INFINITY;
#pragma unroll
            for (int c = 0; c < CW; c += 32) {
                uint32_t v[32];
                tmem_ld32(s_addr + c, v);
                tmem_wait_ld();
                if (!EXTRA && plain) {
                    float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        x0 = fmaxf(x0, __uint_as_float(v[e]));
                        x1 = fmaxf(x1, __uint_as_float(v[e + 1]));
                    }
                    top = fmaxf(top, fmaxf(x0, x1));
                } else {
#pragma unroll
                    for (int e = 0; e < 32; e++) {
                        const int64_t j = k0 + c + e;
                        float x = __uint_as_float(v[e]);
                        if (EXTRA) x = score_log2(x, rf, a.softcap, row.slope, fabsf((float)(row.i - j)));
                        bool seen = plain || (j >= row.lo && j < row.hi);
                        if (docs) seen = seen && docs_s[(jj % S::DOCS) * KT + half * 32 + c + e] == row.doc;
                        x = seen ? x : -INFINITY;
                        top = fmaxf(top, x);
                        v[e] = __float_as_uint(x);
                    }
                    tmem_st32(s_addr + c, v);
                    tmem_wait_st();
                }
            }
            const float fs = EXTRA ? 1.0f : rf;
            top = top == -INFINITY ? top : top * fs;
            if constexpr (HD == 256) {  // the other half's maximum; the columns alternate with the tiles
                const uint32_t x_addr = tmem + lane_base + S::X_COL + 2 * (jj & 1);
                tmem_st1(x_addr + wg, top);
                tmem_wait_st();
                tc_fence_before();
                named_sync<2, 256>();
                tc_fence_after();
                const float other = tmem_ld1(x_addr + (wg ^ 1));
                tmem_wait_ld();
                top = fmaxf(top, other);
            }
            const float mn = fmaxf(m, top);
            const float al = mn == m ? 1.0f : ex2(m - mn);
            m = mn;
            // weights times 2^10: small ones keep their f16 bits, and the sum carries the same factor
            const float base = m == -INFINITY ? 0.0f : 10.0f - m;
            float l0 = 0.0f, l1 = 0.0f;
#pragma unroll
            for (int c = 0; c < CW; c += 32) {
                uint32_t v[32], p[32];
                tmem_ld32(s_addr + c, v);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                    const float x = ex2(fmaf(__uint_as_float(v[e]), fs, base));
                    const float y = ex2(fmaf(__uint_as_float(v[e + 1]), fs, base));
                    l0 += x;
                    l1 += y;
                    split_f16x2(x, y, p[e / 2], p[16 + e / 2]);
                }
                tmem_st32(s_addr + c, p);
            }
            tmem_wait_st();
            l = fmaf(l, al, l0 + l1);
            if constexpr (HD == 256) {
                // the last tile's product was computed while this softmax ran
                if (jj) {
                    wait(o_full + 0, (jj - 1) & 1);
                    __syncwarp();
                    tc_fence_after();
                    add_o();
                }
                alpha = al;
                tc_fence_before();
                mbar_arrive(p_full + 0);
            } else {
                alpha = al;
                tc_fence_before();
                mbar_arrive(p_full + tile);
                wait(o_full + tile, jj & 1);
                __syncwarp();
                tc_fence_after();
                add_o();
            }
        }
        if constexpr (HD == 256) {
            if (jj) {
                wait(o_full + 0, (jj - 1) & 1);
                __syncwarp();
                tc_fence_after();
                add_o();
            }
            // both halves' sums
            const uint32_t x_addr = tmem + lane_base + S::X_COL + 4;
            tmem_st1(x_addr + wg, l);
            tmem_wait_st();
            tc_fence_before();
            named_sync<2, 256>();
            tc_fence_after();
            l += tmem_ld1(x_addr + (wg ^ 1));
            tmem_wait_ld();
        }
        if (real) {
            float *dst = a.out + (uint64_t)(c0 + token) * a.out_stride + (uint64_t)head * HD + half * 128;
            const float inv = l > 0.0f ? __fdiv_rn(1.0f, l) : (l == 0.0f ? 0.0f : l);
            float bad = 0.0f;
#pragma unroll
            for (int e = 0; e < OW; e++) bad += (o[e] - o[e]);
            if (bad == 0.0f && l - l == 0.0f) {
#pragma unroll
                for (int e = 0; e < OW; e += 4)
                    *reinterpret_cast<float4 *>(dst + e) = make_float4(o[e] * inv, o[e + 1] * inv, o[e + 2] * inv, o[e + 3] * inv);
            } else {
                pp_slow_row(a, row, table, docs, kh, f0, half * 128, OW, dst - half * 128);
            }
        }
        tc_fence_before();
    }
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

namespace {

template <int HD, bool EXTRA>
cudaError_t pp_launch(const LaunchCfg &c, const PagedAttnArgs &a) {
    using S = PpShape<HD>;
    const uint64_t rows = (uint64_t)a.max_q * a.group;
    return launch_k(c, "paged_prompt", k_paged_prompt<HD, EXTRA>,
                    dim3((uint32_t)((rows + S::ROWS - 1) / S::ROWS), a.kv.n_kv, a.n_seq), dim3(kPpThreads), S::SMEM, a);
}

// The register split needs the registers that 168 per thread give a block.
template <int HD, bool EXTRA>
bool pp_regs() {
    cudaFuncAttributes f;
    return cudaFuncGetAttributes(&f, k_paged_prompt<HD, EXTRA>) == cudaSuccess && f.numRegs >= 168;
}

}  // namespace

bool paged_prompt_supported(const PagedAttnArgs &a) {
    static const bool regs = pp_regs<64, false>() && pp_regs<64, true>() && pp_regs<128, false>() &&
                             pp_regs<128, true>() && pp_regs<256, false>() && pp_regs<256, true>();
    return regs && a.kv.f16 && (uint64_t)a.max_q * a.group >= 64;
}

cudaError_t launch_paged_prompt(const LaunchCfg &c, PagedAttnArgs a) {
    a.err = c.dev_err;
    const bool extra = a.softcap != 0.0f || a.slopes;
    switch (a.kv.hd) {
    case 64: return extra ? pp_launch<64, true>(c, a) : pp_launch<64, false>(c, a);
    case 128: return extra ? pp_launch<128, true>(c, a) : pp_launch<128, false>(c, a);
    case 256: return extra ? pp_launch<256, true>(c, a) : pp_launch<256, false>(c, a);
    default: return cudaErrorInvalidValue;
    }
}

}  // namespace lt
