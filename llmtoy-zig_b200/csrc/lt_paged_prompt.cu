// lt_paged_prompt.cu — attention of many queries per sequence over a paged cache of
// f16 values or 8-bit codes, on the 5th-generation tensor cores.
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
//   warps 9-11 (-15) bring K and V tiles from their pages into a ring of stages of
//                    128-byte-swizzled rows: tiles that lie wholly within the
//                    sequence by TMA, a box per page and 64 columns; the ragged
//                    ends, and pages that are no multiple of 8 slots, by 16-byte
//                    asynchronous copies with zero fill.  8-bit codes: from their pages through
//                    registers, where they become f16 numbers (exactly), the next stage's
//                    codes on their way; scales enter as lt_paged_q8.cuh puts them, a
//                    factor and a summand for 16 columns of scores
// While one tile's softmax runs, the tensor cores work for the other: per tile
// of keys the MMA order is PV0 QK0' PV1 QK1' (' the next keys), PV in two halves so
// that the first can start while the softmax is at the second.  S and P share
// their columns of tensor memory; P lies as it is read: per 16 keys 8 columns
// of high terms, then 8 of low ones, over the 16 columns of S they come from.
//
// Bound: the tensor cores, from a few hundred rows on.  One B200, 8192 tokens,
// 32/4 heads of 128, causal (550 GFLOP, 1.1 TFLOP as done): 0.91 to 0.94 ms in a row,
// that is 1.17 to 1.21 PFLOP/s of products against 1.38 sustained by a cuBLAS bf16
// GEMM on this part (1.65 in a burst); 0.78 ms when launches are far enough apart to
// stay clear of the power cap.  With few rows, latency: a 257-token follow-up on 1243
// cached ones (14/2 heads of 64) takes 19 us with its keys shared by 6 CTAs, 37 us
// without.  head_dim 256 (6320 tokens of packed documents, 231 us) waits for K: the
// queries leave room for three stages only, and a K tile's copy starts when the
// product before the last is done.  Prefetching tiles into L2 made every case slower
// (8192 tokens 1.15 ms, 1.00 without), as did one KV head after the other (1.01 ms).
//
// 8-bit codes, the same cases: 8192 tokens 0.95 to 0.98 ms, the follow-up 20.4 us, the packed documents 241 us,
// 4096 tokens of 16/8 heads of 256 0.31 ms (f16 0.35): half the bytes, and the copying warps' conversion instead.  With
// three copying warps 1.27 ms and 351 us; with seven, whose registers the softmax warps gave, 1.00 and 299; with each
// head_dim's own split of the registers (PpShape) what stands above.  Spills at head_dim 256: 152 bytes with cap or bias, 140
// without; at 128 36 and 8.
#include <cuda.h>  // CUtensorMap (encoded through the runtime's driver entry point)

#include "lt_paged_q8.cuh"
#include "lt_umma.cuh"

namespace lt {

// Tiles whose documents are looked at beforehand: 512 bytes of bits, what shared memory leaves beside the queries and
// the ring at head_dim 128.  Longer rows (512 K keys; 256 K at head_dim 256) go through every tile.
constexpr int kPpSkipTiles = 4096;

// 8-bit codes: what stands for the logarithm of V's scale where a scale cannot be used.  With a score and its distance bias it is
// still above kQ8NoScore, which the sums of numbers stay below (scores near f32's largest number, 3.4e38, aside); it is finite, so
// that a masked score, -inf, stays that.
constexpr float kQ8NoScale = 3.3e38f, kQ8NoScore = 3.2e38f;

template <int HD, bool Q8 = false>
struct PpShape {
    static constexpr int TILES = HD == 256 ? 1 : 2;       // row tiles of 128
    static constexpr int ROWS = TILES * 128;
    static constexpr int KT = HD == 256 ? 64 : 128;       // keys per tile
    static constexpr int NBLK = HD / 64;                  // 128-byte-wide column blocks
    static constexpr int STAGE = KT * HD * 2;
    static constexpr int STAGES = HD == 64 ? 6 : 3;
    static constexpr int DOCS = HD == 64 ? 4 : 2;         // document-number buffers
    // 8-bit codes: seven copying warps instead of three, since a stage is refilled only as fast as its codes become f16
    // (8192 tokens, 32/4 heads of 128: 1.22 ms with three, head_dim 256, 4096 tokens: 0.56)
    static constexpr int THREADS = Q8 ? 512 : 384, REST = THREADS - 256, PRODUCERS = REST - 32;
    // registers per thread after the split: 256 softmax threads and the others share those of the launch
    static constexpr int REGS = Q8 ? 128 : 168;
    static constexpr int REGS_SOFTMAX = Q8 ? (HD == 64 ? 184 : HD == 128 ? 192 : 176) : HD == 64 ? 200 : 208;
    static constexpr int REGS_REST = Q8 ? (HD == 64 ? 72 : HD == 128 ? 64 : 80) : HD == 64 ? 104 : 88;
    static_assert(256 * REGS_SOFTMAX + REST * REGS_REST <= THREADS * REGS, "more registers than the launch holds");
    static constexpr int QPLANE = 128 * HD * 2;
    static constexpr int Q_BYTES = TILES * 2 * QPLANE;
    static constexpr int OFF_RING = Q_BYTES;
    static constexpr int OFF_OFFS = OFF_RING + STAGES * STAGE;
    static constexpr int GROUPS = KT / 16;                // of 16 keys, each within a page and a block
    // f16: places of a tile's rows; 8-bit codes: places and scales of the groups of two tiles
    static constexpr int OFF_DOCS = OFF_OFFS + (Q8 ? 2 * GROUPS * 16 : KT * 8);
    static constexpr int OFF_SCALES = OFF_DOCS + DOCS * KT * 4;  // 8-bit codes: k, log2 v and 1 / v of each group
    static constexpr int OFF_SKIP = OFF_SCALES + (Q8 ? DOCS * GROUPS * 12 + 16 : 0);
    static constexpr int OFF_BARS = OFF_SKIP + kPpSkipTiles / 8;
    static constexpr int SMEM = OFF_BARS + 256;
    static constexpr uint32_t S_COL(int i) { return (HD == 256 ? 64 : 128) * i; }
    static constexpr uint32_t O_COL(int i) { return 256 + (HD == 256 ? 0 : 128 * i); }
    static constexpr uint32_t X_COL = 128;                // head_dim 256: the halves' row maxima and sums
};

// 16 consecutive TMEM columns of this thread's lane.
LT_DEVINL void tmem_ld16(uint32_t taddr, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr));
}
LT_DEVINL void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
            taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
LT_DEVINL void tmem_st1(uint32_t taddr, float v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(taddr), "r"(__float_as_uint(v)) : "memory");
}
// One column, there when the call returns.
LT_DEVINL float tmem_ld1(uint32_t taddr) {
    uint32_t v;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n tcgen05.wait::ld.sync.aligned;"
                 : "=r"(v)
                 : "r"(taddr)
                 : "memory");
    return __uint_as_float(v);
}
LT_DEVINL void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// MMAs with descriptors as a changing low word and a constant high one, so that
// the issuing thread adds a constant per product.  High word: see umma_desc_sw128.
constexpr uint32_t kUmmaDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
LT_DEVINL uint32_t umma_lo(uint32_t saddr) { return ((saddr & 0x3FFFFu) >> 4) | (1u << 16); }
// Operand whose rows run along K (V: one row of 64 N values per key): 64-wide
// blocks of N lie `block` bytes apart, groups of 8 keys 1024 bytes.
LT_DEVINL uint32_t umma_lo_mn(uint32_t saddr, uint32_t block) { return ((saddr & 0x3FFFFu) >> 4) | ((block >> 4) << 16); }

template <bool ACC>
LT_DEVINL void umma_ss(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc) {
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 a, b;\n setp.ne.b32 p, %5, 0;\n mov.b64 a, {%1, %4};\n mov.b64 b, {%2, %4};\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n}\n" ::"r"(d_tmem),
        "r"(a_lo), "r"(b_lo), "r"(idesc), "n"(kUmmaDescHi), "n"(ACC ? 1 : 0));
}
// A in tensor memory: 128 lanes, two f16 of K per column.
template <bool ACC>
LT_DEVINL void umma_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc) {
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 b;\n setp.ne.b32 p, %5, 0;\n mov.b64 b, {%2, %4};\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n}\n" ::"r"(d_tmem),
        "r"(a_tmem), "r"(b_lo), "r"(idesc), "n"(kUmmaDescHi), "n"(ACC ? 1 : 0));
}
LT_DEVINL bool elect_one() {
    uint32_t p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
    return p != 0;
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

// K and V pools as [page][head][slot][head_dim] tensors, read in boxes of `rows`
// slots (a divisor of the page and of a tile; 0: no maps) by 64 columns.
struct PpMaps {
    alignas(64) CUtensorMap k;
    alignas(64) CUtensorMap v;
    uint32_t rows;
};
LT_DEVINL void tma_load_4d(uint32_t dst, const CUtensorMap *map, uint32_t x, uint32_t slot, uint32_t head, uint32_t page,
                           uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(slot), "r"(head), "r"(page), "r"(smem_u32(bar))
        : "memory");
}

// Two weights as packed f16 high and low terms: low = x - high by one
// f16 x f16 + f32 product-sum per element.
LT_DEVINL void split_weights(float x, float y, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(x, y);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    float dx, dy;
    asm("{\n .reg .b16 a, b, m;\n mov.b32 {a, b}, %2;\n mov.b16 m, 0xBC00;\n"
        " fma.rn.f32.f16 %0, a, m, %3;\n fma.rn.f32.f16 %1, b, m, %4;\n}\n"
        : "=f"(dx), "=f"(dy)
        : "r"(hi), "f"(x), "f"(y));
    const __half2 l = __floats2half2_rn(dx, dy);
    lo = *reinterpret_cast<const uint32_t *>(&l);
}

template <int N>
struct IntC {
    static constexpr int value = N;
};

template <int HD, bool EXTRA, bool Q8, int kPpThreads = PpShape<HD, Q8>::THREADS>
__global__ void __launch_bounds__(kPpThreads, 1) k_paged_prompt(const __grid_constant__ PagedAttnArgs a, const __grid_constant__ PpMaps maps) {
    using S = PpShape<HD, Q8>;
    constexpr int KT = S::KT, NS = S::STAGES, kPpProducers = S::PRODUCERS;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint64_t *offs = reinterpret_cast<uint64_t *>(smem + S::OFF_OFFS);
    uint32_t *docs_s = reinterpret_cast<uint32_t *>(smem + S::OFF_DOCS);
    float *scales_s = reinterpret_cast<float *>(smem + S::OFF_SCALES);  // [DOCS][3][GROUPS]
    uint32_t *skip = reinterpret_cast<uint32_t *>(smem + S::OFF_SKIP);  // bit set: some row may see the tile
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + S::OFF_BARS), *empty = full + NS;
    uint64_t *s_full = empty + NS, *p_full = s_full + 2, *o_full = p_full + 2, *p_half = o_full + 2;
    uint64_t *mma_end = p_half + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(mma_end + 1);
    volatile uint32_t *dead = tmem_slot + 1;
    // warp-uniform values go through a shuffle where the compiler cannot see that
    // they are: the MMA operands then stay in uniform registers (65 instead of 90
    // to 150 clocks per 128 x 128 x 16 product)
    auto uniform = [](uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); };
    const int tid = threadIdx.x, warp = (int)uniform(tid >> 5), lane = tid & 31;
    pdl_launch_dependents();
    pdl_wait();

    // this CTA's rows; the last row blocks of all prompts, the longest of causal ones, come first
    // (a row block may be shared by nsplit CTAs, each with its part of the keys)
    uint32_t at = blockIdx.x;
    const uint32_t split = at % a.nsplit, kh = (at /= a.nsplit) % a.kv.n_kv, s = (at /= a.kv.n_kv) % a.n_seq;
    const uint32_t rb = a.row_blocks - 1 - at / a.n_seq;
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
    const uint32_t hi = (uint32_t)max((int64_t)0, hi64), first = (uint32_t)min(lo64, (int64_t)hi);
    const uint32_t lo = Q8 ? first & ~15u : maps.rows ? first - first % maps.rows : first;  // tiles start on a box, or a group
    const uint32_t all_tiles = (hi - lo + KT - 1) / KT, share = (all_tiles + a.nsplit - 1) / a.nsplit;
    const uint32_t begin = uniform(min(all_tiles, split * share)), tiles = uniform(min(all_tiles, begin + share));
    const uint32_t *table = a.table + (uint64_t)s * a.kv.max_pages;
    const uint32_t *docs = a.docs ? a.docs + (uint64_t)s * a.doc_stride : nullptr;
    const bool skipping = docs && all_tiles <= kPpSkipTiles;

    if (tid == 0) {
        for (int i = 0; i < NS; i++) {
            mbar_init(full + i, kPpProducers);
            mbar_init(empty + i, 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(s_full + i, 1);
            mbar_init(p_full + i, HD == 256 ? 256 : 128);
            mbar_init(o_full + i, 1);
            mbar_init(p_half + i, 128);
        }
        mbar_init(mma_end, 1);
        *dead = 0;
        fence_barrier_init();
    }
    if (warp == 8) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = uniform(*tmem_slot);

    // A wait that runs out lets all others pass (*dead): no copy is issued after that, and the CTA ends
    // when what is in flight has ended, or has had as long again.
    auto wait_always = [&](uint64_t *bar, uint32_t phase) {
        if (mbar_wait_bounded(bar, phase, kWaitLimitNs)) return true;
        *dead = 1;
        atomicExch(a.err, DEV_ERR_TMA_TIMEOUT);
        return false;
    };
    auto wait = [&](uint64_t *bar, uint32_t phase) { return !*dead && wait_always(bar, phase); };
    // the first tile at or after t that is worked on
    auto next_tile = [&](uint32_t t) {
        if (skipping)
            while (t < tiles && !(uniform(skip[t / 32]) >> (t % 32) & 1u)) t++;
        return t;
    };

    if (warp >= 8) {
        regs_dec<S::REGS_REST>();
        if (skipping) {
            // a tile is left out when the ranges of document numbers do not meet
            for (int i = tid - 256; i < kPpSkipTiles / 32; i += S::REST) skip[i] = 0;
            uint32_t dmin = 0xffffffffu, dmax = 0;
            for (int64_t i = max((int64_t)0, i0) + lane; i <= i1; i += 32) {
                dmin = min(dmin, docs[i]);
                dmax = max(dmax, docs[i]);
            }
            dmin = __reduce_min_sync(0xffffffffu, dmin);
            dmax = __reduce_max_sync(0xffffffffu, dmax);
            named_sync<4, S::REST>();
            for (uint32_t t = begin + warp - 8; t < tiles; t += S::REST / 32) {
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
            named_sync<3, kPpThreads>();
        }
        if (warp > 8) {
            // ── K and V tiles into the ring ──
            const int pt = tid - 288, pw = warp - 9;
            if constexpr (Q8) {
                constexpr int CH = HD / 16, CHUNKS = KT * CH, PER = (CHUNKS + kPpProducers - 1) / kPpProducers;
                uint4 v[PER];  // the next stage's codes: chunk c = pt + i PRODUCERS, column c % CH of row c / CH
                struct Group {
                    uint64_t at;  // ~0: not there
                    float k, v;
                };
                Group *groups = reinterpret_cast<Group *>(offs);  // of two tiles
                auto look = [&](uint32_t tt, uint32_t buf) {
                    if (pt >= S::GROUPS) return;
                    Group x = {~0ull, 0.0f, 0.0f};
                    const uint32_t key = lo + tt * KT + 16 * pt;
                    if (key < hi && key + 16 > first) {
                        const uint32_t page = table[page_of(a.kv, key)];
                        if (page < a.kv.n_pages) {
                            const uint64_t sc = q8_scale_at(a.kv, page, key, kh);
                            x = {paged_offset(a.kv, page, key, kh), a.kv.k_scale[sc], a.kv.v_scale[sc]};
                        } else {
                            atomicExch(a.err, DEV_ERR_BAD_INDEX);
                        }
                    }
                    groups[buf * S::GROUPS + pt] = x;
                };
                auto fetch = [&](const uint8_t *pool, uint32_t buf) {
                    pool += pt % CH * 16;
#pragma unroll
                    for (int i = 0; i < PER; i++) {
                        static_assert(kPpProducers % CH == 0, "one column per thread");
                        const uint32_t r = pt / CH + i * (kPpProducers / CH);
                        const uint64_t o = r < KT ? groups[buf * S::GROUPS + r / 16].at : ~0ull;
                        v[i] = make_uint4(0, 0, 0, 0);  // groups that are not there: zeros, which no weight of 0 makes NaN
                        if (o != ~0ull) v[i] = *reinterpret_cast<const uint4 *>(pool + o + (uint64_t)(r % 16) * (uint32_t)a.kv.slot_stride);
                    }
                };
                uint32_t st = 0, turn = 0;
                // the stage's turn, then its codes as f16: 16 of them fill two 16-byte columns of a 128-byte-swizzled row
                auto hand_over = [&](bool k_stage, uint32_t t, uint32_t jj) {
                    const bool ok = __all_sync(0xffffffffu, wait(empty + st, (turn & 1) ^ 1));
                    if (ok) {
                        if (k_stage) {
                            if (docs)
                                for (int r = pt; r < KT; r += kPpProducers) {
                                    const uint32_t j = lo + t * KT + r;
                                    docs_s[(jj % S::DOCS) * KT + r] = j < hi ? docs[j] : 0;
                                }
                            if (pt < S::GROUPS) {
                                // Scales that cannot be used: scores above all others', by which their rows' sums become NaN.
                                // The factor on scores stays a number: masked ones must stay -inf.
                                const Group &x = groups[(jj & 1) * S::GROUPS + pt];
                                const Q8Scale z = q8_scale(x.k, x.v);
                                const bool good = z.k == z.k;
                                float *to = scales_s + (jj % S::DOCS) * 3 * S::GROUPS + pt;
                                to[0] = good ? z.k : 0.0f;
                                to[S::GROUPS] = good ? z.v_log2 : kQ8NoScale;
                                to[2 * S::GROUPS] = good ? z.v_inv : __int_as_float(0x7fffffff);
                            }
                        }
                        uint8_t *stage = smem + S::OFF_RING + st * S::STAGE;
#pragma unroll
                        for (int i = 0; i < PER; i++) {
                            const int r = pt / CH + i * (kPpProducers / CH), col = 2 * (pt % CH);
                            if (r >= KT) break;
                            uint4 h0, h1;
                            s8_to_f16(v[i].x, h0.x, h0.y);
                            s8_to_f16(v[i].y, h0.z, h0.w);
                            s8_to_f16(v[i].z, h1.x, h1.y);
                            s8_to_f16(v[i].w, h1.z, h1.w);
                            uint8_t *row = stage + col / 8 * (KT * 128) + r * 128;
                            *reinterpret_cast<uint4 *>(row + (((col & 7) ^ (r & 7)) << 4)) = h0;
                            *reinterpret_cast<uint4 *>(row + ((((col & 7) + 1) ^ (r & 7)) << 4)) = h1;
                        }
                        fence_async_smem();
                        mbar_arrive(full + st);
                    }
                    if (++st == NS) st = 0, turn++;
                };
                uint32_t t = next_tile(begin), jj = 0;
                if (t < tiles) {
                    look(t, 0);
                    named_sync<1, kPpProducers>();
                    fetch(a.kv.k, 0);
                }
                while (t < tiles) {
                    const uint32_t tn = next_tile(t + 1);
                    hand_over(true, t, jj);
                    fetch(a.kv.v, jj & 1);
                    if (tn < tiles) look(tn, (jj + 1) & 1);  // its buffer's tile is fetched since the last barrier
                    hand_over(false, t, jj);
                    if (tn < tiles) {
                        named_sync<1, kPpProducers>();
                        fetch(a.kv.k, (jj + 1) & 1);
                    }
                    t = tn;
                    jj++;
                }
            } else {
                constexpr int CH = HD / 8, RPI = 32 / CH;  // 16-byte chunks per row, rows per warp and step
                const int col = lane % CH;
                constexpr int PER = (KT + kPpProducers - 1) / kPpProducers;
                uint64_t mine[PER];  // pool offsets of this thread's rows, looked up one tile ahead
                auto look = [&](uint32_t t) {
#pragma unroll
                    for (int u = 0; u < PER; u++) {
                        const uint32_t r = pt + u * kPpProducers, j = lo + t * KT + r;
                        mine[u] = ~0ull;
                        if (r < KT && j >= first && j < hi) {
                            const uint32_t page = table[j / a.kv.page_size];
                            if (page < a.kv.n_pages)
                                mine[u] = paged_offset(a.kv, page, j, kh);
                            else
                                atomicExch(a.err, DEV_ERR_BAD_INDEX);
                        }
                    }
                };
                auto landed = [&](uint32_t stage) {  // this thread's copies are in place: hand the stage on
                    fence_async_smem();
                    mbar_arrive(full + stage);
                };
                uint32_t jj = 0, st = 0, turn = 0;  // tile count; ring stage and how often it went round
                uint32_t boxes_in = 0, boxes_phase = 0;  // bit per stage: last filled by TMA, and in which phase
                uint32_t t = next_tile(begin);
                bool owed = false;                // the stage before st is copied but not handed on
                // tiles of whole boxes: every slot holds a cached position
                auto boxed = [&](uint32_t tt) {
                    const uint32_t k0 = lo + tt * KT;
                    return maps.rows && k0 >= first && (uint64_t)k0 + KT <= len;
                };
                const uint32_t boxes = maps.rows ? KT / maps.rows : 0;  // per 64 columns
                uint32_t box_page = 0;
                auto look_boxed = [&](uint32_t tt) {  // lane l of warp 9: box l % boxes of column block l / boxes
                    if (pw == 0 && (uint32_t)lane < boxes * S::NBLK) {
                        box_page = table[(lo + tt * KT + lane % boxes * maps.rows) / a.kv.page_size];
                        if (box_page >= a.kv.n_pages) atomicExch(a.err, DEV_ERR_BAD_INDEX);
                    }
                };
                auto ahead = [&](uint32_t tt) {
                    if (tt >= tiles) return;
                    if (boxed(tt))
                        look_boxed(tt);
                    else
                        look(tt);
                };
                ahead(t);
                while (t < tiles) {
                    const bool by_box = boxed(t);
                    if (!by_box) {
                        named_sync<1, kPpProducers>();  // the last such tile's offsets are read
#pragma unroll
                        for (int u = 0; u < PER; u++)
                            if (pt + u * kPpProducers < KT) offs[pt + u * kPpProducers] = mine[u];
                        named_sync<1, kPpProducers>();
                    }
                    const uint32_t tn = next_tile(t + 1), page = box_page;
#pragma unroll 1
                    for (int kv = 0; kv < 2; kv++) {
                        if (owed && (by_box || !mbar_try_wait(empty + st, (turn & 1) ^ 1))) {
                            cp_async_wait<0>();
                            landed(st ? st - 1 : NS - 1);
                            owed = false;
                        }
                        if (!__all_sync(0xffffffffu, wait(empty + st, (turn & 1) ^ 1))) continue;
                        const uint32_t bit = 1u << st;
                        boxes_in = by_box ? boxes_in | bit : boxes_in & ~bit;
                        boxes_phase = turn & 1 ? boxes_phase | bit : boxes_phase & ~bit;
                        if (docs && kv == 0)
                            for (int r = pt; r < KT; r += kPpProducers) {
                                const uint32_t j = lo + t * KT + r;
                                docs_s[(jj % S::DOCS) * KT + r] = j < hi ? docs[j] : 0;
                            }
                        const uint32_t stage = smem_u32(smem) + S::OFF_RING + st * S::STAGE;
                        if (by_box) {
                            if (pw == 0) {
                                if (lane == 0) mbar_arrive_expect_tx(full + st, S::STAGE);
                                __syncwarp();
                                if ((uint32_t)lane < boxes * S::NBLK) {
                                    const uint32_t r = lane % boxes * maps.rows, blk = lane / boxes;
                                    tma_load_4d(stage + blk * (KT * 128) + r * 128, kv ? &maps.v : &maps.k, blk * 64,
                                                (lo + t * KT + r) % a.kv.page_size, kh, page, full + st);
                                }
                                if (lane) mbar_arrive(full + st);
                            } else {
                                mbar_arrive(full + st);
                            }
                            if (kv == 0) ahead(tn);
                        } else {
                            const uint8_t *src = (kv ? a.kv.v : a.kv.k) + col * 16;
                            const uint32_t dst = stage + (col / 8) * (KT * 128);
#pragma unroll 4
                            for (int r = pw * RPI + lane / CH; r < KT; r += 3 * RPI) {
                                const uint64_t o = offs[r];
                                const bool take = o != ~0ull;
                                cp_async16(dst + r * 128 + (((col & 7) ^ (r & 7)) << 4), src + (take ? o : 0), take);
                            }
                            cp_async_commit();
                            if (kv == 0) ahead(tn);
                            if (owed) {
                                cp_async_wait<1>();
                                landed(st ? st - 1 : NS - 1);
                            }
                            owed = true;
                        }
                        if (++st == NS) st = 0, turn++;
                    }
                    t = tn;
                    jj++;
                }
                if (owed) {
                    cp_async_wait<0>();
                    landed(st ? st - 1 : NS - 1);
                }
                if (pw == 0)  // no copy of this CTA is under way when it ends
                    for (int i = 0; i < NS; i++)
                        if ((boxes_in >> i & 1u) && !wait_always(full + i, boxes_phase >> i & 1u)) break;
            }
        } else {
            // ── MMAs ──
            constexpr uint32_t IQK = umma_idesc_f16_f32(128, KT);
            constexpr uint32_t IPV = umma_idesc_f16_f32(128, HD) | kUmmaBTransposed;
            const uint32_t q_u = smem_u32(smem), ring = q_u + S::OFF_RING;
            // one lane issues; the loop around it stays uniform across the warp
            auto qk = [&](int tile, uint32_t stage, uint32_t d, uint64_t *done, uint64_t *release) {
                const uint32_t qa = umma_lo(q_u + tile * 2 * S::QPLANE), kb = umma_lo(ring + stage * S::STAGE);
                if (elect_one()) {
                    // low plane first: small terms while the sum is small
#pragma unroll
                    for (int i = 0; i < HD / 16; i++) {
                        const uint32_t qi = qa + ((S::QPLANE + (i / 4) * 16384 + (i % 4) * 32) >> 4);
                        const uint32_t ki = kb + (((i / 4) * (KT * 128) + (i % 4) * 32) >> 4);
                        if (i == 0)
                            umma_ss<false>(d, qi, ki, IQK);
                        else
                            umma_ss<true>(d, qi, ki, IQK);
                    }
#pragma unroll
                    for (int i = 0; i < HD / 16; i++)
                        umma_ss<true>(d, qa + (((i / 4) * 16384 + (i % 4) * 32) >> 4),
                                      kb + (((i / 4) * (KT * 128) + (i % 4) * 32) >> 4), IQK);
                    umma_commit(done);
                    if (release) umma_commit(release);
                }
                __syncwarp();
            };
            // the products of `STEPS` 16-key steps from step FROM on
            auto pv_steps = [&](auto from, auto steps, uint32_t p, uint32_t vb, uint32_t d) {
                constexpr int FROM = decltype(from)::value, STEPS = decltype(steps)::value;
#pragma unroll
                for (int i = FROM; i < FROM + STEPS; i++) {
                    if (i == 0)
                        umma_ts<false>(d, p + 8, vb, IPV);
                    else
                        umma_ts<true>(d, p + 16 * i + 8, vb + ((i * 2048) >> 4), IPV);
                }
#pragma unroll
                for (int i = FROM; i < FROM + STEPS; i++) umma_ts<true>(d, p + 16 * i, vb + ((i * 2048) >> 4), IPV);
            };
            auto pv = [&](uint32_t p, uint32_t stage, uint32_t d, uint64_t *half, uint64_t *rest, uint32_t turn,
                          uint64_t *done, uint64_t *release) {
                const uint32_t vb = umma_lo_mn(ring + stage * S::STAGE, KT * 128);
                constexpr int STEPS = KT / 16;
                if constexpr (HD == 256) {
                    wait(rest, turn ^ 1);
                    tc_fence_after();
                    if (elect_one()) {
                        pv_steps(IntC<0>(), IntC<STEPS>(), p, vb, d);
                        umma_commit(done);
                        umma_commit(release);
                    }
                } else {
                    // the first keys' weights while the softmax is still at the others
                    wait(half, turn);
                    tc_fence_after();
                    if (elect_one()) pv_steps(IntC<0>(), IntC<STEPS / 2>(), p, vb, d);
                    __syncwarp();
                    wait(rest, turn ^ 1);
                    tc_fence_after();
                    if (elect_one()) {
                        pv_steps(IntC<STEPS / 2>(), IntC<STEPS / 2>(), p, vb, d);
                        umma_commit(done);
                        if (release) umma_commit(release);
                    }
                }
                __syncwarp();
            };
            uint32_t t = next_tile(begin), jj = 0;
            if (t < tiles) {
                // the queries are in place once both softmax groups have arrived on p_full the first time
                wait(p_full + 0, 0);
                if (HD != 256) wait(p_full + 1, 0);
                wait(full + 0, 0);
                tc_fence_after();
                if constexpr (HD == 256) {
                    qk(0, 0, tmem + S::S_COL(0), s_full + 0, empty + 0);
                } else {
                    qk(0, 0, tmem + S::S_COL(0), s_full + 0, nullptr);
                    qk(1, 0, tmem + S::S_COL(1), s_full + 1, empty + 0);
                }
                while (t < tiles) {
                    const uint32_t tn = next_tile(t + 1);
                    const uint32_t nv = 2 * jj + 1, nk = 2 * jj + 2;
                    if constexpr (HD == 256) {
                        if (tn < tiles) {
                            wait(full + nk % NS, (nk / NS) & 1);
                            tc_fence_after();
                            qk(0, nk % NS, tmem + S::S_COL((jj + 1) & 1), s_full + ((jj + 1) & 1), empty + nk % NS);
                        }
                        wait(full + nv % NS, (nv / NS) & 1);
                        pv(tmem + S::S_COL(jj & 1), nv % NS, tmem + S::O_COL(0), nullptr, p_full + 0, jj & 1, o_full + 0,
                           empty + nv % NS);
                    } else {
                        wait(full + nv % NS, (nv / NS) & 1);
                        pv(tmem + S::S_COL(0), nv % NS, tmem + S::O_COL(0), p_half + 0, p_full + 0, jj & 1, o_full + 0, nullptr);
                        if (tn < tiles) {
                            wait(full + nk % NS, (nk / NS) & 1);
                            tc_fence_after();
                            qk(0, nk % NS, tmem + S::S_COL(0), s_full + 0, nullptr);
                        }
                        pv(tmem + S::S_COL(1), nv % NS, tmem + S::O_COL(1), p_half + 1, p_full + 1, jj & 1, o_full + 1,
                           empty + nv % NS);
                        if (tn < tiles) qk(1, nk % NS, tmem + S::S_COL(1), s_full + 1, empty + nk % NS);
                    }
                    t = tn;
                    jj++;
                }
                // no product either, nor its arrival
                if (elect_one()) umma_commit(mma_end);
                __syncwarp();
                wait_always(mma_end, 0);
            }
        }
    } else {
        // ── softmax: one row per thread ──
        regs_inc<S::REGS_SOFTMAX>();
        const int wg = warp >> 2, r = tid & 127, tile = HD == 256 ? 0 : wg;
        constexpr int CW = HD == 256 ? 32 : KT;          // score columns of this thread
        constexpr int OW = HD == 256 ? 128 : HD;         // output columns
        const int half = HD == 256 ? wg : 0;
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t R = R0 + tile * 128 + r;
        const bool real = R < rows;
        // Registers are what this part is short of (o alone takes OW): positions are 32 bits
        // wide here (a length is at most 2^30), and the row's addresses are computed again at the end.
        auto token_of = [&]() { return real ? R / a.group : 0; };
        auto head_of = [&]() { return kh * a.group + (real ? R % a.group : 0); };
        auto q_of = [&]() { return a.q + (uint64_t)(c0 + token_of()) * a.q_stride + (uint64_t)head_of() * HD; };
        const int row_i = (int)((int64_t)len - nq + token_of());
        const int row_lo = a.window ? (int)max((int64_t)0, (int64_t)row_i - a.window + 1) : 0;
        int row_hi = a.causal ? (int)min((int64_t)len, max((int64_t)row_i + 1, (int64_t)prefix)) : (int)len;
        uint32_t row_doc = 0;
        const float row_slope = EXTRA && a.slopes ? a.slopes[head_of()] : 0.0f;
        if (docs) {
            if (row_i >= 0)
                row_doc = docs[row_i];
            else
                row_hi = 0;
        }
        if (!real) row_hi = 0;
        // Queries to two f16 planes: a warp takes its 32 rows (head_dim 256: each group half of
        // them) eight at a time, the next eight on their way.  A rolled loop: unrolled over
        // the rows, fetching its instructions took longer than its loads.
        const float f0 = EXTRA && a.softcap != 0.0f ? a.scale / a.softcap : a.scale * 1.4426950408889634f;
        float rf = 0.0f;
        {
            constexpr int PER = HD / 32, B = 8, MINE = HD == 256 ? 16 : 32;
            const int x_first = HD == 256 ? 16 * wg : 0;
            const int n_rows = (int)min((int64_t)32, max((int64_t)0, (int64_t)rows - (R - lane)));  // of this warp's 32
            const uint64_t row_q = reinterpret_cast<uint64_t>(q_of());
            float v[2][B][PER];
            auto load = [&](int x0, float(&w)[B][PER]) {
#pragma unroll
                for (int y = 0; y < B; y++) {
                    const float *src = reinterpret_cast<const float *>(__shfl_sync(0xffffffffu, row_q, (x0 + y) & 31));
#pragma unroll
                    for (int e = 0; e < PER; e += 2) {
                        const float2 z = x0 + y < n_rows ? *reinterpret_cast<const float2 *>(src + 32 * e + 2 * lane) : make_float2(0.0f, 0.0f);
                        w[y][e] = z.x;
                        w[y][e + 1] = z.y;
                    }
                }
            };
            auto convert = [&](int x0, const float(&w)[B][PER]) {
#pragma unroll
                for (int y = 0; y < B; y++) {
                    const uint32_t rr = (warp & 3) * 32 + x0 + y;
                    float top = 0.0f;
#pragma unroll
                    for (int e = 0; e < PER; e++) top = fmaxf(top, fabsf(w[y][e]));
                    top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
                    float up = 1.0f;
                    if (top > 0.0f && top < INFINITY) {
                        const int ex = min(max(8 - (int)(__float_as_uint(top) >> 23) + 127, -126), 126);
                        up = __uint_as_float((uint32_t)(ex + 127) << 23);
                    }
                    if (lane == x0 + y) rf = f0 / up;
                    const float sg = f0 < 0.0f ? -up : up;  // the factor on the scores stays positive
#pragma unroll
                    for (int e = 0; e < PER; e += 2) {
                        uint32_t h, l;
                        split_f16x2(w[y][e] * sg, w[y][e + 1] * sg, h, l);
                        const uint32_t at = tile * 2 * S::QPLANE + (e / 2) * 16384 + sw128_offset(rr, 2 * lane);
                        *reinterpret_cast<uint32_t *>(smem + at) = h;
                        *reinterpret_cast<uint32_t *>(smem + at + S::QPLANE) = l;
                    }
                }
            };
            load(x_first, v[0]);
#pragma unroll 1
            for (int x0 = x_first; x0 < x_first + MINE; x0 += 2 * B) {
                load(x0 + B, v[1]);
                convert(x0, v[0]);
                if (x0 + 2 * B < x_first + MINE) load(x0 + 2 * B, v[0]);
                convert(x0 + B, v[1]);
            }
            fence_async_smem();
        }
        if constexpr (HD == 256) {  // the two groups have each other's rows' factors
            tmem_st1(tmem + lane_base + S::X_COL + wg, rf);
            tmem_wait_st();
            tc_fence_before();
            named_sync<2, 256>();
            tc_fence_after();
            const float r0 = tmem_ld1(tmem + lane_base + S::X_COL), r1 = tmem_ld1(tmem + lane_base + S::X_COL + 1);
            rf = lane < 16 ? r0 : r1;
            tc_fence_before();
            named_sync<2, 256>();
            tc_fence_after();
        }
        // never 0, by which a masked score's -inf would become NaN: products are below 1e10, so the least
        // normal number makes nothing of them either
        rf = fmaxf(fabsf(rf), 1.17549435e-38f);
        if (skipping) named_sync<3, kPpThreads>();
        mbar_arrive(p_full + tile);

        float o[OW];
#pragma unroll
        for (int e = 0; e < OW; e++) o[e] = 0.0f;
        float m = -INFINITY, l = 0.0f, alpha = 1.0f;
        const uint32_t o_addr = tmem + lane_base + S::O_COL(tile) + half * 128;
        auto add_o = [&]() {  // o = o * alpha + this tile's product
            uint32_t v[2][16];
            const float2 al2 = make_float2(alpha, alpha);
            tmem_ld16(o_addr, v[0]);
#pragma unroll
            for (int c = 0; c < OW; c += 16) {
                uint32_t(&u)[16] = v[(c / 16) & 1];
                tmem_wait_ld(u);
                if (c + 16 < OW) tmem_ld16(o_addr + c + 16, v[(c / 16 + 1) & 1]);
#pragma unroll
                for (int e = 0; e < 16; e += 2) {
                    const float2 x = ffma2(make_float2(o[c + e], o[c + e + 1]), al2,
                                           make_float2(__uint_as_float(u[e]), __uint_as_float(u[e + 1])));
                    o[c + e] = x.x;
                    o[c + e + 1] = x.y;
                }
            }
        };
        uint32_t jj = 0;
        for (uint32_t t = next_tile(begin); t < tiles; t = next_tile(t + 1), jj++) {
            const int sb = HD == 256 ? (jj & 1) : tile;
            const uint32_t s_addr = tmem + lane_base + S::S_COL(sb) + half * 32;
            const int k0 = (int)(lo + t * KT) + half * 32;
            wait(s_full + sb, HD == 256 ? (jj / 2) & 1 : jj & 1);
            __syncwarp();
            tc_fence_after();
            // whether every row of the warp sees all of its columns, documents aside and altogether
            const bool in_range = __all_sync(0xffffffffu, (row_lo <= k0 && k0 + CW <= row_hi) || !real);
            const bool plain = in_range && !docs;
            // pass 1: the row's maximum; capped, biased or masked scores go back to tensor
            // memory.  Each load runs while the columns before it are worked on.
            float top = -INFINITY;
            const float *zs = scales_s + (jj % S::DOCS) * 3 * S::GROUPS + half * 2;  // this thread's columns' scales, 16 to each
            // the factor on 16 columns' raw scores: not 0, by which a masked score's -inf would become NaN
            auto factor = [&](int c) { return fmaxf(rf * zs[c / 16], 1.17549435e-38f); };
            {
                uint32_t v[2][16];
                tmem_ld16(s_addr, v[0]);
                const int from = max(0, min(CW, row_lo - k0));
                const int to = max(0, min(CW, row_hi - k0));
                const float dist = (float)(row_i - k0);
                constexpr int UNROLL = EXTRA ? 2 : CW / 16;  // the capped path is long: keep it in the instruction cache
#pragma unroll UNROLL
                for (int c = 0; c < CW; c += 16) {
                    uint32_t(&u)[16] = v[(c / 16) & 1];
                    tmem_wait_ld(u);
                    if (c + 16 < CW) tmem_ld16(s_addr + c + 16, v[(c / 16 + 1) & 1]);
                    if (!EXTRA && plain) {
                        float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
                        for (int e = 0; e < 16; e += 4) {
                            x0 = fmaxf(fmaxf(x0, __uint_as_float(u[e])), __uint_as_float(u[e + 1]));
                            x1 = fmaxf(fmaxf(x1, __uint_as_float(u[e + 2])), __uint_as_float(u[e + 3]));
                        }
                        if constexpr (Q8) {
                            top = fmaxf(top, fmaf(fmaxf(x0, x1), factor(c), zs[S::GROUPS + c / 16]));
                        } else {
                            top = fmaxf(top, fmaxf(x0, x1));
                        }
                        continue;
                    }
                    if (EXTRA) {  // score_log2, the usual case two at a time
                        constexpr float kLog2e = 1.4426950408889634f;
                        float big = 0.0f;
#pragma unroll
                        for (int e = 0; e < 16; e++) big = fmaxf(big, fabsf(__uint_as_float(u[e])));
                        const float f1 = Q8 ? rf * zs[c / 16] : rf;
                        const float2 f2 = make_float2(f1, f1);
                        if (a.softcap == 0.0f) {
#pragma unroll
                            for (int e = 0; e < 16; e += 2) {
                                const float2 x = fmul2(make_float2(__uint_as_float(u[e]), __uint_as_float(u[e + 1])), f2);
                                u[e] = __float_as_uint(x.x);
                                u[e + 1] = __float_as_uint(x.y);
                            }
                        } else if (__all_sync(0xffffffffu, big * f1 <= kTanhSmall)) {
                            const float2 cl = make_float2(a.softcap * kLog2e, a.softcap * kLog2e);
#pragma unroll
                            for (int e = 0; e < 16; e += 2) {
                                float2 x = fmul2(make_float2(__uint_as_float(u[e]), __uint_as_float(u[e + 1])), f2);
                                x = fmul2(tanh_small2(x), cl);
                                u[e] = __float_as_uint(x.x);
                                u[e + 1] = __float_as_uint(x.y);
                            }
                        } else {
#pragma unroll
                            for (int e = 0; e < 16; e++)
                                u[e] = __float_as_uint(tanh_any(__uint_as_float(u[e]) * f1) * (a.softcap * kLog2e));
                        }
                        if (a.slopes) {
                            const float sl = -row_slope * kLog2e;
#pragma unroll
                            for (int e = 0; e < 16; e++)
                                u[e] = __float_as_uint(fmaf(sl, fabsf(dist - (float)(c + e)), __uint_as_float(u[e])));
                        }
                    }
                    constexpr uint32_t kMinusInf = 0xff800000u;
                    if (!in_range) {
#pragma unroll
                        for (int e = 0; e < 16; e++) u[e] = c + e >= from && c + e < to ? u[e] : kMinusInf;
                    }
                    if (docs) {
                        const uint4 *dn = reinterpret_cast<const uint4 *>(docs_s + (jj % S::DOCS) * KT + half * 32 + c);
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const uint4 d = dn[e];
                            u[4 * e] = d.x == row_doc ? u[4 * e] : kMinusInf;
                            u[4 * e + 1] = d.y == row_doc ? u[4 * e + 1] : kMinusInf;
                            u[4 * e + 2] = d.z == row_doc ? u[4 * e + 2] : kMinusInf;
                            u[4 * e + 3] = d.w == row_doc ? u[4 * e + 3] : kMinusInf;
                        }
                    }
                    if constexpr (Q8) {
                        float x = -INFINITY;
#pragma unroll
                        for (int e = 0; e < 16; e++) x = fmaxf(x, __uint_as_float(u[e]));
                        top = fmaxf(top, fmaf(x, EXTRA ? 1.0f : factor(c), zs[S::GROUPS + c / 16]));
                    } else {
#pragma unroll
                        for (int e = 0; e < 16; e++) top = fmaxf(top, __uint_as_float(u[e]));
                    }
                    tmem_st16(s_addr + c, u);
                }
                if (EXTRA || !plain) tmem_wait_st();
            }
            const float fs = EXTRA ? 1.0f : rf;
            if (!Q8) top = top == -INFINITY ? top : top * fs;
            if constexpr (HD == 256) {  // the other half's maximum; the columns alternate with the tiles
                const uint32_t x_addr = tmem + lane_base + S::X_COL + 2 * (jj & 1);
                tmem_st1(x_addr + wg, top);
                tmem_wait_st();
                tc_fence_before();
                named_sync<2, 256>();
                tc_fence_after();
                const float other = tmem_ld1(x_addr + (wg ^ 1));
                top = fmaxf(top, other);
            }
            const float mn = fmaxf(m, top);
            const float al = mn == m ? 1.0f : ex2(m - mn);
            m = mn;
            // weights times 2^10: small ones keep their f16 bits, and the sum carries the same factor
            const float base = m == -INFINITY ? 0.0f : 10.0f - m;
            float2 sum = make_float2(0.0f, 0.0f);
            // 8-bit codes: the columns' sums, each times its 1 / v.  NaN where the row sees a scale that cannot be used, whatever
            // the distance bias leaves of the weights there (asked of every 16 columns: 8-bit 4096 tokens with a bias,
            // 32/4 heads of 128, 311 -> 323 us; so 311)
            float weight = Q8 && top > kQ8NoScore ? __int_as_float(0x7fffffff) : 0.0f;
            {
                float2 fs2 = make_float2(fs, fs), base2 = make_float2(base, base);
                uint32_t v[2][16];
                tmem_ld16(s_addr, v[0]);
#pragma unroll
                for (int c = 0; c < CW; c += 16) {
                    uint32_t(&u)[16] = v[(c / 16) & 1];
                    uint32_t p[16];
                    tmem_wait_ld(u);
                    if (c + 16 < CW) tmem_ld16(s_addr + c + 16, v[(c / 16 + 1) & 1]);
                    if constexpr (Q8) {
                        const float f1 = EXTRA ? 1.0f : factor(c), b1 = base + zs[S::GROUPS + c / 16];
                        fs2 = make_float2(f1, f1);
                        base2 = make_float2(b1, b1);
                        sum = make_float2(0.0f, 0.0f);
                    }
#pragma unroll
                    for (int e = 0; e < 16; e += 2) {
                        float2 x = ffma2(make_float2(__uint_as_float(u[e]), __uint_as_float(u[e + 1])), fs2, base2);
                        x.x = ex2(x.x);
                        x.y = ex2(x.y);
                        sum = fadd2(sum, x);
                        split_weights(x.x, x.y, p[e / 2], p[8 + e / 2]);
                    }
                    if constexpr (Q8) {
                        const float all = sum.x + sum.y;
                        if (all != 0.0f) weight = fmaf(all, zs[2 * S::GROUPS + c / 16], weight);
                    }
                    tmem_st16(s_addr + c, p);
                    if (HD != 256 && c + 16 == CW / 2) {
                        tmem_wait_st();
                        tc_fence_before();
                        mbar_arrive(p_half + tile);
                    }
                }
            }
            tmem_wait_st();
            l = fmaf(l, al, Q8 ? weight : sum.x + sum.y);
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
        }
        // rows to the output through shared memory (this row tile's query planes are
        // no longer read), 32 columns at a time, so that stores fill whole lines
        float inv = l > 0.0f ? __fdiv_rn(1.0f, l) : (l == 0.0f ? 0.0f : l);
        float off = l - l;
#pragma unroll
        for (int e = 0; e < OW; e++) off += o[e] - o[e];
        bool fine = Q8 || off == 0.0f;  // codes are always finite: a masked one is nothing times a weight of 0
        constexpr int PITCH = 36;
        float *st = reinterpret_cast<float *>(smem + tile * 2 * S::QPLANE) + (HD == 256 ? warp : warp & 3) * 32 * PITCH;
        uint64_t dst = reinterpret_cast<uint64_t>(a.out + (uint64_t)(c0 + token_of()) * a.out_stride + (uint64_t)head_of() * HD + half * 128);
        if (a.nsplit > 1) {  // a record for k_paged_prompt_join: sums as they are, maximum and weight sum
            const uint64_t rec = (((uint64_t)s * a.kv.n_kv + kh) * a.row_blocks + rb) * a.nsplit + split;
            const uint64_t row = rec * S::ROWS + tile * 128 + r;
            dst = reinterpret_cast<uint64_t>(a.part_o + row * HD + half * 128);
            if (real && half == 0) *reinterpret_cast<float2 *>(a.part_ml + 2 * row) = make_float2(m, l);
            inv = 1.0f;
            fine = true;
        }
        const uint32_t fine_rows = __ballot_sync(0xffffffffu, fine && real);
#pragma unroll
        for (int c = 0; c < OW; c += 32) {
            __syncwarp();
#pragma unroll
            for (int e = 0; e < 32; e += 4)
                *reinterpret_cast<float4 *>(st + lane * PITCH + e) =
                    make_float4(o[c + e] * inv, o[c + e + 1] * inv, o[c + e + 2] * inv, o[c + e + 3] * inv);
            __syncwarp();
#pragma unroll
            for (int x = 0; x < 8; x++) {
                const int rr = x * 4 + lane / 8;
                float *to = reinterpret_cast<float *>(__shfl_sync(0xffffffffu, dst, rr));
                if (fine_rows >> rr & 1u)
                    *reinterpret_cast<float4 *>(to + c + lane % 8 * 4) =
                        *reinterpret_cast<const float4 *>(st + rr * PITCH + lane % 8 * 4);
            }
        }
        if constexpr (!Q8) {
            uint32_t again = __ballot_sync(0xffffffffu, real && !fine && !*dead);
            for (; again; again &= again - 1) slow_row<HD>(a, s, kh, R - lane + __ffs(again) - 1, half * 128, OW);
        }
        tc_fence_before();
    }
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Rows whose keys several CTAs share: one warp per row, the records in order.
// Grid (row steps, n_kv, n_seq).
constexpr int kPpJoinRows = 8;

template <int HD, bool Q8>
__global__ void __launch_bounds__(kPpJoinRows * 32) k_paged_prompt_join(const __grid_constant__ PagedAttnArgs a) {
    using S = PpShape<HD>;
    constexpr int PER = HD / 64;  // float2 per lane
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t s = blockIdx.z, kh = blockIdx.y, R = blockIdx.x * kPpJoinRows + threadIdx.x / 32;
    const int lane = threadIdx.x & 31;
    const uint32_t c0 = a.cu[s], c1 = a.cu[s + 1];
    if (!(c0 <= c1 && c1 <= a.total_q && c1 - c0 <= a.max_q) || R >= (c1 - c0) * a.group) return;
    const uint64_t rec = (((uint64_t)s * a.kv.n_kv + kh) * a.row_blocks + R / S::ROWS) * a.nsplit;
    const uint64_t row = rec * S::ROWS + R % S::ROWS;  // of split 0; a split's is S::ROWS further
    float m = -INFINITY, l = 0.0f;
    if ((uint32_t)lane < a.nsplit) {  // nsplit <= 32
        const float2 ml = *reinterpret_cast<const float2 *>(a.part_ml + 2 * (row + (uint64_t)lane * S::ROWS));
        m = ml.x;
        l = ml.y;
    }
    float top = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float w = m == -INFINITY ? 0.0f : ex2(m - top);
    l = warp_sum(l * w);
    float2 acc[PER];
#pragma unroll
    for (int e = 0; e < PER; e++) acc[e] = make_float2(0.0f, 0.0f);
#pragma unroll 4
    for (uint32_t i = 0; i < a.nsplit; i++) {
        const float wi = __shfl_sync(0xffffffffu, w, i);
        const float *src = a.part_o + (row + (uint64_t)i * S::ROWS) * HD + 2 * lane;
#pragma unroll
        for (int e = 0; e < PER; e++) {
            const float2 v = *reinterpret_cast<const float2 *>(src + 64 * e);
            acc[e].x = fmaf(v.x, wi, acc[e].x);
            acc[e].y = fmaf(v.y, wi, acc[e].y);
        }
    }
    const float inv = l > 0.0f ? __fdiv_rn(1.0f, l) : (l == 0.0f ? 0.0f : l);
    float off = l - l;
#pragma unroll
    for (int e = 0; e < PER; e++) off += (acc[e].x - acc[e].x) + (acc[e].y - acc[e].y);
    if (Q8 || __all_sync(0xffffffffu, off == 0.0f)) {
        float *dst = a.out + (uint64_t)(c0 + R / a.group) * a.out_stride + (uint64_t)(kh * a.group + R % a.group) * HD + 2 * lane;
#pragma unroll
        for (int e = 0; e < PER; e++) *reinterpret_cast<float2 *>(dst + 64 * e) = make_float2(acc[e].x * inv, acc[e].y * inv);
    } else if constexpr (!Q8) {
        slow_row<HD>(a, s, kh, R, 0, HD);
    }
}

namespace {

using EncodeTiledFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                   const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_tiled() {
    static EncodeTiledFn fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
                        q == cudaDriverEntryPointSuccess;
        if (!ok) cudaGetLastError();
        return ok ? reinterpret_cast<EncodeTiledFn>(p) : nullptr;
    }();
    return fn;
}

// Maps of the pool, or rows = 0 where its pages or strides do not allow them.
void pp_maps(const PagedKvDev &kv, uint32_t tile, PpMaps &m) {
    m.rows = 0;
    uint32_t rows = tile;
    while (kv.page_size % rows) rows /= 2;  // tile is a power of two: the largest box in both
    const uint64_t most = 1ull << 40;
    if (rows < 8 || kv.slot_stride >= most || kv.head_stride >= most || kv.page_stride >= most) return;
    EncodeTiledFn fn = encode_tiled();
    if (!fn) return;
    const cuuint64_t dims[4] = {kv.hd, kv.page_size, kv.n_kv, kv.n_pages};
    const cuuint64_t strides[3] = {kv.slot_stride, kv.head_stride, kv.page_stride};
    const cuuint32_t box[4] = {64, rows, 1, 1}, step[4] = {1, 1, 1, 1};
    for (int i = 0; i < 2; i++)
        if (fn(i ? &m.v : &m.k, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, i ? kv.v : kv.k, dims, strides, box, step,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return;
    m.rows = rows;
}

// Row blocks that leave SMs without work share their keys among several CTAs:
// as many as fill the SMs, each with at least two tiles of the longest row.
template <int HD>
void pp_split(PagedAttnArgs &a, int num_sms) {
    using S = PpShape<HD>;
    a.row_blocks = (uint32_t)(((uint64_t)a.max_q * a.group + S::ROWS - 1) / S::ROWS);
    const uint64_t ctas = (uint64_t)a.row_blocks * a.kv.n_kv * a.n_seq, tiles = (a.max_len + S::KT - 1) / S::KT;
    a.nsplit = (uint32_t)max((uint64_t)1, min(min((uint64_t)num_sms / ctas, tiles / 2), (uint64_t)32));
}

void pp_split(PagedAttnArgs &a, int num_sms) {
    a.kv.hd == 64 ? pp_split<64>(a, num_sms) : a.kv.hd == 128 ? pp_split<128>(a, num_sms) : pp_split<256>(a, num_sms);
}

uint32_t pp_rows(const PagedAttnArgs &a) { return a.kv.hd == 256 ? PpShape<256>::ROWS : PpShape<128>::ROWS; }
static_assert(PpShape<64>::ROWS == PpShape<128>::ROWS, "one branch for both");

uint64_t pp_records(const PagedAttnArgs &a) {  // rows of all records
    return (uint64_t)a.n_seq * a.kv.n_kv * a.row_blocks * a.nsplit * pp_rows(a);
}

// Most rows for the kernel of single tokens, over a cache of more than 256 positions and of fewer (see paged_prompt_supported).
struct PpFew {
    uint32_t rows, rows_short;
};
PpFew pp_few(const PagedKvDev &kv) {
    if (!kv.k_scale) return {16, 32};
    return kv.hd == 64 ? PpFew{56, 56} : kv.hd == 128 ? PpFew{36, 80} : PpFew{26, 16};
}

template <int HD, bool EXTRA, bool Q8>
cudaError_t pp_launch(const LaunchCfg &c, const PagedAttnArgs &a) {
    using S = PpShape<HD, Q8>;
    PpMaps maps;
    maps.rows = 0;
    if (!Q8) pp_maps(a.kv, S::KT, maps);
    const uint64_t ctas = (uint64_t)a.row_blocks * a.nsplit * a.kv.n_kv * a.n_seq;
    if (ctas > 0x7fffffffull) return cudaErrorInvalidValue;
    cudaError_t e = launch_k(c, "paged_prompt", k_paged_prompt<HD, EXTRA, Q8>, dim3((uint32_t)ctas), dim3(S::THREADS), S::SMEM, a,
                             maps);
    if (e != cudaSuccess || a.nsplit == 1) return e;
    const uint32_t rows = a.max_q * a.group;
    return launch_k(c, "paged_prompt_join", k_paged_prompt_join<HD, Q8>,
                    dim3((rows + kPpJoinRows - 1) / kPpJoinRows, a.kv.n_kv, a.n_seq), dim3(kPpJoinRows * 32), 0, a);
}

// The register split needs the registers that a block is launched with.
template <int HD, bool EXTRA, bool Q8>
bool pp_regs() {
    cudaFuncAttributes f;
    if (cudaFuncGetAttributes(&f, k_paged_prompt<HD, EXTRA, Q8>) == cudaSuccess) return f.numRegs >= PpShape<HD, Q8>::REGS;
    cudaGetLastError();
    return false;
}

template <bool Q8>
bool pp_regs_all() {
    return pp_regs<64, false, Q8>() && pp_regs<64, true, Q8>() && pp_regs<128, false, Q8>() && pp_regs<128, true, Q8>() &&
           pp_regs<256, false, Q8>() && pp_regs<256, true, Q8>();
}

template <bool Q8>
cudaError_t pp_launch_hd(const LaunchCfg &c, const PagedAttnArgs &a) {
    const bool extra = a.softcap != 0.0f || a.slopes;
    switch (a.kv.hd) {
    case 64: return extra ? pp_launch<64, true, Q8>(c, a) : pp_launch<64, false, Q8>(c, a);
    case 128: return extra ? pp_launch<128, true, Q8>(c, a) : pp_launch<128, false, Q8>(c, a);
    case 256: return extra ? pp_launch<256, true, Q8>(c, a) : pp_launch<256, false, Q8>(c, a);
    default: return cudaErrorInvalidValue;
    }
}

}  // namespace

bool paged_prompt_supported(const PagedAttnArgs &a) {
    static const bool regs = pp_regs_all<false>(), regs_q8 = pp_regs_all<true>();
    // Few rows: the kernel for single tokens reads the cache once per 8 rows.  Measured there and here,
    // over head_dim 64, 128 and 256: 8 rows of 8 sequences of 8000 cached tokens 23, 41 and 114 us and
    // 30, 65 and 206; 16 rows of them 33, 59 and 218 us and 30, 69 and 206; 32 rows 52, 99 and 424 us and
    // 30, 68 and 207.  A cache of 60 tokens: 28 to 32 rows 7.3, 7.8 and 19.5 us and 10.2, 12.6 and 13.7,
    // 56 rows 16, 18 and 20 us and 10, 13 and 14; of 200 tokens, 16 rows 16, 17 and 19 us and 13, 16 and 16.
    // 8-bit codes, the same shapes: 56 rows of 8000 tokens 34 and 34 us (head_dim 64), 32 and 48 rows 64, 90 and 70, 73 (128),
    // 24 and 32 rows 165, 222 and 176, 176 (256); of 200 tokens, 64 and 96 rows 14, 20 and 18, 18.5 (128), 16 rows 18.5 and 18 (256).
    const uint64_t rows = (uint64_t)a.max_q * a.group;
    if (a.kv.k_scale ? !regs_q8 : !regs || !a.kv.f16) return false;
    const PpFew few = pp_few(a.kv);
    return rows > (a.max_len > 256 ? few.rows : few.rows_short);
}

size_t paged_prompt_scratch(PagedAttnArgs a, int num_sms) {
    pp_split(a, num_sms);
    return a.nsplit == 1 ? 0 : pp_records(a) * (a.kv.hd + 2) * 4;
}

// Enough for this call and for every smaller one, so that an op run once at its largest sizes has its scratch when a
// smaller call is recorded.  Only smaller calls may share their keys, and there are records only where a launch has no
// more CTAs than SMs; the fewest rows take the other kernel with its own scratch (a call that does so itself may have
// smaller ones of as many rows here, where a shorter cache has the lower bound).
size_t paged_prompt_scratch_most(const PagedAttnArgs &a, int num_sms) {
    const uint32_t least = min(pp_few(a.kv).rows, pp_few(a.kv).rows_short), most = max(pp_few(a.kv).rows, pp_few(a.kv).rows_short);
    const size_t records = (uint64_t)a.max_q * a.group > least ? (size_t)num_sms * pp_rows(a) * (a.kv.hd + 2) * 4 : 0;
    PagedAttnArgs few = a;
    few.max_q = min(a.max_q, most / a.group);
    if (!few.max_q) return records;
    return max(records, few.kv.k_scale ? paged_q8_attn_scratch(few, num_sms) : paged_attn_scratch(few, num_sms));
}

cudaError_t launch_paged_prompt(const LaunchCfg &c, PagedAttnArgs a, uint8_t *scratch) {
    a.err = c.dev_err;
    pp_split(a, c.num_sms);
    a.part_o = (float *)scratch;
    a.part_ml = a.part_o + (a.nsplit == 1 ? 0 : pp_records(a) * a.kv.hd);
    return a.kv.k_scale ? pp_launch_hd<true>(c, a) : pp_launch_hd<false>(c, a);
}

}  // namespace lt
