// lt_paged_q8_attn.cu — attention over a paged cache of 8-bit codes: one new token
// per sequence, and a few.
//
// The formulas are lt_paged_attn.cu's, with the blocks' scales as lt_paged_q8.cuh puts
// them, in one pass over the keys with the running maximum m and sum l.
//
// Bound: memory for many or long sequences (K and V are read once per 8 query heads of a
// KV head), latency for few; the work is shared as lt_paged_walk.cuh says.  One B200: 64
// sequences of 200 to 8192 positions (32/4 heads of 128) 36.6 us, 4.0 TB/s; one of 130001
// 31.8 us, 4.2 TB/s; one of 8192 10.3 us; a window of 1024 (16/8 heads of 256) 10.7 us;
// 64 sequences, 14/2 heads of 64, 17.3 us.  Some 11 us of the long ones are the start (2 us of launch,
// lengths -> table -> codes), the merge and the join; while the codes stream, two warps to a scheduler
// issue in 39% of the cycles and wait for their own results in most others.  Three CTAs to an SM instead of two at
// head_dim 128, with pieces of 16 keys or rings of 2: 46.7 and 47.8 us.
// - Each warp owns KB keys of a tile and a ring of STAGES such pieces in shared memory,
//   filled by 16-byte asynchronous copies, with the pieces' scales beside them.  Rows of
//   codes lie one behind the other, their 16-byte columns permuted so that neither matrix
//   load meets a bank conflict.
// - Scores are sums of exact products: a query row becomes 32-bit integers (a power of two times
//   the row, its largest element in [2^29, 2^30)), those four signed 8-bit digits, in rows r and r + 8
//   of two operands of the integer tensor-core product with K's codes as they lie in memory.
// - Weights go in as two f16 terms (22 bits) in rows r and r + 8, against V's codes in
//   f16, where they are exact: a transposing 8-bit matrix load gives 4 keys of a dimension,
//   and a byte b next to 0x64 is the f16 number 1024 + b.
// - Keys are dealt to the columns of the score product so that a thread's scores are
//   those of 4 consecutive keys, as its weights have to be for the second product.
#include "lt_paged_q8.cuh"
#include "lt_paged_walk.cuh"

namespace lt {

template <int HD>
struct Q8Shape {
    static constexpr int KB = HD == 256 ? 16 : 32;          // keys per warp and tile
    static constexpr int NG = KB / 16;                      // groups of 16, each within a block and a page
    static constexpr int TILE = KB * kPaWarps;
    static constexpr int STAGES = 3;
    static constexpr int HALF = KB * HD;                    // bytes of K's codes, and of V's
    static constexpr int PIECE = 2 * HALF;
    static constexpr int RING = PIECE * STAGES * kPaWarps;
    static constexpr int SCALES = NG * 8;                   // bytes per piece: K and V scale of each group
    static constexpr int QSTEPS = HD / 32;
    static constexpr int QBYTES = QSTEPS * 1024;
    static constexpr int RECS = HD == 256 ? 2 : kPaWarps;   // merge records
    static constexpr int MERGE = RECS * kPaRows * HD * 4;
    static constexpr int UNION = QBYTES > MERGE ? QBYTES : MERGE;
    static constexpr int OFF_SCALES = RING + UNION;
    static constexpr int OFF_ML = OFF_SCALES + SCALES * STAGES * kPaWarps;  // (m, l) of each warp's rows
    static constexpr int OFF_ROWF = OFF_ML + kPaWarps * kPaRows * 8;
    static constexpr int SMEM = OFF_ROWF + kPaRows * 4;
    static constexpr int CTAS = HD == 64 ? 3 : 2;
};

// Place of 16-byte column c of row r of a piece.  Eight rows of a matrix load are 0-7 or 8-15 (V), or the 8
// of 16 whose second bit is alike (K, see key_of): the column's permutation differs among the rows of each.
template <int HD>
LT_DEVINL uint32_t q8_at(uint32_t r, uint32_t c) {
    const uint32_t b = ((r >> 1) ^ (r >> 3)) & 1;
    const uint32_t f = HD == 64 ? (r & 4) >> 1 | b : (r & 4) | (r & 1) << 1 | b;
    return r * HD + ((c ^ f) << 4);
}

// C[16x8] += A[16x32] B[32x8], signed bytes, exact.  Not volatile, as the f16 product: products may
// move between loads (which keep their order).
LT_DEVINL void mma_s8(int (&c)[4], const uint4 &a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
LT_DEVINL void mma_w(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Byte p of four words to a register each: d[p] = bytes p of x[0], x[1], x[2], x[3].
LT_DEVINL void bytes_across(const uint32_t (&x)[4], uint32_t (&d)[4]) {
    const uint32_t l01 = __byte_perm(x[0], x[1], 0x5140), l23 = __byte_perm(x[2], x[3], 0x5140);
    const uint32_t h01 = __byte_perm(x[0], x[1], 0x7362), h23 = __byte_perm(x[2], x[3], 0x7362);
    d[0] = __byte_perm(l01, l23, 0x5410), d[1] = __byte_perm(l01, l23, 0x7632);
    d[2] = __byte_perm(h01, h23, 0x5410), d[3] = __byte_perm(h01, h23, 0x7632);
}
// Two 16x16 matrices of bytes, transposed: lanes 0-15 give the first's rows, 16-31 the second's.
// Register i: bytes 4 (lane % 4) .. + 3 of column lane / 4 + 8 (i % 2) of matrix i / 2.
LT_DEVINL void ldsm_t8(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
LT_DEVINL void cp_async4(uint32_t dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
LT_DEVINL uint4 lds_u4(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}

// What the join needs to know of a unit that CTAs first .. first + n - 1 share.  The list has a place per unit
// (a.join_units: decode, where every unit is there) or, where there are more units than CTAs and for rows of prompts,
// one per CTA, for the unit that begins there and goes on elsewhere (n = 0: none does).
struct Q8Join {
    uint32_t first, n, rows, kh, rb, q0, unused[2];
};

// PLAIN: neither cap nor distance bias.
template <int HD, bool PROMPT, bool PLAIN>
__global__ void __launch_bounds__(kPaThreads, Q8Shape<HD>::CTAS) k_paged_q8(const __grid_constant__ PagedAttnArgs a) {
    using S = Q8Shape<HD>;
    constexpr int KB = S::KB, NG = S::NG, TILE = S::TILE, NB = HD / 8;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t s_scan[kPaWarps];
    __shared__ uint64_t s_rem;
    __shared__ uint32_t s_seq;
    __shared__ PaSeq s_q;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, j4 = lane & 3;
    uint8_t *qm = smem + S::RING;  // query fragments, then the merge records
    float *rec = reinterpret_cast<float *>(qm);
    float2 *ml = reinterpret_cast<float2 *>(smem + S::OFF_ML);
    float *rowf = reinterpret_cast<float *>(smem + S::OFF_ROWF);
    const uint32_t ring_u = smem_u32(smem) + warp * (S::PIECE * S::STAGES), qm_u = smem_u32(qm);
    const uint32_t scale_u = smem_u32(smem) + S::OFF_SCALES + warp * (S::SCALES * S::STAGES);
    const uint32_t c = blockIdx.x;
    pdl_launch_dependents();
    // Lengths, page table and queries towards L2 while the kernel before still runs (hints only: the values
    // are read after the wait).
    {
        const uint64_t line = ((uint64_t)c * kPaThreads + tid) * 32, entries = (uint64_t)a.n_seq * a.kv.max_pages;
        if (line < entries) prefetch_l2(a.table + line);
        if (tid < 32 && tid * 32 < a.n_seq) prefetch_l2(a.lens + tid * 32);
        if (tid == 32) prefetch_l2(a.q);
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
    if (c >= G) {
        if (!a.join_units && tid == 0) reinterpret_cast<Q8Join *>(a.unit_info)[c].n = 0;
        return;
    }
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
        if (f0 >= f1) {
            if (!a.join_units && tid == 0) reinterpret_cast<Q8Join *>(a.unit_info)[c].n = 0;
            return;
        }
        cw.template next_unit<TILE>(a);
    } else {
        cw.set_unit(a);
    }
    lw = cw;
    uint64_t lf = f0;  // lw's place in the count

    // a unit's queries: warp w takes rows 2 w and 2 w + 1, a lane 4 consecutive elements of each 128
    constexpr int QV = HD == 256 ? 2 : 1;
    float4 qv[2][QV];
    auto load_q = [&]() {
        const uint32_t rows = min((uint32_t)kPaRows, cw.q.nq * a.group - cw.rb * kPaRows);
#pragma unroll
        for (int rr = 0; rr < 2; rr++) {
            const uint32_t r = warp * 2 + rr, R = cw.rb * kPaRows + r;
            const float *src = a.q + (uint64_t)(cw.q.q0 + R / a.group) * a.q_stride + (uint64_t)(cw.kh * a.group + R % a.group) * HD;
#pragma unroll
            for (int e = 0; e < QV; e++)
                qv[rr][e] = r < rows && (HD != 64 || lane < 16) ? *reinterpret_cast<const float4 *>(src + 128 * e + 4 * lane)
                                                              : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
    };
    load_q();

    // The piece to copy next: a page for each of its groups, and where its slots begin there.  Whole groups are copied,
    // what lies outside the unit's positions too (codes may be anything, scores there are masked); groups wholly
    // outside are not.  This is a third of the instructions of a piece if left to 64-bit products of strides:
    // strides are below 2^32, and what the unit fixes is added up once per unit.
    constexpr int CH = HD / 16, STEP = 32 / CH;  // columns of a row, rows per copy instruction
    const uint32_t row0 = lane / CH, col0 = lane % CH;
    const uint32_t page_stride = (uint32_t)a.kv.page_stride, slot_stride = (uint32_t)a.kv.slot_stride;
    const uint64_t v_off = a.kv.v - a.kv.k, step_off = (uint64_t)STEP * slot_stride;
    uint32_t row_at[16 / STEP];
#pragma unroll
    for (int i = 0; i < 16 / STEP; i++) row_at[i] = ring_u + q8_at<HD>(row0 + i * STEP, col0);
    const uint32_t *row_table;   // of lw's unit: its sequence's page table,
    const uint8_t *head_k;       // its head's codes, from this lane's row and column on,
    const float *head_scale;     // and its head's scales, K's or (odd lanes) V's
    auto unit_base = [&]() {
        row_table = a.table + (uint64_t)lw.s * a.kv.max_pages;
        head_k = a.kv.k + (uint64_t)lw.kh * (uint32_t)a.kv.head_stride + (uint64_t)row0 * slot_stride + col0 * 16;
        head_scale = (lane & 1 ? a.kv.v_scale : a.kv.k_scale) + (uint64_t)lw.kh * a.kv.page_blocks;
    };
    unit_base();
    const uint32_t scales_per_page = a.kv.n_kv * a.kv.page_blocks;  // below 2^32: checked on the host
    struct Job {
        uint32_t page[NG], slot[NG];
        const uint8_t *k;
        const float *scale;
        bool there;
    };
    constexpr uint32_t kNone = 0xffffffffu;
    auto look = [&](Job &j) {
        const uint32_t key0 = lw.base + lw.tile * TILE + warp * KB;
#pragma unroll
        for (int n = 0; n < NG; n++) {
            const uint32_t key = key0 + 16 * n;
            uint32_t at;
            if (a.kv.page_shift != kNoShift) {
                at = key >> a.kv.page_shift;
                j.slot[n] = key & (a.kv.page_size - 1);
            } else {
                at = key / a.kv.page_size;
                j.slot[n] = key - at * a.kv.page_size;
            }
            j.page[n] = key < lw.hi && key + 16 > lw.lo ? row_table[at] : kNone;
        }
        j.k = head_k;
        j.scale = head_scale;
    };
    auto copy = [&](const Job &j, int stage) {
#pragma unroll
        for (int n = 0; n < NG; n++) {
            const uint32_t page = j.page[n];
            if (page >= a.kv.n_pages) {
                if (page != kNone) atomicExch(a.err, DEV_ERR_BAD_INDEX);
                continue;
            }
            const uint8_t *pk = j.k + (uint64_t)page * page_stride + (uint64_t)j.slot[n] * slot_stride;
            const uint32_t to = stage * S::PIECE + n * 16 * HD;
#pragma unroll
            for (int i = 0; i < 16 / STEP; i++) {
                cp_async16(to + row_at[i], pk, true);
                cp_async16(to + row_at[i] + S::HALF, pk + v_off, true);
                pk += step_off;
            }
            if (lane < 2)
                cp_async4(scale_u + stage * S::SCALES + n * 8 + lane * 4,
                          j.scale + (uint64_t)page * scales_per_page + (j.slot[n] >> a.kv.block_shift));
        }
    };
    // all pages of the first pieces are looked up before the first copy waits for its own
    Job jobs[S::STAGES];
    auto look_next = [&](Job &j) {
        j.there = lf < f1;
        if (!j.there) return;
        look(j);
        if (++lw.tile < lw.q.tiles) {
            lf++;
        } else {
            lf += 1 + kUnitCost;
            if (lf < f1) {
                lw.template next_unit<TILE>(a);
                unit_base();
            }
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
    bool continues = false;  // a unit begins here and goes on elsewhere
    while (f < f1) {
        // ── one segment: this CTA's tiles of one unit ──
        const uint32_t seg = (uint32_t)min((uint64_t)(cw.q.tiles - cw.tile), f1 - f);
        const uint64_t unit_f0 = f - cw.tile;
        const uint32_t rows = min((uint32_t)kPaRows, cw.q.nq * a.group - cw.rb * kPaRows);
        // queries to digits
#pragma unroll
        for (int rr = 0; rr < 2; rr++) {
            const uint32_t r = warp * 2 + rr;
            uint32_t top = 0;  // bits: NaN above infinity above every number
#pragma unroll
            for (int e = 0; e < QV; e++) {
                const float4 &v = qv[rr][e];
                top = max(max(top, max(__float_as_uint(v.x) & 0x7fffffffu, __float_as_uint(v.y) & 0x7fffffffu)),
                          max(__float_as_uint(v.z) & 0x7fffffffu, __float_as_uint(v.w) & 0x7fffffffu));
            }
            top = __reduce_max_sync(0xffffffffu, top);
            const int ex = min(max(29 - (int)(top >> 23) + 127, -126), 126);
            const float up = __uint_as_float((uint32_t)(ex + 127) << 23);
            const float f1 = a.softcap != 0.0f ? a.scale / a.softcap : a.scale * 1.4426950408889634f;
            if (lane == 0) rowf[r] = top < 0x7f800000u ? f1 / up : __int_as_float(0x7fffffff);
#pragma unroll
            for (int e = 0; e < QV; e++) {
                const float4 &v = qv[rr][e];
                uint32_t d[4];
                const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int i = 0; i < 4; i++) d[i] = ((uint32_t)__float2int_rn(x[i] * up) + 0x00808080u) ^ 0x00808080u;
                uint32_t p[4];
                bytes_across(d, p);
                const uint32_t k = 128 * e + 4 * lane;  // element: step k / 32, its half (k / 16) % 2, column (k / 4) % 4
                if (HD != 64 || lane < 16) {
                    uint8_t *at = qm + (k / 32) * 1024 + (r * 4 + (k / 4) % 4) * 16 + (k / 16) % 2 * 8;
                    *reinterpret_cast<uint2 *>(at) = make_uint2(p[3], p[2]);
                    *reinterpret_cast<uint2 *>(at + 512) = make_uint2(p[1], p[0]);
                }
            }
        }
        __syncthreads();
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
                if (a.prefix) row_hi = max(row_hi, (int)min(a.prefix[cw.s], cw.q.len));
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
        // Sums in registers; each piece's product is computed from zero and added here: the tensor core
        // truncates where it accumulates.
        float2 o[NB];
#pragma unroll
        for (int n = 0; n < NB; n++) o[n] = make_float2(0.0f, 0.0f);
        float m = -INFINITY, l = 0.0f;

        for (uint32_t it = 0; it < seg; it++) {
            cp_async_wait<S::STAGES - 2>();
            __syncwarp();
            // the piece before is done with: its place is filled before this one's products, so that two pieces
            // of each warp are on their way all the time (behind them: 64 ragged sequences 39.0 us, 36.6 so)
            int fill = stage + S::STAGES - 1;
            if (fill >= S::STAGES) fill -= S::STAGES;
            if (job.there) {
                copy(job, fill);
                look_next(job);
            }
            cp_async_commit();
            const uint32_t k0 = cw.base + cw.tile * TILE + warp * KB;  // the piece's first position
            if (k0 < cw.hi && k0 + KB > cw.lo) {
                const uint32_t kb = ring_u + stage * S::PIECE, vb = kb + S::HALF;
                float sc[4 * NG];  // positions k0 + 16 (i / 4) + 4 j4 + i % 4
                {
                    int s0[2 * NG][4], s1[2 * NG][4];
#pragma unroll
                    for (int n = 0; n < 2 * NG; n++)
#pragma unroll
                        for (int e = 0; e < 4; e++) s0[n][e] = s1[n][e] = 0;
                    // column x of product 2 n + h is key 16 n + 4 (x / 2) + 2 h + x % 2
                    const uint32_t x = lane & 7, key = 4 * (x >> 1) + (x & 1) + 2 * (lane >> 4), half = (lane >> 3) & 1;
#pragma unroll
                    for (int i = 0; i < S::QSTEPS; i++) {
                        const uint4 q0 = lds_u4(qm_u + i * 1024 + lane * 16), q1 = lds_u4(qm_u + i * 1024 + 512 + lane * 16);
#pragma unroll
                        for (int n = 0; n < NG; n++) {
                            uint32_t b[4];
                            ldsm4(b, kb + n * 16 * HD + q8_at<HD>(key, 2 * i + half));
                            mma_s8(s0[2 * n], q0, b[0], b[1]);
                            mma_s8(s1[2 * n], q1, b[0], b[1]);
                            mma_s8(s0[2 * n + 1], q0, b[2], b[3]);
                            mma_s8(s1[2 * n + 1], q1, b[2], b[3]);
                        }
                    }
#pragma unroll
                    for (int n = 0; n < 2 * NG; n++)
#pragma unroll
                        for (int e = 0; e < 2; e++)
                            sc[4 * (n / 2) + 2 * (n % 2) + e] =
                                fmaf((float)(s0[n][e] * 256 + s0[n][2 + e]), 65536.0f, (float)(s1[n][e] * 256 + s1[n][2 + e]));
                }
                float top = -INFINITY, v_inv[NG];
                const bool whole = !PROMPT && k0 >= cw.lo && k0 + KB <= cw.hi;
                const float dist = (float)(row_i - (int)(k0 + 4 * j4));
#pragma unroll
                for (int n = 0; n < NG; n++) {
                    float ks, vs;
                    asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(ks), "=f"(vs) : "r"(scale_u + stage * S::SCALES + n * 8) : "memory");
                    const Q8Scale z = q8_scale(ks, vs);
                    const float rk = rf * z.k;
                    v_inv[n] = z.v_inv;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        float &t = sc[4 * n + e];
                        const int j = (int)k0 + 16 * n + 4 * j4 + e;
                        t = PLAIN ? fmaf(t, rk, z.v_log2)
                                  : score_log2(t, rk, a.softcap, slope, fabsf(dist - (float)(16 * n + e))) + z.v_log2;
                        if (PROMPT) {
                            bool seen = j >= row_lo && j < row_hi;
                            if (docs && seen) seen = docs[j] == my_doc;
                            if (!seen) t = -INFINITY;
                        }
                    }
                }
                if (!PROMPT && !whole) {
#pragma unroll
                    for (int i = 0; i < 4 * NG; i++) {
                        const int j = (int)k0 + 16 * (i / 4) + 4 * j4 + i % 4;
                        if (j < row_lo || j >= row_hi) sc[i] = -INFINITY;
                    }
                }
#pragma unroll
                for (int i = 0; i < 4 * NG; i++) top = fmaxf(top, sc[i]);
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float mn = fmaxf(m, top);
                const float al = mn > m ? ex2(m - mn) : 1.0f;  // m = -inf: 0
                l *= al;
                m = mn;
                // weights scaled by 2^10 so that small ones keep their f16 bits; l carries the same factor
                const float base = m == -INFINITY ? 0.0f : m - 10.0f;
                uint32_t pa[NG][4];
#pragma unroll
                for (int n = 0; n < NG; n++) {
                    float sum = 0.0f;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        sc[4 * n + e] = ex2(sc[4 * n + e] - base);
                        sum += sc[4 * n + e];
                    }
                    l = fmaf(sum, v_inv[n], l);
                    split_f16x2(sc[4 * n], sc[4 * n + 1], pa[n][0], pa[n][1]);
                    split_f16x2(sc[4 * n + 2], sc[4 * n + 3], pa[n][2], pa[n][3]);
                }
                const float2 al2 = make_float2(al, al);
#pragma unroll
                for (int i = 0; i < HD / 32; i++) {
                    float p[4][4] = {};  // dims 32 i + 8 x ..
#pragma unroll
                    for (int n = 0; n < NG; n++) {
                        uint32_t w[4];
                        ldsm_t8(w, vb + n * 16 * HD + q8_at<HD>(lane & 15, 2 * i + (lane >> 4)));
#pragma unroll
                        for (int x = 0; x < 4; x++) {
                            uint32_t b0, b1;
                            s8_to_f16(w[x], b0, b1);
                            mma_w(p[x], pa[n], b0, b1);
                        }
                    }
#pragma unroll
                    for (int x = 0; x < 4; x++)
                        o[4 * i + x] = ffma2(o[4 * i + x], al2, fadd2(make_float2(p[x][0], p[x][1]), make_float2(p[x][2], p[x][3])));
                }
            }
            if (++stage == S::STAGES) stage = 0;
            if (it + 1 < seg) cw.tile++;
        }

        // ── merge the warps: each leaves its sums, then every thread adds up dims of its own, row by row.  This runs
        // once per unit: short loops, since fetching its instructions is most of its time (unrolled in registers, from
        // half the warps to the other half: 2.7 us) ──
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if (j4 == 0) ml[warp * kPaRows + g] = make_float2(m, l);
        // column of a record's row: 8 floats apart in the rows that a store of a warp's half touches
        auto rec_at = [](uint32_t w, uint32_t r, uint32_t d) { return (w * kPaRows + r) * HD + (d ^ ((r & 3) << 3)); };
        __syncthreads();  // every warp is done with the query fragments
        if constexpr (S::RECS == kPaWarps) {
#pragma unroll
            for (int n = 0; n < NB; n++) *reinterpret_cast<float2 *>(rec + rec_at(warp, g, 8 * n + 2 * j4)) = o[n];
        } else {  // two records: the upper warps' sums, to which the lower ones add theirs
            if (warp >= 2)
#pragma unroll
                for (int n = 0; n < NB; n++) *reinterpret_cast<float2 *>(rec + rec_at(warp - 2, g, 8 * n + 2 * j4)) = o[n];
            __syncthreads();
            if (warp < 2) {
                const float m2 = ml[(warp + 2) * kPaRows + g].x, mn = fmaxf(m, m2), from = mn == -INFINITY ? 0.0f : mn;
                const float w1 = ex2(m - from), w2 = ex2(m2 - from);
#pragma unroll
                for (int n = 0; n < NB; n++) {
                    float2 *at = reinterpret_cast<float2 *>(rec + rec_at(warp, g, 8 * n + 2 * j4));
                    const float2 t = *at;
                    *at = make_float2(o[n].x * w1 + t.x * w2, o[n].y * w1 + t.y * w2);
                }
            }
        }
        const uint32_t first = share.owner(unit_f0), last = share.owner(unit_f0 + cw.q.tiles - 1);
        const bool whole_unit = first == last, begins = unit_f0 == f;
        const uint64_t u = pa_unit(a, cw.s, cw.kh, cw.rb), part = 2 * (uint64_t)c + (begins ? 1 : 0);
        if (begins && tid == 0 && (a.join_units || !whole_unit))
            reinterpret_cast<Q8Join *>(a.unit_info)[a.join_units ? u : c] = {first, last - first + 1, rows, cw.kh, cw.rb, cw.q.q0, {0, 0}};
        continues |= begins && !whole_unit;
        __syncthreads();
        constexpr int D = HD / 4, RSTEP = kPaThreads / D;  // threads to a row, rows at a time
#pragma unroll 1
        for (uint32_t r = tid / D; r < rows; r += RSTEP) {
            const int d = tid % D * 4;
            float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            float top = ml[r].x, all = 0.0f;
#pragma unroll
            for (int w = 1; w < kPaWarps; w++) top = fmaxf(top, ml[w * kPaRows + r].x);
            const float from = top == -INFINITY ? 0.0f : top;
#pragma unroll
            for (int w = 0; w < kPaWarps; w++) {
                const float2 x = ml[w * kPaRows + r];
                all = fmaf(x.y, ex2(x.x - from), all);  // m = -inf: times 0, and l and the sums are 0 or NaN
                if (w >= S::RECS) continue;
                // a record's reference: its warp's, or the larger of the two that are in it
                const float y = S::RECS == kPaWarps ? x.x : fmaxf(x.x, ml[(w + 2) * kPaRows + r].x);
                const float f = ex2(y - from);
                const float4 v = *reinterpret_cast<const float4 *>(rec + rec_at(w, r, d));
                sum.x = fmaf(v.x, f, sum.x);
                sum.y = fmaf(v.y, f, sum.y);
                sum.z = fmaf(v.z, f, sum.z);
                sum.w = fmaf(v.w, f, sum.w);
            }
            float *dst;
            if (whole_unit) {
                const uint32_t row = cw.rb * kPaRows + r;
                const float inv = all > 0.0f ? __fdiv_rn(1.0f, all) : (all == 0.0f ? 0.0f : all);
                sum = make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv);
                dst = a.out + (uint64_t)(cw.q.q0 + row / a.group) * a.out_stride + (uint64_t)(cw.kh * a.group + row % a.group) * HD;
            } else {
                dst = a.part_o + (part * kPaRows + r) * HD;
                if (d == 0) {
                    a.part_ml[part * 16 + r] = top;
                    a.part_ml[part * 16 + 8 + r] = all;
                }
            }
            *reinterpret_cast<float4 *>(dst + d) = sum;
        }
        __syncthreads();  // the merge records are read before the next queries overwrite them
        f = unit_f0 + cw.q.cost();  // the next unit, unless this one goes on elsewhere
        if (f < f1) {
            cw.template next_unit<TILE>(a);
            load_q();
        }
    }
    cp_async_wait<0>();
    if (!a.join_units && !continues && tid == 0) reinterpret_cast<Q8Join *>(a.unit_info)[c].n = 0;
}

// Row r of a unit that several CTAs share: out = sum_p 2^(m_p - m) o_p / sum_p 2^(m_p - m) l_p over its records
// in CTA order.  Grid (8 rows of each entry of the list).  Few entries: 256 threads, so that nearly all records' sums
// are on their way at once (74 records for each row: 31.8 us in all, 34.5 with 128); many, with few records each:
// 128, of which more fit an SM (64 ragged sequences: 38.9 us, 43.0 with 256).
template <int HD, int THREADS>
__global__ void __launch_bounds__(THREADS) k_paged_q8_join(const __grid_constant__ PagedAttnArgs a) {
    constexpr int LANES = HD / 4, GROUPS = THREADS / LANES, EARLY = THREADS == 256 ? 10 : 4, PER = kPaMaxParts / THREADS;
    __shared__ float s_w[kPaMaxParts], s_top[THREADS / 32], s_sum[THREADS / 32];
    __shared__ float4 s_o[THREADS];
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, grp = tid / LANES, x = tid % LANES;
    const uint32_t r = blockIdx.x % kPaRows;
    const Q8Join in = reinterpret_cast<const Q8Join *>(a.unit_info)[blockIdx.x / kPaRows];
    if (in.n < 2 || in.n > kPaMaxParts || r >= in.rows) return;
    const auto sums = [&](uint32_t p) {
        return *reinterpret_cast<const float4 *>(a.part_o + (pa_part(in.first, p) * kPaRows + r) * HD + 4 * x);
    };
    float4 v[EARLY];
#pragma unroll
    for (int i = 0; i < EARLY; i++)
        if (grp + i * GROUPS < in.n) v[i] = sums(grp + i * GROUPS);
    float pm[PER], pl[PER], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const uint32_t p = tid + THREADS * i;
        pm[i] = -INFINITY;
        pl[i] = 0.0f;
        if (p < in.n) {
            const float *ml = a.part_ml + pa_part(in.first, p) * 16 + r;
            pm[i] = ml[0];
            pl[i] = ml[8];
        }
        m = fmaxf(m, pm[i]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) s_top[warp] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 32; w++) m = fmaxf(m, s_top[w]);
    const float from = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const float w = ex2(pm[i] - from);
        if (tid + THREADS * i < in.n) s_w[tid + THREADS * i] = w;
        l = fmaf(pl[i], w, l);
    }
    l = warp_sum(l);
    if (lane == 0) s_sum[warp] = l;
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
        if (grp + i * GROUPS < in.n) add(v[i], s_w[grp + i * GROUPS]);
#pragma unroll 4
    for (uint32_t p = grp + EARLY * GROUPS; p < in.n; p += GROUPS) add(sums(p), s_w[p]);
    s_o[tid] = acc;
    __syncthreads();
    if (grp) return;
    l = 0.0f;
#pragma unroll
    for (int w = 0; w < THREADS / 32; w++) l += s_sum[w];
#pragma unroll
    for (int i = 1; i < GROUPS; i++) add(s_o[i * LANES + x], 1.0f);
    const float inv = l > 0.0f ? __fdiv_rn(1.0f, l) : (l == 0.0f ? 0.0f : l);
    const uint32_t R = in.rb * kPaRows + r;
    float *dst = a.out + (uint64_t)(in.q0 + R / a.group) * a.out_stride + (uint64_t)(in.kh * a.group + R % a.group) * HD + 4 * x;
    *reinterpret_cast<float4 *>(dst) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
}

namespace {

size_t up256(size_t v) { return (v + 255) & ~(size_t)255; }

struct Q8Scratch {
    size_t part_o, part_ml, unit_info, total;
};
uint32_t q8_grid(uint32_t hd, int num_sms) {
    return min((uint32_t)num_sms * (hd == 256 ? Q8Shape<256>::CTAS : hd == 128 ? Q8Shape<128>::CTAS : Q8Shape<64>::CTAS), kPaMaxParts);
}
uint32_t q8_row_blocks(const PagedAttnArgs &a) {
    return (uint32_t)(((uint64_t)(a.cu ? a.max_q : 1) * a.group + kPaRows - 1) / kPaRows);
}
Q8Scratch q8_layout(const PagedAttnArgs &a, uint32_t G) {
    Q8Scratch s;
    s.part_o = 0;
    s.part_ml = up256((size_t)2 * G * kPaRows * a.kv.hd * 4);
    s.unit_info = s.part_ml + up256((size_t)2 * G * 16 * 4);
    s.total = s.unit_info + up256((size_t)G * sizeof(Q8Join));
    return s;
}

template <int HD, bool PROMPT>
cudaError_t q8_launch(const LaunchCfg &c, const PagedAttnArgs &a) {
    const char *label = PROMPT ? "paged_q8_attn_rows" : "paged_q8_attn";
    const dim3 grid(q8_grid(HD, c.num_sms)), block(kPaThreads);
    cudaError_t e;
    if (a.softcap == 0.0f && !a.slopes)
        e = launch_k(c, label, k_paged_q8<HD, PROMPT, true>, grid, block, Q8Shape<HD>::SMEM, a);
    else
        e = launch_k(c, label, k_paged_q8<HD, PROMPT, false>, grid, block, Q8Shape<HD>::SMEM, a);
    if (e != cudaSuccess) return e;
    const uint32_t places = a.join_units ? a.n_seq * a.kv.n_kv * a.row_blocks : grid.x;
    const dim3 rows(places * kPaRows);
    if (rows.x <= 3u * (uint32_t)c.num_sms) return launch_k(c, "paged_q8_join", k_paged_q8_join<HD, 256>, rows, dim3(256), 0, a);
    return launch_k(c, "paged_q8_join", k_paged_q8_join<HD, 128>, rows, dim3(128), 0, a);
}

}  // namespace

size_t paged_q8_attn_scratch(const PagedAttnArgs &a, int num_sms) { return q8_layout(a, q8_grid(a.kv.hd, num_sms)).total; }

cudaError_t launch_paged_q8_attn(const LaunchCfg &c, PagedAttnArgs a, uint8_t *scratch) {
    const Q8Scratch s = q8_layout(a, q8_grid(a.kv.hd, c.num_sms));
    a.part_o = (float *)(scratch + s.part_o);
    a.part_ml = (float *)(scratch + s.part_ml);
    a.unit_info = (uint32_t *)(scratch + s.unit_info);
    a.err = c.dev_err;
    a.row_blocks = q8_row_blocks(a);
    a.join_units = !a.cu && (uint64_t)a.n_seq * a.kv.n_kv * a.row_blocks <= q8_grid(a.kv.hd, c.num_sms);
    switch (a.kv.hd) {
    case 64: return a.cu ? q8_launch<64, true>(c, a) : q8_launch<64, false>(c, a);
    case 128: return a.cu ? q8_launch<128, true>(c, a) : q8_launch<128, false>(c, a);
    case 256: return a.cu ? q8_launch<256, true>(c, a) : q8_launch<256, false>(c, a);
    default: return cudaErrorInvalidValue;
    }
}

}  // namespace lt
