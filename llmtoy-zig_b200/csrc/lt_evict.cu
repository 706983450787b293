// lt_evict.cu — eviction from a paged cache by accumulated attention weight.
//
// Per sequence of n > budget positions and per KV head: the newest `recent`
// positions stay, and of the others the budget - recent with the largest
// accumulated weight (the lowest position first among equals).  What stays keeps
// its order; its K and V rows and its weights move to slots 0 .. budget - 1.
//
// k_evict_select: one CTA per (sequence, KV head), or a cluster of four.  The weights become
// order-preserving 32-bit keys; three passes of 11, 11 and 10 bits narrow the
// budget-th largest key down (histograms in shared memory), and one ordered
// pass writes what stays: a kept position's slot is the number of larger keys
// before it plus the equal ones before it, as far as equal ones are taken.
// k_evict_move: the rows.  Bound: memory.  Into other pages any order will do
// and every row is its own work.  Within the same pages row i comes from a
// position >= i, so a CTA that goes up in steps, reading a step before it writes
// it, never overwrites what a later step reads; 32-byte columns of the rows are
// independent of each other and give the parallelism.
//
// One B200, 16 sequences of 20000 to 32768 with 4 KV heads of 128 in f16, budget
// 8192: 116 us, the moves 82 us of it (6.5 TB/s).  8 sequences of about 1100: 11 us,
// two launches.
#include <cooperative_groups.h>

#include "lt_paged.cuh"

namespace lt {

namespace cg = cooperative_groups;

constexpr int kSelThreads = 1024;
constexpr int kSelPer = 4;
constexpr int kSelBins = 2048;
// Rows longer than this take a cluster where all clusters run at once.  The selection by one CTA and by four,
// 4 or 16 rows: 9000 positions 17.8 and 18.5 us, 12000 18.6 and 18.6, 16000 20.6 and 18.7, 32768 32.9 and 24.
// 64 rows, whose 256 CTAs take turns: 22.4 and 28.7 us at 16000, 34.9 and 37.0 at 32768.
constexpr uint32_t kSelCluster = 12288;
constexpr int kMoveThreads = 256;
constexpr int kMoveRows = 64;

// Ascending with the weight; NaN counts as the largest, -0 as 0.
LT_DEVINL uint32_t mass_key(float m) {
    if (m != m) return 0xffffffffu;
    const uint32_t u = __float_as_uint(m + 0.0f);
    return (u >> 31) ? ~u : u | 0x80000000u;
}

// Exclusive sum over the block of one packed value per thread.
LT_DEVINL uint64_t block_excl(uint64_t v, uint64_t *s_warp, uint64_t *total) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint64_t x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();  // the last call's reads are over
    if (lane == 31) s_warp[warp] = x;
    __syncthreads();
    if (warp == 0) {
        uint64_t w = s_warp[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t y = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += y;
        }
        s_warp[lane] = w;
    }
    __syncthreads();
    *total = s_warp[31];
    return x - v + (warp ? s_warp[warp - 1] : 0);
}

// CL CTAs (a cluster) per (sequence, KV head), each with a contiguous part of the positions.
template <int CL>
__global__ void __launch_bounds__(kSelThreads) k_evict_select(EvictArgs a) {
    __shared__ uint32_t s_hist[kSelBins];
    __shared__ uint64_t s_warp[32], s_mine;
    __shared__ uint32_t s_bin, s_left;
    pdl_launch_dependents();
    pdl_wait();
    const cg::cluster_group cluster = cg::this_cluster();
    const uint32_t rank = CL > 1 ? cluster.block_rank() : 0, tid = threadIdx.x;
    auto sync_all = [&]() {
        if constexpr (CL > 1)
            cluster.sync();
        else
            __syncthreads();
    };
    const uint32_t h = blockIdx.x / CL, s = blockIdx.y;
    const uint64_t pair = (uint64_t)s * a.kv.n_kv + h;
    uint32_t n = a.lens[s];
    if (n > a.max_len || (n + a.kv.page_size - 1) / a.kv.page_size > a.kv.max_pages) {
        if (tid == 0) atomicExch(a.err, DEV_ERR_BAD_INDEX);
        n = min((uint64_t)a.max_len, (uint64_t)a.kv.max_pages * a.kv.page_size);
    }
    const uint32_t keep = min(n, a.budget);
    const float *mass = a.mass + pair * a.mass_stride;
    float *mass_out = a.mass_out + pair * a.mass_out_stride;
    uint32_t *kept = a.kept + pair * a.kept_stride;
    if (h == 0 && rank == 0 && tid == 0) a.new_len[s] = keep;
    const uint32_t old = n > a.budget ? n - a.recent : 0;  // positions that compete
    uint32_t want = n > a.budget ? a.budget - a.recent : 0;
    constexpr uint32_t CHUNK = kSelThreads * kSelPer;
    const uint32_t part = ((n + CL - 1) / CL + CHUNK - 1) / CHUNK * CHUNK;
    const uint32_t from = min(n, rank * part), to = min(n, from + part);  // this CTA's positions
    const bool wide = (reinterpret_cast<uintptr_t>(mass) & 15) == 0;

    // four weights in a row per thread and chunk; a part of one chunk is loaded once
    float m[kSelPer];
    auto load = [&](uint32_t j, float(&w)[kSelPer]) {
        if (wide && j + kSelPer <= to) {
            const float4 v = *reinterpret_cast<const float4 *>(mass + j);
            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        } else {
#pragma unroll
            for (int u = 0; u < kSelPer; u++) w[u] = j + u < to ? mass[j + u] : 0.0f;
        }
    };
    const bool once = to - from <= CHUNK;
    if (once) load(from + tid * kSelPer, m);

    // the want-th largest key among the first `old`, bits from the top
    uint32_t prefix = 0, done = 0;
    for (int pass = 0; pass < 3 && want; pass++) {
        const int bits = pass == 2 ? 10 : 11, shift = 32 - (int)done - bits, bins = 1 << bits;
        for (int i = tid; i < kSelBins; i += kSelThreads) s_hist[i] = 0;
        __syncthreads();
        auto count = [&](uint32_t j, const float(&w)[kSelPer]) {
#pragma unroll
            for (int u = 0; u < kSelPer; u++) {
                const uint32_t k = mass_key(w[u]);
                if (j + u < old && j + u < to && (done == 0 || k >> (32 - done) == prefix))
                    atomicAdd(&s_hist[(k >> shift) & (bins - 1)], 1u);
            }
        };
        if (once) {
            count(from + tid * kSelPer, m);
        } else {
            for (uint32_t j = from + tid * kSelPer; j < min(to, old); j += 2 * CHUNK) {
                float w0[kSelPer], w1[kSelPer];
                load(j, w0);
                load(j + CHUNK, w1);
                count(j, w0);
                count(j + CHUNK, w1);
            }
        }
        sync_all();
        // bins from the top: thread t takes bins - 1 - 2 t and the one below, of all parts
        const int b0 = bins - 1 - 2 * (int)tid, b1 = b0 - 1;
        uint32_t c0 = 0, c1 = 0;
        if (b1 >= 0) {
#pragma unroll
            for (int r = 0; r < CL; r++) {
                const uint32_t *hist = CL > 1 ? cluster.map_shared_rank(s_hist, r) : s_hist;
                c0 += hist[b0];
                c1 += hist[b1];
            }
        }
        uint64_t total;
        const uint32_t before = (uint32_t)block_excl((uint64_t)c0 + c1, s_warp, &total);
        if (before < want && want <= before + c0) {
            s_bin = b0;
            s_left = want - before;
        } else if (before + c0 < want && want <= before + c0 + c1) {
            s_bin = b1;
            s_left = want - before - c0;
        }
        sync_all();  // and nobody reads this part's bins any more
        prefix = (prefix << bits) | s_bin;
        want = s_left;
        done += bits;
    }
    // want now counts the keys equal to prefix that stay
    const bool any = n > a.budget && a.budget > a.recent;
    auto sides = [&](uint32_t j, const float(&w)[kSelPer], uint32_t &gt, uint32_t &eq) {  // bit u: element j + u
        gt = eq = 0;
#pragma unroll
        for (int u = 0; u < kSelPer; u++) {
            if (j + u >= to) continue;
            const uint32_t k = mass_key(w[u]);
            if (j + u >= old || (any && k > prefix))
                gt |= 1u << u;  // newest, or nothing is evicted, or heavier
            else if (any && k == prefix)
                eq |= 1u << u;
        }
    };
    uint32_t greater = 0, equal = 0;  // so far, the parts before this one included
    if constexpr (CL > 1) {
        uint64_t mine = 0;
        for (uint32_t j = from + tid * kSelPer; j < to; j += CHUNK) {
            if (!once) load(j, m);
            uint32_t gt, eq;
            sides(j, m, gt, eq);
            mine += ((uint64_t)__popc(gt) << 32) | __popc(eq);
        }
        uint64_t total;
        block_excl(mine, s_warp, &total);
        if (tid == 0) s_mine = total;
        cluster.sync();
        for (uint32_t r = 0; r < rank; r++) {
            const uint64_t t = *cluster.map_shared_rank(&s_mine, r);
            greater += (uint32_t)(t >> 32);
            equal += (uint32_t)t;
        }
        cluster.sync();  // nobody leaves before its count is read
    }
    for (uint32_t j0 = from; j0 < to; j0 += CHUNK) {
        const uint32_t j = j0 + tid * kSelPer;
        if (!once) load(j, m);
        uint32_t gt, eq;
        sides(j, m, gt, eq);
        uint64_t total;
        const uint64_t before = block_excl(((uint64_t)__popc(gt) << 32) | __popc(eq), s_warp, &total);
        uint32_t g = greater + (uint32_t)(before >> 32), e = equal + (uint32_t)before;
#pragma unroll
        for (int u = 0; u < kSelPer; u++) {
            const bool is_eq = eq >> u & 1u;
            if ((gt >> u & 1u) || (is_eq && e < want)) {
                const uint32_t at = g + min(e, want);
                kept[at] = j + u;
                mass_out[at] = m[u];
            }
            g += gt >> u & 1u;
            e += is_eq;
        }
        greater += (uint32_t)(total >> 32);
        equal += (uint32_t)total;
    }
}

// Byte offset of a position of sequence s in the pool; false: a bad page id.
LT_DEVINL bool evict_offset(const EvictArgs &a, const uint32_t *table, uint32_t s, uint32_t j, uint32_t h, uint64_t &off) {
    const uint32_t p = j / a.kv.page_size;
    const uint32_t page = p < a.kv.max_pages ? table[(uint64_t)s * a.kv.max_pages + p] : a.kv.n_pages;
    if (page >= a.kv.n_pages) {
        atomicExch(a.err, DEV_ERR_BAD_INDEX);
        return false;
    }
    off = paged_offset(a.kv, page, j, h);
    return true;
}

// Into other pages: grid (row steps, n_kv, n_seq); 16 bytes per thread at a time.
__global__ void __launch_bounds__(kMoveThreads) k_evict_move(EvictArgs a) {
    __shared__ uint64_t s_from[kMoveRows], s_to[kMoveRows];
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t h = blockIdx.y, s = blockIdx.z, i0 = blockIdx.x * kMoveRows, tid = threadIdx.x;
    const uint32_t keep = a.new_len[s];
    if (h == 0 && i0 == 0 && tid == 0) a.lens_out[s] = keep;
    if (i0 >= keep) return;
    const uint32_t rows = min((uint32_t)kMoveRows, keep - i0);
    const uint64_t pair = (uint64_t)s * a.kv.n_kv + h;
    if (tid < rows) {
        uint64_t f = ~0ull, t = ~0ull;
        const bool ok = evict_offset(a, a.table, s, a.kept[pair * a.kept_stride + i0 + tid], h, f) &&
                        evict_offset(a, a.dst_table, s, i0 + tid, h, t);
        s_from[tid] = ok ? f : ~0ull;
        s_to[tid] = t;
    }
    __syncthreads();
    const uint32_t lanes = a.kv.hd * (a.kv.f16 ? 2 : 4) / 16;  // 8 .. 64, a power of two
    const uint32_t col = tid % lanes * 16, step = kMoveThreads / lanes;
    for (uint32_t r0 = tid / lanes; r0 < rows; r0 += 4 * step) {
        uint4 k[4], v[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const uint32_t r = r0 + u * step;
            if (r < rows && s_from[r] != ~0ull) {
                k[u] = *reinterpret_cast<const uint4 *>(a.kv.k + s_from[r] + col);
                v[u] = *reinterpret_cast<const uint4 *>(a.kv.v + s_from[r] + col);
            }
        }
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const uint32_t r = r0 + u * step;
            if (r < rows && s_from[r] != ~0ull) {
                *reinterpret_cast<uint4 *>(a.kv.k + s_to[r] + col) = k[u];
                *reinterpret_cast<uint4 *>(a.kv.v + s_to[r] + col) = v[u];
            }
        }
    }
}

// Within the same pages: grid (32-byte columns of K, then of V; n_kv, n_seq).
__global__ void __launch_bounds__(kMoveThreads) k_evict_move_in_place(EvictArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t h = blockIdx.y, s = blockIdx.z, tid = threadIdx.x;
    const uint32_t cols = a.kv.hd * (a.kv.f16 ? 2 : 4) / 32;
    uint8_t *base = blockIdx.x < cols ? a.kv.k : a.kv.v;
    const uint32_t byte = blockIdx.x % cols * 32 + (tid & 1) * 16;
    const uint32_t keep = a.new_len[s];
    if (h == 0 && blockIdx.x == 0 && tid == 0) a.lens_out[s] = keep;
    const uint32_t *kept = a.kept + ((uint64_t)s * a.kv.n_kv + h) * a.kept_stride;
    constexpr int U = 4, R = kMoveThreads / 2;
    for (uint32_t i0 = 0; i0 < keep; i0 += R * U) {
        uint4 x[U];
        uint64_t to[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t i = i0 + u * R + tid / 2;
            to[u] = ~0ull;
            if (i < keep && kept[i] != i) {
                uint64_t f, t;
                if (evict_offset(a, a.table, s, kept[i], h, f) && evict_offset(a, a.table, s, i, h, t)) {
                    x[u] = *reinterpret_cast<const uint4 *>(base + f + byte);
                    to[u] = t;
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < U; u++)
            if (to[u] != ~0ull) *reinterpret_cast<uint4 *>(base + to[u] + byte) = x[u];
        __syncthreads();
    }
}

namespace {

// launch_k with a cluster along x.
template <typename Kern, typename... Args>
cudaError_t launch_cluster(const LaunchCfg &c, const char *label, Kern kern, dim3 grid, dim3 block, uint32_t size, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.stream = c.stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = size;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const bool timed = c.prof && c.prof->on;
    if (c.pdl && !timed) {
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.numAttrs = 2;
    }
    Profiler::Rec rec;
    if (timed) c.prof->begin(label, c.stream, rec);
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
    if (timed) c.prof->end(rec, c.stream);
    return e;
}

}  // namespace

// Positions a row can keep: a budget may say "no limit".
static uint32_t evict_most(const EvictArgs &a) { return min(a.budget, a.max_len); }

size_t evict_scratch(const EvictArgs &a, bool have_kept) {
    const size_t lens = ((size_t)a.n_seq * 4 + 255) & ~(size_t)255;
    return lens + (have_kept ? 0 : (size_t)a.n_seq * a.kv.n_kv * evict_most(a) * 4);
}

cudaError_t launch_evict(const LaunchCfg &c, EvictArgs a, uint8_t *scratch) {
    a.new_len = (uint32_t *)scratch;
    a.kept_stride = a.kept ? a.budget : evict_most(a);
    if (!a.kept) a.kept = (uint32_t *)(scratch + (((size_t)a.n_seq * 4 + 255) & ~(size_t)255));
    a.err = c.dev_err;
    // Long rows by clusters of four (kSelCluster).  Not where the weights are compacted in place: a CTA writes where
    // those before it read, which only one CTA's own order makes safe.
    cudaError_t e;
    if (a.max_len > kSelCluster && 4 * a.kv.n_kv * a.n_seq <= (uint32_t)c.num_sms && a.mass_out != a.mass)
        e = launch_cluster(c, "evict_select", k_evict_select<4>, dim3(4 * a.kv.n_kv, a.n_seq), dim3(kSelThreads), 4, a);
    else
        e = launch_k(c, "evict_select", k_evict_select<1>, dim3(a.kv.n_kv, a.n_seq), dim3(kSelThreads), 0, a);
    if (e != cudaSuccess) return e;
    if (a.in_place) {
        const uint32_t cols = a.kv.hd * (a.kv.f16 ? 2 : 4) / 32;
        return launch_k(c, "evict_move", k_evict_move_in_place, dim3(2 * cols, a.kv.n_kv, a.n_seq), dim3(kMoveThreads),
                        0, a);
    }
    return launch_k(c, "evict_move", k_evict_move, dim3((evict_most(a) + kMoveRows - 1) / kMoveRows, a.kv.n_kv, a.n_seq),
                    dim3(kMoveThreads), 0, a);
}

}  // namespace lt
