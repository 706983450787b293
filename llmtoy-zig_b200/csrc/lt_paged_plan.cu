// lt_paged_plan.cu — pages and slots of the coming tokens of a batch, on the
// device: what a host would do with a list of free pages and a loop over the
// sequences.
//
// Of sequence s keep[s] cached positions stay and new[s] come.  With pages of P
// slots, have = ceil(lens / P), stay = ceil(keep / P), want = ceil((keep + new) / P):
// pages stay .. have - 1 go back to the stack of free pages, then pages
// stay .. want - 1 are taken from its top.  Returned last sequence first and last
// page first, taken first sequence first and first page first, so that giving
// back what was just taken restores the stack.  With
//   G(s) = sum_{t < s} (have - stay),  T(s) = sum_{t < s} (want - stay),  n' = n_free + G(n_seq)
// the page returned from entry j lies at n' - 1 - (G(s) + j - stay), and entry j
// takes the page at n' - 1 - (T(s) + j - stay): every page and token finds its place by itself.
//
// Bound: latency (dependent loads and block barriers).  One B200, calls of a recorded graph: a
// token for each of 64 sequences 4.5 us; prompts of 512 (325661 tokens, 10426 pages back and as
// many taken) 10.6 us (in three launches, threads with pages and tokens to place alike, 15.9).
// One CTA scans the sequences, a thread to each as far as they go round, and refuses what
// cannot be done before anything is changed: page numbers past the pool, too, wherever the plan
// makes a table entry or a slot of them.  Few tokens: the same CTA moves the pages and places
// the tokens.  Many: all SMs, in two launches (one CTA alone for the pages of those prompts:
// 22 us, by its instructions): every CTA scans the sequences for itself and looks at its share
// of the pages that go or come, then everything is written.
// Pages and tokens are dealt to threads one by one, wherever their sequences begin.  Up to
// 2048 sequences are kept in shared memory between the steps; more are scanned by one CTA,
// and the pages looked at in a launch of their own.
#include "lt_launch.cuh"

namespace lt {

constexpr int kPlanThreads = 1024, kPlanWarps = kPlanThreads / 32;
constexpr uint32_t kPlanNoPage = 0xffffffffu;
constexpr uint32_t kPlanMaxLen = 1u << 30;

// Divisions by the page size, in 32 bits and for powers of two as shifts.
LT_DEVINL uint32_t page_of(const PagedPlanArgs &a, uint32_t n) { return a.page_shift != kNoShift ? n >> a.page_shift : n / a.page; }
LT_DEVINL uint32_t pages_for(const PagedPlanArgs &a, uint32_t n) { return n ? page_of(a, n - 1) + 1 : 0; }

// The last s with first[s] <= i, of n ascending entries whose first is 0.
LT_DEVINL uint32_t owner_of(const uint32_t *first, uint32_t n, uint32_t i) {
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (first[mid] <= i)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

// What the steps know of sequence s: its first token among all, its first pages among those taken and among those that
// go, how many positions stay, and on how many pages.  And of all: the stack's top before anything is taken.
struct PlanSeqs {
    const uint32_t *cu, *take, *gone, *keep, *stay;
    uint32_t top, n_gone, n_take, n_tokens;
};

// The page that the k-th place among those taken gets; ids: of the pages that go, where they are not yet on the stack.
LT_DEVINL uint32_t taken(const PagedPlanArgs &a, const PlanSeqs &q, const uint32_t *ids, uint32_t k) {
    return ids && k < q.n_gone ? ids[k] : a.free[q.top - 1 - k];
}

// Whether one of the pages that go, or that come from the stack as it was, has a number past the pool; thread `at` of
// `step` looks at its share.  gone, stay: of each sequence.  ids: where the numbers of those that go are left.
LT_DEVINL bool plan_look(const PagedPlanArgs &a, const uint32_t *gone, const uint32_t *stay, uint32_t top, uint32_t n_gone, uint32_t n_take,
                         uint32_t *ids, uint32_t at, uint32_t step) {
    bool off = false;
    const uint32_t more = n_take > n_gone ? n_take - n_gone : 0, n = max(n_gone, more);
    for (uint32_t i = at; i < n; i += step) {
        const uint32_t comes = i < more ? a.free[top - 1 - n_gone - i] : 0;  // on its way during the search
        if (i < n_gone) {
            const uint32_t s = owner_of(gone, a.n_seq, i);
            const uint32_t id = a.table[(uint64_t)s * a.max_pages + stay[s] + (i - gone[s])];
            if (ids) ids[i] = id;
            off |= id >= a.n_pages;
        }
        off |= comes >= a.n_pages;
    }
    return off;
}

// Table entries and token rows, thread `at` of `step`; entries from the middle thread on, so that few threads have
// both.  Nothing that is read here is written here.
LT_DEVINL void plan_fill(const PagedPlanArgs &a, const PlanSeqs &q, const uint32_t *ids, uint32_t at, uint32_t step) {
    const uint32_t n = a.n_seq;
    for (uint32_t k = at < step / 2 ? at + step - step / 2 : at - step / 2; k < q.n_take; k += step) {
        const uint32_t s = owner_of(q.take, n, k);
        a.table[(uint64_t)s * a.max_pages + q.stay[s] + (k - q.take[s])] = taken(a, q, ids, k);
    }
    if (!a.seq && !a.pos && !a.slot) return;
    for (uint32_t t = at; t < q.n_tokens; t += step) {
        const uint32_t s = owner_of(q.cu, n, t), p = q.keep[s] + (t - q.cu[s]);
        if (a.seq) a.seq[t] = s;
        if (a.pos) a.pos[t] = p;
        if (a.slot) {
            const uint32_t stay = q.stay[s], j = page_of(a, p);
            const uint32_t id = j < stay ? a.table[(uint64_t)s * a.max_pages + j] : taken(a, q, ids, q.take[s] + j - stay);
            a.slot[t] = id * a.page + (p - j * a.page);
        }
    }
}

struct PlanSum {
    uint64_t tokens, gone, take;
};

constexpr uint32_t kPlanInShared = 2048;  // sequences

// ALONE: the one CTA does everything.  Else what was found goes to scratch, by CTA 0, and nothing to the caller's; all CTAs
// look at the pages that go or come where the sequences are in shared memory.  One CTA to an SM, said to the compiler: without it
// it keeps to 32 registers and spills (prompts of 512: 12.0 us instead of 11.4, both by events around calls from the host).
template <bool ALONE>
__global__ void __launch_bounds__(kPlanThreads, 1) k_paged_plan(const __grid_constant__ PagedPlanArgs a) {
    __shared__ PlanSum s_warp[kPlanWarps], s_all;
    __shared__ int s_bad, s_bad_page;
    __shared__ uint32_t s_cu[kPlanInShared], s_take[kPlanInShared], s_gone[kPlanInShared], s_keep[kPlanInShared], s_stay[kPlanInShared];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const bool in_shared = a.n_seq <= kPlanInShared;
    uint32_t *const cu = in_shared ? s_cu : a.cu_copy, *const take = in_shared ? s_take : a.take;
    uint32_t *const gone = in_shared ? s_gone : a.gone, *const keeps = in_shared ? s_keep : a.keeps, *const stays = in_shared ? s_stay : a.stay;
    pdl_launch_dependents();
    if (tid == 0) s_bad = s_bad_page = DEV_ERR_NONE;
    pdl_wait();
    const uint32_t n_free = *a.n_free;
    __syncthreads();
    const uint32_t per = (a.n_seq + kPlanThreads - 1) / kPlanThreads;
    const uint32_t sa = min(a.n_seq, tid * per), sb = min(a.n_seq, sa + per);
    const uint64_t cap = min((uint64_t)a.max_pages * a.page, (uint64_t)kPlanMaxLen);
    PlanSum mine = {0, 0, 0};
    bool bad = false, off = false;  // off: a page number past the pool
    uint32_t held = 0;              // one that is on its way, looked at only when the sums are scanned
    for (uint32_t s = sa; s < sb; s++) {  // within this thread for now, in what belongs to it alone
        const uint32_t len = a.lens[s], keep = a.keep ? a.keep[s] : len, add = a.add[s];
        cu[s] = (uint32_t)mine.tokens;
        take[s] = (uint32_t)mine.take;
        gone[s] = (uint32_t)mine.gone;
        keeps[s] = keep;
        if (len > cap || keep > len || (uint64_t)keep + add > cap) {
            bad = true;
            continue;
        }
        const uint32_t stay = pages_for(a, keep);
        stays[s] = stay;
        if (add && stay * a.page != keep && (ALONE || !in_shared || s % gridDim.x == blockIdx.x)) {
            off |= held >= a.n_pages;
            held = a.table[(uint64_t)s * a.max_pages + stay - 1];  // the page that the coming tokens go on with
        }
        mine.tokens += add;
        mine.gone += pages_for(a, len) - stay;
        mine.take += pages_for(a, keep + add) - stay;
    }
    auto scan = [&](PlanSum &v) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t x = __shfl_up_sync(0xffffffffu, v.tokens, o), y = __shfl_up_sync(0xffffffffu, v.gone, o),
                           z = __shfl_up_sync(0xffffffffu, v.take, o);
            if (lane >= o) v.tokens += x, v.gone += y, v.take += z;
        }
    };
    PlanSum incl = mine;
    scan(incl);
    if (lane == 31) s_warp[warp] = incl;
    if (bad) s_bad = DEV_ERR_BAD_INDEX;
    __syncthreads();
    if (warp == 0) {
        PlanSum v = s_warp[lane];
        const PlanSum own = v;
        scan(v);
        s_warp[lane] = {v.tokens - own.tokens, v.gone - own.gone, v.take - own.take};
        if (lane == 31) {
            s_all = v;
            if (s_bad == DEV_ERR_NONE) {
                const uint64_t top = (uint64_t)n_free + v.gone;
                if (v.tokens > a.total_q || n_free > a.n_pages || top > a.n_pages)
                    s_bad = DEV_ERR_BAD_INDEX;
                else if (v.take > top)
                    s_bad = DEV_ERR_NO_PAGES;
            }
        }
    }
    off |= held >= a.n_pages;
    if (ALONE && off) s_bad_page = DEV_ERR_BAD_INDEX;
    __syncthreads();
    const PlanSum all = s_all;
    const uint32_t top = n_free + (uint32_t)all.gone;  // where it counts, nothing is bad
    const PlanSum at = {s_warp[warp].tokens + incl.tokens - mine.tokens, s_warp[warp].gone + incl.gone - mine.gone,
                        s_warp[warp].take + incl.take - mine.take};
    for (uint32_t s = sa; s < sb; s++) {
        cu[s] += (uint32_t)at.tokens;
        take[s] += (uint32_t)at.take;
        gone[s] += (uint32_t)at.gone;
    }
    bool ok = s_bad == DEV_ERR_NONE;
    if (!ALONE) {
        for (uint32_t s = sa; in_shared && blockIdx.x == 0 && s < sb; s++) {
            a.cu_copy[s] = cu[s];
            a.take[s] = take[s];
            a.gone[s] = gone[s];
            a.keeps[s] = keeps[s];
            a.stay[s] = stays[s];
        }
        int wrong = s_bad;
        if (!in_shared && __syncthreads_or(off) && ok) wrong = DEV_ERR_BAD_INDEX;
        if (blockIdx.x == 0 && tid == 0) *a.head = {top, (uint32_t)all.gone, (uint32_t)all.take, (uint32_t)all.tokens, wrong, n_free};
        if (!in_shared) return;
        __syncthreads();
        if (ok)
            off |= plan_look(a, gone, stays, top, (uint32_t)all.gone, (uint32_t)all.take, a.ids, blockIdx.x * kPlanThreads + tid,
                             gridDim.x * kPlanThreads);
        off = __syncthreads_or(off);
        if (tid == 0) a.flags[blockIdx.x] = off;
        return;
    }
    ok = ok && s_bad_page == DEV_ERR_NONE;  // written before the barrier above only
    if (ok && (all.gone || all.take)) {
        // the pages that go and those from the stack, one to a thread: their numbers are looked at before any moves
        if (all.gone) __syncthreads();
        ok = !__syncthreads_or(plan_look(a, gone, stays, top, (uint32_t)all.gone, (uint32_t)all.take, nullptr, tid, kPlanThreads));
        if (ok && all.gone) {
            for (uint32_t r = tid; r < all.gone; r += kPlanThreads) {
                const uint32_t s = owner_of(gone, a.n_seq, r);
                uint32_t *entry = a.table + (uint64_t)s * a.max_pages + stays[s] + (r - gone[s]);
                a.free[top - 1 - r] = *entry;
                *entry = kPlanNoPage;
            }
            __syncthreads();
        }
    }
    for (uint32_t s = sa; s < sb; s++) {
        a.cu[s] = ok ? cu[s] : 0;
        if (ok) a.lens[s] = keeps[s] + ((s + 1 < sb ? cu[s + 1] : (uint32_t)(at.tokens + mine.tokens)) - cu[s]);
    }
    if (tid == 0) {
        a.cu[a.n_seq] = ok ? (uint32_t)all.tokens : 0;
        if (ok)
            *a.n_free = (uint32_t)(top - all.take);
        else
            atomicExch(a.err, s_bad != DEV_ERR_NONE ? s_bad : DEV_ERR_BAD_INDEX);
    }
    if (!ok) return;
    __syncthreads();
    const PlanSeqs q = {cu, take, gone, keeps, stays, top, (uint32_t)all.gone, (uint32_t)all.take, (uint32_t)all.tokens};
    plan_fill(a, q, nullptr, tid, kPlanThreads);
}

constexpr int kPlanFillThreads = 256;

// The pages that go and those from the stack, looked at: of more sequences than shared memory holds.
__global__ void __launch_bounds__(kPlanFillThreads) k_paged_plan_gone(const __grid_constant__ PagedPlanArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    const PlanHead h = *a.head;
    if (h.bad != DEV_ERR_NONE) return;
    const uint32_t at = blockIdx.x * kPlanFillThreads + threadIdx.x, step = gridDim.x * kPlanFillThreads;
    if (plan_look(a, a.gone, a.stay, h.top, h.gone, h.take, a.ids, at, step)) a.head->bad_page = DEV_ERR_BAD_INDEX;
}

// Everything that is written.  Pages that go are read from ids: their table entries may be written here.
__global__ void __launch_bounds__(kPlanFillThreads) k_paged_plan_fill(const __grid_constant__ PagedPlanArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    const PlanHead h = *a.head;
    const uint32_t at = blockIdx.x * kPlanFillThreads + threadIdx.x, step = gridDim.x * kPlanFillThreads;
    bool off = false;
    for (uint32_t i = threadIdx.x; i < a.n_flags; i += kPlanFillThreads) off |= a.flags[i] != 0;
    off = __syncthreads_or(off) || h.bad_page != DEV_ERR_NONE;
    const int bad = h.bad != DEV_ERR_NONE ? h.bad : off ? DEV_ERR_BAD_INDEX : DEV_ERR_NONE;
    if (bad != DEV_ERR_NONE) {
        for (uint32_t s = at; s <= a.n_seq; s += step) a.cu[s] = 0;
        if (at == 0) atomicExch(a.err, bad);
        return;
    }
    for (uint32_t s = at; s <= a.n_seq; s += step) {
        const uint32_t first = s < a.n_seq ? a.cu_copy[s] : h.tokens, next = s + 1 < a.n_seq ? a.cu_copy[s + 1] : h.tokens;
        a.cu[s] = first;
        if (s < a.n_seq) a.lens[s] = a.keeps[s] + (next - first);
    }
    if (at == 0) *a.n_free = h.top - h.take;
    for (uint32_t r = step - 1 - at; r < h.gone; r += step) {  // from the last thread on
        a.free[h.top - 1 - r] = a.ids[r];
        const uint32_t s = owner_of(a.gone, a.n_seq, r), j = r - a.gone[s];
        const uint32_t takes = (s + 1 < a.n_seq ? a.take[s + 1] : h.take) - a.take[s];
        if (j >= takes) a.table[(uint64_t)s * a.max_pages + a.stay[s] + j] = kPlanNoPage;
    }
    const PlanSeqs q = {a.cu_copy, a.take, a.gone, a.keeps, a.stay, h.top, h.gone, h.take, h.tokens};
    plan_fill(a, q, a.ids, at, step);
}

namespace {
constexpr size_t kPlanHead = 4096;  // and the flags behind it
constexpr uint32_t kPlanMostFlags = (4096 - 256) / 4;
size_t plan_row(const PagedPlanArgs &a) { return ((size_t)a.n_seq * 4 + 255) & ~(size_t)255; }
}  // namespace

size_t paged_plan_scratch(const PagedPlanArgs &a) { return kPlanHead + 5 * plan_row(a) + (size_t)a.n_pages * 4; }

cudaError_t launch_paged_plan(const LaunchCfg &c, PagedPlanArgs a, uint8_t *scratch) {
    a.err = c.dev_err;
    a.head = (PlanHead *)scratch;
    a.flags = (uint32_t *)(scratch + 256);
    a.take = (uint32_t *)(scratch + kPlanHead);
    a.gone = a.take + plan_row(a) / 4;
    a.keeps = a.gone + plan_row(a) / 4;
    a.stay = a.keeps + plan_row(a) / 4;
    a.cu_copy = a.stay + plan_row(a) / 4;
    a.ids = a.cu_copy + plan_row(a) / 4;
    a.page_shift = kNoShift;
    for (uint32_t i = 0; i < 32; i++)
        if (a.page == 1u << i) a.page_shift = i;
    const uint64_t steps = ((uint64_t)a.total_q + kPlanFillThreads - 1) / kPlanFillThreads;
    if (steps <= 16) return launch_k(c, "paged_plan", k_paged_plan<true>, dim3(1), dim3(kPlanThreads), 0, a);
    const uint32_t grid = (uint32_t)min(steps, (uint64_t)c.num_sms * 8), look = min(grid, min((uint32_t)c.num_sms, kPlanMostFlags));
    const bool in_shared = a.n_seq <= kPlanInShared;
    a.n_flags = in_shared ? look : 0;
    cudaError_t e = launch_k(c, "paged_plan", k_paged_plan<false>, dim3(in_shared ? look : 1), dim3(kPlanThreads), 0, a);
    if (e != cudaSuccess) return e;
    if (!in_shared) {
        e = launch_k(c, "paged_plan_gone", k_paged_plan_gone, dim3(look), dim3(kPlanFillThreads), 0, a);
        if (e != cudaSuccess) return e;
    }
    return launch_k(c, "paged_plan_fill", k_paged_plan_fill, dim3(grid), dim3(kPlanFillThreads), 0, a);
}

}  // namespace lt
