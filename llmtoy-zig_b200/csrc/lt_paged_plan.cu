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
// Bound: latency (the sums over the sequences, one block barrier after the other);
// many tokens: the writes, 12 bytes each.  One CTA scans the sequences, refuses what
// cannot be done before anything is changed, and puts the returned pages on the
// stack.  Few tokens are then placed by the same CTA, many by a second launch over
// all SMs.
#include "lt_launch.cuh"

namespace lt {

constexpr int kPlanThreads = 1024, kPlanWarps = kPlanThreads / 32;
constexpr uint32_t kPlanNoPage = 0xffffffffu;
constexpr uint32_t kPlanMaxLen = 1u << 30;

LT_DEVINL uint32_t pages_for(uint64_t n, uint32_t page) { return (uint32_t)((n + page - 1) / page); }

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

// Table entries and token rows, thread `at` of `step`.  Nothing that is read here is written here.
LT_DEVINL void plan_fill(const PagedPlanArgs &a, uint32_t at, uint32_t step) {
    const uint32_t top = a.head[0], takes = a.head[1], tokens = a.head[2], n = a.n_seq;
    for (uint32_t k = at; k < takes; k += step) {
        const uint32_t s = owner_of(a.take, n, k);
        const uint32_t kept = a.lens[s] - (a.cu[s + 1] - a.cu[s]);
        a.table[(uint64_t)s * a.max_pages + pages_for(kept, a.page) + (k - a.take[s])] = a.free[top - 1 - k];
    }
    if (!a.seq && !a.pos && !a.slot) return;
    for (uint32_t t = at; t < tokens; t += step) {
        const uint32_t s = owner_of(a.cu, n, t);
        const uint32_t kept = a.lens[s] - (a.cu[s + 1] - a.cu[s]), p = kept + (t - a.cu[s]);
        if (a.seq) a.seq[t] = s;
        if (a.pos) a.pos[t] = p;
        if (a.slot) {
            const uint32_t stay = pages_for(kept, a.page), j = p / a.page;
            const uint32_t id = j < stay ? a.table[(uint64_t)s * a.max_pages + j] : a.free[top - 1 - (a.take[s] + j - stay)];
            a.slot[t] = id * a.page + p % a.page;
        }
    }
}

struct PlanSum {
    uint64_t tokens, gone, take;
};

// FILL: the same CTA places the tokens.
template <bool FILL>
__global__ void __launch_bounds__(kPlanThreads) k_paged_plan(const __grid_constant__ PagedPlanArgs a) {
    __shared__ PlanSum s_warp[kPlanWarps];
    __shared__ int s_bad, s_bad_page;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_launch_dependents();
    pdl_wait();
    if (tid == 0) s_bad = s_bad_page = DEV_ERR_NONE;
    __syncthreads();
    const uint32_t per = (a.n_seq + kPlanThreads - 1) / kPlanThreads;
    const uint32_t sa = min(a.n_seq, tid * per), sb = min(a.n_seq, sa + per);
    const uint64_t cap = min((uint64_t)a.max_pages * a.page, (uint64_t)kPlanMaxLen);
    PlanSum mine = {0, 0, 0};
    bool bad = false;
    for (uint32_t s = sa; s < sb; s++) {
        const uint32_t len = a.lens[s], keep = a.keep ? a.keep[s] : len, add = a.add[s];
        if (len > cap || keep > len || (uint64_t)keep + add > cap) {
            bad = true;
            continue;
        }
        const uint32_t stay = pages_for(keep, a.page);
        mine.tokens += add;
        mine.gone += pages_for(len, a.page) - stay;
        mine.take += pages_for((uint64_t)keep + add, a.page) - stay;
    }
    PlanSum incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t x = __shfl_up_sync(0xffffffffu, incl.tokens, o), y = __shfl_up_sync(0xffffffffu, incl.gone, o),
                       z = __shfl_up_sync(0xffffffffu, incl.take, o);
        if (lane >= o) incl.tokens += x, incl.gone += y, incl.take += z;
    }
    if (lane == 31) s_warp[warp] = incl;
    if (bad) s_bad = DEV_ERR_BAD_INDEX;
    __syncthreads();
    PlanSum at = {incl.tokens - mine.tokens, incl.gone - mine.gone, incl.take - mine.take}, all = {0, 0, 0};
#pragma unroll 8
    for (int w = 0; w < kPlanWarps; w++) {
        const PlanSum x = s_warp[w];
        if (w < warp) at.tokens += x.tokens, at.gone += x.gone, at.take += x.take;
        all.tokens += x.tokens, all.gone += x.gone, all.take += x.take;
    }
    const uint32_t n_free = *a.n_free;
    const uint64_t top = (uint64_t)n_free + all.gone;
    if (tid == 0 && s_bad == DEV_ERR_NONE) {
        if (all.tokens > a.total_q || n_free > a.n_pages || top > a.n_pages)
            s_bad = DEV_ERR_BAD_INDEX;
        else if (all.take > top)
            s_bad = DEV_ERR_NO_PAGES;
    }
    __syncthreads();
    // where each sequence's pages and tokens begin, and which pages go: of scratch, nothing of the caller's
    if (s_bad == DEV_ERR_NONE) {
        for (uint32_t s = sa; s < sb; s++) {
            const uint32_t len = a.lens[s], keep = a.keep ? a.keep[s] : len, add = a.add[s];
            const uint32_t stay = pages_for(keep, a.page), have = pages_for(len, a.page);
            a.take[s] = (uint32_t)at.take;
            a.gone[s] = (uint32_t)at.gone;
            a.stay[s] = stay;
            a.have[s] = have;
            at.gone += have - stay;
            at.take += pages_for((uint64_t)keep + add, a.page) - stay;
        }
    }
    __syncthreads();
    // the pages that go, 32 sequences to a warp: first their numbers are looked at, then they move
    bool ok = s_bad == DEV_ERR_NONE;
    for (int pass = 0; pass < 2 && ok; pass++) {
        for (uint32_t s0 = warp * 32; s0 < a.n_seq; s0 += kPlanThreads) {
            const uint32_t s = s0 + lane;
            const bool in = s < a.n_seq;
            const uint32_t stay = in ? a.stay[s] : 0, have = in ? a.have[s] : 0, first = in ? a.gone[s] : 0;
            for (uint32_t some = __ballot_sync(0xffffffffu, have > stay); some; some &= some - 1) {
                const int x = __ffs(some) - 1;
                const uint32_t j0 = __shfl_sync(0xffffffffu, stay, x), j1 = __shfl_sync(0xffffffffu, have, x);
                const uint32_t g = __shfl_sync(0xffffffffu, first, x);
                uint32_t *row = a.table + (uint64_t)(s0 + x) * a.max_pages;
#pragma unroll 4
                for (uint32_t j = j0 + lane; j < j1; j += 32) {
                    const uint32_t id = row[j];
                    if (pass == 0) {
                        if (id >= a.n_pages) s_bad_page = DEV_ERR_BAD_INDEX;
                    } else {
                        a.free[top - 1 - (g + j - j0)] = id;
                        row[j] = kPlanNoPage;
                    }
                }
            }
        }
        __syncthreads();  // s_bad_page is written in the first pass only, and read after it
        ok = s_bad_page == DEV_ERR_NONE;
    }
    for (uint32_t s = sa; s < sb; s++) {
        a.cu[s] = ok ? (uint32_t)at.tokens : 0;
        if (!ok) continue;
        const uint32_t keep = a.keep ? a.keep[s] : a.lens[s], add = a.add[s];
        at.tokens += add;
        a.lens[s] = keep + add;
    }
    if (tid == 0) {
        a.cu[a.n_seq] = ok ? (uint32_t)all.tokens : 0;
        a.head[0] = ok ? (uint32_t)top : 0;
        a.head[1] = ok ? (uint32_t)all.take : 0;
        a.head[2] = ok ? (uint32_t)all.tokens : 0;
        if (ok)
            *a.n_free = (uint32_t)(top - all.take);
        else
            atomicExch(a.err, s_bad != DEV_ERR_NONE ? s_bad : s_bad_page);
    }
    if (FILL) {
        __syncthreads();
        plan_fill(a, tid, kPlanThreads);
    }
}

constexpr int kPlanFillThreads = 256;

__global__ void __launch_bounds__(kPlanFillThreads) k_paged_plan_fill(const __grid_constant__ PagedPlanArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    plan_fill(a, blockIdx.x * kPlanFillThreads + threadIdx.x, gridDim.x * kPlanFillThreads);
}

namespace {
constexpr size_t kPlanHead = 256;
size_t plan_row(const PagedPlanArgs &a) { return ((size_t)a.n_seq * 4 + 255) & ~(size_t)255; }
}  // namespace

size_t paged_plan_scratch(const PagedPlanArgs &a) { return kPlanHead + 4 * plan_row(a); }

cudaError_t launch_paged_plan(const LaunchCfg &c, PagedPlanArgs a, uint8_t *scratch) {
    a.err = c.dev_err;
    a.head = (uint32_t *)scratch;
    a.take = (uint32_t *)(scratch + kPlanHead);
    a.gone = a.take + plan_row(a) / 4;
    a.stay = a.gone + plan_row(a) / 4;
    a.have = a.stay + plan_row(a) / 4;
    const uint64_t steps = ((uint64_t)a.total_q + kPlanFillThreads - 1) / kPlanFillThreads;
    if (steps <= 16) return launch_k(c, "paged_plan", k_paged_plan<true>, dim3(1), dim3(kPlanThreads), 0, a);
    cudaError_t e = launch_k(c, "paged_plan", k_paged_plan<false>, dim3(1), dim3(kPlanThreads), 0, a);
    if (e != cudaSuccess) return e;
    const uint32_t grid = (uint32_t)min(steps, (uint64_t)c.num_sms * 8);
    return launch_k(c, "paged_plan_fill", k_paged_plan_fill, dim3(grid), dim3(kPlanFillThreads), 0, a);
}

}  // namespace lt
