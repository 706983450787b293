// lt_logits.cu — what a request asks of its logits before a token is chosen.
//
// For token t of a row with history counts c(t) (lt_logit_rule):
//   y = x                                                       c(t) = 0
//   y = (x > 0 ? x / rep : x * rep) - (c(t) freq + pres)        c(t) > 0
//   y = y + bias(t)
//   y = -inf where the row's grammar mask has bit t clear.
//
// Bound: memory (a row is read and written once; logits behind a run of masked
// tokens are not even read).  A CTA owns a chunk of one row's tokens and keeps
// their counts and biases in shared memory; a cluster of eight CTAs shares one
// reading of the row's history, each taking every eighth part and counting into
// the chunk's owner (every chunk reading all of it took four times as long at 64
// rows of 262144 with histories of 8192).  The counts are integers, so their
// order does not matter; of a token that the bias list names twice the last
// entry counts: the list index goes through an integer maximum.
#include <cooperative_groups.h>

#include "llmtoy_cuda.h"
#include "lt_paged.cuh"

namespace lt {

namespace cg = cooperative_groups;

constexpr int kLgThreads = 256, kLgCluster = 8;
constexpr int kLgPer = 4;                              // 4-token groups per thread
constexpr int kLgChunk = kLgThreads * kLgPer * 4;      // tokens per CTA

// Calls f(index, id) for this thread's share of list[0 .. n): every kLgCluster * kLgThreads-th
// entry, four loads in flight.
template <typename F>
LT_DEVINL void each_listed(const uint32_t *list, uint32_t n, uint32_t first, F f) {
    constexpr uint32_t STEP = kLgCluster * kLgThreads;
    for (uint32_t i = first; i < n; i += 4 * STEP) {
        uint32_t id[4];
#pragma unroll
        for (int u = 0; u < 4; u++) id[u] = i + u * STEP < n ? list[i + u * STEP] : 0xffffffffu;
#pragma unroll
        for (int u = 0; u < 4; u++)
            if (i + u * STEP < n) f(i + u * STEP, id[u]);
    }
}

__global__ void __cluster_dims__(kLgCluster, 1, 1) __launch_bounds__(kLgThreads) k_logits(LogitArgs a) {
    __shared__ __align__(16) uint32_t s_count[kLgChunk];
    __shared__ __align__(16) uint32_t s_bias[kLgChunk];
    pdl_launch_dependents();
    pdl_wait();
    const cg::cluster_group cluster = cg::this_cluster();
    const uint32_t rank = cluster.block_rank(), tid = threadIdx.x;
    const uint32_t row = blockIdx.y, t0 = blockIdx.x * kLgChunk, span0 = (blockIdx.x - rank) * kLgChunk;
    const uint32_t nt = t0 < a.n ? min((uint32_t)kLgChunk, a.n - t0) : 0;
    const uint32_t span = min((uint32_t)(kLgCluster * kLgChunk), a.n - span0);  // the cluster's tokens
    const lt_logit_rule r = static_cast<const lt_logit_rule *>(a.rules)[row];
    const uint32_t hist_len = a.history ? r.history_len : 0, bias_len = a.bias_ids ? r.bias_len : 0;
    const float *x = a.logits + row * a.in_stride + t0;
    float *y = a.out + row * a.out_stride + t0;
    const uint32_t *mask = r.mask_row == LT_NO_MASK || !a.masks ? nullptr : a.masks + (uint64_t)r.mask_row * ((a.n + 31) / 32);
    const bool wide = ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) & 15) == 0;

    // this thread's tokens: groups of four, kLgThreads groups apart; allowed ones are on their way
    // while the lists are counted
    uint32_t keep[kLgPer];
    float v[kLgPer][4];
#pragma unroll
    for (int u = 0; u < kLgPer; u++) {
        const uint32_t i = (u * kLgThreads + tid) * 4;
        keep[u] = i < nt ? (mask ? mask[(t0 + i) >> 5] >> ((t0 + i) & 31) & 15u : 15u) : 0u;  // chunks start on a word
    }
#pragma unroll
    for (int u = 0; u < kLgPer; u++) {
        const uint32_t i = (u * kLgThreads + tid) * 4;
        v[u][0] = v[u][1] = v[u][2] = v[u][3] = 0.0f;
        if (keep[u]) {
            if (wide && i + 4 <= nt) {
                const float4 t = *reinterpret_cast<const float4 *>(x + i);
                v[u][0] = t.x, v[u][1] = t.y, v[u][2] = t.z, v[u][3] = t.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (i + e < nt) v[u][e] = x[i + e];
            }
        }
    }
    const bool counted = hist_len != 0, biased = bias_len != 0;  // the same for the whole cluster
    if (counted || biased) {
#pragma unroll
        for (int u = 0; u < kLgPer; u++) {
            const uint32_t i = (u * kLgThreads + tid) * 4;
            *reinterpret_cast<uint4 *>(s_count + i) = make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4 *>(s_bias + i) = make_uint4(0, 0, 0, 0);
        }
        cluster.sync();
        const uint32_t first = rank * kLgThreads + tid;
        each_listed(a.history + r.history_first, hist_len, first, [&](uint32_t, uint32_t id) {
            const uint32_t d = id - span0;
            if (d < span) atomicAdd(cluster.map_shared_rank(s_count, d / kLgChunk) + d % kLgChunk, 1u);
        });
        each_listed(a.bias_ids + r.bias_first, bias_len, first, [&](uint32_t i, uint32_t id) {
            const uint32_t d = id - span0;
            if (d < span) atomicMax(cluster.map_shared_rank(s_bias, d / kLgChunk) + d % kLgChunk, i + 1);
        });
        cluster.sync();
    }
#pragma unroll
    for (int u = 0; u < kLgPer; u++) {
        const uint32_t i = (u * kLgThreads + tid) * 4;
        if (i >= nt) continue;
        if (counted) {
            const uint4 c4 = *reinterpret_cast<const uint4 *>(s_count + i);
            const uint32_t c[4] = {c4.x, c4.y, c4.z, c4.w};
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (c[e])
                    v[u][e] = (v[u][e] > 0.0f ? __fdiv_rn(v[u][e], r.repetition) : v[u][e] * r.repetition) -
                              ((float)c[e] * r.frequency + r.presence);
        }
        if (biased) {
            const uint4 b4 = *reinterpret_cast<const uint4 *>(s_bias + i);
            const uint32_t b[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (b[e]) v[u][e] += a.bias_values[(uint64_t)r.bias_first + b[e] - 1];
        }
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (!(keep[u] >> e & 1u)) v[u][e] = -INFINITY;
        if (wide && i + 4 <= nt) {
            *reinterpret_cast<float4 *>(y + i) = make_float4(v[u][0], v[u][1], v[u][2], v[u][3]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (i + e < nt) y[i + e] = v[u][e];
        }
    }
}

cudaError_t launch_logits(const LaunchCfg &c, const LogitArgs &a) {
    const uint32_t chunks = (a.n + kLgChunk - 1) / kLgChunk;
    return launch_k(c, "logits", k_logits, dim3((chunks + kLgCluster - 1) / kLgCluster * kLgCluster, a.n_rows),
                    dim3(kLgThreads), 0, a);
}

}  // namespace lt
