// lt_logits.cu — what a request asks of its logits before a token is chosen.
//
// For token t of a row with history counts c(t) (lt_logit_rule):
//   y = x                                                       c(t) = 0
//   y = (x > 0 ? x / rep : x * rep) - (c(t) freq + pres)        c(t) > 0
//   y = y + bias(t)
//   y = -inf where the row's grammar mask has bit t clear.
//
// Bound: memory (a row is read and written once; logits behind a run of masked
// tokens are not even read).  A CTA owns a chunk of one row's tokens.  It copies
// the chunk with its mask and does the few tokens that the lists name one by one:
// every history entry of the chunk counts in a table in shared memory (integers:
// the order does not matter), whoever comes first puts the token on a work list,
// and the work list is gone through when all are counted.  Then the same with the
// biases, the table holding the largest list index, so that of a token listed
// twice the last entry counts.
//
// One B200, 64 rows of 262144: 20.8 us without lists (6.6 TB/s), 42 us with
// histories of up to 8192 and 300 biases, which every chunk of a row scans.  Counts
// and biases applied to every token instead of a work list: 95 us; one scan per
// cluster of eight chunks, counting into each other's shared memory: 41 to 52 us
// (the cluster barriers cost more than the scans); 512 threads: 44 us and more.
#include "llmtoy_cuda.h"
#include "lt_paged.cuh"

namespace lt {

constexpr int kLgThreads = 256;
constexpr int kLgPer = 4;                          // 4-token groups per thread
constexpr int kLgChunk = kLgThreads * kLgPer * 4;  // tokens per CTA
static_assert(kLgChunk <= 65536, "work list entries are 16 bits wide");

// Calls f(index, token - t0) for every entry of list[0 .. n) in [t0, t0 + nt), four loads in flight.
template <typename F>
LT_DEVINL void each_listed(const uint32_t *list, uint32_t n, uint32_t t0, uint32_t nt, F f) {
    constexpr int U = 4;
    uint32_t i = threadIdx.x;
    for (; i + (U - 1) * kLgThreads < n; i += U * kLgThreads) {
        uint32_t id[U];
#pragma unroll
        for (int u = 0; u < U; u++) id[u] = list[i + u * kLgThreads];
#pragma unroll
        for (int u = 0; u < U; u++)
            if (id[u] - t0 < nt) f(i + u * kLgThreads, id[u] - t0);
    }
    for (; i < n; i += kLgThreads) {
        const uint32_t d = list[i] - t0;
        if (d < nt) f(i, d);
    }
}

__global__ void __launch_bounds__(kLgThreads) k_logits(LogitArgs a) {
    __shared__ __align__(16) uint32_t s_table[kLgChunk];
    __shared__ uint16_t s_work[kLgChunk];
    __shared__ uint32_t s_n;
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t tid = threadIdx.x, row = blockIdx.y, t0 = blockIdx.x * kLgChunk, nt = min((uint32_t)kLgChunk, a.n - t0);
    const lt_logit_rule r = static_cast<const lt_logit_rule *>(a.rules)[row];
    const uint32_t hist_len = a.history ? r.history_len : 0, bias_len = a.bias_ids ? r.bias_len : 0;
    const float *x = a.logits + (uint64_t)row * a.n + t0;
    float *y = a.out + (uint64_t)row * a.n + t0;
    const uint32_t *mask = r.mask_row == LT_NO_MASK || !a.masks ? nullptr : a.masks + (uint64_t)r.mask_row * ((a.n + 31) / 32);
    const bool wide = ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) & 15) == 0;

    // the chunk: groups of four tokens, kLgThreads groups apart; only allowed ones are read
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
        v[u][0] = v[u][1] = v[u][2] = v[u][3] = -INFINITY;
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
    if (hist_len || bias_len) {
#pragma unroll
        for (int u = 0; u < kLgPer; u++)
            *reinterpret_cast<uint4 *>(s_table + (u * kLgThreads + tid) * 4) = make_uint4(0, 0, 0, 0);
        if (tid == 0) s_n = 0;
        __syncthreads();
        each_listed(a.history + r.history_first, hist_len, t0, nt, [&](uint32_t, uint32_t d) {
            if (atomicAdd(&s_table[d], 1u) == 0) s_work[atomicAdd(&s_n, 1u)] = (uint16_t)d;
        });
    }
#pragma unroll
    for (int u = 0; u < kLgPer; u++) {
        const uint32_t i = (u * kLgThreads + tid) * 4;
        if (i >= nt) continue;
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
    auto allowed = [&](uint32_t d) { return !mask || (mask[(t0 + d) >> 5] >> ((t0 + d) & 31) & 1u); };
    if (hist_len) {
        __syncthreads();
        const uint32_t n = s_n;
        for (uint32_t i = tid; i < n; i += kLgThreads) {
            const uint32_t d = s_work[i];
            const float c = (float)s_table[d];
            s_table[d] = 0;
            if (allowed(d)) {
                const float w = y[d];
                y[d] = (w > 0.0f ? __fdiv_rn(w, r.repetition) : w * r.repetition) - (c * r.frequency + r.presence);
            }
        }
    }
    if (bias_len) {
        __syncthreads();
        if (tid == 0) s_n = 0;
        __syncthreads();
        each_listed(a.bias_ids + r.bias_first, bias_len, t0, nt, [&](uint32_t i, uint32_t d) {
            if (atomicMax(&s_table[d], i + 1) == 0) s_work[atomicAdd(&s_n, 1u)] = (uint16_t)d;
        });
        __syncthreads();
        const uint32_t n = s_n;
        for (uint32_t i = tid; i < n; i += kLgThreads) {
            const uint32_t d = s_work[i];
            if (allowed(d)) y[d] += a.bias_values[(uint64_t)r.bias_first + s_table[d] - 1];
        }
    }
}

cudaError_t launch_logits(const LaunchCfg &c, const LogitArgs &a) {
    return launch_k(c, "logits", k_logits, dim3((a.n + kLgChunk - 1) / kLgChunk, a.n_rows), dim3(kLgThreads), 0, a);
}

}  // namespace lt
