// lt_logits.cu — what a request asks of its logits before a token is chosen.
//
// For token t of a row with history counts c(t) (lt_logit_rule):
//   y = x                                                       c(t) = 0
//   y = (x > 0 ? x / rep : x * rep) - (c(t) freq + pres)        c(t) > 0
//   y = y + bias(t)
//   y = -inf where the row's grammar mask has bit t clear.
//
// Bound: memory (a row is read and written once).  A CTA owns a chunk of one
// row's tokens: it counts the row's history into shared memory for its chunk
// only (integer atomics, so the order does not matter), then streams the chunk.
// Of a token that the bias list names twice the last entry counts: the list
// index goes through an integer maximum.
#include "lt_paged.cuh"
#include "llmtoy_cuda.h"

namespace lt {

constexpr int kLgThreads = 256;
constexpr int kLgChunk = 4096;

__global__ void __launch_bounds__(kLgThreads) k_logits(LogitArgs a) {
    __shared__ uint32_t s_count[kLgChunk];
    __shared__ uint32_t s_bias[kLgChunk];
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t row = blockIdx.y, t0 = blockIdx.x * kLgChunk, nt = min((uint32_t)kLgChunk, a.n - t0);
    const lt_logit_rule r = static_cast<const lt_logit_rule *>(a.rules)[row];
    for (uint32_t i = threadIdx.x; i < kLgChunk; i += kLgThreads) s_count[i] = s_bias[i] = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; a.history && i < r.history_len; i += kLgThreads) {
        const uint32_t d = a.history[(uint64_t)r.history_first + i] - t0;
        if (d < nt) atomicAdd(&s_count[d], 1u);
    }
    for (uint32_t i = threadIdx.x; a.bias_ids && i < r.bias_len; i += kLgThreads) {
        const uint32_t d = a.bias_ids[(uint64_t)r.bias_first + i] - t0;
        if (d < nt) atomicMax(&s_bias[d], i + 1);
    }
    __syncthreads();
    const float *x = a.logits + row * a.in_stride + t0;
    float *y = a.out + row * a.out_stride + t0;
    const uint32_t *mask = r.mask_row == LT_NO_MASK || !a.masks ? nullptr : a.masks + (uint64_t)r.mask_row * ((a.n + 31) / 32);
    for (uint32_t i = threadIdx.x; i < nt; i += kLgThreads) {
        float v = x[i];
        const uint32_t c = s_count[i], b = s_bias[i];
        if (c) v = (v > 0.0f ? __fdiv_rn(v, r.repetition) : v * r.repetition) - ((float)c * r.frequency + r.presence);
        if (b) v += a.bias_values[(uint64_t)r.bias_first + b - 1];
        if (mask && !(mask[(t0 + i) >> 5] >> ((t0 + i) & 31) & 1u)) v = -INFINITY;
        y[i] = v;
    }
}

cudaError_t launch_logits(const LaunchCfg &c, const LogitArgs &a) {
    return launch_k(c, "logits", k_logits, dim3((a.n + kLgChunk - 1) / kLgChunk, a.n_rows), dim3(kLgThreads), 0, a);
}

}  // namespace lt
