// lt_paged_q8.cuh — a paged cache of 8-bit codes: where a block's scales lie, and
// how attention uses them.
//
// A block is 2^block_shift slots of a page and one KV head; value = code * scale.
// With ks and vs the scales of the block that position j lies in,
//   q . k_j = ks (q . code_j),      p_j v_j = (p_j vs) code_j.
// The weights' factor goes into their exponent: with t_j = s_j + log2 vs (s in units
// of log2) and m the largest t, P_j = 2^(t_j - m) is what multiplies the codes, and the
// sum of the weights is  l = sum over blocks of (1 / vs) sum_{j in block} P_j.  So neither
// scale costs an operation per position and dimension, and out = sum_j P_j code_j / l
// holds whatever m is.  vs is held to [2^-60, 2^60]: the exponents' span then leaves
// room for 2^30 positions in f32.
#pragma once

#include "lt_paged.cuh"

namespace lt {

// Place of the scales of position j of a sequence, on page `page`, for head h.
LT_DEVINL uint64_t q8_scale_at(const PagedKvDev &kv, uint32_t page, uint32_t j, uint32_t h) {
    return ((uint64_t)page * kv.n_kv + h) * kv.page_blocks + (slot_of(kv, j) >> kv.block_shift);
}

constexpr float kQ8Most = 1.152921504606847e18f, kQ8Least = 8.673617379884035e-19f;  // 2^60, 2^-60

// What scores and weights need of a block's scales: the factor on q . code, log2 of the weights'
// factor and its inverse.  Scales that cannot be used make the scores NaN, and nothing else.
struct Q8Scale {
    float k, v_log2, v_inv;
};
LT_DEVINL Q8Scale q8_scale(float ks, float vs) {
    Q8Scale r;
    const bool ok = ks >= 0.0f && ks <= 3.402823466e38f && vs >= 0.0f && vs <= kQ8Most;
    const float v = ok ? fmaxf(vs, kQ8Least) : 1.0f;
    r.k = ok ? ks : __int_as_float(0x7fffffff);
    // the approximations are off by 2^-22 (lg2, absolute between 1/2 and 2) and one unit in the last place, of f32: as much as a weight's
    // two terms; log2 and inverse need not agree better
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r.v_log2) : "f"(v));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.v_inv) : "f"(v));
    return r;
}

// Four signed bytes as f16, exactly: a byte b next to 0x64 is the f16 number 1024 + b.
LT_DEVINL void s8_to_f16(uint32_t w, uint32_t &b0, uint32_t &b1) {
    const uint32_t x = w ^ 0x80808080u;
    const uint32_t p = __byte_perm(x, 0x64646464u, 0x4140), q = __byte_perm(x, 0x64646464u, 0x4342);
    const __half2 off = __float2half2_rn(1152.0f);
    const __half2 u = __hsub2(*reinterpret_cast<const __half2 *>(&p), off), v = __hsub2(*reinterpret_cast<const __half2 *>(&q), off);
    b0 = *reinterpret_cast<const uint32_t *>(&u);
    b1 = *reinterpret_cast<const uint32_t *>(&v);
}

}  // namespace lt
