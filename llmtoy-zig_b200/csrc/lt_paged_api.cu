// lt_paged_api.cu — entry points of the batched-serving operators: argument
// checks, scratch, launches (lt_paged_append.cu, lt_paged_attn.cu, lt_paged_q8_append.cu,
// lt_paged_q8_attn.cu, lt_paged_plan.cu, lt_evict.cu, lt_logits.cu).
#include <cmath>

#include "llmtoy_cuda.h"
#include "lt_internal.h"

namespace {

using lt::ctx_fail;

lt_status st_of(int s) { return (lt_status)s; }

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

constexpr uint32_t kMaxLen = 1u << 30;  // positions of a sequence: 32-bit position arithmetic stays exact

lt_status paged_kv(lt_ctx *ctx, const lt_paged_kv *kv, const char *who, lt::PagedKvDev &d) {
    if (!kv || !kv->dev_k || !kv->dev_v) return st_of(ctx_fail(ctx, LT_EINVAL, "%s: null cache", who));
    if (kv->head_dim != 64 && kv->head_dim != 128 && kv->head_dim != 256)
        return st_of(ctx_fail(ctx, LT_EINVAL, "%s: head_dim %u (64, 128 or 256)", who, kv->head_dim));
    if (kv->n_kv_heads == 0 || kv->n_kv_heads > 1024)
        return st_of(ctx_fail(ctx, LT_EINVAL, "%s: %u KV heads", who, kv->n_kv_heads));
    if (kv->page_size == 0 || kv->n_pages == 0 || kv->max_pages == 0)
        return st_of(ctx_fail(ctx, LT_EINVAL, "%s: page_size %u, n_pages %u, max_pages %u", who, kv->page_size,
                              kv->n_pages, kv->max_pages));
    const uint64_t size = kv->kv_f16 ? 2 : 4;
    const bool plain = !kv->page_stride && !kv->slot_stride && !kv->head_stride;
    if (!plain && (!kv->page_stride || !kv->slot_stride || !kv->head_stride))
        return st_of(ctx_fail(ctx, LT_EINVAL, "%s: give all three strides or none", who));
    d.head_stride = (plain ? kv->head_dim : kv->head_stride) * size;
    d.slot_stride = (plain ? (uint64_t)kv->n_kv_heads * kv->head_dim : kv->slot_stride) * size;
    d.page_stride = plain ? kv->page_size * d.slot_stride : kv->page_stride * size;
    if (d.head_stride % 16 || d.slot_stride % 16 || d.page_stride % 16 || !aligned16(kv->dev_k) || !aligned16(kv->dev_v))
        return st_of(ctx_fail(ctx, LT_EINVAL, "%s: cache addresses and strides must be multiples of 16 bytes", who));
    d.k = (uint8_t *)kv->dev_k;
    d.v = (uint8_t *)kv->dev_v;
    d.n_kv = kv->n_kv_heads;
    d.hd = kv->head_dim;
    d.f16 = kv->kv_f16 != 0;
    d.page_size = kv->page_size;
    d.n_pages = kv->n_pages;
    d.max_pages = kv->max_pages;
    d.page_shift = lt::kNoShift;
    for (uint32_t i = 0; i < 32; i++)
        if (kv->page_size == 1u << i) d.page_shift = i;
    return LT_OK;
}

lt_status paged_q8(lt_ctx *ctx, const lt_paged_q8 *kv, const char *who, lt::PagedKvDev &d) {
    if (!kv || !kv->dev_k || !kv->dev_v || !kv->dev_k_scale || !kv->dev_v_scale)
        return st_of(ctx_fail(ctx, LT_EINVAL, "%s: null cache", who));
    if (kv->head_dim != 64 && kv->head_dim != 128 && kv->head_dim != 256)
        return st_of(ctx_fail(ctx, LT_EINVAL, "%s: head_dim %u (64, 128 or 256)", who, kv->head_dim));
    if (kv->n_kv_heads == 0 || kv->n_kv_heads > 1024)
        return st_of(ctx_fail(ctx, LT_EINVAL, "%s: %u KV heads", who, kv->n_kv_heads));
    if (kv->block != 16 && kv->block != 32 && kv->block != 64 && kv->block != 128)
        return st_of(ctx_fail(ctx, LT_EINVAL, "%s: blocks of %u positions (16, 32, 64 or 128)", who, kv->block));
    if (kv->page_size == 0 || kv->page_size % kv->block || kv->n_pages == 0 || kv->max_pages == 0)
        return st_of(ctx_fail(ctx, LT_EINVAL, "%s: page_size %u (a multiple of %u), n_pages %u, max_pages %u", who,
                              kv->page_size, kv->block, kv->n_pages, kv->max_pages));
    const bool plain = !kv->page_stride && !kv->slot_stride && !kv->head_stride;
    if (!plain && (!kv->page_stride || !kv->slot_stride || !kv->head_stride))
        return st_of(ctx_fail(ctx, LT_EINVAL, "%s: give all three strides or none", who));
    d.slot_stride = plain ? kv->head_dim : kv->slot_stride;
    d.head_stride = plain ? (uint64_t)kv->page_size * kv->head_dim : kv->head_stride;
    d.page_stride = plain ? kv->n_kv_heads * d.head_stride : kv->page_stride;
    if (d.head_stride % 16 || d.slot_stride % 16 || d.page_stride % 16 || !aligned16(kv->dev_k) || !aligned16(kv->dev_v))
        return st_of(ctx_fail(ctx, LT_EINVAL, "%s: cache addresses and strides must be multiples of 16 bytes", who));
    if ((d.head_stride | d.slot_stride | d.page_stride) >> 32 || (uint64_t)kv->n_kv_heads * (kv->page_size / kv->block) >> 32)
        return st_of(ctx_fail(ctx, LT_EINVAL, "%s: strides must be below 2^32 bytes", who));
    if (((uintptr_t)kv->dev_k_scale | (uintptr_t)kv->dev_v_scale) & 3)
        return st_of(ctx_fail(ctx, LT_EINVAL, "%s: scales must be 4-byte aligned", who));
    d.k = (uint8_t *)kv->dev_k;
    d.v = (uint8_t *)kv->dev_v;
    d.k_scale = kv->dev_k_scale;
    d.v_scale = kv->dev_v_scale;
    d.n_kv = kv->n_kv_heads;
    d.hd = kv->head_dim;
    d.f16 = 0;
    d.page_size = kv->page_size;
    d.n_pages = kv->n_pages;
    d.max_pages = kv->max_pages;
    d.page_shift = lt::kNoShift;
    for (uint32_t i = 0; i < 32; i++) {
        if (kv->page_size == 1u << i) d.page_shift = i;
        if (kv->block == 1u << i) d.block_shift = i;
    }
    d.page_blocks = kv->page_size / kv->block;
    return LT_OK;
}

// The rest of an attention call's arguments, a.kv being checked.
lt_status paged_attn_rest(lt_ctx *ctx, const char *who, const lt_paged_attn_cfg *cfg, lt::PagedAttnArgs &a) {
    const lt::PagedKvDev *kv = &a.kv;
    if (!cfg) return st_of(ctx_fail(ctx, LT_EINVAL, "%s: null configuration", who));
    if (cfg->n_heads == 0 || cfg->n_heads > 4096 || cfg->n_heads % kv->n_kv)
        return st_of(ctx_fail(ctx, LT_EINVAL, "%s: %u query heads over %u KV heads", who, cfg->n_heads, kv->n_kv));
    if (!(cfg->scale - cfg->scale == 0.0f) || !(cfg->softcap >= 0.0f) || cfg->softcap - cfg->softcap != 0.0f)
        return st_of(ctx_fail(ctx, LT_EINVAL, "%s: scale %g, softcap %g", who, cfg->scale, cfg->softcap));
    const uint64_t row = (uint64_t)cfg->n_heads * kv->hd;
    a.q_stride = cfg->q_stride ? cfg->q_stride : row;
    a.out_stride = cfg->out_stride ? cfg->out_stride : row;
    if (a.q_stride < row || a.out_stride < row || a.q_stride % 4 || a.out_stride % 4)
        return st_of(ctx_fail(ctx, LT_EINVAL, "%s: row strides must be multiples of 4 and at least %llu", who,
                              (unsigned long long)row));
    if (!aligned16(a.q) || !aligned16(a.out))
        return st_of(ctx_fail(ctx, LT_EINVAL, "%s: queries and output must be 16-byte aligned", who));
    if (a.n_seq > 65535) return st_of(ctx_fail(ctx, LT_EINVAL, "%s: %u sequences (at most 65535)", who, a.n_seq));
    if (a.max_len == 0 || a.max_len > kMaxLen)
        return st_of(ctx_fail(ctx, LT_EINVAL, "%s: max_len %u (1 to %u)", who, a.max_len, kMaxLen));
    a.n_heads = cfg->n_heads;
    a.group = cfg->n_heads / kv->n_kv;
    a.window = cfg->window;
    a.causal = cfg->causal != 0;
    a.scale = cfg->scale;
    a.softcap = cfg->softcap;
    a.slopes = cfg->dev_slopes;
    return LT_OK;
}

lt_status paged_attn(lt_ctx *ctx, const char *who, const lt_paged_attn_cfg *cfg, const lt_paged_kv *kv,
                     lt::PagedAttnArgs &a) {
    const lt_status st = paged_kv(ctx, kv, who, a.kv);
    return st != LT_OK ? st : paged_attn_rest(ctx, who, cfg, a);
}

// What a prompt call gives beside the cache and the configuration.
lt_status paged_prompt_rest(lt_ctx *ctx, const char *who, uint32_t &max_q, uint32_t total_q, uint64_t doc_stride,
                            const uint32_t *docs, const lt::PagedAttnArgs &a) {
    if (docs && (doc_stride < a.max_len || doc_stride > 0xffffffffull))
        return st_of(ctx_fail(ctx, LT_EINVAL, "%s: doc_stride %llu, max_len %u", who, (unsigned long long)doc_stride, a.max_len));
    if (max_q > total_q) max_q = total_q;
    if ((uint64_t)max_q * a.group > 0x7fffffffull || (uint64_t)max_q * a.n_heads / 8 * a.n_seq > 0x3fffffffull)
        return st_of(ctx_fail(ctx, LT_EINVAL, "%s: max_q %u of %u sequences is too large", who, max_q, a.n_seq));
    return LT_OK;
}

}  // namespace

extern "C" {

lt_status lt_paged_append(lt_ctx *ctx, const lt_attn_cfg *cfg, const lt_paged_kv *kv, const float *dev_qkv,
                          uint32_t ntok, const float *dev_q_norm, const float *dev_k_norm, const uint32_t *dev_seq,
                          const uint32_t *dev_pos, const uint32_t *dev_slot, const uint32_t *dev_page_table,
                          uint32_t n_seq, float *dev_q) {
    lt_status st = st_of(lt::ctx_enter(ctx));
    if (st != LT_OK) return st;
    lt::PagedAppendArgs a = {};
    if ((st = paged_kv(ctx, kv, "lt_paged_append", a.kv)) != LT_OK) return st;
    if (!cfg || !dev_qkv || !dev_seq || !dev_pos || !dev_page_table || !dev_q)
        return st_of(ctx_fail(ctx, LT_EINVAL, "lt_paged_append: null argument"));
    if (cfg->head_dim != kv->head_dim || cfg->n_kv_heads != kv->n_kv_heads)
        return st_of(ctx_fail(ctx, LT_EINVAL, "lt_paged_append: cfg has %u KV heads of %u, the cache %u of %u",
                              cfg->n_kv_heads, cfg->head_dim, kv->n_kv_heads, kv->head_dim));
    if (cfg->n_heads == 0 || cfg->n_heads > 4096)
        return st_of(ctx_fail(ctx, LT_EINVAL, "lt_paged_append: %u query heads", cfg->n_heads));
    if (!aligned16(dev_qkv) || !aligned16(dev_q))
        return st_of(ctx_fail(ctx, LT_EINVAL, "lt_paged_append: dev_qkv and dev_q must be 16-byte aligned"));
    if (ntok == 0) return LT_OK;
    if (n_seq == 0) return st_of(ctx_fail(ctx, LT_EINVAL, "lt_paged_append: no sequences"));
    a.n_heads = cfg->n_heads;
    a.rope_neox = cfg->rope_neox;
    a.v_norm = cfg->v_norm;
    a.n_seq = n_seq;
    a.ntok = ntok;
    a.theta = cfg->rope_theta;
    a.eps = cfg->eps;
    a.qkv = dev_qkv;
    a.q_norm = dev_q_norm;
    a.k_norm = dev_k_norm;
    a.seq = dev_seq;
    a.pos = dev_pos;
    a.slot = dev_slot;
    a.table = dev_page_table;
    a.q = dev_q;
    return st_of(lt::ctx_launched(ctx, lt::launch_paged_append(lt::ctx_cfg(ctx), a), "paged append"));
}

lt_status lt_paged_attn_decode(lt_ctx *ctx, const lt_paged_attn_cfg *cfg, const lt_paged_kv *kv, const float *dev_q,
                               uint32_t n_seq, const uint32_t *dev_page_table, const uint32_t *dev_lens,
                               uint32_t max_len, float *dev_mass, uint64_t mass_stride, float *dev_out) {
    lt_status st = st_of(lt::ctx_enter(ctx));
    if (st != LT_OK) return st;
    if (!dev_q || !dev_page_table || !dev_lens || !dev_out)
        return st_of(ctx_fail(ctx, LT_EINVAL, "lt_paged_attn_decode: null argument"));
    lt::PagedAttnArgs a = {};
    a.q = dev_q;
    a.out = dev_out;
    a.n_seq = n_seq;
    a.max_len = max_len;
    if ((st = paged_attn(ctx, "lt_paged_attn_decode", cfg, kv, a)) != LT_OK) return st;
    if (dev_mass && mass_stride < max_len)
        return st_of(ctx_fail(ctx, LT_EINVAL, "lt_paged_attn_decode: mass_stride %llu < max_len %u",
                              (unsigned long long)mass_stride, max_len));
    if (n_seq == 0) return LT_OK;
    a.max_q = 1;
    a.total_q = n_seq;
    a.table = dev_page_table;
    a.lens = dev_lens;
    a.mass = dev_mass;
    a.mass_stride = mass_stride;
    const lt::LaunchCfg c = lt::ctx_cfg(ctx);
    uint8_t *scratch = nullptr;
    const size_t need = lt::paged_attn_scratch(a, c.num_sms);
    if ((st = st_of(lt::ctx_scratch(ctx, need, need, &scratch))) != LT_OK) return st;
    return st_of(lt::ctx_launched(ctx, lt::launch_paged_attn(c, a, scratch), "paged attention"));
}

lt_status lt_paged_attn_prompt(lt_ctx *ctx, const lt_paged_attn_cfg *cfg, const lt_paged_kv *kv, const float *dev_q,
                               uint32_t n_seq, const uint32_t *dev_cu_q, uint32_t total_q, uint32_t max_q,
                               const uint32_t *dev_page_table, const uint32_t *dev_lens, uint32_t max_len,
                               const uint32_t *dev_prefix, const uint32_t *dev_docs, uint64_t doc_stride,
                               float *dev_out) {
    lt_status st = st_of(lt::ctx_enter(ctx));
    if (st != LT_OK) return st;
    if (!dev_q || !dev_cu_q || !dev_page_table || !dev_lens || !dev_out)
        return st_of(ctx_fail(ctx, LT_EINVAL, "lt_paged_attn_prompt: null argument"));
    lt::PagedAttnArgs a = {};
    a.q = dev_q;
    a.out = dev_out;
    a.n_seq = n_seq;
    a.max_len = max_len;
    if ((st = paged_attn(ctx, "lt_paged_attn_prompt", cfg, kv, a)) != LT_OK) return st;
    if ((st = paged_prompt_rest(ctx, "lt_paged_attn_prompt", max_q, total_q, doc_stride, dev_docs, a)) != LT_OK) return st;
    if (n_seq == 0 || max_q == 0) return LT_OK;
    a.max_q = max_q;
    a.total_q = total_q;
    a.cu = dev_cu_q;
    a.table = dev_page_table;
    a.lens = dev_lens;
    a.prefix = dev_prefix;
    a.docs = dev_docs;
    a.doc_stride = (uint32_t)doc_stride;
    const lt::LaunchCfg c = lt::ctx_cfg(ctx);
    uint8_t *scratch = nullptr;
    if (lt::paged_prompt_supported(a)) {
        const size_t need = lt::paged_prompt_scratch(a, c.num_sms), most = lt::paged_prompt_scratch_most(a, c.num_sms);
        if ((st = st_of(lt::ctx_scratch(ctx, most, need, &scratch))) != LT_OK) return st;
        return st_of(lt::ctx_launched(ctx, lt::launch_paged_prompt(c, a, scratch), "paged prompt attention"));
    }
    const size_t need = lt::paged_attn_scratch(a, c.num_sms);
    if ((st = st_of(lt::ctx_scratch(ctx, need, need, &scratch))) != LT_OK) return st;
    return st_of(lt::ctx_launched(ctx, lt::launch_paged_attn(c, a, scratch), "paged prompt attention"));
}

lt_status lt_kv_evict(lt_ctx *ctx, const lt_paged_kv *kv, uint32_t n_seq, const uint32_t *dev_page_table,
                      const uint32_t *dev_lens, uint32_t max_len, const float *dev_mass, uint64_t mass_stride,
                      uint32_t budget, uint32_t recent, const uint32_t *dev_dst_table, uint32_t *dev_lens_out,
                      float *dev_mass_out, uint64_t mass_out_stride, uint32_t *dev_kept) {
    lt_status st = st_of(lt::ctx_enter(ctx));
    if (st != LT_OK) return st;
    lt::EvictArgs a = {};
    if ((st = paged_kv(ctx, kv, "lt_kv_evict", a.kv)) != LT_OK) return st;
    if (!dev_page_table || !dev_lens || !dev_mass || !dev_lens_out || !dev_mass_out)
        return st_of(ctx_fail(ctx, LT_EINVAL, "lt_kv_evict: null argument"));
    if (budget == 0 || recent > budget)
        return st_of(ctx_fail(ctx, LT_EINVAL, "lt_kv_evict: budget %u, recent %u", budget, recent));
    if (max_len == 0 || max_len > kMaxLen || n_seq > 65535)
        return st_of(ctx_fail(ctx, LT_EINVAL, "lt_kv_evict: max_len %u, %u sequences", max_len, n_seq));
    if (mass_stride < max_len || mass_out_stride < (budget < max_len ? budget : max_len))
        return st_of(ctx_fail(ctx, LT_EINVAL, "lt_kv_evict: mass strides %llu and %llu", (unsigned long long)mass_stride,
                              (unsigned long long)mass_out_stride));
    if (dev_mass_out == dev_mass && mass_out_stride != mass_stride)
        return st_of(ctx_fail(ctx, LT_EINVAL, "lt_kv_evict: masses updated in place need one stride"));
    if (n_seq == 0) return LT_OK;
    a.n_seq = n_seq;
    a.max_len = max_len;
    a.budget = budget;
    a.recent = recent;
    a.table = dev_page_table;
    a.lens = dev_lens;
    a.dst_table = dev_dst_table;
    a.in_place = !dev_dst_table || dev_dst_table == dev_page_table;
    a.mass = dev_mass;
    a.mass_stride = mass_stride;
    a.mass_out_stride = mass_out_stride;
    a.lens_out = dev_lens_out;
    a.kept = dev_kept;
    a.mass_out = dev_mass_out;
    uint8_t *scratch = nullptr;
    const size_t need = lt::evict_scratch(a, dev_kept != nullptr);
    if ((st = st_of(lt::ctx_scratch(ctx, need, need, &scratch))) != LT_OK) return st;
    return st_of(lt::ctx_launched(ctx, lt::launch_evict(lt::ctx_cfg(ctx), a, scratch), "evict"));
}

lt_status lt_paged_q8_append(lt_ctx *ctx, const lt_attn_cfg *cfg, const lt_paged_q8 *kv, const float *dev_qkv,
                             uint32_t n_seq, const uint32_t *dev_cu_q, uint32_t total_q, uint32_t max_q,
                             const float *dev_q_norm, const float *dev_k_norm, const uint32_t *dev_pos,
                             const uint32_t *dev_page_table, const uint32_t *dev_lens, float *dev_q) {
    lt_status st = st_of(lt::ctx_enter(ctx));
    if (st != LT_OK) return st;
    lt::PagedQ8AppendArgs a = {};
    if ((st = paged_q8(ctx, kv, "lt_paged_q8_append", a.kv)) != LT_OK) return st;
    if (!cfg || !dev_qkv || !dev_cu_q || !dev_page_table || !dev_lens || !dev_q)
        return st_of(ctx_fail(ctx, LT_EINVAL, "lt_paged_q8_append: null argument"));
    if (cfg->head_dim != kv->head_dim || cfg->n_kv_heads != kv->n_kv_heads)
        return st_of(ctx_fail(ctx, LT_EINVAL, "lt_paged_q8_append: cfg has %u KV heads of %u, the cache %u of %u",
                              cfg->n_kv_heads, cfg->head_dim, kv->n_kv_heads, kv->head_dim));
    if (cfg->n_heads == 0 || cfg->n_heads > 4096)
        return st_of(ctx_fail(ctx, LT_EINVAL, "lt_paged_q8_append: %u query heads", cfg->n_heads));
    if (!(cfg->rope_theta > 0.0f) || cfg->rope_theta - cfg->rope_theta != 0.0f)
        return st_of(ctx_fail(ctx, LT_EINVAL, "lt_paged_q8_append: rope_theta %g", cfg->rope_theta));
    if (!aligned16(dev_qkv) || !aligned16(dev_q))
        return st_of(ctx_fail(ctx, LT_EINVAL, "lt_paged_q8_append: dev_qkv and dev_q must be 16-byte aligned"));
    if (n_seq > 65535 || total_q > kMaxLen)
        return st_of(ctx_fail(ctx, LT_EINVAL, "lt_paged_q8_append: %u sequences (at most 65535), %u tokens (at most %u)",
                              n_seq, total_q, kMaxLen));
    if (max_q > total_q) max_q = total_q;
    if (n_seq == 0 || max_q == 0) return LT_OK;
    a.n_heads = cfg->n_heads;
    a.rope_neox = cfg->rope_neox;
    a.v_norm = cfg->v_norm;
    a.n_seq = n_seq;
    a.total_q = total_q;
    a.max_q = max_q;
    a.log2_theta = log2((double)cfg->rope_theta);
    a.eps = cfg->eps;
    a.qkv = dev_qkv;
    a.q_norm = dev_q_norm;
    a.k_norm = dev_k_norm;
    a.cu = dev_cu_q;
    a.pos = dev_pos;
    a.table = dev_page_table;
    a.lens = dev_lens;
    a.q = dev_q;
    return st_of(lt::ctx_launched(ctx, lt::launch_paged_q8_append(lt::ctx_cfg(ctx), a), "8-bit paged append"));
}

lt_status lt_paged_q8_attn_decode(lt_ctx *ctx, const lt_paged_attn_cfg *cfg, const lt_paged_q8 *kv, const float *dev_q,
                                  uint32_t n_seq, const uint32_t *dev_page_table, const uint32_t *dev_lens,
                                  uint32_t max_len, float *dev_out) {
    lt_status st = st_of(lt::ctx_enter(ctx));
    if (st != LT_OK) return st;
    if (!dev_q || !dev_page_table || !dev_lens || !dev_out)
        return st_of(ctx_fail(ctx, LT_EINVAL, "lt_paged_q8_attn_decode: null argument"));
    lt::PagedAttnArgs a = {};
    a.q = dev_q;
    a.out = dev_out;
    a.n_seq = n_seq;
    a.max_len = max_len;
    if ((st = paged_q8(ctx, kv, "lt_paged_q8_attn_decode", a.kv)) != LT_OK) return st;
    if ((st = paged_attn_rest(ctx, "lt_paged_q8_attn_decode", cfg, a)) != LT_OK) return st;
    if (n_seq == 0) return LT_OK;
    a.max_q = 1;
    a.total_q = n_seq;
    a.table = dev_page_table;
    a.lens = dev_lens;
    const lt::LaunchCfg c = lt::ctx_cfg(ctx);
    uint8_t *scratch = nullptr;
    const size_t need = lt::paged_q8_attn_scratch(a, c.num_sms);
    if ((st = st_of(lt::ctx_scratch(ctx, need, need, &scratch))) != LT_OK) return st;
    return st_of(lt::ctx_launched(ctx, lt::launch_paged_q8_attn(c, a, scratch), "8-bit paged attention"));
}

lt_status lt_paged_q8_attn_prompt(lt_ctx *ctx, const lt_paged_attn_cfg *cfg, const lt_paged_q8 *kv, const float *dev_q,
                                  uint32_t n_seq, const uint32_t *dev_cu_q, uint32_t total_q, uint32_t max_q,
                                  const uint32_t *dev_page_table, const uint32_t *dev_lens, uint32_t max_len,
                                  const uint32_t *dev_prefix, const uint32_t *dev_docs, uint64_t doc_stride,
                                  float *dev_out) {
    lt_status st = st_of(lt::ctx_enter(ctx));
    if (st != LT_OK) return st;
    if (!dev_q || !dev_cu_q || !dev_page_table || !dev_lens || !dev_out)
        return st_of(ctx_fail(ctx, LT_EINVAL, "lt_paged_q8_attn_prompt: null argument"));
    lt::PagedAttnArgs a = {};
    a.q = dev_q;
    a.out = dev_out;
    a.n_seq = n_seq;
    a.max_len = max_len;
    if ((st = paged_q8(ctx, kv, "lt_paged_q8_attn_prompt", a.kv)) != LT_OK) return st;
    if ((st = paged_attn_rest(ctx, "lt_paged_q8_attn_prompt", cfg, a)) != LT_OK) return st;
    if ((st = paged_prompt_rest(ctx, "lt_paged_q8_attn_prompt", max_q, total_q, doc_stride, dev_docs, a)) != LT_OK) return st;
    if (n_seq == 0 || max_q == 0) return LT_OK;
    a.max_q = max_q;
    a.total_q = total_q;
    a.cu = dev_cu_q;
    a.table = dev_page_table;
    a.lens = dev_lens;
    a.prefix = dev_prefix;
    a.docs = dev_docs;
    a.doc_stride = (uint32_t)doc_stride;
    const lt::LaunchCfg c = lt::ctx_cfg(ctx);
    uint8_t *scratch = nullptr;
    const size_t most = lt::paged_prompt_scratch_most(a, c.num_sms);
    if (lt::paged_prompt_supported(a)) {
        const size_t need = lt::paged_prompt_scratch(a, c.num_sms);
        if ((st = st_of(lt::ctx_scratch(ctx, most, need, &scratch))) != LT_OK) return st;
        return st_of(lt::ctx_launched(ctx, lt::launch_paged_prompt(c, a, scratch), "8-bit paged prompt attention"));
    }
    const size_t need = lt::paged_q8_attn_scratch(a, c.num_sms);
    if ((st = st_of(lt::ctx_scratch(ctx, most > need ? most : need, need, &scratch))) != LT_OK) return st;
    return st_of(lt::ctx_launched(ctx, lt::launch_paged_q8_attn(c, a, scratch), "8-bit paged prompt attention"));
}

lt_status lt_paged_plan(lt_ctx *ctx, const lt_paged_state *state, const uint32_t *dev_keep, const uint32_t *dev_new,
                        uint32_t total_q, uint32_t *dev_cu_q, uint32_t *dev_seq, uint32_t *dev_pos,
                        uint32_t *dev_pool_slot) {
    lt_status st = st_of(lt::ctx_enter(ctx));
    if (st != LT_OK) return st;
    if (!state || !state->dev_lens || !state->dev_page_table || !state->dev_free || !state->dev_n_free || !dev_new || !dev_cu_q)
        return st_of(ctx_fail(ctx, LT_EINVAL, "lt_paged_plan: null argument"));
    if (state->page_size == 0 || state->n_pages == 0 || state->max_pages == 0)
        return st_of(ctx_fail(ctx, LT_EINVAL, "lt_paged_plan: page_size %u, n_pages %u, max_pages %u", state->page_size,
                              state->n_pages, state->max_pages));
    if ((uint64_t)state->n_pages * state->page_size > 0xffffffffull)
        return st_of(ctx_fail(ctx, LT_EINVAL, "lt_paged_plan: %u pages of %u slots (fewer than 2^32 slots)", state->n_pages,
                              state->page_size));
    if (state->n_seq > 65535 || total_q > kMaxLen)
        return st_of(ctx_fail(ctx, LT_EINVAL, "lt_paged_plan: %u sequences (at most 65535), %u tokens (at most %u)",
                              state->n_seq, total_q, kMaxLen));
    if (state->n_seq == 0)  // the sums of nothing: one 0
        return st_of(lt::ctx_launched(ctx, cudaMemsetAsync(dev_cu_q, 0, sizeof(uint32_t), lt::ctx_stream(ctx)), "page plan"));
    lt::PagedPlanArgs a = {};
    a.n_seq = state->n_seq;
    a.page = state->page_size;
    a.n_pages = state->n_pages;
    a.max_pages = state->max_pages;
    a.total_q = total_q;
    a.keep = dev_keep;
    a.add = dev_new;
    a.lens = state->dev_lens;
    a.table = state->dev_page_table;
    a.free = state->dev_free;
    a.n_free = state->dev_n_free;
    a.cu = dev_cu_q;
    a.seq = dev_seq;
    a.pos = dev_pos;
    a.slot = dev_pool_slot;
    uint8_t *scratch = nullptr;
    const size_t need = lt::paged_plan_scratch(a);
    if ((st = st_of(lt::ctx_scratch(ctx, need, need, &scratch))) != LT_OK) return st;
    return st_of(lt::ctx_launched(ctx, lt::launch_paged_plan(lt::ctx_cfg(ctx), a, scratch), "page plan"));
}

lt_status lt_logits_process(lt_ctx *ctx, const float *dev_logits, uint32_t n, uint32_t n_rows,
                            const lt_logit_rule *dev_rules, const uint32_t *dev_history,
                            const uint32_t *dev_bias_ids, const float *dev_bias_values, const uint32_t *dev_masks,
                            float *dev_out) {
    lt_status st = st_of(lt::ctx_enter(ctx));
    if (st != LT_OK) return st;
    if (!dev_logits || !dev_rules || !dev_out) return st_of(ctx_fail(ctx, LT_EINVAL, "lt_logits_process: null argument"));
    if (n > 0x7fffffffu || n_rows > 65535)
        return st_of(ctx_fail(ctx, LT_EINVAL, "lt_logits_process: %u rows of %u logits", n_rows, n));
    if ((dev_bias_ids == nullptr) != (dev_bias_values == nullptr))
        return st_of(ctx_fail(ctx, LT_EINVAL, "lt_logits_process: bias ids and values go together"));
    if (n == 0 || n_rows == 0) return LT_OK;
    lt::LogitArgs a = {dev_logits, n, n_rows, dev_rules, dev_history, dev_bias_ids, dev_bias_values, dev_masks, dev_out};
    return st_of(lt::ctx_launched(ctx, lt::launch_logits(lt::ctx_cfg(ctx), a), "logits"));
}

}  // extern "C"
