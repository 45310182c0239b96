// qmm_attn_check.h — the argument checks of the cache append and the attention,
// as plain C++ (no HIP): the entry points refuse by them, and a host program
// can check them without a device. Contents of device arrays are checked where
// the kernels use them.
#pragma once

#include <cmath>
#include <cstdint>

#include "../../include/qmm_hip.h"

namespace qmm {

struct Refusal {
    int code;         // QMM_OK: none
    const char *why;
};
constexpr Refusal kFine{QMM_OK, ""};

inline bool on(const void *p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

inline Refusal check_kv(const qmm_kv_batch *b, const qmm_kv_cache *c) {
    if (!b || !c) return {QMM_EINVAL, "null batch or cache"};
    if (b->n_seqs < 0 || b->n_rows < 0 || b->max_pages <= 0 || b->max_new < 0 || b->max_kv < 0)
        return {QMM_EINVAL, "negative batch size or no pages"};
    if (c->type != QMM_KV_F16 && c->type != QMM_KV_Q8) return {QMM_ETYPE, "unknown cache type"};
    if (c->page_tokens < 16 || c->page_tokens > 1024 || (c->page_tokens & (c->page_tokens - 1)))
        return {QMM_ESHAPE, "page_tokens must be a power of two, 16..1024"};
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return {QMM_ESHAPE, "head_dim must be 64, 128 or 256"};
    if (c->n_pages <= 0 || c->n_heads <= 0 || c->n_heads > 65535) return {QMM_EINVAL, "bad cache size"};
    if (int64_t(b->n_seqs) * c->n_heads >= (int64_t(1) << 24)) return {QMM_ESHAPE, "n_seqs * n_heads must stay below 2^24"};
    if (!c->k || !c->v) return {QMM_EINVAL, "null cache"};
    if (!on(c->k, 16) || !on(c->v, 16)) return {QMM_EALIGN, "cache must be 16-B aligned"};
    if (c->type == QMM_KV_Q8) {
        if (!c->k_scale || !c->v_scale) return {QMM_EINVAL, "8-bit cache without scales"};
        if (!on(c->k_scale, 16) || !on(c->v_scale, 16)) return {QMM_EALIGN, "cache scales must be 16-B aligned"};
    }
    if (b->n_seqs > 0 && b->n_rows > 0) {
        if (!b->row_start || !b->kv_len || !b->pages) return {QMM_EINVAL, "null batch array"};
        if (!on(b->row_start, 4) || !on(b->kv_len, 4) || !on(b->pages, 4)) return {QMM_EALIGN, "batch arrays must be 4-B aligned"};
    }
    return kFine;
}

inline Refusal check_attention(const qmm_kv_batch *b, const qmm_kv_cache *c, const qmm_attention_args *t) {
    const Refusal r = check_kv(b, c);
    if (r.code) return r;
    if (!t) return {QMM_EINVAL, "null attention arguments"};
    if (t->q_heads <= 0 || t->q_heads > (1 << 20) || t->q_heads % c->n_heads)
        return {QMM_ESHAPE, "q_heads must be a multiple of the cache's heads"};
    if (int64_t(b->n_rows) * (t->q_heads / c->n_heads) >= (int64_t(1) << 30))
        return {QMM_ESHAPE, "n_rows * q_heads / n_heads must stay below 2^30"};
    if (!(t->scale > 0.0f) || !std::isfinite(t->scale)) return {QMM_EINVAL, "scale must be positive and finite"};
    if (t->window < 0 || t->sinks < 0) return {QMM_EINVAL, "negative window or sinks"};
    if (t->out_type != QMM_TYPE_F16 && t->out_type != QMM_TYPE_F32) return {QMM_ETYPE, "out_type must be F16 or F32"};
    if (b->n_rows > 0) {
        const size_t width = size_t(t->q_heads) * size_t(c->head_dim);
        if (!t->q || !t->out) return {QMM_EINVAL, "null q or out"};
        if (t->q_stride < width || t->out_stride < width) return {QMM_EINVAL, "row stride below q_heads * head_dim"};
        if (!on(t->q, 16) || t->q_stride % 8) return {QMM_EALIGN, "q rows must be 16-B aligned"};
        if (!on(t->out, t->out_type == QMM_TYPE_F32 ? 16 : 8) || t->out_stride % 4)
            return {QMM_EALIGN, "output rows must be 8-B (F32: 16-B) aligned"};
    }
    return kFine;
}

// rot_dim: of the rotation table, 0 without one
inline Refusal check_append(const qmm_kv_batch *b, const qmm_kv_cache *c, const qmm_kv_rows *t, int rot_dim) {
    const Refusal r = check_kv(b, c);
    if (r.code) return r;
    if (!t) return {QMM_EINVAL, "null rows"};
    if (b->n_rows > 0) {
        const size_t kw = size_t(c->n_heads) * size_t(c->head_dim);
        if (!t->k || !t->v) return {QMM_EINVAL, "null keys or values"};
        if (t->k_stride < kw || t->v_stride < kw) return {QMM_EINVAL, "row stride below n_heads * head_dim"};
        if (!on(t->k, 16) || !on(t->v, 16) || t->k_stride % 4 || t->v_stride % 4)
            return {QMM_EALIGN, "key and value rows must be 16-B aligned"};
        if (t->q) {
            if (t->q_heads <= 0 || t->q_heads > (1 << 20)) return {QMM_EINVAL, "bad q_heads"};
            const size_t qw = size_t(t->q_heads) * size_t(c->head_dim);
            if (!t->q_out) return {QMM_EINVAL, "q without q_out"};
            if (t->q_stride < qw || t->q_out_stride < qw) return {QMM_EINVAL, "row stride below q_heads * head_dim"};
            if (!on(t->q, 16) || t->q_stride % 4) return {QMM_EALIGN, "query rows must be 16-B aligned"};
            if (!on(t->q_out, 8) || t->q_out_stride % 4) return {QMM_EALIGN, "q_out rows must be 8-B aligned"};
        }
    }
    if (!on(t->q_gamma, 16) || !on(t->k_gamma, 16)) return {QMM_EALIGN, "norm weights must be 16-B aligned"};
    if (!(t->eps >= 0.0f) || !std::isfinite(t->eps)) return {QMM_EINVAL, "eps must be finite and not negative"};
    if (rot_dim > c->head_dim) return {QMM_ESHAPE, "rot_dim above head_dim"};
    if (rot_dim && t->pos) {
        if (t->pos_stride < size_t(b->n_rows)) return {QMM_EINVAL, "pos_stride below n_rows"};
        if (!on(t->pos, 4)) return {QMM_EALIGN, "pos must be 4-B aligned"};
    }
    return kFine;
}

inline Refusal check_rope(const qmm_rope_params *t) {
    if (!t) return {QMM_EINVAL, "null rotation parameters"};
    if (t->rot_dim < 8 || t->rot_dim > 256 || t->rot_dim % 8) return {QMM_ESHAPE, "rot_dim must be a multiple of 8, 8..256"};
    if (t->style != QMM_ROPE_HALF && t->style != QMM_ROPE_PAIRS) return {QMM_EINVAL, "unknown rotation style"};
    if (t->n_axes < 1 || t->n_axes > 3) return {QMM_EINVAL, "n_axes must be 1..3"};
    if (!t->pair_freq && !(t->base > 0.0 && std::isfinite(t->base))) return {QMM_EINVAL, "base must be positive and finite"};
    if (!std::isfinite(t->scale)) return {QMM_EINVAL, "scale must be finite"};
    for (int j = 0; j < t->rot_dim / 2; ++j) {
        if (t->pair_freq && !std::isfinite(t->pair_freq[j])) return {QMM_EINVAL, "frequency not finite"};
        if (t->pair_axis && t->pair_axis[j] >= t->n_axes) return {QMM_EINVAL, "pair axis past n_axes"};
    }
    return kFine;
}

}  // namespace qmm
