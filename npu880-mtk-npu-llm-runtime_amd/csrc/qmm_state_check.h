// qmm_state_check.h — the argument checks of the short convolution, the gated
// delta rule, the beam selection and the copy of slots, as plain C++ (no HIP), so
// that a host program can check them without a device. Contents of device arrays
// are checked where the kernels use them.
#pragma once

#include "qmm_attn_check.h"
#include "qmm_state.h"

namespace qmm {

constexpr int kMaxBeams = 64, kMaxKeep = 64;

inline Refusal check_state_batch(const qmm_state_batch *b) {
    if (!b) return {QMM_EINVAL, "null batch"};
    if (b->n_seqs < 0 || b->n_rows < 0 || b->n_slots < 0 || b->max_new < 0) return {QMM_EINVAL, "negative batch size"};
    if (b->n_rows >= (1 << 30)) return {QMM_ESHAPE, "n_rows must stay below 2^30"};
    if (b->n_seqs > 0 && !b->row_start) return {QMM_EINVAL, "null row_start"};
    if (!on(b->row_start, 4) || !on(b->slot_in, 4) || !on(b->slot_out, 4)) return {QMM_EALIGN, "batch arrays must be 4-B aligned"};
    return kFine;
}

inline Refusal check_conv(const qmm_state_batch *b, const qmm_conv_args *t) {
    const Refusal r = check_state_batch(b);
    if (r.code) return r;
    if (!t) return {QMM_EINVAL, "null convolution arguments"};
    if (t->width < 2 || t->width > 4) return {QMM_ESHAPE, "width must be 2..4"};
    if (t->channels <= 0 || t->channels % 4) return {QMM_ESHAPE, "channels must be a positive multiple of 4"};
    if (t->channels > (1 << 24)) return {QMM_ESHAPE, "channels must not pass 2^24"};
    if (int64_t(b->n_seqs) * ((t->channels + 1023) / 1024) >= (int64_t(1) << 24))
        return {QMM_ESHAPE, "n_seqs * channels / 1024 must stay below 2^24"};
    if (!t->weight) return {QMM_EINVAL, "null weights"};
    if (!on(t->weight, 16) || !on(t->bias, 16)) return {QMM_EALIGN, "weights and bias must be 16-B aligned"};
    if ((b->slot_in || b->slot_out) && b->n_slots > 0 && !t->state) return {QMM_EINVAL, "slots without a state"};
    if (!on(t->state, 16)) return {QMM_EALIGN, "state must be 16-B aligned"};
    if (b->n_rows > 0) {
        if (!t->x || !t->out) return {QMM_EINVAL, "null x or out"};
        if (t->x_stride < size_t(t->channels) || t->out_stride < size_t(t->channels)) return {QMM_EINVAL, "row stride below channels"};
        if (!on(t->x, 16) || !on(t->out, 16) || t->x_stride % 4 || t->out_stride % 4) return {QMM_EALIGN, "rows must be 16-B aligned"};
    }
    return kFine;
}

inline Refusal check_delta(const qmm_state_batch *b, const qmm_delta_args *t) {
    const Refusal r = check_state_batch(b);
    if (r.code) return r;
    if (!t) return {QMM_EINVAL, "null delta rule arguments"};
    if ((t->key_dim != 64 && t->key_dim != 128) || (t->value_dim != 64 && t->value_dim != 128))
        return {QMM_ESHAPE, "key_dim and value_dim must be 64 or 128"};
    if (t->qk_heads <= 0 || t->v_heads <= 0 || t->v_heads > 65535 || t->v_heads % t->qk_heads)
        return {QMM_ESHAPE, "v_heads must be a multiple of qk_heads, up to 65535"};
    if (int64_t(b->n_seqs) * t->v_heads >= (int64_t(1) << 24)) return {QMM_ESHAPE, "n_seqs * v_heads must stay below 2^24"};
    if (!t->rate || !t->dt_bias) return {QMM_EINVAL, "null rate or dt_bias"};
    if (!on(t->rate, 4) || !on(t->dt_bias, 4)) return {QMM_EALIGN, "rate and dt_bias must be 4-B aligned"};
    if (!(t->scale > 0.0f) || !std::isfinite(t->scale)) return {QMM_EINVAL, "scale must be positive and finite"};
    if (!(t->qk_eps > 0.0f) || !std::isfinite(t->qk_eps)) return {QMM_EINVAL, "qk_eps must be positive and finite"};
    if (!(t->gamma_eps >= 0.0f) || !std::isfinite(t->gamma_eps)) return {QMM_EINVAL, "gamma_eps must be finite and not negative"};
    if ((b->slot_in || b->slot_out) && b->n_slots > 0 && !t->state) return {QMM_EINVAL, "slots without a state"};
    if (!on(t->state, 16) || !on(t->gamma, 16)) return {QMM_EALIGN, "state and gamma must be 16-B aligned"};
    if (b->n_rows > 0) {
        const size_t kw = size_t(t->qk_heads) * size_t(t->key_dim), vw = size_t(t->v_heads) * size_t(t->value_dim);
        if (!t->q || !t->k || !t->v || !t->a || !t->b || !t->out) return {QMM_EINVAL, "null row tensor"};
        if (t->q_stride < kw || t->k_stride < kw || t->v_stride < vw || t->out_stride < vw || (t->z && t->z_stride < vw))
            return {QMM_EINVAL, "row stride below heads * dim"};
        if (t->a_stride < size_t(t->v_heads) || t->b_stride < size_t(t->v_heads)) return {QMM_EINVAL, "row stride below v_heads"};
        if (!on(t->q, 16) || !on(t->k, 16) || !on(t->v, 16) || !on(t->z, 16) || !on(t->out, 16) || t->q_stride % 4 ||
            t->k_stride % 4 || t->v_stride % 4 || (t->z && t->z_stride % 4) || t->out_stride % 4)
            return {QMM_EALIGN, "rows must be 16-B aligned"};
        if (!on(t->a, 4) || !on(t->b, 4)) return {QMM_EALIGN, "a and b must be 4-B aligned"};
    }
    return kFine;
}

inline Refusal check_beam(const qmm_beam_args *t) {
    if (!t) return {QMM_EINVAL, "null beam arguments"};
    if (t->vocab <= 0 || t->vocab >= (1 << 30)) return {QMM_EINVAL, "vocab must be 1..2^30 - 1"};
    if (t->n_items < 0 || t->n_beams < 1 || t->n_beams > kMaxBeams) return {QMM_EINVAL, "n_beams must be 1..64, n_items not negative"};
    if (int64_t(t->n_items) * t->n_beams >= (int64_t(1) << 20)) return {QMM_ESHAPE, "n_items * n_beams must stay below 2^20"};
    if (int64_t(t->n_items) * t->n_beams * beam_slices(t->vocab) >= (int64_t(1) << 26))
        return {QMM_ESHAPE, "n_items * n_beams * vocab / 2048 must stay below 2^26"};
    if (t->n_keep < 1 || t->n_keep > kMaxKeep || t->n_keep > int64_t(t->n_beams) * t->vocab)
        return {QMM_EINVAL, "n_keep must be 1..64, at most n_beams * vocab"};
    if (t->stride < size_t(t->vocab)) return {QMM_EINVAL, "row stride below vocab"};
    if (t->ended && (t->end_token < 0 || t->end_token >= t->vocab)) return {QMM_EINVAL, "end_token past the vocabulary"};
    if (t->n_items > 0 && (!t->logits || !t->token || !t->parent || !t->score_out)) return {QMM_EINVAL, "null logits or outputs"};
    if (!on(t->logits, 4) || !on(t->score, 4) || !on(t->ended, 4) || !on(t->token, 4) || !on(t->parent, 4) || !on(t->score_out, 4))
        return {QMM_EALIGN, "beam arrays must be 4-B aligned"};
    return kFine;
}

inline Refusal check_copy(const qmm_slot_pool *pools, int n_pools, const int32_t *src, const int32_t *dst, int n) {
    if (n_pools < 0 || n < 0) return {QMM_EINVAL, "negative number of pools or pairs"};
    if (n_pools > 0 && !pools) return {QMM_EINVAL, "null pools"};
    if (n > 0 && (!src || !dst)) return {QMM_EINVAL, "null slot array"};
    if (!on(src, 4) || !on(dst, 4)) return {QMM_EALIGN, "slot arrays must be 4-B aligned"};
    for (int i = 0; i < n_pools; ++i) {
        if (pools[i].n_slots < 0) return {QMM_EINVAL, "negative number of slots"};
        if (pools[i].n_slots > 0 && !pools[i].base) return {QMM_EINVAL, "null pool"};
        if (pools[i].slot_bytes > (size_t(1) << 40)) return {QMM_ESHAPE, "slot_bytes past 2^40"};
        if (!on(pools[i].base, 16) || pools[i].slot_bytes % 16) return {QMM_EALIGN, "pools and slots must be 16-B aligned"};
    }
    return kFine;
}

}  // namespace qmm
