// qmm_state.h — what the kernels of layers with a carried state share: the batch
// as kernels see it, and the launchers' interface to the C ABI. What finds a
// sequence's rows and slots is plain C++: a host program can check it without a
// device.
#pragma once

#include <cstddef>
#include <cstdint>

#include "qmm_attn.h"

namespace qmm {

struct StateView {
    const int32_t *row_start, *slot_in, *slot_out;  // slot arrays may be nullptr
    int n_seqs, n_rows, n_slots;
};

// A sequence's rows, clamped to the tensors, and its slots: -1 where there is none.
struct StateSeq {
    int r0, n, in, out;
};
QMM_HD inline StateSeq state_seq(const StateView &b, int s) {
    StateSeq v;
    v.r0 = clamped(b.row_start[s], 0, b.n_rows);
    v.n = clamped(b.row_start[s + 1], v.r0, b.n_rows) - v.r0;
    const int in = b.slot_in ? b.slot_in[s] : -1, out = b.slot_out ? b.slot_out[s] : -1;
    v.in = unsigned(in) < unsigned(b.n_slots) ? in : -1;
    v.out = unsigned(out) < unsigned(b.n_slots) ? out : -1;
    return v;
}

constexpr int kConvRows = 8;  // rows of one workgroup of the convolution

// The convolution's workgroups a sequence and 1024 channels: one per 8 rows as far as the host knows
// (they take turns where there are more), below 2^24 in all.
inline int conv_tiles(const StateView &b, int channels, int max_new) {
    const int64_t lists = int64_t(b.n_seqs) * ((channels + 1023) / 1024);
    const int64_t want = (int64_t(max_new > 0 ? max_new : b.n_rows) + kConvRows - 1) / kConvRows;
    const int64_t most = lists > 0 ? ((int64_t(1) << 24) - 1) / lists : 1;
    const int64_t n = want < most ? want : most;
    return n < 1 ? 1 : int(n);
}

struct ConvArgs {
    StateView b;
    const float *x, *weight, *bias;
    size_t x_stride, out_stride;
    int channels, width, silu, max_new;
    float *state, *out;
};

struct DeltaArgs {
    StateView b;
    const float *q, *k, *v, *a, *beta, *rate, *dt_bias, *z, *gamma;
    size_t q_stride, k_stride, v_stride, a_stride, b_stride, z_stride, out_stride;
    int qk_heads, v_heads, key_dim, value_dim, max_new;
    float scale, qk_eps, gamma_eps;
    float *state, *out;
};

// Prompts go through the delta rule in groups of 32 tokens. Group i of sequence s has number
// row_start[s] / 32 + s + i: different for all groups of ascending sequences, and below
// n_rows / 32 + n_seqs for any starts. Of every group the workspace holds, per value head, two 32 x 32
// matrices as pairs of fp16 in operand order (8 KB) and 96 factors; per key head 64 inverse lengths.
constexpr int kChunk = 32;
constexpr int64_t delta_groups(int n_rows, int n_seqs) { return int64_t(n_rows) / kChunk + n_seqs; }
constexpr size_t kDeltaMatrices = 8192;
constexpr int kFactors = 96;
inline size_t delta_group_bytes(const DeltaArgs &a) {
    return size_t(delta_groups(a.b.n_rows, a.b.n_seqs)) * (size_t(a.v_heads) * (kDeltaMatrices + kFactors * 4) + size_t(a.qk_heads) * 256) + 256;
}
// Where few heads (of all sequences together at most kHalfLists) walk long sequences in halves, it also holds three
// matrices of each and a row of key_dim values for every token and head of a second half. A workspace serves calls of
// fewer rows and sequences, too: it has that place (of 32768 rows and 32 heads of 128 as much again as the groups) if
// one sequence of all rows would use it, and without it the groups are walked in one.
constexpr int64_t kHalfLists = 64;
constexpr int kHalfGroups = 16;  // groups of a sequence from which on halves are faster (32 heads, 512 tokens: 47 us either way)
inline size_t delta_scratch_bytes(const DeltaArgs &a) {
    const size_t groups = delta_group_bytes(a);
    if (a.v_heads > kHalfLists || a.b.n_rows <= (kHalfGroups - 1) * kChunk) return groups;
    const int64_t lists = int64_t(a.b.n_seqs) * a.v_heads;
    return groups + size_t(lists < kHalfLists ? lists : kHalfLists) * size_t(a.key_dim) * size_t(2 * a.value_dim + a.key_dim) * 4 +
           size_t(a.b.n_rows / 2) * size_t(a.v_heads) * size_t(a.key_dim) * 4;
}

// The selection's lists: every wave of the first kernel reads 2048 logits of one
// beam and leaves its best n_keep and what the sum of exponentials needs.
constexpr int kBeamSlice = 2048;
struct BeamArgs {
    const float *logits, *score;
    const int32_t *ended;
    size_t stride;
    int vocab, n_items, n_beams, n_keep, end_token;
    int32_t *token, *parent;
    float *score_out;
    uint64_t *list;  // [rows][slices][n_keep]
    float *stat;     // [rows][slices][2]: maximum, sum of exp(x - maximum)
};
constexpr int beam_slices(int vocab) { return (vocab + kBeamSlice - 1) / kBeamSlice; }
inline size_t beam_list_bytes(int64_t rows, int vocab, int n_keep) {
    return (size_t(rows) * size_t(beam_slices(vocab)) * size_t(n_keep) * 8 + 255) & ~size_t(255);
}
inline size_t beam_scratch_bytes(int64_t rows, int vocab, int n_keep) {
    return beam_list_bytes(rows, vocab, n_keep) + size_t(rows) * size_t(beam_slices(vocab)) * 8 + 256;
}

struct CopyArgs {
    struct {
        char *base;
        size_t bytes;
        int slots;
    } pool[64];
    const int32_t *src, *dst;
    int n;
};

}  // namespace qmm

#ifdef __HIPCC__
namespace qmm {
hipError_t launch_conv(const ConvArgs &a, hipStream_t s);
hipError_t launch_delta(const DeltaArgs &a, void *scratch, size_t scratch_bytes, int cu_count, hipStream_t s);
hipError_t launch_beam(const BeamArgs &a, hipStream_t s);
// n_pools <= 64, their largest slot
hipError_t launch_copy(const CopyArgs &a, int n_pools, size_t most_bytes, hipStream_t s);
}  // namespace qmm
#endif
