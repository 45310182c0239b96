// qmm_attn.h — what the cache append and the attention kernels share: the
// batch as kernels see it, the tiles of tokens a row block attends to, and the
// launchers' interface to the C ABI. What finds a row's tokens and their pages
// is plain C++: a host program can check it without a device.
#pragma once

#include <cstddef>
#include <cstdint>

#ifdef __HIPCC__
#include <hip/hip_runtime.h>
#endif

namespace qmm {

constexpr int kTileKeys = 64;  // tokens of one attention tile

// The visible part of a sequence for rows at positions pmin..pmax (pmax < len)
// as tiles of 64 tokens: `sink` tiles from token 0 on (the first tokens a window
// keeps), then those from tile `lo` to the one that holds pmax; n in all. Tile i
// of the list is i below `sink`, else lo + i - sink.
struct TileSpan {
    int sink, lo, n;
    constexpr int at(int i) const { return i < sink ? i : lo + i - sink; }
};
constexpr TileSpan tile_span(int pmin, int pmax, int window, int sinks) {
    if (pmax < 0) return TileSpan{0, 0, 0};
    const int hi = pmax / kTileKeys + 1;
    if (window <= 0 || pmin < window) return TileSpan{0, 0, hi};
    const int lo = (pmin - window + 1) / kTileKeys;
    const int s = sinks > 0 ? (sinks - 1) / kTileKeys + 1 : 0;
    const int sink = s < lo ? s : lo;
    return TileSpan{sink, lo, sink + hi - lo};
}
#ifdef __HIPCC__
#define QMM_HD __host__ __device__
#else
#define QMM_HD
#endif

struct KvView {
    const int32_t *row_start, *kv_len, *pages;
    int n_seqs, n_rows, max_pages, n_pages, page_shift, n_heads;
};

// tokens a page table's row can hold (positions stay clear of the largest int)
constexpr int kv_capacity(int max_pages, int page_shift) {
    const int64_t n = int64_t(max_pages) << page_shift;
    return n > 0x7fffff00 ? 0x7fffff00 : int(n);
}

constexpr int clamped(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }

// A sequence's rows and length, clamped to what the tensors hold. The first
// new token's place is pos0 (negative where kv_len is less than the new rows).
struct SeqView {
    int r0, n_new, len, pos0;
};
QMM_HD inline SeqView seq_view(const KvView &b, int s) {
    SeqView v;
    v.r0 = clamped(b.row_start[s], 0, b.n_rows);
    v.n_new = clamped(b.row_start[s + 1], v.r0, b.n_rows) - v.r0;
    v.len = clamped(b.kv_len[s], 0, kv_capacity(b.max_pages, b.page_shift));
    v.pos0 = v.len - v.n_new;
    return v;
}
// page id that holds `token` of sequence s, or -1 (past its end, or no page)
QMM_HD inline int page_of(const KvView &b, int s, int token, int len) {
    if (token < 0 || token >= len) return -1;
    const int id = b.pages[size_t(s) * size_t(b.max_pages) + size_t(token >> b.page_shift)];
    return unsigned(id) < unsigned(b.n_pages) ? id : -1;
}

// The aligned groups of 16 slots that hold a sequence's new tokens: first .. end - 1. By their own
// number, not their first slot: groups past the end are looked at too, and 16 times those can be past
// the largest int.
struct SlotGroups {
    int first, end;
};
QMM_HD constexpr SlotGroups slot_groups(const SeqView &v) {  // (rows at negative places have no cell)
    return SlotGroups{(v.pos0 < 0 ? 0 : v.pos0) >> 4, v.n_new > 0 ? (v.len + 15) >> 4 : 0};
}

struct AttnArgs {
    KvView b;
    const uint16_t *q;
    size_t q_stride;
    void *out;
    size_t out_stride;
    int out_f32;
    int head_dim, group;  // query heads per key-value head; n_rows * group < 2^30
    unsigned group_inv;   // ceil(2^32 / group)
    float scale;
    int window, sinks;
    const void *kc, *vc;
    const float *ks, *vs;
    int max_new, max_kv;  // the host's hints, > 0
};

}  // namespace qmm

#ifdef __HIPCC__
namespace qmm {

// A rotation: each pair's turns (not radians) per position, and its position axis.
struct RopeTable {
    double turns[128];
    int32_t axis[128];
};
// writes it to device memory (by a kernel: nothing is copied from the host's stack later)
hipError_t launch_rope_table(const RopeTable &t, RopeTable *dst, hipStream_t s);

struct AppendArgs {
    KvView b;
    const float *q, *k, *v;
    size_t q_stride, k_stride, v_stride;
    int q_heads, head_dim;
    const float *q_gamma, *k_gamma;
    float eps;
    const RopeTable *rope;  // device; nullptr: no rotation
    int rot_dim, style;
    float rope_scale;
    const int32_t *pos;
    size_t pos_stride;
    uint16_t *q_out;
    size_t q_out_stride;
    void *kc, *vc;
    float *ks, *vs;  // 8-bit cache: scales (else nullptr)
    int max_new;
};
hipError_t launch_kv_append(const AppendArgs &a, hipStream_t s);

hipError_t launch_attention(const AttnArgs &a, void *scratch, size_t scratch_bytes, int cu_count, hipStream_t s);

}  // namespace qmm
#endif
