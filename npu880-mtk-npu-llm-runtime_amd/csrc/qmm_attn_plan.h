// qmm_attn_plan.h — how an append and a call of the attention are launched: the
// append's workgroups; row tiles, who shares which work, and the scratch that
// takes. Plain C++: a host program can check it without a device.
#pragma once

#include <algorithm>

#include "qmm_attn.h"

namespace qmm {

// Workgroups of an append: njobs for each row of queries and keys, and for each sequence ngroups (in
// turn) for its groups of 16 slots of values, times nchunks of 1024 values. workgroups 0: more than one
// launch has (2^32 threads in 256s).
struct AppendGrid {
    int njobs, ngroups, nchunks;
    unsigned workgroups;
};
inline AppendGrid append_grid(int n_rows, int n_seqs, int n_heads, int head_dim, int q_heads, int max_new) {
    constexpr int64_t kMost = (int64_t(1) << 24) - 1;
    const int hpw = 256 / head_dim, groups = (q_heads + n_heads + hpw - 1) / hpw;  // head groups of a row, one a wave
    AppendGrid g{1, 0, int((int64_t(n_heads) * head_dim + 1023) / 1024), 0};
    const int64_t values = int64_t(n_seqs) * g.nchunks;
    if (n_rows + values > kMost) return g;
    // few rows: every head group its own wave; many: one workgroup a row, the angles reduced once
    while (g.njobs * 4 < groups && int64_t(n_rows) * g.njobs < 1024 && int64_t(n_rows) * (g.njobs + 1) + values <= kMost) ++g.njobs;
    // aligned groups that max_new tokens can touch, or as many as there is room for
    g.ngroups = int(std::min<int64_t>((int64_t(max_new) + 14) / 16 + 1, (kMost - int64_t(n_rows) * g.njobs) / values));
    g.workgroups = unsigned(int64_t(n_rows) * g.njobs + values * g.ngroups);
    return g;
}

constexpr int kMaxShared = 512;  // sequences of a call whose tiles workers share
// A segment (a row tile of a sequence's head) whose tiles several workers of the
// split kernel share, as the worker that has its first tile leaves it for the join.
struct SharedSegment {
    int pieces;  // its own and those of the next workers; below 2: nothing to join
    int seq, head, row0, rows, pad[3];
};

// Units (tiles of row tiles) of one head, summed over sequences: at the top instead of past it, and
// those of all heads: 0, nothing to share, from 2^31 on. Row starts that fall let every sequence claim
// all rows, so the count can pass what the host allowed for.
constexpr int64_t kMostUnits = int64_t(1) << 31;
QMM_HD constexpr uint32_t capped_sum(uint32_t x, uint32_t y) { return x + y < x ? ~0u : x + y; }
QMM_HD constexpr int call_units(uint32_t of_head, int heads) {
    return uint64_t(of_head) * unsigned(heads) < uint64_t(kMostUnits) ? int(of_head * unsigned(heads)) : 0;
}

// How sequences of a call are launched.
struct SplitPlan {
    int rows;      // of a row tile: 16 or 128
    int workers;   // that share all tiles (0: a workgroup for each head, or with 128 rows each row tile)
    int nw;        // waves, with 16 rows
    bool lines;    // loads of whole cache lines, with 16 rows
    int row_tiles;
    int new_min, new_max;
    size_t slots, bytes;  // partial rows; all of the scratch
};

inline int few_tokens(const AttnArgs &a) { return a.group > 16 ? 1 : 16 / a.group; }

// tiles of a row tile of R rows, as the host knows it
inline int64_t hinted_tiles(const AttnArgs &a, int R) {
    const int64_t tiles = (a.max_kv - 1) / kTileKeys + 1;
    if (a.window <= 0) return tiles;
    const int64_t most = (int64_t(a.window) + R / a.group + 1) / kTileKeys + (int64_t(a.sinks) + kTileKeys - 1) / kTileKeys + 3;
    return most < tiles ? most : tiles;
}

// Tiles up to which a head of a sequence is one workgroup's. A workgroup takes 5 us and 0.62 us
// a tile; shared work 11.5 us and 4.5 us for 1000 tiles of all heads, its join included. us,
// whole / shared (8 heads of 128): 8 heads of 11 tiles 11.1 / 13.9, of 16 14.2 / 11.1; 32 of 16
// 15.9 / 13.0; 64 of 16 16.1 / 16.0, of 28 23.4 / 18.4; 128 of 16 17.0 / 22.0; 256 of 32 44 / 53.
// Heads of 64, and 8-bit ones of 128: 8 of 16 11.2 / 10.2, 13.0 / 11.2; 64 of 22 15.4 / 16.5,
// 18.3 / 19.6; 256 of 30 24.4 / 29.8, 29.0 / 34.5. Heads of 256 have 4 waves, not 8, and 1.6 to
// 2 us a tile: 8 of 9 17.7 / 19.5, of 12 21.5 / 16.2; 64 of 20 36.9 / 25.6; 128 of 9 20.7 / 27.6,
// of 18 38.4 / 35.4; 256 of 20 58.9 / 64.6; 8-bit 64 of 12 25.6 / 19.4, 256 of 20 45.5 / 42.5.
inline int64_t short_tiles(int64_t heads, int head_dim) {
    return std::min<int64_t>(32, head_dim <= 128 ? 10 + heads / 6 : 10 + heads * heads / 6000);
}

// Whether row tiles of 128 are shared: `whole` of them, `tiles` tiles long, of `rows` rows in use. Whole,
// they take us_tile for each tile of the longest; shared, what they leave idle of the chip is used (two
// 8-bit ones on a CU, bound by their conversions, cost each other less), but 8 us and those of the
// partial results are added. us, whole / shared (8 heads of 128, group 4), new tokens x tiles:
//   fp16    1 x 512 rows: of 8 18.8 / 36.3, of 24 43.1 / 49.9, of 47 78.7 / 64.4; 1 x 1024 of 16 31.8 / 53.4,
//           of 79 124 / 136; 1 x 128 of 13 26.2 / 28.0, of 18 33.6 / 28.6; 4 x 256 of 36 61.8 / 86.5
//   drafts  8 rows: 1 of 12 21.9 / 16.7; 16 of 19 32.3 / 32.0, of 63 94.6 / 66.7; 24 of 24 43.1 / 54.0
//   8-bit   1 x 512 of 8 25.1 / 39.3, of 24 62.2 / 54.6; 1 x 1024 of 16 44.8 / 58.2, of 79 189 / 161; drafts
//           24 of 24 61.4 / 54.7, 32 of 125 296 / 223; 1 x 2048 of 32 86.1 / 115
//   of 64   1 x 512 of 24 32.5 / 39.5, of 47 60.2 / 47.8; drafts 16 of 19 25.7 / 23.2, of 63 75.4 / 45.6
//   of 256  1 x 512 of 8 34.6 / 55.4, of 24 81.2 / 79.1; drafts 16 of 11 45.8 / 42.5, 32 of 125 392 / 451;
//           8-bit 1 x 512 of 8 42.4 / 57.9, of 24 106 / 90.1, 1 x 1024 of 79 323 / 369
inline bool shares_row_tiles(const AttnArgs &a, int64_t tiles, int64_t whole, int64_t rows, int cu_count) {
    constexpr double kTile[] = {1.2, 1.6, 3.0}, kPartial[] = {7, 12, 24};
    const bool q8 = a.ks != nullptr;
    const int kind = a.head_dim == 64 ? 0 : a.head_dim == 128 ? 1 : 2;
    const double us_tile = kTile[kind] * (q8 ? 1.5 : 1.0), us_partial = kPartial[kind];
    const double idle = 1.0 - (q8 && kind < 2 ? 0.65 : 1.0) * double(whole) / cu_count;
    return us_tile * double(tiles) * idle > 8.0 + us_partial * double(rows) / 128;
}

// Bytes of cache (as the hints have it: the longest sequence times all) from which loads take whole
// lines and leave them in no cache: what is less
// may be there from one call to the next (the last one holds 256 MB). us, as operands have
// them / whole lines: 57 MB 21.7 / 23.0, 86 MB 25.8 / 28.6, 115 MB 33.3 / 31.9, 230 MB
// 56.0 / 49.8; 0.4 MB 8.0 / 8.5 (more code to fetch). 8-bit, and heads of 64: 48 MB 18.9 / 20.7,
// 16.1 / 17.4, 193 MB 48.7 / 46.0, 44.8 / 40.5; heads of 256 as well either way (102 MB 33.5 / 32.7,
// 195 MB 61.8 / 62.5). Where the cache has been driven out in between, whole lines are no slower from
// 5 MB on (13 MB 8.9 / 7.9, 51 MB 17.9 / 16.8): the rule leaves up to 10 % there.
constexpr int64_t kLargeBytes = int64_t(96) << 20;

// All workers of shared work with row tiles of R rows, and what one takes of the scratch: partial
// results of two pieces, and a segment.
struct Sharing {
    int64_t workers;
    size_t each;
    size_t bytes() const { return size_t(workers) * each + sizeof(SharedSegment); }
};
inline int workgroups_of_cu(const AttnArgs &a, int R) { return R == 128 && a.head_dim > 128 ? 1 : 2; }
inline Sharing sharing(const AttnArgs &a, int R, int cu_count) {
    return Sharing{std::min(cu_count, 512) * int64_t(workgroups_of_cu(a, R)), 2 * size_t(R) * (size_t(a.head_dim) * 4 + 8) + sizeof(SharedSegment)};
}

// max_new: the most new tokens of the sequences it is for
inline SplitPlan plan_split(const AttnArgs &a, int max_new, int cu_count, size_t scratch) {
    SplitPlan p{};
    const int64_t rows = int64_t(max_new) * a.group;
    const int R = p.rows = max_new <= few_tokens(a) ? 16 : 128;
    const int64_t tiles = hinted_tiles(a, R), units = int64_t(a.b.n_seqs) * a.b.n_heads, row_tiles = (rows + R - 1) / R;
    const Sharing all = sharing(a, R, cu_count);
    // Room for fewer workers than all: only where they are no fewer than the workgroups that run at
    // once without sharing.
    int64_t workers = all.workers;
    bool enough = workers > units / 4;
    if (all.bytes() > scratch) {
        workers = int64_t(scratch / all.each) - 1;
        enough = workers >= std::min(all.workers, R == 16 ? units : units * row_tiles);
    }
    // Units of the shared work, were every row tile to see all that a sequence can hold (row starts that
    // ascend; others are counted where they are read)
    const int64_t most_tiles = int64_t(a.b.n_rows) * a.group / R + a.b.n_seqs, most_span = kv_capacity(a.b.max_pages, a.b.page_shift) / kTileKeys + 1;
    const bool countable = most_tiles * most_span < kMostUnits / a.b.n_heads;
    const int64_t whole = a.b.n_heads * std::min(a.b.n_seqs * row_tiles, int64_t(a.b.n_rows) * a.group / R + a.b.n_seqs);
    const bool few_tiles = R == 16 ? tiles <= short_tiles(units, a.head_dim) : !shares_row_tiles(a, tiles, whole, std::min<int64_t>(rows, R), cu_count);
    p.new_max = 0x7fffffff;
    if (!few_tiles && a.b.n_seqs <= kMaxShared && enough && countable) {
        p.workers = int(workers);
        p.slots = size_t(workers) * 2 * R;
        p.bytes = Sharing{workers, all.each}.bytes();
    }
    // 8 waves: one workgroup a CU (registers), so for no more heads than CUs. us, 4 / 8 waves: 8 heads of 4
    // tiles 6.9 / 7.2, of 5 8.2 / 7.9, of 10 10.8 / 10.6; 256 of 10 17.2 / 16.4; 512 of 8 24.7 / 28.2; heads of 64,
    // and 8-bit ones: 256 of 10 11.0 / 10.4, 14.3 / 13.2; 512 of 8 14.0 / 17.2, 17.0 / 20.7
    p.nw = R == 16 && !p.workers && a.head_dim <= 128 && units <= cu_count && tiles > 4 ? 8 : 4;
    p.lines = R == 16 && tiles * units >= kLargeBytes / (int64_t(kTileKeys) * a.head_dim * (a.ks ? 2 : 4));
    p.row_tiles = int(std::min<int64_t>(row_tiles, 65535));
    return p;
}

// one or two plans; the number of them
inline int plan_call(const AttnArgs &a, int cu_count, size_t scratch, SplitPlan out[2]) {
    const int few = few_tokens(a);
    out[0] = plan_split(a, a.max_new, cu_count, scratch);
    // one row tile at most; one sequence, or all of the same many rows: nothing is left for another kernel
    if (int64_t(a.max_new) * a.group <= 128 || a.b.n_seqs == 1 || int64_t(a.b.n_seqs) * a.max_new <= a.b.n_rows) return 1;
    out[0].new_min = few + 1;
    out[1] = plan_split(a, few, cu_count, scratch - out[0].bytes);
    out[1].new_max = few;
    return 2;
}

// Scratch with which no call is short of workers: this one, or any other over as many heads of this
// size with no more new tokens of a sequence. (How many workers share does not depend on the lengths.)
inline size_t attn_scratch_bytes(const AttnArgs &a, int cu_count) {
    size_t n = sharing(a, 16, cu_count).bytes();
    if (a.max_new > few_tokens(a)) n += sharing(a, 128, cu_count).bytes();  // (both, where a call has sequences of both kinds)
    return n;
}

}  // namespace qmm
