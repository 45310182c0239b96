// qmm_attn.hip — attention of new tokens over a paged key-value cache.
//
// A key-value head's query heads times a sequence's new tokens are the rows of
//   S^T [tokens x rows] = K Q^T,   O^T [values x rows] = V^T P^T
// on fp16 MFMA, 64 tokens a tile, with the running maximum m and sum l of the
// softmax in base 2 (exp2(s scale log2 e - m)), fp32. The weights P are rounded
// to fp16 for the second product, 2^15 times as large (half a step, 2^-11, of each
// down to 2^-29 of the largest, 2^-40 of it below; their sum l is of the unrounded
// ones), outputs once more. Which token a row of an MFMA operand stands for is
// free, so it is chosen that P stays in the lane that computed it.
//
// Two kernels, by the rows of a sequence's head:
//  - up to 16 rows (single tokens; a few drafts): memory-bound, every cache byte
//    is used once, so keys and values go from memory straight to the operands of
//    a wave that has all the rows and 64 tokens of its own (split_piece). 5.5 TB/s
//    for 32 sequences of 210 to 8000 tokens (537 MB in 97 us), 6.0 for one of
//    131071, with 8 heads of 128; a plain read reaches 6.0, and 6.9 when it
//    keeps nothing in the caches.
//  - more rows (prompts, drafts): 128 of them a workgroup that shares the tile
//    through LDS (tile_piece). Bound by the matrix cores and the exponentials
//    beside them: 830 to 870 TFLOP/s for a causal prompt of 8192 (32 heads of 128 on 8;
//    the library's own fp16 product of 16384 reaches 1330).
// 8-bit caches: codes become fp16 exactly, a key's scale multiplies its scores,
// a value's scale its weights.
//
// Who takes which tiles: even shares of all tiles for the workers (2 a CU), and
// partial results joined by a second kernel; or, where that costs more than it
// evens out, a workgroup for each head of a sequence or row tile (plan_split).
// The order of all sums is fixed by the lengths, the hints, the workspace's size and the CUs: the same
// call, the same bits.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "qmm_attn_plan.h"
#include "qmm_device.h"

namespace qmm {
namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef unsigned short us2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

struct SplitArgs {
    AttnArgs a;
    float sl2;             // scale log2(e)
    int new_min, new_max;  // only sequences of this many new tokens
    float *part_o;         // partial results, and (m, l) of the same rows
    float2 *part_ml;
    // [worker][2][row tile][D]: a piece that goes on from the worker before, one that the next goes on with
    int workers;  // 0: a workgroup takes a head of a sequence whole, nothing is partial
    SharedSegment *shared;  // [workers + 1], the last one's pieces: the workers there were
};

// The largest of three (a NaN counts for nothing), as one instruction. Not as inline assembly: the
// compiler puts no wait between an MFMA and assembly that reads its result.
__device__ inline float max3(float a, float b, float c) {
    return __builtin_elementwise_maximumnum(__builtin_elementwise_maximumnum(a, b), c);
}
// maximum / sum over the four lane groups (lanes l, l ^ 16, l ^ 32, l ^ 48)
__device__ inline float groups_max(float v) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ inline float groups_sum(float v) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// 8 signed codes -> fp16, exactly: a code + 128 in the mantissa of 1024, less 1152
__device__ inline h8 codes8(uint32_t w0, uint32_t w1) {
    const h2 off = {_Float16(1152.0f), _Float16(1152.0f)};
    h8 r;
    const uint32_t x[2] = {w0 ^ 0x80808080u, w1 ^ 0x80808080u};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const h2 a = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, x[i], 0x04010400u)) - off;
        const h2 b = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, x[i], 0x04030402u)) - off;
        r[4 * i] = a[0], r[4 * i + 1] = a[1], r[4 * i + 2] = b[0], r[4 * i + 3] = b[1];
    }
    return r;
}

// Bit j < N: token key0 + j is visible to the row at position p, i.e. key <= p and
// (key > low or key < sinks). Whole masks from the three bounds, no test per token.
template <int N> __device__ inline uint32_t seen_bits(int key0, int p, int low, int sinks) {
    auto below = [&](int bound) { return (1u << min(max(bound - key0, 0), N)) - 1u; };  // tokens before `bound`
    return below(p + 1) & (~below(low + 1) | below(sinks));
}

// all ones where bit j of `bits` is set, else 0
__device__ inline uint32_t whole(uint32_t bits, int j) { return uint32_t(int32_t(bits << (31 - j)) >> 31); }
// x where bit j of `bits` is set, else -infinity
__device__ inline float seen_or_none(uint32_t bits, int j, float x) {
    const uint32_t w = whole(bits, j);
    return __uint_as_float((__float_as_uint(x) & w) | (0xff800000u & ~w));
}
// |x|, 0 where it is no number
__device__ inline float magnitude_or_0(float x) { return fabsf(x) < __builtin_inff() ? fabsf(x) : 0.0f; }

// An 8-bit cache's weights are p 2^-k times the value's scale, in fp16: k (kept as a float)
// puts the largest scale the row has seen between 2^14 and 2^15, and 2^-k is part of the
// running maximum, so it costs no operation and the row's sum has it too. From -16 (scales
// below 1/2 lose the room they do not need: outputs are fp16) to 106 (no finite scale
// overflows), so that a change of k never takes a sum below fp32's range.
// The exponent is taken from the bits: 0, where a row sees no scale, has the least of all.
constexpr float kLeastShift = -16.0f;
// An fp16 cache's weights are p 2^15: all of an fp16's bits down to 2^-29 of the row's largest (the tail
// of a long context behind one strong key is made of many such weights).
constexpr float kWeightShift = -15.0f;
constexpr float kNoScore = -3.402823466e38f;  // the maximum of no score: finite, so that a row of none has weights of 0 without a test
__device__ inline float scale_shift(float largest) {  // (no number below 0)
    return fminf(fmaxf(float(int(__float_as_uint(largest) >> 23) - (126 + 15)), kLeastShift), 106.0f);
}
// What a row's exponents are taken relative to: its maximum and the shift, or above by up to two units
// in the maximum's last place, never below. Both were rounded, so a score of 2^24 and more (a float's
// digits end above the point there) could else make a weight twice what fp16 has room for.
__device__ inline float raised(float m, float shift) { return m + __builtin_fmaf(fabsf(m), 0x1p-23f, shift); }
// 8 halves of ones where the token's bit is set, else of zeros
__device__ inline u4 halves_of(uint32_t bits) {
    u4 r;
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = ((bits >> 2 * j & 1u) ? 0xffffu : 0u) | ((bits >> (2 * j + 1) & 1u) ? 0xffff0000u : 0u);
    return r;
}

// A value that is no number, made a count: +inf 1, -inf 128, NaN 16384 (64
// tokens' counts stay apart in a sum); finite values 0.
__device__ inline uint32_t nonfinite_code(uint32_t h) {
    if ((h & 0x7c00u) != 0x7c00u) return 0u;
    return (h & 0x3ffu) ? 0x7400u : (h & 0x8000u) ? 0x5800u : 0x3c00u;  // fp16 16384, 128, 1
}
// 8 values -> their counts; they are 0 afterwards where they were no numbers
__device__ inline u4 take_nonfinite(u4 &w) {
    u4 code;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t lo = nonfinite_code(w[j] & 0xffffu), hi = nonfinite_code(w[j] >> 16);
        code[j] = lo | hi << 16;
        w[j] &= (lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u);
    }
    return code;
}
// the largest magnitudes of 8 values and `top`'s two, as integers: 0x7c00 and above are no numbers
__device__ inline us2 magnitudes(us2 top, u4 w) {
#pragma unroll
    for (int j = 0; j < 4; ++j) top = __builtin_elementwise_max(top, __builtin_bit_cast(us2, w[j] & 0x7fff7fffu));
    return top;
}
__device__ inline bool no_number(us2 top) { return top[0] >= 0x7c00 || top[1] >= 0x7c00; }
// what those counts of a row's visible tokens make of its sum
__device__ inline float nonfinite_sum(float count) {
    const int n = int(count);
    float r = 0.0f;
    if (n & 127) r += __builtin_inff();
    if ((n >> 7) & 127) r -= __builtin_inff();
    if (n >> 14) r = __builtin_nanf("");
    return r;
}

// 4 values of a row, rounded to fp16
__device__ inline void put_row(const AttnArgs &a, size_t at, f4 o) {
    const h4 y = {_Float16(o[0]), _Float16(o[1]), _Float16(o[2]), _Float16(o[3])};
    if (a.out_f32) *reinterpret_cast<f4 *>(static_cast<float *>(a.out) + at) = f4{float(y[0]), float(y[1]), float(y[2]), float(y[3])};
    else *reinterpret_cast<h4 *>(static_cast<uint16_t *>(a.out) + at) = y;
}

constexpr int kJoinWaves = 8;  // of a workgroup that joins partial results

// A wave's share of a row's partial results, k = first, first + step, .. below n
// (slot(k): the k-th's place), a lane D / 64 values.
template <int D, class Slot>
__device__ inline void join_pieces(const SplitArgs &p, int first, int step, int n, Slot slot, float (&o)[D / 64], float &m, float &l) {
    constexpr int N = D / 64;
    const int lane = threadIdx.x & 63;
    m = -__builtin_inff();
    l = 0.0f;
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = 0.0f;
#pragma unroll 8
    for (int k = first; k < n; k += step) {
        const int64_t s = slot(k);
        const float2 x = p.part_ml[s];
        float y[N];
#pragma unroll
        for (int j = 0; j < N; ++j) y[j] = p.part_o[s * D + 64 * j + lane];
        const float top = fmaxf(m, x.x), base = top == -__builtin_inff() ? 0.0f : top;
        const float wa = __builtin_amdgcn_exp2f(m - base), wb = __builtin_amdgcn_exp2f(x.x - base);
        m = top;
        l = l * wa + x.y * wb;
#pragma unroll
        for (int j = 0; j < N; ++j) o[j] = o[j] * wa + y[j] * wb;
    }
}
// One row from n partial results, by a workgroup: its waves' shares in turn, in this
// order whatever ran when.
template <int D, class Slot>
__device__ inline void join_row(const SplitArgs &p, int n, Slot slot, float (*part)[D], float2 *ml, size_t dst) {
    constexpr int W = kJoinWaves;
    constexpr int N = D / 64;
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
    float o[N], m, l;
    join_pieces<D>(p, wid, W, n, slot, o, m, l);
    if (lane == 0) ml[wid] = make_float2(m, l);
#pragma unroll
    for (int j = 0; j < N; ++j) part[wid][64 * j + lane] = o[j];
    __syncthreads();
    if (threadIdx.x < D) {
        float top = ml[0].x;
        for (int w = 1; w < W; ++w) top = fmaxf(top, ml[w].x);
        const float base = top == -__builtin_inff() ? 0.0f : top;
        float total = 0.0f, sum = 0.0f;
        for (int w = 0; w < W; ++w) {
            const float e = __builtin_amdgcn_exp2f(ml[w].x - base);
            total += ml[w].y * e;
            sum += part[w][threadIdx.x] * e;
        }
        const _Float16 y = _Float16(total > 0.0f || total != total ? sum / total : 0.0f);
        if (p.a.out_f32) static_cast<float *>(p.a.out)[dst + threadIdx.x] = float(y);
        else static_cast<_Float16 *>(p.a.out)[dst + threadIdx.x] = y;
    }
    __syncthreads();
}

// The split kernel's work: segments in the order of sequence, head, row tile,
// each of as many units as its span has tiles (one where it has none: its rows
// are zeros). Worker w of W takes units bound(w) .. bound(w + 1): even shares, so
// that ragged batches load every CU alike, moved to a head's border where one is
// near (a segment in one piece needs no join). The host sees to it that all units
// are below 2^31.
struct Work {
    const int *upto;  // [n_seqs + 1]: units of one head of the sequences before
    int n_seqs, heads, workers, total, share, more;
    __device__ void set(int n_units, int most_workers) {
        total = n_units;
        workers = most_workers;
        share = workers ? total / workers : 0;
        more = total - share * workers;
    }
    __device__ int seq_of(int unit) const {  // the sequence that holds it
        int lo = 0, hi = n_seqs - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (upto[mid] * heads <= unit) lo = mid;
            else hi = mid - 1;
        }
        return lo;
    }
    __device__ int bound(int w) const {
        if (w >= workers) return total;
        const int even = share * w + more * w / workers;  // (more < workers <= 2^10)
        const int s = seq_of(even);
        const int n = upto[s + 1] - upto[s], first = upto[s] * heads;
        const int border = first + (even - first + n / 2) / n * n;
        return abs(border - even) <= share / 8 ? border : even;
    }
};

// row / group, where inv = ceil(2^32 / group): the product's quotient is that or one more
__device__ inline int token_of(const AttnArgs &a, int row) {
    const int q = a.group == 1 ? row : int(__umulhi(unsigned(row), a.group_inv));
    return q - int(q * a.group > row);
}

// a sequence's row tile: rows row0 .. row0 + nrows - 1, their span, and its units
struct RowTile {
    int row0, nrows, pmin, pmax, units;
    TileSpan span;
};
template <int R> __device__ inline RowTile row_tile(const AttnArgs &a, const SeqView &v, int rt) {
    RowTile t;
    t.row0 = rt * R;
    t.nrows = min(v.n_new * a.group - t.row0, R);
    t.pmin = v.pos0 + token_of(a, t.row0);
    t.pmax = v.pos0 + token_of(a, t.row0 + t.nrows - 1);
    t.span = tile_span(t.pmin, t.pmax, a.window, a.sinks);
    t.units = t.span.n > 0 ? t.span.n : 1;
    return t;
}

// 16 B that no other workgroup reads
__device__ inline u4 once(const void *p) { return __builtin_nontemporal_load(static_cast<const u4 *>(p)); }
// Loads that cover whole 128-B lines, made operands: lane l has loaded row l % 8 (a) and row
// 8 + l % 8 (b), of each the piece 2 (l / 16) + (l / 8) % 2; afterwards row l % 16, pieces
// 2 (l / 16) and 2 (l / 16) + 1. (Lanes 8 apart exchange halves in the lane network.)
__device__ inline void rows_of_lines(u4 &a, u4 &b) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int x = int(a[j]), y = int(b[j]);
        a[j] = uint32_t(__builtin_amdgcn_update_dpp(x, y, 0x128, 15, 12, false));
        b[j] = uint32_t(__builtin_amdgcn_update_dpp(y, x, 0x128, 15, 3, false));
    }
}

template <int D, int NW> struct SplitShared {
    f4 joined[NW][D < 128 ? D / 16 : 8][64];  // value tiles joined at a time
    float2 ml[NW][16];
    h8 queries[D > 128 ? NW : 1][D > 128 ? D / 32 : 1][64];  // where 256 registers do not hold them too
};

// One piece of a segment: the up to 16 rows of `tile` of head h of sequence s over
// tiles begin .. end - 1 of its span, the waves' steps in turn; the rows themselves
// (direct), or their partial results at slot0.
// 16x16x32 MFMA; lane group c = lane / 16 has tokens TL c .. TL c + TL - 1 of a step:
//   S:  operand row i of MFMA t is token TL (i / 4) + 4 t + i % 4, and the lane
//       finds its scores of tokens TL c + 4t + r in register r of result t;
//   PV: operand k index 8c + j of step u is token TL c + 8u + j.
// A page holds 16 tokens or more, so a lane's tokens are in one page. A step's
// values are under way during its scores, the next step's keys during its softmax
// and second product; 8 waves of 16 to 32 KB a CU keep memory busy, and the
// products and exponentials (a tenth of the time) lie under it.
template <int D, int NW, bool Q8, bool LINES>
__device__ inline __attribute__((always_inline)) void split_piece(const SplitArgs &p, SplitShared<D, NW> &sh, const SeqView &v,
                                                                  const RowTile &tile, int s, int h, int begin, int end,
                                                                  bool direct, int slot0) {
    constexpr int KS = D / 32;           // MFMA steps of a score
    constexpr int DT = D / 16;           // value tiles
    constexpr int KR = Q8 ? D / 64 : KS;  // 16-B registers of a key operand
    constexpr int KT = D <= 128 ? 64 : 32;  // tokens of a wave's step
    constexpr int NT = KT / 16;          // score MFMAs of a step
    constexpr int TL = KT / 4;           // tokens of a lane: TL c .. TL c + TL - 1
    constexpr int NU = TL / 8;           // MFMA steps of the second product
    constexpr int SUB = kTileKeys / KT;
    // what 256 registers hold: the next step's keys beside this one's values, and the queries
    constexpr bool AHEAD = D <= 128, QLDS = D > 128;
    // A load of 16 rows of 64 B, as an operand has them, takes half a cache line of each; two of
    // 8 rows take whole lines, which non-temporal loads need: 6.9 TB/s of 6.0
    constexpr bool KLINES = LINES && KR >= 2, VLINES = LINES && !Q8 && NU == 2;
    constexpr int DG = DT < 8 ? DT : 8;  // value tiles joined at a time
    const AttnArgs &a = p.a;
    const int H = a.b.n_heads, G = a.group;
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, c = lane >> 4;
    const int P = 1 << a.b.page_shift, shift = a.b.page_shift;
    const TileSpan span = tile.span;
    const int row0 = tile.row0, nrows = tile.nrows, pmin = tile.pmin, pmax = tile.pmax;

    // this lane's row: its queries, position, the last token its window hides
    h8 q[QLDS ? 1 : KS];
    const int row = row0 + (col < nrows ? col : 0);
    const int qi = token_of(a, row), qg = row - qi * G, pos = v.pos0 + qi;
    const int low = a.window > 0 ? max(max(pos, 0) - a.window, -1) : -1;
    {
        const uint16_t *src = a.q + size_t(v.r0 + qi) * a.q_stride + size_t(h * G + qg) * D;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            // (the values that the key operand of step k holds)
            const int at = KLINES ? (Q8 ? 128 * (k / 4) + 32 * c + 8 * (k % 4) : 64 * (k / 2) + 16 * c + 8 * (k % 2))
                                  : (Q8 ? 64 * (k / 2) + 16 * c + 8 * (k % 2) : 32 * k + 8 * c);
            const h8 x = *reinterpret_cast<const h8 *>(src + at);
            if constexpr (QLDS) sh.queries[wid][k][lane] = x;
            else q[k] = x;
        }
    }
    float m = kNoScore, base = m, l = 0.0f, shift_v = kLeastShift;  // (base: m and the shift, raised)
    f4 acc[DT];

    u4 kr[NT][KR], vr[DT][Q8 ? (NU + 1) / 2 : NU];
    f4 ksc[NT], vsc[NT];
    int id_v = -1;
    bool wild_steps = false;
    // the lane groups whose tokens this lane loads keys of, and its piece of a line
    const int ck = KLINES ? (lane & 7) >> 2 : col >> 2, piece = 2 * c + (lane >> 3 & 1);
    // the wave's steps are wid, wid + NW, .. of SUB (end - begin)
    const int steps = (end - begin) * SUB;
    auto step_at = [&](int i) { return span.at(begin + i / SUB) * kTileKeys + i % SUB * KT; };
    auto is_full = [&](int t0, bool page_ok) {  // every row sees every token
        return __all(page_ok) && t0 + KT - 1 <= pmin &&
               (a.window <= 0 || t0 > pmax - a.window || t0 + KT <= a.sinks);
    };
    auto look_up = [&](int i, int2 &ik, int &iv) {
        const int t = step_at(i);
        ik.x = page_of(a.b, s, t + TL * ck, v.len);
        if constexpr (KLINES) ik.y = page_of(a.b, s, t + TL * (ck + 2), v.len);
        iv = page_of(a.b, s, t + TL * c, v.len);
    };
    auto load_k = [&](int i, int2 id) {
        constexpr int RB = Q8 ? D : 2 * D;  // bytes of a key
        auto row = [&](int id, int group) {
            const int slot = (step_at(i) + TL * group) & (P - 1);
            const size_t cell = ((size_t(max(id, 0)) * H + h) << shift) + size_t(slot + (lane & 3));
            return static_cast<const uint8_t *>(a.kc) + cell * RB;
        };
        const uint8_t *src = row(id.x, ck) + 16 * (KLINES ? piece : c);
        if constexpr (KLINES) {
            const uint8_t *next = row(id.y, ck + 2) + 16 * piece;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int k = 0; k < KR; k += 2) {
                    kr[t][k] = once(src + t * 4 * RB + k * 64);
                    kr[t][k + 1] = once(next + t * 4 * RB + k * 64);
                }
        } else {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int k = 0; k < KR; ++k) kr[t][k] = *reinterpret_cast<const u4 *>(src + t * 4 * RB + k * 64);
        }
    };
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[d] = f4{0.f, 0.f, 0.f, 0.f};
    // pages are looked up a step ahead of their loads: loads return in order
    int2 nk = make_int2(-1, -1);
    int nv = -1;
    if (wid < steps) {
        look_up(wid, nk, id_v);
        load_k(wid, nk);
    }
    if (wid + NW < steps) look_up(wid + NW, nk, nv);
    for (int i = wid; i < steps; i += NW) {
        int2 nnk = make_int2(-1, -1);
        int nnv = -1;
        if (i + 2 * NW < steps) look_up(i + 2 * NW, nnk, nnv);
        const int t0 = step_at(i), key0 = t0 + TL * c;
        auto load_v = [&] {  // this step's values (and scales)
            const size_t hv = size_t(max(id_v, 0)) * H + h;
            const int slot = key0 & (P - 1);
            const int row = VLINES ? lane & 7 : col, at = VLINES ? slot + (lane & 8) : slot;
            const uint8_t *src = static_cast<const uint8_t *>(a.vc) + ((hv * D + row) * size_t(P) + at) * (Q8 ? 1 : 2);
            const size_t next = size_t(16 * (Q8 ? 1 : 2)) << shift;
#pragma unroll
            for (int d = 0; d < DT; ++d, src += next) {
                if constexpr (VLINES) {
                    vr[d][0] = once(src);
                    vr[d][1] = once(src + next / 2);
                } else if constexpr (!Q8) {
#pragma unroll
                    for (int u = 0; u < NU; ++u) vr[d][u] = reinterpret_cast<const u4 *>(src)[u];
                } else if constexpr (NU == 2) {
                    vr[d][0] = LINES ? once(src) : *reinterpret_cast<const u4 *>(src);
                } else {
                    const uint2 w = *reinterpret_cast<const uint2 *>(src);
                    vr[d][0] = u4{w.x, w.y, 0, 0};
                }
            }
            if constexpr (Q8) {
                const size_t cell = (hv << shift) + size_t(slot);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    ksc[t] = *reinterpret_cast<const f4 *>(a.ks + cell + 4 * t);
                    vsc[t] = *reinterpret_cast<const f4 *>(a.vs + cell + 4 * t);
                }
            }
        };
        if constexpr (AHEAD) load_v();
        const bool page_ok = id_v >= 0;
        __builtin_amdgcn_sched_barrier(0);

        f4 sc[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            sc[t] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < (KLINES ? KR : 0); k += 2) rows_of_lines(kr[t][k], kr[t][k + 1]);
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                h8 kk, qq;
                if constexpr (Q8) kk = codes8(kr[t][k / 2][2 * (k % 2)], kr[t][k / 2][2 * (k % 2) + 1]);
                else kk = __builtin_bit_cast(h8, kr[t][k]);
                if constexpr (QLDS) qq = sh.queries[wid][k][lane];
                else qq = q[k];
                sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk, qq, sc[t], 0, 0, 0);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (AHEAD) {
            if (i + NW < steps) load_k(i + NW, nk);
        } else {
            load_v();
        }
        __builtin_amdgcn_sched_barrier(0);

        const bool full = is_full(t0, page_ok);
        uint32_t seen = (1u << TL) - 1u;  // bit j: token key0 + j is visible to the row
        if constexpr (Q8) {
#pragma unroll
            for (int t = 0; t < NT; ++t) sc[t] *= ksc[t];
        }
        if (!full) {
            seen = page_ok ? seen_bits<TL>(key0, pos, low, a.sinks) : 0u;
#pragma unroll
            for (int j = 0; j < TL; ++j) sc[j / 4][j % 4] = seen_or_none(seen, j, sc[j / 4][j % 4]);
        }
        float top = max3(sc[0][0], sc[0][1], sc[0][2]);
#pragma unroll
        for (int j = 3; j + 1 < TL; j += 2) top = max3(top, sc[j / 4][j % 4], sc[(j + 1) / 4][(j + 1) % 4]);
        top = fmaxf(top, sc[NT - 1][3]);
        m = fmaxf(m, groups_max(top) * p.sl2);
        if constexpr (Q8) {  // of the value scales that the row sees, the largest
            float big = 0.0f;
#pragma unroll
            for (int j = 0; j < TL; ++j) {
                float x = vsc[j / 4][j % 4];
                if (!full) x = __uint_as_float(__float_as_uint(x) & whole(seen, j));
                big = fmaxf(big, magnitude_or_0(x));
            }
            shift_v = fmaxf(shift_v, scale_shift(groups_max(big)));
        }
        const float ms = raised(m, Q8 ? shift_v : kWeightShift);
        const float alpha = __builtin_amdgcn_exp2f(base - ms);
        base = ms;
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < TL; ++j) {
            const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[j / 4][j % 4], p.sl2, -ms));
            sc[j / 4][j % 4] = e;
            sum += e;
        }
        l = l * alpha + sum;
        if (!__all(alpha == 1.0f)) {
#pragma unroll
            for (int d = 0; d < DT; ++d) acc[d] *= alpha;
        }
        if constexpr (!Q8) {
            if (!full) {
                // values that are no numbers in a step of which a row does not see all: a weight of 0
                // does not hide a NaN, so they leave the product and come back below
                us2 top = {0, 0};
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int u = 0; u < NU; ++u) top = magnitudes(top, vr[d][u]);
                if (__any(no_number(top))) {
                    wild_steps = true;
#pragma unroll
                    for (int d = 0; d < DT; ++d)
#pragma unroll
                        for (int u = 0; u < NU; ++u) (void)take_nonfinite(vr[d][u]);
                }
            }
        }
        h8 pb[NU];
#pragma unroll
        for (int j = 0; j < TL; ++j) {
            float w = sc[j / 4][j % 4];
            if constexpr (Q8) w *= vsc[j / 4][j % 4];  // the weights of the codes
            pb[j / 8][j % 8] = _Float16(w);
        }
        if constexpr (Q8) {  // (a hidden token's scale may be no number)
            if (!full) {
#pragma unroll
                for (int u = 0; u < NU; ++u) pb[u] = __builtin_bit_cast(h8, u4(__builtin_bit_cast(u4, pb[u]) & halves_of(seen >> 8 * u)));
            }
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            if constexpr (VLINES) rows_of_lines(vr[d][0], vr[d][1]);
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                h8 vv;
                if constexpr (Q8) vv = codes8(vr[d][0][2 * u], vr[d][0][2 * u + 1]);
                else vv = __builtin_bit_cast(h8, vr[d][u]);
                acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vv, pb[u], acc[d], 0, 0, 0);
            }
        }
        if constexpr (!AHEAD) {
            if (i + NW < steps) load_k(i + NW, nk);
        }
        id_v = nv;
        nk = nnk;
        nv = nnv;
    }

    if constexpr (!Q8) {
        if (wild_steps) {  // of what each row sees of those values, counts, and what they make of its sum
            for (int i = wid; i < steps; i += NW) {
                const int t0 = step_at(i), key0 = t0 + TL * c;
                look_up(i, nk, id_v);
                if (is_full(t0, id_v >= 0)) continue;
                const uint8_t *src = static_cast<const uint8_t *>(a.vc) +
                                     (((size_t(max(id_v, 0)) * H + h) * D + col) * size_t(P) + size_t(key0 & (P - 1))) * 2;
                const uint32_t bits = id_v >= 0 ? seen_bits<TL>(key0, pos, low, a.sinks) : 0u;
                h8 sb[NU];
#pragma unroll
                for (int j = 0; j < TL; ++j) sb[j / 8][j % 8] = _Float16(float(bits >> j & 1u));
#pragma unroll
                for (int d = 0; d < DT; ++d, src += size_t(32) << shift) {
                    asm volatile("" : "+v"(src));  // (one address, not all of them)
                    f4 cnt = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int u = 0; u < NU; ++u) {
                        u4 w = reinterpret_cast<const u4 *>(src)[u];
                        cnt = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, take_nonfinite(w)), sb[u], cnt, 0, 0, 0);
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[d][r] += nonfinite_sum(cnt[r]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
    }

    // the waves' results, joined in LDS
    l = groups_sum(l);
    if (c == 0) sh.ml[wid][col] = make_float2(base, l);
    __syncthreads();
    float top = -__builtin_inff(), total = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) top = fmaxf(top, sh.ml[w][col].x);
    const float ref = top == -__builtin_inff() ? 0.0f : top;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        const float2 x = sh.ml[w][col];
        total += x.y * __builtin_amdgcn_exp2f(x.x - ref);
    }
    const float mine = __builtin_amdgcn_exp2f(base - ref);
    const float inv = direct ? (total > 0.0f || total != total ? 1.0f / total : 0.0f) : 1.0f;
    const bool in = col < nrows;
    const int slot = slot0 + col;
    if (!direct && in && threadIdx.x < 16) p.part_ml[slot] = make_float2(top, total);
    const size_t dst = size_t(v.r0 + qi) * a.out_stride + size_t(h * G + qg) * D;
#pragma unroll
    for (int d0 = 0; d0 < DT; d0 += DG) {
        if (d0) __syncthreads();
#pragma unroll
        for (int d = 0; d < DG; ++d) sh.joined[wid][d][lane] = acc[d0 + d] * mine;
        __syncthreads();
#pragma unroll
        for (int d = wid; d < DG; d += NW) {
            f4 o = sh.joined[0][d][lane];
#pragma unroll
            for (int w = 1; w < NW; ++w) o += sh.joined[w][d][lane];
            if (!in) continue;
            const int at = 16 * (d0 + d) + 4 * c;
            if (direct) put_row(a, dst + size_t(at), o * inv);
            else *reinterpret_cast<f4 *>(p.part_o + size_t(slot) * D + at) = o;
        }
    }
    __syncthreads();
}
// maximum / sum over the two lane halves (lanes l, l ^ 32)
__device__ inline float halves_max(float v) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ inline float halves_sum(float v) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// Many rows: 128 of them a workgroup, 32 a wave, the columns of 32x32x16 MFMA. (64 rows
// a workgroup read each tile twice as often; 64 a wave need more than 256 registers.)
// The tile's keys and values are staged through LDS (8-bit ones as fp16) and
// shared by the four waves; the next tile's loads are in flight meanwhile. A
// lane (half hh = lane / 32) holds scores of tokens 16u + 8 hh + 0..7, u < 4:
// result row i = 8a + 4 hh + r of a 32-token MFMA is given token 16 (a / 2) +
// 8 hh + 4 (a % 2) + r (bits 2 and 3 of i exchanged in the key operand's row),
// so the weights are the second product's operand as they stand. 16-B pieces of
// an LDS row are exchanged by an XOR with the row, so that 16 rows' equal pieces
// lie in 64 different banks.
template <int D> struct TileShared {  // (the buffers first: sh_at below is its LDS address)
    __attribute__((aligned(16))) uint8_t kbuf[2][128 * D];  // 64 keys, as fp16
    __attribute__((aligned(16))) uint8_t vbuf[2][128 * D];
    float ksc[4][64], vsc[2][64], vmax[2][4];               // 8-bit cache: their scales; the largest of each 16 values'
    int wild;                                               // a tile had values that are no numbers, hidden from some row
};

// lane l's 16 B at src land at LDS byte address lds + 16 l (counted by vmcnt)
__device__ inline void dma16g(const void *src, uint32_t lds) {
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(src), "s"(lds) : "memory", "m0");
#pragma clang diagnostic pop
}

// One row tile over tiles begin .. end - 1 of its span. A step takes tile i's
// weights and second product beside tile i + 1's scores, so the matrix cores work
// while the weights' exponentials are computed; the keys of tile i + 2 and the
// values of tile i + 1 are on their way to LDS meanwhile (fp16 straight from
// memory, the XOR of an LDS row's pieces in the lanes' addresses). Against scores
// and product in turn: a prompt of 8192 727 -> 648 us. Nothing may spill in this
// loop: a spilled value's load waits for all of the loads above (8-bit: 10 to
// 25 %). Three of the forms of 128 values keep up to 8 registers in scratch, read
// between pieces.
template <int D, bool Q8>
__device__ inline __attribute__((always_inline)) void tile_piece(const SplitArgs &p, TileShared<D> &sh, uint32_t sh_at, const SeqView &v,
                                                                 const RowTile &tile, int s, int h, int begin, int end,
                                                                 bool direct, int slot0) {
    constexpr int KS = D / 16, DB = D / 32;
    constexpr int RK = D * 2;                 // bytes of a key's row in LDS
    constexpr int NL = Q8 ? D / 64 : D / 32;  // 16-B loads of a thread for its keys, and for its values
    const AttnArgs &a = p.a;
    const int H = a.b.n_heads, G = a.group;
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, hh = lane >> 5;
    const int P = 1 << a.b.page_shift, shift = a.b.page_shift;
    const int krow = (col & ~12) | ((col & 4) << 1) | ((col & 8) >> 1);  // the key this lane's operand row stands for
    auto k_at = [](int row, int ch) { return row * RK + ((ch ^ (D == 64 ? (row >> 1) & 7 : row & 15)) << 4); };
    auto v_at = [](int d, int ch) { return d * 128 + ((ch ^ ((d >> 1) & 7)) << 4); };
    const int row0 = tile.row0, nrows = tile.nrows;
    const TileSpan span = tile.span;

    const int wr = 32 * wid, wrows = min(nrows - wr, 32);  // this wave's rows of the tile (none: <= 0)
    const int row = row0 + (wrows > 0 ? wr + (col < wrows ? col : 0) : 0);
    const int qi = token_of(a, row), qg = row - qi * G, pos = v.pos0 + qi;
    const int pmin = v.pos0 + token_of(a, row0 + min(wr, nrows - 1)), pmax = v.pos0 + token_of(a, row0 + min(wr + 31, nrows - 1));
    const int low = a.window > 0 ? max(max(pos, 0) - a.window, -1) : -1;  // the last token the row's window hides
    h8 q[KS];
    {
        const uint16_t *src = a.q + size_t(v.r0 + qi) * a.q_stride + size_t(h * G + qg) * D + 8 * hh;
#pragma unroll
        for (int k = 0; k < KS; ++k) q[k] = *reinterpret_cast<const h8 *>(src + 16 * k);
    }
    float m = kNoScore, base = m, l = 0.0f, shift_v = kLeastShift;  // (base: m and the shift, raised)
    f16v acc[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] = 0.0f;

    // Staging: wave w brings the tile's keys 16w .. 16w + 15 (of one page) and D / 4 of
    // its values' rows. Lane l looks up the page of the tile's tokens 16 (l % 4) ..
    auto look_up = [&](int i) { return i < end ? page_of(a.b, s, span.at(i) * kTileKeys + 16 * (lane & 3), v.len) : -1; };
    auto k_cell = [&](int i, int g) {  // this wave's first key
        const int id = max(__builtin_amdgcn_readlane(g, wid), 0);
        return ((size_t(id) * H + h) << shift) + size_t((span.at(i) * kTileKeys + 16 * wid) & (P - 1));
    };
    u4 kr[Q8 ? NL : 1], vr[Q8 ? NL : 1];
    float sreg = 0.0f;
    auto bring_k = [&](int i, int g, int b) {
        const uint8_t *src = static_cast<const uint8_t *>(a.kc) + k_cell(i, g) * (Q8 ? D : 2 * D);
        if constexpr (Q8) {
#pragma unroll
            for (int j = 0; j < NL; ++j) kr[j] = *reinterpret_cast<const u4 *>(src + 1024 * j + 16 * lane);
        } else {
#pragma unroll
            for (int j = 0; j < NL; ++j) {
                const int r = (64 * j + lane) / (D / 8), ch = (64 * j + lane) % (D / 8);
                dma16g(src + k_at(r, ch), sh_at + uint32_t(b * 128 * D + 16 * wid * RK + 1024 * j));
            }
        }
    };
    auto bring_v = [&](int i, int g, int b) {
        const int t = span.at(i) * kTileKeys;
        if constexpr (Q8) {
            const int slot = (t + 16 * (lane & 3)) & (P - 1), d0 = wid * (D / 4) + (lane >> 2);
            const uint8_t *src = static_cast<const uint8_t *>(a.vc) + ((size_t(max(g, 0)) * H + h) * D + d0) * size_t(P) + slot;
#pragma unroll
            for (int j = 0; j < NL; ++j) vr[j] = *reinterpret_cast<const u4 *>(src + size_t(16 * j) * P);
        } else {
            // rows d = w D / 4 + 8 j + l / 8; the piece that lands at place l % 8 is that XOR (d / 2) % 8
            const int ch = (lane & 7) ^ (lane >> 4);
#pragma unroll
            for (int e = 0; e < 2; ++e) {  // (even and odd j: pieces ch and ch ^ 4)
                const int c = ch ^ (4 * e), id = max(__shfl(g, c >> 1), 0), slot = (t + 16 * (c >> 1)) & (P - 1);
                const int d0 = wid * (D / 4) + 8 * e + (lane >> 3);
                const uint8_t *src = static_cast<const uint8_t *>(a.vc) +
                                     (((size_t(id) * H + h) * D + d0) * size_t(P) + slot) * 2 + 16 * (c & 1);
#pragma unroll
                for (int j = e; j < NL; j += 2)
                    dma16g(src + size_t(8 * (j - e) * 2) * P, sh_at + uint32_t((2 + b) * 128 * D + wid * (D / 4) * 128 + 1024 * j));
            }
        }
    };
    // 8-bit: the scales of tile ik's keys and tile iv's values; then codes to LDS as fp16
    auto bring_scales = [&](int ik, int gk, int iv, int gv) {
        if (lane < 16 && ik < end) sreg = a.ks[k_cell(ik, gk) + lane];
        else if (lane >= 16 && lane < 32 && iv < end) sreg = a.vs[k_cell(iv, gv) + (lane & 15)];
    };
    auto put_k = [&](int b, int slot) {
        int ln = lane;  // (addresses made anew each time: kept, they would spill)
        asm volatile("" : "+v"(ln));
#pragma unroll
        for (int j = 0; j < (Q8 ? NL : 0); ++j) {
            const int u = 64 * j + ln, r = 16 * wid + u / (D / 16), ch = u % (D / 16) * 2;
            *reinterpret_cast<h8 *>(&sh.kbuf[b][k_at(r, ch)]) = codes8(kr[j][0], kr[j][1]);
            *reinterpret_cast<h8 *>(&sh.kbuf[b][k_at(r, ch + 1)]) = codes8(kr[j][2], kr[j][3]);
        }
        if (ln < 16) sh.ksc[slot & 3][16 * wid + ln] = sreg;
    };
    auto put_v = [&](int b) {
        int ln = lane;
        asm volatile("" : "+v"(ln));
#pragma unroll
        for (int j = 0; j < (Q8 ? NL : 0); ++j) {
            const int d = wid * (D / 4) + 16 * j + (ln >> 2), c = 2 * (ln & 3);
            *reinterpret_cast<h8 *>(&sh.vbuf[b][v_at(d, c)]) = codes8(vr[j][0], vr[j][1]);
            *reinterpret_cast<h8 *>(&sh.vbuf[b][v_at(d, c + 1)]) = codes8(vr[j][2], vr[j][3]);
        }
        float big = magnitude_or_0(sreg);
#pragma unroll
        for (int o = 1; o < 16; o *= 2) big = fmaxf(big, __shfl_xor(big, o));
        if (ln == 16) sh.vmax[b][wid] = big;
        if (ln >= 16 && ln < 32) sh.vsc[b][16 * wid + (ln & 15)] = sreg;
    };
    // Values that are no numbers in a tile of which some row of the workgroup does not see
    // all: out of the product (a weight of 0 does not hide a NaN), and back after the loop.
    // A wave looks through what it brought itself.
    auto partial = [&](int i, unsigned ok) {
        const int t = span.at(i) * kTileKeys;
        return ok != 15 || t + kTileKeys - 1 > tile.pmin ||
               (a.window > 0 && t <= tile.pmax - a.window && t + kTileKeys > a.sinks);
    };
    auto take_wild = [&](int b) {
        u4 *mine = reinterpret_cast<u4 *>(&sh.vbuf[b][wid * (D / 4) * 128 + 16 * lane]);
        us2 top = {0, 0};
#pragma unroll
        for (int j = 0; j < NL; ++j) top = magnitudes(top, mine[64 * j]);
        if (__any(no_number(top))) {
            sh.wild = 1;
#pragma unroll 1
            for (int j = 0; j < NL; ++j) {
                u4 w = mine[64 * j];
                (void)take_nonfinite(w);
                mine[64 * j] = w;
            }
        }
    };
    auto groups = [&](int g) { return unsigned(__ballot(g >= 0) & 15); };  // which 16 tokens have a page
    // Operand pieces in LDS, from one offset each (that of buffer b, with the XOR of the
    // row in it): the step's own bits are exchanged by another XOR. The offsets are made
    // anew for each tile: as constants of the loop they would fill the registers.
    auto key_base = [&](int b) {
        uint32_t at = uint32_t(b * 64 * RK + k_at(krow, hh));
        asm volatile("" : "+v"(at));
        return at;
    };
    auto value_base = [&](int b) {
        uint32_t at = uint32_t(b * 128 * D + v_at(col, hh));
        asm volatile("" : "+v"(at));
        return at;
    };
    auto key = [&](uint32_t base, int n, int k) {
        return *reinterpret_cast<const h8 *>(&sh.kbuf[0][0] + (base ^ uint32_t(k << 5)) + 32 * n * RK);
    };
    auto value = [&](uint32_t base, int d, int u) {
        return *reinterpret_cast<const u4 *>(&sh.vbuf[0][0] + (base ^ uint32_t(u << 5)) + 32 * d * 128);
    };

    // a lane's scores of a tile: token t0 + 16 u + 8 hh + j is sc[u / 2][8 (u % 2) + j]
    f16v sc[2];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) sc[n][r] = 0.0f;
    unsigned ok = 0;
    int g1 = -1, g2 = -1;  // pages of the next two tiles
    if (threadIdx.x == 0) sh.wild = 0;
    if (begin < end) {
        const int g0 = look_up(begin);
        g1 = look_up(begin + 1);
        g2 = look_up(begin + 2);
        ok = groups(g0);
        bring_k(begin, g0, 0);
        bring_v(begin, g0, 0);
        if constexpr (Q8) {
            bring_scales(begin, g0, begin, g0);
            put_k(0, 0);
            put_v(0);
        }
        if (begin + 1 < end) {
            bring_k(begin + 1, g1, 1);
            if constexpr (Q8) {
                bring_scales(begin + 1, g1, end, g1);
                put_k(1, 1);
            }
        }
        wait_vmcnt<0>();
        __syncthreads();
        const uint32_t kb = key_base(0);
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int n = 0; n < 2; ++n) sc[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(key(kb, n, k), q[k], sc[n], 0, 0, 0);
    }
    for (int i = begin; i < end; ++i) {
        const int b = (i - begin) & 1;
        wait_vmcnt<0>();
        if constexpr (!Q8) {
            if (partial(i, ok)) take_wild(b);
        }
        __syncthreads();  // tile i's values and tile i + 1's keys are in LDS, the buffers filled below are read no more
        const int g3 = look_up(i + 3);
        if (i + 2 < end) bring_k(i + 2, g2, b);
        if (i + 1 < end) bring_v(i + 1, g1, 1 - b);
        if constexpr (Q8) bring_scales(i + 2, g2, i + 1, g1);
        __builtin_amdgcn_sched_barrier(0);

        if (Q8 || wrows > 0) {  // (a wave without rows only brings its part; 8-bit: not worth the registers)
            const int t0 = span.at(i) * kTileKeys;
            const uint32_t vb = value_base(b), kb = key_base(1 - b);
            // (8-bit: the scales of the lane's tokens 4x .. 4x + 3 of 32)
            auto key_scales = [&](int x) { return *reinterpret_cast<const f4 *>(&sh.ksc[(i - begin) & 3][16 * (x / 2) + 8 * hh + 4 * (x % 2)]); };
            auto value_scales = [&](int x) { return *reinterpret_cast<const f4 *>(&sh.vsc[b][16 * (x / 2) + 8 * hh + 4 * (x % 2)]); };
            if constexpr (Q8) {
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    const f4 kx = key_scales(x);
#pragma unroll
                    for (int r = 0; r < 4; ++r) sc[x / 4][4 * (x % 4) + r] *= kx[r];
                }
            }
            const bool full = ok == 15 && t0 + kTileKeys - 1 <= pmin &&
                              (a.window <= 0 || t0 > pmax - a.window || t0 + kTileKeys <= a.sinks);
            uint32_t seen = 0xffffffffu;
            if (!full) {
                seen = 0;
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    seen |= ((ok >> u & 1u) ? seen_bits<8>(t0 + 16 * u + 8 * hh, pos, low, a.sinks) : 0u) << (8 * u);
#pragma unroll
                for (int j = 0; j < 32; ++j) sc[j / 16][j % 16] = seen_or_none(seen, j, sc[j / 16][j % 16]);
            }
            float top = max3(sc[0][0], sc[0][1], sc[0][2]);
#pragma unroll
            for (int j = 3; j < 31; j += 2) top = max3(top, sc[j / 16][j % 16], sc[(j + 1) / 16][(j + 1) % 16]);
            top = fmaxf(top, sc[1][15]);
            m = fmaxf(m, halves_max(top) * p.sl2);
            if constexpr (Q8) {
                const f4 most = *reinterpret_cast<const f4 *>(sh.vmax[b]);
                float big = fmaxf(max3(most[0], most[1], most[2]), most[3]);
                if (!full && __any(scale_shift(big) > shift_v)) {  // of those that the row sees, where that can matter
                    big = 0.0f;
#pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        const f4 vx = value_scales(x);
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const float y = fabsf(vx[r]);
                            const bool in = ((seen >> (4 * x + r) & 1u) != 0) & (y < __builtin_inff());
                            big = fmaxf(big, in ? y : 0.0f);
                        }
                    }
                    big = halves_max(big);
                }
                shift_v = fmaxf(shift_v, scale_shift(big));
            }
            const float ms = raised(m, Q8 ? shift_v : kWeightShift);
            const float alpha = __builtin_amdgcn_exp2f(base - ms);
            base = ms;
            l *= alpha;
            if (!__all(alpha == 1.0f)) {
#pragma unroll
                for (int d = 0; d < DB; ++d) acc[d] *= alpha;
            }

            f16v sn[2];  // (past the last tile: of what the buffer holds, not used)
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r) sn[n][r] = 0.0f;
            h8 pb[4];
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
            auto product = [&](int u) {
#pragma unroll
                for (int d = 0; d < DB; ++d)
                    acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, value(vb, d, u)), pb[u], acc[d], 0, 0, 0);
            };
            // in quarters, each between fences: exponentials of 16 tokens, a quarter of the next
            // scores, and from the third on the product of the quarter two before. The scores' keys
            // are read a quarter ahead (a prompt of 8192 661 -> 653 us); with 8-bit ones that spills
            // (window prompts 94 -> 101 us).
            h8 kk[Q8 ? 1 : KS / 2];
            if constexpr (!Q8) {
#pragma unroll
                for (int k = 0; k < KS / 2; ++k) kk[k] = key(kb, 0, k);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                f4 vx[2];
                if constexpr (Q8) {
                    vx[0] = value_scales(2 * u);
                    vx[1] = value_scales(2 * u + 1);
                }
#pragma unroll
                for (int k = 0; k < KS / 2; ++k)
                    sn[u / 2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(Q8 ? key(kb, u / 2, u % 2 * KS / 2 + k) : kk[k],
                                                                       q[u % 2 * KS / 2 + k], sn[u / 2], 0, 0, 0);
                if constexpr (!Q8) {
#pragma unroll
                    for (int k = 0; k < (u < 3 ? KS / 2 : 0); ++k) kk[k] = key(kb, (u + 1) / 2, (u + 1) % 2 * KS / 2 + k);
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    float e = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[u / 2][8 * (u % 2) + j], p.sl2, -ms));
                    sum[u] += e;
                    if constexpr (Q8) e *= vx[j / 4][j % 4];
                    pb[u][j] = _Float16(e);
                }
                if constexpr (Q8) {  // (a hidden token's scale may be no number)
                    if (!full) pb[u] = __builtin_bit_cast(h8, u4(__builtin_bit_cast(u4, pb[u]) & halves_of(seen >> 8 * u)));
                }
                if (u >= 2) product(u - 2);
                __builtin_amdgcn_sched_barrier(0);
            }
            product(2);
            product(3);
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
            for (int n = 0; n < 2; ++n) sc[n] = sn[n];
        }
        if constexpr (Q8) {
            __builtin_amdgcn_sched_barrier(0);
            if (i + 2 < end) put_k(b, i + 2 - begin);
            if (i + 1 < end) put_v(1 - b);
        }
        ok = groups(g1);
        g1 = g2;
        g2 = g3;
    }

    if constexpr (!Q8) {
        __syncthreads();
        if (sh.wild) {  // of what each row sees of those values, counts, and what they make of its sum
            for (int i = begin; i < end; ++i) {
                const int t0 = span.at(i) * kTileKeys;
                if (!partial(i, groups(look_up(i)))) continue;
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    f16v cnt;
#pragma unroll
                    for (int r = 0; r < 16; ++r) cnt[r] = 0.0f;
#pragma unroll 1
                    for (int u = 0; u < 4; ++u) {
                        const int at = t0 + 16 * u + 8 * hh, id = page_of(a.b, s, t0 + 16 * u, v.len);
                        u4 w = *reinterpret_cast<const u4 *>(static_cast<const uint8_t *>(a.vc) +
                            (((size_t(max(id, 0)) * H + h) * D + 32 * d + col) * size_t(P) + size_t(at & (P - 1))) * 2);
                        const uint32_t bits = id >= 0 ? seen_bits<8>(at, pos, low, a.sinks) : 0u;
                        h8 sb;
#pragma unroll
                        for (int j = 0; j < 8; ++j) sb[j] = _Float16(float(bits >> j & 1u));
                        cnt = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, take_nonfinite(w)), sb, cnt, 0, 0, 0);
                    }
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[d][r] += nonfinite_sum(cnt[r]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
    }
    const float total = halves_sum(l);
    if (col < wrows) {
        if (!direct) {
            const size_t slot = size_t(slot0 + wr + col);
            if (hh == 0) p.part_ml[slot] = make_float2(base, total);
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    *reinterpret_cast<f4 *>(p.part_o + slot * D + 32 * d + 8 * x + 4 * hh) =
                        f4{acc[d][4 * x], acc[d][4 * x + 1], acc[d][4 * x + 2], acc[d][4 * x + 3]};
        } else {
            const float inv = (total > 0.0f || total != total ? 1.0f / total : 0.0f);
            const size_t dst = size_t(v.r0 + qi) * a.out_stride + size_t(h * G + qg) * D + size_t(4 * hh);
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    h4 y;
#pragma unroll
                    for (int r = 0; r < 4; ++r) y[r] = _Float16(acc[d][4 * x + r] * inv);
                    if (a.out_f32)
                        *reinterpret_cast<f4 *>(static_cast<float *>(a.out) + dst + 32 * d + 8 * x) =
                            f4{float(y[0]), float(y[1]), float(y[2]), float(y[3])};
                    else
                        *reinterpret_cast<h4 *>(static_cast<uint16_t *>(a.out) + dst + 32 * d + 8 * x) = y;
                }
        }
    }
    __syncthreads();  // (the next row tile's first store)
}
// The shared work (or, with no workers, a workgroup for each head of a sequence).
// R 16: few rows, a wave's tokens its own; R 128: the waves' rows, the tokens in LDS.
template <int D, int R, int NW, bool Q8, bool LINES>
__global__ __launch_bounds__(64 * NW, R == 128 && D > 128 ? 1 : 2) void attn_split_kernel(SplitArgs p) {
    constexpr int kLeast = R == 16 ? NW : 4;  // units of a worker, where all are fewer than the workers could take
    __shared__ std::conditional_t<R == 16, SplitShared<D, NW>, TileShared<D>> sh;
    __shared__ int upto[kMaxShared + 1];
    __shared__ uint32_t sums[NW];
    const AttnArgs &a = p.a;
    const int H = a.b.n_heads, G = a.group;
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int worker = int(blockIdx.x);

    Work work{upto, a.b.n_seqs, H, 0, 0, 0, 0};
    int at = 0, stop = 1;
    if (p.workers) {  // the units of every sequence, summed
        constexpr int N = kMaxShared / (64 * NW);  // sequences of a thread
        uint32_t mine[N], sum = 0;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int q = int(threadIdx.x) * N + j;
            mine[j] = 0;
            if (q < a.b.n_seqs) {
                const SeqView v = seq_view(a.b, q);
                if (v.n_new >= p.new_min && v.n_new <= p.new_max)  // (one sequence's stay below 2^31)
                    for (int rt = 0; rt * R < v.n_new * G; ++rt) mine[j] += unsigned(row_tile<R>(a, v, rt).units);
            }
            sum = capped_sum(sum, mine[j]);
        }
        uint32_t before = sum;
#pragma unroll
        for (int o = 1; o < 64; o *= 2) {
            const uint32_t x = __shfl_up(before, o);
            before = capped_sum(before, lane >= o ? x : 0);
        }
        if (lane == 63) sums[wid] = before;
        before -= sum;
        __syncthreads();
        uint32_t total = 0;
        for (int w = 0; w < NW; ++w) {
            if (w < wid) before += sums[w];
            total = capped_sum(total, sums[w]);
        }
        if (threadIdx.x == 0) upto[0] = 0;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            before += mine[j];
            upto[threadIdx.x * N + j + 1] = int(before);
        }
        __syncthreads();
        const int units = call_units(__builtin_amdgcn_readfirstlane(total), H);  // (none: no worker reads upto)
        work.set(units, min(p.workers, units / kLeast + (units % kLeast != 0)));
        if (threadIdx.x == 0 && blockIdx.x == 0) p.shared[p.workers].pieces = work.workers;  // (for the join)
        if constexpr (R == 128) {
            // workgroups b, b + 8, .. run on one XCD: they are neighbours in the work, and the
            // row tiles of one head, at the same tokens at one time, meet in that XCD's L2
            const int per = (work.workers + 7) / 8;
            if (int(blockIdx.x / 8) >= per) return;
            worker = int(blockIdx.x % 8) * per + int(blockIdx.x / 8);
        }
        if (worker >= work.workers) return;
        const int edge = work.bound(worker + (lane & 1));  // (both ends at once)
        at = __builtin_amdgcn_readlane(edge, 0);
        stop = __builtin_amdgcn_readlane(edge, 1);
        if (threadIdx.x == 0) p.shared[worker].pieces = 0;
    }

    int next_tile = 0;  // (nothing shared: the head's row tiles in turn)
    while (at < stop) {
        // the segment that holds unit `at`, and this worker's piece of it
        int s, h, rt = 0, off = 0;
        if (p.workers) {
            s = __builtin_amdgcn_readfirstlane(work.seq_of(at));
            const int n = upto[s + 1] - upto[s], u = at - upto[s] * H;
            h = __builtin_amdgcn_readfirstlane(u / n);
            off = __builtin_amdgcn_readfirstlane(u - h * n);
        } else {
            s = worker / H;
            h = worker - s * H;
            rt = next_tile++;
        }
        const SeqView v = seq_view(a.b, s);
        if (!p.workers && (v.n_new < p.new_min || v.n_new > p.new_max || rt * R >= v.n_new * G)) return;
        RowTile tile = row_tile<R>(a, v, rt);
        while (off >= tile.units) {
            off -= tile.units;
            tile = row_tile<R>(a, v, ++rt);
        }
        const int begin = off;
        int end = tile.units;
        if (p.workers) {
            end = min(end, begin + (stop - at));
            at += end - begin;
        }
        const bool direct = end - begin == tile.units;
        const int slot0 = (worker * 2 + (begin == 0)) * R;
        if (!direct && begin == 0 && wid == 0) {
            // the workers up to the one of the segment's last unit, 64 borders at a time
            const int last = at - end + tile.units - 1;
            int n = 2;
            for (;; n += 64) {
                const uint64_t past = __ballot(work.bound(worker + n + lane) > last);
                if (past) {
                    n += __builtin_ctzll(past);
                    break;
                }
            }
            if (lane == 0) p.shared[worker] = SharedSegment{n, s, h, tile.row0, tile.nrows};
        }
        end = min(end, tile.span.n);  // (a span of no tiles)
        if constexpr (R == 16) split_piece<D, NW, Q8, LINES>(p, sh, v, tile, s, h, begin, end, direct, slot0);
        else tile_piece<D, Q8>(p, sh, lds_addr(&sh), v, tile, s, h, begin, end, direct, slot0);
    }
}

// A workgroup for each row tile, nothing shared: a call of many rows.
template <int D, bool Q8>
__global__ __launch_bounds__(256, D > 128 ? 1 : 2) void attn_tile_kernel(SplitArgs p) {
    __shared__ TileShared<D> sh;
    const AttnArgs &a = p.a;
    const int h = int(blockIdx.x) % a.b.n_heads, s = int(blockIdx.x) / a.b.n_heads;
    const SeqView v = seq_view(a.b, s);
    if (v.n_new < p.new_min || v.n_new > p.new_max) return;
    // the last row tiles see most: they go first
    for (int rt = int(gridDim.y) - 1 - int(blockIdx.y); rt * 128 < v.n_new * a.group; rt += int(gridDim.y)) {
        const RowTile tile = row_tile<128>(a, v, rt);
        tile_piece<D, Q8>(p, sh, lds_addr(&sh), v, tile, s, h, 0, tile.span.n, true, 0);
    }
}

// Joins the segments' pieces, for each worker that has a segment's first tile. A wave
// a row; or (ROWS: few segments of many pieces, so the owners are some workers apart) a
// workgroup a row, which looks at kOwners workers: a quarter of the workgroups.
constexpr int kOwners = 4;
template <int D, int R, bool ROWS>
__global__ __launch_bounds__(64 * kJoinWaves) void attn_pieces_kernel(SplitArgs p) {
    __shared__ float part[ROWS ? kJoinWaves : 1][D];
    __shared__ float2 ml[kJoinWaves];
    constexpr int N = D / 64, OWN = ROWS ? kOwners : 1;
    const int first = int(blockIdx.y) * OWN, workers = p.shared[p.workers].pieces;  // (rows across the XCDs: owners may be 8 workers apart)
    int pieces[OWN];
#pragma unroll
    for (int i = 0; i < OWN; ++i) pieces[i] = first + i < workers ? p.shared[first + i].pieces : 0;
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
        if (pieces[i] < 2) continue;
        const int w = first + i;
        const SharedSegment seg = p.shared[w];
        const AttnArgs &a = p.a;
        const SeqView v = seq_view(a.b, seg.seq);
        auto slot = [&](int k, int r) { return int64_t((w + k) * 2 + (k == 0)) * R + r; };
        auto place = [&](int r) {
            const int row = seg.row0 + r, i = token_of(a, row), g = row - i * a.group;
            return size_t(v.r0 + i) * a.out_stride + size_t(seg.head * a.group + g) * D;
        };
        if constexpr (ROWS) {
            for (int r = int(blockIdx.x); r < seg.rows; r += int(gridDim.x))
                join_row<D>(p, seg.pieces, [&](int k) { return slot(k, r); }, part, ml, place(r));
        } else {
            const int lane = threadIdx.x & 63;
            for (int r = kJoinWaves * int(blockIdx.x) + int(threadIdx.x >> 6); r < seg.rows; r += kJoinWaves * int(gridDim.x)) {
                float o[N], m, l;
                join_pieces<D>(p, 0, 1, seg.pieces, [&](int k) { return slot(k, r); }, o, m, l);
                const size_t dst = place(r);
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const _Float16 y = _Float16(l > 0.0f || l != l ? o[j] / l : 0.0f);
                    if (a.out_f32) static_cast<float *>(a.out)[dst + 64 * j + lane] = float(y);
                    else static_cast<_Float16 *>(a.out)[dst + 64 * j + lane] = y;
                }
            }
        }
    }
}

template <int D, int R, int NW, bool LINES> void launch_split(const SplitArgs &p, dim3 grid, hipStream_t s) {
    if (p.a.ks) hipLaunchKernelGGL((attn_split_kernel<D, R, NW, true, LINES>), grid, dim3(64 * NW), 0, s, p);
    else hipLaunchKernelGGL((attn_split_kernel<D, R, NW, false, LINES>), grid, dim3(64 * NW), 0, s, p);
}

template <int D> hipError_t launch_plan(SplitArgs &p, const SplitPlan &pl, hipStream_t s) {
    const AttnArgs &a = p.a;
    const unsigned units = unsigned(a.b.n_seqs) * unsigned(a.b.n_heads);
    // (128 rows: the workers of an XCD are workgroups 8 apart, so all eight need as many)
    const dim3 grid(!pl.workers ? units : pl.rows == 128 ? unsigned(pl.workers + 7) / 8 * 8 : unsigned(pl.workers));
    if (pl.rows == 128) {
        const dim3 tiles(units, unsigned(pl.row_tiles));
        if (pl.workers) launch_split<D, 128, 4, false>(p, grid, s);
        else if (a.ks) hipLaunchKernelGGL((attn_tile_kernel<D, true>), tiles, dim3(256), 0, s, p);
        else hipLaunchKernelGGL((attn_tile_kernel<D, false>), tiles, dim3(256), 0, s, p);
    } else if constexpr (D <= 128) {
        if (pl.nw == 8 && pl.lines) launch_split<D, 16, 8, true>(p, grid, s);
        else if (pl.nw == 8) launch_split<D, 16, 8, false>(p, grid, s);
        else if (pl.lines) launch_split<D, 16, 4, true>(p, grid, s);
        else launch_split<D, 16, 4, false>(p, grid, s);
    } else {
        if (pl.lines) launch_split<D, 16, 4, true>(p, grid, s);
        else launch_split<D, 16, 4, false>(p, grid, s);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !pl.workers) return e;
    const int64_t rows = std::min<int64_t>(int64_t(a.max_new) * a.group, pl.rows);
    const unsigned rows8 = unsigned((rows + kJoinWaves - 1) / kJoinWaves), owners4 = (grid.x + kOwners - 1) / kOwners;
    const dim3 block(64 * kJoinWaves);
    if (pl.rows == 128) hipLaunchKernelGGL((attn_pieces_kernel<D, 128, false>), dim3(rows8, grid.x), block, 0, s, p);
    else if (grid.x > kOwners * units) hipLaunchKernelGGL((attn_pieces_kernel<D, 16, true>), dim3(unsigned(rows), owners4), block, 0, s, p);
    else hipLaunchKernelGGL((attn_pieces_kernel<D, 16, false>), dim3(rows8, grid.x), block, 0, s, p);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_attention(const AttnArgs &a, void *scratch, size_t scratch_bytes, int cu_count, hipStream_t s) {
    SplitPlan plans[2];
    const int n = plan_call(a, cu_count, scratch ? scratch_bytes : 0, plans);
    uint8_t *base = static_cast<uint8_t *>(scratch);
    for (int i = 0; i < n; ++i) {
        const SplitPlan &pl = plans[i];
        SplitArgs p{};
        p.a = a;
        p.sl2 = a.scale * 1.44269504088896341f;
        p.new_min = pl.new_min;
        p.new_max = pl.new_max;
        p.workers = pl.workers;
        if (pl.bytes) {
            p.part_o = reinterpret_cast<float *>(base);
            p.part_ml = reinterpret_cast<float2 *>(p.part_o + pl.slots * size_t(a.head_dim));
            p.shared = reinterpret_cast<SharedSegment *>(p.part_ml + pl.slots);
            base += pl.bytes;
        }
        const hipError_t e = a.head_dim == 64    ? launch_plan<64>(p, pl, s)
                             : a.head_dim == 128 ? launch_plan<128>(p, pl, s)
                                                 : launch_plan<256>(p, pl, s);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace qmm
