// qmm_attn.hip — attention of new tokens over a paged key-value cache.
//
// A key-value head's query heads times a sequence's new tokens are the rows;
// 16 NC of them are the columns of the products
//   S^T [tokens x rows] = K Q^T,   O^T [values x rows] = V^T P^T
// on 16x16x32 fp16 MFMA, 64 tokens a tile, with the running maximum m and sum l
// of the softmax in base 2 (exp2(s scale log2 e - m)), fp32. Which token a row
// of an MFMA operand stands for is free, so each lane is given 16 consecutive
// tokens of the tile's 64 (lane group c = lane / 16: tokens 16c .. 16c + 15):
//   S:  operand row i of MFMA t is token 16 (i / 4) + 4 t + i % 4, and the lane
//       finds its scores of tokens 16c + 4t + r in register r of result t;
//   PV: operand k index 8c + j of step u is token 16c + 8u + j: P stays in the
//       lane that computed it, and V (stored with a value's tokens side by
//       side) is read 32 B a lane. A page holds 16 tokens or more, so a lane
//       looks up one page for its keys and one for its values.
// Keys and values go from memory straight to the operands.
#include <hip/hip_runtime.h>

#include "qmm_attn.h"
#include "qmm_device.h"

namespace qmm {
namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

struct SplitArgs {
    AttnArgs a;
    float sl2;  // scale log2(e)
    int nsplit, chunk, row_tiles;
    float *part_o;   // [seq][head][split][rows][D], rows = row_tiles * 16 NC
    float2 *part_ml;  // (m, l) of the same rows
};

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

// A value that is no number, made a count: +inf 1, -inf 128, NaN 16384 (64
// tokens' counts stay apart in a sum); finite values 0.
__device__ inline uint32_t nonfinite_code(uint32_t h) {
    if ((h & 0x7c00u) != 0x7c00u) return 0u;
    return (h & 0x3ffu) ? 0x7400u : (h & 0x8000u) ? 0x5800u : 0x3c00u;  // fp16 16384, 128, 1
}
// what those counts of a row's visible tokens make of its sum
__device__ inline float nonfinite_sum(float count) {
    const int n = int(count);
    float r = 0.0f;
    if (n & 127) r += __builtin_inff();
    if ((n >> 7) & 127) r -= __builtin_inff();
    if (n >> 14) r = __builtin_nanf("");
    return r;
}

template <int D, int NC, bool Q8>
__global__ __launch_bounds__(256, NC == 1 && D <= 128 ? 2 : 1) void attn_split_kernel(SplitArgs p) {
    constexpr int R = 16 * NC;           // rows of a row tile
    constexpr int KS = D / 32;           // MFMA steps of a score
    constexpr int DT = D / 16;           // value tiles
    constexpr int KR = Q8 ? D / 64 : KS;  // 16-B registers of a key operand
    constexpr int VR = Q8 ? 1 : 2;
    constexpr int DG = DT < 8 ? DT : 8;  // value tiles joined at a time
    __shared__ f4 joined[4][DG][64];
    __shared__ float2 ml[4][R];

    const AttnArgs &a = p.a;
    const int H = a.b.n_heads, G = a.group;
    const int h = int(blockIdx.x) % H, s = int(blockIdx.x) / H, split = int(blockIdx.y);
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, col = lane & 15, c = lane >> 4;
    const SeqView v = seq_view(a.b, s);
    const int64_t rows = int64_t(v.n_new) * G;
    const int P = 1 << a.b.page_shift, shift = a.b.page_shift;

    for (int64_t rt = blockIdx.z; rt * R < rows; rt += gridDim.z) {
        const int64_t row0 = rt * R;
        const int nrows = int(rows - row0 < R ? rows - row0 : R);
        const int pmin = v.pos0 + int(row0 / G), pmax = v.pos0 + int((row0 + nrows - 1) / G);
        const TileSpan span = tile_span(pmin, pmax, a.window, a.sinks);
        // row tiles past what the host said have no place for partial results: one split takes them whole
        const bool planned = rt < p.row_tiles;
        const int per = planned ? split_tiles(span.n, p.nsplit, p.chunk) : span.n;
        const int begin = split * per, end = min(begin + per, span.n);
        if (begin >= end && split > 0) continue;
        const bool direct = per >= span.n;  // the only split

        // this lane's rows: queries, positions
        h8 q[NC][KS];
        int pos[NC];
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            const int r = 16 * n + col;
            const int64_t row = row0 + (r < nrows ? r : 0);
            const int i = int(row / G), g = int(row % G);
            pos[n] = v.pos0 + i;
            const uint16_t *src = a.q + size_t(v.r0 + i) * a.q_stride + size_t(h * G + g) * D;
#pragma unroll
            for (int k = 0; k < KS; ++k)
                q[n][k] = *reinterpret_cast<const h8 *>(src + (Q8 ? 64 * (k / 2) + 16 * c + 8 * (k % 2) : 32 * k + 8 * c));
        }
        float m[NC], l[NC], vref[NC];
        f4 acc[NC][DT];
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            m[n] = -__builtin_inff();
            l[n] = 0.0f;
            vref[n] = 1e-30f;
#pragma unroll
            for (int d = 0; d < DT; ++d) acc[n][d] = f4{0.f, 0.f, 0.f, 0.f};
        }

        u4 kr[4][KR], vr[DT][VR];
        f4 ksc[4], vsc[4];
        int id_k = -1, id_v = -1, tile = 0;
        const int ck = col >> 2;  // the lane group whose tokens this lane loads keys of
        auto look_up = [&](int i, int &ik, int &iv) {
            const int t = span.at(i) * kTileKeys;
            ik = page_of(a.b, s, t + 16 * ck, v.len);
            iv = page_of(a.b, s, t + 16 * c, v.len);
        };
        auto load_k = [&](int i, int id) {
            const int slot = (span.at(i) * kTileKeys + 16 * ck) & (P - 1);
            const size_t cell = ((size_t(max(id, 0)) * H + h) << shift) + size_t(slot + (lane & 3));
            const uint8_t *src = static_cast<const uint8_t *>(a.kc) + cell * (Q8 ? D : 2 * D) + 16 * c;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int k = 0; k < KR; ++k)
                    kr[t][k] = *reinterpret_cast<const u4 *>(src + t * 4 * (Q8 ? D : 2 * D) + k * 64);
        };
        if (begin + wid < end) {
            look_up(begin + wid, id_k, id_v);
            load_k(begin + wid, id_k);
        }
        for (int i = begin + wid; i < end; i += 4) {
            tile = span.at(i);
            const int t0 = tile * kTileKeys, slot_v = (t0 + 16 * c) & (P - 1);
            {   // this tile's values (and scales)
                const size_t hv = size_t(max(id_v, 0)) * H + h;
                const uint8_t *src = static_cast<const uint8_t *>(a.vc) + ((hv * D + col) * size_t(P) + slot_v) * (Q8 ? 1 : 2);
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int j = 0; j < VR; ++j)
                        vr[d][j] = *reinterpret_cast<const u4 *>(src + size_t(d) * 16 * P * (Q8 ? 1 : 2) + 16 * j);
                if constexpr (Q8) {
                    const size_t cell = (hv << shift) + size_t(slot_v);
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        ksc[t] = *reinterpret_cast<const f4 *>(a.ks + cell + 4 * t);
                        vsc[t] = *reinterpret_cast<const f4 *>(a.vs + cell + 4 * t);
                    }
                }
            }
            const bool page_ok = id_v >= 0;
            int nk = -1, nv = -1;
            if (i + 4 < end) look_up(i + 4, nk, nv);
            __builtin_amdgcn_sched_barrier(0);

            f4 sc[NC][4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
#pragma unroll
                for (int n = 0; n < NC; ++n) sc[n][t] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    h8 kk;
                    if constexpr (Q8) kk = codes8(kr[t][k / 2][2 * (k % 2)], kr[t][k / 2][2 * (k % 2) + 1]);
                    else kk = __builtin_bit_cast(h8, kr[t][k]);
#pragma unroll
                    for (int n = 0; n < NC; ++n)
                        sc[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk, q[n][k], sc[n][t], 0, 0, 0);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            if (i + 4 < end) load_k(i + 4, nk);
            id_k = nk;
            id_v = nv;
            __builtin_amdgcn_sched_barrier(0);

            // tokens of this lane: key0 .. key0 + 15
            const int key0 = t0 + 16 * c;
            const bool full = __all(page_ok) && t0 + kTileKeys - 1 <= pmin &&
                              (a.window <= 0 || t0 > pmax - a.window || t0 + kTileKeys <= a.sinks);
            uint32_t seen[NC];  // bit j: token key0 + j is visible to the row
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                if constexpr (Q8) {
#pragma unroll
                    for (int t = 0; t < 4; ++t) sc[n][t] *= ksc[t];
                }
                seen[n] = 0xffffu;
                if (!full) {
                    uint32_t bits = 0;
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const int key = key0 + j;
                        const bool ok = page_ok && key <= pos[n] &&
                                        (a.window <= 0 || key > pos[n] - a.window || key < a.sinks);
                        bits |= ok ? 1u << j : 0u;
                        if (!ok) sc[n][j / 4][j % 4] = -__builtin_inff();
                    }
                    seen[n] = bits;
                }
                float top = sc[n][0][0];
#pragma unroll
                for (int j = 1; j < 16; ++j) top = fmaxf(top, sc[n][j / 4][j % 4]);
                const float mn = fmaxf(m[n], groups_max(top) * p.sl2);
                const float ms = mn == -__builtin_inff() ? 0.0f : mn;
                const float lscale = __builtin_amdgcn_exp2f(m[n] - ms);
                float alpha = lscale, vinv = 1.0f;
                if constexpr (Q8) {  // the largest value scale the row has seen: its weights below are relative to it
                    float big = vref[n];
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const float x = fabsf(vsc[j / 4][j % 4]);
                        big = fmaxf(big, ((seen[n] >> j) & 1u) && x < __builtin_inff() ? x : 0.0f);
                    }
                    big = groups_max(big);
                    alpha *= vref[n] / big;
                    vref[n] = big;
                    vinv = 1.0f / big;
                }
                m[n] = mn;
                float sum = 0.0f;
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[n][j / 4][j % 4], p.sl2, -ms));
                    sc[n][j / 4][j % 4] = e;
                    sum += e;
                }
                l[n] = l[n] * lscale + sum;
                if (!__all(alpha == 1.0f)) {
#pragma unroll
                    for (int d = 0; d < DT; ++d) acc[n][d] *= alpha;
                }
                if constexpr (Q8) {  // the weights of the codes: p * scale
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const float w = sc[n][j / 4][j % 4] * (vsc[j / 4][j % 4] * vinv);
                        sc[n][j / 4][j % 4] = (seen[n] >> j) & 1u ? w : 0.0f;
                    }
                }
            }
            if constexpr (!Q8) {
                if (!full) {
                    // cells no row of the tile sees: their bits may be anything, a weight of 0 does not hide a NaN
                    uint32_t any = 0;
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const int key = key0 + j;
                        const bool ok = page_ok && key <= pmax && (a.window <= 0 || key > pmin - a.window || key < a.sinks);
                        any |= ok ? 1u << j : 0u;
                    }
                    u4 keep[2];
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        keep[j / 4][j % 4] = ((any >> (2 * j)) & 1u ? 0xffffu : 0u) | ((any >> (2 * j + 1)) & 1u ? 0xffff0000u : 0u);
                    uint32_t wild = 0;
#pragma unroll
                    for (int d = 0; d < DT; ++d)
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            vr[d][u] &= keep[u];
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const uint32_t x = vr[d][u][j] & 0x7c007c00u;
                                wild |= uint32_t((x & 0xffffu) == 0x7c00u) | uint32_t((x >> 16) == 0x7c00u);
                            }
                        }
                    // values that are no numbers, seen by some rows of the tile and hidden from
                    // others: out of the product, and back as counts of what each row sees
                    if (pmin != pmax && __any(wild != 0)) {
                        h8 sb[NC][2];
#pragma unroll
                        for (int n = 0; n < NC; ++n)
#pragma unroll
                            for (int j = 0; j < 16; ++j) sb[n][j / 8][j % 8] = _Float16(float((seen[n] >> j) & 1u));
#pragma unroll
                        for (int d = 0; d < DT; ++d) {
                            f4 cnt[NC];
#pragma unroll
                            for (int n = 0; n < NC; ++n) cnt[n] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                            for (int u = 0; u < 2; ++u) {
                                u4 code;
#pragma unroll
                                for (int j = 0; j < 4; ++j) {
                                    const uint32_t w = vr[d][u][j];
                                    const uint32_t lo = nonfinite_code(w & 0xffffu), hi = nonfinite_code(w >> 16);
                                    code[j] = lo | hi << 16;
                                    vr[d][u][j] = w & ((lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u));
                                }
#pragma unroll
                                for (int n = 0; n < NC; ++n)
                                    cnt[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, code), sb[n][u],
                                                                                   cnt[n], 0, 0, 0);
                            }
#pragma unroll
                            for (int n = 0; n < NC; ++n)
#pragma unroll
                                for (int r = 0; r < 4; ++r) acc[n][d][r] += nonfinite_sum(cnt[n][r]);
                        }
                    }
                }
            }
            h8 pb[NC][2];
#pragma unroll
            for (int n = 0; n < NC; ++n)
#pragma unroll
                for (int j = 0; j < 16; ++j) pb[n][j / 8][j % 8] = _Float16(sc[n][j / 4][j % 4]);
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    h8 vv;
                    if constexpr (Q8) vv = codes8(vr[d][0][2 * u], vr[d][0][2 * u + 1]);
                    else vv = __builtin_bit_cast(h8, vr[d][u]);
#pragma unroll
                    for (int n = 0; n < NC; ++n)
                        acc[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vv, pb[n][u], acc[n][d], 0, 0, 0);
                }
        }

        // the four waves' results, joined in LDS
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            const float sum = groups_sum(l[n]);
            if (c == 0) ml[wid][16 * n + col] = make_float2(m[n], sum);
        }
        __syncthreads();
        const size_t slot0 = ((size_t(s) * H + h) * size_t(p.nsplit) + size_t(split)) * size_t(p.row_tiles) * R + size_t(row0);
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            float top = ml[0][16 * n + col].x;
#pragma unroll
            for (int w = 1; w < 4; ++w) top = fmaxf(top, ml[w][16 * n + col].x);
            const float base = top == -__builtin_inff() ? 0.0f : top;
            float total = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) total += ml[w][16 * n + col].y * __builtin_amdgcn_exp2f(ml[w][16 * n + col].x - base);
            const float mine = __builtin_amdgcn_exp2f(m[n] - base) * (Q8 ? vref[n] : 1.0f);
            const float inv = direct ? (total > 0.0f || total != total ? 1.0f / total : 0.0f) : 1.0f;
            const int r = 16 * n + col;
            const int64_t row = row0 + r;
            const bool on = r < nrows;
            if (!direct && on && threadIdx.x < 16) p.part_ml[slot0 + r] = make_float2(top, total);
#pragma unroll
            for (int d0 = 0; d0 < DT; d0 += DG) {
                if (n || d0) __syncthreads();
#pragma unroll
                for (int d = 0; d < DG; ++d) joined[wid][d][lane] = acc[n][d0 + d] * mine;
                __syncthreads();
#pragma unroll
                for (int d = wid; d < DG; d += 4) {
                    f4 o = (joined[0][d][lane] + joined[1][d][lane]) + (joined[2][d][lane] + joined[3][d][lane]);
                    if (!on) continue;
                    const int at = 16 * (d0 + d) + 4 * c;
                    if (!direct) {
                        *reinterpret_cast<f4 *>(p.part_o + (slot0 + r) * D + at) = o;
                        continue;
                    }
                    o *= inv;
                    const int i = int(row / G), g = int(row % G);
                    const size_t dst = size_t(v.r0 + i) * a.out_stride + size_t(h * G + g) * D + size_t(at);
                    const h4 y = {_Float16(o[0]), _Float16(o[1]), _Float16(o[2]), _Float16(o[3])};
                    if (a.out_f32)
                        *reinterpret_cast<f4 *>(static_cast<float *>(a.out) + dst) =
                            f4{float(y[0]), float(y[1]), float(y[2]), float(y[3])};
                    else
                        *reinterpret_cast<h4 *>(static_cast<uint16_t *>(a.out) + dst) = y;
                }
            }
        }
        __syncthreads();
    }
}

// Joins a row's splits: one workgroup a row and head, its waves' shares of the
// splits in turn, a lane D / 64 values.
template <int D>
__global__ __launch_bounds__(256) void attn_join_kernel(SplitArgs p, int rows_per_tile) {
    constexpr int N = D / 64;
    __shared__ float part[4][D];
    __shared__ float2 ml[4];
    const AttnArgs &a = p.a;
    const int H = a.b.n_heads, G = a.group;
    const int h = int(blockIdx.x) % H, s = int(blockIdx.x) / H;
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
    const SeqView v = seq_view(a.b, s);
    const int64_t cap = int64_t(p.row_tiles) * rows_per_tile, rows = min(int64_t(v.n_new) * G, cap);
    for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
        const int64_t row0 = row / rows_per_tile * rows_per_tile;
        const int64_t last = min(row0 + rows_per_tile, int64_t(v.n_new) * G) - 1;
        const TileSpan span = tile_span(v.pos0 + int(row0 / G), v.pos0 + int(last / G), a.window, a.sinks);
        const int per = split_tiles(span.n, p.nsplit, p.chunk);
        if (per >= span.n) continue;  // (the split kernel wrote the row itself)
        const int n = (span.n + per - 1) / per;
        const size_t slot0 = (size_t(s) * H + h) * size_t(p.nsplit) * size_t(cap) + size_t(row);
        float o[N], m = -__builtin_inff(), l = 0.0f;
#pragma unroll
        for (int j = 0; j < N; ++j) o[j] = 0.0f;
        for (int i = wid; i < n; i += 4) {
            const size_t slot = slot0 + size_t(i) * size_t(cap);
            const float2 x = p.part_ml[slot];
            float y[N];
#pragma unroll
            for (int j = 0; j < N; ++j) y[j] = p.part_o[slot * D + 64 * j + lane];
            const float top = fmaxf(m, x.x), base = top == -__builtin_inff() ? 0.0f : top;
            const float wa = __builtin_amdgcn_exp2f(m - base), wb = __builtin_amdgcn_exp2f(x.x - base);
            m = top;
            l = l * wa + x.y * wb;
#pragma unroll
            for (int j = 0; j < N; ++j) o[j] = o[j] * wa + y[j] * wb;
        }
        if (lane == 0) ml[wid] = make_float2(m, l);
#pragma unroll
        for (int j = 0; j < N; ++j) part[wid][64 * j + lane] = o[j];
        __syncthreads();
        if (threadIdx.x < D) {
            float top = ml[0].x;
            for (int w = 1; w < 4; ++w) top = fmaxf(top, ml[w].x);
            const float base = top == -__builtin_inff() ? 0.0f : top;
            float total = 0.0f, sum = 0.0f;
            for (int w = 0; w < 4; ++w) {
                const float e = __builtin_amdgcn_exp2f(ml[w].x - base);
                total += ml[w].y * e;
                sum += part[w][threadIdx.x] * e;
            }
            const float y = total > 0.0f || total != total ? sum / total : 0.0f;
            const int i = int(row / G), g = int(row % G);
            const size_t dst = size_t(v.r0 + i) * a.out_stride + size_t(h * G + g) * D + threadIdx.x;
            if (a.out_f32) static_cast<float *>(a.out)[dst] = float(_Float16(y));
            else static_cast<_Float16 *>(a.out)[dst] = _Float16(y);
        }
        __syncthreads();
    }
}

struct SplitPlan {
    int nc, row_tiles, nsplit, chunk;
    size_t bytes;
};

SplitPlan plan_split(const AttnArgs &a, int cu_count, size_t scratch) {
    SplitPlan p;
    const int64_t rows = int64_t(a.max_new) * a.group;
    p.nc = rows <= 16 ? 1 : rows <= 32 || a.head_dim > 128 ? 2 : 4;
    const int R = 16 * p.nc;
    p.row_tiles = int((rows + R - 1) / R);
    if (p.row_tiles > 65535) p.row_tiles = 65535;
    int tiles = (a.max_kv - 1) / kTileKeys + 1;
    if (a.window > 0) {
        const int64_t most = (int64_t(a.window) + a.max_new + a.sinks) / kTileKeys + 3;
        if (most < tiles) tiles = int(most);
    }
    const int64_t units = int64_t(a.b.n_seqs) * a.b.n_heads * p.row_tiles;
    const int64_t want = (int64_t(cu_count) * 4 + units - 1) / units;  // four workgroups per CU
    int64_t n = want < 1 ? 1 : want;
    const int64_t most = (tiles + 3) / 4;  // a tile for each wave at least
    if (n > most) n = most;
    const size_t slot = size_t(a.b.n_seqs) * a.b.n_heads * p.row_tiles * R * (size_t(a.head_dim) * 4 + 8);
    if (n > 1 && size_t(n) * slot > scratch) n = int64_t(scratch / slot);
    if (n < 1) n = 1;
    p.chunk = int((tiles + n - 1) / n);
    p.nsplit = (tiles + p.chunk - 1) / p.chunk;
    p.bytes = p.nsplit > 1 ? size_t(p.nsplit) * slot : 0;
    return p;
}

template <int D, int NC, bool Q8> void launch_split(const SplitArgs &p, dim3 grid, hipStream_t s) {
    hipLaunchKernelGGL((attn_split_kernel<D, NC, Q8>), grid, dim3(256), 0, s, p);
}
template <int D> hipError_t launch_split_d(const SplitArgs &p, int nc, bool q8, dim3 grid, hipStream_t s) {
    if (nc == 1) q8 ? launch_split<D, 1, true>(p, grid, s) : launch_split<D, 1, false>(p, grid, s);
    else if (nc == 2) q8 ? launch_split<D, 2, true>(p, grid, s) : launch_split<D, 2, false>(p, grid, s);
    else if constexpr (D <= 128) q8 ? launch_split<D, 4, true>(p, grid, s) : launch_split<D, 4, false>(p, grid, s);
    return hipGetLastError();
}

}  // namespace

size_t attn_scratch_bytes(const AttnArgs &a, int cu_count) { return plan_split(a, cu_count, ~size_t(0)).bytes; }

hipError_t launch_attention(const AttnArgs &a, void *scratch, size_t scratch_bytes, int cu_count, hipStream_t s) {
    const SplitPlan pl = plan_split(a, cu_count, scratch ? scratch_bytes : 0);
    SplitArgs p;
    p.a = a;
    p.sl2 = a.scale * 1.44269504088896341f;
    p.nsplit = pl.nsplit;
    p.chunk = pl.chunk;
    p.row_tiles = pl.row_tiles;
    const size_t slots = size_t(a.b.n_seqs) * a.b.n_heads * pl.nsplit * pl.row_tiles * 16 * pl.nc;
    p.part_o = static_cast<float *>(scratch);
    p.part_ml = pl.nsplit > 1 ? reinterpret_cast<float2 *>(p.part_o + slots * size_t(a.head_dim)) : nullptr;
    const dim3 grid(unsigned(a.b.n_seqs) * unsigned(a.b.n_heads), unsigned(pl.nsplit), unsigned(pl.row_tiles));
    const bool q8 = a.ks != nullptr;
    hipError_t e = a.head_dim == 64    ? launch_split_d<64>(p, pl.nc, q8, grid, s)
                   : a.head_dim == 128 ? launch_split_d<128>(p, pl.nc, q8, grid, s)
                                       : launch_split_d<256>(p, pl.nc, q8, grid, s);
    if (e != hipSuccess || pl.nsplit == 1) return e;
    const int64_t rows = int64_t(a.max_new) * a.group;
    const dim3 jg(grid.x, unsigned(rows < 65535 ? rows : 65535));
    if (a.head_dim == 64) hipLaunchKernelGGL(attn_join_kernel<64>, jg, dim3(256), 0, s, p, 16 * pl.nc);
    else if (a.head_dim == 128) hipLaunchKernelGGL(attn_join_kernel<128>, jg, dim3(256), 0, s, p, 16 * pl.nc);
    else hipLaunchKernelGGL(attn_join_kernel<256>, jg, dim3(256), 0, s, p, 16 * pl.nc);
    return hipGetLastError();
}

}  // namespace qmm
