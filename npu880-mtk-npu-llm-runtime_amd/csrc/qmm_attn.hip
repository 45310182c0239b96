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
typedef float f16v __attribute__((ext_vector_type(16)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

struct SplitArgs {
    AttnArgs a;
    float sl2;  // scale log2(e)
    int nsplit, chunk, row_tiles;
    int new_min, new_max;  // only sequences of this many new tokens
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

// Bit j < N: token key0 + j is visible to the row at position p, i.e. key <= p and
// (key > low or key < sinks). Whole masks from the three bounds, no test per token.
template <int N> __device__ inline uint32_t seen_bits(int key0, int p, int low, int sinks) {
    auto below = [&](int bound) { return (1u << min(max(bound - key0, 0), N)) - 1u; };  // tokens before `bound`
    return below(p + 1) & (~below(low + 1) | below(sinks));
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
__device__ inline uint32_t any_nonfinite(u4 w) {
    uint32_t r = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) r |= uint32_t((w[j] & 0x7c00u) == 0x7c00u) | uint32_t((w[j] & 0x7c000000u) == 0x7c000000u);
    return r;
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
    if (v.n_new < p.new_min || v.n_new > p.new_max) return;
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
        int pos[NC], low[NC];  // a row's position; the last token its window hides
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            const int r = 16 * n + col;
            const int64_t row = row0 + (r < nrows ? r : 0);
            const int i = int(row / G), g = int(row % G);
            pos[n] = v.pos0 + i;
            low[n] = a.window > 0 ? max(pos[n] - a.window, -1) : -1;
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
        int id_k = -1, id_v = -1;
        bool wild_tiles = false;
        const int ck = col >> 2;  // the lane group whose tokens this lane loads keys of
        auto is_full = [&](int t0, bool page_ok) {  // every row of the tile sees every token
            return __all(page_ok) && t0 + kTileKeys - 1 <= pmin &&
                   (a.window <= 0 || t0 > pmax - a.window || t0 + kTileKeys <= a.sinks);
        };
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
            const int t0 = span.at(i) * kTileKeys, slot_v = (t0 + 16 * c) & (P - 1);
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
            const bool full = is_full(t0, page_ok);
            uint32_t seen[NC];  // bit j: token key0 + j is visible to the row
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                if constexpr (Q8) {
#pragma unroll
                    for (int t = 0; t < 4; ++t) sc[n][t] *= ksc[t];
                }
                seen[n] = 0xffffu;
                if (!full) {
                    seen[n] = page_ok ? seen_bits<16>(key0, pos[n], low[n], a.sinks) : 0u;
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        sc[n][j / 4][j % 4] = (seen[n] >> j & 1u) ? sc[n][j / 4][j % 4] : -__builtin_inff();
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
                // values that are no numbers in a tile of which a row does not see all: a weight of 0
                // does not hide a NaN, so they leave the product and come back below
                uint32_t wild = 0;
                if (!full) {
#pragma unroll
                    for (int d = 0; d < DT; ++d) wild |= any_nonfinite(vr[d][0]) | any_nonfinite(vr[d][1]);
                }
                if (!full && __any(wild != 0)) {
                    wild_tiles = true;
#pragma unroll
                    for (int d = 0; d < DT; ++d) {
                        (void)take_nonfinite(vr[d][0]);
                        (void)take_nonfinite(vr[d][1]);
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

        if constexpr (!Q8) {
            if (wild_tiles) {  // of what each row sees of those values, counts, and what they make of its sum
                for (int i = begin + wid; i < end; i += 4) {
                    const int t0 = span.at(i) * kTileKeys, key0 = t0 + 16 * c;
                    look_up(i, id_k, id_v);
                    if (is_full(t0, id_v >= 0)) continue;
                    const uint8_t *src = static_cast<const uint8_t *>(a.vc) +
                                         (((size_t(max(id_v, 0)) * H + h) * D + col) * size_t(P) + size_t(key0 & (P - 1))) * 2;
                    h8 sb[NC][2];
#pragma unroll
                    for (int n = 0; n < NC; ++n) {
                        const uint32_t bits = id_v >= 0 ? seen_bits<16>(key0, pos[n], low[n], a.sinks) : 0u;
#pragma unroll
                        for (int j = 0; j < 16; ++j) sb[n][j / 8][j % 8] = _Float16(float(bits >> j & 1u));
                    }
#pragma unroll
                    for (int d = 0; d < DT; ++d) {
                        u4 w[2] = {reinterpret_cast<const u4 *>(src + size_t(d) * 32 * P)[0],
                                   reinterpret_cast<const u4 *>(src + size_t(d) * 32 * P)[1]};
                        const h8 code[2] = {__builtin_bit_cast(h8, take_nonfinite(w[0])), __builtin_bit_cast(h8, take_nonfinite(w[1]))};
#pragma unroll
                        for (int n = 0; n < NC; ++n) {
                            f4 cnt = {0.f, 0.f, 0.f, 0.f};
                            cnt = __builtin_amdgcn_mfma_f32_16x16x32_f16(code[0], sb[n][0], cnt, 0, 0, 0);
                            cnt = __builtin_amdgcn_mfma_f32_16x16x32_f16(code[1], sb[n][1], cnt, 0, 0, 0);
#pragma unroll
                            for (int r = 0; r < 4; ++r) acc[n][d][r] += nonfinite_sum(cnt[r]);
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
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

// maximum / sum over the two lane halves (lanes l, l ^ 32)
__device__ inline float halves_max(float v) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ inline float halves_sum(float v) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// Many rows: 128 of them a workgroup, 32 a wave, the columns of 32x32x16 MFMA.
// The tile's keys and values are staged through LDS (8-bit ones as fp16) and
// shared by the four waves; the next tile's loads are in flight meanwhile. A
// lane (half hh = lane / 32) holds scores of tokens 16u + 8 hh + 0..7, u < 4:
// result row i = 8a + 4 hh + r of a 32-token MFMA is given token 16 (a / 2) +
// 8 hh + 4 (a % 2) + r (bits 2 and 3 of i exchanged in the key operand's row),
// so the weights are the second product's operand as they stand. 16-B pieces of
// an LDS row are exchanged by an XOR with the row, so that 16 rows' equal pieces
// lie in 64 different banks.
template <int D, bool Q8>
__global__ __launch_bounds__(256, D <= 128 ? 2 : 1) void attn_tile_kernel(SplitArgs p) {
    constexpr int R = 128, KS = D / 16, DB = D / 32;
    constexpr int RK = D * 2;                       // bytes of a key's row in LDS
    constexpr int NL = Q8 ? D / 64 : D / 32;        // 16-B loads of a thread for its keys, and for its values
    __shared__ __attribute__((aligned(16))) uint8_t kbuf[2][64 * RK];
    __shared__ __attribute__((aligned(16))) uint8_t vbuf[2][D * 128];
    __shared__ float scales[2][2][64];              // 8-bit cache: of keys, of values
    __shared__ int wild;                            // a tile had values that are no numbers, hidden from some row

    const AttnArgs &a = p.a;
    const int H = a.b.n_heads, G = a.group;
    const int h = int(blockIdx.x) % H, s = int(blockIdx.x) / H, split = int(blockIdx.y);
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, hh = lane >> 5;
    const SeqView v = seq_view(a.b, s);
    if (v.n_new < p.new_min || v.n_new > p.new_max) return;
    const int64_t rows = int64_t(v.n_new) * G;
    const int P = 1 << a.b.page_shift, shift = a.b.page_shift;
    const int krow = (col & ~12) | ((col & 4) << 1) | ((col & 8) >> 1);  // the key this lane's operand row stands for
    auto k_at = [](int row, int ch) { return row * RK + ((ch ^ (D == 64 ? (row >> 1) & 7 : row & 15)) << 4); };
    auto v_at = [](int d, int ch) { return d * 128 + ((ch ^ ((d >> 1) & 7)) << 4); };

    // the last row tiles see most: they go first
    for (int64_t rt = int64_t(gridDim.z) - 1 - blockIdx.z; rt * R < rows; rt += gridDim.z) {
        const int64_t row0 = rt * R;
        const int nrows = int(rows - row0 < R ? rows - row0 : R);
        const int first = v.pos0 + int(row0 / G), last = v.pos0 + int((row0 + nrows - 1) / G);
        const TileSpan span = tile_span(first, last, a.window, a.sinks);
        const bool planned = rt < p.row_tiles;
        const int per = planned ? split_tiles(span.n, p.nsplit, p.chunk) : span.n;
        const int begin = split * per, end = min(begin + per, span.n);
        if (begin >= end && split > 0) continue;
        const bool direct = per >= span.n;

        const int wr = 32 * wid, wrows = min(nrows - wr, 32);  // this wave's rows of the tile (none: <= 0)
        const int64_t row = row0 + wr + (col < wrows ? col : 0);
        const int64_t safe = wrows > 0 ? row : row0;
        const int qi = int(safe / G), qg = int(safe % G), pos = v.pos0 + qi;
        const int pmin = v.pos0 + int((row0 + wr) / G), pmax = v.pos0 + int((row0 + wr + max(wrows, 1) - 1) / G);
        h8 q[KS];
        {
            const uint16_t *src = a.q + size_t(v.r0 + qi) * a.q_stride + size_t(h * G + qg) * D + 8 * hh;
#pragma unroll
            for (int k = 0; k < KS; ++k) q[k] = *reinterpret_cast<const h8 *>(src + 16 * k);
        }
        float m = -__builtin_inff(), l = 0.0f, vref = 1e-30f;
        f16v acc[DB];
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[d][r] = 0.0f;

        // staging: wave w loads the tile's keys 16w .. 16w + 15 (one page) and D / 4 of its values' rows
        u4 kr[NL], vr[NL];
        float sreg = 0.0f;
        const int vgroup = Q8 ? lane & 3 : (lane & 7) >> 1;  // the 16 tokens this lane loads values of
        int idk = -1, idv = -1;
        auto look_up = [&](int i, int &ik, int &iv) {
            const int t = span.at(i) * kTileKeys;
            ik = page_of(a.b, s, t + 16 * wid, v.len);
            iv = page_of(a.b, s, t + 16 * vgroup, v.len);
        };
        auto load = [&](int i, int ik, int iv) {
            const int t = span.at(i) * kTileKeys;
            const size_t kcell = ((size_t(max(ik, 0)) * H + h) << shift) + size_t((t + 16 * wid) & (P - 1));
            const uint8_t *ksrc = static_cast<const uint8_t *>(a.kc) + kcell * (Q8 ? D : 2 * D) + 16 * lane;
#pragma unroll
            for (int j = 0; j < NL; ++j) kr[j] = *reinterpret_cast<const u4 *>(ksrc + 1024 * j);
            const size_t hv = size_t(max(iv, 0)) * H + h;
            const int slot = (t + 16 * vgroup) & (P - 1);
            const int d0 = wid * (D / 4) + (Q8 ? lane >> 2 : lane >> 3);
            const uint8_t *vsrc = static_cast<const uint8_t *>(a.vc) + ((hv * D + d0) * size_t(P) + slot) * (Q8 ? 1 : 2) +
                                  (Q8 ? 0 : 16 * (lane & 1));
#pragma unroll
            for (int j = 0; j < NL; ++j) vr[j] = *reinterpret_cast<const u4 *>(vsrc + size_t(j) * (Q8 ? 16 : 8 * 2) * P);
            if constexpr (Q8) {
                if (lane < 32) sreg = (lane < 16 ? a.ks : a.vs)[kcell + (lane & 15)];
            }
        };
        const int low = a.window > 0 ? max(pos - a.window, -1) : -1;  // the last token the row's window hides
        // a tile of which some row of the workgroup does not see some cell
        auto partial = [&](int i, unsigned ok) {
            const int t = span.at(i) * kTileKeys;
            return ok != 15 || t + kTileKeys - 1 > first ||
                   (a.window > 0 && t <= last - a.window && t + kTileKeys > a.sinks);
        };
        auto store = [&](int i, int b, unsigned ok) {
            if constexpr (!Q8) {
                if (partial(i, ok)) {
                    uint32_t w = 0;
#pragma unroll
                    for (int j = 0; j < NL; ++j) w |= any_nonfinite(vr[j]);
                    if (__any(w != 0)) {  // (a weight of 0 does not hide a NaN: out of the product, and back below)
                        wild = 1;
#pragma unroll
                        for (int j = 0; j < NL; ++j) (void)take_nonfinite(vr[j]);
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < NL; ++j) {
                const int u = 64 * j + lane;
                if constexpr (Q8) {
                    const int r = 16 * wid + u / (D / 16), ch = u % (D / 16) * 2;
                    *reinterpret_cast<h8 *>(&kbuf[b][k_at(r, ch)]) = codes8(kr[j][0], kr[j][1]);
                    *reinterpret_cast<h8 *>(&kbuf[b][k_at(r, ch + 1)]) = codes8(kr[j][2], kr[j][3]);
                    const int d = wid * (D / 4) + 16 * j + (lane >> 2), c = 2 * (lane & 3);
                    *reinterpret_cast<h8 *>(&vbuf[b][v_at(d, c)]) = codes8(vr[j][0], vr[j][1]);
                    *reinterpret_cast<h8 *>(&vbuf[b][v_at(d, c + 1)]) = codes8(vr[j][2], vr[j][3]);
                } else {
                    *reinterpret_cast<u4 *>(&kbuf[b][k_at(16 * wid + u / (D / 8), u % (D / 8))]) = kr[j];
                    *reinterpret_cast<u4 *>(&vbuf[b][v_at(wid * (D / 4) + 8 * j + (lane >> 3), lane & 7)]) = vr[j];
                }
            }
            if constexpr (Q8) {
                if (lane < 32) scales[b][lane >> 4][16 * wid + (lane & 15)] = sreg;
            }
        };
        // which of the tile's four groups of 16 tokens have a page
        auto groups = [&](int iv) {
            const uint64_t bal = __ballot(iv >= 0);
            return Q8 ? unsigned(bal & 15) : unsigned((bal & 1) | (bal >> 1 & 2) | (bal >> 2 & 4) | (bal >> 3 & 8));
        };
        unsigned ok = 0, ok_next = 0;
        int nk = -1, nv = -1;
        if (threadIdx.x == 0) wild = 0;
        __syncthreads();
        if (begin < end) {
            look_up(begin, idk, idv);
            ok = groups(idv);
            load(begin, idk, idv);
            if (begin + 1 < end) look_up(begin + 1, nk, nv);
            store(begin, 0, ok);
        }
        for (int i = begin; i < end; ++i) {
            const int b = (i - begin) & 1;
            __syncthreads();
            if (i + 1 < end) {
                ok_next = groups(nv);
                load(i + 1, nk, nv);
                if (i + 2 < end) look_up(i + 2, nk, nv);
            }
            __builtin_amdgcn_sched_barrier(0);
            const int t0 = span.at(i) * kTileKeys;
            // (a tile that none of this wave's rows sees)
            const bool none = wrows <= 0 || t0 > pmax ||
                              (a.window > 0 && t0 + kTileKeys - 1 <= pmin - a.window && t0 >= a.sinks);
            if (!none) {
                f16v sc[2];
#pragma unroll
                for (int n = 0; n < 2; ++n) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) sc[n][r] = 0.0f;
#pragma unroll
                    for (int k = 0; k < KS; ++k) {
                        const h8 kk = *reinterpret_cast<const h8 *>(&kbuf[b][k_at(32 * n + krow, 2 * k + hh)]);
                        sc[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kk, q[k], sc[n], 0, 0, 0);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
                // the lane's scores: token t0 + 16 u + 8 hh + j is sc[u / 2][8 (u % 2) + j]
                float vsc[Q8 ? 32 : 1];
                if constexpr (Q8) {
#pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        const int at = 16 * (x / 2) + 8 * hh + 4 * (x % 2);
                        const f4 kx = *reinterpret_cast<const f4 *>(&scales[b][0][at]);
                        const f4 vx = *reinterpret_cast<const f4 *>(&scales[b][1][at]);
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            sc[x / 4][4 * (x % 4) + r] *= kx[r];
                            vsc[4 * x + r] = vx[r];
                        }
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
                    for (int j = 0; j < 32; ++j) sc[j / 16][j % 16] = (seen >> j & 1u) ? sc[j / 16][j % 16] : -__builtin_inff();
                }
                float top = sc[0][0];
#pragma unroll
                for (int j = 1; j < 32; ++j) top = fmaxf(top, sc[j / 16][j % 16]);
                const float mn = fmaxf(m, halves_max(top) * p.sl2);
                const float ms = mn == -__builtin_inff() ? 0.0f : mn;
                const float lscale = __builtin_amdgcn_exp2f(m - ms);
                float alpha = lscale, vinv = 1.0f;
                if constexpr (Q8) {
                    float big = vref;
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        const float x = fabsf(vsc[j]);
                        big = fmaxf(big, (seen >> j & 1u) && x < __builtin_inff() ? x : 0.0f);
                    }
                    big = halves_max(big);
                    alpha *= vref / big;
                    vref = big;
                    vinv = 1.0f / big;
                }
                m = mn;
                float sum = 0.0f;
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[j / 16][j % 16], p.sl2, -ms));
                    sum += e;
                    sc[j / 16][j % 16] = e;
                }
                l = l * lscale + sum;
                if (!__all(alpha == 1.0f)) {
#pragma unroll
                    for (int d = 0; d < DB; ++d) acc[d] *= alpha;
                }
                if constexpr (Q8) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        const float w = sc[j / 16][j % 16] * (vsc[j] * vinv);
                        sc[j / 16][j % 16] = (seen >> j & 1u) ? w : 0.0f;
                    }
                }
                h8 pb[4];
#pragma unroll
                for (int j = 0; j < 32; ++j) pb[j / 8][j % 8] = _Float16(sc[j / 16][j % 16]);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int d = 0; d < DB; ++d) {
                        const h8 vv = *reinterpret_cast<const h8 *>(&vbuf[b][v_at(32 * d + col, 2 * u + hh)]);
                        acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vv, pb[u], acc[d], 0, 0, 0);
                    }
            }
            __builtin_amdgcn_sched_barrier(0);
            if (i + 1 < end) {
                store(i + 1, 1 - b, ok_next);
                ok = ok_next;
            }
        }

        if constexpr (!Q8) {
            __syncthreads();
            if (wild) {  // of what each row sees of those values, counts, and what they make of its sum
                for (int i = begin; i < end; ++i) {
                    const int t0 = span.at(i) * kTileKeys;
                    look_up(i, idk, idv);
                    if (!partial(i, groups(idv))) continue;
#pragma unroll
                    for (int d = 0; d < DB; ++d) {
                        f16v cnt;
#pragma unroll
                        for (int r = 0; r < 16; ++r) cnt[r] = 0.0f;
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            const int key = t0 + 16 * u + 8 * hh, id = page_of(a.b, s, t0 + 16 * u, v.len);
                            const uint8_t *src = static_cast<const uint8_t *>(a.vc) +
                                (((size_t(max(id, 0)) * H + h) * D + 32 * d + col) * size_t(P) + size_t(key & (P - 1))) * 2;
                            u4 w = *reinterpret_cast<const u4 *>(src);
                            const uint32_t bits = id >= 0 ? seen_bits<8>(key, pos, low, a.sinks) : 0u;
                            h8 sb;
#pragma unroll
                            for (int j = 0; j < 8; ++j) sb[j] = _Float16(float(bits >> j & 1u));
                            cnt = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, take_nonfinite(w)), sb, cnt, 0, 0, 0);
                            __builtin_amdgcn_sched_barrier(0);
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
            const float unit = Q8 ? vref : 1.0f;
            if (!direct) {
                const size_t slot = (((size_t(s) * H + h) * size_t(p.nsplit) + size_t(split)) * size_t(p.row_tiles)) * R + size_t(row);
                if (hh == 0) p.part_ml[slot] = make_float2(m, total);
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        *reinterpret_cast<f4 *>(p.part_o + slot * D + 32 * d + 8 * x + 4 * hh) =
                            f4{acc[d][4 * x], acc[d][4 * x + 1], acc[d][4 * x + 2], acc[d][4 * x + 3]} * unit;
            } else {
                const float inv = (total > 0.0f || total != total ? 1.0f / total : 0.0f) * unit;
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
    if (v.n_new < p.new_min || v.n_new > p.new_max) return;
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

// How a call's sequences are launched: those of up to `few` new tokens (64 rows)
// by the split kernel, longer ones by the tile kernel.
struct SplitPlan {
    int nc, row_tiles, nsplit, chunk;  // nc: columns / 16 of the split kernel, 8: the tile kernel
    int new_min, new_max;
    size_t slots, bytes;
    int rows() const { return 16 * nc; }
};

int few_tokens(const AttnArgs &a) {
    const int most = a.head_dim > 128 ? 16 : 64;
    return a.group > most ? 1 : most / a.group;
}

// nc 0: as the rows ask. max_new: the most new tokens of the sequences it is for.
SplitPlan plan_split(const AttnArgs &a, int nc, int max_new, int cu_count, size_t scratch) {
    SplitPlan p{};
    const int64_t rows = int64_t(max_new) * a.group;
    p.nc = nc ? nc : rows <= 16 || a.head_dim > 128 ? 1 : rows <= 32 ? 2 : 4;
    const int R = p.rows();
    const int64_t rt = (rows + R - 1) / R;
    p.row_tiles = int(rt < 65535 ? rt : 65535);
    int tiles = (a.max_kv - 1) / kTileKeys + 1;
    if (a.window > 0) {
        const int64_t most = (int64_t(a.window) + R / a.group + 1) / kTileKeys + (int64_t(a.sinks) + kTileKeys - 1) / kTileKeys + 3;
        if (most < tiles) tiles = int(most);
    }
    const int64_t units = int64_t(a.b.n_seqs) * a.b.n_heads * p.row_tiles;
    const int64_t aim = int64_t(cu_count) * (p.nc == 8 ? 2 : 4);  // workgroups
    int64_t n = (aim + units - 1) / units;
    const int64_t most = p.nc == 8 ? (tiles + 3) / 4 : (tiles + 3) / 4;  // a tile for each wave at least
    if (n > most) n = most;
    const size_t slot = size_t(a.b.n_seqs) * a.b.n_heads * p.row_tiles * R;
    const size_t slot_bytes = slot * (size_t(a.head_dim) * 4 + 8);
    if (n > 1 && size_t(n) > scratch / slot_bytes) n = int64_t(scratch / slot_bytes);
    if (n < 1) n = 1;
    p.chunk = int((tiles + n - 1) / n);
    p.nsplit = (tiles + p.chunk - 1) / p.chunk;
    p.slots = slot * size_t(p.nsplit);
    p.bytes = p.nsplit > 1 ? slot_bytes * size_t(p.nsplit) : 0;
    p.new_min = 0;
    p.new_max = 0x7fffffff;
    return p;
}

// one or two plans; the number of them
int plan_call(const AttnArgs &a, int cu_count, size_t scratch, SplitPlan out[2]) {
    const int few = few_tokens(a);
    if (a.max_new <= few) {
        out[0] = plan_split(a, 0, a.max_new, cu_count, scratch);
        return 1;
    }
    out[0] = plan_split(a, 8, a.max_new, cu_count, scratch);
    // one sequence, or all of the same many rows: nothing is left for the split kernel
    if (a.b.n_seqs == 1 || int64_t(a.b.n_seqs) * a.max_new <= a.b.n_rows) return 1;
    out[0].new_min = few + 1;
    out[1] = plan_split(a, 0, few, cu_count, scratch - out[0].bytes);
    out[1].new_max = few;
    return 2;
}

template <int D, int NC, bool Q8> void launch_split(const SplitArgs &p, dim3 grid, hipStream_t s) {
    hipLaunchKernelGGL((attn_split_kernel<D, NC, Q8>), grid, dim3(256), 0, s, p);
}
template <int D> hipError_t launch_split_d(const SplitArgs &p, int nc, bool q8, dim3 grid, hipStream_t s) {
    if (nc == 8) {
        if (q8) hipLaunchKernelGGL((attn_tile_kernel<D, true>), grid, dim3(256), 0, s, p);
        else hipLaunchKernelGGL((attn_tile_kernel<D, false>), grid, dim3(256), 0, s, p);
    } else if (nc == 1) q8 ? launch_split<D, 1, true>(p, grid, s) : launch_split<D, 1, false>(p, grid, s);
    else if constexpr (D <= 128) {
        if (nc == 2) q8 ? launch_split<D, 2, true>(p, grid, s) : launch_split<D, 2, false>(p, grid, s);
        else q8 ? launch_split<D, 4, true>(p, grid, s) : launch_split<D, 4, false>(p, grid, s);
    }
    return hipGetLastError();
}

}  // namespace

size_t attn_scratch_bytes(const AttnArgs &a, int cu_count) {
    SplitPlan pl[2];
    size_t n = 0;
    for (int i = plan_call(a, cu_count, ~size_t(0), pl); i-- > 0;) n += pl[i].bytes;
    return n;
}

hipError_t launch_attention(const AttnArgs &a, void *scratch, size_t scratch_bytes, int cu_count, hipStream_t s) {
    SplitPlan plans[2];
    const int n = plan_call(a, cu_count, scratch ? scratch_bytes : 0, plans);
    uint8_t *base = static_cast<uint8_t *>(scratch);
    for (int i = 0; i < n; ++i) {
        const SplitPlan &pl = plans[i];
        SplitArgs p;
        p.a = a;
        p.sl2 = a.scale * 1.44269504088896341f;
        p.nsplit = pl.nsplit;
        p.chunk = pl.chunk;
        p.row_tiles = pl.row_tiles;
        p.new_min = pl.new_min;
        p.new_max = pl.new_max;
        p.part_o = reinterpret_cast<float *>(base);
        p.part_ml = pl.nsplit > 1 ? reinterpret_cast<float2 *>(p.part_o + pl.slots * size_t(a.head_dim)) : nullptr;
        if (base) base += pl.bytes;
        const dim3 grid(unsigned(a.b.n_seqs) * unsigned(a.b.n_heads), unsigned(pl.nsplit), unsigned(pl.row_tiles));
        const bool q8 = a.ks != nullptr;
        const hipError_t e = a.head_dim == 64    ? launch_split_d<64>(p, pl.nc, q8, grid, s)
                             : a.head_dim == 128 ? launch_split_d<128>(p, pl.nc, q8, grid, s)
                                                 : launch_split_d<256>(p, pl.nc, q8, grid, s);
        if (e != hipSuccess) return e;
        if (pl.nsplit == 1) continue;
        const int64_t rows = int64_t(pl.row_tiles) * pl.rows();
        const dim3 jg(grid.x, unsigned(rows < 65535 ? rows : 65535));
        if (a.head_dim == 64) hipLaunchKernelGGL(attn_join_kernel<64>, jg, dim3(256), 0, s, p, pl.rows());
        else if (a.head_dim == 128) hipLaunchKernelGGL(attn_join_kernel<128>, jg, dim3(256), 0, s, p, pl.rows());
        else hipLaunchKernelGGL(attn_join_kernel<256>, jg, dim3(256), 0, s, p, pl.rows());
        const hipError_t ej = hipGetLastError();
        if (ej != hipSuccess) return ej;
    }
    return hipSuccess;
}

}  // namespace qmm
