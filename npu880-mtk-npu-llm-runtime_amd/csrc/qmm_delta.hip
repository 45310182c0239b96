// qmm_delta.hip — the gated delta rule.
//
// Every token of a head, in order, on its state S [DK][DV]:
//   S <- e^g S;  d = beta (v - S' k);  S <- S + k d';  o = S' q
// with k and q of unit length. The columns of S are independent of each other.
#include <hip/hip_runtime.h>

#include "qmm_lanes.h"
#include "qmm_state.h"

namespace qmm {
namespace {

constexpr int kStepRows = 24;  // new rows up to which a token at a time is faster
constexpr int kGroup = 8;  // tokens whose inputs are in LDS at a time

__device__ inline float softplus(float x) { return x > 0.0f ? x + log1pf(expf(-x)) : log1pf(expf(x)); }
__device__ inline float log_decay(const DeltaArgs &a, int row, int h) {
    return fminf(a.rate[h] * softplus(a.a[size_t(row) * a.a_stride + h] + a.dt_bias[h]), 0.0f);
}
__device__ inline float step_size(const DeltaArgs &a, int row, int h) {
    return 1.0f / (1.0f + expf(-a.beta[size_t(row) * a.b_stride + h]));
}

__device__ inline float4 load4(const float *p) { return *reinterpret_cast<const float4 *>(p); }
__device__ inline float dot4(float4 x, float4 y) { return x.x * y.x + x.y * y.y + (x.z * y.z + x.w * y.w); }

// One token after another through the state, for few new rows: a workgroup per
// sequence and head, a wave 16 * CL / 4 columns (4 a lane) of all rows, in
// registers; a lane has rows 4 (rl + RL g) .. + 3. Both products with S are taken
// before it changes: S' q after the step is e^g S' q + (k.q) d, so one pass and one
// sum over the lanes serve both, and no wave waits for another between tokens.
template <int DK, int DV>
__global__ __launch_bounds__(256, 3) void delta_step_kernel(DeltaArgs a) {
    constexpr int CL = DV / 16, RL = 64 / CL, NG = DK / (4 * RL), NV = (kGroup * DV + 1023) / 1024, HL = 32;  // HL: lanes that hold one row of q or k
    __shared__ float qk[kGroup][2][DK];
    __shared__ float vo[kGroup][DV];  // values, then outputs
    __shared__ float sc[kGroup][4];   // decay, beta, k.q
    const int t = threadIdx.x, lane = t & 63, wid = __builtin_amdgcn_readfirstlane(t >> 6);
    const int s = int(blockIdx.x / unsigned(a.v_heads)), h = int(blockIdx.x % unsigned(a.v_heads));
    const int hk = h / (a.v_heads / a.qk_heads);
    const StateSeq v = state_seq(a.b, s);
    const int cl = lane % CL, rl = lane / CL, col = wid * (DV / 4) + 4 * cl;
    const int sub = lane % HL, is_k = lane / HL;
    const float *src = (is_k ? a.k : a.q) + size_t(hk) * DK + 4 * sub;
    const size_t src_stride = is_k ? a.k_stride : a.q_stride;
    const size_t place = size_t(h) * DK * DV + col;
    const size_t pool = size_t(a.v_heads) * DK * DV;

    float4 x[kGroup / 4], val[NV];
    auto load = [&](int t0) {
#pragma unroll
        for (int i = 0; i < kGroup / 4; ++i) {
            const int m = t0 + 4 * i + wid;
            x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (m < v.n && 4 * sub < DK) x[i] = load4(src + size_t(v.r0 + m) * src_stride);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int e = i * 1024 + 4 * t, m = t0 + e / DV;
            val[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (m < v.n && e < kGroup * DV) val[i] = load4(a.v + size_t(v.r0 + m) * a.v_stride + size_t(h) * DV + e % DV);
        }
    };
    if (v.n > 0) load(0);
    float4 S[NG][4];
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            S[g][j] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (v.in >= 0) S[g][j] = load4(a.state + size_t(v.in) * pool + place + size_t(4 * (rl + RL * g) + j) * DV);
        }
    for (int t0 = 0; t0 < v.n; t0 += kGroup) {
        const int nt = min(kGroup, v.n - t0);
        if (t < nt) {
            sc[t][0] = expf(log_decay(a, v.r0 + t0 + t, h));
            sc[t][1] = step_size(a, v.r0 + t0 + t, h);
        }
#pragma unroll
        for (int i = 0; i < kGroup / 4; ++i) {
            if (4 * i + wid >= nt) break;
            const float r = inv_root(lanes_sum<HL>(dot4(x[i], x[i])) + a.qk_eps) * (is_k ? 1.0f : a.scale);
            const float4 y = make_float4(x[i].x * r, x[i].y * r, x[i].z * r, x[i].w * r);
            if (4 * sub < DK) *reinterpret_cast<float4 *>(&qk[4 * i + wid][is_k][4 * sub]) = y;
            const float4 z = make_float4(__shfl_xor(y.x, 32), __shfl_xor(y.y, 32), __shfl_xor(y.z, 32), __shfl_xor(y.w, 32));
            const float kq = lanes_sum<HL>(dot4(y, z));
            if (lane == 0) sc[4 * i + wid][2] = kq;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (i * 1024 + 4 * t < kGroup * DV) *reinterpret_cast<float4 *>(&vo[0][0] + i * 1024 + 4 * t) = val[i];
        __syncthreads();
        if (t0 + kGroup < v.n) load(t0 + kGroup);
        for (int m = 0; m < nt; ++m) {
            const float decay = sc[m][0], beta = sc[m][1], kq = sc[m][2];
            const float4 val = load4(&vo[m][col]);
            float4 kr[NG];
            float ks[4] = {}, qs[4] = {};
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                kr[g] = load4(&qk[m][1][4 * (rl + RL * g)]);
                const float4 qr = load4(&qk[m][0][4 * (rl + RL * g)]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float kj = reinterpret_cast<const float *>(&kr[g])[j], qj = reinterpret_cast<const float *>(&qr)[j];
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const float sv = reinterpret_cast<const float *>(&S[g][j])[c];
                        ks[c] = __builtin_fmaf(kj, sv, ks[c]);
                        qs[c] = __builtin_fmaf(qj, sv, qs[c]);
                    }
                }
            }
            float d[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float old = columns_sum<CL>(ks[c]) * decay;
                d[c] = beta * (reinterpret_cast<const float *>(&val)[c] - old);
                qs[c] = __builtin_fmaf(kq, d[c], columns_sum<CL>(qs[c]) * decay);
            }
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        float &sv = reinterpret_cast<float *>(&S[g][j])[c];
                        sv = __builtin_fmaf(reinterpret_cast<const float *>(&kr[g])[j], d[c], sv * decay);
                    }
            if (rl == 0) *reinterpret_cast<float4 *>(&vo[m][col]) = make_float4(qs[0], qs[1], qs[2], qs[3]);
        }
        __syncthreads();
        // rows out: half a wave each, with the norm and the gate
        for (int m = 2 * wid + lane / HL; m < nt; m += 8) {
            const bool on = 4 * sub < DV;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
            if (on) o = load4(&vo[m][4 * sub]);
            const size_t row = size_t(v.r0 + t0 + m);
            if (a.gamma) {
                const float r = inv_root(lanes_sum<HL>(dot4(o, o)) * (1.0f / DV) + a.gamma_eps);
                if (on) {
                    const float4 w = load4(a.gamma + 4 * sub);
                    o = make_float4(o.x * r * w.x, o.y * r * w.y, o.z * r * w.z, o.w * r * w.w);
                }
            }
            if (on && a.z) {
                const float4 z = load4(a.z + row * a.z_stride + size_t(h) * DV + 4 * sub);
                o = make_float4(o.x * silu(z.x), o.y * silu(z.y), o.z * silu(z.z), o.w * silu(z.w));
            }
            if (on) *reinterpret_cast<float4 *>(a.out + row * a.out_stride + size_t(h) * DV + 4 * sub) = o;
        }
        __syncthreads();
    }
    if (v.out >= 0) {
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *reinterpret_cast<float4 *>(a.state + size_t(v.out) * pool + place + size_t(4 * (rl + RL * g) + j) * DV) = S[g][j];
    }
}

// ------------------------------------------------------------- prompts
// Of a group of up to 32 tokens, with G_i the sum of its log decays up to token i, k and q its unit rows and
// S the state before it:
//   A_ij = beta_i e^(G_i - G_j) k_i.k_j  (j < i),   T = (I + A)^-1,   P_ij = e^(G_i - G_j) q_i.k_j  (j <= i)
//   D = (T diag(beta)) (V - diag(e^G) K S),   O = diag(e^G) Q S + P D,   S <- e^(G_last) S + K' diag(e^(G_last - G)) D
// The first kernel makes T diag(beta) and P of every group at once; the second walks a
// sequence's groups. All products but the inverse run on the matrix units in fp16, each operand as a
// pair hi + lo of 22 bits (three products: hi hi, hi lo, lo hi), sums in fp32. K, Q, T diag(beta) and P are at
// most 1 in size and kept 2^4 times as large, so that their low parts are no subnormals; the scale of S, D
// and V is a power of two for each column, from a bound of the column that holds for the group
// (|S column| grows by |v| at most, as a step makes no column longer).
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));

// An operand of 16 rows and 32 columns k in LDS: lane (row r, group g of lanes) reads 16 B at 272 g + 16 r: columns
// 4 g .. + 3 and 16 + 4 g .. + 3. That is the order in which a group of lanes holds the rows of two tiles of
// a product, so a product's result is the next product's right operand as it stands. (272, not 256: pieces of
// 8 B of four columns then lie on all banks when they are written.)
constexpr int kBlock = 4 * 272;
__device__ inline int operand_at(int row, int col) {  // of the aligned 4 columns from `col` (of 32)
    return (col % 16 / 4) * 272 + (row % 16) * 16 + col / 16 * 8;
}
__device__ inline f4 mfma(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
// x = hi + lo + at most 2^-22 |x| (and 2^-25)
__device__ inline void split4(f4 x, h4 &hi, h4 &lo) {
    hi = __builtin_convertvector(x, h4);
    f4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __builtin_fmaf(float(hi[i]), -1.0f, x[i]);
    lo = __builtin_convertvector(r, h4);
}
struct Pair {
    h8 hi, lo;
};
__device__ inline Pair split(f4 x, f4 y) {
    h4 a, b, c, d;
    split4(x, a, b);
    split4(y, c, d);
    return Pair{__builtin_shufflevector(a, c, 0, 1, 2, 3, 4, 5, 6, 7), __builtin_shufflevector(b, d, 0, 1, 2, 3, 4, 5, 6, 7)};
}
__device__ inline Pair operand(const char *p) {  // p: this lane's place in the block of the high parts; the low parts follow
    return Pair{*reinterpret_cast<const h8 *>(p), *reinterpret_cast<const h8 *>(p + kBlock)};
}
__device__ inline f4 product(const Pair &a, const Pair &b, f4 c) { return mfma(a.lo, b.hi, mfma(a.hi, b.lo, mfma(a.hi, b.hi, c))); }

struct DeltaScratch {
    char *matrices;  // [groups][v_heads]: T diag(beta), then P: two tiles of 16 rows, each 1 KB hi and 1 KB lo
    float *decays;   // [groups][v_heads][64]: e^G_i, e^(G_last - G_i)
    float *inverse;  // [groups][qk_heads][64]: 1 / |k_i|, 1 / |q_i|
};
__device__ inline int64_t first_group(const StateSeq &v, int s) { return v.r0 / kChunk + s; }

// 4 tokens x 4 values of q or k for item `i` of a group's 2 * 8 * DK / 4: eight lanes side by side take 128 B
template <int DK> struct Item {
    int is_q, token, at;
    __device__ explicit Item(int i) {
        constexpr int kAll = 8 * DK / 4;
        is_q = i / kAll;
        const int r = i % kAll;
        token = r / 8 % 8 * 4;
        at = (r / 64 * 8 + r % 8) * 4;
    }
    __device__ void load(const DeltaArgs &a, int hk, int r0, int left, float4 x[4]) const {
        const float *src = (is_q ? a.q : a.k) + size_t(hk) * DK + at;
        const size_t stride = is_q ? a.q_stride : a.k_stride;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[j] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (token + j < left) x[j] = load4(src + size_t(r0 + token + j) * stride);
        }
    }
    // as left operand, rows the tokens: tiles of 16 tokens, each DK / 32 blocks of hi and lo
    __device__ void store(char *base, const float4 x[4], const float *inv) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float f = inv[j] * 16.0f;
            h4 hi, lo;
            split4(f4{x[j].x * f, x[j].y * f, x[j].z * f, x[j].w * f}, hi, lo);
            char *p = base + ((token / 16) * (DK / 32) + at / 32) * 2 * kBlock + operand_at(token + j, at % 32);
            *reinterpret_cast<h4 *>(p) = hi;
            *reinterpret_cast<h4 *>(p + kBlock) = lo;
        }
    }
    // as left operand, rows the values: tiles of 16 values, each one block of hi and lo
    __device__ void store_turned(char *base, const float4 x[4], const float *inv) const {
        f4 y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float f = inv[j] * 16.0f;
            y[0][j] = x[j].x * f;
            y[1][j] = x[j].y * f;
            y[2][j] = x[j].z * f;
            y[3][j] = x[j].w * f;
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            h4 hi, lo;
            split4(y[c], hi, lo);
            char *p = base + (at / 16) * 2 * kBlock + operand_at(at + c, token);
            *reinterpret_cast<h4 *>(p) = hi;
            *reinterpret_cast<h4 *>(p + kBlock) = lo;
        }
    }
};

__device__ inline double shfl_up(double x, int d) {
    const uint64_t u = __double_as_longlong(x);
    return __longlong_as_double((uint64_t(uint32_t(__shfl_up(int(u >> 32), d, 32))) << 32) | uint32_t(__shfl_up(int(u), d, 32)));
}

// T diag(beta) and P of one group and key head, for its value heads two at a time. The inverse of the unit
// lower triangle: two 16 x 16 triangles a head by substitution, a column per lane (both heads in one wave), then
// T21 = -T22 A21 T11 on the matrix units in fp32.
template <int DK>
__global__ __launch_bounds__(256) void delta_prepare_kernel(DeltaArgs a, DeltaScratch w, int tiles) {
    constexpr int NU = DK / 32, NI = DK / 64, kRow = 36;
    __shared__ __attribute__((aligned(16))) char rows[2][2 * NU * 2 * kBlock];  // k and q as operands
    __shared__ float sums[2][32][NU];
    __shared__ float inv[2][32];
    __shared__ float kk[32][kRow], qk[32][kRow];
    __shared__ float A[2][32][kRow], T[2][32][kRow];
    __shared__ double G[2][32];
    __shared__ float beta[2][32];
    const int t = threadIdx.x, lane = t & 63, wid = __builtin_amdgcn_readfirstlane(t >> 6);
    const int hk = int(blockIdx.x % unsigned(a.qk_heads)), st = int(blockIdx.x / unsigned(a.qk_heads));
    const int s = st / tiles, of = a.v_heads / a.qk_heads;
    const StateSeq v = state_seq(a.b, s);
    for (int tile = st % tiles; int64_t(tile) * kChunk < v.n; tile += tiles) {
        const int r0 = v.r0 + tile * kChunk, left = v.n - tile * kChunk;
        const size_t group = size_t(first_group(v, s) + tile);
        float4 x[NI][4];
#pragma unroll
        for (int i = 0; i < NI; ++i) Item<DK>(t + 256 * i).load(a, hk, r0, left, x[i]);
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const Item<DK> it(t + 256 * i);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float ss = dot4(x[i][j], x[i][j]);  // over the eight lanes that share a token
                ss += lane_moved<0xB1>(ss);
                ss += lane_moved<0x4E>(ss);
                ss += lane_moved<0x141>(ss);
                if (lane % 8 == 0) sums[it.is_q][it.token + j][it.at / 32] = ss;
            }
        }
        __syncthreads();
        if (t < 64) {
            float ss = a.qk_eps;
#pragma unroll
            for (int u = 0; u < NU; ++u) ss += sums[t / 32][t % 32][u];
            const float r = inv_root(ss);
            inv[t / 32][t % 32] = r;
            w.inverse[(group * a.qk_heads + hk) * 64 + t] = r;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const Item<DK> it(t + 256 * i);
            it.store(rows[it.is_q], x[i], &inv[it.is_q][it.token]);
        }
        __syncthreads();
        for (int task = wid; task < 6; task += 4) {  // k k' and q k', the tiles on and below the diagonal
            const int is_q = task / 3, ti = task % 3 != 0, tj = task % 3 == 2;
            const int at = (lane / 16) * 272 + (lane % 16) * 16;
            f4 c{};
#pragma unroll
            for (int u = 0; u < NU; ++u)
                c = product(operand(rows[is_q] + (ti * NU + u) * 2 * kBlock + at), operand(rows[0] + (tj * NU + u) * 2 * kBlock + at), c);
            float(*to)[kRow] = is_q ? qk : kk;
#pragma unroll
            for (int r = 0; r < 4; ++r) to[16 * ti + 4 * (lane / 16) + r][16 * tj + lane % 16] = c[r] * 0x1p-8f;
        }
        for (int h0 = 0; h0 < of; h0 += 2) {
            const int nh = min(2, of - h0);
            if (wid == 0) {  // a head in half a wave, a token per lane
                const int hh = lane / 32, m = lane % 32, h = hk * of + h0 + hh;
                const bool on = hh < nh && m < left;
                double g = on ? double(log_decay(a, r0 + m, h)) : 0.0;
#pragma unroll
                for (int d = 1; d < 32; d *= 2) {
                    const double o = shfl_up(g, d);
                    if (m >= d) g += o;
                }
                G[hh][m] = g;
                beta[hh][m] = on ? step_size(a, r0 + m, h) : 0.0f;
            }
            __syncthreads();
            if (t < 64 * nh) {
                const int hh = t / 64, m = t % 32;
                w.decays[(group * a.v_heads + hk * of + h0 + hh) * 64 + t % 64] = expf(float(t % 64 < 32 ? G[hh][m] : G[hh][31] - G[hh][m]));
            }
            const int i = t / 8, c = t % 8 * 4;  // row i, columns c .. c + 3
            for (int hh = 0; hh < nh; ++hh) {
                f4 p;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float e = c + j <= i ? expf(float(G[hh][i] - G[hh][c + j])) : 0.0f;
                    A[hh][i][c + j] = c + j < i ? beta[hh][i] * e * kk[i][c + j] : 0.0f;
                    p[j] = c + j <= i ? e * qk[i][c + j] * 16.0f : 0.0f;  // (above the diagonal's tiles nothing was written)
                }
                h4 hi, lo;
                split4(p, hi, lo);
                char *to = w.matrices + (group * a.v_heads + hk * of + h0 + hh) * kDeltaMatrices + 4096 + i / 16 * 2048 + (c % 16 / 4) * 256 + i % 16 * 16 + c / 16 * 8;
                *reinterpret_cast<h4 *>(to) = hi;
                *reinterpret_cast<h4 *>(to + 1024) = lo;
            }
            __syncthreads();
            if (wid == 0 && lane / 32 < nh) {
                const int hh = lane / 32, b = lane / 16 % 2 * 16, col = lane % 16;
                float x[16];
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    float y = r == col ? 1.0f : 0.0f;
#pragma unroll
                    for (int j = 0; j < r; ++j) y = __builtin_fmaf(-A[hh][b + r][b + j], x[j], y);
                    x[r] = y;
                    T[hh][b + r][b + col] = y;
                }
            }
            __syncthreads();
            if (wid < nh) {
                const int g = lane / 16, col = lane % 16;
                f4 y{}, z{};
#pragma unroll
                for (int k = 0; k < 16; k += 4) y = __builtin_amdgcn_mfma_f32_16x16x4f32(A[wid][16 + col][k + g], T[wid][k + g][col], y, 0, 0, 0);
#pragma unroll
                for (int r = 0; r < 4; ++r) z = __builtin_amdgcn_mfma_f32_16x16x4f32(T[wid][16 + col][16 + 4 * g + r], y[r], z, 0, 0, 0);
#pragma unroll
                for (int r = 0; r < 4; ++r) T[wid][16 + 4 * g + r][col] = -z[r];
            }
            __syncthreads();
            for (int hh = 0; hh < nh; ++hh) {
                f4 p;
#pragma unroll
                for (int j = 0; j < 4; ++j) p[j] = c / 16 <= i / 16 ? T[hh][i][c + j] * beta[hh][c + j] * 16.0f : 0.0f;
                h4 hi, lo;
                split4(p, hi, lo);
                char *to = w.matrices + (group * a.v_heads + hk * of + h0 + hh) * kDeltaMatrices + i / 16 * 2048 + (c % 16 / 4) * 256 + i % 16 * 16 + c / 16 * 8;
                *reinterpret_cast<h4 *>(to) = hi;
                *reinterpret_cast<h4 *>(to + 1024) = lo;
            }
            __syncthreads();
        }
        __syncthreads();
    }
}

__device__ inline float two_to(int e) { return __uint_as_float(uint32_t(e + 127) << 23); }
// the power of two that takes numbers up to `bound` below 2^15; within 2^-60 .. 2^60, so that two of them
// have a quotient in fp32 (columns below 2^-46 lose bits under 2^-85)
__device__ inline int scale_for(float bound) { return min(max(141 - int(__float_as_uint(bound) >> 23 & 255), -60), 60); }
__device__ inline float over_groups(float x) {  // sum over the four lanes of a column
    auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(p[0]) + __uint_as_float(p[1]);
    auto q = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(q[0]) + __uint_as_float(q[1]);
}

// The walk over a sequence's groups. A workgroup has 16 NT columns of the state in each of its NW first waves, all
// rows, as sums of matrix products; nothing of it leaves the wave's registers from group to group. Four
// more waves bring the next group's K, Q, T diag(beta) and P into LDS as operands meanwhile.
template <int DK, int NW, int NT>
__global__ __launch_bounds__(64 * (NW + 4)) void delta_walk_kernel(DeltaArgs a, DeltaScratch w, int splits) {
    constexpr int NU = DK / 32, NI = DK / 64;
    constexpr int kK = 0, kQ = kK + 2 * NU * 2 * kBlock, kTurned = kQ + 2 * NU * 2 * kBlock, kM = kTurned + DK / 16 * 2 * kBlock;
    constexpr int kP = kM + 4 * kBlock, kDecays = kP + 4 * kBlock, kBuffer = kDecays + 256;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int of = a.v_heads / a.qk_heads, per = of * splits;
    // workgroups that read the same keys on one XCD (they go to the eight in turns)
    const int unit = int(blockIdx.x / 8 / unsigned(per)) * 8 + int(blockIdx.x % 8), part = int(blockIdx.x / 8 % unsigned(per));
    if (unit >= a.b.n_seqs * a.qk_heads) return;
    const int s = unit / a.qk_heads, hk = unit % a.qk_heads, h = hk * of + part / splits, split_no = part % splits;
    const StateSeq v = state_seq(a.b, s);
    const int n_groups = (v.n + kChunk - 1) / kChunk;
    const size_t group0 = size_t(first_group(v, s));
    const int t = threadIdx.x, lane = t & 63, wid = __builtin_amdgcn_readfirstlane(t >> 6);

    if (wid >= NW) {
        const int i = t - 64 * NW;  // of 256
        float4 x[NI][4];
        float inv[NI][4];
        uint4 m0, m1;
        float decay = 0.0f;
        auto load = [&](int n) {
            const size_t group = group0 + n;
#pragma unroll
            for (int j = 0; j < NI; ++j) {
                const Item<DK> it(i + 256 * j);
                it.load(a, hk, v.r0 + n * kChunk, v.n - n * kChunk, x[j]);
                const float4 r = load4(w.inverse + (group * a.qk_heads + hk) * 64 + it.is_q * 32 + it.token);
                inv[j][0] = r.x;
                inv[j][1] = r.y;
                inv[j][2] = r.z;
                inv[j][3] = r.w;
            }
            const uint4 *src = reinterpret_cast<const uint4 *>(w.matrices + (group * a.v_heads + h) * kDeltaMatrices);
            m0 = src[i];
            m1 = src[i + 256];
            if (i < 64) decay = w.decays[(group * a.v_heads + h) * 64 + i];
        };
        auto store = [&](char *buf) {
#pragma unroll
            for (int j = 0; j < NI; ++j) {
                const Item<DK> it(i + 256 * j);
                it.store(buf + (it.is_q ? kQ : kK), x[j], inv[j]);
                if (!it.is_q) it.store_turned(buf + kTurned, x[j], inv[j]);
            }
            char *to = buf + kM + i / 64 * kBlock + i % 64 / 16 * 272 + i % 16 * 16;
            *reinterpret_cast<uint4 *>(to) = m0;
            *reinterpret_cast<uint4 *>(to + 4 * kBlock) = m1;
            if (i < 64) reinterpret_cast<float *>(buf + kDecays)[i] = decay;
        };
        if (n_groups > 0) {
            load(0);
            store(lds);
        }
        if (n_groups > 1) load(1);
        __syncthreads();
        for (int n = 0; n < n_groups; ++n) {
            if (n + 1 < n_groups) store(lds + (n + 1) % 2 * kBuffer);
            if (n + 2 < n_groups) load(n + 2);
            __syncthreads();
        }
        return;
    }

    const int g = lane / 16, lane_at = g * 272 + (lane % 16) * 16;
    const int col = (split_no * NW + wid) * 16 * NT + lane % 16;  // of column tile 0
    const int DV = a.value_dim;
    const size_t place = size_t(h) * DK * DV + col, pool = size_t(a.v_heads) * DK * DV;
    f4 S[2 * NU][NT];
    f4 val[2][NT];
    float bound[NT], sum[NT];  // of the column's length; of the next values' sizes
    int scale[NT];             // S is kept times 2^scale
    auto load_values = [&](int n) {
#pragma unroll
        for (int ti = 0; ti < 2; ++ti)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int m = n * kChunk + 16 * ti + 4 * g + r;
#pragma unroll
                for (int j = 0; j < NT; ++j) val[ti][j][r] = m < v.n ? a.v[size_t(v.r0 + m) * a.v_stride + size_t(h) * DV + col + 16 * j] : 0.0f;
            }
    };
    auto sum_values = [&](int j) {
        float x = 0.0f;
#pragma unroll
        for (int ti = 0; ti < 2; ++ti)
#pragma unroll
            for (int r = 0; r < 4; ++r) x += fabsf(val[ti][j][r]);
        return over_groups(x);
    };
    load_values(0);
#pragma unroll
    for (int k = 0; k < 2 * NU; ++k)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                S[k][j][r] = v.in >= 0 ? a.state[size_t(v.in) * pool + place + size_t(16 * k + 4 * g + r) * DV + 16 * j] : 0.0f;
    if (n_groups == 0) {
        __syncthreads();
        if (v.out >= 0)
#pragma unroll
            for (int k = 0; k < 2 * NU; ++k)
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) a.state[size_t(v.out) * pool + place + size_t(16 * k + 4 * g + r) * DV + 16 * j] = S[k][j][r];
        return;
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        float x = 0.0f;
#pragma unroll
        for (int k = 0; k < 2 * NU; ++k)
#pragma unroll
            for (int r = 0; r < 4; ++r) x += fabsf(S[k][j][r]);
        bound[j] = over_groups(x);
        sum[j] = sum_values(j);
        scale[j] = scale_for(bound[j] + sum[j]);
#pragma unroll
        for (int k = 0; k < 2 * NU; ++k) S[k][j] *= two_to(scale[j]);
    }
    __syncthreads();
    for (int n = 0; n < n_groups; ++n) {
        const char *buf = lds + n % 2 * kBuffer + lane_at;
        const float *decays = reinterpret_cast<const float *>(lds + n % 2 * kBuffer + kDecays);
        f4 ks[2][NT], qs[2][NT];
#pragma unroll
        for (int ti = 0; ti < 2; ++ti)
#pragma unroll
            for (int j = 0; j < NT; ++j) ks[ti][j] = qs[ti][j] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            Pair b[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j) b[j] = split(S[2 * u][j], S[2 * u + 1][j]);
#pragma unroll
            for (int ti = 0; ti < 2; ++ti) {
                const Pair k = operand(buf + kK + (ti * NU + u) * 2 * kBlock), q = operand(buf + kQ + (ti * NU + u) * 2 * kBlock);
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    ks[ti][j] = product(k, b[j], ks[ti][j]);
                    qs[ti][j] = product(q, b[j], qs[ti][j]);
                }
            }
        }
        f4 eg[2], el[2];
#pragma unroll
        for (int ti = 0; ti < 2; ++ti) {
            eg[ti] = *reinterpret_cast<const f4 *>(decays + 16 * ti + 4 * g);
            el[ti] = *reinterpret_cast<const f4 *>(decays + 32 + 16 * ti + 4 * g);
        }
        const float all = decays[31];
        Pair xb[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) {  // V - e^G K S, times 2^(scale - 4)
            f4 x[2];
#pragma unroll
            for (int ti = 0; ti < 2; ++ti)
#pragma unroll
                for (int r = 0; r < 4; ++r) x[ti][r] = __builtin_fmaf(eg[ti][r] * -0x1p-8f, ks[ti][j][r], val[ti][j][r] * two_to(scale[j] - 4));
            xb[j] = split(x[0], x[1]);
        }
        load_values(n + 1);
        f4 d[2][NT];  // D times 2^scale
#pragma unroll
        for (int ti = 0; ti < 2; ++ti) {
            const Pair m = operand(buf + kM + ti * 2 * kBlock);
#pragma unroll
            for (int j = 0; j < NT; ++j) d[ti][j] = product(m, xb[j], f4{0.f, 0.f, 0.f, 0.f});
        }
        f4 o[2][NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) xb[j] = split(d[0][j], d[1][j]);
#pragma unroll
        for (int ti = 0; ti < 2; ++ti) {
            const Pair p = operand(buf + kP + ti * 2 * kBlock);
#pragma unroll
            for (int j = 0; j < NT; ++j) o[ti][j] = product(p, xb[j], qs[ti][j] * eg[ti]);
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const float f = a.scale * two_to(-(scale[j] + 4));
#pragma unroll
            for (int ti = 0; ti < 2; ++ti)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int m = n * kChunk + 16 * ti + 4 * g + r;
                    if (m < v.n) a.out[size_t(v.r0 + m) * a.out_stride + size_t(h) * DV + col + 16 * j] = o[ti][j][r] * f;
                }
            bound[j] = __builtin_fmaf(all, bound[j], sum[j]);
            sum[j] = sum_values(j);
            const int next = scale_for(bound[j] + sum[j]);
            const float turn = two_to(next - scale[j]);
            scale[j] = next;
#pragma unroll
            for (int k = 0; k < 2 * NU; ++k) S[k][j] *= all * turn;
            xb[j] = split(d[0][j] * (el[0] * (turn * 0x1p-4f)), d[1][j] * (el[1] * (turn * 0x1p-4f)));
        }
#pragma unroll
        for (int k = 0; k < 2 * NU; ++k) {
            const Pair kt = operand(buf + kTurned + k * 2 * kBlock);
#pragma unroll
            for (int j = 0; j < NT; ++j) S[k][j] = product(kt, xb[j], S[k][j]);
        }
        __syncthreads();
    }
    if (v.out >= 0) {
#pragma unroll
        for (int k = 0; k < 2 * NU; ++k)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    a.state[size_t(v.out) * pool + place + size_t(16 * k + 4 * g + r) * DV + 16 * j] = S[k][j][r] * two_to(-scale[j]);
    }
}

// The norm and the gate of rows as the walk leaves them, in place: half a wave per row and head
template <int DV>
__global__ __launch_bounds__(256) void delta_norm_kernel(DeltaArgs a, int tiles) {
    const int lane = threadIdx.x & 31, h = int(blockIdx.x % unsigned(a.v_heads)), st = int(blockIdx.x / unsigned(a.v_heads));
    const int s = st / tiles;
    const StateSeq v = state_seq(a.b, s);
    const bool on = 4 * lane < DV;
    float4 w = make_float4(1.f, 1.f, 1.f, 1.f);
    if (on && a.gamma) w = load4(a.gamma + 4 * lane);
    for (int64_t m0 = int64_t(st % tiles) * kChunk; m0 < v.n; m0 += int64_t(tiles) * kChunk)
#pragma unroll
        for (int i = 0; i < kChunk / 8; ++i) {
            const int m = int(m0) + 8 * i + int(threadIdx.x) / 32;
            if (m >= v.n) continue;
            float *p = a.out + size_t(v.r0 + m) * a.out_stride + size_t(h) * DV + 4 * lane;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
            if (on) o = load4(p);
            if (a.gamma) {
                const float r = inv_root(lanes_sum<32>(dot4(o, o)) * (1.0f / DV) + a.gamma_eps);
                o = make_float4(o.x * r * w.x, o.y * r * w.y, o.z * r * w.z, o.w * r * w.w);
            }
            if (on && a.z) {
                const float4 z = load4(a.z + size_t(v.r0 + m) * a.z_stride + size_t(h) * DV + 4 * lane);
                o = make_float4(o.x * silu(z.x), o.y * silu(z.y), o.z * silu(z.z), o.w * silu(z.w));
            }
            if (on) *reinterpret_cast<float4 *>(p) = o;
        }
}

template <int DK, int NW, int NT> hipError_t launch_walk(const DeltaArgs &a, const DeltaScratch &w, hipStream_t s) {
    constexpr int kBuffer = ((2 * 2 * (DK / 32) + DK / 16) * 2 + 8) * kBlock + 256;
    const int splits = a.value_dim / (16 * NW * NT), per = a.v_heads / a.qk_heads * splits;
    const int units = a.b.n_seqs * a.qk_heads;
    hipLaunchKernelGGL((delta_walk_kernel<DK, NW, NT>), dim3(unsigned((units + 7) / 8) * 8u * unsigned(per)), dim3(64 * (NW + 4)),
                       2 * kBuffer, s, a, w, splits);
    return hipGetLastError();
}

template <int DK> hipError_t launch_groups(const DeltaArgs &a, const DeltaScratch &w, int cu_count, hipStream_t s) {
    const int64_t lists = int64_t(a.b.n_seqs) * a.v_heads;
    const int64_t want = (int64_t(a.max_new) + kChunk - 1) / kChunk, most = ((int64_t(1) << 24) - 1) / lists;
    const int tiles = int(want < 1 ? 1 : want < most ? want : most);  // (the others in turns)
    hipLaunchKernelGGL(delta_prepare_kernel<DK>, dim3(unsigned(a.b.n_seqs) * unsigned(tiles) * unsigned(a.qk_heads)), dim3(256), 0, s, a, w, tiles);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (lists < cu_count) e = launch_walk<DK, 2, 1>(a, w, s);
    else if (a.value_dim == 64) e = launch_walk<DK, 2, 2>(a, w, s);
    else e = launch_walk<DK, 4, 2>(a, w, s);
    if (e != hipSuccess || (!a.gamma && !a.z)) return e;
    const dim3 grid(unsigned(lists) * unsigned(tiles));
    if (a.value_dim == 64) hipLaunchKernelGGL(delta_norm_kernel<64>, grid, dim3(256), 0, s, a, tiles);
    else hipLaunchKernelGGL(delta_norm_kernel<128>, grid, dim3(256), 0, s, a, tiles);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_delta(const DeltaArgs &a, void *scratch, size_t scratch_bytes, int cu_count, hipStream_t s) {
    // (a walk of 2^22 heads would be past 2^32 threads)
    if (a.max_new > kStepRows && scratch && scratch_bytes >= delta_scratch_bytes(a) && int64_t(a.b.n_seqs) * a.v_heads < (1 << 22)) {
        const size_t groups = size_t(delta_groups(a.b.n_rows, a.b.n_seqs));
        DeltaScratch w;
        w.matrices = static_cast<char *>(scratch);
        w.decays = reinterpret_cast<float *>(w.matrices + groups * a.v_heads * kDeltaMatrices);
        w.inverse = w.decays + groups * a.v_heads * 64;
        return a.key_dim == 128 ? launch_groups<128>(a, w, cu_count, s) : launch_groups<64>(a, w, cu_count, s);
    }
    const dim3 grid(unsigned(a.b.n_seqs) * unsigned(a.v_heads));
#define QMM_STEP(K, V) hipLaunchKernelGGL((delta_step_kernel<K, V>), grid, dim3(256), 0, s, a)
    if (a.key_dim == 128) {
        if (a.value_dim == 128) QMM_STEP(128, 128);
        else QMM_STEP(128, 64);
    } else {
        if (a.value_dim == 128) QMM_STEP(64, 128);
        else QMM_STEP(64, 64);
    }
#undef QMM_STEP
    return hipGetLastError();
}

}  // namespace qmm
