// qmm_delta.hip — the gated delta rule.
//
// Every token of a head, in order, on its state S [DK][DV]:
//   S <- e^g S;  d = beta (v - S' k);  S <- S + k d';  o = S' q
// with k and q of unit length. The columns of S are independent of each other. Three ways, one for all sequences of a
// call, by the new rows of the longest: a token at a time (up to 8), groups of 32 in one launch, groups in three
// (launch_delta has the rule). Bound: a token at a time and one group by the states' way through memory, or the latency
// of a launch where they are few; prompts by the chain of groups, one product after the other (figures at the kernels,
// heads of 128).
#include <hip/hip_runtime.h>

#include "qmm_lanes.h"
#include "qmm_state.h"

namespace qmm {
namespace {

constexpr int kStepRows = 8;  // new rows up to which a token at a time is as fast as a group of 32 (heads of 128 and of 64)
constexpr int kGroup = 8;  // tokens whose inputs are in LDS at a time

__device__ inline float softplus(float x) { return x > 0.0f ? x + log1pf(expf(-x)) : log1pf(expf(x)); }
// Between -200, whose e^x is 0 in fp32 (sums over tokens keep their small parts, and no infinity meets another), and 0;
// NaN stays.
__device__ inline float log_decay(const DeltaArgs &a, int row, int h) {
    const float g = a.rate[h] * softplus(a.a[size_t(row) * a.a_stride + h] + a.dt_bias[h]);
    return g > 0.0f ? 0.0f : g < -200.0f ? -200.0f : g;
}
__device__ inline float step_size(const DeltaArgs &a, int row, int h) {
    return 1.0f / (1.0f + expf(-a.beta[size_t(row) * a.b_stride + h]));
}

__device__ inline float4 load4(const float *p) { return *reinterpret_cast<const float4 *>(p); }
__device__ inline float dot4(float4 x, float4 y) { return x.x * y.x + x.y * y.y + (x.z * y.z + x.w * y.w); }

// Rows r0 .. below r0 + n out, half a wave each, with the norm and the gate; get(m, e): four values of row r0 + m
template <int DV, typename F> __device__ inline void write_rows(const DeltaArgs &a, int h, int r0, int n, int t, int threads, F get) {
    const int e = 4 * (t % 32);
    const bool on = e < DV;
    for (int m = t / 32; m < n; m += threads / 32) {
        const size_t row = size_t(r0 + m);
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        if (on) o = get(m, e);
        if (a.gamma) {
            const float r = inv_root(lanes_sum<32>(dot4(o, o)) * (1.0f / DV) + a.gamma_eps);
            if (on) {
                const float4 w = load4(a.gamma + e);
                o = make_float4(o.x * r * w.x, o.y * r * w.y, o.z * r * w.z, o.w * r * w.w);
            }
        }
        if (on && a.z) {
            const float4 z = load4(a.z + row * a.z_stride + size_t(h) * DV + e);
            o = make_float4(o.x * silu(z.x), o.y * silu(z.y), o.z * silu(z.z), o.w * silu(z.w));
        }
        if (on) *reinterpret_cast<float4 *>(a.out + row * a.out_stride + size_t(h) * DV + e) = o;
    }
}

// One token after another through the state, for few new rows: a workgroup per sequence and head, a wave 16 * CL / 4
// columns (4 a lane) of all rows, in registers; a lane has rows 4 (rl + RL g) .. + 3. Both products with S are taken
// before it changes: S' q after the step is e^g S' q + (k.q) d, so one pass and one sum over the lanes serve both, and
// no wave waits for another between tokens. 32 heads: one sequence of a token 5.5 us (a launch and one way through
// memory), 64 sequences 49.2 us (5.5 TB/s of 273 MB); another token adds 0.75 us.
//
// MANY: more workgroups than three a CU. Then four: places are worked out again for every use, and k is read from LDS
// twice (kept over the tokens they take the registers of the fourth), and states of more than 32 MB in all go past the
// caches: 32 sequences of 4 tokens 29 us become 22, 64 of one 57 become 49. For fewer that only costs: one sequence of
// 8 tokens 10.7 us, so 11.6.
template <int DK, int DV, bool MANY>
__global__ __launch_bounds__(256, MANY ? 4 : 3) void delta_step_kernel(DeltaArgs a) {
    constexpr int CL = DV / 16, RL = 64 / CL, NG = DK / (4 * RL), NV = (kGroup * DV + 1023) / 1024;
    constexpr int HL = 32;  // lanes that hold one row of q or k
    __shared__ float qk[kGroup][2][DK];
    __shared__ float vo[kGroup][DV];  // values, then outputs
    __shared__ float sc[kGroup][4];   // decay, beta, k.q
    const int t = threadIdx.x, lane = t & 63, wid = __builtin_amdgcn_readfirstlane(t >> 6);
    const int s = int(blockIdx.x / unsigned(a.v_heads)), h = int(blockIdx.x % unsigned(a.v_heads));
    const int hk = h / (a.v_heads / a.qk_heads);
    const StateSeq v = state_seq(a.b, s);
    const int cl = lane % CL, rl = lane / CL, col = wid * (DV / 4) + 4 * cl;
    const int sub = lane % HL, is_k = lane / HL;
    const size_t pool = size_t(a.v_heads) * DK * DV;
    auto now = [](int x) {
        if (MANY) asm("" : "+v"(x));
        return x;
    };
    auto state = [&](int slot, int at) {
        return a.state + size_t(slot) * pool + size_t(h) * DK * DV + size_t(4 * (at / CL)) * DV + wid * (DV / 4) + 4 * (at % CL);
    };

    float4 x[kGroup / 4], val[NV];
    auto load = [&](int t0, int t) {
        const int sub = t % HL, is_k = t / HL % 2;
        const float *src = (is_k ? a.k : a.q) + size_t(hk) * DK + 4 * sub;
        const size_t src_stride = is_k ? a.k_stride : a.q_stride;
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
    if (v.n > 0) load(0, t);
    const bool past = MANY && size_t(gridDim.x) * (DK * DV * 4) > (32u << 20);
    float4 S[NG][4];
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float4 *p = reinterpret_cast<const float4 *>(state(v.in, lane) + size_t(4 * RL * g + j) * DV);
            S[g][j] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (v.in >= 0) S[g][j] = past ? load_past(p) : *p;
        }
    for (int t0 = 0; t0 < v.n; t0 += kGroup) {
        const int nt = min(kGroup, v.n - t0);
        if (t0 > 0) load(t0, now(t) & 255);
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
        for (int m = 0; m < nt; ++m) {
            const float decay = sc[m][0], beta = sc[m][1], kq = sc[m][2];
            const float4 val = load4(&vo[m][col]);
            float4 kept[NG];
            float ks[4] = {}, qs[4] = {};
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const float4 kr = load4(&qk[m][1][4 * (rl + RL * g)]);
                kept[g] = kr;
                const float4 qr = load4(&qk[m][0][4 * (rl + RL * g)]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float kj = reinterpret_cast<const float *>(&kr)[j], qj = reinterpret_cast<const float *>(&qr)[j];
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
            const int again = now(m);
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const float4 kr = MANY ? load4(&qk[again][1][4 * (rl + RL * g)]) : kept[g];
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        float &sv = reinterpret_cast<float *>(&S[g][j])[c];
                        sv = __builtin_fmaf(reinterpret_cast<const float *>(&kr)[j], d[c], sv * decay);
                    }
            }
            if (rl == 0) *reinterpret_cast<float4 *>(&vo[m][col]) = make_float4(qs[0], qs[1], qs[2], qs[3]);
        }
        __syncthreads();
        write_rows<DV>(a, h, v.r0 + t0, nt, now(t) & 255, 256, [&](int m, int e) { return load4(&vo[m][e]); });
        __syncthreads();
    }
    if (v.out >= 0) {
        float *to = state(v.out, now(lane) & 63);
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float4 *p = reinterpret_cast<float4 *>(to + size_t(4 * RL * g + j) * DV);
                if (past) store_past(p, S[g][j]);
                else *p = S[g][j];
            }
    }
}

// ------------------------------------------------------------- prompts
// Of a group of up to 32 tokens, with G_i the sum of its log decays up to token i, k and q its unit rows and
// S the state before it:
//   A_ij = beta_i e^(G_i - G_j) k_i.k_j  (j < i),   T = (I + A)^-1,   P_ij = e^(G_i - G_j) q_i.k_j  (j <= i)
//   D = T diag(beta) (V - diag(e^G) K S),   O = diag(e^G) Q S + P D,   S <- e^(G_last) S + K' diag(e^(G_last - G)) D
// The first kernel makes T and P of every group at once; the second walks a sequence's groups. All products but the
// inverse run on the matrix units in fp16, each operand as a pair hi + lo of 22 bits (three products: hi hi, hi lo, lo
// hi), sums in fp32. A low part is a multiple of 2^-24, so operands are kept large: K, at most 1 in size and of length
// 1, 2^4 times; Q, T and P, at most 1 in size, 2^14 times (their small values meet large ones of D where decays are
// strong); the scale of a column of S, D and V is a power of two, from a bound of the column that holds for the group
// (|S column| grows by |v| at most, as a step makes no column longer; and it is measured now and then). What is left of
// a value is good to 2^-22, or 2^-39 of that bound (D in the state's update, 2^-4 times for the keys' 2^4, 2^-36). beta
// is no part of T: small ones would lose bits there.
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));

// An operand of 16 rows and 32 columns k in LDS, 1 KB: lane (row r, group g of lanes) reads the 16 B of place 16 g + (r
// ^ g), columns 4 g .. + 3 and 16 + 4 g .. + 3. That is the order in which a group of lanes holds the rows of two tiles
// of a product, so a product's result is the next product's right operand as it stands. (r ^ g, not r: pieces of 8 B of
// four columns, written by the lanes of four rows and all g at once, then lie on all banks.)
constexpr int kBlock = 1024;
__device__ inline int operand_at(int row, int col) {  // of the aligned 4 columns from `col` (of 32)
    const int g = col % 16 / 4;
    return g * 256 + (row % 16 ^ g) * 16 + col / 16 * 8;
}
__device__ inline f4 mfma(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
// x f = hi + lo + at most 2^-22 |x f| (and 2^-25). `f` is no constant the compiler sees, so that the low part is one
// operation on the fp16 high part.
__device__ inline void split4(f4 x, float f, h4 &hi, h4 &lo) {
    hi = __builtin_convertvector(x * f, h4);
    f4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __builtin_fmaf(x[i], f, -float(hi[i]));
    lo = __builtin_convertvector(r, h4);
}
__device__ inline void split4(f4 x, h4 &hi, h4 &lo) {
    float one = 1.0f;
    asm("" : "+s"(one));
    hi = __builtin_convertvector(x, h4);
    f4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __builtin_fmaf(x[i], one, -float(hi[i]));
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

// The products of two tiles of rows, the three of each pair apart, as each adds to the one before
__device__ inline void products(const Pair (&op)[2], const Pair &b, f4 (&c)[2]) {
#pragma unroll
    for (int part = 0; part < 3; ++part)
#pragma unroll
        for (int i = 0; i < 2; ++i) c[i] = mfma(part < 2 ? op[i].hi : op[i].lo, part == 1 ? b.lo : b.hi, c[i]);
}
// the order of what stands since the last barrier of the scheduler: N times one matrix product and K vector
// instructions
template <int N, int K> __device__ inline void mix() {
    if constexpr (N > 0) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, K, 0);
        mix<N - 1, K>();
    }
}

struct DeltaScratch {
    char *matrices;  // [groups][v_heads]: T, then P: two tiles of 16 rows, each 1 KB hi and 1 KB lo
    float *factors;  // [groups][v_heads][96]: e^G_i, e^(G_last - G_i), beta_i
    float *inverse;  // [groups][qk_heads][64]: 1 / |k_i|, 1 / |q_i|
    // of sequences that are walked in halves, per sequence and value head: the state after the first one; the second
    // one's end from a state of zeros; and what it makes of the unit vectors; of the second one's tokens, what they
    // read of those
    float *middle, *end, *carry, *reads;
};
// A sequence's second half begins at this group (its number of groups: it has none).
__device__ inline int second_half(int n_groups, bool halves) { return halves && n_groups >= kHalfGroups ? (n_groups + 1) / 2 : n_groups; }
__device__ inline int64_t first_group(const StateSeq &v, int s) { return v.r0 / kChunk + s; }

// Up to 32 rows from `p` on, of which `left` are the sequence's, as a buffer: loads past them give 0 and stores
// nothing, without a branch. p: row 0 of one head, `before` values into its row; stride below 2^24 values, so that all
// offsets fit.
__device__ inline __amdgpu_buffer_rsrc_t group_rows(const float *p, size_t stride, int before, int left) {
    const uint32_t rows = uint32_t(min(max(left, 0), kChunk));
    const uint32_t bytes = (rows * uint32_t(stride) - (rows ? uint32_t(before) : 0u)) * 4u;
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(p), short(0), __builtin_amdgcn_readfirstlane(int(bytes)), 0x00020000);
}

// 4 tokens x 4 values of q or k, one of a group's 2 * 8 * DK / 4: eight lanes side by side take 128 B
template <int DK> struct Item {
    int is_q, token, at;
    __device__ Item(int t, int j) {  // thread t's j-th of DK / 64; a wave has one kind
        constexpr int kAll = 8 * DK / 4;
        is_q = DK == 128 ? j : __builtin_amdgcn_readfirstlane(t / kAll);
        const int r = t % kAll;
        token = r / 8 % 8 * 4;
        at = (r / 64 * 8 + r % 8) * 4;
    }
    // from rows r0 .. of which `left` are the sequence's
    __device__ void load(const DeltaArgs &a, int hk, int r0, int left, f4 x[4]) const {
        const size_t stride = is_q ? a.q_stride : a.k_stride;
        const __amdgpu_buffer_rsrc_t rows = group_rows((is_q ? a.q : a.k) + size_t(r0) * stride + size_t(hk) * DK, stride, hk * DK, left);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            x[j] = __builtin_bit_cast(f4, __builtin_amdgcn_raw_buffer_load_b128(
                                              rows, (unsigned(token + j) * unsigned(stride) + unsigned(at)) * 4u, 0, 0));
    }
    // times 2^4 (k) or 2^14 (q) / length as left operand, rows the tokens (tiles of 16, each DK / 32 blocks of hi and
    // lo) and, where `turned`, rows the values (tiles of 16, each one block)
    __device__ void convert(const f4 x[4], f4 inv, h4 hi[4], h4 lo[4]) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) split4(x[j], inv[j] * (is_q ? 0x1p14f : 0x1p4f), hi[j], lo[j]);
    }
    __device__ void store(char *base, char *turned, const h4 hi[4], const h4 lo[4]) const {
        char *p = base + ((token / 16) * (DK / 32) + at / 32) * 2 * kBlock;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            *reinterpret_cast<h4 *>(p + operand_at(token + j, at % 32)) = hi[j];
            *reinterpret_cast<h4 *>(p + operand_at(token + j, at % 32) + kBlock) = lo[j];
        }
        if (!turned) return;
        p = turned + (at / 16) * 2 * kBlock;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            *reinterpret_cast<h4 *>(p + operand_at(at + c, token)) = h4{hi[0][c], hi[1][c], hi[2][c], hi[3][c]};
            *reinterpret_cast<h4 *>(p + operand_at(at + c, token) + kBlock) = h4{lo[0][c], lo[1][c], lo[2][c], lo[3][c]};
        }
    }
};

__device__ inline double shfl_up(double x, int d) {
    const uint64_t u = __double_as_longlong(x);
    return __longlong_as_double((uint64_t(uint32_t(__shfl_up(int(u >> 32), d, 32))) << 32) | uint32_t(__shfl_up(int(u), d, 32)));
}

constexpr int kRow = 36;  // floats of a row of a 32 x 32 matrix in LDS
typedef float Square[32][kRow];

// The pieces of T and P of one group: squares of an item's rows, summed over the eight lanes that share them, to
// sums[kind][token][of 32 values]
template <int DK> __device__ inline void row_squares(const Item<DK> &it, const f4 x[4], float (*sums)[32][DK / 32]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float ss = (x[j][0] * x[j][0] + x[j][1] * x[j][1]) + (x[j][2] * x[j][2] + x[j][3] * x[j][3]);
        ss += lane_moved<0xB1>(ss);
        ss += lane_moved<0x4E>(ss);
        ss += lane_moved<0x141>(ss);
        if (threadIdx.x % 8 == 0) sums[it.is_q][it.token + j][it.at / 32] = ss;
    }
}
template <int DK> __device__ inline float inverse_length(const float (&sums)[DK / 32], float eps) {
#pragma unroll
    for (int u = 0; u < DK / 32; ++u) eps += sums[u];
    return inv_root(eps);
}
// 2^x, x rounded to fp32 first: |x| 2^-24 off
__device__ inline float power_of_two(double x) { return __builtin_amdgcn_exp2f(float(x)); }
// sums of the log decays of a head (of 2: the decays are powers of two, one instruction each) and its step sizes, a
// token per lane of half a wave
__device__ inline void head_steps(const DeltaArgs &a, int row, int h, int m, bool on, double *G, float *beta) {
    double g = on ? double(log_decay(a, row, h)) * 1.4426950408889634 : 0.0;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const double o = shfl_up(g, d);
        if (m >= d) g += o;
    }
    G[m] = g;
    beta[m] = on ? step_size(a, row, h) : 0.0f;
}
// one of the six tiles of k k' (0..2) and q k' (3..5) on and below the diagonal, by a wave; and its way to LDS
template <int DK> __device__ inline f4 tile_of(int task, int lane, const char *k, const char *q) {
    constexpr int NU = DK / 32;
    const int ti = task % 3 != 0, tj = task % 3 == 2, at = (lane / 16) * 256 + (lane % 16 ^ lane / 16) * 16;
    f4 c{};
#pragma unroll
    for (int u = 0; u < NU; ++u)
        c = product(operand((task < 3 ? k : q) + (ti * NU + u) * 2 * kBlock + at), operand(k + (tj * NU + u) * 2 * kBlock + at), c);
    return c * (task < 3 ? 0x1p-8f : 0x1p-18f);
}
__device__ inline void store_tile(int task, int lane, f4 c, Square &kk, Square &qk) {
    Square &to = task < 3 ? kk : qk;
#pragma unroll
    for (int r = 0; r < 4; ++r) to[16 * (task % 3 != 0) + 4 * (lane / 16) + r][16 * (task % 3 == 2) + lane % 16] = c[r];
}
// four values of a 32 x 32 matrix as operand: `place` is that of row and column (operand_at) in the row's tile
__device__ inline void store_operand(char *matrix, int i, int place, f4 x) {
    h4 hi, lo;
    split4(x, hi, lo);
    *reinterpret_cast<h4 *>(matrix + i / 16 * 2 * kBlock + place) = hi;
    *reinterpret_cast<h4 *>(matrix + i / 16 * 2 * kBlock + place + kBlock) = lo;
}
// row i, columns c .. c + 3 of A, and of P times 2^14 (above the diagonal's tiles nothing was written: any value)
__device__ inline f4 mask_and_decay(const Square &kk, const Square &qk, const double *G, const float *beta, int i, int c, Square &A) {
    const f4 kv = *reinterpret_cast<const f4 *>(&kk[i][c]), qv = *reinterpret_cast<const f4 *>(&qk[i][c]);
    const double row = G[i];
    f4 p, x;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float e = power_of_two(row - G[c + j]);
        x[j] = c + j < i ? beta[i] * e * kv[j] : 0.0f;
        p[j] = c + j <= i ? e * qv[j] * 0x1p14f : 0.0f;
    }
    *reinterpret_cast<f4 *>(&A[i][c]) = x;
    return p;
}
// The inverse of I + A: its two 16 x 16 triangles by substitution, a column per lane, then T21 = -T22 A21 T11 on the
// matrix units in fp32.
__device__ inline void invert_half(const Square &A, int b, int col, Square &T) {
    float x[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        float y = r == col ? 1.0f : 0.0f;
#pragma unroll
        for (int j = 0; j < r; ++j) y = __builtin_fmaf(-A[b + r][b + j], x[j], y);
        x[r] = y;
        T[b + r][b + col] = y;
    }
}
__device__ inline void invert_corner(const Square &A, int lane, Square &T) {  // (a wave)
    const int g = lane / 16, col = lane % 16;
    f4 y{}, z{};
#pragma unroll
    for (int k = 0; k < 16; k += 4) y = __builtin_amdgcn_mfma_f32_16x16x4f32(A[16 + col][k + g], T[k + g][col], y, 0, 0, 0);
#pragma unroll
    for (int r = 0; r < 4; ++r) z = __builtin_amdgcn_mfma_f32_16x16x4f32(T[16 + col][16 + 4 * g + r], y[r], z, 0, 0, 0);
#pragma unroll
    for (int r = 0; r < 4; ++r) T[16 + 4 * g + r][col] = -z[r];
}
// row i, columns c .. c + 3 of T, times 2^14
__device__ inline f4 enlarged(const Square &T, int i, int c) {
    return c / 16 <= i / 16 ? *reinterpret_cast<const f4 *>(&T[i][c]) * 0x1p14f : f4{0.f, 0.f, 0.f, 0.f};
}
// of 96 factors: e^G_i, then e^(G_last - G_i), then beta_i
__device__ inline float factor_of(const double *G, const float *beta, int i) {
    return i < 64 ? power_of_two(i < 32 ? G[i] : G[31] - G[i - 32]) : beta[i - 64];
}

// T and P of one group and key head, for its value heads two at a time (both inverses in one wave). Bound: the chain of
// ten barriers at four workgroups of a CU (35 KB of LDS; with three, k k' and q k' beside the rows, 58 us): 8192 tokens
// of 16 key and 32 value heads 53 us. Of 58, loads, conversion and products were 31, inverses 6, stores 4.
template <int DK>
__global__ __launch_bounds__(256) void delta_prepare_kernel(DeltaArgs a, DeltaScratch w, int tiles) {
    constexpr int NU = DK / 32, NI = DK / 64;
    constexpr int kRows = 2 * NU * 2 * kBlock, kSquares = 6 * sizeof(Square);
    __shared__ __attribute__((aligned(16))) char shared[2 * kRows > kSquares ? 2 * kRows : kSquares];
    char *const rows = shared;  // k and q as operands; after their products those, and A and T of two heads
    Square *const A = reinterpret_cast<Square *>(shared), *const T = A + 2;
    Square &kk = A[4], &qk = A[5];
    __shared__ float sums[2][32][NU];
    __shared__ __attribute__((aligned(16))) float inv[2][32];
    __shared__ double G[2][32];
    __shared__ float beta[2][32];
    const int t = threadIdx.x, lane = t & 63, wid = __builtin_amdgcn_readfirstlane(t >> 6);
    const int hk = int(blockIdx.x % unsigned(a.qk_heads)), st = int(blockIdx.x / unsigned(a.qk_heads));
    const int s = st / tiles, of = a.v_heads / a.qk_heads;
    const StateSeq v = state_seq(a.b, s);
    for (int tile = st % tiles; int64_t(tile) * kChunk < v.n; tile += tiles) {
        const int r0 = v.r0 + tile * kChunk, left = v.n - tile * kChunk;
        const size_t group = size_t(first_group(v, s) + tile);
        f4 x[NI][4];
#pragma unroll
        for (int i = 0; i < NI; ++i) Item<DK>(t, i).load(a, hk, r0, left, x[i]);
#pragma unroll
        for (int i = 0; i < NI; ++i) row_squares<DK>(Item<DK>(t, i), x[i], sums);
        __syncthreads();
        if (t < 64) {
            const float r = inverse_length<DK>(sums[t / 32][t % 32], a.qk_eps);
            inv[t / 32][t % 32] = r;
            w.inverse[(group * a.qk_heads + hk) * 64 + t] = r;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const Item<DK> it(t, i);
            h4 hi[4], lo[4];
            it.convert(x[i], *reinterpret_cast<const f4 *>(&inv[it.is_q][it.token]), hi, lo);
            it.store(rows + it.is_q * kRows, nullptr, hi, lo);
        }
        __syncthreads();
        const f4 first = tile_of<DK>(wid, lane, rows, rows + kRows);
        f4 second{};
        if (wid < 2) second = tile_of<DK>(wid + 4, lane, rows, rows + kRows);
        __syncthreads();
        store_tile(wid, lane, first, kk, qk);
        if (wid < 2) store_tile(wid + 4, lane, second, kk, qk);
        __syncthreads();
        for (int h0 = 0; h0 < of; h0 += 2) {
            const int nh = min(2, of - h0);
            const size_t first = group * a.v_heads + hk * of + h0;
            if (wid == 0) {
                const int hh = lane / 32, m = lane % 32;
                head_steps(a, r0 + m, hk * of + h0 + hh, m, hh < nh && m < left, G[hh], beta[hh]);
            }
            __syncthreads();
            if (t < kFactors * nh) w.factors[first * kFactors + t] = factor_of(G[t / kFactors], beta[t / kFactors], t % kFactors);
            const int i = t / 8, c = t % 8 * 4, place = (c % 16 / 4) * 256 + i % 16 * 16 + c / 16 * 8;
            for (int hh = 0; hh < nh; ++hh)
                store_operand(w.matrices + (first + hh) * kDeltaMatrices + 4 * kBlock, i, place,
                              mask_and_decay(kk, qk, G[hh], beta[hh], i, c, A[hh]));
            __syncthreads();
            if (wid == 0 && lane / 32 < nh) invert_half(A[lane / 32], lane / 16 % 2 * 16, lane % 16, T[lane / 32]);
            __syncthreads();
            if (wid < nh) invert_corner(A[wid], lane, T[wid]);
            __syncthreads();
            for (int hh = 0; hh < nh; ++hh) store_operand(w.matrices + (first + hh) * kDeltaMatrices, i, place, enlarged(T[hh], i, c));
            __syncthreads();
        }
        __syncthreads();
    }
}

__device__ inline float two_to(int e) { return __uint_as_float(uint32_t(e + 127) << 23); }
// The power of two that takes numbers up to `bound` below 2^15, from 2^-32 (2^30 rows of values below 65520 sum to less
// than 2^46) to 2^94, so that two of them have a quotient in fp32. Columns that sum to less than 2^-80 lose the bits
// below 2^-119. It is kept less 30: its largest is then 64, the largest constant of an instruction (8192 tokens of 8
// heads otherwise 268 us, so 263).
constexpr int kScale = 30;
__device__ inline int scale_for(float bound) {
    return min(max(141 - kScale - int(__float_as_uint(bound) >> 23 & 255), -32 - kScale), 94 - kScale);
}
__device__ inline float grown(int scale) { return two_to(scale + kScale); }
__device__ inline float shrunk(int scale, int more = 0) { return two_to(-(scale + kScale + more)); }
__device__ inline float over_groups(float x) {  // sum over the four lanes of a column
    auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(p[0]) + __uint_as_float(p[1]);
    auto q = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(q[0]) + __uint_as_float(q[1]);
}

__device__ inline float most_over_groups(float x) {
    auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
    auto q = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(q[0]), __uint_as_float(q[1]));
}
// A column's length is at most sqrt(DK) of its largest value, and at most what it was, decayed, and what the values
// added. The second grows with every token where nothing decays, so the walk measures the first after every second
// group (8192 tokens of 32 heads 387 us, 385 without; after each one 391).
constexpr int kMeasured = 2;
__device__ inline float larger(float m, float x, float y) { return fmaxf(fmaxf(m, fabsf(x)), fabsf(y)); }

// The i-th longest of up to 64 sequences, a lane each: the longest walks begin first (prompts of 951, 677, 403, 129,
// 1500 and 1225 tokens: 107 us in their order, 97 so). More than a wave can rank keep their order (2000 tokens behind
// 64 of 100 in all 490 us, in front of them 415).
__device__ inline int by_length(const StateView &b, int i) {
    if (b.n_seqs > 64) return i;
    const int lane = threadIdx.x % 64, n = lane < b.n_seqs ? state_seq(b, lane).n : -1;
    int longer = 0;
    for (int j = 0; j < b.n_seqs; ++j) {
        const int other = __builtin_amdgcn_readlane(n, j);
        longer += other > n || (other == n && j < lane);
    }
    return int(__builtin_ctzll(__ballot(longer == i)));
}

// The walk over a sequence's groups. A workgroup has 16 columns of the state in each of its NW first waves, all rows,
// as sums of matrix products; nothing of it leaves the wave's registers from group to group. Four more waves bring the
// next group's K, Q, T and P into LDS as operands meanwhile. Bound: one wave's chain of 84 matrix products and 300
// vector instructions a group, beside 62 KB of LDS reads a wave and 57 KB of writes: 1.6 us a group of 32 columns, 1.65
// to 2.0 of 64, where the products alone take 0.57 (16.2 cycles each). 417 tokens 26.8 us. Measured and not kept: 16
// columns a workgroup, operands made by the first kernel (480 us for 8192 tokens against 411), output products in waves
// of their own, K S of the next group beside this one's.
//
// HALVES: a sequence of many groups goes in two halves at once, where compute units are left. The rule is linear in the
// state: what follows from S is what follows from zeros, with the values, and M S without them, M from the unit matrix.
// So the second half is walked twice, for the values (kind 1) and for M (kind 2), and joined with the first one's last
// state afterwards. 8192 tokens: 411 us in one, 240 in halves.
template <int DK, int NW, bool HALVES>
__global__ __launch_bounds__(512) void delta_walk_kernel(DeltaArgs a, DeltaScratch w, int splits) {
    constexpr int NU = DK / 32, NI = DK / 64;
    constexpr int kK = 0, kQ = kK + 2 * NU * 2 * kBlock, kTurned = kQ + 2 * NU * 2 * kBlock, kM = kTurned + DK / 16 * 2 * kBlock;
    constexpr int kP = kM + 4 * kBlock, kFactor = kP + 4 * kBlock, kBuffer = kFactor + kFactors * 4;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int of = a.v_heads / a.qk_heads, parts = HALVES ? 2 * splits + DK / (16 * NW) : splits, per = of * parts;
    // workgroups that read the same keys on one XCD (they go to the eight in turns)
    const int unit = int(blockIdx.x / 8 / unsigned(per)) * 8 + int(blockIdx.x % 8), part = int(blockIdx.x / 8 % unsigned(per));
    if (unit >= a.b.n_seqs * a.qk_heads) return;
    const int s = HALVES ? unit / a.qk_heads : by_length(a.b, unit / a.qk_heads), hk = unit % a.qk_heads, h = hk * of + part / parts;
    StateSeq v = state_seq(a.b, s);
    const int kind = HALVES ? min(part % parts / splits, 2) : 0;
    const int all_groups = (v.n + kChunk - 1) / kChunk, middle = second_half(all_groups, HALVES), first = kind ? middle : 0;
    if (HALVES && kind && middle == all_groups) return;
    const int n_groups = HALVES ? (kind ? all_groups - middle : middle) : all_groups;
    const size_t group0 = size_t(first_group(v, s)) + size_t(first), read0 = size_t(v.r0) / 2;
    if (HALVES) {
        v.n = kind ? v.n - first * kChunk : min(v.n, middle * kChunk);
        v.r0 += first * kChunk;
    }
    const int t = threadIdx.x, lane = t & 63, wid = __builtin_amdgcn_readfirstlane(t >> 6);

    if (wid >= NW) {
        // (waves go to the four SIMDs in turns: with two walking ones, the two after the first four would share theirs)
        if (NW == 2 && (wid & 2) == 0) return;
        const int i = NW == 2 ? (wid / 4 * 2 + wid % 2) * 64 + lane : t - 64 * NW;  // of 256
        // what a thread holds of a group while it comes from memory
        struct Held {
            f4 x[NI][4];
            f4 inv[NI];
            f4 m0, m1;
            float factor;
        };
        auto load = [&](int n, Held &y) {  // (past the last group: rows of zeros, the last one's matrices)
            const size_t group = group0 + min(n, n_groups - 1);
#pragma unroll
            for (int j = 0; j < NI; ++j) {
                const Item<DK> it(i, j);
                it.load(a, hk, v.r0 + n * kChunk, v.n - n * kChunk, y.x[j]);
                y.inv[j] = *reinterpret_cast<const f4 *>(w.inverse + (group * a.qk_heads + hk) * 64 + it.is_q * 32 + it.token);
            }
            const f4 *src = reinterpret_cast<const f4 *>(w.matrices + (group * a.v_heads + h) * kDeltaMatrices);
            y.m0 = src[i];
            y.m1 = src[i + 256];
            y.factor = w.factors[(group * a.v_heads + h) * kFactors + i % kFactors];
        };
        // One step: group n from the registers to LDS, and group n + 2 on its way to them. The writes come last: LDS is
        // the walking waves' while they read the first operands of their step.
        auto pass = [&](int n, Held &y) {
            char *buf = lds + n % 2 * kBuffer;
            h4 hi[NI][4], lo[NI][4];
#pragma unroll
            for (int j = 0; j < NI; ++j) Item<DK>(i, j).convert(y.x[j], y.inv[j], hi[j], lo[j]);
            const f4 m0 = y.m0, m1 = y.m1;
            const float factor = y.factor;
            __builtin_amdgcn_sched_barrier(0);
            load(n + 2, y);
            __builtin_amdgcn_sched_barrier(0);
            char *to = buf + kM + i / 64 * kBlock + i % 64 / 16 * 256 + (i % 16 ^ i % 64 / 16) * 16;
            *reinterpret_cast<f4 *>(to) = m0;
            *reinterpret_cast<f4 *>(to + 4 * kBlock) = m1;
            reinterpret_cast<float *>(buf + kFactor)[i % kFactors] = factor;
#pragma unroll
            for (int j = 0; j < NI; ++j) {
                const Item<DK> it(i, j);
                it.store(buf + (it.is_q ? kQ : kK), it.is_q ? nullptr : buf + kTurned, hi[j], lo[j]);
            }
        };
        if (n_groups == 0) {
            __syncthreads();
            return;
        }
        Held even, odd;  // two groups are under way, so that a walk's step may be shorter than the memory's latency
        load(0, even);
        load(1, odd);
        pass(0, even);
        __syncthreads();
        int n = 0;  // (no way out between the two steps: the waits count the loads of one path)
        for (; n + 1 < n_groups; n += 2) {
            pass(n + 1, odd);
            __syncthreads();
            pass(n + 2, even);
            __syncthreads();
        }
        if (n < n_groups) __syncthreads();
        return;
    }

    __builtin_amdgcn_s_setprio(2);  // before the waves that bring operands
    const int g = lane / 16, lane_at = g * 256 + (lane % 16 ^ g) * 16;
    const int DV = a.value_dim, columns = kind == 2 ? DK : DV;
    const int col = ((part % parts - kind * splits) * NW + wid) * 16 + lane % 16;
    const size_t pool = size_t(a.v_heads) * DK * DV, list = size_t(s) * a.v_heads + h;
    const float *from = v.in >= 0 ? a.state + size_t(v.in) * pool + size_t(h) * DK * DV : nullptr;
    float *to = v.out >= 0 ? a.state + size_t(v.out) * pool + size_t(h) * DK * DV : nullptr;
    float *out = a.out + size_t(v.r0) * a.out_stride + size_t(h) * DV;
    size_t out_stride = a.out_stride;
    float out_factor = a.scale;
    if (HALVES && kind) from = nullptr;
    if (HALVES && (kind || middle < all_groups)) to = kind == 2 ? w.carry + list * DK * DK : (kind ? w.end : w.middle) + list * DK * DV;
    if (HALVES && kind == 2) {
        out_stride = size_t(a.v_heads) * DK;
        out = w.reads + read0 * out_stride + size_t(h) * DK;
        out_factor = 1.0f;
    }
    const f4 zero = {0.f, 0.f, 0.f, 0.f};
    f4 S[2 * NU], val[2], ahead[2];     // values of this group and the next
    unsigned v_at[2][4], out_at[2][4];  // bytes from a group's first row to this lane's, of its row tensors
#pragma unroll
    for (int ti = 0; ti < 2; ++ti)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            v_at[ti][r] = (unsigned(16 * ti + 4 * g + r) * unsigned(a.v_stride) + unsigned(col)) * 4u;
            out_at[ti][r] = (unsigned(16 * ti + 4 * g + r) * unsigned(out_stride) + unsigned(col)) * 4u;
        }
    auto load_values = [&](int n, f4 (&to)[2]) {
        const __amdgpu_buffer_rsrc_t rows =
            group_rows(a.v + size_t(v.r0 + n * kChunk) * a.v_stride + size_t(h) * DV, a.v_stride, h * DV,
                       kind == 2 ? 0 : v.n - n * kChunk);
#pragma unroll
        for (int ti = 0; ti < 2; ++ti)
#pragma unroll
            for (int r = 0; r < 4; ++r) to[ti][r] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rows, v_at[ti][r], 0, 0));
    };
    auto sizes = [](const f4 (&x)[2]) {
        float y = 0.0f;
#pragma unroll
        for (int ti = 0; ti < 2; ++ti)
#pragma unroll
            for (int r = 0; r < 4; ++r) y += fabsf(x[ti][r]);
        return over_groups(y);
    };
    load_values(0, val);
    load_values(1, ahead);
#pragma unroll
    for (int k = 0; k < 2 * NU; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = 16 * k + 4 * g + r;
            S[k][r] = from ? from[size_t(row) * DV + col] : kind == 2 && row == col ? 1.0f : 0.0f;
        }
    if (n_groups == 0) {
        __syncthreads();
        if (to)
#pragma unroll
            for (int k = 0; k < 2 * NU; ++k)
#pragma unroll
                for (int r = 0; r < 4; ++r) to[size_t(16 * k + 4 * g + r) * DV + col] = S[k][r];
        return;
    }
    float bound = 0.0f, sum = sizes(val);  // of the column's length; of the values' sizes
#pragma unroll
    for (int k = 0; k < 2 * NU; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r) bound += fabsf(S[k][r]);
    bound = over_groups(bound);
    int scale = scale_for(bound + sum);  // S is kept times grown(scale)
#pragma unroll
    for (int k = 0; k < 2 * NU; ++k) S[k] *= grown(scale);
    __syncthreads();
    int n = 0;
    do {
        const char *buf = lds + n % 2 * kBuffer + lane_at;
        const float *factors = reinterpret_cast<const float *>(lds + n % 2 * kBuffer + kFactor);
        // A wave has no other beside it to fill its gaps: operands are read ahead of their products, and Q S, for which
        // nothing waits, runs beside the steps from K S to D.
        f4 ks[2] = {zero, zero}, qs[2] = {zero, zero}, eg[2], el[2], beta[2];
        Pair ops[2][2], b[NU], m[2], p[2];
        auto read_rows = [&](int at, int u, Pair (&to)[2]) {  // both token tiles
#pragma unroll
            for (int ti = 0; ti < 2; ++ti) to[ti] = operand(buf + at + (ti * NU + u) * 2 * kBlock);
        };
        read_rows(kK, 0, ops[0]);
        read_rows(kK, 1, ops[1]);
        b[0] = split(S[0], S[1]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            products(ops[u % 2], b[u], ks);
            if (u + 1 < NU) b[u + 1] = split(S[2 * u + 2], S[2 * u + 3]);
            mix<6, 3>();
            __builtin_amdgcn_sched_barrier(0);
            if (u + 2 < NU) {
                read_rows(kK, u + 2, ops[u % 2]);
            } else if (u + 2 == NU) {
#pragma unroll
                for (int ti = 0; ti < 2; ++ti) {
                    m[ti] = operand(buf + kM + ti * 2 * kBlock);
                    eg[ti] = *reinterpret_cast<const f4 *>(factors + 16 * ti + 4 * g);
                    beta[ti] = *reinterpret_cast<const f4 *>(factors + 64 + 16 * ti + 4 * g);
                }
                read_rows(kQ, 0, ops[u % 2]);
            } else {
                read_rows(kQ, 1, ops[u % 2]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        const float all = factors[31];
        f4 x[2];  // diag(beta) (V - diag(e^G) K S), times grown(scale)
#pragma unroll
        for (int ti = 0; ti < 2; ++ti)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                x[ti][r] = beta[ti][r] * __builtin_fmaf(eg[ti][r] * -0x1p-4f, ks[ti][r], val[ti][r] * grown(scale));
        const Pair xb = split(x[0], x[1]);
        products(ops[0], b[0], qs);
        mix<6, 6>();
        __builtin_amdgcn_sched_barrier(0);
        if (NU > 2) read_rows(kQ, 2, ops[0]);
#pragma unroll
        for (int ti = 0; ti < 2; ++ti) {
            p[ti] = operand(buf + kP + ti * 2 * kBlock);
            val[ti] = ahead[ti];
        }
        load_values(n + 2, ahead);
        __builtin_amdgcn_sched_barrier(0);
        f4 d[2] = {zero, zero};  // D times 2^14 grown(scale)
        products(m, xb, d);
        products(ops[1], b[1], qs);
        bound = __builtin_fmaf(all, bound, sum);
        sum = sizes(val);
        const int next = scale_for(bound + sum);
        const float turn = two_to(next - scale), out_scale = out_factor * shrunk(scale, 14);
        scale = next;
#pragma unroll
        for (int k = 0; k < 2 * NU; ++k) S[k] *= all * turn;
        mix<12, 5>();
        __builtin_amdgcn_sched_barrier(0);
        Pair kt[2][2];
        auto read_turned = [&](int k, Pair (&to)[2]) {
            to[0] = operand(buf + kTurned + k * 2 * kBlock);
            to[1] = operand(buf + kTurned + (k + 1) * 2 * kBlock);
        };
        if (NU > 2) read_rows(kQ, 3, ops[1]);
#pragma unroll
        for (int ti = 0; ti < 2; ++ti) el[ti] = *reinterpret_cast<const f4 *>(factors + 32 + 16 * ti + 4 * g);
        read_turned(0, kt[0]);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (NU > 2) products(ops[0], b[2], qs);
        const Pair db = split(d[0] * (el[0] * (turn * 0x1p-18f)), d[1] * (el[1] * (turn * 0x1p-18f)));
        const Pair dp = split(d[0] * 0x1p-14f, d[1] * 0x1p-14f);
        mix<6, 10>();
        __builtin_amdgcn_sched_barrier(0);
        f4 o[2];
        if constexpr (NU > 2) products(ops[1], b[3], qs);
#pragma unroll
        for (int k = 0; k < 2 * NU; k += 2) {
            if (k + 2 < 2 * NU) read_turned(k + 2, kt[k / 2 % 2 ^ 1]);
            __builtin_amdgcn_sched_barrier(0);
            f4 step[2] = {S[k], S[k + 1]};
            products(kt[k / 2 % 2], db, step);
            S[k] = step[0];
            S[k + 1] = step[1];
            if (k == 0) {
                o[0] = qs[0] * eg[0];
                o[1] = qs[1] * eg[1];
            }
            if (k == (NU > 2 ? 2 : 0)) products(p, dp, o);
            if (k == 2 * NU - 2) {
                const __amdgpu_buffer_rsrc_t rows =
                    group_rows(out + size_t(n * kChunk) * out_stride, out_stride, h * columns, v.n - n * kChunk);
#pragma unroll
                for (int ti = 0; ti < 2; ++ti)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(o[ti][r] * out_scale), rows, out_at[ti][r], 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if (n % kMeasured == kMeasured - 1) {
            float most = 0.0f;
#pragma unroll
            for (int k = 0; k < 2 * NU; ++k) most = larger(larger(most, S[k][0], S[k][1]), S[k][2], S[k][3]);
            bound = fminf(bound, most_over_groups(most) * ((DK == 128 ? 11.32f : 8.0f) * shrunk(scale)));
        }
        __syncthreads();
    } while (++n < n_groups);
    if (to) {
        int now = lane;
        asm("" : "+v"(now));  // (places worked out here, not kept over the walk)
        float *p = to + size_t(4 * (now / 16 & 3)) * columns + ((part % parts - kind * splits) * NW + wid) * 16 + now % 16;
#pragma unroll
        for (int k = 0; k < 2 * NU; ++k)
#pragma unroll
            for (int r = 0; r < 4; ++r) p[size_t(16 * k + r) * columns] = S[k][r] * shrunk(scale);
    }
}

// Few groups, drafts mostly: all of the above in one workgroup per sequence and head, that makes a group's matrices
// itself and has all columns of the state (16 a wave), so that the norm needs no launch of its own. Two workgroups of a
// CU. 8 sequences of 5 to 16 tokens and 32 heads 15.2 us: launch and loads, then eleven steps between barriers.
template <int DK, int DV>
__global__ __launch_bounds__(512, 4) void delta_group_kernel(DeltaArgs a) {
    constexpr int NU = DK / 32, kRows = 2 * NU * 2 * kBlock;
    __shared__ __attribute__((aligned(16))) char rows[3 * kRows];  // k, its transpose and q as operands
    __shared__ __attribute__((aligned(16))) char matrices[8 * kBlock];
    __shared__ __attribute__((aligned(16))) Square squares[4];  // k k', q k', A, T; then the outputs
    static_assert(sizeof(squares) >= 32 * (DV + 4) * 4);
    __shared__ float sums[2][32][NU];
    __shared__ __attribute__((aligned(16))) float inv[2][32], factors[kFactors];
    __shared__ double G[32];
    __shared__ float beta[32];
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // (24 and 32 sequences of 9 to 192 tokens 100 and 125 us in their order, 75 and 112 longest first; of up to 64
    // tokens 47 and 44 but 56 and 58, 64 sequences 112 and 122: no order for up to three groups)
    const int number = int(blockIdx.x / unsigned(a.v_heads)), h = int(blockIdx.x % unsigned(a.v_heads));
    const int s = a.max_new > 3 * kChunk ? by_length(a.b, number) : number;
    const int hk = h / (a.v_heads / a.qk_heads);
    const StateSeq v = state_seq(a.b, s);
    const int col = wid * 16 + threadIdx.x % 16;
    const bool walks = wid < DV / 16, has_item = DK == 128 || wid < 4;
    const size_t place = size_t(h) * DK * DV + size_t(4 * (threadIdx.x % 64 / 16)) * DV + col, pool = size_t(a.v_heads) * DK * DV;
    const f4 zero = {0.f, 0.f, 0.f, 0.f};
    f4 x[4], S[2 * NU];
    auto load_rows = [&](int t, int n) {
        if (has_item) Item<DK>(t % 256, wid / 4).load(a, hk, v.r0 + n * kChunk, v.n - n * kChunk, x);
    };
    load_rows(threadIdx.x, 0);
#pragma unroll
    for (int k = 0; k < 2 * NU; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r) S[k][r] = walks && v.in >= 0 ? a.state[size_t(v.in) * pool + place + size_t(16 * k + r) * DV] : 0.0f;
    float bound = __builtin_huge_valf();
    int scale = -kScale;  // S is kept times grown(scale)
    const int n_groups = (v.n + kChunk - 1) / kChunk;
    for (int n = 0; n < n_groups; ++n) {
        const int r0 = v.r0 + n * kChunk, left = v.n - n * kChunk;
        int t = threadIdx.x;
        asm("" : "+v"(t));  // there is one group mostly: no places in LDS are worked out ahead of the loop, for which registers lack
        t &= 511;
        const int lane = t % 64, g = lane / 16, lane_at = g * 256 + (lane % 16 ^ g) * 16;
        f4 val[2];
        const __amdgpu_buffer_rsrc_t v_rows = group_rows(a.v + size_t(r0) * a.v_stride + size_t(h) * DV, a.v_stride, h * DV, left);
#pragma unroll
        for (int ti = 0; ti < 2; ++ti)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                val[ti][r] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(
                    v_rows, (unsigned(16 * ti + 4 * g + r) * unsigned(a.v_stride) + unsigned(walks ? col : 0)) * 4u, 0, 0));
        const Item<DK> it(t % 256, wid / 4);
        if (has_item) row_squares<DK>(it, x, sums);
        if (wid == 7 && lane < 32) head_steps(a, r0 + lane, h, lane, lane < left, G, beta);
        __syncthreads();
        if (wid == 0) inv[lane / 32][lane % 32] = inverse_length<DK>(sums[lane / 32][lane % 32], a.qk_eps);
        if (t >= 512 - kFactors) factors[t - (512 - kFactors)] = factor_of(G, beta, t - (512 - kFactors));
        __syncthreads();
        if (has_item) {
            h4 hi[4], lo[4];
            it.convert(x, *reinterpret_cast<const f4 *>(&inv[it.is_q][it.token]), hi, lo);
            it.store(rows + it.is_q * 2 * kRows, it.is_q ? nullptr : rows + kRows, hi, lo);
        }
        __syncthreads();
        if (n + 1 < n_groups) load_rows(t, n + 1);
        if (wid < 6) store_tile(wid, lane, tile_of<DK>(wid, lane, rows, rows + 2 * kRows), squares[0], squares[1]);
        __syncthreads();
        const int i = t / 8, c = t % 8 * 4;
        if (t < 256)
            store_operand(matrices + 4 * kBlock, i, operand_at(i, c), mask_and_decay(squares[0], squares[1], G, beta, i, c, squares[2]));
        __syncthreads();
        if (wid == 7) {  // (the others have products to make meanwhile)
            if (lane < 32) invert_half(squares[2], lane / 16 * 16, lane % 16, squares[3]);
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();  // lanes read what others of the wave wrote
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            invert_corner(squares[2], lane, squares[3]);
        }
        f4 ks[2] = {zero, zero}, qs[2] = {zero, zero};
        float sum = 0.0f;
        if (walks) {
#pragma unroll
            for (int ti = 0; ti < 2; ++ti)
#pragma unroll
                for (int r = 0; r < 4; ++r) sum += fabsf(val[ti][r]);
            sum = over_groups(sum);
            float state = 0.0f;
#pragma unroll
            for (int k = 0; k < 2 * NU; ++k)
#pragma unroll
                for (int r = 0; r < 4; ++r) state += fabsf(S[k][r]);
            bound = fminf(bound, over_groups(state) * shrunk(scale));  // (what the steps add up to, if that is less)
            const int next = scale_for(bound + sum);
            const float turn = two_to(next - scale);
            scale = next;
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                S[2 * u] *= turn;
                S[2 * u + 1] *= turn;
                const Pair b = split(S[2 * u], S[2 * u + 1]);
                Pair k[2], q[2];
#pragma unroll
                for (int ti = 0; ti < 2; ++ti) {
                    k[ti] = operand(rows + (ti * NU + u) * 2 * kBlock + lane_at);
                    q[ti] = operand(rows + 2 * kRows + (ti * NU + u) * 2 * kBlock + lane_at);
                }
                products(k, b, ks);
                products(q, b, qs);
                __builtin_amdgcn_sched_barrier(0);  // (registers: not all operands ahead)
            }
        }
        __syncthreads();
        if (t < 256) store_operand(matrices, i, operand_at(i, c), enlarged(squares[3], i, c));
        __syncthreads();
        float(*const out)[DV + 4] = reinterpret_cast<float(*)[DV + 4]>(squares);
        if (walks) {
            f4 eg[2], el[2], y[2], d[2] = {zero, zero};
            Pair m[2], p[2];
#pragma unroll
            for (int ti = 0; ti < 2; ++ti) {
                eg[ti] = *reinterpret_cast<const f4 *>(factors + 16 * ti + 4 * g);
                el[ti] = *reinterpret_cast<const f4 *>(factors + 32 + 16 * ti + 4 * g);
                const f4 bt = *reinterpret_cast<const f4 *>(factors + 64 + 16 * ti + 4 * g);
                m[ti] = operand(matrices + ti * 2 * kBlock + lane_at);
                p[ti] = operand(matrices + (4 + ti * 2) * kBlock + lane_at);
#pragma unroll
                for (int r = 0; r < 4; ++r) y[ti][r] = bt[r] * __builtin_fmaf(eg[ti][r] * -0x1p-4f, ks[ti][r], val[ti][r] * grown(scale));
            }
            products(m, split(y[0], y[1]), d);
            f4 o[2] = {qs[0] * eg[0], qs[1] * eg[1]};
            products(p, split(d[0] * 0x1p-14f, d[1] * 0x1p-14f), o);
            const float f = a.scale * shrunk(scale, 14), all = factors[31];
#pragma unroll
            for (int ti = 0; ti < 2; ++ti)
#pragma unroll
                for (int r = 0; r < 4; ++r) out[16 * ti + 4 * g + r][col] = o[ti][r] * f;
            const Pair db = split(d[0] * (el[0] * 0x1p-18f), d[1] * (el[1] * 0x1p-18f));
            bound = __builtin_fmaf(all, bound, sum);
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                Pair kt[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) kt[j] = operand(rows + kRows + (2 * u + j) * 2 * kBlock + lane_at);
                f4 step[2] = {S[2 * u] * all, S[2 * u + 1] * all};
                products(kt, db, step);
                S[2 * u] = step[0];
                S[2 * u + 1] = step[1];
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        __syncthreads();
        write_rows<DV>(a, h, r0, min(left, kChunk), t, 512, [&](int m, int e) { return *reinterpret_cast<const float4 *>(&out[m][e]); });
        __syncthreads();
    }
    if (walks && v.out >= 0) {
#pragma unroll
        for (int k = 0; k < 2 * NU; ++k)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float y = S[k][r];
                a.state[size_t(v.out) * pool + place + size_t(16 * k + r) * DV] = n_groups ? y * shrunk(scale) : y;
            }
    }
}

// The norm and the gate of rows as the walk leaves them, in place: half a wave per row and head. Bound: memory (8192
// tokens of 32 heads 77 us, 5.2 TB/s).
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

// What a first half left goes to the second half's tokens and last state: O + scale R S and E + M S, with S the state
// in the middle, R what the tokens read of the unit vectors, O and E what the values gave; 32 rows at a time. Then, and
// for all other rows, norm and gate. S has a scale for each column, as above, and R and M one for each row, from what
// it sums to: they fall with the decays of the second half, far below 1, and what is left of the state in the middle is
// to keep its bits. Bound: memory (8192 tokens of 32 heads 100 us, 4.7 TB/s; with scales summed over waves, through LDS
// and one more barrier, 117).
template <int DK, int DV>
__global__ __launch_bounds__(512, 4) void delta_join_kernel(DeltaArgs a, DeltaScratch w, int tiles) {
    constexpr int NU = DK / 32;
    __shared__ __attribute__((aligned(16))) char rows[2 * NU * 2 * kBlock];
    __shared__ __attribute__((aligned(16))) float sum[32][DV + 4];
    __shared__ float shrink[32];  // what undoes the rows' scales
    const int t = threadIdx.x, lane = t & 63, wid = __builtin_amdgcn_readfirstlane(t >> 6);
    const int h = int(blockIdx.x % unsigned(a.v_heads)), st = int(blockIdx.x / unsigned(a.v_heads)), s = st / tiles;
    const StateSeq v = state_seq(a.b, s);
    const int n_groups = (v.n + kChunk - 1) / kChunk, middle = second_half(n_groups, true);
    const int g = lane / 16, lane_at = g * 256 + (lane % 16 ^ g) * 16, col = wid * 16 + lane % 16;
    const bool multiplies = wid < DV / 16;
    const size_t list = size_t(s) * a.v_heads + h, read_stride = size_t(a.v_heads) * DK;
    Pair b[NU];
    int scale = 0;
    if (middle < n_groups && multiplies) {
        f4 S[2 * NU];
        float bound = 0.0f;
#pragma unroll
        for (int k = 0; k < 2 * NU; ++k)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                S[k][r] = w.middle[list * DK * DV + size_t(16 * k + 4 * g + r) * DV + col];
                bound += fabsf(S[k][r]);
            }
        scale = scale_for(over_groups(bound));
#pragma unroll
        for (int u = 0; u < NU; ++u) b[u] = split(S[2 * u] * grown(scale), S[2 * u + 1] * grown(scale));
    }
    const int items = n_groups + (middle < n_groups ? DK / 32 : 0);
    for (int i = st % tiles; i < items; i += tiles) {
        const int r0 = v.r0 + i * kChunk, left = min(v.n - i * kChunk, kChunk);
        float *const out = a.out + size_t(h) * DV;
        if (i < middle) {
            if (a.gamma || a.z)
                write_rows<DV>(a, h, r0, left, t, 512, [&](int m, int e) { return load4(out + size_t(r0 + m) * a.out_stride + e); });
            continue;
        }
        const bool state = i >= n_groups;
        // DK / 4 lanes a row, so that its scale needs no exchange between waves
        const size_t stride = state ? DK : read_stride;
        const float *from = state ? w.carry + list * DK * DK + size_t(i - n_groups) * 32 * DK
                                  : w.reads + (size_t(v.r0) / 2 + size_t(i - middle) * kChunk) * read_stride + size_t(h) * DK;
        constexpr int kLanes = DK / 4, kTurns = 32 * kLanes / 512;
        const int at = t % kLanes * 4, row = t / kLanes;
        f4 x[kTurns];
#pragma unroll
        for (int j = 0; j < kTurns; ++j) {
            const int m = row + j * (512 / kLanes);
            x[j] = f4{0.f, 0.f, 0.f, 0.f};
            if (state || m < left) x[j] = *reinterpret_cast<const f4 *>(from + size_t(m) * stride + at);
        }
#pragma unroll
        for (int j = 0; j < kTurns; ++j) {
            const int m = row + j * (512 / kLanes);
            const int e = scale_for(lanes_sum<kLanes>((fabsf(x[j][0]) + fabsf(x[j][1])) + (fabsf(x[j][2]) + fabsf(x[j][3]))));
            if (at == 0) shrink[m] = shrunk(e);
            h4 hi, lo;
            split4(x[j], grown(e), hi, lo);
            char *p = rows + (m / 16 * NU + at / 32) * 2 * kBlock + operand_at(m, at % 32);
            *reinterpret_cast<h4 *>(p) = hi;
            *reinterpret_cast<h4 *>(p + kBlock) = lo;
        }
        __syncthreads();
        if (multiplies) {
            f4 c[2] = {};
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                Pair op[2];
#pragma unroll
                for (int ti = 0; ti < 2; ++ti) op[ti] = operand(rows + (ti * NU + u) * 2 * kBlock + lane_at);
                products(op, b[u], c);
            }
            const float f = (state ? 1.0f : a.scale) * shrunk(scale);
#pragma unroll
            for (int ti = 0; ti < 2; ++ti)
#pragma unroll
                for (int r = 0; r < 4; ++r) sum[16 * ti + 4 * g + r][col] = c[ti][r] * f * shrink[16 * ti + 4 * g + r];
        }
        __syncthreads();
        auto plus = [](float4 x, float4 y) { return make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w); };
        if (!state) {
            write_rows<DV>(a, h, r0, left, t, 512, [&](int m, int e) {
                return plus(load4(&sum[m][e]), load4(out + size_t(r0 + m) * a.out_stride + e));
            });
        } else if (v.out >= 0) {
            const size_t at = size_t(i - n_groups) * 32 * DV;
            float *to = a.state + (size_t(v.out) * a.v_heads + size_t(h)) * DK * DV + at;
            for (int e = 4 * t; e < 32 * DV; e += 4 * 512)
                *reinterpret_cast<float4 *>(to + e) = plus(load4(&sum[e / DV][e % DV]), load4(w.end + list * DK * DV + at + e));
        }
        __syncthreads();
    }
}

template <int DK, int NW, bool HALVES> hipError_t launch_walk(const DeltaArgs &a, const DeltaScratch &w, hipStream_t s) {
    constexpr int kBuffer = ((2 * 2 * (DK / 32) + DK / 16) * 2 + 8) * kBlock + kFactors * 4;
    const int splits = a.value_dim / (16 * NW), parts = HALVES ? 2 * splits + DK / (16 * NW) : splits;
    const int per = a.v_heads / a.qk_heads * parts;
    const int units = a.b.n_seqs * a.qk_heads;
    const dim3 grid(unsigned((units + 7) / 8) * 8u * unsigned(per));
    hipLaunchKernelGGL((delta_walk_kernel<DK, NW, HALVES>), grid, dim3(512), 2 * kBuffer, s, a, w, splits);
    return hipGetLastError();
}

template <int DK> hipError_t launch_groups(const DeltaArgs &a, const DeltaScratch &w, bool halves, int cu_count, hipStream_t s) {
    const int64_t lists = int64_t(a.b.n_seqs) * a.v_heads;
    const int64_t want = (int64_t(a.max_new) + kChunk - 1) / kChunk, most = ((int64_t(1) << 24) - 1) / lists;
    const int tiles = int(want < 1 ? 1 : want < most ? want : most);  // (the others in turns)
    const dim3 all_groups(unsigned(a.b.n_seqs) * unsigned(tiles) * unsigned(a.qk_heads));
    hipLaunchKernelGGL(delta_prepare_kernel<DK>, all_groups, dim3(256), 0, s, a, w, tiles);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    // Where workgroups of 32 columns find a CU each they are a little faster (a prompt of 8192 and 32 heads: 411 us,
    // with 64 columns 423), else those of 64 (six prompts of 4885 tokens in all: 106 us, with 32 columns 144). Halves
    // where all their workgroups find a CU: a prompt of 32 heads and 640 tokens 50 us, in one 54; of 2048 109 and 141;
    // of 8192 397 and 559.
    if (halves && want >= kHalfGroups && lists <= kHalfLists && lists * ((2 * a.value_dim + DK) / 64) <= cu_count) {
        if ((e = launch_walk<DK, 4, true>(a, w, s)) != hipSuccess) return e;
        // (each workgroup with about four items, for one reading of the state; more than four past 2^31 threads)
        const int turns = int(min((want + DK / 32 + 3) / 4, (int64_t(1) << 22) / lists));
        const dim3 grid(unsigned(lists) * unsigned(turns));
        if (a.value_dim == 64) hipLaunchKernelGGL((delta_join_kernel<DK, 64>), grid, dim3(512), 0, s, a, w, turns);
        else hipLaunchKernelGGL((delta_join_kernel<DK, 128>), grid, dim3(512), 0, s, a, w, turns);
        return hipGetLastError();
    }
    e = lists * (a.value_dim / 32) <= cu_count ? launch_walk<DK, 2, false>(a, w, s) : launch_walk<DK, 4, false>(a, w, s);
    if (e != hipSuccess || (!a.gamma && !a.z)) return e;
    const dim3 grid(unsigned(lists) * unsigned(tiles));
    if (a.value_dim == 64) hipLaunchKernelGGL(delta_norm_kernel<64>, grid, dim3(256), 0, s, a, tiles);
    else hipLaunchKernelGGL(delta_norm_kernel<128>, grid, dim3(256), 0, s, a, tiles);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_delta(const DeltaArgs &a, void *scratch, size_t scratch_bytes, int cu_count, hipStream_t s) {
    // A token at a time (T tokens) or one group of 32, of 1, 8 and 32 sequences of 32 heads: T = 4 7.8, 10.8, 22.3 us;
    // T = 8 10.8, 14.8, 31.0; T = 12 14.9, 19.6, 44; a group 10.9 to 11.5, 15.0 to 16.5, 40 to 46.
    const size_t widest = max(max(a.q_stride, a.k_stride), max(a.v_stride, a.out_stride));
    const int64_t lists = int64_t(a.b.n_seqs) * a.v_heads;
    const bool grouped = a.max_new > kStepRows && widest < (1 << 24) && lists < (1 << 20);  // (32 rows in 32 bits of bytes; threads)
    // All in one launch takes about 4 us and 8.4 for each group of the longest sequence; three launches 17 us and the
    // longer of 1.9 for each of its groups and 0.029 for each group of any head (one launch has 0.025 of that).
    // Measured, one launch and three: 1 sequence of 64 tokens 19.1, 20.4, of 128 36.7, 24.1; 8 of 64 25.2, 37.2, of 192
    // 64, 69.5; 32 of 192 171, 252. Fitted to heads of 128. Of 64 it is 14.2, 19.0; 26.2, 20.8; 17.2, 23.7; 43.5, 34.6;
    // 114, 126.
    const double steps = double((int64_t(a.max_new) + kChunk - 1) / kChunk);
    const double all = min(steps * a.b.n_seqs, double(a.b.n_rows / kChunk + a.b.n_seqs)) * a.v_heads;
    if (grouped && 8.4 * steps > 13 + max(1.9 * steps, 0.029 * all) && scratch && scratch_bytes >= delta_group_bytes(a)) {
        const bool halves = scratch_bytes >= delta_scratch_bytes(a);
        const size_t groups = size_t(delta_groups(a.b.n_rows, a.b.n_seqs));
        DeltaScratch w;
        w.matrices = static_cast<char *>(scratch);
        w.factors = reinterpret_cast<float *>(w.matrices + groups * a.v_heads * kDeltaMatrices);
        w.inverse = w.factors + groups * a.v_heads * kFactors;
        const size_t half = size_t(min(lists, kHalfLists)) * a.key_dim;
        w.middle = w.inverse + groups * a.qk_heads * 64;
        w.end = w.middle + half * a.value_dim;
        w.carry = w.end + half * a.value_dim;
        w.reads = w.carry + half * a.key_dim;
        return a.key_dim == 128 ? launch_groups<128>(a, w, halves, cu_count, s) : launch_groups<64>(a, w, halves, cu_count, s);
    }
    const dim3 grid(unsigned(a.b.n_seqs) * unsigned(a.v_heads));
#define QMM_STEP(K, V) \
    do { \
        if (grouped) hipLaunchKernelGGL((delta_group_kernel<K, V>), grid, dim3(512), 0, s, a); \
        else if (lists > 3 * int64_t(cu_count)) hipLaunchKernelGGL((delta_step_kernel<K, V, true>), grid, dim3(256), 0, s, a); \
        else hipLaunchKernelGGL((delta_step_kernel<K, V, false>), grid, dim3(256), 0, s, a); \
    } while (0)
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
