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

constexpr int kGroup = 8;   // tokens whose inputs are in LDS at a time

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

}  // namespace

hipError_t launch_delta(const DeltaArgs &a, void *, size_t, int, hipStream_t s) {
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
