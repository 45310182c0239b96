// qmm_kv.hip — new tokens into a paged key-value cache: head norms of queries
// and keys, position rotation, rounding to the cache's type.
//
//   norm      y = x / sqrt(mean(x^2) + eps) * gamma   over a head's D values, fp32
//   rotation  (a, b) -> f (a cos t - b sin t, b cos t + a sin t), t = pos * freq(pair)
//   store     fp16, or code = rint(x 127 / max|x|) with scale max|x| / 127
//
// Bound: memory. Every projection value is read once as fp32 and written once
// as fp16 (or 8 bits). One launch, two kinds of workgroups:
//  - a row of queries and keys: a head is D / 4 lanes of four consecutive
//    values (16-B loads), so its sums are a few lane exchanges; the row's
//    angles are reduced once per workgroup in 64 bits (positions up to 2^31
//    keep an error below 1e-6 rad) into a table in LDS that all heads share.
//  - 16 slots of one page's values, 1024 values of each token: the cache keeps
//    a value's tokens side by side, so a thread collects 4 values of up to 16
//    tokens and writes 32 B (16 B of 8-bit codes) of each; single tokens write
//    2 B (1 B) pieces.
#include <hip/hip_runtime.h>

#include "qmm_attn.h"

namespace qmm {
namespace {

typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

constexpr float kZeroAmax = 7.8886090522101181e-31f;  // 2^-100: smaller rows are zeros (127 / max|x| stays finite)

// sum / maximum over the LPH lanes that hold one head
template <int LPH> __device__ inline float head_sum(float v) {
#pragma unroll
    for (int o = 1; o < LPH; o *= 2) v += __shfl_xor(v, o);
    return v;
}
template <int LPH> __device__ inline float head_max(float v) {
#pragma unroll
    for (int o = 1; o < LPH; o *= 2) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}
__device__ inline float abs_max4(float4 x) {
    return fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
}
__device__ inline int code8(float x, float inv) { return int(fminf(fmaxf(rintf(x * inv), -127.0f), 127.0f)); }

// one row's queries and keys; job j of nj takes its share of the head groups
template <int D>
__device__ inline void append_qk(const AppendArgs &a, int m, int job, int njobs, float2 *cs, int *found) {
    constexpr int LPH = D / 4, HPW = 64 / LPH;  // lanes per head, heads per wave
    const int t = threadIdx.x, lane = t & 63, wid = t >> 6;
    // the sequence that holds row m (the last one where the starts are not ascending)
    if (t == 0) *found = -1;
    __syncthreads();
    for (int s = t; s < a.b.n_seqs; s += 256)
        if (a.b.row_start[s] <= m && m < a.b.row_start[s + 1]) atomicMax(found, s);
    __syncthreads();
    const int s = *found;
    if (s < 0) return;
    const SeqView v = seq_view(a.b, s);
    const int place = v.pos0 + (m - v.r0);
    const int rot = a.rope.rot_dim, half = rot / 2;
    if (rot) {
        if (t < half) {
            const int pos = a.pos ? a.pos[size_t(a.rope.axis[t]) * a.pos_stride + size_t(m)] : place;
            const double turns = double(pos) * a.rope.turns[t];
            float sn, co;
            sincospif(2.0f * float(turns - rint(turns)), &sn, &co);
            cs[t] = make_float2(co * a.rope.scale, sn * a.rope.scale);
        }
        __syncthreads();
    }
    const int page = page_of(a.b, s, place, v.len);
    const int slot = place & ((1 << a.b.page_shift) - 1);
    const int H = a.b.n_heads, HQ = a.q ? a.q_heads : 0, heads = HQ + H;
    const int e = 4 * (lane % LPH);  // this lane's first value of its head
    const bool turned = e < rot, half_style = a.rope.style == 0;
    const bool first = e < half;
    const int other = (lane & ~(LPH - 1)) + (half_style && turned ? (first ? e + half : e - half) / 4 : lane % LPH);
    for (int g = job * 4 + wid; g * HPW < heads; g += njobs * 4) {
        const int head = g * HPW + lane / LPH;
        const bool on = head < heads, is_q = head < HQ;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (on)
            x = is_q ? *reinterpret_cast<const float4 *>(a.q + size_t(m) * a.q_stride + size_t(head) * D + e)
                     : *reinterpret_cast<const float4 *>(a.k + size_t(m) * a.k_stride + size_t(head - HQ) * D + e);
        const float *gamma = is_q ? a.q_gamma : a.k_gamma;
        const float ss = head_sum<LPH>(x.x * x.x + x.y * x.y + (x.z * x.z + x.w * x.w));
        if (gamma) {
            const float r = 1.0f / sqrtf(ss / float(D) + a.eps);
            const float4 w = *reinterpret_cast<const float4 *>(gamma + e);
            x = make_float4(x.x * r * w.x, x.y * r * w.y, x.z * r * w.z, x.w * r * w.w);
        }
        if (rot) {
            if (half_style) {
                const float4 y = make_float4(__shfl(x.x, other), __shfl(x.y, other), __shfl(x.z, other), __shfl(x.w, other));
                if (turned) {
                    const float2 *c = cs + (first ? e : e - half);
                    const float sg = first ? -1.0f : 1.0f;
                    x = make_float4(x.x * c[0].x + sg * (y.x * c[0].y), x.y * c[1].x + sg * (y.y * c[1].y),
                                    x.z * c[2].x + sg * (y.z * c[2].y), x.w * c[3].x + sg * (y.w * c[3].y));
                }
            } else if (turned) {
                const float2 c0 = cs[e / 2], c1 = cs[e / 2 + 1];
                x = make_float4(x.x * c0.x - x.y * c0.y, x.y * c0.x + x.x * c0.y, x.z * c1.x - x.w * c1.y,
                                x.w * c1.x + x.z * c1.y);
            }
        }
        const float am = a.ks ? head_max<LPH>(abs_max4(x)) : 0.0f;
        if (!on) continue;
        const h4 y = {_Float16(x.x), _Float16(x.y), _Float16(x.z), _Float16(x.w)};
        if (is_q) {
            *reinterpret_cast<h4 *>(a.q_out + size_t(m) * a.q_out_stride + size_t(head) * D + e) = y;
        } else if (page >= 0) {
            const size_t cell = ((size_t(page) * H + size_t(head - HQ)) << a.b.page_shift) + size_t(slot);
            if (!a.ks) {
                *reinterpret_cast<h4 *>(static_cast<uint16_t *>(a.kc) + cell * D + e) = y;
            } else {
                const float inv = am < kZeroAmax ? 0.0f : 127.0f / am;
                const uint32_t w = (code8(x.x, inv) & 255) | (code8(x.y, inv) & 255) << 8 | (code8(x.z, inv) & 255) << 16 |
                                   uint32_t(code8(x.w, inv)) << 24;
                *reinterpret_cast<uint32_t *>(static_cast<uint8_t *>(a.kc) + cell * D + e) = w;
                if (e == 0) a.ks[cell] = am < kZeroAmax ? 0.0f : am / 127.0f;
            }
        }
    }
}

// the values of sequence s's new tokens in aligned groups of 16 slots, 1024
// values of a token (4 a thread) from `chunk` on
template <int D>
__device__ inline void append_v(const AppendArgs &a, int s, int group0, int ngroups, int chunk) {
    constexpr int LPH = D / 4;
    const SeqView v = seq_view(a.b, s);
    const int H = a.b.n_heads;
    const int i = chunk * 1024 + 4 * int(threadIdx.x);  // this thread's values i .. i + 3 of H * D
    const bool on = i < H * D;
    const int head = i / D, d = i % D;
    const int P = 1 << a.b.page_shift;
    const int first = max(v.pos0, 0) >> 4;  // (rows at negative places have no cell)
    for (int g = first + group0; g * 16 < v.len; g += ngroups) {
        const int lo = max(max(v.pos0, 0), g * 16), hi = min(v.len, g * 16 + 16);
        if (lo >= hi) break;
        const int page = page_of(a.b, s, lo, v.len);
        if (page < 0) continue;
        const int slot = (g * 16) & (P - 1);
        float4 x[16];
        const float *src = a.v + size_t(v.r0 - v.pos0 + lo) * a.v_stride + i;  // (row of place p: r0 + p - pos0)
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const int p = g * 16 + j;
            x[j] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (on && p >= lo && p < hi) x[j] = *reinterpret_cast<const float4 *>(src + size_t(p - lo) * a.v_stride);
        }
        const size_t row = (size_t(page) * H + size_t(head)) * D + size_t(d);  // the first value's row of P slots
        const bool whole = hi - lo == 16;
        if (!a.vs) {
            if (!on) continue;
            uint16_t *dst = static_cast<uint16_t *>(a.vc) + row * size_t(P) + slot;
            if (whole) {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    h8 y[2];
#pragma unroll
                    for (int j = 0; j < 16; ++j) y[j / 8][j % 8] = _Float16(reinterpret_cast<const float *>(&x[j])[c]);
                    *reinterpret_cast<h8 *>(dst + size_t(c) * P) = y[0];
                    *reinterpret_cast<h8 *>(dst + size_t(c) * P + 8) = y[1];
                }
            } else {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const int p = g * 16 + j;
                    if (p < lo || p >= hi) continue;
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        reinterpret_cast<_Float16 *>(dst)[size_t(c) * P + j] = _Float16(reinterpret_cast<const float *>(&x[j])[c]);
                }
            }
            continue;
        }
        uint32_t w[4][4] = {};  // codes: value c's 16 tokens
        uint8_t *dst = static_cast<uint8_t *>(a.vc) + row * size_t(P) + slot;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const int p = g * 16 + j;
            if (p < lo || p >= hi) continue;
            const float am = head_max<LPH>(abs_max4(x[j]));
            const float inv = am < kZeroAmax ? 0.0f : 127.0f / am;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const uint32_t code = uint32_t(code8(reinterpret_cast<const float *>(&x[j])[c], inv)) & 255u;
                w[c][j / 4] |= code << (8 * (j % 4));
                if (!whole && on) dst[size_t(c) * P + j] = uint8_t(code);
            }
            if (on && d == 0)
                a.vs[((size_t(page) * H + size_t(head)) << a.b.page_shift) + size_t(slot + j)] = am < kZeroAmax ? 0.0f : am / 127.0f;
        }
        if (whole && on) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
                *reinterpret_cast<uint4 *>(dst + size_t(c) * P) = make_uint4(w[c][0], w[c][1], w[c][2], w[c][3]);
        }
    }
}

// Workgroups 0 .. n_rows * njobs - 1: queries and keys of a row; then
// (sequence, group of 16 slots, 1024 values) of the values.
template <int D>
__global__ __launch_bounds__(256) void kv_append_kernel(AppendArgs a, int njobs, int ngroups, int nchunks) {
    __shared__ float2 cs[128];
    __shared__ int found;
    const unsigned nqk = unsigned(a.b.n_rows) * unsigned(njobs);
    if (blockIdx.x < nqk) {
        append_qk<D>(a, int(blockIdx.x / unsigned(njobs)), int(blockIdx.x % unsigned(njobs)), njobs, cs, &found);
        return;
    }
    const unsigned u = blockIdx.x - nqk;
    const int chunk = int(u % unsigned(nchunks));
    const unsigned sg = u / unsigned(nchunks);
    append_v<D>(a, int(sg / unsigned(ngroups)), int(sg % unsigned(ngroups)), ngroups, chunk);
}

}  // namespace

hipError_t launch_kv_append(const AppendArgs &a, hipStream_t s) {
    const int D = a.head_dim, hpw = 256 / D;
    const int groups = ((a.q ? a.q_heads : 0) + a.b.n_heads + hpw - 1) / hpw;  // head groups of a row, one a wave
    // few rows: every head group its own wave; many: one workgroup a row, the angles reduced once
    int njobs = 1;
    while (njobs * 4 < groups && int64_t(a.b.n_rows) * njobs < 1024) ++njobs;
    const int ngroups = (a.max_new + 14) / 16 + 1;  // aligned groups that max_new tokens can touch
    const int nchunks = (a.b.n_heads * D + 1023) / 1024;
    const uint64_t grid = uint64_t(a.b.n_rows) * uint64_t(njobs) + uint64_t(a.b.n_seqs) * uint64_t(ngroups) * uint64_t(nchunks);
    if (grid >= (uint64_t(1) << 31)) return hipErrorInvalidValue;
#define QMM_KV(DD) hipLaunchKernelGGL(kv_append_kernel<DD>, dim3(unsigned(grid)), dim3(256), 0, s, a, njobs, ngroups, nchunks)
    if (D == 64) QMM_KV(64);
    else if (D == 128) QMM_KV(128);
    else QMM_KV(256);
#undef QMM_KV
    return hipGetLastError();
}

}  // namespace qmm
