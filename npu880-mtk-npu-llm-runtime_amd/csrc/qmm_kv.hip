// qmm_kv.hip — new tokens into a paged key-value cache: head norms of queries
// and keys, position rotation, rounding to the cache's type.
//
//   norm      y = x / sqrt(mean(x^2) + eps) * gamma   over a head's D values, fp32
//   rotation  (a, b) -> f (a cos t - b sin t, b cos t + a sin t), t = pos * freq(pair)
//   store     fp16, or code = rint(x 127 / max|x|) with scale max|x| / 127; a head with a value that is
//             no number has none: codes of 0 with a scale of NaN
//
// Bound: memory. Every projection value is read once as fp32 and written once
// as fp16 (or 8 bits): 8192 tokens of 32 + 8 + 8 heads of 128 (302 MB) in 70 us (8-bit 73),
// 4.3 TB/s, where a plain fp32 -> fp16 copy of that size reaches 5.8; one token
// 4 us, of which a launch is 3. One launch, two kinds of workgroups, with 7 waves
// a SIMD (4 were a quarter slower: what is left is latency):
//  - 16 slots of one page's values, 1024 values of each token, first, as they
//    are the longer ones: the cache keeps a value's tokens side by side, so a
//    thread collects 4 values of 8 tokens, twice, and writes 16 B (8 B of codes)
//    of each; single tokens write 2 B (1 B) pieces.
//  - a row of queries and keys: a head is D / 4 lanes of four consecutive values
//    (16-B loads), so its sums stay in the lanes' own network. The row's angles
//    are reduced once per workgroup in 64 bits (positions up to 2^31 keep an
//    error below 1e-6 rad) into a table in LDS that all heads share.
#include <hip/hip_runtime.h>

#include "qmm_attn_plan.h"

namespace qmm {
namespace {

typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

constexpr float kZeroAmax = 7.8886090522101181e-31f;  // 2^-100: smaller rows are zeros (127 / max|x| stays finite)

// sum / maximum over the LPH lanes (16, 32 or 64) that hold one head: neighbours, pairs, mirrored
// halves and rows of 16 in the vector registers' own lane network, then across the rows
template <int CTRL> __device__ inline uint32_t moved(uint32_t v) {
    return uint32_t(__builtin_amdgcn_update_dpp(0, int(v), CTRL, 15, 15, true));
}
template <int LPH, typename F> __device__ inline uint32_t over_head(uint32_t v, F f) {
    v = f(v, moved<0xB1>(v));
    v = f(v, moved<0x4E>(v));
    v = f(v, moved<0x141>(v));
    v = f(v, moved<0x140>(v));
    if constexpr (LPH >= 32) {
        auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = f(a[0], a[1]);
    }
    if constexpr (LPH == 64) {
        auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        v = f(a[0], a[1]);
    }
    return v;
}
template <int LPH> __device__ inline float head_sum(float v) {
    return __uint_as_float(over_head<LPH>(
        __float_as_uint(v), [](uint32_t a, uint32_t b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); }));
}
// 1 / sqrt(x) to one step of fp32; the instruction takes no number below 2^-126
__device__ inline float inv_sqrt(float x) {
    const bool tiny = x < 0x1p-100f;
    return __builtin_amdgcn_rsqf(tiny ? x * 0x1p100f : x) * (tiny ? 0x1p50f : 1.0f);
}
// What an 8-bit cache keeps of one head: its scale, what makes codes of its values, and the codes' bits
// (none where a value is no number: 255 otherwise).
struct HeadCodes {
    float scale, inv;
    uint32_t bits;
};
// The largest magnitude over a head's lanes as an integer: there an infinity is above all numbers and
// a NaN above both, where a maximum of floats would pass over the NaN.
template <int LPH> __device__ inline HeadCodes head_codes(float4 x) {
    auto top = [](uint32_t a, uint32_t b) { return max(a, b); };
    auto size = [](float v) { return __float_as_uint(v) & 0x7fffffffu; };
    const uint32_t most = over_head<LPH>(max(max(size(x.x), size(x.y)), max(size(x.z), size(x.w))), top);
    const float am = __uint_as_float(most);
    if (most >= 0x7f800000u) return HeadCodes{__builtin_nanf(""), 0.0f, 0u};
    return am < kZeroAmax ? HeadCodes{0.0f, 0.0f, 255u} : HeadCodes{am / 127.0f, 127.0f / am, 255u};
}
__device__ inline uint32_t code8(float x, const HeadCodes &h) {
    return uint32_t(int(fminf(fmaxf(rintf(x * h.inv), -127.0f), 127.0f))) & h.bits;
}

// One row's queries and keys: workgroup `job` of `njobs` takes its share of the head
// groups, a wave HPW heads at a time. A wave's loads are all under way before it
// looks for the row's sequence, its page and its angles.
template <int D>
__device__ inline void append_qk(const AppendArgs &a, int m, int job, int njobs, float2 *cs) {
    constexpr int LPH = D / 4, HPW = 64 / LPH, NI = 5;  // lanes per head, heads per wave, groups at a time
    const int t = threadIdx.x, lane = t & 63, wid = __builtin_amdgcn_readfirstlane(t >> 6);
    const int H = a.b.n_heads, HQ = a.q ? a.q_heads : 0, heads = HQ + H;
    const int e = 4 * (lane % LPH), step = njobs * 4;  // this lane's first value of its head
    float4 x[NI];
    auto load = [&](int g0) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int head = (g0 + i * step) * HPW + lane / LPH;
            x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (head < heads)
                x[i] = head < HQ ? *reinterpret_cast<const float4 *>(a.q + size_t(m) * a.q_stride + size_t(head) * D + e)
                                 : *reinterpret_cast<const float4 *>(a.k + size_t(m) * a.k_stride + size_t(head - HQ) * D + e);
        }
    };
    const int g_first = job * 4 + wid;
    const int rot = a.rope ? a.rot_dim : 0, half = rot / 2;
    int from = 0, to = 0, axis = 0;
    double turn = 0.0;
    if (lane < a.b.n_seqs) {
        from = a.b.row_start[lane];
        to = a.b.row_start[lane + 1];
    }
    if (t < half) {
        axis = a.rope->axis[t];
        turn = a.rope->turns[t];
    }
    __builtin_amdgcn_sched_barrier(0);
    load(g_first);
    __builtin_amdgcn_sched_barrier(0);
    // the sequence that holds row m (the last one where the starts are not ascending)
    int s = -1;
    for (int s0 = 0;;) {
        const uint64_t found = __ballot(from <= m && m < to);
        if (found) s = s0 + 63 - __builtin_clzll(found);
        s0 += 64;
        if (s0 >= a.b.n_seqs) break;
        from = to = 0;
        if (s0 + lane < a.b.n_seqs) {
            from = a.b.row_start[s0 + lane];
            to = a.b.row_start[s0 + lane + 1];
        }
    }
    if (s < 0) return;  // (all waves alike)
    s = __builtin_amdgcn_readfirstlane(s);
    const SeqView v = seq_view(a.b, s);
    const int place = v.pos0 + (m - v.r0);
    if (rot) {
        if (t < half) {
            const int pos = a.pos ? a.pos[size_t(axis) * a.pos_stride + size_t(m)] : place;
            const double turns = double(pos) * turn;
            float sn, co;
            sincospif(2.0f * float(turns - rint(turns)), &sn, &co);
            cs[t] = make_float2(co * a.rope_scale, sn * a.rope_scale);
        }
        __syncthreads();
    }
    const int page = page_of(a.b, s, place, v.len);
    const int slot = place & ((1 << a.b.page_shift) - 1);
    const bool turned = e < rot, half_style = a.style == 0, first = e < half;
    const int other = (lane & ~(LPH - 1)) + (half_style && turned ? (first ? e + half : e - half) / 4 : lane % LPH);
    float2 c[4];  // this lane's cosines and sines (two of them in PAIRS style)
    if (turned) {
#pragma unroll
        for (int j = 0; j < 4; ++j) c[j] = half_style ? cs[(first ? e : e - half) + j] : cs[e / 2 + (j & 1)];
    }
    const float sg = first ? -1.0f : 1.0f;
    for (int g0 = g_first;;) {
        asm volatile("" : "+s"(g0));  // (addresses from g0 each time: five hoisted sets of them cost a third of the waves)
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int g = g0 + i * step;
            if (g * HPW >= heads) break;  // (the same for the wave)
            const int head = g * HPW + lane / LPH;
            const bool is_q = head < HQ;
            float4 y = x[i];
            const float ss = head_sum<LPH>(y.x * y.x + y.y * y.y + (y.z * y.z + y.w * y.w));
            const float *gamma = is_q ? a.q_gamma : a.k_gamma;
            if (gamma) {
                const float r = inv_sqrt(ss * (1.0f / D) + a.eps);
                const float4 w = *reinterpret_cast<const float4 *>(gamma + e);
                y = make_float4(y.x * r * w.x, y.y * r * w.y, y.z * r * w.z, y.w * r * w.w);
            }
            if (rot) {
                if (half_style) {
                    const float4 z = make_float4(__shfl(y.x, other), __shfl(y.y, other), __shfl(y.z, other), __shfl(y.w, other));
                    if (turned)
                        y = make_float4(y.x * c[0].x + sg * (z.x * c[0].y), y.y * c[1].x + sg * (z.y * c[1].y),
                                        y.z * c[2].x + sg * (z.z * c[2].y), y.w * c[3].x + sg * (z.w * c[3].y));
                } else if (turned) {
                    y = make_float4(y.x * c[0].x - y.y * c[0].y, y.y * c[0].x + y.x * c[0].y, y.z * c[1].x - y.w * c[1].y,
                                    y.w * c[1].x + y.z * c[1].y);
                }
            }
            const HeadCodes hc = a.ks ? head_codes<LPH>(y) : HeadCodes{};
            if (head >= heads) continue;
            const h4 r = {_Float16(y.x), _Float16(y.y), _Float16(y.z), _Float16(y.w)};
            if (is_q) {
                *reinterpret_cast<h4 *>(a.q_out + size_t(m) * a.q_out_stride + size_t(head) * D + e) = r;
            } else if (page >= 0) {
                const size_t cell = ((size_t(page) * H + size_t(head - HQ)) << a.b.page_shift) + size_t(slot);
                if (!a.ks) {
                    *reinterpret_cast<h4 *>(static_cast<uint16_t *>(a.kc) + cell * D + e) = r;
                } else {
                    const uint32_t w = code8(y.x, hc) | code8(y.y, hc) << 8 | code8(y.z, hc) << 16 | code8(y.w, hc) << 24;
                    *reinterpret_cast<uint32_t *>(static_cast<uint8_t *>(a.kc) + cell * D + e) = w;
                    if (e == 0) a.ks[cell] = hc.scale;
                }
            }
        }
        g0 += NI * step;
        if (g0 * HPW >= heads) break;
        load(g0);
    }
}

// the values of sequence s's new tokens in aligned groups of 16 slots, 1024
// values of a token (4 a thread) from `chunk` on; a group in two halves of 8
// slots, so that a thread holds 32 values at most
template <int D>
__device__ inline void append_v(const AppendArgs &a, int s, int group0, int ngroups, int chunk) {
    constexpr int LPH = D / 4;
    const SeqView v = seq_view(a.b, s);
    const int H = a.b.n_heads;
    const int i = chunk * 1024 + 4 * int(threadIdx.x);  // this thread's values i .. i + 3 of H * D
    const bool on = i < H * D;
    const int head = i / D, d = i % D;
    const int P = 1 << a.b.page_shift;
    const int start = max(v.pos0, 0);  // (rows at negative places have no cell)
    const SlotGroups groups = slot_groups(v);
    for (int g = groups.first + group0; g < groups.end; g += ngroups) {
        const int page = page_of(a.b, s, max(start, g * 16), v.len);
        if (page < 0) continue;
        const size_t row = (size_t(page) * H + size_t(head)) * D + size_t(d);  // the first value's row of P slots
#pragma unroll 1
        for (int p0 = g * 16; p0 < g * 16 + 16; p0 += 8) {
            const int lo = max(start, p0), hi = min(v.len, p0 + 8);
            if (lo >= hi) continue;
            const int slot = p0 & (P - 1);
            const bool whole = hi - lo == 8;
            float4 x[8];
            const float *src = a.v + size_t(v.r0 - v.pos0 + lo) * a.v_stride + i;  // (row of place p: r0 + p - pos0)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int p = p0 + j;
                x[j] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (on && p >= lo && p < hi) x[j] = *reinterpret_cast<const float4 *>(src + size_t(p - lo) * a.v_stride);
            }
            if (!a.vs) {
                if (!on) continue;
                uint16_t *dst = static_cast<uint16_t *>(a.vc) + row * size_t(P) + slot;
                if (whole) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        h8 y;
#pragma unroll
                        for (int j = 0; j < 8; ++j) y[j] = _Float16(reinterpret_cast<const float *>(&x[j])[c]);
                        *reinterpret_cast<h8 *>(dst + size_t(c) * P) = y;
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int p = p0 + j;
                        if (p < lo || p >= hi) continue;
#pragma unroll
                        for (int c = 0; c < 4; ++c)
                            reinterpret_cast<_Float16 *>(dst)[size_t(c) * P + j] = _Float16(reinterpret_cast<const float *>(&x[j])[c]);
                    }
                }
                continue;
            }
            uint32_t w[4][2] = {};  // codes: value c's 8 tokens
            uint8_t *dst = static_cast<uint8_t *>(a.vc) + row * size_t(P) + slot;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int p = p0 + j;
                if (p < lo || p >= hi) continue;
                const HeadCodes hc = head_codes<LPH>(x[j]);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const uint32_t code = code8(reinterpret_cast<const float *>(&x[j])[c], hc);
                    w[c][j / 4] |= code << (8 * (j % 4));
                    if (!whole && on) dst[size_t(c) * P + j] = uint8_t(code);
                }
                if (on && d == 0) a.vs[((size_t(page) * H + size_t(head)) << a.b.page_shift) + size_t(slot + j)] = hc.scale;
            }
            if (whole && on) {
#pragma unroll
                for (int c = 0; c < 4; ++c) *reinterpret_cast<uint2 *>(dst + size_t(c) * P) = make_uint2(w[c][0], w[c][1]);
            }
        }
    }
}

// First the values: (sequence, group of 16 slots, 1024 values) a workgroup; then the
// queries and keys, njobs workgroups a row.
template <int D>
__global__ __launch_bounds__(256) void kv_append_kernel(AppendArgs a, int njobs, int ngroups, int nchunks) {
    __shared__ float2 cs[128];
    const unsigned nv = unsigned(a.b.n_seqs) * unsigned(ngroups) * unsigned(nchunks);
    if (blockIdx.x >= nv) {
        const unsigned u = blockIdx.x - nv;
        append_qk<D>(a, int(u / unsigned(njobs)), int(u % unsigned(njobs)), njobs, cs);
        return;
    }
    const unsigned sg = blockIdx.x / unsigned(nchunks);
    append_v<D>(a, int(sg / unsigned(ngroups)), int(sg % unsigned(ngroups)), ngroups, int(blockIdx.x % unsigned(nchunks)));
}

__global__ __launch_bounds__(128) void rope_table_kernel(RopeTable t, RopeTable *dst) {
    dst->turns[threadIdx.x] = t.turns[threadIdx.x];
    dst->axis[threadIdx.x] = t.axis[threadIdx.x];
}

}  // namespace

hipError_t launch_rope_table(const RopeTable &t, RopeTable *dst, hipStream_t s) {
    hipLaunchKernelGGL(rope_table_kernel, dim3(1), dim3(128), 0, s, t, dst);
    return hipGetLastError();
}

hipError_t launch_kv_append(const AppendArgs &a, hipStream_t s) {
    const AppendGrid g = append_grid(a.b.n_rows, a.b.n_seqs, a.b.n_heads, a.head_dim, a.q ? a.q_heads : 0, a.max_new);
    if (!g.workgroups) return hipErrorInvalidValue;
    const int D = a.head_dim;
#define QMM_KV(DD) hipLaunchKernelGGL(kv_append_kernel<DD>, dim3(g.workgroups), dim3(256), 0, s, a, g.njobs, g.ngroups, g.nchunks)
    if (D == 64) QMM_KV(64);
    else if (D == 128) QMM_KV(128);
    else QMM_KV(256);
#undef QMM_KV
    return hipGetLastError();
}

}  // namespace qmm
