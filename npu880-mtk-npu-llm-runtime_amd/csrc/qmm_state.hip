// qmm_state.hip — the short causal convolution in front of the gated delta rule,
// and copies of the slots that states (and cache pages) are kept in.
//
//   y[t][c] = act(bias[c] + sum_i w[c][i] x[t - W + 1 + i][c]),  act(y) = y / (1 + exp(-y))
//
// Bound: memory; every input is read once (and W - 1 of 8 rows again, from the caches) and every output written once.
// 8192 channels: 16 sequences of a token 4.5 us (one launch), five prompts of 5581 73.5 us, 5.0 TB/s. Inputs of more
// than 32 MB are loaded past the caches, in which the outputs then lie for what reads them: 6 prompts of 800 tokens
// with the delta rule behind 237 us, 245 without. Outputs past them too are faster alone (64.5 us) and slower together
// (241). With 16 rows a workgroup 78.5 us, with 4 80.
#include <hip/hip_runtime.h>

#include "qmm_lanes.h"
#include "qmm_state.h"

namespace qmm {
namespace {

__device__ inline float4 fma4(float4 w, float4 x, float4 y) {
    return make_float4(__builtin_fmaf(w.x, x.x, y.x), __builtin_fmaf(w.y, x.y, y.y), __builtin_fmaf(w.z, x.z, y.z),
                       __builtin_fmaf(w.w, x.w, y.w));
}
template <bool PAST> __device__ inline float4 load4(const float *p) {
    if (PAST) return load_past(reinterpret_cast<const float4 *>(p));
    return *reinterpret_cast<const float4 *>(p);
}
// A workgroup: 1024 channels (4 a thread) of 8 rows of a sequence. A thread keeps the last W - 1
// inputs in registers. The first rows' workgroup alone reads and writes the carried inputs (a slot may be
// both read and written), and it reads them before it writes.
template <int W, bool PAST>
__global__ __launch_bounds__(256) void conv_kernel(ConvArgs a, int tiles, int chunks) {
    const int chunk = int(blockIdx.x % unsigned(chunks)), st = int(blockIdx.x / unsigned(chunks));
    const int s = st / tiles;
    const int c = chunk * 1024 + 4 * int(threadIdx.x);
    if (c >= a.channels) return;
    const StateSeq v = state_seq(a.b, s);
    const float *x = a.x + size_t(v.r0) * a.x_stride + c;
    float *out = a.out + size_t(v.r0) * a.out_stride + c;
    float4 w[W], bias = make_float4(0.f, 0.f, 0.f, 0.f);
    const float *wc = a.weight + size_t(c) * W;
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = make_float4(wc[i], wc[W + i], wc[2 * W + i], wc[3 * W + i]);
    if (a.bias) bias = *reinterpret_cast<const float4 *>(a.bias + c);
    auto carried = [&](int slot, int i) { return a.state + (size_t(slot) * (W - 1) + size_t(i)) * size_t(a.channels) + c; };
    for (int tile = st % tiles; tile == 0 || tile * int64_t(kConvRows) < v.n; tile += tiles) {
        const int t0 = tile * kConvRows, t1 = min(t0 + kConvRows, v.n);
        float4 last[W - 1];  // inputs t - W + 1 .. t - 1
#pragma unroll
        for (int i = 0; i < W - 1; ++i) {
            const int p = t0 - (W - 1) + i;
            last[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (tile > 0) last[i] = *reinterpret_cast<const float4 *>(x + size_t(p) * a.x_stride);
            else if (v.in >= 0) last[i] = *reinterpret_cast<const float4 *>(carried(v.in, i));
        }
        float4 in[kConvRows];
#pragma unroll
        for (int j = 0; j < kConvRows; ++j) {
            in[j] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (t0 + j < t1) in[j] = load4<PAST>(x + size_t(t0 + j) * a.x_stride);
        }
#pragma unroll
        for (int j = 0; j < kConvRows; ++j) {
            if (t0 + j >= t1) break;
            float4 y = bias;
#pragma unroll
            for (int i = 0; i < W - 1; ++i) y = fma4(w[i], last[i], y);
            y = fma4(w[W - 1], in[j], y);
            if (a.silu) y = make_float4(silu(y.x), silu(y.y), silu(y.z), silu(y.w));
            *reinterpret_cast<float4 *>(out + size_t(t0 + j) * a.out_stride) = y;
#pragma unroll
            for (int i = 0; i + 1 < W - 1; ++i) last[i] = last[i + 1];
            last[W - 2] = in[j];
        }
        if (tile == 0 && v.out >= 0) {
            float4 left[W - 1];  // the inputs after the last row, all read before the first is written
#pragma unroll
            for (int i = 0; i < W - 1; ++i) {
                const int p = v.n - (W - 1) + i;
                left[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (p >= 0) left[i] = *reinterpret_cast<const float4 *>(x + size_t(p) * a.x_stride);
                else if (v.in >= 0) left[i] = *reinterpret_cast<const float4 *>(carried(v.in, W - 1 + p));
            }
#pragma unroll
            for (int i = 0; i < W - 1; ++i) *reinterpret_cast<float4 *>(carried(v.out, i)) = left[i];
        }
    }
}

// 16 KB of one pair's slot in one pool a workgroup: four 16-B loads of a thread under way. Bound: memory, 6.1 to 6.6
// TB/s at 200 MB (stores past the caches: 7 more of 51 us here, but lost again where the copies are read next).
constexpr int kCopyChunk = 16384;
__global__ __launch_bounds__(256) void copy_kernel(CopyArgs a) {
    const auto pool = a.pool[blockIdx.z];
    for (int i = int(blockIdx.y); i < a.n; i += int(gridDim.y)) {
        const int src = a.src[i], dst = a.dst[i];
        if (unsigned(src) >= unsigned(pool.slots) || unsigned(dst) >= unsigned(pool.slots) || src == dst) continue;
        const uint4 *from = reinterpret_cast<const uint4 *>(pool.base + size_t(src) * pool.bytes);
        uint4 *to = reinterpret_cast<uint4 *>(pool.base + size_t(dst) * pool.bytes);
        const size_t n = pool.bytes / 16;
        for (size_t at = size_t(blockIdx.x) * (kCopyChunk / 16); at < n; at += size_t(gridDim.x) * (kCopyChunk / 16)) {
            uint4 x[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const size_t e = at + size_t(j) * 256 + threadIdx.x;
                x[j] = e < n ? from[e] : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const size_t e = at + size_t(j) * 256 + threadIdx.x;
                if (e < n) to[e] = x[j];
            }
        }
    }
}

}  // namespace

hipError_t launch_conv(const ConvArgs &a, hipStream_t s) {
    const int chunks = (a.channels + 1023) / 1024, tiles = conv_tiles(a.b, a.channels, a.max_new);
    const dim3 grid(unsigned(a.b.n_seqs) * unsigned(tiles) * unsigned(chunks));
    const bool past = size_t(a.b.n_rows) * size_t(a.channels) * 4 > (32u << 20);
#define QMM_CONV(W) \
    do { \
        if (past) hipLaunchKernelGGL((conv_kernel<W, true>), grid, dim3(256), 0, s, a, tiles, chunks); \
        else hipLaunchKernelGGL((conv_kernel<W, false>), grid, dim3(256), 0, s, a, tiles, chunks); \
    } while (0)
    if (a.width == 2) QMM_CONV(2);
    else if (a.width == 3) QMM_CONV(3);
    else QMM_CONV(4);
#undef QMM_CONV
    return hipGetLastError();
}

hipError_t launch_copy(const CopyArgs &a, int n_pools, size_t most_bytes, hipStream_t s) {
    const size_t chunks = (most_bytes + kCopyChunk - 1) / kCopyChunk;
    const unsigned pairs = unsigned(a.n < 4096 ? a.n : 4096);  // (the others in turns; below 2^31 workgroups)
    const size_t most = ((size_t(1) << 31) - 1) / 256 / (size_t(pairs) * size_t(n_pools));
    const dim3 grid(unsigned(chunks < most ? chunks : most < 1 ? 1 : most), pairs, unsigned(n_pools));
    hipLaunchKernelGGL(copy_kernel, grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace qmm
