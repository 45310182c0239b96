// qmm_beam.hip — the best continuations of an item's beams over the vocabulary.
//
//   total(b, j) = score[b] + x_bj - lse_b,  lse_b = m + log(sum_j exp(x_bj - m))
//
// Within a beam the order of totals is that of the logits (equal ones: the lower
// token first), so a logit and its place make one key of 64 bits, all different:
// the logit's bits as an ordered whole number, then the place's complement. Two
// launches:
//  - a wave reads 2048 logits once, into registers: their maximum, the sum of
//    exponentials (fp32), and the n_keep best keys. Those lie above the n_keep-th
//    of the lanes' own best keys, which few others do; they are collected in LDS
//    and put in order by counting.
//  - a workgroup per item: a wave per beam joins the beam's lists the same way and
//    the sums in 64 bits; then every candidate's rank is the number of those before
//    it, by bisection in the beams' lists, which are in order.
// Bound: memory (the logits are read once) for many rows, else the latency of the two launches. 4 beams over 151936
// tokens, 8 kept: 5.8 + 5.8 us; 128 beams of 16 items, 16 kept: 17.9 (3.7 TB/s: some 500 vector instructions a wave,
// 8.6 us of issue in all, and the scalar ones of its searches between them) + 8.7. Keys are found by their upper half
// first: a search of 16 ballots, not 64 (35.1 us for both launches with 64, 28.5 so).
#include <hip/hip_runtime.h>

#include "qmm_lanes.h"
#include "qmm_state.h"

namespace qmm {
namespace {

constexpr int kPerLane = kBeamSlice / 64;
constexpr float kInf = __builtin_huge_valf(), kLog2e = 1.4426950408889634f;

__device__ inline uint32_t ordered(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);  // (-0 counts as 0)
    return u ^ (u & 0x80000000u ? 0xffffffffu : 0x80000000u);
}
__device__ inline float unordered(uint32_t u) { return __uint_as_float(u ^ (u & 0x80000000u ? 0x80000000u : 0xffffffffu)); }
__device__ inline float allowed(float x) { return x < kInf ? x : -kInf; }  // NaN and +infinity count as ruled out

// What the wave's lanes wrote to LDS is read by its other lanes after this.
__device__ inline void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// The largest T of the bits `from` .. `to` - 1 (the lower ones 0, those above as in T) that at least n of the lanes
// where `on` have at or above.
__device__ inline uint32_t nth_bits(uint32_t x, bool on, int n, uint32_t T, int from, int to) {
#pragma unroll 1
    for (int bit = to - 1; bit >= from; --bit) {
        const uint32_t c = T | 1u << bit;
        if (__popcll(__ballot(on && x >= c)) >= n) T = c;
    }
    return T;
}
// The largest key T with at least `n` of the lanes' keys (all different, or 0 for none) at or above it; 0
// where there are fewer.
__device__ inline uint64_t nth_key(uint64_t key, int n) {
    const uint32_t hi = uint32_t(key >> 32), lo = uint32_t(key);
    const uint32_t T = nth_bits(hi, true, n, 0, 0, 32);
    const int need = n - __popcll(__ballot(hi > T));
    if (__popcll(__ballot(hi == T)) <= need) return uint64_t(T) << 32;
    return uint64_t(T) << 32 | nth_bits(lo, hi == T, need, 0, 0, 32);
}

// The n_keep best of `n` different keys in LDS, in order, to `out` (0 where there are fewer): by counting
// the larger ones. More than 64 are first cut down to those at or above the n_keep-th, found by its bits.
__device__ inline void keep_best(uint64_t *key, int n, int n_keep, uint64_t *out) {
    const int lane = threadIdx.x & 63;
    wave_sync();
    if (n > 64) {
        uint64_t T = 0;
#pragma unroll 1
        for (int bit = 63; bit >= 0; --bit) {
            const uint64_t c = T | uint64_t(1) << bit;
            int count = 0;
            for (int i = lane; i - lane < n; i += 64) count += __popcll(__ballot(i < n && key[i] >= c));
            if (count >= n_keep) T = c;
        }
        int kept = 0;  // (written at or before where they were read)
        for (int i = lane; i - lane < n; i += 64) {
            const uint64_t k = i < n ? key[i] : 0;
            const bool in = i < n && k >= T;
            const uint64_t who = __ballot(in);
            if (in) key[kept + __popcll(who & ((uint64_t(1) << lane) - 1))] = k;
            kept += __popcll(who);
        }
        n = kept;
    }
    wave_sync();
    const uint64_t mine = lane < n ? key[lane] : 0;
    int before = 0;
    for (int i = 0; i < n; ++i) before += key[i] > mine;
    if (lane < n && before < n_keep) out[before] = mine;
    if (lane >= n && lane < n_keep) out[lane] = 0;
}

__global__ __launch_bounds__(256) void beam_slice_kernel(BeamArgs a, int slices) {
    extern __shared__ uint64_t found[];  // a wave's candidates: at most n_keep lanes' logits
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t u = int64_t(blockIdx.x) * 4 + wid;
    const int row = int(u / slices), slice = int(u % slices);
    if (row >= a.n_items * a.n_beams) return;
    if (a.ended && a.ended[row]) return;
    const int first = slice * kBeamSlice, n = min(kBeamSlice, a.vocab - first);
    const float *x = a.logits + size_t(row) * a.stride + first;
    uint64_t *list = found + wid * a.n_keep * kPerLane;
    float v[kPerLane];
    // Place of this lane's value i: 4 neighbours, one load, at whatever 4-B address the row begins (16-B loads need no
    // more). The same for all rows: beams alike add their exponentials in one order and get the same bits, so that the
    // lower one comes first. 6 rows of 50257 logits without a gap, whose addresses differ: 12.3 us (13.0 with a load a
    // value where a row was not 16-B aligned).
    typedef float AnyFour __attribute__((ext_vector_type(4), aligned(4)));
    auto place = [&](int i) { return (i / 4) * 256 + 4 * lane + i % 4; };
#pragma unroll
    for (int i = 0; i < kPerLane; i += 4) {
        const int e = place(i);
        if (e + 3 < n) {
            const AnyFour y = *reinterpret_cast<const AnyFour *>(x + e);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[i + j] = y[j];
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[i + j] = e + j < n ? x[e + j] : -kInf;
        }
    }
    // First as if all were numbers or -infinity; where one is not, the sum is no number, or infinite.
    float top, m, sum;
    auto look = [&] {
        top = fmaxf(v[0], v[1]);
#pragma unroll
        for (int i = 2; i < kPerLane; i += 2) top = fmaxf(fmaxf(top, v[i]), v[i + 1]);
        m = lanes_max<64>(top);
        const float base = m == -kInf ? 0.0f : m;
        float s[4] = {};
#pragma unroll
        for (int i = 0; i < kPerLane; ++i) s[i % 4] += __builtin_amdgcn_exp2f((v[i] - base) * kLog2e);  // (a rounded base would shift all)
        sum = lanes_sum<64>((s[0] + s[1]) + (s[2] + s[3]));
    };
    look();
    if (!(sum < kInf)) {
#pragma unroll
        for (int i = 0; i < kPerLane; ++i) v[i] = allowed(v[i]);
        look();
    }
    if (lane == 0) {
        float *st = a.stat + (size_t(row) * slices + slice) * 2;
        st[0] = m;
        st[1] = sum;
    }
    // The n_keep-th of the lanes' largest values, first by its upper half: seldom do more lanes reach that.
    uint32_t T = nth_bits(ordered(top), true, a.n_keep, 0, 16, 32), T_place = 0;
    if (__popcll(__ballot(ordered(top) >= T)) > a.n_keep) {
        T = nth_bits(ordered(top), true, a.n_keep, T, 0, 16);
        const bool at_T = ordered(top) == T;
        const int need = a.n_keep - __popcll(__ballot(ordered(top) > T));
        if (__popcll(__ballot(at_T)) > need) {  // equal values: those of the lanes whose first one comes first
            uint32_t first_at = 0;
#pragma unroll
            for (int i = kPerLane - 1; i >= 0; --i)
                if (v[i] == top && place(i) < n) first_at = ~uint32_t(first + place(i));
            T_place = nth_bits(first_at, at_T, need, 0, 0, 32);
        }
    }
    const uint64_t T_key = uint64_t(T) << 32 | T_place;
    // (the least float that is at or above T; all of them where T is below -infinity)
    const float T_value = T < ordered(-kInf) ? -kInf : unordered(T);
    int count = 0;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
        if (__ballot(v[i] >= T_value) == 0) continue;
        const uint64_t key = uint64_t(ordered(v[i])) << 32 | uint32_t(~uint32_t(first + place(i)));
        const bool in = key >= T_key && place(i) < n;
        const uint64_t who = __ballot(in);
        if (in) list[count + __popcll(who & ((uint64_t(1) << lane) - 1))] = key;
        count += __popcll(who);
    }
    keep_best(list, count, a.n_keep, a.list + (size_t(row) * slices + slice) * a.n_keep);
}

constexpr int kJoinCap = 512;  // candidates of one beam in LDS

// The n_keep best of a beam's lists (each in order, 0 past its end) by one wave. Collected are those at or
// above the n_keep-th of the lanes' best keys (a lane has every 64th list) or, of fewer lists, above the
// least of their keys at a depth that makes n_keep of them. Where values lie so that those are too many, the
// best is taken n_keep times instead.
__device__ inline void join_lists(const uint64_t *lists, int slices, int full, int n_keep, uint64_t *cand, int *counter, uint64_t *out) {
    const int lane = threadIdx.x & 63;
    uint64_t T = 0;
    constexpr int kFirst = 4;  // keys of a list that are read at once
    uint64_t first[2][kFirst];  // of this lane's first two lists
#pragma unroll
    for (int l = 0; l < 2; ++l)
#pragma unroll
        for (int i = 0; i < kFirst; ++i) first[l][i] = lane + 64 * l < slices && i < n_keep ? lists[size_t(lane + 64 * l) * n_keep + i] : 0;
    if (full >= n_keep) {
        uint64_t head = first[0][0] > first[1][0] ? first[0][0] : first[1][0];  // the best of this lane's lists
        for (int s = lane + 128; s < slices; s += 64) {
            const uint64_t k = lists[size_t(s) * n_keep];
            head = k > head ? k : head;
        }
        T = nth_key(head, n_keep);
    } else if (full > 0) {  // (lists of full slices have n_keep keys; fewer than 64 lists)
        const uint64_t k = lane < full ? lists[size_t(lane) * n_keep + (n_keep + full - 1) / full - 1] : ~uint64_t(0);
        const uint32_t hi = ~lanes_max<64>(~uint32_t(k >> 32));
        T = uint64_t(hi) << 32 | uint32_t(~lanes_max<64>(uint32_t(k >> 32) == hi ? ~uint32_t(k) : 0u));
    }
    if (lane == 0) *counter = 0;
    wave_sync();
    auto take = [&](uint64_t k) {
        if (k == 0 || k < T) return false;
        const int at = atomicAdd(counter, 1);
        if (at < kJoinCap) cand[at] = k;
        return true;
    };
#pragma unroll
    for (int l = 0; l < 2; ++l) {
        bool more = true;
#pragma unroll
        for (int i = 0; i < kFirst; ++i) more = more && take(first[l][i]);
        for (int i = kFirst; more && i < n_keep; ++i) more = take(lists[size_t(lane + 64 * l) * n_keep + i]);
    }
    for (int s = lane + 128; s < slices; s += 64)
        for (int i = 0; i < n_keep && take(lists[size_t(s) * n_keep + i]); ++i) {}
    wave_sync();
    const int n = __builtin_amdgcn_readfirstlane(*counter);
    if (n <= kJoinCap) {
        keep_best(cand, n, n_keep, out);
        return;
    }
    uint64_t below = ~uint64_t(0);
    for (int r = 0; r < n_keep; ++r) {  // the largest key below the last one taken
        uint64_t k = 0;
        for (int s = lane; s < slices; s += 64)
            for (int i = 0; i < n_keep; ++i) {
                const uint64_t y = lists[size_t(s) * n_keep + i];
                if (y < below) {
                    k = y > k ? y : k;
                    break;
                }
            }
        const uint32_t hi = lanes_max<64>(uint32_t(k >> 32));
        const uint32_t lo = lanes_max<64>(uint32_t(k >> 32) == hi ? uint32_t(k) : 0u);
        below = uint64_t(hi) << 32 | lo;
        if (lane == 0) out[r] = below;
    }
}

__global__ __launch_bounds__(1024) void beam_item_kernel(BeamArgs a, int slices) {
    extern __shared__ uint64_t lds[];
    const int B = a.n_beams, K = a.n_keep, n = B * K;
    uint64_t *key = lds;                                   // [B][K]
    double *total = reinterpret_cast<double *>(lds + n);   // [B][K]
    int *rank = reinterpret_cast<int *>(lds + 2 * n);      // [B][K]
    uint64_t *cand = lds + 2 * n + (n + 1) / 2;            // [16][kJoinCap]
    __shared__ int counter[16];
    const int t = threadIdx.x, lane = t & 63, wid = __builtin_amdgcn_readfirstlane(t >> 6);
    const int item = int(blockIdx.x);
    const int have = min(K, a.vocab);  // keys of a beam's list
    for (int i = t; i < n; i += 1024) rank[i] = 0;
    for (int b = wid; b < B; b += 16) {
        const int row = item * B + b;
        float score = a.score ? a.score[row] : 0.0f;
        score = allowed(score);
        const bool ended = a.ended && a.ended[row];
        double lse = 0.0;
        bool none = score == -kInf;
        if (!ended && !none) {
            const float *st = a.stat + size_t(row) * slices * 2;
            float m = -kInf;
            for (int s = lane; s < slices; s += 64) m = fmaxf(m, st[2 * s]);
            m = lanes_max<64>(m);
            none = m == -kInf;
            double sum = 0.0;
            for (int s = lane; s < slices; s += 64)
                if (st[2 * s] > -kInf) sum += double(st[2 * s + 1]) * double(__builtin_amdgcn_exp2f((st[2 * s] - m) * kLog2e));
            for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
            lse = double(m) + log(sum);
        }
        uint64_t *mine = key + b * K;
        if (none || ended) {  // in the tokens' order, an ended beam's only continuation first
            if (lane < K) {
                const int e = a.end_token, j = ended && !none ? (lane == 0 ? e : lane - 1 < e ? lane - 1 : lane) : lane;
                mine[lane] = uint32_t(~uint32_t(j));
                total[b * K + lane] = ended && !none && lane == 0 ? double(score) : double(-kInf);
            }
        } else {
            join_lists(a.list + size_t(row) * slices * K, slices, a.vocab / kBeamSlice, K, cand + wid * kJoinCap, counter + wid, mine);
            wave_sync();
            if (lane < K) {
                const uint64_t k = mine[lane];
                total[b * K + lane] = double(score) + (double(unordered(uint32_t(k >> 32))) - lse);
            }
        }
    }
    __syncthreads();
    // how many of beam o's candidates come before candidate c: its list is in order
    for (int p = t; p < n * B; p += 1024) {
        const int c = p % n, o = p / n, b = c / K, i = c % K;
        if (i >= have) continue;
        int before = i;
        if (o != b) {
            const double x = total[c];
            int lo = 0, hi = have;
            while (lo < hi) {
                const int mid = (lo + hi) / 2;
                const double y = total[o * K + mid];
                if (y > x || (y == x && o < b)) lo = mid + 1;
                else hi = mid;
            }
            before = lo;
        }
        if (before) atomicAdd(rank + c, before);
    }
    __syncthreads();
    for (int c = t; c < n; c += 1024) {
        if (c % K >= have || rank[c] >= K) continue;
        const size_t at = size_t(item) * K + rank[c];
        a.token[at] = int(~uint32_t(key[c]));
        a.parent[at] = c / K;
        a.score_out[at] = float(total[c]);
    }
}

}  // namespace

hipError_t launch_beam(const BeamArgs &a, hipStream_t s) {
    const int slices = beam_slices(a.vocab);
    const int64_t waves = int64_t(a.n_items) * a.n_beams * slices;
    const size_t n = size_t(a.n_beams) * a.n_keep;
    hipLaunchKernelGGL(beam_slice_kernel, dim3(unsigned((waves + 3) / 4)), dim3(256), size_t(4) * a.n_keep * kPerLane * 8, s, a, slices);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(beam_item_kernel, dim3(unsigned(a.n_items)), dim3(1024), (2 * n + (n + 1) / 2 + size_t(16) * kJoinCap) * 8, s, a, slices);
    return hipGetLastError();
}

}  // namespace qmm
