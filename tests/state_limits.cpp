// What the host decides for the layers with a carried state and the beam search, without a device: a size is given for
// exactly the calls that are taken, and covers the smaller ones. Prints one line per failure and "ok" at the end.
#include <cstdio>
#include <initializer_list>

#include "../npu880-mtk-npu-llm-runtime_amd/csrc/qmm_state.h"
#include "../npu880-mtk-npu-llm-runtime_amd/csrc/qmm_state_check.h"

using namespace qmm;

static int bad = 0;
#define EXPECT(c, ...) do { if (!(c)) { ++bad; std::printf("%s: ", #c); std::printf(__VA_ARGS__); std::printf("\n"); } } while (0)

alignas(16) static float mem[64];
static int32_t ints[8];

// a launch has at most 2^26 slices of 2048 logits: more are refused where the size is asked for, too
static void slices() {
    for (int items : {1, 100, (1 << 20) - 1})
        for (int beams : {1, 4, 64})
            for (int vocab : {1, 2048, 2049, 151936, 131072, (1 << 30) - 1}) {
                const qmm_beam_args t{mem, size_t(vocab), vocab, items, beams, mem, ints, 0, 1, ints, ints, mem};
                const int64_t rows = int64_t(items) * beams;
                const bool fits = rows < (1 << 20) && rows * ((int64_t(vocab) + 2047) / 2048) < (int64_t(1) << 26);
                EXPECT(check_beam(&t).code == (fits ? QMM_OK : QMM_ESHAPE), "%d x %d x %d", items, beams, vocab);
            }
}

// A workspace serves all calls of no more rows and sequences; the place for second halves is there where one of those would use it,
// and nowhere else.
static void workspaces() {
    auto args = [](int seqs, int rows, int hk, int of, int dk, int dv) {
        DeltaArgs a{};
        a.b = StateView{nullptr, nullptr, nullptr, seqs, rows, 0};
        a.qk_heads = hk;
        a.v_heads = hk * of;
        a.key_dim = dk;
        a.value_dim = dv;
        return a;
    };
    for (int hk : {1, 8, 16, 64, 65})
        for (int of : {1, 2, 3})
            for (int dk : {64, 128})
                for (int dv : {64, 128}) {
                    size_t last = 0;
                    for (int seqs : {1, 2, 65, 1000})
                        for (int rows : {1, 31, 480, 481, 512, 8192, 1 << 20}) {
                            const DeltaArgs a = args(seqs, rows, hk, of, dk, dv);
                            const size_t n = delta_scratch_bytes(a), groups = delta_group_bytes(a), lists = size_t(seqs) * a.v_heads;
                            const size_t half = (lists < 64 ? lists : 64) * dk * (2 * dv + dk) * 4 + size_t(rows / 2) * a.v_heads * dk * 4;
                            EXPECT(n == groups + (a.v_heads <= 64 && rows > 480 ? half : 0), "%d x %d, %d rows of %d", hk, of, rows, seqs);
                            EXPECT(groups >= size_t(rows / 32 + seqs) * (a.v_heads * (8192 + 384) + hk * 256), "%d rows of %d", rows, seqs);
                            for (int s2 : {1, 2, 65, 1000})
                                for (int r2 : {1, 31, 480, 481, 512, 8192, 1 << 20})
                                    if (s2 <= seqs && r2 <= rows) {
                                        const DeltaArgs less = args(s2, r2, hk, of, dk, dv);
                                        EXPECT(delta_scratch_bytes(less) <= n && delta_group_bytes(less) <= groups, "%d of %d, %d of %d", r2, rows, s2, seqs);
                                    }
                            last = n;
                        }
                    EXPECT(last > 0, "none");
                }
}

int main() {
    slices();
    workspaces();
    if (!bad) std::printf("ok\n");
    return bad != 0;
}
