// What the host decides for the layers with a carried state and the beam search, without a device: a size is given for
// exactly the calls that are taken. Prints one line per failure and "ok" at the end.
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

int main() {
    slices();
    if (!bad) std::printf("ok\n");
    return bad != 0;
}
