// How calls of the attention are launched, without a device: when work is
// shared, and what a workspace made for one call does to others. Prints one line per failure and "ok" at the end.
#include <cstdio>
#include <random>

#include "../npu880-mtk-npu-llm-runtime_amd/csrc/qmm_attn_plan.h"

using namespace qmm;

static int bad = 0;
#define EXPECT(c, ...) do { if (!(c)) { if (++bad < 20) { std::printf("%s: ", #c); std::printf(__VA_ARGS__); std::printf("\n"); } } } while (0)

static AttnArgs call(int seqs, int rows, int max_new, int max_kv, int heads = 8, int group = 4, int dim = 128) {
    AttnArgs a{};
    a.b = KvView{nullptr, nullptr, nullptr, seqs, rows, 1 << 14, 1 << 20, 6, heads};
    a.group = group;
    a.head_dim = dim;
    a.max_new = max_new;
    a.max_kv = max_kv;
    return a;
}
static const size_t kAny = ~size_t(0) / 2;
static const int kCus = 256;

static bool same(const SplitPlan &x, const SplitPlan &y) {
    return x.rows == y.rows && x.workers == y.workers && x.nw == y.nw && x.lines == y.lines && x.row_tiles == y.row_tiles &&
           x.new_min == y.new_min && x.new_max == y.new_max && x.bytes == y.bytes;
}

// `later` with the workspace of `made` runs as with any
static void covered(const AttnArgs &made, const AttnArgs &later, const char *what) {
    SplitPlan with[2], free[2];
    const int n = plan_call(later, kCus, attn_scratch_bytes(made, kCus), with);
    EXPECT(plan_call(later, kCus, kAny, free) == n, "%s", what);
    for (int i = 0; i < n; ++i) EXPECT(same(with[i], free[i]), "%s: %d workers of %d", what, with[i].workers, free[i].workers);
}

// workgroups of a plan that can run at once
static int64_t at_once(const AttnArgs &a, const SplitPlan &p, int max_new) {
    const int64_t units = int64_t(a.b.n_seqs) * a.b.n_heads, most = sharing(a, p.rows, kCus).workers;
    const int64_t tiles = (int64_t(max_new) * a.group + p.rows - 1) / p.rows;
    return std::min(most, p.workers ? p.workers : p.rows == 16 ? units : units * tiles);
}
static void no_worse_than_none(const AttnArgs &a, size_t scratch, const char *what) {
    SplitPlan with[2], none[2];
    const int n = plan_call(a, kCus, scratch, with);
    EXPECT(plan_call(a, kCus, 0, none) == n, "%s", what);
    size_t bytes = 0;
    for (int i = 0; i < n; ++i) {
        const int rows = i ? few_tokens(a) : a.max_new;
        bytes += with[i].bytes;
        EXPECT(at_once(a, with[i], rows) >= at_once(a, none[i], rows), "%s: %d workers, %lld workgroups without", what, with[i].workers,
               (long long)at_once(a, none[i], rows));
    }
    EXPECT(bytes <= scratch, "%s: %zu bytes of %zu", what, bytes, scratch);
}

// Where work is shared, its units stay below 2^31 for every ragged batch of ascending row starts;
// and page tables of room for long sequences do not keep short ones from sharing.
static void counts() {
    SplitPlan p[2];
    AttnArgs a = call(256, 256, 1, 9000, 4, 8);
    a.b.max_pages = 1 << 14;  // of 64 tokens
    plan_call(a, kCus, kAny, p);
    EXPECT(p[0].workers == 512, "%d workers for 256 sequences with tables of 2^20 tokens", p[0].workers);
    std::mt19937 rng(6);
    auto any = [&](int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(rng); };
    int shared = 0;
    for (int i = 0; i < 20000; ++i) {
        const int seqs = any(1, 1 << any(0, 9)), rows = any(1, 1 << any(0, 16));
        AttnArgs a = call(seqs, rows, any(1, rows), any(1, 1 << 20), any(1, 1 << any(0, 8)), any(1, 40));
        a.b.max_pages = any(1, 1 << any(0, 24));
        for (int n = plan_call(a, kCus, kAny, p), k = 0; k < n; ++k) {
            if (!p[k].workers) continue;
            ++shared;
            const int64_t span = kv_capacity(a.b.max_pages, a.b.page_shift) / kTileKeys + 1;
            int64_t units = 0, left = rows;
            for (int s = 0; s < seqs; ++s) {
                const int64_t mine = s + 1 < seqs ? any(0, int(left)) : left;
                units += (mine * a.group + p[k].rows - 1) / p[k].rows * span;
                left -= mine;
            }
            EXPECT(units * a.b.n_heads < kMostUnits, "%lld units", (long long)(units * a.b.n_heads));
            EXPECT(call_units(uint32_t(units), a.b.n_heads) == units * a.b.n_heads, "units");
        }
    }
    EXPECT(shared > 2000, "%d plans that share", shared);
    EXPECT(capped_sum(~0u - 3, 3) == ~0u && capped_sum(~0u - 3, 4) == ~0u && capped_sum(~0u, ~0u) == ~0u && capped_sum(7, 8) == 15, "sums");
    EXPECT(call_units(1u << 30, 2) == 0 && call_units((1u << 30) - 1, 2) == 0x7ffffffe && call_units(~0u, 65535) == 0 && call_units(~0u, 1) == 0 &&
               call_units(0, 9) == 0 && call_units(0x7fffffffu, 1) == 0x7fffffff, "units of a call");
}

// heads of 256 values take a workgroup three times as long a tile: they share sooner
static void short_heads() {
    SplitPlan p[2];
    auto workers = [&](int heads, int seqs, int dim, int tiles) {
        const AttnArgs a = call(seqs, seqs, 1, tiles * 64, heads, 4, dim);
        plan_call(a, kCus, kAny, p);
        return p[0].workers;
    };
    EXPECT(workers(8, 1, 256, 8) == 0 && workers(8, 1, 256, 12) == 512 && workers(8, 8, 256, 18) == 512 && workers(8, 16, 256, 9) == 0 &&
               workers(8, 16, 256, 18) == 512 && workers(8, 32, 256, 18) == 0 && workers(8, 32, 256, 33) == 512, "heads of 256");
    EXPECT(workers(8, 1, 128, 11) == 0 && workers(8, 1, 128, 16) == 512 && workers(8, 8, 128, 20) == 0 && workers(8, 8, 128, 28) == 512 &&
               workers(8, 16, 64, 22) == 0 && workers(8, 32, 128, 32) == 0, "heads of 64 and 128");
}

// a workgroup of 8 waves takes a CU: for no more heads than CUs, and more tiles than 4
static void waves() {
    SplitPlan p[2];
    auto waves = [&](int seqs, int tiles, int dim) {
        const AttnArgs a = call(seqs, seqs, 1, tiles * 64, 8, 4, dim);
        EXPECT(plan_call(a, kCus, 0, p) == 1 && p[0].workers == 0, "waves");
        return p[0].nw;
    };
    EXPECT(waves(1, 5, 128) == 8 && waves(32, 10, 64) == 8 && waves(1, 4, 128) == 4 && waves(1, 10, 256) == 4, "few heads");
    EXPECT(waves(33, 8, 128) == 4 && waves(64, 8, 128) == 4 && waves(64, 10, 64) == 4, "more heads than CUs");
}

// row tiles of 128: a prompt of its own is not shared, as its row tiles do not differ enough for what
// that costs; long pasts and drafts are
static void row_tiles() {
    SplitPlan p[2];
    auto workers = [&](int seqs, int rows, int past, bool q8 = false) {
        AttnArgs a = call(seqs, seqs * rows, rows, rows + past);
        static const float scale = 1;
        a.ks = q8 ? &scale : nullptr;
        plan_call(a, kCus, kAny, p);
        return p[0].workers;
    };
    EXPECT(workers(1, 512, 0) == 0 && workers(1, 1024, 0) == 0 && workers(1, 2048, 0) == 0 && workers(4, 256, 2000) == 0 &&
               workers(1, 8192, 0) == 0 && workers(1, 1024, 0, true) == 0 && workers(1, 2048, 0, true) == 0, "prompts whole");
    EXPECT(workers(1, 512, 4000) == 512 && workers(1, 256, 2000) == 512 && workers(8, 12, 2000) == 512 && workers(1, 8, 760) == 512 &&
               workers(1, 1024, 4000, true) == 512 && workers(24, 8, 1500, true) == 512, "long pasts shared");
    AttnArgs a = call(8, 519, 512, 4512);  // one long prompt among single tokens: the rows there are count
    plan_call(a, kCus, kAny, p);
    EXPECT(p[0].rows == 128 && p[0].workers == 512, "%d workers for one prompt among single tokens", p[0].workers);
}

// every group of 16 slots and every row of an append has its workgroup, in one launch (below 2^32 threads)
static void append_grids() {
    std::mt19937 rng(7);
    auto any = [&](int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(rng); };
    const int64_t most = (int64_t(1) << 32) / 256;
    for (int i = 0; i < 200000; ++i) {
        const int rows = any(1, 1 << any(0, 26)), heads = any(1, 1 << any(0, 16)) % 65536 + 1, dim = 64 << any(0, 2);
        const int seqs = any(1, std::max(1, std::min(1 << any(0, 24), ((1 << 24) - 1) / heads)));
        const int max_new = any(1, rows), q_heads = any(0, 8) * heads;
        const int64_t chunks = (int64_t(heads) * dim + 1023) / 1024;
        const AppendGrid g = append_grid(rows, seqs, heads, dim, q_heads, max_new);
        if (rows + seqs * chunks >= most) {
            EXPECT(g.workgroups == 0, "%d rows %d sequences %d heads", rows, seqs, heads);
            continue;
        }
        EXPECT(g.workgroups > 0 && g.workgroups < most && g.njobs >= 1 && g.ngroups >= 1 && g.nchunks == chunks &&
                   g.workgroups == int64_t(rows) * g.njobs + int64_t(seqs) * g.ngroups * g.nchunks,
               "%d rows %d sequences %d heads of %d, %d new: %u workgroups", rows, seqs, heads, dim, max_new, g.workgroups);
        EXPECT(g.ngroups <= (max_new + 14) / 16 + 1, "%d groups", g.ngroups);
    }
    const AppendGrid g = append_grid(65536, 256, 64, 256, 0, 65536);  // one long prompt, or max_new not known
    EXPECT(g.workgroups && g.ngroups > 4000, "%u workgroups, %d groups a sequence", g.workgroups, g.ngroups);
    const AppendGrid one = append_grid(1, 1, 8, 128, 32, 1), many = append_grid(8192, 1, 8, 128, 32, 8192);
    EXPECT(one.njobs == 5 && one.ngroups == 1 && one.workgroups == 6 && many.njobs == 1 && many.workgroups == 8192 + 513, "%d %u %u", one.njobs,
           one.workgroups, many.workgroups);
}

// a sequence's workgroups take each of its groups of slots once and end, up to the largest length
static void slots() {
    std::mt19937 rng(8);
    auto any = [&](int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(rng); };
    const int cap = kv_capacity(1 << 30, 10);
    for (int i = 0; i < 3000; ++i) {
        const int len = i % 2 ? cap - any(0, 40) : any(0, 3000), n_new = any(0, 1 << any(0, 11)), ngroups = any(1, 1 << any(0, 23));
        const SeqView v{0, n_new, len, len - n_new};
        const SlotGroups g = slot_groups(v);
        int seen = 0;
        for (int group0 = 0; group0 < std::min(ngroups, 200); ++group0)
            for (int k = g.first + group0; k < g.end; k += ngroups) {
                EXPECT(k >= 0 && k * 16 < len && (k + 1) * 16 > v.pos0, "group %d of %d..%d", k, v.pos0, len);
                if (++seen > 1000) break;
            }
        const int want = n_new && len ? (len - 1) / 16 - std::max(v.pos0, 0) / 16 + 1 : 0;
        EXPECT(seen == want, "%d groups of %d: %d new of %d, %d at a time", seen, want, n_new, len, ngroups);
    }
}

int main() {
    counts();
    slots();
    short_heads();
    row_tiles();
    waves();
    append_grids();
    const AttnArgs prompt = call(1, 8192, 8192, 8192), token = call(1, 1, 1, 131071), batch = call(32, 32, 1, 8000);
    const AttnArgs drafts = call(28, 28 * 8, 8, 4000), many = call(600, 600, 1, 2000), mixed = call(9, 600, 512, 9000);
    covered(prompt, token, "a prompt's workspace, one token");
    covered(prompt, batch, "a prompt's workspace, a batch");
    covered(prompt, drafts, "a prompt's workspace, drafts");
    covered(prompt, mixed, "a prompt's workspace, prompts and tokens");
    covered(many, token, "that of many sequences, one token");
    covered(batch, token, "a batch's, one token");
    covered(token, batch, "one token's, a batch");
    for (size_t scratch : {size_t(0), size_t(1) << 16, size_t(1) << 20, attn_scratch_bytes(token, kCus), attn_scratch_bytes(prompt, kCus), kAny})
        for (const AttnArgs *a : {&prompt, &token, &batch, &drafts, &many, &mixed}) no_worse_than_none(*a, scratch, "scratch of any size");

    std::mt19937 rng(5);
    auto any = [&](int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(rng); };
    for (int i = 0; i < 20000; ++i) {
        const int heads = any(1, 16), group = any(1, 20), dim = 64 << any(0, 2);
        auto one = [&](int most_new) {
            const int seqs = any(1, 1 << any(0, 10)), max_new = any(1, most_new);
            return call(seqs, any(max_new, std::max(max_new, seqs * max_new)), max_new, any(max_new, 1 << any(13, 19)), heads, group, dim);
        };
        const AttnArgs made = one(1 << any(0, 12)), later = one(made.max_new);
        covered(made, later, "any call");
        no_worse_than_none(later, size_t(any(0, 1 << any(4, 30))), "any scratch");
    }
    std::printf(bad ? "%d failures\n" : "ok\n", bad);
    return bad != 0;
}
