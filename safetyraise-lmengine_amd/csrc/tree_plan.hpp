// Host rules of the tree calls, without a GPU: the tree's shape, and how a
// tree attention launch is cut.
#pragma once

#include <algorithm>
#include <cstdint>

#include "sr_internal.hpp"

namespace sr {

constexpr uint32_t kMaxTreeRows = SAFETYRAISE_MI355X_MAX_TREE_ROWS;
constexpr uint32_t kMaxGdnTreeRows = SAFETYRAISE_MI355X_MAX_GDN_TREE_ROWS;

// Every parent is an earlier row of the sequence, or -1.
inline bool tree_valid(const int32_t *parents, uint32_t rows) {
    for (uint32_t r = 0; r < rows; ++r) {
        if (parents[r] < -1 || parents[r] >= (int32_t)r) return false;
    }
    return true;
}

// The rows from the root to `row`, as bits (a parent has a smaller index, so
// ascending bits are the path's order); rows < 64.
inline uint64_t tree_path(const int32_t *parents, int32_t row) {
    uint64_t path = 0;
    for (; row >= 0; row = parents[row]) path |= 1ull << row;
    return path;
}

// One stage of the tree kernel: 32 KB of K and V.
constexpr uint32_t tree_stage_keys(uint32_t head_dim) { return 8192 / head_dim; }
// Query vectors (rows x heads of a KV head) per wave, and waves of vectors per
// workgroup: as many for few vectors too, as the waves without any still load keys (1..3
// rows of 4 heads at width 128 behind 8192..20000 tokens: 69 us with four, 78 with one).
constexpr uint32_t kTreeVectors = 32;
constexpr uint32_t tree_vector_waves(uint32_t head_dim) { return head_dim == 64 ? 2 : 4; }
// LDS entries for the page ids of one partition.
constexpr uint32_t kTreePageSlots = 1024;

// Bytes of a partition's record of one query vector: max, sum, 2 unused, o.
constexpr uint32_t tree_record_floats(uint32_t head_dim) { return head_dim + 4; }

// Partitions of a sequence are equal: its keys over their number, up to whole stages.
constexpr uint32_t tree_part_keys(uint32_t keys, uint32_t parts, uint32_t head_dim) {
    const uint32_t stage = tree_stage_keys(head_dim);
    return ((keys + parts - 1) / parts + stage - 1) / stage * stage;
}

// Time of a key in tenths: one where every SIMD has two waves with query vectors.  With
// fewer vectors it has one, with half the products but nothing beside it.  The 7 tenths are
// by what the plan makes of eight sequences of unlike rows and contexts (160 -> 149 us);
// with the same rows in every sequence, all CUs busy, a stage at width 128 takes 1.6 us
// with 128 vectors and 1.4 with two (f32 result).
inline uint32_t tree_key_cost(uint32_t head_dim, uint64_t vectors) {
    const uint32_t key_waves = tree_stage_keys(head_dim) / 32, vector_waves = tree_vector_waves(head_dim);
    const uint64_t tiles = std::min<uint64_t>(vector_waves, (vectors + kTreeVectors - 1) / kTreeVectors);
    return tiles * key_waves > 4 ? 10 : vector_waves * key_waves > 4 ? 7 : 10;
}

// The number of partitions of a sequence of `keys` (with the call's rows).
inline uint32_t tree_parts(const TreePlan &plan, uint32_t head_dim, uint32_t keys, uint64_t vectors) {
    const uint64_t stage = tree_stage_keys(head_dim);
    uint64_t part = plan.budget / tree_key_cost(head_dim, vectors) / stage * stage;
    part = std::min<uint64_t>(std::max(part, stage), plan.max_part);
    const uint64_t parts = (keys + part - 1) / part;
    // (equal partitions of whole stages may be fewer)
    const uint64_t equal = tree_part_keys(keys, (uint32_t)parts, head_dim);
    return (uint32_t)((keys + equal - 1) / equal);
}

// A workgroup fills its CU and costs its keys plus a start and an end, about 8 us; the
// merge of records is 4.5 us and the writing and reading of them at 4 TB/s (17 / D^2 tenths
// of a key per float).  These are counted in keys as if a stage took D / 64 x 0.5 us, in
// inverse proportion to D^2: 300 tokens at width 256 take 21 us in partitions of two
// stages, 45 in one.  The stages measured with all CUs busy (128 vectors, 40 to 80 stages):
// 2.3 us at width 64, 1.6 at 128, 1.7 at 256 for an f32 result, 1.4, 1.1 and 1.1 for bf16;
// so the ends and the merge weigh up to four times what they take at width 64 and up to
// twice at 128, for fewer and longer partitions.  The candidates are the least budgets
// that make one to four rounds of workgroups over the CUs, and one partition per sequence.
inline TreePlan tree_plan(uint32_t heads, uint32_t kv_heads, uint32_t head_dim,
                          uint32_t page_tokens, int num_cus, const SeqMeta *seqs, int nseq) {
    const uint64_t stage = tree_stage_keys(head_dim);
    const uint64_t cus = std::max(num_cus, 1);
    const uint64_t group = heads / kv_heads;
    auto up = [](uint64_t x, uint64_t unit) { return (x + unit - 1) / unit; };
    TreePlan plan{};
    uint64_t longest = 0, dearest = 0;
    // (a partition that starts inside a page touches part / page + 2 pages)
    plan.max_part = (uint32_t)((uint64_t)(kTreePageSlots - 2) * page_tokens / stage * stage);
    const uint64_t per_group = (uint64_t)tree_vector_waves(head_dim) * kTreeVectors;
    for (int i = 0; i < nseq; ++i) {
        const uint64_t keys = (uint64_t)seqs[i].ctx + seqs[i].rows;
        longest = std::max(longest, keys);
        dearest = std::max(dearest, up(keys, stage) * stage * tree_key_cost(head_dim, seqs[i].rows * group));
    }
    uint64_t records = 0;  // of the budget that blocks() last looked at
    auto blocks = [&](uint64_t budget) {
        TreePlan p = plan;
        p.budget = budget;
        uint64_t n = 0;
        records = 0;
        for (int i = 0; i < nseq; ++i) {
            const uint64_t vectors = seqs[i].rows * group;
            const uint64_t parts = tree_parts(p, head_dim, seqs[i].ctx + seqs[i].rows, vectors);
            n += parts * up(vectors, per_group);
            records += parts * seqs[i].rows * heads;
        }
        return n * kv_heads;
    };
    const uint64_t square = (uint64_t)head_dim * head_dim;
    const uint64_t ends = 20000 * 4096 / square, merge = 11000 * 4096 / square;  // (tenths of a key)
    constexpr uint64_t kLeast = 2;  // stages of a partition
    const bool may_whole = up(longest, stage) * stage <= plan.max_part;
    uint64_t best = 0, best_time = ~0ull;
    if (may_whole) {
        // (costs in tenths differ between sequences: with `dearest * 2` none is cut)
        best = dearest * 2;
        best_time = up(blocks(best), cus) * (dearest + ends);
    }
    for (uint64_t rounds = 1; rounds <= 4; ++rounds) {
        uint64_t lo = kLeast * stage * 10, hi = std::max(lo, dearest);  // (to 1 part in 1024)
        const uint64_t step = std::max(stage, (hi - lo) / 1024);
        if (blocks(lo) <= rounds * cus) hi = lo;
        while (hi - lo > step) {
            const uint64_t mid = (lo + hi) / 2;
            if (blocks(mid) > rounds * cus) lo = mid;
            else hi = mid;
        }
        const uint64_t time = up(blocks(hi), cus) * (hi + ends) + merge +
                              records * tree_record_floats(head_dim) * 17 / square;
        if (time < best_time) {
            best_time = time;
            best = hi;
        }
        if (hi == kLeast * stage * 10) break;  // more rounds make the same partitions
    }
    plan.budget = best;
    (void)blocks(best);
    uint64_t rows = 0;
    for (int i = 0; i < nseq; ++i) rows += seqs[i].rows;
    plan.direct = records == rows * heads;
    if (!plan.direct) plan.record_bytes = records * tree_record_floats(head_dim) * sizeof(float);
    return plan;
}

}  // namespace sr
