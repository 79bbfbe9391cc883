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
// workgroup at most.
constexpr uint32_t kTreeVectors = 32;
constexpr uint32_t tree_vector_waves(uint32_t head_dim) { return head_dim == 64 ? 2 : 4; }
// LDS entries for the page ids of one partition.
constexpr uint32_t kTreePageSlots = 1024;

struct TreePlan {
    uint32_t vector_waves;  // waves of 32 query vectors per workgroup: 1, 2 or 4
    uint32_t part_keys;     // keys per partition, a multiple of the stage
    bool direct;            // one partition per sequence: no records
    uint64_t record_bytes;
};

// Bytes of a partition's record of one query vector: max, sum, 2 unused, o.
constexpr uint32_t tree_record_floats(uint32_t head_dim) { return head_dim + 4; }

// A workgroup fills its CU and costs its keys plus a start and end worth
// kEnds keys; the merge of records costs kMerge.  The candidates are the
// partitions that make one to four rounds of workgroups over the CUs, and one
// partition per sequence.
inline TreePlan tree_plan(uint32_t heads, uint32_t kv_heads, uint32_t head_dim,
                          uint32_t page_tokens, int num_cus, const SeqMeta *seqs, int nseq) {
    const uint64_t stage = tree_stage_keys(head_dim);
    const uint64_t cus = std::max(num_cus, 1);
    const uint64_t group = heads / kv_heads;
    auto up = [](uint64_t x, uint64_t unit) { return (x + unit - 1) / unit; };
    TreePlan plan{};
    uint64_t most_vectors = 0, longest = 0;
    for (int i = 0; i < nseq; ++i) {
        most_vectors = std::max<uint64_t>(most_vectors, seqs[i].rows * group);
        longest = std::max<uint64_t>(longest, (uint64_t)seqs[i].ctx + seqs[i].rows);
    }
    plan.vector_waves = 1;
    while (plan.vector_waves < tree_vector_waves(head_dim) &&
           plan.vector_waves * kTreeVectors < most_vectors) {
        plan.vector_waves *= 2;
    }
    const uint64_t per_group = (uint64_t)plan.vector_waves * kTreeVectors;
    auto blocks = [&](uint64_t part) {
        uint64_t n = 0;
        for (int i = 0; i < nseq; ++i) {
            n += up((uint64_t)seqs[i].ctx + seqs[i].rows, part) * up(seqs[i].rows * group, per_group);
        }
        return n * kv_heads;
    };
    // (a partition that starts inside a page touches part / page + 2 pages)
    const uint64_t max_part = (uint64_t)(kTreePageSlots - 2) * page_tokens / stage * stage;
    const uint64_t whole = up(longest, stage) * stage;
    constexpr uint64_t kEnds = 384, kMerge = 256;
    uint64_t best = 0, best_time = ~0ull;
    if (whole <= max_part) {
        best = whole;
        best_time = up(blocks(whole), cus) * (whole + kEnds);
    }
    for (uint64_t rounds = 1; rounds <= 4; ++rounds) {
        uint64_t part = 4 * stage;
        while (part < std::min(whole, max_part) && blocks(part) > rounds * cus) {
            part += std::max<uint64_t>(stage, part / 16 / stage * stage);
        }
        part = std::min(part, max_part);
        const uint64_t time = up(blocks(part), cus) * (part + kEnds) + kMerge;
        if (part < whole && time < best_time) {
            best_time = time;
            best = part;
        }
    }
    plan.part_keys = (uint32_t)best;
    plan.direct = best >= whole;
    if (!plan.direct) {
        uint64_t records = 0;
        for (int i = 0; i < nseq; ++i) {
            records += up((uint64_t)seqs[i].ctx + seqs[i].rows, best) * seqs[i].rows * heads;
        }
        plan.record_bytes = records * tree_record_floats(head_dim) * sizeof(float);
    }
    return plan;
}

}  // namespace sr
