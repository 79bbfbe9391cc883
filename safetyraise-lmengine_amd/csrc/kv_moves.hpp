// The description of a kv_compact or kv_gather call as its kernels read it: 32-bit
// words, entries first; offsets count words from the beginning.
#pragma once

#include <cstdint>

#include <hip/hip_runtime.h>

namespace sr {

struct MoveEntry {
    uint16_t *k_pages;
    uint16_t *v_pages;
    const int32_t *from;  // page-table row of the source
    uint64_t num_pages;
    uint32_t kv_heads, head_dim, log2_page;
    uint32_t start;       // kept tokens from here on come from the list
    uint32_t first_page;  // first page of `pages`
    uint32_t pages;       // page ids of the new sequence from first_page on
    uint32_t tokens;      // the list
    uint32_t unused;
};
// Tokens of the new sequence; next: the range that the same workgroup moves
// after this one (0: none; the first ranges of the chains come first)
struct MoveRange {
    uint32_t entry, begin, end, next;
};
// page ids for a row of the page table
struct MoveLink {
    int32_t *row;
    uint32_t pages, count;
};
struct GatherEntry {
    const uint16_t *k_pages;
    const uint16_t *v_pages;
    const int32_t *from;
    uint64_t first;  // the entry's first token in the output
    uint32_t num_pages, log2_page, start, count;
    uint32_t tokens;  // 0: consecutive tokens
    uint32_t unused;
};
// a workgroup's tokens: block_tokens of the entry from `begin` on, as far as it has them
struct GatherBlock {
    uint32_t entry, begin;
};
static_assert(sizeof(MoveEntry) % 8 == 0 && sizeof(MoveRange) % 8 == 0 && sizeof(MoveLink) % 8 == 0 &&
                  sizeof(GatherEntry) % 8 == 0,
              "pointers stay aligned");

constexpr uint32_t kMoveInlineWords = 1008;  // what fits the kernel arguments
constexpr uint32_t kGatherInlineWords = 992;

// Workgroups of 256 threads that a launch has at most: its threads are counted in 32 bits.
constexpr uint32_t kMostBlocks = UINT32_MAX / 256, kMostBlocksY = 65535;

// Rows (one token of one head) that a workgroup of the move kernel has in flight.
constexpr uint32_t kMovePasses = 4;
constexpr uint32_t move_rows(uint32_t head_dim) {
    const uint32_t units = head_dim % 8 == 0 ? head_dim / 8 : head_dim;
    return kMovePasses * (units <= 256 ? 256 / units : 1);
}

struct MoveCall {
    const uint32_t *host_words;
    const uint32_t *device_words;  // nullptr: the words travel in the arguments
    uint32_t words;
    uint32_t entries, ranges, chains;
    uint32_t links;       // rows that no range of the call reads
    uint32_t late_links;  // rows written after the ranges
    uint32_t log2_heads, head_groups;  // a workgroup moves 2^log2_heads heads of a range
};
struct GatherCall {
    const uint32_t *host_words;
    const uint32_t *device_words;
    uint32_t words;
    uint32_t entries, blocks, kv_heads, head_dim, block_tokens;
    void *keys, *values;
    bool bf16_out;
};
// the moves, and the rows that no range reads; then the other rows
hipError_t launch_kv_moves(hipStream_t stream, const MoveCall &call);
hipError_t launch_kv_links(hipStream_t stream, const MoveCall &call);
hipError_t launch_kv_gather_rows(hipStream_t stream, const GatherCall &call);

}  // namespace sr
