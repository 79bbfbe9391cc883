// Tokens moved inside a KV pool and copied out of it, for lists of tokens of many
// sequences and pools in one launch.
//
// Both are copies: bound by the bytes they read and write, or for a few tokens by the
// launch (4.6 us).  14500 of 53000 tokens of two sequences, 8 heads of width 128, to free
// pages, 119 MB: 29.4 us; 33300 of three, 2 heads of width 256, to f32 rows, 205 MB: 38.6 us
// (each call with inputs of its own).  Serial ranges are bound by one workgroup's round
// trips: 12800 tokens of two sequences in place, 105 MB, 29 us to free pages, 224 without any.
//
// The call's description (entries, ranges, token lists, page ids) travels in the
// kernel arguments where it fits, else through pinned host memory into a device buffer.
#include "kv_moves.hpp"
#include "sr_device.hpp"

namespace sr {

namespace {

typedef uint32_t Unit16 __attribute__((ext_vector_type(4)));  // 8 values

struct MoveArgs {
    const uint32_t *words;  // nullptr: inline_words
    uint32_t entries, ranges, chains, links, log2_heads;
    alignas(16) uint32_t inline_words[kMoveInlineWords];
};
static_assert(sizeof(MoveArgs) <= 4096, "kernel arguments stay within 4 KiB");

// A workgroup moves the tokens of one range, K or V of 2^lh heads, in the order of the
// tokens: a chunk is read whole before any of it is written.  A row (one token of one
// head) is `per` units; a thread has one of them in every pass of 256 / per rows (rows
// of more than 256 units: a thread takes every 256th unit of one row).
template <typename Unit>
__device__ __forceinline__ void move_range(uint16_t *pages, const MoveEntry &e, const MoveRange &r,
                                           const int32_t *from, const int32_t *to,
                                           const uint32_t *tokens, uint32_t head0, uint32_t lh) {
    const uint32_t per = (uint32_t)(e.head_dim * 2 / sizeof(Unit));  // at most 512 units
    const uint32_t lpt = e.log2_page, mask = (1u << lpt) - 1;
    Unit *base = global_from_bits<Unit>((uint64_t)pages);
    const size_t head_rows = (size_t)e.num_pages << lpt;
    const uint32_t rows = per <= 256 ? 256 / per : 1;  // of a pass
    const uint32_t my_row = per <= 256 ? threadIdx.x / per : 0;
    const uint32_t my_unit = per <= 256 ? threadIdx.x % per : threadIdx.x;
    const uint32_t chunk = max(1u, (rows * kMovePasses) >> lh);  // tokens
    for (uint32_t t0 = r.begin; t0 < r.end; t0 += chunk) {
        for (uint32_t u0 = 0; u0 < per; u0 += 256) {  // (once, but for rows of more than 256 units)
            const uint32_t u = min(u0 + my_unit, per - 1);
            Unit x[kMovePasses];
            Unit *dst[kMovePasses];
            bool ok[kMovePasses];
            uint32_t s[kMovePasses];
            size_t head[kMovePasses];
#pragma unroll
            for (uint32_t i = 0; i < kMovePasses; ++i) {
                const uint32_t at = rows * i + my_row, t = t0 + (at >> lh);
                const uint32_t hh = head0 + (at & ((1u << lh) - 1));
                ok[i] = my_row < rows && u0 + my_unit < per && (at >> lh) < chunk && t < r.end && hh < e.kv_heads;
                const uint32_t tc = ok[i] ? t : r.begin;
                head[i] = (ok[i] ? hh : head0) * head_rows;
                s[i] = tc < e.start ? tc : e.start + tokens[tc - e.start];
                dst[i] = base + (head[i] + ((size_t)to[(tc >> lpt) - e.first_page] << lpt) + (tc & mask)) * per + u;
            }
#pragma unroll
            for (uint32_t i = 0; i < kMovePasses; ++i) {
                x[i] = base[(head[i] + ((size_t)from[s[i] >> lpt] << lpt) + (s[i] & mask)) * per + u];
            }
            // every wave's reads are done before any wave writes
            __builtin_amdgcn_s_waitcnt(0x0F70);
            __syncthreads();
#pragma unroll
            for (uint32_t i = 0; i < kMovePasses; ++i) {
                if (ok[i]) *dst[i] = x[i];
            }
        }
    }
}

// grid (range that begins a chain, 2 x groups of heads); then links: blocks past the
// ranges write page-table rows of targets that no range reads
__global__ void __launch_bounds__(256) kv_move_kernel(const MoveArgs a) {
    const uint32_t *w = a.words != nullptr ? a.words : a.inline_words;
    const MoveEntry *entries = (const MoveEntry *)w;
    const MoveRange *ranges = (const MoveRange *)(entries + a.entries);
    if (blockIdx.x >= a.chains) {
        if (blockIdx.y != 0) return;
        const MoveLink l = ((const MoveLink *)(ranges + a.ranges))[blockIdx.x - a.chains];
        for (uint32_t i = threadIdx.x; i < l.count; i += 256) l.row[i] = (int32_t)w[l.pages + i];
        return;
    }
    MoveRange r = ranges[blockIdx.x];
    const MoveEntry e = entries[r.entry];
    const int32_t *from = global_from_bits<const int32_t>((uint64_t)e.from);
    const uint32_t head0 = (blockIdx.y >> 1) << a.log2_heads;
    if (head0 >= e.kv_heads) return;
    uint16_t *pages = (blockIdx.y & 1) ? e.v_pages : e.k_pages;
    const int32_t *to = (const int32_t *)(w + e.pages);
    const uint32_t *tokens = w + e.tokens;
    for (;;) {
        if (e.head_dim % 8 == 0) move_range<Unit16>(pages, e, r, from, to, tokens, head0, a.log2_heads);
        else move_range<uint16_t>(pages, e, r, from, to, tokens, head0, a.log2_heads);
        if (r.next == 0) break;
        r = ranges[r.next];
    }
}

__global__ void __launch_bounds__(256) kv_link_kernel(const uint32_t *words, const MoveArgs a) {
    const uint32_t *w = words != nullptr ? words : a.inline_words;
    const MoveLink l = ((const MoveLink *)((const MoveRange *)((const MoveEntry *)w + a.entries) + a.ranges))[a.links + blockIdx.x];
    for (uint32_t i = threadIdx.x; i < l.count; i += 256) l.row[i] = (int32_t)w[l.pages + i];
}

struct GatherArgs {
    const uint32_t *words;
    void *keys;
    void *values;
    uint32_t entries, kv_heads, head_dim, block_tokens;
    int bf16_out;
    alignas(16) uint32_t inline_words[kGatherInlineWords];
};
static_assert(sizeof(GatherArgs) <= 4096, "kernel arguments stay within 4 KiB");

// Unit `at` of an output, past the caches: written once, and as a rule more than they
// hold (205 MB: 58 us with plain stores, 47 with these, where each call has inputs and
// outputs of its own).
__device__ __forceinline__ void put8(void *out, size_t at, Unit16 x, bool bf16) {
    typedef float Half __attribute__((ext_vector_type(4)));
    if (bf16) {
        __builtin_nontemporal_store(x, (Unit16 *)out + at);
    } else {
        Half *to = (Half *)out + 2 * at;
        __builtin_nontemporal_store(Half{bf16lo(x.x), bf16hi(x.x), bf16lo(x.y), bf16hi(x.y)}, to);
        __builtin_nontemporal_store(Half{bf16lo(x.z), bf16hi(x.z), bf16lo(x.w), bf16hi(x.w)}, to + 1);
    }
}

// One workgroup per block of at most block_tokens tokens of one entry; a thread
// takes 8 values (kVec) or one value of a token's K and V rows at a time.
template <bool kVec>
__global__ void __launch_bounds__(256) kv_gather_rows_kernel(const GatherArgs a) {
    const uint32_t *w = a.words != nullptr ? a.words : a.inline_words;
    const GatherEntry *entries = (const GatherEntry *)w;
    const GatherBlock b = ((const GatherBlock *)(entries + a.entries))[blockIdx.x];
    const GatherEntry e = entries[b.entry];
    const uint16_t *k_pages = global_from_bits<const uint16_t>((uint64_t)e.k_pages);
    const uint16_t *v_pages = global_from_bits<const uint16_t>((uint64_t)e.v_pages);
    const int32_t *from = global_from_bits<const int32_t>((uint64_t)e.from);
    const uint32_t per_head = kVec ? a.head_dim / 8 : a.head_dim;
    const uint32_t per = a.kv_heads * per_head;
    const uint32_t n = min(a.block_tokens, e.count - b.begin) * per;
    constexpr uint32_t kBatch = 4;
    for (uint32_t i0 = threadIdx.x; i0 < n; i0 += 256 * kBatch) {
        size_t src[kBatch], dst[kBatch];
        bool ok[kBatch];
#pragma unroll
        for (uint32_t u = 0; u < kBatch; ++u) {
            ok[u] = i0 + 256 * u < n;
            const uint32_t i = ok[u] ? i0 + 256 * u : i0;
            const uint32_t at = b.begin + i / per, r = i % per, h = r / per_head, c = r % per_head;
            const uint32_t s = e.start + (e.tokens != 0 ? w[e.tokens + at] : at);
            const size_t row = (((size_t)h * e.num_pages + from[s >> e.log2_page]) << e.log2_page) +
                               (s & ((1u << e.log2_page) - 1));
            src[u] = row * a.head_dim + (kVec ? 8 * c : c);
            dst[u] = (e.first + at) * per + r;
        }
        if constexpr (kVec) {
            Unit16 k[kBatch], v[kBatch];
#pragma unroll
            for (uint32_t u = 0; u < kBatch; ++u) {
                k[u] = *(const Unit16 *)(k_pages + src[u]);
                v[u] = *(const Unit16 *)(v_pages + src[u]);
            }
#pragma unroll
            for (uint32_t u = 0; u < kBatch; ++u) {
                if (!ok[u]) break;
                put8(a.keys, dst[u], k[u], a.bf16_out != 0);
                put8(a.values, dst[u], v[u], a.bf16_out != 0);
            }
        } else {
#pragma unroll
            for (uint32_t u = 0; u < kBatch; ++u) {
                if (!ok[u]) break;
                if (a.bf16_out) {
                    ((uint16_t *)a.keys)[dst[u]] = k_pages[src[u]];
                    ((uint16_t *)a.values)[dst[u]] = v_pages[src[u]];
                } else {
                    ((float *)a.keys)[dst[u]] = bf16_to_f32(k_pages[src[u]]);
                    ((float *)a.values)[dst[u]] = bf16_to_f32(v_pages[src[u]]);
                }
            }
        }
    }
}

}  // namespace

namespace {

bool move_args(const MoveCall &c, MoveArgs &a) {
    a.words = c.device_words;
    a.entries = c.entries;
    a.ranges = c.ranges;
    a.chains = c.chains;
    a.links = c.links;
    a.log2_heads = c.log2_heads;
    if (a.words == nullptr) {
        if (c.words > kMoveInlineWords) return false;
        for (uint32_t i = 0; i < c.words; ++i) a.inline_words[i] = c.host_words[i];
    }
    return true;
}

}  // namespace

hipError_t launch_kv_moves(hipStream_t stream, const MoveCall &c) {
    if (c.chains + c.links == 0) return hipSuccess;
    MoveArgs a{};
    if (!move_args(c, a)) return hipErrorInvalidValue;
    SR_LAUNCH("kv_move_kernel", kv_move_kernel, dim3(c.chains + c.links, 2 * c.head_groups), dim3(256),
              0, stream, a);
    return hipGetLastError();
}

hipError_t launch_kv_links(hipStream_t stream, const MoveCall &c) {
    if (c.late_links == 0) return hipSuccess;
    MoveArgs a{};
    if (!move_args(c, a)) return hipErrorInvalidValue;
    SR_LAUNCH("kv_link_kernel", kv_link_kernel, dim3(c.late_links), dim3(256), 0, stream, c.device_words, a);
    return hipGetLastError();
}

hipError_t launch_kv_gather_rows(hipStream_t stream, const GatherCall &c) {
    GatherArgs a{};
    a.words = c.device_words;
    a.keys = c.keys;
    a.values = c.values;
    a.entries = c.entries;
    a.kv_heads = c.kv_heads;
    a.head_dim = c.head_dim;
    a.block_tokens = c.block_tokens;
    a.bf16_out = c.bf16_out ? 1 : 0;
    if (a.words == nullptr) {
        if (c.words > kGatherInlineWords) return hipErrorInvalidValue;
        for (uint32_t i = 0; i < c.words; ++i) a.inline_words[i] = c.host_words[i];
    }
    if (c.head_dim % 8 == 0) {
        SR_LAUNCH("kv_gather_rows_kernel", kv_gather_rows_kernel<true>, dim3(c.blocks), dim3(256), 0, stream, a);
    } else {
        SR_LAUNCH("kv_gather_rows_kernel", kv_gather_rows_kernel<false>, dim3(c.blocks), dim3(256), 0, stream, a);
    }
    return hipGetLastError();
}

}  // namespace sr
