// Tokens moved inside a KV pool and copied out of it, for lists of tokens of many
// sequences and pools in one launch.
//
// Both are copies: bound by the bytes they read and write, or for a few tokens
// by the launch.  The call's description (entries, ranges, token lists, page
// ids) travels in the kernel arguments where it fits, else through pinned host
// memory into a device buffer.
#include "kv_moves.hpp"
#include "sr_device.hpp"

namespace sr {

namespace {

struct MoveArgs {
    const uint32_t *words;  // nullptr: inline_words
    uint32_t entries, ranges, chains, links;
    alignas(16) uint32_t inline_words[kMoveInlineWords];
};
static_assert(sizeof(MoveArgs) <= 4096, "kernel arguments stay within 4 KiB");

// A workgroup moves the tokens of one range of one head's K or V, in the order
// of the tokens: a chunk is read whole before any of it is written.
template <typename Unit, uint32_t kUnits>
__device__ __forceinline__ void move_range(uint16_t *pages, const MoveEntry &e, const MoveRange &r,
                                           const int32_t *from, const int32_t *to,
                                           const uint32_t *tokens, uint32_t kvh) {
    const uint32_t per = (uint32_t)(e.head_dim * 2 / sizeof(Unit));  // units per row
    const uint32_t lpt = e.log2_page, mask = (1u << lpt) - 1;
    Unit *base = (Unit *)(pages + (((size_t)kvh * e.num_pages) << lpt) * e.head_dim);
    const uint64_t total = (uint64_t)(r.end - r.begin) * per;
    for (uint64_t u0 = 0; u0 < total; u0 += 256 * kUnits) {
        Unit x[kUnits];
        size_t dst[kUnits];
#pragma unroll
        for (uint32_t i = 0; i < kUnits; ++i) {
            const uint64_t u = min(u0 + threadIdx.x + 256 * i, total - 1);
            const uint32_t t = r.begin + (uint32_t)(u / per), at = (uint32_t)(u % per);
            const uint32_t s = t < e.start ? t : e.start + tokens[t - e.start];
            const int32_t src_page = from[s >> lpt], dst_page = to[(t >> lpt) - e.first_page];
            x[i] = base[(((size_t)src_page << lpt) + (s & mask)) * per + at];
            dst[i] = (((size_t)dst_page << lpt) + (t & mask)) * per + at;
        }
        // every wave's reads are done before any wave writes
        __builtin_amdgcn_s_waitcnt(0x0F70);
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < kUnits; ++i) {
            if (u0 + threadIdx.x + 256 * i < total) base[dst[i]] = x[i];
        }
    }
}

// grid (range that begins a chain, 2 x KV heads); then links: blocks past the ranges write page-table
// rows of targets that no range reads
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
    const uint32_t kvh = blockIdx.y >> 1;
    if (kvh >= e.kv_heads) return;
    uint16_t *pages = (blockIdx.y & 1) ? e.v_pages : e.k_pages;
    const int32_t *to = (const int32_t *)(w + e.pages);
    const uint32_t *tokens = w + e.tokens;
    for (;;) {
        if (e.head_dim % 8 == 0) move_range<uint4, 4>(pages, e, r, e.from, to, tokens, kvh);
        else move_range<uint16_t, 8>(pages, e, r, e.from, to, tokens, kvh);
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
    uint64_t tokens;
    uint32_t entries, kv_heads, head_dim;
    int bf16_out;
    alignas(16) uint32_t inline_words[kMoveInlineWords - 16];
};
static_assert(sizeof(GatherArgs) <= 4096, "kernel arguments stay within 4 KiB");

// One thread per 8 values (kVec) or one value of a token's K and V rows.
template <bool kVec>
__global__ void __launch_bounds__(256) kv_gather_rows_kernel(const GatherArgs a) {
    const uint32_t *w = a.words != nullptr ? a.words : a.inline_words;
    const GatherEntry *entries = (const GatherEntry *)w;
    const uint32_t per_head = kVec ? a.head_dim / 8 : a.head_dim;
    const uint32_t per = a.kv_heads * per_head;
    const uint64_t n = a.tokens * per;
    for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < n; i += (uint64_t)gridDim.x * 256) {
        const uint64_t t = i / per;
        const uint32_t r = (uint32_t)(i % per), h = r / per_head, c = r % per_head;
        uint32_t lo = 0, hi = a.entries - 1;  // the entry that holds token t
        while (lo < hi) {
            const uint32_t mid = (lo + hi + 1) / 2;
            if (entries[mid].first <= t) lo = mid;
            else hi = mid - 1;
        }
        const GatherEntry e = entries[lo];
        const uint32_t at = (uint32_t)(t - e.first);
        const uint32_t s = e.start + (e.tokens != 0 ? w[e.tokens + at] : at);
        const size_t row = (((size_t)h * e.num_pages + e.from[s >> e.log2_page]) << e.log2_page) +
                           (s & ((1u << e.log2_page) - 1));
        if constexpr (kVec) {
            const size_t src = row * a.head_dim + 8 * c;
            const uint4 k = *(const uint4 *)(e.k_pages + src), v = *(const uint4 *)(e.v_pages + src);
            if (a.bf16_out) {
                ((uint4 *)a.keys)[i] = k;
                ((uint4 *)a.values)[i] = v;
            } else {
                float4 *dk = (float4 *)a.keys + 2 * i, *dv = (float4 *)a.values + 2 * i;
                dk[0] = make_float4(bf16lo(k.x), bf16hi(k.x), bf16lo(k.y), bf16hi(k.y));
                dk[1] = make_float4(bf16lo(k.z), bf16hi(k.z), bf16lo(k.w), bf16hi(k.w));
                dv[0] = make_float4(bf16lo(v.x), bf16hi(v.x), bf16lo(v.y), bf16hi(v.y));
                dv[1] = make_float4(bf16lo(v.z), bf16hi(v.z), bf16lo(v.w), bf16hi(v.w));
            }
        } else {
            const size_t src = row * a.head_dim + c;
            if (a.bf16_out) {
                ((uint16_t *)a.keys)[i] = e.k_pages[src];
                ((uint16_t *)a.values)[i] = e.v_pages[src];
            } else {
                ((float *)a.keys)[i] = bf16_to_f32(e.k_pages[src]);
                ((float *)a.values)[i] = bf16_to_f32(e.v_pages[src]);
            }
        }
    }
}

}  // namespace

hipError_t launch_kv_moves(hipStream_t stream, const MoveCall &c) {
    MoveArgs a{};
    a.words = c.device_words;
    a.entries = c.entries;
    a.ranges = c.ranges;
    a.chains = c.chains;
    a.links = c.links;
    if (a.words == nullptr) {
        if (c.words > kMoveInlineWords) return hipErrorInvalidValue;
        for (uint32_t i = 0; i < c.words; ++i) a.inline_words[i] = c.host_words[i];
    }
    if (c.chains + c.links > 0) {
        SR_LAUNCH("kv_move_kernel", kv_move_kernel, dim3(c.chains + c.links, 2 * c.kv_heads), dim3(256),
                  0, stream, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    if (c.late_links > 0) {
        SR_LAUNCH("kv_link_kernel", kv_link_kernel, dim3(c.late_links), dim3(256), 0, stream,
                  c.device_words, a);
    }
    return hipGetLastError();
}

hipError_t launch_kv_gather_rows(hipStream_t stream, const GatherCall &c) {
    GatherArgs a{};
    a.words = c.device_words;
    a.keys = c.keys;
    a.values = c.values;
    a.tokens = c.tokens;
    a.entries = c.entries;
    a.kv_heads = c.kv_heads;
    a.head_dim = c.head_dim;
    a.bf16_out = c.bf16_out ? 1 : 0;
    if (a.words == nullptr) {
        if (c.words > kMoveInlineWords - 16) return hipErrorInvalidValue;
        for (uint32_t i = 0; i < c.words; ++i) a.inline_words[i] = c.host_words[i];
    }
    const bool vec = c.head_dim % 8 == 0;
    const uint64_t n = c.tokens * c.kv_heads * (vec ? c.head_dim / 8 : c.head_dim);
    const uint32_t blocks = (uint32_t)std::min<uint64_t>((n + 255) / 256, 65536);
    if (vec) SR_LAUNCH("kv_gather_rows_kernel", kv_gather_rows_kernel<true>, dim3(blocks), dim3(256), 0, stream, a);
    else SR_LAUNCH("kv_gather_rows_kernel", kv_gather_rows_kernel<false>, dim3(blocks), dim3(256), 0, stream, a);
    return hipGetLastError();
}

}  // namespace sr
