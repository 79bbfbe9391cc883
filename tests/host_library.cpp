// The library's host code without a GPU: the runtime's calls on host memory, and the page
// copies, table writes and token moves done there, the workgroups of a launch in random
// order.  Calls that compute do nothing.  test_fail makes a launch fail.
#include <cmath>
#include <cstdlib>
#include <cstring>
#include <string>
#include <vector>

#include "kv_moves.hpp"
#include "sr_internal.hpp"

namespace {

using Pool = safetyraise_kernel_kv_pool;

uint64_t g_random = 1;
uint32_t random_below(uint32_t n) {
    g_random = g_random * 6364136223846793005ull + 1442695040888963407ull;
    return (uint32_t)((g_random >> 33) % n);
}

std::string g_fail;
int g_fail_after = 0, g_null_copies = 0, g_waits = 0;

// a launch: an error where the test asks for one
hipError_t launch(const char *name) {
    if (g_fail != name || g_fail_after-- > 0) return hipSuccess;
    g_fail.clear();
    return hipErrorLaunchFailure;
}

float as_float(uint16_t x) {
    const uint32_t w = (uint32_t)x << 16;
    float f;
    std::memcpy(&f, &w, 4);
    return f;
}
uint16_t as_bf16(float f) {
    uint32_t w;
    std::memcpy(&w, &f, 4);
    return (uint16_t)((w + 0x7fffu + ((w >> 16) & 1)) >> 16);
}

// the row of a token and head
size_t row_of(const Pool *p, int32_t page, uint64_t token, uint32_t head) {
    return ((size_t)head * p->num_pages + page) * p->page_tokens + token % p->page_tokens;
}

// One workgroup of a launch's moves: a head of K or V, and where it is in its chain.
struct Group {
    uint32_t range, head;
    bool values;
    uint32_t at;
};

}  // namespace

extern "C" {

void test_seed(uint64_t seed) { g_random = seed; }
// the launch of this name after `after` others of it fails; whether one is still to fail
void test_fail(const char *name, int after) { g_fail = name, g_fail_after = after; }
int test_failing() { return !g_fail.empty(); }
int test_null_copies() { return g_null_copies; }
int test_waits() { return g_waits; }

void *__real_memcpy(void *to, const void *from, size_t n);
void *__wrap_memcpy(void *to, const void *from, size_t n) {
    if (to == nullptr || from == nullptr) {
        ++g_null_copies;
        return to;
    }
    return __real_memcpy(to, from, n);
}

// 0, or what is wrong with a pool's page lists: 1 reference counts, 2 the free list, 3 the page
// table, 4 too few pages
int test_pool(const Pool *p) {
    std::vector<uint32_t> held(p->num_pages, 0);
    for (uint32_t s = 0; s < p->max_sequences; ++s) {
        const auto &q = p->seqs[s];
        if (!q.open) continue;
        for (int32_t page : q.pages) ++held[page];
        const uint64_t need = (q.len + p->page_tokens - 1) / p->page_tokens;
        if (q.pages.size() < need) return 4;
        for (uint64_t i = 0; i < need; ++i) {
            if (p->d_page_table[(size_t)s * p->pages_per_seq + i] != q.pages[i]) return 3;
        }
    }
    std::vector<uint8_t> is_free(p->num_pages, 0);
    for (int32_t page : p->free_pages) {
        if (is_free[page]++ != 0) return 2;
    }
    for (uint64_t i = 0; i < p->num_pages; ++i) {
        if (held[i] != p->refcount[i]) return 1;
        if ((held[i] == 0) != (is_free[i] == 1)) return 2;
    }
    return 0;
}
uint64_t test_free_pages(const Pool *p) { return p->free_pages.size(); }

// ------------------------------------------------------------------ the runtime

hipError_t hipGetDeviceCount(int *n) { return *n = 1, hipSuccess; }
hipError_t hipGetDevice(int *d) { return *d = 0, hipSuccess; }
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipGetDevicePropertiesR0600(hipDeviceProp_tR0600 *p, int) {
    std::memset((void *)p, 0, sizeof *p);
    p->multiProcessorCount = 256;
    return hipSuccess;
}
hipError_t hipGetLastError() { return hipSuccess; }
const char *hipGetErrorName(hipError_t) { return "error"; }
const char *hipGetErrorString(hipError_t) { return "a launch that the test made fail"; }
hipError_t hipStreamCreate(hipStream_t *s) { return *s = (hipStream_t)std::malloc(1), hipSuccess; }
hipError_t hipStreamDestroy(hipStream_t s) { return std::free((void *)s), hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return ++g_waits, hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus *c) {
    return *c = hipStreamCaptureStatusNone, hipSuccess;
}
hipError_t hipMalloc(void **p, size_t n) {
    *p = std::malloc(n + 1);
    std::memset(*p, 0xff, n);  // (bf16 and f32 NaN)
    return hipSuccess;
}
hipError_t hipFree(void *p) { return std::free(p), hipSuccess; }
hipError_t hipHostMalloc(void **p, size_t n, unsigned) { return hipMalloc(p, n); }
hipError_t hipHostFree(void *p) { return std::free(p), hipSuccess; }
hipError_t hipHostGetDevicePointer(void **d, void *h, unsigned) { return *d = h, hipSuccess; }
hipError_t hipMemset(void *p, int v, size_t n) { return std::memset(p, v, n), hipSuccess; }
hipError_t hipMemsetAsync(void *p, int v, size_t n, hipStream_t) { return hipMemset(p, v, n); }
hipError_t hipMemcpy(void *to, const void *from, size_t n, hipMemcpyKind) {
    return std::memmove(to, from, n), hipSuccess;
}
hipError_t hipMemcpyAsync(void *to, const void *from, size_t n, hipMemcpyKind k, hipStream_t) {
    return hipMemcpy(to, from, n, k);
}
hipError_t hipEventCreate(hipEvent_t *e) { return *e = (hipEvent_t)std::malloc(1), hipSuccess; }
hipError_t hipEventCreateWithFlags(hipEvent_t *e, unsigned) { return hipEventCreate(e); }
hipError_t hipEventDestroy(hipEvent_t e) { return std::free((void *)e), hipSuccess; }
hipError_t hipEventRecord(hipEvent_t, hipStream_t) { return launch("event"); }
hipError_t hipEventSynchronize(hipEvent_t) { return hipSuccess; }
hipError_t hipEventElapsedTime(float *t, hipEvent_t, hipEvent_t) { return *t = 0, hipSuccess; }

}  // extern "C"

namespace sr {

// ------------------------------------------------------------------ pages

hipError_t launch_page_table_set(hipStream_t, int32_t *table, const uint32_t *idx, const int32_t *val, int n) {
    const hipError_t e = launch("page_table_set");
    for (int i = 0; e == hipSuccess && i < n; ++i) table[idx[i]] = val[i];
    return e;
}
hipError_t launch_page_copy(hipStream_t, const Pool *p, int32_t dst, int32_t src) {
    const size_t bytes = (size_t)p->page_tokens * p->head_dim * 2;
    for (uint32_t h = 0; h < p->kv_heads; ++h) {
        for (uint16_t *pages : {p->k_pages, p->v_pages}) {
            std::memcpy(pages + row_of(p, dst, 0, h) * p->head_dim, pages + row_of(p, src, 0, h) * p->head_dim, bytes);
        }
    }
    return launch("page_copy");
}
hipError_t launch_kv_scatter(hipStream_t, const Pool *p, uint32_t slot, uint64_t start, uint64_t tokens,
                             const void *keys, const void *values, bool bf16_in, uint32_t *) {
    const int32_t *table = p->d_page_table + (size_t)slot * p->pages_per_seq;
    for (uint64_t t = 0; t < tokens; ++t) {
        for (uint32_t i = 0; i < p->kv_heads * p->head_dim; ++i) {
            const size_t from = t * p->kv_heads * p->head_dim + i;
            const size_t to = row_of(p, table[(start + t) / p->page_tokens], start + t, i / p->head_dim) *
                                  p->head_dim + i % p->head_dim;
            p->k_pages[to] = bf16_in ? ((const uint16_t *)keys)[from] : as_bf16(((const float *)keys)[from]);
            p->v_pages[to] = bf16_in ? ((const uint16_t *)values)[from] : as_bf16(((const float *)values)[from]);
        }
    }
    return launch("kv_scatter");
}
hipError_t launch_kv_gather(hipStream_t, const Pool *p, uint32_t slot, uint64_t start, uint64_t tokens,
                            float *keys, float *values) {
    const int32_t *table = p->d_page_table + (size_t)slot * p->pages_per_seq;
    for (uint64_t t = 0; t < tokens; ++t) {
        for (uint32_t i = 0; i < p->kv_heads * p->head_dim; ++i) {
            const size_t from = row_of(p, table[(start + t) / p->page_tokens], start + t, i / p->head_dim) *
                                    p->head_dim + i % p->head_dim;
            keys[t * p->kv_heads * p->head_dim + i] = as_float(p->k_pages[from]);
            values[t * p->kv_heads * p->head_dim + i] = as_float(p->v_pages[from]);
        }
    }
    return launch("kv_gather");
}
hipError_t launch_linear_input(hipStream_t, const float *src, float *dst, uint64_t count) {
    const hipError_t e = launch("linear_input");
    if (e == hipSuccess) std::memcpy(dst, src, count * 4);
    return e;
}

hipError_t launch_kv_moves(hipStream_t, const MoveCall &c) {
    if (c.chains + c.links == 0) return hipSuccess;
    const hipError_t e = launch("kv_moves");
    if (e != hipSuccess) return e;
    const uint32_t *w = c.device_words != nullptr ? c.device_words : c.host_words;
    const MoveEntry *entries = (const MoveEntry *)w;
    const MoveRange *ranges = (const MoveRange *)(entries + c.entries);
    const MoveLink *links = (const MoveLink *)(ranges + c.ranges);
    std::vector<Group> groups;
    for (uint32_t i = 0; i < c.chains; ++i) {
        for (uint32_t h = 0; h < entries[ranges[i].entry].kv_heads; ++h) {
            for (bool values : {false, true}) groups.push_back({i, h, values, ranges[i].begin});
        }
    }
    std::vector<uint32_t> open_links;
    for (uint32_t i = 0; i < c.links; ++i) open_links.push_back(i);
    while (!groups.empty() || !open_links.empty()) {
        if (!open_links.empty() && random_below(8) == 0) {
            const MoveLink &l = links[open_links.back()];
            open_links.pop_back();
            for (uint32_t i = 0; i < l.count; ++i) l.row[i] = (int32_t)w[l.pages + i];
            continue;
        }
        if (groups.empty()) continue;
        // a few tokens of some workgroup: all are read, then all are written
        Group &g = groups[random_below((uint32_t)groups.size())];
        const MoveRange &r = ranges[g.range];
        const MoveEntry &m = entries[r.entry];
        const uint32_t n = std::min(1 + random_below(24), r.end - g.at), mask = (1u << m.log2_page) - 1;
        uint16_t *pages = g.values ? m.v_pages : m.k_pages;
        auto place = [&](int32_t page, uint32_t t) {
            return ((((size_t)g.head * m.num_pages + page) << m.log2_page) + (t & mask)) * m.head_dim;
        };
        std::vector<uint16_t> rows((size_t)n * m.head_dim);
        for (uint32_t i = 0; i < n; ++i) {
            const uint32_t t = g.at + i, s = t < m.start ? t : m.start + w[m.tokens + t - m.start];
            std::memcpy(&rows[(size_t)i * m.head_dim], pages + place(m.from[s >> m.log2_page], s), m.head_dim * 2);
        }
        for (uint32_t i = 0; i < n; ++i) {
            const uint32_t t = g.at + i;
            std::memcpy(pages + place((int32_t)w[m.pages + (t >> m.log2_page) - m.first_page], t),
                        &rows[(size_t)i * m.head_dim], m.head_dim * 2);
        }
        g.at += n;
        if (g.at < r.end) continue;
        if (r.next != 0) {
            g.range = r.next;
            g.at = ranges[r.next].begin;
        } else {
            std::swap(g, groups.back());
            groups.pop_back();
        }
    }
    return hipSuccess;
}
hipError_t launch_kv_links(hipStream_t, const MoveCall &c) {
    if (c.late_links == 0) return hipSuccess;
    const hipError_t e = launch("kv_links");
    const uint32_t *w = c.device_words != nullptr ? c.device_words : c.host_words;
    const MoveLink *links = (const MoveLink *)((const MoveRange *)((const MoveEntry *)w + c.entries) + c.ranges);
    for (uint32_t k = 0; e == hipSuccess && k < c.late_links; ++k) {
        const MoveLink &l = links[c.links + k];
        for (uint32_t i = 0; i < l.count; ++i) l.row[i] = (int32_t)w[l.pages + i];
    }
    return e;
}
hipError_t launch_kv_gather_rows(hipStream_t, const GatherCall &c) {
    const hipError_t e = launch("kv_gather_rows");
    const uint32_t *w = c.device_words != nullptr ? c.device_words : c.host_words;
    const GatherEntry *entries = (const GatherEntry *)w;
    for (uint32_t k = 0; e == hipSuccess && k < c.entries; ++k) {
        const GatherEntry &g = entries[k];
        for (uint32_t t = 0; t < g.count; ++t) {
            const uint32_t s = g.start + (g.tokens != 0 ? w[g.tokens + t] : t);
            for (uint32_t i = 0; i < c.kv_heads * c.head_dim; ++i) {
                const size_t from = ((((size_t)(i / c.head_dim) * g.num_pages + g.from[s >> g.log2_page])
                                      << g.log2_page) + (s & ((1u << g.log2_page) - 1))) * c.head_dim + i % c.head_dim;
                const size_t to = (g.first + t) * c.kv_heads * c.head_dim + i;
                if (c.bf16_out) {
                    ((uint16_t *)c.keys)[to] = g.k_pages[from];
                    ((uint16_t *)c.values)[to] = g.v_pages[from];
                } else {
                    ((float *)c.keys)[to] = as_float(g.k_pages[from]);
                    ((float *)c.values)[to] = as_float(g.v_pages[from]);
                }
            }
        }
    }
    return e;
}

// ------------------------------------------------------------------ not here

bool generic_head_dim(uint32_t) { return true; }
bool prefill_supported(const AttnLaunch &) { return false; }
size_t prefill_rope_bytes(const AttnLaunch &, uint64_t) { return 0; }
bool verify_supported(const AttnLaunch &, uint32_t) { return false; }
bool split_fits(const AttnLaunch &, const SeqMeta *, int, int, uint64_t) { return false; }
hipError_t launch_attn_decode(hipStream_t, const AttnLaunch &, const SeqMeta *, int, const DecodePlanInput &) {
    return hipErrorNotSupported;
}
hipError_t launch_attn_prefill(hipStream_t, const AttnLaunch &, const SeqMeta *, int, void *) {
    return hipErrorNotSupported;
}
hipError_t launch_attn_generic(hipStream_t, const AttnLaunch &, const SeqMeta *, int) { return hipErrorNotSupported; }
hipError_t launch_attn_verify(hipStream_t, const AttnLaunch &, const SeqMeta *, int, void *, const DecodePlanInput &,
                              uint64_t) {
    return hipErrorNotSupported;
}
TreeScratch tree_scratch(const TreeLaunch &, const SeqMeta *, int, uint64_t, int) { return {}; }
hipError_t launch_tree_attn(hipStream_t, const TreeLaunch &, const SeqMeta *, int, const uint8_t *, const TreePlan &) {
    return hipErrorNotSupported;
}
// (launched, and computing nothing)
hipError_t launch_gdn(hipStream_t, const GdnLaunch &, const GdnSeq *, int, uint32_t) { return launch("gdn"); }
size_t gdn_chunk_rec_bytes(const safetyraise_kernel_gdn_pool *, const GdnSeq *, int, bool, bool) { return 0; }
hipError_t launch_gdn_rollback(hipStream_t, const GdnRollback &) { return launch("gdn_rollback"); }
size_t gdn_tree_scratch_bytes(const safetyraise_kernel_gdn_pool *, uint32_t) { return 0; }
hipError_t launch_gdn_tree(hipStream_t, const GdnLaunch &, const GdnSeq *, int, const uint8_t *, float *) {
    return launch("gdn_tree");
}
hipError_t launch_gdn_tree_commit(hipStream_t, const GdnCommitEntry *, uint32_t, const GdnCommitEntry *) {
    return launch("gdn_tree_commit");
}
uint32_t gdn_key_dim() { return 128; }
uint32_t gdn_row_block() { return 64; }
uint32_t gdn_max_kernel() { return 8; }
size_t linear_scratch_bytes(uint32_t, uint32_t, uint32_t, uint32_t, int, bool, bool) { return 0; }
size_t linear_weight_bytes(uint64_t, uint64_t, uint32_t) { return 1; }
hipError_t linear_pack_bf16(hipStream_t, const void *, void *, uint64_t, uint64_t) { return hipErrorNotSupported; }
hipError_t launch_linear(hipStream_t, const float *, const void *, uint32_t, float *, uint32_t, uint32_t, uint32_t,
                         const LinScratch &, int) {
    return hipErrorNotSupported;
}

}  // namespace sr
