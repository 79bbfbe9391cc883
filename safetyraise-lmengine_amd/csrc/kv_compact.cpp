// kv_compact and kv_gather: chosen tokens of sequences kept, or copied out.
//
// The page lists change on the host when the call is made, as in kv.cpp; the
// copies and the page tables follow on the context's stream.  Every entry is
// checked and planned before anything changes.

#include <algorithm>
#include <cstring>
#include <map>
#include <utility>
#include <vector>

#include "kv_moves.hpp"
#include "kv_plan.hpp"
#include "sr_internal.hpp"

namespace sr {

int32_t upload_words(Ctx *ctx, const uint32_t *words, size_t count, const uint32_t **out) {
    UploadSlot &u = ctx->upload[ctx->upload_next];
    ctx->upload_next = (ctx->upload_next + 1) % kUploadSlots;
    const size_t bytes = (count * 4 + 15) & ~(size_t)15;
    if (u.pending) {
        SR_HIP(ctx, hipEventSynchronize(u.fetched));
        u.pending = false;
    }
    if (u.fetched == nullptr) SR_HIP(ctx, hipEventCreateWithFlags(&u.fetched, hipEventDisableTiming));
    if (u.bytes < bytes) {
        const size_t want = std::max<size_t>(2 * bytes, 65536);
        if (u.host != nullptr) SR_HIP(ctx, hipHostFree(u.host));
        u.host = nullptr;
        u.bytes = 0;
        SR_HIP(ctx, hipHostMalloc(&u.host, want, hipHostMallocDefault));
        SR_HIP(ctx, hipHostGetDevicePointer(&u.host_dev, u.host, 0));
        u.bytes = want;
    }
    const int32_t st = ensure_buffer(ctx, u.dev, u.bytes, false);
    if (st != kOk) return st;
    std::memcpy(u.host, words, count * 4);
    SR_HIP(ctx, launch_linear_input(ctx->stream, (const float *)u.host_dev, (float *)u.dev.ptr, bytes / 4));
    SR_HIP(ctx, hipEventRecord(u.fetched, ctx->stream));
    u.pending = true;
    *out = (const uint32_t *)u.dev.ptr;
    return kOk;
}

namespace {

using Pool = safetyraise_kernel_kv_pool;

bool is_open(const Pool *pool, uint32_t seq) {
    return seq < pool->max_sequences && pool->seqs[seq].open;
}

template <class T>
void put(std::vector<uint32_t> &words, const T &x) {
    const size_t at = words.size();
    words.resize(at + sizeof(T) / 4);
    std::memcpy(words.data() + at, &x, sizeof(T));
}

int32_t compact(Ctx *ctx, const safetyraise_kernel_kv_keep *entries, uint32_t n, uint32_t flags) {
    if (entries == nullptr || n == 0 || (flags & ~SAFETYRAISE_MI355X_ASYNC) != 0) {
        return fail(ctx, kInvalid, "kv_compact needs entries, and no flag but ASYNC");
    }
    const bool async = (flags & SAFETYRAISE_MI355X_ASYNC) != 0;
    // who is source and target of which entries
    std::vector<std::pair<std::pair<Pool *, uint32_t>, uint32_t>> uses;  // (sequence, entry)
    for (uint32_t i = 0; i < n; ++i) {
        const auto &e = entries[i];
        if (e.kv == nullptr || !is_open(e.kv, e.source) || !is_open(e.kv, e.target)) {
            return fail(ctx, kInvalid, "KV sequence handle is not open");
        }
        const uint64_t len = e.kv->seqs[e.source].len;
        if (e.start > len || e.count > len - e.start || (e.count > 0 && e.tokens == nullptr)) {
            return fail(ctx, kInvalid, "KV token index out of range");
        }
        for (uint64_t j = 0; j < e.count; ++j) {
            if (e.tokens[j] >= len - e.start || (j > 0 && e.tokens[j] <= e.tokens[j - 1])) {
                return fail(ctx, kInvalid,
                            "kv_compact tokens must ascend strictly and stay within the sequence");
            }
        }
        uses.push_back({{e.kv, e.source}, i});
        if (e.target != e.source) uses.push_back({{e.kv, e.target}, i});
    }
    std::sort(uses.begin(), uses.end());
    for (size_t i = 0; i < uses.size();) {
        size_t end = i;
        bool target = false;
        while (end < uses.size() && uses[end].first == uses[i].first) {
            target = target || entries[uses[end].second].target == uses[i].first.second;
            ++end;
        }
        if (target && end - i > 1) {
            return fail(ctx, kInvalid, "a target of kv_compact may not appear in another entry");
        }
        i = end;
    }
    if (!async) {
        const int32_t st = report_pending_async(ctx);
        if (st != kOk) return st;
    }

    // plans, against the pages that are free now or that a target gives up
    std::map<Pool *, uint64_t> free_pages;
    for (uint32_t i = 0; i < n; ++i) {
        Pool *pool = entries[i].kv;
        auto at = free_pages.emplace(pool, pool->free_pages.size()).first;
        if (entries[i].target == entries[i].source) continue;
        for (int32_t page : pool->seqs[entries[i].target].pages) at->second += pool->refcount[page] == 1;
    }
    std::vector<CompactPlan> plans(n);
    for (uint32_t i = 0; i < n; ++i) {
        const auto &e = entries[i];
        const auto &src = e.kv->seqs[e.source];
        const KeepList keep{e.start, e.count, e.tokens};
        uint64_t &free = free_pages[e.kv];
        plans[i] = compact_plan(keep, e.kv->page_tokens, e.target == e.source, free, [&](uint64_t q) {
            return e.kv->refcount[src.pages[q]] == 1;
        });
        if (plans[i].fresh > free) return fail(ctx, kNoMemory, "KV page pool exhausted");
        free -= plans[i].fresh;
    }

    // the new page lists, as the kernels' words
    MoveCall call{};
    std::vector<uint32_t> words, lists;
    std::vector<MoveEntry> moves(n);
    std::vector<MoveRange> heads, tails;
    std::vector<MoveLink> links, late;
    std::vector<std::vector<int32_t>> pages(n);
    size_t ranges = 0;
    for (const CompactPlan &p : plans) ranges += p.ranges.size();
    size_t link_count = 0;
    for (uint32_t i = 0; i < n; ++i) {
        const uint64_t len = entries[i].start + entries[i].count;
        link_count += len > plans[i].first * entries[i].kv->page_tokens ? 1 : 0;
    }
    const size_t fixed = (n * sizeof(MoveEntry) + ranges * sizeof(MoveRange) +
                          (link_count + 1) * sizeof(MoveLink)) / 4;
    // pages that targets give up first, so that they are free for the call
    for (uint32_t i = 0; i < n; ++i) {
        const auto &e = entries[i];
        if (e.target == e.source) continue;
        auto &t = e.kv->seqs[e.target];
        for (int32_t page : t.pages) {
            if (--e.kv->refcount[page] == 0) e.kv->free_pages.push_back(page);
        }
        t.pages.clear();
        t.len = 0;
    }
    std::map<std::pair<const uint32_t *, uint64_t>, uint32_t> shared;  // token lists already there
    for (uint32_t i = 0; i < n; ++i) {
        const auto &e = entries[i];
        Pool *pool = e.kv;
        const CompactPlan &p = plans[i];
        const auto &old = pool->seqs[e.source].pages;
        std::vector<int32_t> &now = pages[i];
        now.assign(old.begin(), old.begin() + (ptrdiff_t)p.first);
        for (int64_t take : p.take) {
            if (take >= 0) {
                now.push_back(old[(size_t)take]);
            } else {
                now.push_back(pool->free_pages.back());
                pool->free_pages.pop_back();
                pool->refcount[now.back()] = 0;
            }
        }
        for (int32_t page : now) ++pool->refcount[page];
        MoveEntry &m = moves[i];
        m.k_pages = pool->k_pages;
        m.v_pages = pool->v_pages;
        m.from = pool->d_page_table + (size_t)e.source * pool->pages_per_seq;
        m.num_pages = pool->num_pages;
        m.kv_heads = pool->kv_heads;
        m.head_dim = pool->head_dim;
        m.log2_page = (uint32_t)__builtin_ctz(pool->page_tokens);
        m.start = (uint32_t)e.start;
        m.first_page = (uint32_t)p.first;
        m.pages = (uint32_t)(fixed + lists.size());
        for (size_t q = p.first; q < now.size(); ++q) lists.push_back((uint32_t)now[q]);
        if (!p.ranges.empty()) {
            // layers usually keep the same tokens
            const auto known = shared.emplace(std::make_pair(e.tokens, e.count), (uint32_t)(fixed + lists.size()));
            if (known.second) lists.insert(lists.end(), e.tokens, e.tokens + e.count);
            m.tokens = known.first->second;
            call.kv_heads = std::max(call.kv_heads, pool->kv_heads);
        }
        bool changed = e.target != e.source;
        for (size_t q = p.first; q < now.size() && !changed; ++q) changed = now[q] != old[q];
        if (changed && now.size() > p.first) {
            const MoveLink l{pool->d_page_table + (size_t)e.target * pool->pages_per_seq + p.first,
                             m.pages, (uint32_t)(now.size() - p.first)};
            (e.target != e.source ? links : late).push_back(l);
        }
        for (size_t r = 0; r < p.ranges.size(); ++r) {
            const MoveRange range{i, (uint32_t)p.ranges[r].begin, (uint32_t)p.ranges[r].end, 0};
            (p.serial && r > 0 ? tails : heads).push_back(range);
        }
    }
    // chains: a serial entry's later ranges follow its first
    {
        size_t at = 0, head = 0;
        for (uint32_t i = 0; i < n; ++i) {
            const size_t count = plans[i].ranges.size();
            if (plans[i].serial && count > 1) {
                MoveRange *last = &heads[head];
                for (size_t r = 1; r < count; ++r) {
                    last->next = (uint32_t)(heads.size() + at);
                    last = &tails[at++];
                }
            }
            head += plans[i].serial ? std::min<size_t>(count, 1) : count;
        }
    }
    call.entries = n;
    call.chains = (uint32_t)heads.size();
    call.ranges = (uint32_t)(heads.size() + tails.size());
    call.links = (uint32_t)links.size();
    call.late_links = (uint32_t)late.size();
    if (call.kv_heads == 0) call.kv_heads = 1;
    for (const MoveEntry &m : moves) put(words, m);
    for (const MoveRange &r : heads) put(words, r);
    for (const MoveRange &r : tails) put(words, r);
    for (const MoveLink &l : links) put(words, l);
    for (const MoveLink &l : late) put(words, l);
    words.resize(fixed);
    words.insert(words.end(), lists.begin(), lists.end());
    // the sequences have their new pages from here on, whatever the launches say
    for (uint32_t i = 0; i < n; ++i) {
        const auto &e = entries[i];
        auto &t = e.kv->seqs[e.target];
        if (e.target == e.source) {
            for (int32_t page : t.pages) {
                if (--e.kv->refcount[page] == 0) e.kv->free_pages.push_back(page);
            }
        }
        t.pages = std::move(pages[i]);
        t.len = e.start + e.count;
    }
    call.host_words = words.data();
    call.words = (uint32_t)words.size();
    if (call.chains + call.links + call.late_links > 0) {
        if (words.size() > kMoveInlineWords) {
            const int32_t st = upload_words(ctx, words.data(), words.size(), &call.device_words);
            if (st != kOk) return st;
        }
        SR_HIP(ctx, launch_kv_moves(ctx->stream, call));
    }
    return finish_call(ctx, async);
}

int32_t gather(Ctx *ctx, const safetyraise_kernel_kv_rows *entries, uint32_t n, void *keys, void *values,
               uint32_t flags) {
    const bool device = (flags & SAFETYRAISE_MI355X_DEVICE_POINTERS) != 0;
    const bool async = (flags & SAFETYRAISE_MI355X_ASYNC) != 0;
    const bool out16 = (flags & SAFETYRAISE_MI355X_OUTPUT_BF16) != 0;
    if (entries == nullptr || n == 0 ||
        (flags & ~(SAFETYRAISE_MI355X_DEVICE_POINTERS | SAFETYRAISE_MI355X_ASYNC |
                   SAFETYRAISE_MI355X_OUTPUT_BF16)) != 0) {
        return fail(ctx, kInvalid, "kv_gather needs entries, and no flags but DEVICE_POINTERS, ASYNC, OUTPUT_BF16");
    }
    if (async && !device) return fail(ctx, kInvalid, "ASYNC needs DEVICE_POINTERS");
    uint64_t total = 0;
    for (uint32_t i = 0; i < n; ++i) {
        const auto &e = entries[i];
        if (e.kv == nullptr || !is_open(e.kv, e.sequence) || e.reserved != 0) {
            return fail(ctx, kInvalid, "KV sequence handle is not open");
        }
        if (e.kv->kv_heads != entries[0].kv->kv_heads || e.kv->head_dim != entries[0].kv->head_dim) {
            return fail(ctx, kInvalid, "kv_gather pools differ in kv_heads or head_dim");
        }
        const uint64_t len = e.kv->seqs[e.sequence].len;
        if (e.start > len || (e.tokens == nullptr && e.count > len - e.start)) {
            return fail(ctx, kInvalid, "KV token index out of range");
        }
        for (uint64_t j = 0; e.tokens != nullptr && j < e.count; ++j) {
            if (e.tokens[j] >= len - e.start) return fail(ctx, kInvalid, "KV token index out of range");
        }
        if (e.count > INT32_MAX) return fail(ctx, kOverflow, "too many tokens");
        total += e.count;
    }
    if (!async) {
        const int32_t st = report_pending_async(ctx);
        if (st != kOk) return st;
    }
    if (total == 0) return finish_call(ctx, async);
    if (keys == nullptr || values == nullptr) return fail(ctx, kInvalid, "NULL argument");
    if (device && (((uintptr_t)keys | (uintptr_t)values) & 15u) != 0) {
        return fail(ctx, kInvalid, "device pointers must be 16-byte aligned");
    }
    GatherCall call{};
    call.kv_heads = entries[0].kv->kv_heads;
    call.head_dim = entries[0].kv->head_dim;
    call.tokens = total;
    call.bf16_out = out16;
    uint64_t bytes = 0;
    if (!checked_mul(total, (uint64_t)call.kv_heads * call.head_dim * (out16 ? 2 : 4), &bytes)) {
        return fail(ctx, kOverflow, "kv_gather size overflows");
    }
    std::vector<uint32_t> words, lists;
    std::map<std::pair<const uint32_t *, uint64_t>, uint32_t> shared;
    const size_t fixed = n * sizeof(GatherEntry) / 4;
    uint64_t first = 0;
    for (uint32_t i = 0; i < n; ++i) {
        const auto &e = entries[i];
        if (e.count == 0) continue;  // no token searches for it
        GatherEntry g{};
        g.k_pages = e.kv->k_pages;
        g.v_pages = e.kv->v_pages;
        g.from = e.kv->d_page_table + (size_t)e.sequence * e.kv->pages_per_seq;
        g.num_pages = e.kv->num_pages;
        g.first = first;
        g.log2_page = (uint32_t)__builtin_ctz(e.kv->page_tokens);
        g.start = (uint32_t)e.start;
        if (e.tokens != nullptr) {
            const auto known = shared.emplace(std::make_pair(e.tokens, e.count), (uint32_t)(fixed + lists.size()));
            if (known.second) lists.insert(lists.end(), e.tokens, e.tokens + e.count);
            g.tokens = known.first->second;
        }
        put(words, g);
        ++call.entries;
        first += e.count;
    }
    words.resize(fixed);
    words.insert(words.end(), lists.begin(), lists.end());
    call.host_words = words.data();
    call.words = (uint32_t)words.size();
    if (words.size() > kMoveInlineWords - 16) {
        const int32_t st = upload_words(ctx, words.data(), words.size(), &call.device_words);
        if (st != kOk) return st;
    }
    call.keys = keys;
    call.values = values;
    const size_t half = (bytes + 255) & ~(size_t)255;
    if (!device) {
        const int32_t st = ensure_buffer(ctx, ctx->staging, 2 * half, false);
        if (st != kOk) return st;
        call.keys = ctx->staging.ptr;
        call.values = (char *)ctx->staging.ptr + half;
    }
    SR_HIP(ctx, launch_kv_gather_rows(ctx->stream, call));
    if (!device) {
        SR_HIP(ctx, hipMemcpyAsync(keys, call.keys, bytes, hipMemcpyDeviceToHost, ctx->stream));
        SR_HIP(ctx, hipMemcpyAsync(values, call.values, bytes, hipMemcpyDeviceToHost, ctx->stream));
    }
    return finish_call(ctx, async);
}

}  // namespace

}  // namespace sr

using namespace sr;

extern "C" {

SAFETYRAISE_KERNEL_EXPORT int32_t safetyraise_kernel_kv_compact(
    safetyraise_kernel_context *context, const safetyraise_kernel_kv_keep *entries,
    uint32_t num_entries, uint32_t flags) {
    if (context == nullptr) return kInvalid;
    const int32_t capture = refuse_under_capture(context, "kv_compact");
    if (capture != kOk) return capture;
    DeviceScope device_scope(context);
    TimerScope timer_scope(context);
    return no_throw(context, [&] { return compact(context, entries, num_entries, flags); });
}

SAFETYRAISE_KERNEL_EXPORT int32_t safetyraise_kernel_kv_gather(
    safetyraise_kernel_context *context, const safetyraise_kernel_kv_rows *entries,
    uint32_t num_entries, void *keys, void *values, uint32_t flags) {
    if (context == nullptr) return kInvalid;
    const int32_t capture = refuse_under_capture(context, "kv_gather");
    if (capture != kOk) return capture;
    DeviceScope device_scope(context);
    TimerScope timer_scope(context);
    return no_throw(context, [&] { return gather(context, entries, num_entries, keys, values, flags); });
}

}  // extern "C"
