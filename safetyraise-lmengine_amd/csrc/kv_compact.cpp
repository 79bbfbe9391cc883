// kv_compact and kv_gather: chosen tokens of sequences kept, or copied out.
//
// The page lists change on the host when the call is made, as in kv.cpp; the
// copies and the page tables follow on the context's stream.  Every entry is
// checked and planned before anything changes.

#include <algorithm>
#include <atomic>
#include <cstring>
#include <utility>
#include <vector>

#include "kv_moves.hpp"
#include "kv_plan.hpp"
#include "sr_internal.hpp"

namespace sr {

int32_t upload_room(Ctx *ctx, size_t count, uint32_t **host) {
    UploadSlot &u = ctx->upload[ctx->upload_next];
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
    *host = (uint32_t *)u.host;
    return kOk;
}

int32_t upload_words(Ctx *ctx, size_t count, const uint32_t **device) {
    UploadSlot &u = ctx->upload[ctx->upload_next];
    ctx->upload_next = (ctx->upload_next + 1) % kUploadSlots;
    SR_HIP(ctx, launch_linear_input(ctx->stream, (const float *)u.host_dev, (float *)u.dev.ptr,
                                    (count + 3) / 4 * 4));
    const hipError_t e = hipEventRecord(u.fetched, ctx->stream);
    if (e != hipSuccess) {
        (void)hipStreamSynchronize(ctx->stream);  // the slot's words are still being read
        return hip_fail(ctx, e, "hipEventRecord");
    }
    u.pending = true;
    *device = (const uint32_t *)u.dev.ptr;
    return kOk;
}

namespace {

using Pool = safetyraise_kernel_kv_pool;

bool is_open(const Pool *pool, uint32_t seq) {
    return seq < pool->max_sequences && pool->seqs[seq].open;
}

// The words of a call: in the kernel arguments (`small`) or in an upload slot.
struct Words {
    alignas(16) uint32_t small[kMoveInlineWords];
    uint32_t *at = nullptr;

    int32_t open(Ctx *ctx, size_t count, size_t most_inline) {
        if (count <= most_inline) {
            at = small;
            return kOk;
        }
        return upload_room(ctx, count, &at);
    }
    // the device address, or nullptr for words in the arguments
    int32_t send(Ctx *ctx, size_t count, const uint32_t **device) {
        *device = nullptr;
        return at == small ? kOk : upload_words(ctx, count, device);
    }
};

// Whether all tokens are below the limit (> 0).  The sign of t | (limit - 1 - t) says so for
// a limit up to 2^31, in operations of every vector unit.
bool all_below(const uint32_t *tokens, uint64_t count, uint64_t limit) {
    uint32_t bad = 0;
    if (limit <= 1ull << 31) {
        const uint32_t top = (uint32_t)limit - 1;
        for (uint64_t j = 0; j < count; ++j) bad |= tokens[j] | (top - tokens[j]);
        return bad >> 31 == 0;
    }
    for (uint64_t j = 0; j < count; ++j) bad |= tokens[j] >= limit ? 1u : 0u;
    return bad == 0;
}

bool all_ascend(const uint32_t *tokens, uint64_t count) {
    if (count == 0) return true;
    uint32_t bad = 0, high = tokens[0];
    for (uint64_t j = 1; j < count; ++j) {
        bad |= tokens[j] - tokens[j - 1] - 1;
        high |= tokens[j];
    }
    if (high >> 31 == 0) return bad >> 31 == 0;
    for (uint64_t j = 1; j < count; ++j) {
        if (tokens[j] <= tokens[j - 1]) return false;
    }
    return true;
}

// Token lists of a call by address: layers usually share them.
struct Lists {
    struct One {
        const uint32_t *tokens;
        uint64_t count;
        uint64_t below;   // all tokens are below it (0: not looked at)
        bool ascending;   // (likewise)
        uint32_t offset;  // in the words; 0: not yet
    };
    std::vector<One> lists;

    // the index of a list (a shared one may be there twice: only the last few are
    // looked through)
    uint32_t add(const uint32_t *tokens, uint64_t count) {
        for (size_t i = lists.size(); i-- > 0 && i + 32 > lists.size();) {
            if (lists[i].tokens == tokens && lists[i].count == count) return (uint32_t)i;
        }
        lists.push_back({tokens, count, 0, false, 0});
        return (uint32_t)lists.size() - 1;
    }
    bool below(uint32_t i, uint64_t limit) {
        One &l = lists[i];
        if (l.below != 0 && l.below <= limit) return true;
        if (limit == 0 || !all_below(l.tokens, l.count, limit)) return false;
        l.below = limit;
        return true;
    }
    // ascending strictly, and below the limit
    bool ascend_below(uint32_t i, uint64_t limit) {
        One &l = lists[i];
        l.ascending = l.ascending || all_ascend(l.tokens, l.count);
        return l.ascending && l.tokens[l.count - 1] < limit;
    }
};

// A plan, and what it holds for (plans of other layers are often the same)
struct KnownPlan {
    const uint32_t *tokens;
    uint64_t count, start;
    uint32_t page_tokens;
    bool in_place;
    CompactPlan plan;
};

uint64_t next_call() {
    static std::atomic<uint64_t> calls{0};
    return ++calls;
}

// Shared pages of the pool that no sequence holds but targets of the call, which give
// them up before any entry takes one.  (Pages of one target alone are counted for
// every call; this walk over the pool is for one that would be short of pages.)
uint64_t given_up_together(const safetyraise_kernel_kv_keep *entries, uint32_t n, const Pool *pool) {
    std::vector<uint32_t> targets(pool->num_pages);
    uint64_t pages = 0;
    for (uint32_t i = 0; i < n; ++i) {
        const auto &e = entries[i];
        if (e.kv != pool || e.target == e.source) continue;
        for (int32_t page : pool->seqs[e.target].pages) {
            if (pool->refcount[page] > 1 && ++targets[page] == pool->refcount[page]) ++pages;
        }
    }
    return pages;
}

int32_t compact(Ctx *ctx, const safetyraise_kernel_kv_keep *entries, uint32_t n, uint32_t flags) {
    if (entries == nullptr || n == 0 || (flags & ~SAFETYRAISE_MI355X_ASYNC) != 0) {
        return fail(ctx, kInvalid, "kv_compact needs entries, and no flag but ASYNC");
    }
    const bool async = (flags & SAFETYRAISE_MI355X_ASYNC) != 0;
    const uint64_t id = next_call();
    Lists lists;
    std::vector<uint32_t> list_of(n);
    for (uint32_t i = 0; i < n; ++i) {
        const auto &e = entries[i];
        if (e.kv == nullptr || !is_open(e.kv, e.source) || !is_open(e.kv, e.target)) {
            return fail(ctx, kInvalid, "KV sequence handle is not open");
        }
        auto &source = e.kv->seqs[e.source], &target = e.kv->seqs[e.target];
        if (e.start > source.len || e.count > source.len - e.start || (e.count > 0 && e.tokens == nullptr)) {
            return fail(ctx, kInvalid, "KV token index out of range");
        }
        if (e.count > 0) {
            list_of[i] = lists.add(e.tokens, e.count);
            if (!lists.ascend_below(list_of[i], source.len - e.start)) {
                return fail(ctx, kInvalid,
                            "kv_compact tokens must ascend strictly and stay within the sequence");
            }
        }
        if (target.source_of == id || target.target_of == id || source.target_of == id) {
            return fail(ctx, kInvalid, "a target of kv_compact may not appear in another entry");
        }
        source.source_of = id;
        target.target_of = id;
        if (e.kv->compact_call != id) {
            e.kv->compact_call = id;
            e.kv->compact_free = e.kv->free_pages.size();
        }
        if (e.target != e.source) {
            for (int32_t page : target.pages) e.kv->compact_free += e.kv->refcount[page] == 1;
        }
    }
    if (!async) {
        const int32_t st = report_pending_async(ctx);
        if (st != kOk) return st;
    }

    // plans, against the pages that are free now or that targets give up
    std::vector<KnownPlan> known;
    std::vector<uint32_t> plan_of(n);
    size_t ranges = 0, links = 0, words = 0;
    uint32_t chains = 0, kv_heads = 1, in_flight = UINT32_MAX;
    uint64_t longest = 1;
    for (uint32_t i = 0; i < n; ++i) {
        const auto &e = entries[i];
        Pool *pool = e.kv;
        const auto &old = pool->seqs[e.source].pages;
        const bool in_place = e.target == e.source;
        bool own = true;  // (of the pages that may be written)
        const uint64_t pages = (e.start + e.count + pool->page_tokens - 1) / pool->page_tokens;
        for (uint64_t q = e.start / pool->page_tokens; in_place && q < pages; ++q) own = own && pool->refcount[old[q]] == 1;
        size_t at = known.size();
        for (size_t k = known.size(); own && k-- > 0 && k + 16 > known.size();) {
            const KnownPlan &x = known[k];
            if (x.tokens == e.tokens && x.count == e.count && x.start == e.start &&
                x.page_tokens == pool->page_tokens && x.in_place == in_place &&
                x.plan.wanted <= pool->compact_free) {
                at = k;
                break;
            }
        }
        if (at == known.size()) {
            const KeepList keep{e.start, e.count, e.tokens};
            known.push_back({own ? e.tokens : nullptr, own ? e.count : UINT64_MAX, e.start, pool->page_tokens, in_place,
                             compact_plan(keep, pool->page_tokens, in_place, pool->compact_free,
                                          [&](uint64_t q) { return pool->refcount[old[q]] == 1; })});
        }
        const CompactPlan &p = known[at].plan;
        plan_of[i] = (uint32_t)at;
        if (p.fresh > pool->compact_free && pool->compact_shared != id) {
            pool->compact_shared = id;
            pool->compact_free += given_up_together(entries, n, pool);
        }
        if (p.fresh > pool->compact_free) return fail(ctx, kNoMemory, "KV page pool exhausted");
        pool->compact_free -= p.fresh;
        ranges += p.ranges.size();
        chains += (uint32_t)(p.serial ? std::min<size_t>(p.ranges.size(), 1) : p.ranges.size());
        links += p.take.empty() ? 0 : 1;
        words += p.take.size();
        if (p.ranges.empty()) continue;
        kv_heads = std::max(kv_heads, pool->kv_heads);
        in_flight = std::min(in_flight, move_rows(pool->head_dim));
        for (const auto &r : p.ranges) longest = std::max(longest, r.end - r.begin);
    }
    const size_t fixed = (n * sizeof(MoveEntry) + ranges * sizeof(MoveRange) + links * sizeof(MoveLink)) / 4;
    words += fixed;
    for (const Lists::One &l : lists.lists) words += l.count;
    // short ranges: a workgroup takes as many heads as it has in flight at once
    uint32_t log2_heads = 0;
    while ((2u << log2_heads) <= kv_heads && (longest << (log2_heads + 1)) <= in_flight) ++log2_heads;
    const uint32_t head_groups = (kv_heads + (1u << log2_heads) - 1) >> log2_heads;
    if (words > UINT32_MAX || (uint64_t)chains + links > kMostBlocks || head_groups > kMostBlocksY / 2) {
        return fail(ctx, kOverflow, "kv_compact is too large for one call");
    }
    Words w;
    int32_t st = w.open(ctx, words, kMoveInlineWords);
    if (st != kOk) return st;

    // what the targets were, so that a call whose launch fails leaves them so
    struct Before {
        uint64_t len;
        size_t pages;  // from the first changed one on, in one of the lists below
    };
    std::vector<Before> before(n);
    std::vector<int32_t> replaced;  // of targets that are not their entry's source
    std::vector<MoveLink> late;
    std::vector<uint32_t> late_of;
    std::vector<std::pair<Pool *, int32_t>> given_up;
    std::vector<int32_t> now;
    size_t most = 0, old_pages = 0, others = 0;
    for (uint32_t i = 0; i < n; ++i) {
        const auto &e = entries[i];
        const CompactPlan &p = known[plan_of[i]].plan;
        auto &target = e.kv->seqs[e.target];
        most = std::max(most, p.take.size());
        before[i] = {target.len, target.pages.size() - p.first};
        (e.target == e.source ? old_pages : others) += before[i].pages;
        target.pages.reserve(p.first + p.take.size());
    }
    replaced.reserve(others);
    late.reserve(n);
    late_of.reserve(n);
    given_up.reserve(old_pages);
    now.reserve(most);

    // nothing fails from here on but a launch (and nothing is allocated: a pool's free
    // list has room for all its pages): the new page lists, and the words
    for (uint32_t i = 0; i < n; ++i) {
        const auto &e = entries[i];
        if (e.target == e.source) continue;
        auto &t = e.kv->seqs[e.target];
        for (int32_t page : t.pages) {
            if (--e.kv->refcount[page] == 0) e.kv->free_pages.push_back(page);
        }
        replaced.insert(replaced.end(), t.pages.begin(), t.pages.end());
        t.pages.clear();
    }
    // all of it taken back, the last step first
    auto undo = [&]() {
        auto hold = [](Pool *pool, int32_t page) {
            if (pool->refcount[page]++ == 0) pool->free_pages.pop_back();
        };
        for (size_t k = given_up.size(); k-- > 0;) hold(given_up[k].first, given_up[k].second);
        size_t in_place = given_up.size(), other = replaced.size();
        for (uint32_t i = n; i-- > 0;) {
            const auto &e = entries[i];
            const CompactPlan &p = known[plan_of[i]].plan;
            auto &t = e.kv->seqs[e.target];
            for (size_t q = p.take.size(); q-- > 0;) {
                const int32_t page = t.pages[p.first + q];
                if (--e.kv->refcount[page] == 0) e.kv->free_pages.push_back(page);
            }
            t.len = before[i].len;
            t.pages.resize(p.first);
            if (e.target == e.source) {
                in_place -= before[i].pages;
                for (size_t k = 0; k < before[i].pages; ++k) t.pages.push_back(given_up[in_place + k].second);
            } else {
                other -= before[i].pages;
                t.pages.insert(t.pages.end(), replaced.begin() + other, replaced.begin() + other + before[i].pages);
            }
        }
        for (uint32_t i = n; i-- > 0;) {
            const auto &e = entries[i];
            if (e.target == e.source) continue;
            const auto &pages = e.kv->seqs[e.target].pages;
            for (size_t q = pages.size(); q-- > 0;) hold(e.kv, pages[q]);
        }
    };
    MoveEntry *move = (MoveEntry *)w.at;
    MoveRange *head = (MoveRange *)(move + n), *tail = head + chains;
    MoveRange *const first_range = head;
    MoveLink *link = (MoveLink *)(head + ranges);
    uint32_t *list = w.at + fixed;
    MoveCall call{};
    for (uint32_t i = 0; i < n; ++i, ++move) {
        const auto &e = entries[i];
        Pool *pool = e.kv;
        const CompactPlan &p = known[plan_of[i]].plan;
        auto &source = pool->seqs[e.source], &target = pool->seqs[e.target];
        const bool in_place = e.target == e.source;
        bool changed = !in_place;
        now.clear();
        for (size_t q = 0; q < p.take.size(); ++q) {
            int32_t page;
            if (p.take[q] >= 0) {
                page = source.pages[(size_t)p.take[q]];
                ++pool->refcount[page];
                changed = changed || (uint64_t)p.take[q] != p.first + q;
            } else {
                page = pool->free_pages.back();
                pool->free_pages.pop_back();
                pool->refcount[page] = 1;
                changed = true;
            }
            now.push_back(page);
        }
        *move = MoveEntry{};
        move->k_pages = pool->k_pages;
        move->v_pages = pool->v_pages;
        move->from = pool->d_page_table + (size_t)e.source * pool->pages_per_seq;
        move->num_pages = pool->num_pages;
        move->kv_heads = pool->kv_heads;
        move->head_dim = pool->head_dim;
        move->log2_page = (uint32_t)__builtin_ctz(pool->page_tokens);
        move->start = (uint32_t)e.start;
        move->first_page = (uint32_t)p.first;
        move->pages = (uint32_t)(list - w.at);
        if (!now.empty()) std::memcpy(list, now.data(), now.size() * 4);
        list += now.size();
        if (!p.ranges.empty() && e.count > 0) {
            Lists::One &l = lists.lists[list_of[i]];
            if (l.offset == 0) {
                l.offset = (uint32_t)(list - w.at);
                std::memcpy(list, e.tokens, e.count * 4);
                list += e.count;
            }
            move->tokens = l.offset;
        }
        if (changed && !now.empty()) {
            const MoveLink l{pool->d_page_table + (size_t)e.target * pool->pages_per_seq + p.first,
                             move->pages, (uint32_t)now.size()};
            if (in_place) late.push_back(l), late_of.push_back(i);
            else *link++ = l, ++call.links;
        }
        MoveRange *last = nullptr;
        for (size_t r = 0; r < p.ranges.size(); ++r) {
            MoveRange *to = p.serial && r > 0 ? tail++ : head++;
            *to = MoveRange{i, (uint32_t)p.ranges[r].begin, (uint32_t)p.ranges[r].end, 0};
            if (p.serial && last != nullptr) last->next = (uint32_t)(to - first_range);
            last = to;
        }
        // the old pages from the first changed one on are given up, but not to this
        // call's other entries: its ranges read them
        if (in_place) {
            for (size_t q = p.first; q < source.pages.size(); ++q) given_up.emplace_back(pool, source.pages[q]);
            source.pages.resize(p.first);
        }
        target.pages.insert(target.pages.end(), now.begin(), now.end());
        target.len = e.start + e.count;
    }
    for (const MoveLink &l : late) *link++ = l;
    for (const auto &[pool, page] : given_up) {
        if (--pool->refcount[page] == 0) pool->free_pages.push_back(page);
    }
    call.entries = n;
    call.chains = chains;
    call.ranges = (uint32_t)ranges;
    call.late_links = (uint32_t)late.size();
    call.log2_heads = log2_heads;
    call.head_groups = head_groups;
    call.host_words = w.at;
    call.words = (uint32_t)(list - w.at);
    if (call.chains + call.links + call.late_links > 0) {
        st = w.send(ctx, call.words, &call.device_words);
        if (st == kOk) {
            const hipError_t e = launch_kv_moves(ctx->stream, call);
            if (e != hipSuccess) st = hip_fail(ctx, e, "kv_compact launch");
        }
        if (st != kOk) {
            undo();
            return st;
        }
        const hipError_t e = launch_kv_links(ctx->stream, call);
        if (e != hipSuccess) {
            // the tokens have moved: the rows of the page tables follow by another launch
            st = hip_fail(ctx, e, "kv_compact page tables");
            const std::string saved = ctx->error;
            for (uint32_t i : late_of) {
                Pool *pool = entries[i].kv;
                TableBatch batch;
                for (size_t q = known[plan_of[i]].plan.first; q < pool->seqs[entries[i].target].pages.size(); ++q) {
                    batch.idx.push_back((uint32_t)(entries[i].target * pool->pages_per_seq + q));
                    batch.val.push_back(pool->seqs[entries[i].target].pages[q]);
                }
                (void)kv_flush_table(ctx, pool, batch);
            }
            ctx->error = saved;
            return st;
        }
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
    Lists lists;
    std::vector<uint32_t> list_of(n);
    for (uint32_t i = 0; i < n; ++i) {
        const auto &e = entries[i];
        if (e.kv == nullptr || !is_open(e.kv, e.sequence) || e.reserved != 0) {
            return fail(ctx, kInvalid, "KV sequence handle is not open");
        }
        if (e.kv->kv_heads != entries[0].kv->kv_heads || e.kv->head_dim != entries[0].kv->head_dim) {
            return fail(ctx, kInvalid, "kv_gather pools differ in kv_heads or head_dim");
        }
        if (e.count > INT32_MAX) return fail(ctx, kOverflow, "too many tokens");
        const uint64_t len = e.kv->seqs[e.sequence].len;
        bool inside = e.start <= len && (e.tokens != nullptr || e.count <= len - e.start);
        if (inside && e.tokens != nullptr && e.count > 0) {
            list_of[i] = lists.add(e.tokens, e.count);
            inside = lists.below(list_of[i], len - e.start);
        }
        if (!inside) return fail(ctx, kInvalid, "KV token index out of range");
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
    call.bf16_out = out16;
    uint64_t bytes = 0;
    if (!checked_mul(total, (uint64_t)call.kv_heads * call.head_dim * (out16 ? 2 : 4), &bytes)) {
        return fail(ctx, kOverflow, "kv_gather size overflows");
    }
    // tokens of a workgroup: about 1024 of its threads' units
    const uint64_t per = (uint64_t)call.kv_heads * (call.head_dim % 8 == 0 ? call.head_dim / 8 : call.head_dim);
    call.block_tokens = (uint32_t)std::max<uint64_t>(1, 1024 / per);
    uint64_t blocks = 0;
    for (uint32_t i = 0; i < n; ++i) {
        call.entries += entries[i].count > 0;
        blocks += (entries[i].count + call.block_tokens - 1) / call.block_tokens;
    }
    uint64_t words = (call.entries * sizeof(GatherEntry) + blocks * sizeof(GatherBlock)) / 4;
    for (const Lists::One &l : lists.lists) words += l.count;
    if (words > UINT32_MAX || blocks > kMostBlocks) return fail(ctx, kOverflow, "kv_gather is too large for one call");
    Words w;
    int32_t st = w.open(ctx, words, kGatherInlineWords);
    if (st != kOk) return st;
    GatherEntry *g = (GatherEntry *)w.at;
    GatherBlock *block = (GatherBlock *)(g + call.entries);
    uint32_t *list = (uint32_t *)(block + blocks);
    uint64_t first = 0;
    for (uint32_t i = 0, k = 0; i < n; ++i) {
        const auto &e = entries[i];
        if (e.count == 0) continue;
        *g = GatherEntry{};
        g->k_pages = e.kv->k_pages;
        g->v_pages = e.kv->v_pages;
        g->from = e.kv->d_page_table + (size_t)e.sequence * e.kv->pages_per_seq;
        g->num_pages = (uint32_t)e.kv->num_pages;
        g->first = first;
        g->log2_page = (uint32_t)__builtin_ctz(e.kv->page_tokens);
        g->start = (uint32_t)e.start;
        g->count = (uint32_t)e.count;
        if (e.tokens != nullptr) {
            Lists::One &l = lists.lists[list_of[i]];
            if (l.offset == 0) {
                l.offset = (uint32_t)(list - w.at);
                std::memcpy(list, e.tokens, e.count * 4);
                list += e.count;
            }
            g->tokens = l.offset;
        }
        for (uint64_t t = 0; t < e.count; t += call.block_tokens) *block++ = GatherBlock{k, (uint32_t)t};
        first += e.count;
        ++g;
        ++k;
    }
    call.blocks = (uint32_t)blocks;
    call.host_words = w.at;
    call.words = (uint32_t)(list - w.at);
    st = w.send(ctx, call.words, &call.device_words);
    if (st != kOk) return st;
    call.keys = keys;
    call.values = values;
    const size_t half = (bytes + 255) & ~(size_t)255;
    if (!device) {
        st = ensure_buffer(ctx, ctx->staging, 2 * half, false);
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
