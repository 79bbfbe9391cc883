// How kv_compact lays the kept tokens out over pages.  Host code only, so that
// it is tested without a GPU.
#pragma once

#include <algorithm>
#include <cstdint>
#include <vector>

namespace sr {

// Moves of at most this many tokens are made where the pages are, by one
// workgroup per head in the tokens' order; longer ones go to free pages, every
// page at once, as far as the pool has them.  Without enough free pages a long move
// is made in order too, however long: 4872 and 7976 kept tokens of two sequences take
// 224 us at 8 heads of width 128 (29 to free pages), 408 us at 2 heads of 256.
constexpr uint64_t kCompactSerial = 256;

// Tokens that one workgroup copies where ranges run at once.
constexpr uint64_t kCompactRange = 64;

// One sequence's kept tokens: new token t is old token from(t).
struct KeepList {
    uint64_t start, count;
    const uint32_t *tokens;
    uint64_t from(uint64_t t) const { return t < start ? t : start + tokens[t - start]; }
    uint64_t length() const { return start + count; }
};

struct CompactPlan {
    // per page of the new sequence: an old page's index that it takes over, or
    // -1 for a free page, which the copy fills; pages before `first` stay
    uint64_t first = 0;
    std::vector<int64_t> take;  // pages first, first + 1, ...
    uint64_t fresh = 0;         // free pages needed
    uint64_t wanted = 0;        // free pages with which the plan would be the same
    // token ranges to copy; the ranges of a serial plan run in order in one
    // workgroup per head, others at once
    struct Range {
        uint64_t begin, end;
    };
    std::vector<Range> ranges;
    bool serial = false;
};

// Whether new page q holds exactly the tokens that old page *page holds from its
// begin on.
inline bool page_stays_whole(const KeepList &k, uint64_t page_tokens, uint64_t q, uint64_t *page) {
    const uint64_t begin = q * page_tokens, end = std::min(begin + page_tokens, k.length());
    const uint64_t src = k.from(begin);
    if (src % page_tokens != 0 || k.from(end - 1) - src != end - 1 - begin) return false;
    *page = src / page_tokens;
    return true;
}

// `writable`(page index of the old sequence): no other sequence holds it.
// into_source: the old sequence itself becomes the new one; otherwise its pages
// are only linked.  `free`: free pages of the pool.
//
// In place, a token moves to a position at or before its own.  Old page q is
// written by new page q alone, and read by new pages up to q: done in order,
// nothing is overwritten before it is read, and the first page that changes
// is read by its own tokens only.
template <class Writable>
CompactPlan compact_plan(const KeepList &k, uint64_t page_tokens, bool into_source, uint64_t free,
                         Writable writable) {
    CompactPlan plan;
    const uint64_t len = k.length(), pages = (len + page_tokens - 1) / page_tokens;
    uint64_t same = 0;  // kept tokens that stay where they are
    if (into_source) {
        while (same < k.count && k.tokens[same] == same) ++same;
        plan.first = same == k.count ? pages : (k.start + same) / page_tokens;
    }
    const uint64_t moved = k.start + same;  // the first token whose place changes
    std::vector<uint64_t> copied;           // new pages that are filled
    std::vector<uint8_t> taken;             // old pages that a new page takes over
    plan.take.assign(pages - plan.first, -1);
    for (uint64_t q = plan.first; q < pages; ++q) {
        uint64_t page = 0;
        if (page_stays_whole(k, page_tokens, q, &page)) {
            plan.take[q - plan.first] = (int64_t)page;
            if (taken.size() <= page) taken.resize(page + 1, 0);
            taken[page] = 1;
        } else {
            copied.push_back(q);
        }
    }
    auto in_place = [&](uint64_t q) { return into_source && writable(q) && !(q < taken.size() && taken[q]); };
    auto end_of = [&](uint64_t q) { return std::min((q + 1) * page_tokens, len); };
    // the first page in place where it can be, the others on free pages
    uint64_t fresh = 0, tokens = 0;
    for (uint64_t i = 0; i < copied.size(); ++i) {
        const bool stay = i == 0 && copied[i] == plan.first && in_place(copied[i]);
        fresh += stay ? 0 : 1;
        tokens += end_of(copied[i]) - copied[i] * page_tokens;
    }
    uint64_t least = 0;
    for (uint64_t q : copied) least += in_place(q) ? 0 : 1;
    plan.wanted = fresh;
    plan.serial = into_source && least < fresh && (tokens <= kCompactSerial || fresh > free);
    bool first_stays = false;
    for (uint64_t i = 0; i < copied.size(); ++i) {
        const uint64_t q = copied[i];
        const bool stay = in_place(q) && (plan.serial || (i == 0 && q == plan.first));
        if (stay) plan.take[q - plan.first] = (int64_t)q;
        else ++plan.fresh;
        // (tokens before the first moved one are in place already)
        const uint64_t begin = stay ? std::max(q * page_tokens, moved) : q * page_tokens;
        if (begin >= end_of(q)) continue;
        // pages in a row make one range: all of a serial plan's, else up to kCompactRange
        // tokens, but for the page that is filled where it is
        if (i > 0 && !plan.ranges.empty() && plan.ranges.back().end == begin &&
            (plan.serial || (end_of(q) - plan.ranges.back().begin <= kCompactRange && !first_stays))) {
            plan.ranges.back().end = end_of(q);
        } else {
            plan.ranges.push_back({begin, end_of(q)});
        }
        first_stays = stay && !plan.serial;
    }
    return plan;
}

}  // namespace sr
