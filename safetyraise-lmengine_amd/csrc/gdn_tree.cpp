// gdn_tree_forward, gdn_tree_commit and gdn_view on the state pools of gdn.cpp.
//
// A tree call reads a sequence's current state and history and leaves both; what
// it adds is a record per row, and the tree's parents on the host.  A commit
// builds the state of one path into the sequence's other buffers and makes those
// current, so the ones before the tree stay, to commit again from.

#include <algorithm>
#include <cmath>
#include <cstring>
#include <vector>

#include "sr_internal.hpp"
#include "tree_plan.hpp"

namespace sr {

namespace {

using Pool = safetyraise_kernel_gdn_pool;

size_t align_up(size_t x) { return (x + 255) & ~(size_t)255; }

bool is_open(const Pool *pool, uint32_t seq) { return seq < pool->max_sequences && pool->open[seq]; }

float *state_at(const Pool *pool, uint32_t seq, uint32_t par) {
    return pool->d_state + (size_t)(seq * pool->state_buffers() + (pool->keep_rows > 0 ? par : 0)) * pool->state_elems();
}
float *history_at(const Pool *pool, uint32_t seq, uint32_t par) {
    return pool->d_history + ((size_t)par * pool->max_sequences + seq) * pool->history_elems();
}

int32_t tree_forward(Ctx *ctx, const safetyraise_kernel_gdn_tree_args *args) {
    if (args == nullptr || args->struct_size < sizeof(safetyraise_kernel_gdn_tree_args) ||
        args->gdn.struct_size < sizeof(safetyraise_kernel_gdn_args) || args->reserved != 0) {
        return fail(ctx, kInvalid, "gdn tree args pointer or struct_size is invalid");
    }
    const auto &A = args->gdn;
    Pool *pool = A.state;
    const bool device = (A.flags & SAFETYRAISE_MI355X_DEVICE_POINTERS) != 0;
    const bool async = (A.flags & SAFETYRAISE_MI355X_ASYNC) != 0;
    const bool bf16 = (A.flags & SAFETYRAISE_MI355X_INPUT_BF16) != 0;
    if (pool == nullptr) return fail(ctx, kInvalid, "gdn_tree_forward needs a state pool");
    if (async && !device) return fail(ctx, kInvalid, "ASYNC needs DEVICE_POINTERS");
    if ((A.flags & SAFETYRAISE_MI355X_OUTPUT_BF16) != 0) {
        return fail(ctx, kInvalid, "gdn_tree_forward writes f32: it takes no OUTPUT_BF16");
    }
    if ((A.flags & SAFETYRAISE_MI355X_KEEP_ROWS) != 0) {
        return fail(ctx, kInvalid, "gdn_tree_forward takes no KEEP_ROWS: it records every row");
    }
    if (!std::isfinite(A.eps) || A.eps <= 0.0f) {
        return fail(ctx, kInvalid, "RMSNorm shape or epsilon is invalid");
    }
    if (A.num_seqs == 0 || A.num_seqs > SAFETYRAISE_MI355X_MAX_BATCH || A.seq_ids == nullptr ||
        A.seq_rows == nullptr || args->parents == nullptr) {
        return fail(ctx, kInvalid, "GDN batch is empty or too large");
    }
    if (A.qkv == nullptr || A.z == nullptr || A.a == nullptr || A.b == nullptr ||
        A.a_log == nullptr || A.dt_bias == nullptr || A.conv_weight == nullptr ||
        A.norm == nullptr || A.out == nullptr) {
        return fail(ctx, kInvalid, "GDN input or output pointer is NULL");
    }
    std::vector<GdnSeq> seqs(A.num_seqs);
    uint64_t total = 0;
    for (uint32_t i = 0; i < A.num_seqs; ++i) {
        const uint32_t id = A.seq_ids[i], rows = A.seq_rows[i];
        if (!is_open(pool, id)) return fail(ctx, kInvalid, "GDN sequence handle is not open");
        if (rows == 0) return fail(ctx, kInvalid, "input is empty");
        if (rows > kMaxGdnTreeRows || rows > pool->keep_rows) {
            return fail(ctx, kInvalid, "a tree has more rows than the pool's keep_rows");
        }
        if (!tree_valid(args->parents + total, rows)) {
            return fail(ctx, kInvalid, "a tree row's parent must be an earlier row of its sequence, or -1");
        }
        seqs[i] = GdnSeq{id, rows, (uint32_t)total, pool->parity[id], pool->state_index(id, 0),
                         pool->state_index(id, 0)};
        total += rows;
    }
    std::vector<uint32_t> ids(A.seq_ids, A.seq_ids + A.num_seqs);
    std::sort(ids.begin(), ids.end());
    if (std::adjacent_find(ids.begin(), ids.end()) != ids.end()) {
        return fail(ctx, kInvalid, "a sequence appears twice in one call");
    }
    if (total > INT32_MAX / std::max<uint32_t>(pool->channels, 1)) {
        return fail(ctx, kOverflow, "too many rows");
    }
    if (!async) {
        const int32_t st = report_pending_async(ctx);
        if (st != kOk) return st;
    }
    GdnLaunch g{};
    g.pool = pool;
    g.err_word = ctx->d_error_word;
    g.eps = A.eps;
    g.bf16_in = bf16;
    g.qkv = A.qkv;
    g.z = A.z;
    g.a = A.a;
    g.b = A.b;
    g.a_log = A.a_log;
    g.dt_bias = A.dt_bias;
    g.conv_w = A.conv_weight;
    g.norm = A.norm;
    g.out = A.out;
    g.records = pool->d_records;
    g.rec_stride = (uint32_t)pool->record_elems();
    g.keep_rows = pool->keep_rows;
    g.num_cus = ctx->num_cus;
    const size_t esz = bf16 ? 2 : 4;
    const size_t width = (size_t)pool->value_heads * pool->value_dim;
    const size_t out_b = total * width * 4;
    const struct {
        const void *host;
        size_t bytes;
    } regions[8] = {{A.qkv, total * pool->channels * esz}, {A.z, total * width * esz},
                    {A.a, total * pool->value_heads * esz}, {A.b, total * pool->value_heads * esz},
                    {A.a_log, (size_t)pool->value_heads * 4}, {A.dt_bias, (size_t)pool->value_heads * 4},
                    {A.conv_weight, (size_t)pool->channels * pool->conv_kernel * 4},
                    {A.norm, (size_t)pool->value_dim * 4}};
    // launches of at most kGdnTreeSeqs sequences share the scratch
    size_t scratch = 0;
    for (uint32_t i = 0; i < A.num_seqs; i += kGdnTreeSeqs) {
        uint32_t rows = 0;
        for (uint32_t j = i; j < std::min<uint32_t>(i + kGdnTreeSeqs, A.num_seqs); ++j) rows += seqs[j].rows;
        scratch = std::max(scratch, align_up(gdn_tree_scratch_bytes(pool, rows)));
    }
    size_t need = scratch;
    if (!device) {
        for (const auto &r : regions) need += align_up(r.bytes);
        need += align_up(out_b);
    }
    int32_t st = ensure_buffer(ctx, ctx->staging, need, false);
    if (st != kOk) return st;
    char *at = (char *)ctx->staging.ptr + scratch;
    if (!device) {
        const void *dev[8];
        for (int i = 0; i < 8; ++i) {
            SR_HIP(ctx, hipMemcpyAsync(at, regions[i].host, regions[i].bytes, hipMemcpyHostToDevice,
                                       ctx->stream));
            dev[i] = at;
            at += align_up(regions[i].bytes);
        }
        g.qkv = dev[0];
        g.z = dev[1];
        g.a = dev[2];
        g.b = dev[3];
        g.a_log = (const float *)dev[4];
        g.dt_bias = (const float *)dev[5];
        g.conv_w = (const float *)dev[6];
        g.norm = (const float *)dev[7];
        g.out = (float *)at;
    }
    std::vector<uint8_t> parents(total);
    for (uint64_t r = 0; r < total; ++r) parents[r] = (uint8_t)(args->parents[r] + 1);
    std::vector<std::vector<int32_t>> kept(A.num_seqs);
    for (uint32_t i = 0; i < A.num_seqs; ++i) {
        kept[i].assign(args->parents + seqs[i].row0, args->parents + seqs[i].row0 + seqs[i].rows);
    }
    // from the first launch on, the records are no earlier call's
    for (const GdnSeq &q : seqs) {
        pool->kept[q.slot] = Pool::kNoKept;
        pool->trees[q.slot].parents.clear();
    }
    for (uint32_t i = 0; i < A.num_seqs; i += kGdnTreeSeqs) {
        const int n = (int)std::min<uint32_t>(kGdnTreeSeqs, A.num_seqs - i);
        SR_HIP(ctx, launch_gdn_tree(ctx->stream, g, &seqs[i], n, parents.data() + seqs[i].row0,
                                    (float *)ctx->staging.ptr));
    }
    for (uint32_t i = 0; i < A.num_seqs; ++i) {
        const uint32_t id = seqs[i].slot;
        Pool::Tree &t = pool->trees[id];
        t.parents = std::move(kept[i]);
        t.state_par = pool->state_par[id];
        t.parity = pool->parity[id];
    }
    if (!device) {
        SR_HIP(ctx, hipMemcpyAsync(A.out, g.out, out_b, hipMemcpyDeviceToHost, ctx->stream));
    }
    st = finish_call(ctx, async);
    if (st != kOk && !async) {
        for (const GdnSeq &q : seqs) pool->trees[q.slot].parents.clear();
    }
    return st;
}

int32_t commit(Ctx *ctx, const safetyraise_kernel_gdn_commit *commits, uint32_t n, uint32_t flags) {
    if (commits == nullptr || n == 0 || (flags & ~SAFETYRAISE_MI355X_ASYNC) != 0) {
        return fail(ctx, kInvalid, "gdn_tree_commit needs commits, and no flag but ASYNC");
    }
    const bool async = (flags & SAFETYRAISE_MI355X_ASYNC) != 0;
    std::vector<std::pair<Pool *, uint32_t>> who(n);
    for (uint32_t i = 0; i < n; ++i) {
        const auto &c = commits[i];
        if (c.state == nullptr || !is_open(c.state, c.sequence)) {
            return fail(ctx, kInvalid, "GDN sequence handle is not open");
        }
        const auto &t = c.state->trees[c.sequence];
        if (t.parents.empty()) {
            return fail(ctx, kInvalid, "gdn_tree_commit: the sequence's last call was not a tree call");
        }
        if (c.row < -1 || c.row >= (int32_t)t.parents.size()) {
            return fail(ctx, kInvalid, "gdn_tree_commit: the tree has no such row");
        }
        who[i] = {c.state, c.sequence};
    }
    std::sort(who.begin(), who.end());
    if (std::adjacent_find(who.begin(), who.end()) != who.end()) {
        return fail(ctx, kInvalid, "a sequence appears twice in one call");
    }
    if (!async) {
        const int32_t st = report_pending_async(ctx);
        if (st != kOk) return st;
    }
    std::vector<GdnCommitEntry> entries;
    for (uint32_t i = 0; i < n; ++i) {
        const auto &c = commits[i];
        if (c.row < 0) continue;
        const Pool *pool = c.state;
        const Pool::Tree &t = pool->trees[c.sequence];
        GdnCommitEntry e{};
        e.state_in = state_at(pool, c.sequence, t.state_par);
        e.state_out = state_at(pool, c.sequence, t.state_par ^ 1);
        e.hist_in = history_at(pool, c.sequence, t.parity);
        e.hist_out = history_at(pool, c.sequence, t.parity ^ 1);
        e.records = pool->d_records + (size_t)c.sequence * pool->keep_rows * pool->record_elems();
        e.path = tree_path(t.parents.data(), c.row);
        e.rec_stride = (uint32_t)pool->record_elems();
        e.value_heads = pool->value_heads;
        e.key_heads = pool->key_heads;
        e.key_dim = pool->key_dim;
        e.value_dim = pool->value_dim;
        e.channels = pool->channels;
        e.conv_k = pool->conv_kernel;
        entries.push_back(e);
    }
    const uint32_t *device = nullptr;
    constexpr size_t kMost = 32768;  // the launch grid's second dimension
    for (size_t i = 0; i < entries.size(); i += kMost) {
        const size_t count = std::min(kMost, entries.size() - i);
        if (count > kGdnCommitInline) {
            const size_t words = count * sizeof(GdnCommitEntry) / 4;
            uint32_t *host = nullptr;
            int32_t st = upload_room(ctx, words, &host);
            if (st != kOk) return st;
            std::memcpy(host, &entries[i], words * 4);
            st = upload_words(ctx, words, &device);
            if (st != kOk) return st;
        } else {
            device = nullptr;
        }
        SR_HIP(ctx, launch_gdn_tree_commit(ctx->stream, &entries[i], (uint32_t)count,
                                           (const GdnCommitEntry *)device));
    }
    for (uint32_t i = 0; i < n; ++i) {
        const auto &c = commits[i];
        const Pool::Tree &t = c.state->trees[c.sequence];
        const uint32_t flip = c.row < 0 ? 0 : 1;
        c.state->state_par[c.sequence] = t.state_par ^ flip;
        c.state->parity[c.sequence] = t.parity ^ flip;
    }
    return finish_call(ctx, async);
}

}  // namespace

}  // namespace sr

using namespace sr;

extern "C" {

SAFETYRAISE_KERNEL_EXPORT int32_t safetyraise_kernel_gdn_tree_forward(
    safetyraise_kernel_context *context, const safetyraise_kernel_gdn_tree_args *args) {
    if (context == nullptr) return kInvalid;
    const int32_t capture = refuse_under_capture(context, "gdn_tree_forward");
    if (capture != kOk) return capture;
    DeviceScope device_scope(context);
    TimerScope timer_scope(context);
    return no_throw(context, [&] { return tree_forward(context, args); });
}

SAFETYRAISE_KERNEL_EXPORT int32_t safetyraise_kernel_gdn_tree_commit(
    safetyraise_kernel_context *context, const safetyraise_kernel_gdn_commit *commits,
    uint32_t num_commits, uint32_t flags) {
    if (context == nullptr) return kInvalid;
    const int32_t capture = refuse_under_capture(context, "gdn_tree_commit");
    if (capture != kOk) return capture;
    DeviceScope device_scope(context);
    TimerScope timer_scope(context);
    return no_throw(context, [&] { return commit(context, commits, num_commits, flags); });
}

SAFETYRAISE_KERNEL_EXPORT int32_t safetyraise_kernel_gdn_view(
    safetyraise_kernel_context *context, safetyraise_kernel_gdn_pool *pool, uint32_t sequence,
    const float **out_matrix, const float **out_history) {
    if (context == nullptr) return kInvalid;
    const int32_t capture = refuse_under_capture(context, "gdn_view");
    if (capture != kOk) return capture;
    if (pool == nullptr || out_matrix == nullptr || out_history == nullptr) {
        return fail(context, kInvalid, "NULL argument");
    }
    if (!is_open(pool, sequence)) return fail(context, kInvalid, "GDN sequence handle is not open");
    *out_matrix = state_at(pool, sequence, pool->state_par[sequence]);
    *out_history = history_at(pool, sequence, pool->parity[sequence]);
    return kOk;
}

}  // extern "C"
