// safetyraise_kernel_attention_tree_forward: attention of a tree of drafted
// tokens on the paged bf16 KV cache of kv.cpp.  The argument checks are those of
// attention_forward (attention.cpp), with the tree's shape.

#include <algorithm>
#include <cmath>
#include <cstring>
#include <vector>

#include "sr_internal.hpp"
#include "tree_plan.hpp"

namespace sr {

namespace {

size_t align_up(size_t x) { return (x + 255) & ~(size_t)255; }

// Page-table entries of a call that fails before its kernels have written them:
// the host's page lists already hold them (see attention.cpp).
struct TableGuard {
    Ctx *ctx;
    safetyraise_kernel_kv_pool *pool;
    TableBatch &batch;
    bool armed = true;
    ~TableGuard() {
        if (!armed || batch.idx.empty()) return;
        const std::string saved = ctx->error;
        (void)kv_flush_table(ctx, pool, batch);
        ctx->error = saved;
    }
};

int32_t tree_forward(Ctx *ctx, const safetyraise_kernel_attention_tree_args *args) {
    if (args == nullptr || args->struct_size < sizeof(safetyraise_kernel_attention_tree_args) ||
        args->attention.struct_size < sizeof(safetyraise_kernel_attention_args) ||
        args->reserved != 0) {
        return fail(ctx, kInvalid, "attention tree args pointer or struct_size is invalid");
    }
    const auto &A = args->attention;
    auto *pool = A.kv;
    const bool device = (A.flags & SAFETYRAISE_MI355X_DEVICE_POINTERS) != 0;
    const bool async = (A.flags & SAFETYRAISE_MI355X_ASYNC) != 0;
    const bool bf16 = (A.flags & SAFETYRAISE_MI355X_INPUT_BF16) != 0;
    const bool out16 = (A.flags & SAFETYRAISE_MI355X_OUTPUT_BF16) != 0;
    const bool gated = (A.flags & SAFETYRAISE_MI355X_GATED) != 0;
    const bool qk_norm = (A.flags & SAFETYRAISE_MI355X_QK_NORM) != 0;
    if (pool == nullptr) return fail(ctx, kInvalid, "attention needs a KV pool");
    if (async && !device) return fail(ctx, kInvalid, "ASYNC needs DEVICE_POINTERS");
    if (A.heads == 0 || A.kv_heads == 0 || A.head_dim == 0 || A.heads % A.kv_heads != 0 ||
        A.kv_heads != pool->kv_heads || A.head_dim != pool->head_dim) {
        return fail(ctx, kInvalid, "attention head mapping or cache geometry is invalid");
    }
    if (A.rotary_dim == 0 || A.rotary_dim > A.head_dim || A.rotary_dim % 2 != 0) {
        return fail(ctx, kInvalid, "RoPE input shape is invalid");
    }
    if (!(A.rope_theta > 0.0f) || !std::isfinite(A.rope_theta)) {
        return fail(ctx, kInvalid, "RoPE theta must be finite and positive");
    }
    if (qk_norm && (!std::isfinite(A.eps) || A.eps <= 0.0f)) {
        return fail(ctx, kInvalid, "RMSNorm shape or epsilon is invalid");
    }
    if (A.num_seqs == 0 || A.num_seqs > SAFETYRAISE_MI355X_MAX_BATCH || A.seq_ids == nullptr ||
        A.seq_rows == nullptr || args->parents == nullptr) {
        return fail(ctx, kInvalid, "attention batch is empty or too large");
    }
    if (A.q == nullptr || A.k == nullptr || A.v == nullptr || A.positions == nullptr ||
        A.out == nullptr || (qk_norm && (A.q_norm == nullptr || A.k_norm == nullptr))) {
        return fail(ctx, kInvalid, "attention input or output pointer is NULL");
    }
    uint64_t total = 0;
    std::vector<SeqMeta> seqs(A.num_seqs);
    for (uint32_t i = 0; i < A.num_seqs; ++i) {
        const uint32_t id = A.seq_ids[i], rows = A.seq_rows[i];
        if (id >= pool->max_sequences || !pool->seqs[id].open) {
            return fail(ctx, kInvalid, "KV sequence handle is not open");
        }
        if (rows == 0) return fail(ctx, kInvalid, "input is empty");
        if (rows > kMaxTreeRows) {
            return fail(ctx, kInvalid, "a tree has more than MAX_TREE_ROWS (128) rows");
        }
        if (pool->seqs[id].len + rows > pool->max_tokens) {
            return fail(ctx, kInvalid, "KV write would exceed the sequence capacity");
        }
        if (!tree_valid(args->parents + total, rows)) {
            return fail(ctx, kInvalid, "a tree row's parent must be an earlier row of its sequence, or -1");
        }
        seqs[i] = SeqMeta{id, (uint32_t)pool->seqs[id].len, rows, (uint32_t)total, 0};
        total += rows;
    }
    std::vector<uint32_t> ids(A.seq_ids, A.seq_ids + A.num_seqs);
    std::sort(ids.begin(), ids.end());
    if (std::adjacent_find(ids.begin(), ids.end()) != ids.end()) {
        return fail(ctx, kInvalid, "a sequence appears twice in one call");
    }
    if (device && (((uintptr_t)A.q | (uintptr_t)A.k | (uintptr_t)A.v | (uintptr_t)A.out) & 15u)) {
        return fail(ctx, kInvalid, "device pointers must be 16-byte aligned");
    }
    if (!async) {
        const int32_t st = report_pending_async(ctx);
        if (st != kOk) return st;
    }

    TreeLaunch L{};
    L.pool = pool;
    L.flags = A.flags;
    L.heads = A.heads;
    L.kv_heads = A.kv_heads;
    L.head_dim = A.head_dim;
    L.rotary_dim = A.rotary_dim;
    L.eps = A.eps;
    std::memcpy(L.mrope, A.mrope_section, sizeof L.mrope);
    L.err_word = ctx->d_error_word;
    std::vector<float> denom;
    if (A.rotary_dim <= 256) {
        L.rope_denom = rope_table(ctx, A.rope_theta, A.rotary_dim).denom;
    } else {
        denom.resize(A.rotary_dim / 2);
        for (uint32_t i = 0; i < A.rotary_dim / 2; ++i) {
            denom[i] = rope_denominator(A.rope_theta, i, A.rotary_dim);
        }
        L.rope_denom = denom.data();
    }
    L.q = A.q;
    L.k = A.k;
    L.v = A.v;
    L.q_norm = A.q_norm;
    L.k_norm = A.k_norm;
    L.positions = A.positions;
    L.out = A.out;
    const size_t esz = bf16 ? 2 : 4;
    const size_t q_bytes = total * A.heads * A.head_dim * (gated ? 2 : 1) * esz;
    const size_t kv_bytes = total * A.kv_heads * A.head_dim * esz;
    const size_t norm_bytes = qk_norm ? (size_t)A.head_dim * sizeof(float) : 0;
    const size_t out_bytes = total * A.heads * A.head_dim * (out16 ? 2 : 4);
    if (!device) {
        struct {
            const void *host;
            size_t bytes;
        } regions[6] = {{A.q, q_bytes}, {A.k, kv_bytes}, {A.v, kv_bytes},
                        {A.positions, total * 3 * sizeof(int32_t)},
                        {A.q_norm, norm_bytes}, {A.k_norm, norm_bytes}};
        size_t need = align_up(out_bytes);
        for (const auto &r : regions) need += align_up(r.bytes);
        int32_t st = ensure_buffer(ctx, ctx->staging, need, false);
        if (st != kOk) return st;
        char *at = (char *)ctx->staging.ptr;
        L.out = at;
        at += align_up(out_bytes);
        const void *dev[6] = {};
        for (int i = 0; i < 6; ++i) {
            if (regions[i].bytes == 0) continue;
            SR_HIP(ctx, hipMemcpyAsync(at, regions[i].host, regions[i].bytes, hipMemcpyHostToDevice,
                                       ctx->stream));
            dev[i] = at;
            at += align_up(regions[i].bytes);
        }
        L.q = dev[0];
        L.k = dev[1];
        L.v = dev[2];
        L.positions = (const int32_t *)dev[3];
        L.q_norm = (const float *)dev[4];
        L.k_norm = (const float *)dev[5];
    }

    // launches of at most kTreeLaunchSeqs sequences and kTreeLaunchRows rows, which
    // share the scratch one after another
    struct Pack {
        uint32_t first, count;
        TreePlan plan;
    };
    std::vector<Pack> packs;
    uint32_t pack_rows = 0;
    for (uint32_t i = 0; i < A.num_seqs; ++i) {
        if (packs.empty() || packs.back().count == kTreeLaunchSeqs ||
            pack_rows + seqs[i].rows > kTreeLaunchRows) {
            packs.push_back({i, 0, {}});
            pack_rows = 0;
        }
        ++packs.back().count;
        pack_rows += seqs[i].rows;
    }
    TreeScratch most;
    for (Pack &p : packs) {
        const TreeScratch t = tree_scratch(L, &seqs[p.first], (int)p.count, total, ctx->num_cus);
        p.plan = t.plan;
        most.q_bytes = std::max(most.q_bytes, t.q_bytes);
        most.mask_bytes = std::max(most.mask_bytes, t.mask_bytes);
        most.record_bytes = std::max(most.record_bytes, t.record_bytes);
    }
    int32_t st = ensure_buffer(ctx, ctx->tree, align_up(most.mask_bytes) + most.q_bytes, false);
    if (st == kOk && most.record_bytes > 0) st = ensure_buffer(ctx, ctx->partials, most.record_bytes, false);
    if (st != kOk) return st;
    L.masks = ctx->tree.ptr;
    L.q_ops = (char *)ctx->tree.ptr + align_up(most.mask_bytes);
    L.records = (float *)ctx->partials.ptr;

    TableBatch batch;
    for (uint32_t i = 0; i < A.num_seqs; ++i) {
        st = kv_prepare_append(ctx, pool, seqs[i].slot, seqs[i].rows, &batch);
        if (st != kOk) {
            kv_flush_table(ctx, pool, batch);
            return st;
        }
    }
    TableGuard guard{ctx, pool, batch};
    // few page-table entries travel in the first launch's arguments; its own rows'
    // entries are among them, and later launches follow it
    if (batch.idx.size() <= kInlineTable) {
        L.tbl_idx = batch.idx.data();
        L.tbl_val = batch.val.data();
        L.tbl_n = (uint32_t)batch.idx.size();
    } else {
        st = kv_flush_table(ctx, pool, batch);
        if (st != kOk) return st;
    }
    std::vector<uint8_t> parents(kTreeLaunchRows);
    for (const Pack &p : packs) {
        uint32_t n = 0;
        for (uint32_t i = p.first; i < p.first + p.count; ++i) {
            for (uint32_t r = 0; r < seqs[i].rows; ++r) {
                parents[n++] = (uint8_t)(args->parents[seqs[i].row0 + r] + 1);
            }
        }
        const hipError_t e = launch_tree_attn(ctx->stream, L, &seqs[p.first], (int)p.count,
                                              parents.data(), p.plan);
        if (e != hipSuccess) return hip_fail(ctx, e, "tree attention launch");
        L.tbl_n = 0;
    }
    guard.armed = false;
    for (const SeqMeta &m : seqs) pool->seqs[m.slot].len = (uint64_t)m.ctx + m.rows;
    if (!device) {
        SR_HIP(ctx, hipMemcpyAsync(A.out, L.out, out_bytes, hipMemcpyDeviceToHost, ctx->stream));
    }
    st = finish_call(ctx, async);
    if (st != kOk && !async) {
        for (const SeqMeta &m : seqs) pool->seqs[m.slot].len = m.ctx;
    }
    return st;
}

}  // namespace

}  // namespace sr

using namespace sr;

extern "C" SAFETYRAISE_KERNEL_EXPORT int32_t safetyraise_kernel_attention_tree_forward(
    safetyraise_kernel_context *context, const safetyraise_kernel_attention_tree_args *args) {
    if (context == nullptr) return kInvalid;
    const int32_t capture = refuse_under_capture(context, "attention_tree_forward");
    if (capture != kOk) return capture;
    DeviceScope device_scope(context);
    TimerScope timer_scope(context);
    return no_throw(context, [&] { return tree_forward(context, args); });
}
