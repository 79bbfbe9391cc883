// Gated delta net over a tree of drafted rows, for gfx950.
//
// Row r continues from its parent p(r): with a_r its decay, k^ and q^ the
// normalised conv outputs,
//     S_r = a_r S_p(r) + d_r k^_r^T,   d_r = b_r (v_r - a_r S_p(r) k^_r),
//     o_r = S_r q^_r / sqrt(Dk),
// S_-1 = S0 the sequence's state.  No S_r is formed: along the path to r
//     S_r = e^{g_r} S0 + sum_{j in anc(r)} e^{g_r - g_j} d_j k^_j^T,
// g_r the sum of log a over anc(r) (r among them), so
//     d_t = b_t (v_t - e^{g_t} S0 k^_t - sum_{j in anc(t), j < t} e^{g_t - g_j} (k^_j . k^_t) d_j)
//     o_t = (e^{g_t} S0 q^_t + sum_{j in anc(t)} e^{g_t - g_j} (k^_j . q^_t) d_j) / sqrt(Dk):
// S0 is read once for all rows, in any shape of tree, and never written.  Every
// exponent is of a difference along one path, at most 0, taken in f64.  A row's
// conv taps are its ancestors' raw inputs, then the sequence's history.
//
// Records per row (the pool's, see gdn_rollback): a [Hv], d [Hv][Dv], k^ [Hk][Dk],
// raw conv inputs [C]; gdn_tree_commit_kernel builds the state of a path from them.
#include <algorithm>

#include "sr_device.hpp"
#include "tree_plan.hpp"

namespace sr {

namespace {

constexpr uint32_t kRowsMax = kMaxGdnTreeRows;

struct TreeMeta {
    uint32_t slot, rows, row0, parity, state_in;
};

struct GdnTreeParams {
    const float *state;
    const float *history;
    const void *qkv, *z, *a, *b;
    const float *a_log, *dt_bias, *conv_w, *norm;
    float *out;
    float *conv;     // [rows of the launch][C] conv outputs
    float *records;  // [slots][keep_rows][rec_stride]
    uint32_t *err_word;
    float eps;
    uint32_t rec_stride, keep_rows;
    uint32_t key_heads, value_heads, key_dim, value_dim, conv_k, channels, max_slots;
    int bf16_in;
    uint32_t nseq, rows;
    TreeMeta meta[kGdnTreeSeqs];
    uint8_t parent[kGdnTreeSeqs * kRowsMax];  // parent + 1 within the sequence
};
static_assert(sizeof(GdnTreeParams) <= 4096, "kernel arguments stay within 4 KiB");

__device__ __forceinline__ float softplus_ref(float x) {
    return fmaxf(x, 0.0f) + log1pf(expf(-fabsf(x)));
}

// The float offsets of a record's parts behind the decays.
__device__ __forceinline__ uint32_t rec_delta(const GdnTreeParams &p) { return p.value_heads; }
__device__ __forceinline__ uint32_t rec_key(const GdnTreeParams &p) {
    return p.value_heads * (1 + p.value_dim);
}
__device__ __forceinline__ uint32_t rec_raw(const GdnTreeParams &p) {
    return p.value_heads * (1 + p.value_dim + p.key_dim);
}

// Any widths: conv and silu of every row and channel, and the raw inputs into the
// records.  grid (channel blocks, rows)
__global__ void __launch_bounds__(256) gdn_tree_conv_kernel(const GdnTreeParams p) {
    const uint32_t c = blockIdx.x * 256 + threadIdx.x, r = blockIdx.y;
    if (c >= p.channels) return;
    uint32_t s = 0;
    const uint32_t row_first = p.meta[0].row0;
    while (s + 1 < p.nseq && p.meta[s + 1].row0 - row_first <= r) ++s;
    const TreeMeta m = p.meta[s];
    const uint32_t sr = r - (m.row0 - row_first);
    const uint8_t *parent = p.parent + (m.row0 - row_first);
    const uint32_t K = p.conv_k;
    const float *w = p.conv_w + (size_t)c * K;
    const float *hist = p.history + (((size_t)m.parity * p.max_slots + m.slot) * p.channels + c) * (K - 1);
    const float x = load_act(p.qkv, (size_t)(m.row0 + sr) * p.channels + c, p.bf16_in);
    // oldest tap first, as the reference sums them (math.rs:175-185)
    float tap[8];
    uint32_t at = sr + 1;  // row + 1; 0: before the tree
    uint32_t back = 0;     // history taps used
    for (uint32_t j = K; j-- > 0;) {
        if (at != 0) {
            tap[j] = load_act(p.qkv, (size_t)(m.row0 + at - 1) * p.channels + c, p.bf16_in);
            at = parent[at - 1];
        } else {
            tap[j] = hist[K - 2 - back++];
        }
    }
    float acc = 0.0f;
    for (uint32_t j = 0; j < K; ++j) acc = fmaf(tap[j], w[j], acc);
    p.conv[(size_t)r * p.channels + c] = acc * ref_sigmoid(acc);
    p.records[((size_t)m.slot * p.keep_rows + sr) * p.rec_stride + rec_raw(p) + c] = x;
}

// Any widths: one workgroup per (value head, sequence), a thread per value dim.
__global__ void __launch_bounds__(256) gdn_tree_generic_kernel(const GdnTreeParams p) {
    __shared__ float kk[kRowsMax][kRowsMax + 1], qk[kRowsMax][kRowsMax + 1];
    __shared__ double g[kRowsMax];
    __shared__ float beta[kRowsMax], decay[kRowsMax], qn[kRowsMax], kn[kRowsMax], log_a[kRowsMax];
    __shared__ uint64_t anc[kRowsMax];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t h = blockIdx.x;
    const TreeMeta m = p.meta[blockIdx.y];
    const uint32_t row_first = p.meta[0].row0, R = m.rows;
    const uint8_t *parent = p.parent + (m.row0 - row_first);
    const uint32_t groups = p.value_heads / p.key_heads, kh = h / groups;
    const uint32_t Dk = p.key_dim, Dv = p.value_dim;
    const float *conv = p.conv + (size_t)(m.row0 - row_first) * p.channels;
    const uint32_t q_at = kh * Dk, k_at = p.key_heads * Dk + kh * Dk, v_at = 2 * p.key_heads * Dk + h * Dv;
    float *rec = p.records + (size_t)m.slot * p.keep_rows * p.rec_stride;
    if (tid < R) {
        const float av = load_act(p.a, (size_t)(m.row0 + tid) * p.value_heads + h, p.bf16_in);
        const float bv = load_act(p.b, (size_t)(m.row0 + tid) * p.value_heads + h, p.bf16_in);
        log_a[tid] = -expf(p.a_log[h]) * softplus_ref(av + p.dt_bias[h]);
        beta[tid] = ref_sigmoid(bv);
        rec[(size_t)tid * p.rec_stride + h] = expf(log_a[tid]);
    }
    __syncthreads();
    if (tid < R) {
        uint64_t bits = 0;
        double sum = 0.0;
        for (uint32_t t = tid + 1; t != 0; t = parent[t - 1]) {
            bits |= 1ull << (t - 1);
            sum += (double)log_a[t - 1];
        }
        anc[tid] = bits;
        g[tid] = sum;
        decay[tid] = (float)exp(sum);
    }
    for (uint32_t t = wave; t < 2 * R; t += 4) {
        const float *y = conv + (size_t)(t >> 1) * p.channels + ((t & 1) ? k_at : q_at);
        float ss = 0.0f;
        for (uint32_t d = lane; d < Dk; d += 64) ss = fmaf(y[d], y[d], ss);
        ss = sum64(ss);
        if (lane == 0) ((t & 1) ? kn : qn)[t >> 1] = 1.0f / sqrtf(ss + 1e-6f);
    }
    __syncthreads();
    if (h % groups == 0) {
        for (uint32_t i = tid; i < R * Dk; i += 256) {
            const uint32_t t = i / Dk, d = i % Dk;
            rec[(size_t)t * p.rec_stride + rec_key(p) + kh * Dk + d] = conv[(size_t)t * p.channels + k_at + d] * kn[t];
        }
    }
    const float qscale = 1.0f / sqrtf((float)Dk);
    for (uint32_t i = tid; i < R * R; i += 256) {
        const uint32_t t = i / R, j = i % R;
        if (!((anc[t] >> j) & 1)) continue;
        const float *kt = conv + (size_t)t * p.channels + k_at, *kj = conv + (size_t)j * p.channels + k_at;
        const float *qt = conv + (size_t)t * p.channels + q_at;
        float x = 0.0f, y = 0.0f;
        for (uint32_t d = 0; d < Dk; ++d) {
            x = fmaf(kt[d], kj[d], x);
            y = fmaf(qt[d], kj[d], y);
        }
        const float ratio = (float)exp(g[t] - g[j]);
        kk[t][j] = x * kn[t] * kn[j] * ratio * beta[t];
        qk[t][j] = y * qn[t] * kn[j] * ratio;
    }
    __syncthreads();
    const float *S = p.state + ((size_t)m.state_in * p.value_heads + h) * Dv * Dk;
    const size_t width = (size_t)p.value_heads * Dv;
    for (uint32_t v = tid; v < Dv; v += 256) {
        const float *row = S + (size_t)v * Dk;
        for (uint32_t t = 0; t < R; ++t) {
            const float *kt = conv + (size_t)t * p.channels + k_at, *qt = conv + (size_t)t * p.channels + q_at;
            float x = 0.0f, y = 0.0f;
            for (uint32_t d = 0; d < Dk; ++d) {
                x = fmaf(row[d], kt[d], x);
                y = fmaf(row[d], qt[d], y);
            }
            const float vt = conv[(size_t)t * p.channels + v_at + v];
            float delta = beta[t] * (vt - decay[t] * x * kn[t]);
            float o = decay[t] * y * qn[t];
            // a thread's own earlier corrections, from the records
            for (uint64_t bits = anc[t] & ~(1ull << t); bits != 0; bits &= bits - 1) {
                const uint32_t j = (uint32_t)__builtin_ctzll(bits);
                const float dj = rec[(size_t)j * p.rec_stride + rec_delta(p) + h * Dv + v];
                delta = fmaf(-kk[t][j], dj, delta);
                o = fmaf(qk[t][j], dj, o);
            }
            o = fmaf(qk[t][t], delta, o);
            rec[(size_t)t * p.rec_stride + rec_delta(p) + h * Dv + v] = delta;
            p.out[(size_t)(m.row0 + t) * width + h * Dv + v] = o * qscale;
        }
    }
    __syncthreads();
    // RMSNorm without offset, then * silu(z): a row per wave (native.rs:737-740)
    for (uint32_t t = wave; t < R; t += 4) {
        const size_t at = (size_t)(m.row0 + t) * width + (size_t)h * Dv;
        float ss = 0.0f;
        for (uint32_t d = lane; d < Dv; d += 64) ss = fmaf(p.out[at + d], p.out[at + d], ss);
        const float variance = sum64(ss) / (float)Dv;
        if (!isfinite(variance) && lane == 0) atomicOr(p.err_word, kErrNonFiniteVariance);
        const float inv = 1.0f / sqrtf(variance + p.eps);
        for (uint32_t d = lane; d < Dv; d += 64) {
            const float z = load_act(p.z, at + d, p.bf16_in);
            p.out[at + d] = p.out[at + d] * inv * p.norm[d] * (z * ref_sigmoid(z));
        }
    }
}

struct CommitParams {
    const GdnCommitEntry *entries;  // nullptr: in the arguments
    GdnCommitEntry inline_entries[kGdnCommitInline];
};
static_assert(sizeof(CommitParams) <= 4096, "kernel arguments stay within 4 KiB");

constexpr uint32_t kCommitRows = 4;  // state rows per thread

// S = a S + d k^T along the path: 16-byte units of the state, a thread the same
// columns of kCommitRows rows, then the conv channels' last K - 1 inputs.  grid
// (blocks of the largest entry, entries)
template <typename Unit>
__global__ void __launch_bounds__(256) gdn_tree_commit_kernel(const CommitParams p) {
    constexpr uint32_t W = sizeof(Unit) / 4;
    const GdnCommitEntry e = p.entries != nullptr ? p.entries[blockIdx.y] : p.inline_entries[blockIdx.y];
    const uint32_t per = e.key_dim / W;                                  // units per state row
    const uint32_t bands = (e.value_dim + kCommitRows - 1) / kCommitRows;  // of rows, per head
    const uint64_t units = (uint64_t)e.value_heads * bands * per;
    const uint64_t state_blocks = (units + 255) / 256;
    if (blockIdx.x < state_blocks) {
        const uint64_t u = blockIdx.x * 256ull + threadIdx.x;
        if (u >= units) return;
        const uint32_t c = (uint32_t)(u % per);
        const uint32_t band = (uint32_t)(u / per % bands), h = (uint32_t)(u / per / bands);
        const uint32_t kh = h / (e.value_heads / e.key_heads);
        alignas(16) float S[kCommitRows][W];
        uint32_t v[kCommitRows];
#pragma unroll
        for (uint32_t i = 0; i < kCommitRows; ++i) {
            v[i] = min(band + bands * i, e.value_dim - 1);
            *(Unit *)S[i] = *((const Unit *)(e.state_in + ((size_t)h * e.value_dim + v[i]) * e.key_dim) + c);
        }
        for (uint64_t path = e.path; path != 0; path &= path - 1) {
            const float *rec = e.records + (size_t)__builtin_ctzll(path) * e.rec_stride;
            const float alpha = rec[h];
            float k[W];
            const float *key = rec + e.value_heads * (1 + e.value_dim) + kh * e.key_dim + W * c;
#pragma unroll
            for (uint32_t j = 0; j < W; ++j) k[j] = key[j];
#pragma unroll
            for (uint32_t i = 0; i < kCommitRows; ++i) {
                const float delta = rec[e.value_heads + h * e.value_dim + v[i]];
#pragma unroll
                for (uint32_t j = 0; j < W; ++j) S[i][j] = fmaf(delta, k[j], S[i][j] * alpha);
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < kCommitRows; ++i) {
            // (rows past the last repeat it)
            if (band + bands * i < e.value_dim) {
                *((Unit *)(e.state_out + ((size_t)h * e.value_dim + v[i]) * e.key_dim) + c) = *(const Unit *)S[i];
            }
        }
        return;
    }
    const uint32_t c = (uint32_t)(blockIdx.x - state_blocks) * 256 + threadIdx.x, K1 = e.conv_k - 1;
    if (c >= e.channels || K1 == 0) return;
    // the last K - 1 of (history, raw inputs of the path): newest first
    uint64_t path = e.path;
    uint32_t back = 0;
    float x[7];
    for (uint32_t i = K1; i-- > 0;) {
        if (path != 0) {
            const uint32_t r = 63 - (uint32_t)__builtin_clzll(path);
            path &= ~(1ull << r);
            x[i] = e.records[(size_t)r * e.rec_stride + e.value_heads * (1 + e.value_dim + e.key_dim) + c];
        } else {
            x[i] = e.hist_in[(size_t)c * K1 + (K1 - 1 - back++)];
        }
    }
    for (uint32_t i = 0; i < K1; ++i) e.hist_out[(size_t)c * K1 + i] = x[i];
}

}  // namespace

size_t gdn_tree_scratch_bytes(const safetyraise_kernel_gdn_pool *pool, uint32_t rows) {
    return (size_t)rows * pool->channels * sizeof(float);
}

hipError_t launch_gdn_tree(hipStream_t stream, const GdnLaunch &g, const GdnSeq *seqs, int nseq,
                           const uint8_t *parents, float *scratch) {
    const auto *pool = g.pool;
    if (nseq <= 0 || nseq > kGdnTreeSeqs) return hipErrorInvalidValue;
    GdnTreeParams p{};
    p.state = pool->d_state;
    p.history = pool->d_history;
    p.qkv = g.qkv;
    p.z = g.z;
    p.a = g.a;
    p.b = g.b;
    p.a_log = g.a_log;
    p.dt_bias = g.dt_bias;
    p.conv_w = g.conv_w;
    p.norm = g.norm;
    p.out = g.out;
    p.conv = scratch;
    p.records = pool->d_records;
    p.err_word = g.err_word;
    p.eps = g.eps;
    p.rec_stride = g.rec_stride;
    p.keep_rows = g.keep_rows;
    p.key_heads = pool->key_heads;
    p.value_heads = pool->value_heads;
    p.key_dim = pool->key_dim;
    p.value_dim = pool->value_dim;
    p.conv_k = pool->conv_kernel;
    p.channels = pool->channels;
    p.max_slots = pool->max_sequences;
    p.bf16_in = g.bf16_in ? 1 : 0;
    p.nseq = (uint32_t)nseq;
    for (int i = 0; i < nseq; ++i) {
        if (seqs[i].rows > kRowsMax || seqs[i].rows > g.keep_rows) return hipErrorInvalidValue;
        p.meta[i] = TreeMeta{seqs[i].slot, seqs[i].rows, seqs[i].row0, seqs[i].parity, seqs[i].state_in};
        for (uint32_t r = 0; r < seqs[i].rows; ++r) p.parent[p.rows + r] = parents[p.rows + r];
        p.rows += seqs[i].rows;
    }
    SR_LAUNCH("gdn_tree_conv_kernel", gdn_tree_conv_kernel, dim3((p.channels + 255) / 256, p.rows),
              dim3(256), 0, stream, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    SR_LAUNCH("gdn_tree_generic_kernel", gdn_tree_generic_kernel, dim3(p.value_heads, p.nseq), dim3(256),
              0, stream, p);
    return hipGetLastError();
}

hipError_t launch_gdn_tree_commit(hipStream_t stream, const GdnCommitEntry *entries, uint32_t count,
                                  const GdnCommitEntry *device) {
    CommitParams p{};
    p.entries = device;
    if (device == nullptr && count > kGdnCommitInline) return hipErrorInvalidValue;
    uint64_t blocks[2] = {0, 0};
    bool vec = true;
    for (uint32_t i = 0; i < count; ++i) {
        const GdnCommitEntry &e = entries[i];
        if (device == nullptr) p.inline_entries[i] = e;
        vec = vec && e.key_dim % 4 == 0;
        const uint64_t bands = (e.value_dim + kCommitRows - 1) / kCommitRows;
        for (int k = 0; k < 2; ++k) {
            const uint64_t units = e.value_heads * bands * (k == 0 ? e.key_dim / 4 : e.key_dim);
            blocks[k] = std::max<uint64_t>(blocks[k], (units + 255) / 256 + (e.channels + 255) / 256);
        }
    }
    if (vec) {
        SR_LAUNCH("gdn_tree_commit_kernel", gdn_tree_commit_kernel<float4>, dim3((uint32_t)blocks[0], count),
                  dim3(256), 0, stream, p);
    } else {
        SR_LAUNCH("gdn_tree_commit_kernel", gdn_tree_commit_kernel<float>, dim3((uint32_t)blocks[1], count),
                  dim3(256), 0, stream, p);
    }
    return hipGetLastError();
}

}  // namespace sr
