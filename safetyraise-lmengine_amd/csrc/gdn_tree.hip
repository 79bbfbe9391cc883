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
#include <type_traits>

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

// ---------------------------------------------------------------------------
// Dk = Dv = 128: one workgroup of 8 waves per (value head, sequence), everything
// between the inputs and the outputs in LDS and registers.
//
// Wave w owns state rows 16 w .. 16 w + 15 (32 registers, requested first) and
// the same columns of every [row][Dv] matrix:
//   1. raw conv inputs to LDS behind the history; decays, ancestors, conv taps
//      (one wave, pointer doubling over the parents)
//   2. conv + silu in place, last row first (a row reads rows before it)
//   3. q and k normalised, as fp16 parts
//   4. K S0^T and Q S0^T per wave; K K^T and Q K^T blocks over the waves, masked
//      and decayed:  A[t][j] = -b_t e^{g_t - g_j} (k^_t . k^_j),  j above t
//                    P[t][j] = e^{g_t - g_j} (q^_t . k^_j),       j above or t
//   5. T = (I - A_bb)^-1 of each 16-row block
//   6. block by block  D_b = T_b (b_t (V - e^{g_t} K^ S0^T) + sum_{c<b} A_bc D_c),
//      O_b = e^{g_t} Q^ S0^T + sum_{c<=b} P_bc D_c
//   7. RMSNorm and gate, a row per wave.
// The products of step 6 are v_mfma_f32_16x16x4_f32 with 4 consecutive k per lane; an
// accumulator (rows 4 g + i of lane group g) is the next product's B operand as it is.
// RT: 16-row tiles of the longest tree.
// ---------------------------------------------------------------------------
constexpr uint32_t kW = 128;         // Dk and Dv
constexpr uint32_t kPitch = kW + 4;  // floats per LDS row (16 rows of 16 bytes meet no bank twice)
constexpr uint32_t kHist = 7;        // history rows in front of the tree's

template <int RT>
struct HeadShape {
    static constexpr uint32_t kRows = 16 * RT;
    static constexpr uint32_t kPart = (kHist + kRows) * kPitch;  // floats of q, k or v
    static constexpr uint32_t kPair = kRows + 4;                 // pitch of A and P
    static constexpr size_t kLds = (3 * kPart + 2 * kRows * kPair) * sizeof(float);
};

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// A vector of f32 values as two fp16 parts that sum to them (22 bits), held as
// halves [128] and [128] in an LDS row.  Products of two such vectors take three
// fp16 products (without low . low, 2^-22 of a term), where f32 MFMA takes 16
// times one's time.  Normalised vectors are scaled by 2^kSplitExp and state rows
// so that their largest value is about 2^kStateExp, which keeps the low parts
// normal fp16 numbers.
constexpr int kSplitExp = 8, kStateExp = 10;
struct Split {
    f16x8 hi, lo;
};
__device__ __forceinline__ Split split_row(const float *row, int at) {
    const _Float16 *h = (const _Float16 *)row + at;
    return {*(const f16x8 *)h, *(const f16x8 *)(h + 128)};
}
__device__ __forceinline__ f32x4 mma_split(const Split &a, const Split &b, f32x4 acc) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.lo, b.hi, acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.hi, b.lo, acc, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a.hi, b.hi, acc, 0, 0, 0);
}

// Sum over the wave, without LDS.
__device__ __forceinline__ float wave_sum(float x) {
    x = sum16(x);
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_int(x), __float_as_int(x), false, false);
    x = __int_as_float(r[0]) + __int_as_float(r[1]);
    r = __builtin_amdgcn_permlane32_swap(__float_as_int(x), __float_as_int(x), false, false);
    return __int_as_float(r[0]) + __int_as_float(r[1]);
}

// acc += A . B over 16 k: element i of both operands per instruction
__device__ __forceinline__ f32x4 mma16(const f32x4 &a, const f32x4 &b, f32x4 acc) {
#pragma unroll
    for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], acc, 0, 0, 0);
    return acc;
}

// x * sigmoid(x) with the hardware exp2 and reciprocal
__device__ __forceinline__ float silu_fast(float x) {
    return x * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * x));
}

template <int RT>
__global__ void __launch_bounds__(512) gdn_tree_head_kernel(const GdnTreeParams p) {
    using T = HeadShape<RT>;
    constexpr uint32_t kPair = T::kPair;
    extern __shared__ __align__(16) float lds[];
    __shared__ double g_s[kRowsMax];
    __shared__ uint64_t anc_s[kRowsMax];
    __shared__ float beta_s[kRowsMax], decay_s[kRowsMax];
    // a row's conv taps, newest first: byte offsets of their LDS rows
    __shared__ __align__(16) uint16_t tap_s[kRowsMax][8];
    float *xq = lds, *xk = lds + T::kPart, *xv = lds + 2 * T::kPart;
    float *As = lds + 3 * T::kPart, *Ps = As + T::kRows * kPair;

    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = (uint32_t)wave_index();
    const uint32_t h = blockIdx.x;
    const TreeMeta m = p.meta[blockIdx.y];
    const uint32_t R = m.rows, rt = (R + 15) / 16;
    const uint32_t groups = p.value_heads / p.key_heads, kh = h / groups;
    const bool first_of_key = h % groups == 0;
    const bool bf16 = p.bf16_in != 0;
    const uint32_t K = p.conv_k, K1 = K - 1;
    const uint32_t l16 = lane & 15, g4 = lane >> 4;
    float *rec = p.records + (size_t)m.slot * p.keep_rows * p.rec_stride;

    // 1.
    const uint32_t part = wave >> 1, c = tid & 127;  // q, k, v; waves 6 and 7 have no channel
    const uint32_t ch = part == 0 ? kh * kW + c
                      : part == 1 ? (p.key_heads + kh) * kW + c
                                  : 2 * p.key_heads * kW + h * kW + c;
    float *X = lds + part * T::kPart + c;
    // the wave's state rows: row 16 w + l16, dims 32 s + 8 g4 .. + 7, requested behind the
    // inputs, which are waited for first
    f32x4 S[8];
    auto load_state = [&]() __attribute__((always_inline)) {
        const float *src = p.state + (((size_t)m.state_in * p.value_heads + h) * kW + 16 * wave + l16) * kW + 8 * g4;
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            S[s] = __builtin_nontemporal_load((const f32x4 *)(src + 32 * (s >> 1) + 4 * (s & 1)));
        }
    };
    float w[8];
    if (part < 3) {
        const float *hist = p.history + (((size_t)m.parity * p.max_slots + m.slot) * p.channels + ch) * K1;
        float x[T::kRows], old[kHist];
#pragma unroll
        for (uint32_t i = 0; i < T::kRows; ++i) {
            x[i] = load_act_nb(p.qkv, (size_t)(m.row0 + min(i, R - 1)) * p.channels + ch, bf16);
        }
        // (the history holds at least one value, also for K = 1)
#pragma unroll
        for (uint32_t j = 0; j < kHist; ++j) old[j] = hist[j < K1 ? j : 0];
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
            const float x = p.conv_w[(size_t)ch * K + (j < K ? K1 - j : 0)];  // newest first
            w[j] = j < K ? x : 0.0f;
        }
        load_state();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (uint32_t j = 0; j < kHist; ++j) {
            if (j < K1) X[(kHist - K1 + j) * kPitch] = old[j];
        }
        const bool owns = part == 2 || first_of_key;
#pragma unroll
        for (uint32_t i = 0; i < T::kRows; ++i) {
            X[(kHist + i) * kPitch] = i < R ? x[i] : 0.0f;
            if (owns && i < R) rec[(size_t)i * p.rec_stride + rec_raw(p) + ch] = x[i];
        }
    } else if (wave == 6) {
        const uint32_t r = min(lane, R - 1);
        const float av = load_act(p.a, (size_t)(m.row0 + r) * p.value_heads + h, bf16);
        const float bv = load_act(p.b, (size_t)(m.row0 + r) * p.value_heads + h, bf16);
        load_state();
        __builtin_amdgcn_sched_barrier(0);
        const int up = (int)p.parent[m.row0 - p.meta[0].row0 + r] - 1;
        const float log_a = -expf(p.a_log[h]) * softplus_ref(av + p.dt_bias[h]);
        // the path's set and sum up to, not with, `next`: doubling
        int next = up;
        uint32_t lo = r < 32 ? 1u << r : 0u, hi = r < 32 ? 0u : 1u << (r - 32);
        double sum = (double)log_a;
#pragma unroll
        for (int step = 0; step < 6; ++step) {
            const int at = next < 0 ? (int)lane : next;
            const uint32_t l2 = __shfl(lo, at), h2 = __shfl(hi, at);
            const double s2 = __shfl(sum, at);
            const int n2 = __shfl(next, at);
            if (next >= 0) {
                lo |= l2;
                hi |= h2;
                sum += s2;
                next = n2;
            }
        }
        int at = (int)r, back = 0;
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
            // past the kernel's taps: any finite row, its weight is 0
            if (j >= K) at = (int)r;
            if (lane >= R) at = (int)lane;
            const int u = __shfl(up, at < 0 ? 0 : at);
            tap_s[lane][j] = (uint16_t)((at >= 0 ? (int)kHist + at : (int)kHist - 1 - back) * (int)(kPitch * 4));
            back += at < 0 ? 1 : 0;
            at = at < 0 ? -1 : u;
        }
        if (lane < R) {
            g_s[lane] = sum;
            anc_s[lane] = ((uint64_t)hi << 32) | lo;
            beta_s[lane] = ref_sigmoid(bv);
            decay_s[lane] = (float)exp(sum);
            rec[(size_t)lane * p.rec_stride + h] = expf(log_a);
        } else {
            // rows of the last tile past the tree
            g_s[lane] = 0.0;
            anc_s[lane] = 0;
            beta_s[lane] = decay_s[lane] = 0.0f;
        }
    } else {
        load_state();
    }
    // 8. barrier
    __syncthreads();
    // 2. oldest tap first, as the reference sums them (math.rs:175-185); rows past the
    // tree are zeros with themselves as taps
    if (part < 3) {
        auto conv = [&](auto taps_of) __attribute__((always_inline)) {
            constexpr uint32_t KT = decltype(taps_of)::value;  // taps read per row
            constexpr int kBatch = KT == 4 ? 8 : 4;            // rows whose reads are in flight
            for (int t0 = 16 * (int)rt - kBatch; t0 >= 0; t0 -= kBatch) {
                uint32_t tap[kBatch][KT / 2];
                float x[kBatch][KT];
#pragma unroll
                for (int i = 0; i < kBatch; ++i)
#pragma unroll
                    for (uint32_t j = 0; j < KT / 2; ++j) tap[i][j] = ((const uint32_t *)tap_s[t0 + i])[j];
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < kBatch; ++i)
#pragma unroll
                    for (uint32_t j = 0; j < KT / 2; ++j) {
                        const uint32_t two = (uint32_t)__builtin_amdgcn_readfirstlane((int)tap[i][j]);
                        x[i][2 * j] = *(const float *)((const char *)X + (two & 0xffffu));
                        x[i][2 * j + 1] = *(const float *)((const char *)X + (two >> 16));
                    }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    float acc = 0.0f;
#pragma unroll
                    for (uint32_t j = 0; j < KT; ++j) {
                        // (weights past the kernel's are 0)
                        acc = fmaf(x[i][KT - 1 - j], w[KT - 1 - j], acc);
                    }
                    x[i][0] = acc;
                }
#pragma unroll
                for (int i = 0; i < kBatch; ++i) X[(kHist + t0 + i) * kPitch] = silu_fast(x[i][0]);
            }
        };
        if (K <= 4) conv(std::integral_constant<uint32_t, 4>{});
        else conv(std::integral_constant<uint32_t, 8>{});
    }
    __syncthreads();
    // 3. four vectors of a wave at a time; past the last, the last again
    for (uint32_t t0 = wave; t0 < 2 * R; t0 += 32) {
        float2 y[4];
        float inv[4];
        float *row[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t t = min(t0 + 8 * i, (t0 & 1) + 2 * R - 2);
            row[i] = ((t & 1) ? xk : xq) + (kHist + (t >> 1)) * kPitch;
            y[i] = *(const float2 *)(row[i] + 2 * lane);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 4; ++i) inv[i] = fmaf(y[i].y, y[i].y, y[i].x * y[i].x);
#pragma unroll
        for (int i = 0; i < 4; ++i) inv[i] = __builtin_amdgcn_rsqf(wave_sum(inv[i]) + 1e-6f);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a = y[i].x * inv[i], b = y[i].y * inv[i];
            constexpr float kScale = (float)(1 << kSplitExp);
            const f16x2 hi = {(_Float16)(a * kScale), (_Float16)(b * kScale)};
            const f16x2 lo = {(_Float16)(a * kScale - (float)hi.x), (_Float16)(b * kScale - (float)hi.y)};
            if (t0 + 8 * i < 2 * R) {
                ((f16x2 *)row[i])[lane] = hi;
                ((f16x2 *)row[i])[64 + lane] = lo;
                if ((t0 & 1) && first_of_key) {
                    *(float2 *)(rec + (size_t)((t0 + 8 * i) >> 1) * p.rec_stride + rec_key(p) + kh * kW + 2 * lane) = make_float2(a, b);
                }
            }
        }
    }
    // the state rows' parts
    Split Sp[4];
    int back;  // exponent that undoes the scales
    {
        float mx = 0.0f;
#pragma unroll
        for (int s = 0; s < 8; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) mx = fmaxf(mx, fabsf(S[s][i]));
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        // (frexp's exponent: max in [2^(e - 1), 2^e); 0 for 0)
        const int up = kStateExp - __builtin_amdgcn_frexp_expf(mx);
        back = -up - kSplitExp;
#pragma unroll
        for (int s = 0; s < 8; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = __builtin_amdgcn_ldexpf(S[s][i], up);
                const _Float16 hi = (_Float16)x;
                Sp[s >> 1].hi[4 * (s & 1) + i] = hi;
                Sp[s >> 1].lo[4 * (s & 1) + i] = (_Float16)(x - (float)hi);
            }
    }
    __syncthreads();
    // 4.
    f32x4 kS[RT], qS[RT];
#pragma unroll
    for (int b = 0; b < RT; ++b) {
        kS[b] = qS[b] = f32x4{};
        if ((uint32_t)b >= rt) continue;
        const float *kr = xk + (kHist + 16 * b + l16) * kPitch, *qr = xq + (kHist + 16 * b + l16) * kPitch;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            kS[b] = mma_split(split_row(kr, 32 * s + 8 * g4), Sp[s], kS[b]);
            qS[b] = mma_split(split_row(qr, 32 * s + 8 * g4), Sp[s], qS[b]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            kS[b][e] = __builtin_amdgcn_ldexpf(kS[b][e], back);
            qS[b][e] = __builtin_amdgcn_ldexpf(qS[b][e], back);
        }
    }
    {
        // blocks (bt, bj), bj <= bt, of K K^T, then of Q K^T
        const uint32_t blocks = rt * (rt + 1);
        for (uint32_t i = wave; i < blocks; i += 8) {
            const bool is_q = i >= blocks / 2;
            uint32_t bj = is_q ? i - blocks / 2 : i, bt = 0;
            while (bj > bt) bj -= ++bt;
            const float *ar = (is_q ? xq : xk) + (kHist + 16 * bt + l16) * kPitch;
            const float *br = xk + (kHist + 16 * bj + l16) * kPitch;
            f32x4 acc[2] = {f32x4{}, f32x4{}};
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                acc[s & 1] = mma_split(split_row(ar, 32 * s + 8 * g4), split_row(br, 32 * s + 8 * g4), acc[s & 1]);
            }
            const uint32_t j = 16 * bj + l16;
            const double gj = g_s[j];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t t = 16 * bt + 4 * g4 + e;
                const bool sees = (anc_s[t] >> j) & 1;
                const float ratio = __builtin_amdgcn_exp2f((float)(g_s[t] - gj) * kLog2e);
                const float dot = (acc[0][e] + acc[1][e]) * (1.0f / (1 << (2 * kSplitExp)));
                if (is_q) Ps[t * kPair + j] = sees ? dot * ratio : 0.0f;
                else As[t * kPair + j] = sees && t != j ? -dot * ratio * beta_s[t] : 0.0f;
            }
        }
    }
    // (the rows' z, for step 7)
    const size_t width = (size_t)p.value_heads * kW;
    float z0[2 * RT], z1[2 * RT];
#pragma unroll
    for (int i = 0; i < 2 * RT; ++i) {
        const size_t at = (size_t)(m.row0 + min(wave + 8 * i, R - 1)) * width + h * kW + lane;
        z0[i] = load_act_nb(p.z, at, bf16);
        z1[i] = load_act_nb(p.z, at + 64, bf16);
    }
    __syncthreads();
    // 5. column l16 of the inverse per lane
    if (wave < rt) {
        float *Ab = As + 16 * wave * kPair + 16 * wave;
        float x[16];
#pragma unroll
        for (int t = 0; t < 16; ++t) {
            float acc = (uint32_t)t == l16 ? 1.0f : 0.0f;
#pragma unroll
            for (int i = 0; i < t; ++i) acc = fmaf(Ab[t * kPair + i], x[i], acc);
            x[t] = acc;
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (lane < 16) {
#pragma unroll
            for (int t = 0; t < 16; ++t) Ab[t * kPair + lane] = x[t];
        }
    }
    __syncthreads();
    // 6.
    const float qscale = 0.08838834764831845f;  // 1 / sqrt(128)
    f32x4 D[RT];
#pragma unroll
    for (int b = 0; b < RT; ++b) {
        if ((uint32_t)b >= rt) break;
        float *vr = xv + (kHist + 16 * b + 4 * g4) * kPitch + 16 * wave + l16;
        f32x4 rhs, o;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t t = 16 * b + 4 * g4 + e;
            rhs[e] = beta_s[t] * (vr[e * kPitch] - decay_s[t] * kS[b][e]);
            o[e] = decay_s[t] * qS[b][e];
        }
        const float *Ar = As + (16 * b + l16) * kPair + 4 * g4;
        const float *Pr = Ps + (16 * b + l16) * kPair + 4 * g4;
#pragma unroll
        for (int cc = 0; cc < b; ++cc) {
            rhs = mma16(*(const f32x4 *)(Ar + 16 * cc), D[cc], rhs);
            o = mma16(*(const f32x4 *)(Pr + 16 * cc), D[cc], o);
        }
        D[b] = mma16(*(const f32x4 *)(Ar + 16 * b), rhs, f32x4{});
        o = mma16(*(const f32x4 *)(Pr + 16 * b), D[b], o);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t t = 16 * b + 4 * g4 + e;
            vr[e * kPitch] = o[e] * qscale;
            if (t < R) rec[(size_t)t * p.rec_stride + rec_delta(p) + h * kW + 16 * wave + l16] = D[b][e];
        }
    }
    __syncthreads();
    // 7. RMSNorm without offset, then * silu(z) (native.rs:737-740); rows past the
    // wave's last repeat it
    const float n0 = p.norm[lane], n1 = p.norm[lane + 64];
    constexpr int kOut = 2 * RT < 4 ? 2 * RT : 4;  // rows at a time
#pragma unroll
    for (int i0 = 0; i0 < 2 * RT; i0 += kOut) {
        if (wave + 8 * i0 >= R) break;
        float o0[kOut], o1[kOut], inv[kOut];
#pragma unroll
        for (int i = 0; i < kOut; ++i) {
            const float *o = xv + (kHist + min(wave + 8 * (i0 + i), R - 1)) * kPitch;
            o0[i] = o[lane];
            o1[i] = o[lane + 64];
        }
#pragma unroll
        for (int i = 0; i < kOut; ++i) {
            const float variance = wave_sum(fmaf(o1[i], o1[i], o0[i] * o0[i])) / (float)kW;
            if (!isfinite(variance) && lane == 0) atomicOr(p.err_word, kErrNonFiniteVariance);
            inv[i] = 1.0f / sqrtf(variance + p.eps);
        }
#pragma unroll
        for (int i = 0; i < kOut; ++i) {
            const uint32_t t = wave + 8 * (i0 + i);
            if (t >= R) break;
            float *dst = p.out + (size_t)(m.row0 + t) * width + h * kW;
            dst[lane] = o0[i] * inv[i] * n0 * silu_fast(z0[i0 + i]);
            dst[lane + 64] = o1[i] * inv[i] * n1 * silu_fast(z1[i0 + i]);
        }
    }
}

template <int RT>
hipError_t launch_head(hipStream_t stream, const GdnTreeParams &p) {
    using T = HeadShape<RT>;
    static_assert(T::kLds + 8192 <= 160 * 1024, "LDS");
    static const hipError_t configured =
        hipFuncSetAttribute((const void *)gdn_tree_head_kernel<RT>,
                            hipFuncAttributeMaxDynamicSharedMemorySize, (int)T::kLds);
    if (configured != hipSuccess) return configured;
    SR_LAUNCH("gdn_tree_head_kernel", gdn_tree_head_kernel<RT>, dim3(p.value_heads, p.nseq), dim3(512),
              T::kLds, stream, p);
    return hipGetLastError();
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
    if (pool->key_dim == kW && pool->value_dim == kW) return 0;
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
    uint32_t most = 0;
    for (int i = 0; i < nseq; ++i) most = std::max(most, seqs[i].rows);
    if (p.key_dim == kW && p.value_dim == kW) {
        switch ((most + 15) / 16) {
            case 1: return launch_head<1>(stream, p);
            case 2: return launch_head<2>(stream, p);
            case 3: return launch_head<3>(stream, p);
            default: return launch_head<4>(stream, p);
        }
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
