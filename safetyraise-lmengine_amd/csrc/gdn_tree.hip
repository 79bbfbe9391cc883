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

// Least log a that sums of them take: e^x is 0 in f32 from -104 on, and differences of
// sums that hold minus infinity would be NaN.
constexpr float kLeastLog = -1000.0f;
__device__ __forceinline__ float finite_log(float log_a) { return log_a < kLeastLog ? kLeastLog : log_a; }

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

// Any widths: one workgroup per (value head, sequence), a thread per value dim, which
// goes through the rows one after another.  Bound by that chain and by the reads of its
// state row for every row of the tree: eight sequences of 44 rows, 32 value heads of 64 x 64,
// 340 us and 18 for the conv, where inputs, state and outputs are 3.3 us.  It is there for
// widths that no configuration of this framework has.
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
        log_a[tid] = finite_log(-expf(p.a_log[h]) * softplus_ref(av + p.dt_bias[h]));
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
// Wave w owns state rows 16 w .. 16 w + 15 (32 registers, requested with the inputs)
// and the same columns of every [row][Dv] matrix:
//   1. raw conv inputs to LDS behind the history, 16 bytes per lane; decays, ancestors,
//      conv taps (one wave, pointer doubling over the parents)
//   2. v, q, k in turn: conv + silu of a row, two channels per lane, into memory that
//      no row reads any more;
//   3. with them q and k normalised, as fp16 parts
//   4. K S0^T and Q S0^T per wave; on the way K K^T and Q K^T blocks, masked and
//      decayed:  A[t][j] = -b_t e^{g_t - g_j} (k^_t . k^_j),  j above t
//                P[t][j] = e^{g_t - g_j} (q^_t . k^_j),       j above or t
//   5. T = (I - A_bb)^-1 of each 16-row block
//   6. block by block  D_b = T_b (b_t (V - e^{g_t} K^ S0^T) + sum_{c<b} A_bc D_c),
//      O_b = e^{g_t} Q^ S0^T + sum_{c<=b} P_bc D_c
//   7. RMSNorm and gate, a row per wave.
// The products of step 6 are v_mfma_f32_16x16x4_f32 with 4 consecutive k per lane; an
// accumulator (rows 4 g + i of lane group g) is the next product's B operand as it is.
// RT: 16-row tiles of the longest tree.
//
// What bounds it: the chain of phases, each bound by something else.  Eight sequences of
// 24..64 rows, 16 key and 32 value heads: 30.2 us for 40 MB (8.3 us at the copy rate):
// inputs and state 7, conv and norms 6.3 (vector instructions: exponentials and
// reciprocals of the silu; q and k are made once per value head of theirs), products 4.9,
// solve 0.7, step 6 2.2 and 0.8 more for its checks of d, outputs 1.6.  One sequence of 12
// rows: 10.7 us, mostly latency and the fetch of the code.  With 4-byte loads, the conv in
// place and the norms in a pass of their own it took 32 us.
// ---------------------------------------------------------------------------
constexpr uint32_t kW = 128;         // Dk and Dv
constexpr uint32_t kPitch = kW + 4;  // floats per LDS row (16 rows of 16 bytes meet no bank twice)
constexpr uint32_t kHist = 7;        // history rows in front of the tree's

template <int RT>
struct HeadShape {
    static constexpr uint32_t kRows = 16 * RT;
    static constexpr uint32_t kPart = (kHist + kRows) * kPitch;  // floats of raw q, k or v
    static constexpr uint32_t kPair = kRows + 4;                 // pitch of A and P
    // raw q, k, v, and the finished v; the finished q is where v was, the finished k
    // where q was, A and P where k was
    static constexpr size_t kLds = (3 * kPart + kRows * kPitch) * sizeof(float);
    static_assert(2 * kRows * kPair <= kPart, "A and P fit the raw k");
};

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
// (a caller's tensors may begin at any of their values, and a record's rows are aligned
// to 4 bytes)
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef float f32x2u __attribute__((ext_vector_type(2), aligned(4)));
typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2u __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u32u __attribute__((aligned(2)));
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
    __shared__ uint32_t lost_s[2];  // rows whose decay, step or key is not finite
    // a row's conv taps, newest first: byte offsets of their LDS rows
    __shared__ __align__(16) uint16_t tap_s[kRowsMax][8];
    float *xq = lds + 2 * T::kPart, *xk = lds, *xv = lds + 3 * T::kPart;
    float *As = lds + T::kPart, *Ps = As + T::kRows * kPair;

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

    // 1. 4 channels of a row per lane: rows 2 n, 2 n + 1 of q, k or v per load
    const uint32_t l32 = lane & 31, half = lane >> 5;
    const uint32_t head_ch[3] = {kh * kW, (p.key_heads + kh) * kW, 2 * p.key_heads * kW + h * kW};
    const uint32_t r = min(lane, R - 1);
    const size_t ab_at = (size_t)(m.row0 + r) * p.value_heads + h;
    uint32_t a_raw = 0, b_raw = 0, up_raw = 0;
    float a_log = 0.0f, dt_bias = 0.0f;
    if (wave == 0) {
        a_raw = bf16 ? ((const uint16_t *)p.a)[ab_at] : ((const uint32_t *)p.a)[ab_at];
        b_raw = bf16 ? ((const uint16_t *)p.b)[ab_at] : ((const uint32_t *)p.b)[ab_at];
        // (a lane's loads: scalar ones would be waited for here)
        uint32_t at = h;
        asm volatile("" : "+v"(at));
        a_log = p.a_log[at];
        dt_bias = p.dt_bias[at];
        up_raw = p.parent[m.row0 - p.meta[0].row0 + r];
    }
    u32x4 raw[3 * RT];
    u32x2 raw16[3 * RT];
    auto raw_at = [&](int n) __attribute__((always_inline)) {
        const uint32_t row = min(2 * (wave + 8 * (n % RT)) + half, R - 1);
        return (size_t)(m.row0 + row) * p.channels + head_ch[n / RT] + 4 * l32;
    };
    if (bf16) {
#pragma unroll
        for (int n = 0; n < 3 * RT; ++n) raw16[n] = *(const u32x2u *)((const uint16_t *)p.qkv + raw_at(n));
    } else {
#pragma unroll
        for (int n = 0; n < 3 * RT; ++n) raw[n] = *(const u32x4u *)((const float *)p.qkv + raw_at(n));
    }
    // the channels' history, one per thread
    const uint32_t hc = tid & 127, hpart = min(tid >> 7, 2u);
    float old[kHist];
    {
        const uint32_t ch = hc + (hpart < 2 ? (hpart * p.key_heads + kh) * kW : 2 * p.key_heads * kW + h * kW);
        const float *hist = p.history + (((size_t)m.parity * p.max_slots + m.slot) * p.channels + ch) * K1;
#pragma unroll
        for (uint32_t j = 0; j < kHist; ++j) old[j] = j < K1 ? hist[j] : 0.0f;
    }
    // conv weights of channels 2 lane, 2 lane + 1, oldest tap first: of 4 taps, or any
    // (in registers of their own, or the loads of one kind would wait for the other's)
    f32x4 w4[3][2];
    float w[3][8][2];
    if (K == 4) {
#pragma unroll
        for (int part = 0; part < 3; ++part)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                w4[part][e] = *(const f32x4u *)(p.conv_w + (size_t)(head_ch[part] + 2 * lane + e) * 4);
            }
    }
    if (K != 4) {
#pragma unroll
        for (int part = 0; part < 3; ++part)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float *src = p.conv_w + (size_t)(head_ch[part] + 2 * lane + e) * K;
#pragma unroll
                for (uint32_t j = 0; j < 8; ++j) w[part][j][e] = j < K ? src[j] : 0.0f;
            }
    }
    // the wave's state rows: row 16 w + l16, dims 32 s + 8 g4 .. + 7
    f32x4 S[8];
    {
        const float *src = p.state + (((size_t)m.state_in * p.value_heads + h) * kW + 16 * wave + l16) * kW + 8 * g4;
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            S[s] = __builtin_nontemporal_load((const f32x4 *)(src + 32 * (s >> 1) + 4 * (s & 1)));
        }
    }
    __builtin_amdgcn_sched_barrier(0);
    if (wave == 0) {
        // (used from here on: earlier, the compiler would wait for them before the other loads)
        asm volatile("" : "+v"(a_raw), "+v"(b_raw), "+v"(up_raw), "+v"(a_log), "+v"(dt_bias));
        const float av = __uint_as_float(bf16 ? a_raw << 16 : a_raw), bv = __uint_as_float(bf16 ? b_raw << 16 : b_raw);
        const int up = (int)up_raw - 1;
        const float raw_log = finite_log(-expf(a_log) * softplus_ref(av + dt_bias)), raw_beta = ref_sigmoid(bv);
        // (rows that are not finite: see step 6)
        const bool lost = isnan(raw_log) || isnan(raw_beta);
        const uint64_t all_lost = __builtin_amdgcn_ballot_w64(lost && lane < R);
        if (lane < 2) lost_s[lane] = (uint32_t)(all_lost >> (32 * lane));
        const float log_a = lost ? 0.0f : raw_log, beta = lost ? 0.0f : raw_beta;
        // the path's set and sum up to, not with, `next`: doubling
        int next = up;
        uint32_t lo = r < 32 ? 1u << r : 0u, hi = r < 32 ? 0u : 1u << (r - 32);
        double sum = (double)log_a;
#pragma unroll 1
        for (int step = 0; step < 6 && __builtin_amdgcn_ballot_w64(next >= 0) != 0; ++step) {
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
#pragma unroll 1
        for (uint32_t j = 0; j < (K == 4 ? 4u : 8u); ++j) {
            // past the kernel's taps: any finite row, its weight is 0
            if (j >= K) at = (int)r;
            if (lane >= R) at = (int)lane;
            const int u = __shfl(up, at < 0 ? 0 : at);
            tap_s[lane][j < K ? K1 - j : j] =
                (uint16_t)((at >= 0 ? (int)kHist + at : (int)kHist - 1 - back) * (int)(kPitch * 4));
            back += at < 0 ? 1 : 0;
            at = at < 0 ? -1 : u;
        }
        if (lane < R) {
            g_s[lane] = sum;
            anc_s[lane] = ((uint64_t)hi << 32) | lo;
            beta_s[lane] = beta;
            decay_s[lane] = (float)exp(sum);
            rec[(size_t)lane * p.rec_stride + h] = expf(raw_log);
        } else {
            // rows of the last tile past the tree
            g_s[lane] = 0.0;
            anc_s[lane] = 0;
            beta_s[lane] = decay_s[lane] = 0.0f;
        }
    }
#pragma unroll
    for (int n = 0; n < 3 * RT; ++n) {
        const uint32_t row = 2 * (wave + 8 * (n % RT)) + half;
        f32x4 x;
        if (bf16) x = f32x4{bf16lo(raw16[n].x), bf16hi(raw16[n].x), bf16lo(raw16[n].y), bf16hi(raw16[n].y)};
        else x = __builtin_bit_cast(f32x4, raw[n]);
        if (row >= R) x = f32x4{};
        *(f32x4 *)(lds + (n / RT) * T::kPart + (kHist + row) * kPitch + 4 * l32) = x;
        if ((n / RT == 2 || first_of_key) && row < R) {
            *(f32x4u *)(rec + (size_t)row * p.rec_stride + rec_raw(p) + head_ch[n / RT] + 4 * l32) = x;
        }
    }
    if (tid < 3 * kW) {
#pragma unroll
        for (uint32_t j = 0; j < kHist; ++j) {
            if (j < K1) lds[hpart * T::kPart + (kHist - K1 + j) * kPitch + hc] = old[j];
        }
    }
    __syncthreads();
    // 2., 3. v, then q, then k, each into memory that no row reads any more: kBatch rows
    // per wave at a time, two channels per lane.  Oldest tap first, as the reference sums
    // them (math.rs:175-185); rows past the tree are zeros with themselves as taps
    float *const keys = rec + rec_key(p) + kh * kW + 2 * lane;
    const uint32_t rec_stride = p.rec_stride;
    auto conv = [&](auto taps_of) __attribute__((always_inline)) {
        constexpr uint32_t KT = decltype(taps_of)::value;  // taps read per row
        constexpr uint32_t kBatch = 2 * RT < 4 ? 2 * RT : 4;
#pragma unroll 1
        for (int turn = 0; turn < 3; ++turn) {
            const int part = turn == 0 ? 2 : turn - 1;
            const float *from = lds + part * T::kPart + 2 * lane;
            float *to = lds + (turn == 0 ? 3u : turn == 1 ? 2u : 0u) * T::kPart;  // xv, xq, xk
            // (by value: a choice between array elements would put the array in memory)
            auto of_turn = [turn](float first, float second, float third) {
                return turn == 0 ? first : turn == 1 ? second : third;
            };
            float wt[KT][2];
#pragma unroll
            for (uint32_t j = 0; j < KT; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    if constexpr (KT == 4) wt[j][e] = of_turn(w4[2][e][j], w4[0][e][j], w4[1][e][j]);
                    else wt[j][e] = of_turn(w[2][j][e], w[0][j][e], w[1][j][e]);
                }
            for (uint32_t t0 = wave; t0 < 16 * rt; t0 += 8 * kBatch) {
                uint32_t tap[kBatch][KT / 2];
                float2 x[kBatch][KT];
                // (past the last tile: the batch's first row again)
#pragma unroll
                for (uint32_t i = 0; i < kBatch; ++i) {
                    const uint32_t t = t0 + 8 * i < 16 * rt ? t0 + 8 * i : t0;
#pragma unroll
                    for (uint32_t j = 0; j < KT / 2; ++j) tap[i][j] = ((const uint32_t *)tap_s[t])[j];
                }
#pragma unroll
                for (uint32_t i = 0; i < kBatch; ++i)
#pragma unroll
                    for (uint32_t j = 0; j < KT / 2; ++j) {
                        const uint32_t two = (uint32_t)__builtin_amdgcn_readfirstlane((int)tap[i][j]);
                        x[i][2 * j] = *(const float2 *)((const char *)from + (two & 0xffffu));
                        x[i][2 * j + 1] = *(const float2 *)((const char *)from + (two >> 16));
                    }
                __builtin_amdgcn_sched_barrier(0);
                float2 y[kBatch];
#pragma unroll
                for (uint32_t i = 0; i < kBatch; ++i) {
                    float a = 0.0f, b = 0.0f;
#pragma unroll
                    for (uint32_t j = 0; j < KT; ++j) {
                        a = fmaf(x[i][j].x, wt[j][0], a);
                        b = fmaf(x[i][j].y, wt[j][1], b);
                    }
                    y[i] = make_float2(silu_fast(a), silu_fast(b));
                }
                if (turn == 0) {
#pragma unroll
                    for (uint32_t i = 0; i < kBatch; ++i) {
                        if (t0 + 8 * i < 16 * rt) *(float2 *)(to + (t0 + 8 * i) * kPitch + 2 * lane) = y[i];
                    }
                    continue;
                }
                float inv[kBatch];
#pragma unroll
                for (uint32_t i = 0; i < kBatch; ++i) inv[i] = fmaf(y[i].y, y[i].y, y[i].x * y[i].x);
#pragma unroll
                for (uint32_t i = 0; i < kBatch; ++i) inv[i] = __builtin_amdgcn_rsqf(wave_sum(inv[i]) + 1e-6f);
#pragma unroll
                for (uint32_t i = 0; i < kBatch; ++i) {
                    const uint32_t t = t0 + 8 * i;
                    if (t >= 16 * rt) break;
                    float a = y[i].x * inv[i], b = y[i].y * inv[i];
                    if (turn == 2) {
                        if (first_of_key && t < R) *(f32x2u *)(keys + (size_t)t * rec_stride) = f32x2u{a, b};
                        // (a key that is not finite would reach every row: 0 in its place)
                        if (!(inv[i] > 0.0f) && __builtin_amdgcn_ballot_w64(!isfinite(a) || !isfinite(b)) != 0) {
                            a = b = 0.0f;
                            if (lane == 0) atomicOr(&lost_s[t >> 5], 1u << (t & 31));
                        }
                    }
                    constexpr float kScale = (float)(1 << kSplitExp);
                    const f16x2 hi = {(_Float16)(a * kScale), (_Float16)(b * kScale)};
                    const f16x2 lo = {(_Float16)(a * kScale - (float)hi.x), (_Float16)(b * kScale - (float)hi.y)};
                    ((f16x2 *)(to + t * kPitch))[lane] = hi;
                    ((f16x2 *)(to + t * kPitch))[64 + lane] = lo;
                }
            }
            __syncthreads();
        }
    };
    if (K == 4) conv(std::integral_constant<uint32_t, 4>{});
    else conv(std::integral_constant<uint32_t, 8>{});
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
    // 4. a wave reads every block of k and q for its state rows; on the way block `mine`
    // of k (even waves) or q meets the blocks of k up to it
    f32x4 kS[RT], qS[RT];
    const uint32_t mine = wave >> 1;
    const bool is_q = (wave & 1) != 0;
    Split own[4];
    {
        const float *ar = (is_q ? xq : xk) + (16 * min(mine, rt - 1) + l16) * kPitch;
#pragma unroll
        for (int s = 0; s < 4; ++s) own[s] = split_row(ar, 32 * s + 8 * g4);
    }
#pragma unroll
    for (int b = 0; b < RT; ++b) {
        kS[b] = qS[b] = f32x4{};
        if ((uint32_t)b >= rt) continue;
        const float *kr = xk + (16 * b + l16) * kPitch, *qr = xq + (16 * b + l16) * kPitch;
        f32x4 acc[2] = {f32x4{}, f32x4{}};
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const Split kf = split_row(kr, 32 * s + 8 * g4);
            kS[b] = mma_split(kf, Sp[s], kS[b]);
            acc[s & 1] = mma_split(own[s], kf, acc[s & 1]);
            qS[b] = mma_split(split_row(qr, 32 * s + 8 * g4), Sp[s], qS[b]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            kS[b][e] = __builtin_amdgcn_ldexpf(kS[b][e], back);
            qS[b][e] = __builtin_amdgcn_ldexpf(qS[b][e], back);
        }
        if (mine < rt && (uint32_t)b <= mine) {
            const uint32_t j = 16 * b + l16;
            const double gj = g_s[j];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t t = 16 * mine + 4 * g4 + e;
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
    u32x2 z[2 * RT];
#pragma unroll
    for (int i = 0; i < 2 * RT; ++i) {
        const size_t at = (size_t)(m.row0 + min(wave + 8 * i, R - 1)) * width + h * kW + 2 * lane;
        if (bf16) z[i].x = *(const u32u *)((const uint16_t *)p.z + at);
        else z[i] = *(const u32x2u *)((const float *)p.z + at);
    }
    __syncthreads();
    // 5. column l16 of the inverse per lane
    if (wave < rt) {
        float *Ab = As + 16 * wave * kPair + 16 * wave;
        f32x4 n[16][4];
#pragma unroll
        for (int t = 1; t < 16; ++t)
#pragma unroll
            for (int i = 0; i < (t + 3) / 4; ++i) n[t][i] = *(const f32x4 *)(Ab + t * kPair + 4 * i);
        float x[16];
#pragma unroll
        for (int t = 0; t < 16; ++t) x[t] = (uint32_t)t == l16 ? 1.0f : 0.0f;
#pragma unroll
        for (int i = 0; i < 15; ++i)
#pragma unroll
            for (int t = i + 1; t < 16; ++t) x[t] = fmaf(n[t][i / 4][i % 4], x[i], x[t]);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (lane < 16) {
#pragma unroll
            for (int t = 0; t < 16; ++t) Ab[t * kPair + lane] = x[t];
        }
    }
    __syncthreads();
    // 6.  A row of d that is not finite is 0 in the products, or it would reach rows that
    // do not see it (0 x inf); bits of such rows are kept per column.
    uint64_t lost = 0;
    auto finite_rows = [&](f32x4 x, int b) __attribute__((always_inline)) {
        const float zero = fmaf(x[0], 0.0f, x[1] * 0.0f) + fmaf(x[2], 0.0f, x[3] * 0.0f);
        if (__builtin_amdgcn_ballot_w64(zero != 0.0f) == 0) return x;  // (NaN is not 0)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool fine = isfinite(x[e]);
            lost |= fine ? 0ull : 1ull << (16 * b + 4 * g4 + e);
            x[e] = fine ? x[e] : 0.0f;
        }
        return x;
    };
    const float qscale = 0.08838834764831845f;  // 1 / sqrt(128)
    f32x4 D[RT];
#pragma unroll
    for (int b = 0; b < RT; ++b) {
        if ((uint32_t)b >= rt) break;
        float *vr = xv + (16 * b + 4 * g4) * kPitch + 16 * wave + l16;
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
        D[b] = finite_rows(mma16(*(const f32x4 *)(Ar + 16 * b), finite_rows(rhs, b), f32x4{}), b);
        o = mma16(*(const f32x4 *)(Pr + 16 * b), D[b], o);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t t = 16 * b + 4 * g4 + e;
            vr[e * kPitch] = o[e] * qscale;
            if (t < R) rec[(size_t)t * p.rec_stride + rec_delta(p) + h * kW + 16 * wave + l16] = D[b][e];
        }
    }
    const uint64_t lost_rows = ((uint64_t)lost_s[1] << 32) | lost_s[0];
    if (__builtin_amdgcn_ballot_w64((lost | lost_rows) != 0) != 0) {
        // the rows that descend from such rows, in the columns where they are
        uint32_t lo = (uint32_t)(lost | lost_rows), hi = (uint32_t)((lost | lost_rows) >> 32);
        lo |= __shfl_xor(lo, 16), hi |= __shfl_xor(hi, 16);
        lo |= __shfl_xor(lo, 32), hi |= __shfl_xor(hi, 32);
        const uint64_t above = ((uint64_t)hi << 32) | lo;
#pragma unroll 1
        for (uint32_t t = g4; t < R; t += 4) {
            if ((anc_s[t] & above) == 0) continue;
            xv[t * kPitch + 16 * wave + l16] = NAN;
            rec[(size_t)t * p.rec_stride + rec_delta(p) + h * kW + 16 * wave + l16] = NAN;
        }
    }
    __syncthreads();
    // 7. RMSNorm without offset, then * silu(z) (native.rs:737-740); rows past the
    // wave's last repeat it
    const float n0 = p.norm[2 * lane], n1 = p.norm[2 * lane + 1];
    constexpr int kOut = 2 * RT < 4 ? 2 * RT : 4;  // rows at a time
#pragma unroll
    for (int i0 = 0; i0 < 2 * RT; i0 += kOut) {
        if (wave + 8 * i0 >= R) break;
        float2 o[kOut];
        float inv[kOut];
#pragma unroll
        for (int i = 0; i < kOut; ++i) {
            o[i] = *(const float2 *)(xv + min(wave + 8 * (i0 + i), R - 1) * kPitch + 2 * lane);
        }
#pragma unroll
        for (int i = 0; i < kOut; ++i) {
            const float variance = wave_sum(fmaf(o[i].y, o[i].y, o[i].x * o[i].x)) / (float)kW;
            if (!isfinite(variance) && lane == 0) atomicOr(p.err_word, kErrNonFiniteVariance);
            inv[i] = 1.0f / sqrtf(variance + p.eps);
        }
#pragma unroll
        for (int i = 0; i < kOut; ++i) {
            const uint32_t t = wave + 8 * (i0 + i);
            if (t >= R) break;
            const u32x2 zi = z[i0 + i];
            const float z0 = bf16 ? bf16lo(zi.x) : __uint_as_float(zi.x), z1 = bf16 ? bf16hi(zi.x) : __uint_as_float(zi.y);
            *(f32x2u *)(p.out + (size_t)(m.row0 + t) * width + h * kW + 2 * lane) =
                f32x2u{o[i].x * inv[i] * n0 * silu_fast(z0), o[i].y * inv[i] * n1 * silu_fast(z1)};
        }
    }
}

template <int RT>
hipError_t launch_head(hipStream_t stream, const GdnTreeParams &p) {
    using T = HeadShape<RT>;
    static_assert(T::kLds + 8192 <= 160 * 1024, "LDS");
    static LdsLimit limit;
    const hipError_t e = limit.allow((const void *)gdn_tree_head_kernel<RT>, T::kLds);
    if (e != hipSuccess) return e;
    SR_LAUNCH("gdn_tree_head_kernel", gdn_tree_head_kernel<RT>, dim3(p.value_heads, p.nseq), dim3(512),
              T::kLds, stream, p);
    return hipGetLastError();
}

struct CommitParams {
    const GdnCommitEntry *entries;  // nullptr: in the arguments
    GdnCommitEntry inline_entries[kGdnCommitInline];
};
static_assert(sizeof(CommitParams) <= 4096, "kernel arguments stay within 4 KiB");

constexpr uint32_t kCommitRows = 8;  // state rows per thread

// S = a S + d k^T along the path: 16-byte units of the state, a thread the same
// columns of kCommitRows rows, then the conv channels' last K - 1 inputs.  grid
// (blocks of the largest entry, entries).  Bound by the state's bytes: 8 layers of 4
// sequences with 32 heads of 128 x 128, 144 MB: 30 us with inputs of its own each call,
// 4.8 TB/s, the rate of a copy (37.5 through the caches).  The rows of a thread share a
// path row's k (eight rows 28.1 us, four 29.5, one 41.7, sixteen 31.3, all with the
// state still in the last cache).
template <typename Unit, typename Unaligned>
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
        const float *state_in = global_from_bits<const float>((uint64_t)e.state_in);
        float *state_out = global_from_bits<float>((uint64_t)e.state_out);
        const float *records = global_from_bits<const float>((uint64_t)e.records);
        // (read and written once each: past the caches)
        Unit S[kCommitRows];
        uint32_t v[kCommitRows];
#pragma unroll
        for (uint32_t i = 0; i < kCommitRows; ++i) {
            v[i] = min(band + bands * i, e.value_dim - 1);
            S[i] = __builtin_nontemporal_load((const Unit *)(state_in + ((size_t)h * e.value_dim + v[i]) * e.key_dim) + c);
        }
        for (uint64_t path = e.path; path != 0; path &= path - 1) {
            const float *rec = records + (size_t)__builtin_ctzll(path) * e.rec_stride;
            const float alpha = rec[h];
            const Unit k = *(const Unaligned *)(rec + e.value_heads * (1 + e.value_dim) + kh * e.key_dim + W * c);
            float delta[kCommitRows];
#pragma unroll
            for (uint32_t i = 0; i < kCommitRows; ++i) delta[i] = rec[e.value_heads + h * e.value_dim + v[i]];
#pragma unroll
            for (uint32_t i = 0; i < kCommitRows; ++i) {
                if constexpr (W == 1) {
                    S[i] = fmaf(delta[i], k, S[i] * alpha);
                } else {
#pragma unroll
                    for (uint32_t j = 0; j < W; ++j) S[i][j] = fmaf(delta[i], k[j], S[i][j] * alpha);
                }
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < kCommitRows; ++i) {
            // (rows past the last repeat it)
            if (band + bands * i < e.value_dim) {
                __builtin_nontemporal_store(S[i], (Unit *)(state_out + ((size_t)h * e.value_dim + v[i]) * e.key_dim) + c);
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
        SR_LAUNCH("gdn_tree_commit_kernel", (gdn_tree_commit_kernel<f32x4, f32x4u>), dim3((uint32_t)blocks[0], count),
                  dim3(256), 0, stream, p);
    } else {
        SR_LAUNCH("gdn_tree_commit_kernel", (gdn_tree_commit_kernel<float, float>), dim3((uint32_t)blocks[1], count),
                  dim3(256), 0, stream, p);
    }
    return hipGetLastError();
}

}  // namespace sr
