// Attention of a tree of drafted tokens over the paged bf16 cache, for gfx950.
//
// Row r of a sequence (context of `ctx` cached tokens, the call's rows appended
// behind it) sees every context token and its own ancestors anc(r), itself
// among them:
//     o_r = sum_j p_j v_j / sum_j p_j,   p_j = 2^(q_r . k_j - m),
//     j < ctx  or  j - ctx in anc(r),
// with q scaled by log2(e) / sqrt(D).  Three launches:
//   tree_prep_kernel     norms and rotates the new rows; k and v go to the
//                        cache in bf16, q to the scratch in the form that the
//                        attention kernel's matrix instructions take, and each
//                        row's ancestors become a 128-bit mask;
//   tree_attn_kernel     one workgroup per (sequence, KV head, 32..128 query
//                        vectors, partition of the keys);
//   tree_combine_kernel  joins the partitions' records (m, l, o), divides,
//                        applies the output gate.
// tree_generic_kernel takes the head widths other than 64, 128 and 256.
#include <algorithm>
#include <type_traits>

#include "sr_device.hpp"
#include "tree_plan.hpp"

namespace sr {

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kTreeSeqs = kTreeLaunchSeqs;
constexpr uint32_t kTreeRows = kTreeLaunchRows;

struct TreeMeta {
    uint32_t slot, ctx, rows;
    uint32_t row0;     // first row in the call's tensors
    uint32_t tile0;    // first q tile of the sequence (attention kernel)
    uint32_t block0;   // first workgroup (attention kernel)
    uint32_t record0;  // first record (attention and combine kernels)
    uint32_t parts;    // partitions of its keys
};

struct TreeCommon {
    uint16_t *k_pages;
    uint16_t *v_pages;
    const int32_t *page_table;
    const void *q;       // raw rows (the gate's values)
    void *q_ops;         // tiles of q operands, or f32 rows for the generic kernel
    uint4 *masks;        // [rows of the call] ancestors of each row
    float *records;
    void *out;
    uint32_t *err_word;
    uint64_t num_pages;
    uint32_t pages_per_seq, log2_page;
    uint32_t flags, heads, kv_heads, head_dim;
    uint32_t nseq;
    alignas(16) TreeMeta meta[kTreeSeqs];
};

struct PrepParams {
    TreeCommon c;
    const void *k;
    const void *v;
    const float *q_norm;
    const float *k_norm;
    const int32_t *positions;
    uint32_t rotary_dim, mrope[3];
    float eps, qscale;
    uint32_t rows;    // of the launch, from c.meta[0].row0 on
    uint32_t parts;   // bf16 parts of q: 3, 2, or 0 for f32 rows
    uint32_t tbl_n;   // page-table entries that the launch writes
    uint32_t tbl_idx[kInlineTable];
    int32_t tbl_val[kInlineTable];
    float denom[kGenericMaxHeadDim / 2];
    alignas(16) uint8_t parent[kTreeRows];  // parent + 1 within the sequence, 0 for a root
};
static_assert(sizeof(PrepParams) <= 4096, "kernel arguments stay within 4 KiB");

constexpr uint32_t kPrepHeads = 1;  // heads of one row per wave
constexpr uint32_t kPrepDims = kGenericMaxHeadDim / 64;

// The sequence of launch row `r` (rows are numbered from the launch's first), or of
// workgroup `r` of the attention kernel.  The arguments of a launch lie in memory far
// away: a wave reads all the sequences' at once, half of one per lane, instead of one
// after another.
template <bool kBlock>
__device__ __forceinline__ TreeMeta find_meta(const TreeCommon &c, uint32_t r) {
    static_assert(kTreeSeqs == 32 && sizeof(TreeMeta) == 32, "two lanes per sequence");
    const uint32_t lane = threadIdx.x & 63;
    const u32x4 x = ((const u32x4 *)c.meta)[lane];  // {slot, ctx, rows, row0} | {tile0, block0, record0, parts}
    const uint32_t begin = kBlock ? x.y : x.w - (uint32_t)__builtin_amdgcn_readfirstlane((int)x.w);
    const bool before = (lane & 1) == (kBlock ? 1u : 0u) && lane / 2 < c.nseq && begin <= r;
    const int at = 2 * (__popcll(__builtin_amdgcn_ballot_w64(before)) - 1);
    auto get = [&](uint32_t v, int i) { return (uint32_t)__builtin_amdgcn_readlane((int)v, i); };
    return TreeMeta{get(x.x, at), get(x.y, at), get(x.z, at), get(x.w, at),
                    get(x.x, at + 1), get(x.y, at + 1), get(x.z, at + 1), get(x.w, at + 1)};
}

// One wave per (row, head): KV heads first, then query heads.  NI: dims per lane,
// d = lane + 64 i.  Bound by latency: arguments, inputs, one exchange through LDS, and
// the fetch of its code, so that heads are waves and not a loop unrolled (4.5 us for 6
// rows of 16 heads; four heads per wave took 7.8).
template <uint32_t NI>
__global__ void __launch_bounds__(256) tree_prep_kernel(const PrepParams p) {
    extern __shared__ float xs_all[];
    const TreeCommon &c = p.c;
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t wave = (uint32_t)wave_index();
    const uint32_t D = c.head_dim;
    float *xs = xs_all + (size_t)wave * kPrepHeads * D;
    const uint32_t all = c.kv_heads + c.heads;
    const uint32_t groups = (all + kPrepHeads - 1) / kPrepHeads;
    const uint32_t item = blockIdx.x * 4 + wave;
    if (blockIdx.x == 0) {
        for (uint32_t i = threadIdx.x; i < p.tbl_n; i += 256) {
            ((int32_t *)c.page_table)[p.tbl_idx[i]] = p.tbl_val[i];
        }
    }
    if (item >= p.rows * groups) return;
    const uint32_t r = item / groups, h0 = item % groups * kPrepHeads;
    // what the wave needs of the arguments' tables, a part per lane
    constexpr uint32_t kPairs = (NI + 1) / 2;  // rotary pairs per lane
    static_assert(kTreeRows == 64 * 16 && kInlineTable == 64, "a lane's part of the tables");
    float denom[kPairs];
#pragma unroll
    for (uint32_t i = 0; i < kPairs; ++i) denom[i] = p.denom[lane + 64 * i];
    const uint32_t tbl_idx = lane < p.tbl_n ? p.tbl_idx[lane] : ~0u;
    const int32_t tbl_val = p.tbl_val[lane];
    const u32x4 parents = ((const u32x4 *)p.parent)[lane];
    const TreeMeta m = find_meta<false>(c, r);
    const uint32_t row = m.row0 + (r - (m.row0 - c.meta[0].row0));
    const uint32_t sr = row - m.row0;  // row of the sequence
    const bool bf16_in = (c.flags & SAFETYRAISE_MI355X_INPUT_BF16) != 0;
    const bool gated = (c.flags & SAFETYRAISE_MI355X_GATED) != 0;
    const bool norm = (c.flags & SAFETYRAISE_MI355X_QK_NORM) != 0;
    const float add = (c.flags & SAFETYRAISE_MI355X_NORM_OFFSET) ? 1.0f : 0.0f;
    const bool interleaved = (c.flags & SAFETYRAISE_MI355X_MROPE_INTERLEAVED) != 0;
    const size_t hs = gated ? 2 * (size_t)D : D;

    const int32_t *pos = p.positions + (size_t)row * 3;
    const int32_t pos0 = pos[0], pos1 = pos[1], pos2 = pos[2];
    // the row's page: its entry may be among those that this launch writes
    const uint32_t tok = m.ctx + sr;
    const uint32_t entry = m.slot * c.pages_per_seq + (tok >> c.log2_page);
    int32_t page = c.page_table[entry];
    // all of the wave's values are requested before any is used
    float x[kPrepHeads][NI], v[kPrepHeads][NI];
#pragma unroll
    for (uint32_t u = 0; u < kPrepHeads; ++u) {
        const uint32_t hh = min(h0 + u, all - 1);
        const bool kv = hh < c.kv_heads;
        const void *src = kv ? p.k : c.q;
        const size_t at = kv ? ((size_t)row * c.kv_heads + hh) * D
                             : ((size_t)row * c.heads + (hh - c.kv_heads)) * hs;
#pragma unroll
        for (uint32_t i = 0; i < NI; ++i) {
            const uint32_t d = min(lane + 64 * i, D - 1);
            x[u][i] = load_act_nb(src, at + d, bf16_in);
            v[u][i] = kv ? load_act_nb(p.v, at + d, bf16_in) : 0.0f;
        }
    }
    const uint64_t own = __builtin_amdgcn_ballot_w64(tbl_idx == entry);
    if (own != 0) page = __builtin_amdgcn_readlane(tbl_val, __builtin_ctzll(own));
    if (h0 == 0) {
        // the ancestors, walked from the row to its root
        uint32_t w[4] = {0, 0, 0, 0};
        const uint32_t first = m.row0 - c.meta[0].row0;
        for (uint32_t a = sr + 1; a != 0;) {
            const uint32_t b = a - 1;
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) w[k] |= (b >> 5) == k ? 1u << (b & 31) : 0u;
            const uint32_t at = first + b, word = at / 4 % 4;
            uint32_t four = 0;
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) {
                const uint32_t x = (uint32_t)__builtin_amdgcn_readlane((int)parents[k], (int)(at / 16));
                four = word == k ? x : four;
            }
            a = (four >> (at % 4 * 8)) & 0xffu;
        }
        if (lane == 0) c.masks[row] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    // the rotation, while the values are on their way
    const uint32_t half = p.rotary_dim / 2;
    float sn[kPairs], cs[kPairs];
#pragma unroll
    for (uint32_t i = 0; i < kPairs; ++i) {
        const int axis = rope_axis(lane + 64 * i, p.mrope, interleaved);
        sn[i] = 0.0f;
        cs[i] = 1.0f;
        if (lane + 64 * i < half) {
            sincosf((float)(axis == 0 ? pos0 : axis == 1 ? pos1 : pos2) / denom[i], &sn[i], &cs[i]);
        }
    }
    if (norm) {
#pragma unroll
        for (uint32_t u = 0; u < kPrepHeads; ++u) {
            const bool kv = h0 + u < c.kv_heads;
            const float *w = kv ? p.k_norm : p.q_norm;
            float ss = 0.0f;
#pragma unroll
            for (uint32_t i = 0; i < NI; ++i) {
                if (lane + 64 * i < D) ss = fmaf(x[u][i], x[u][i], ss);
            }
            ss = sum64(ss);
            const float variance = ss / (float)D;
            if (!isfinite(variance) && lane == 0) atomicOr(c.err_word, kErrNonFiniteVariance);
            const float inv = 1.0f / sqrtf(variance + p.eps);
#pragma unroll
            for (uint32_t i = 0; i < NI; ++i) {
                x[u][i] = x[u][i] * inv * (w[min(lane + 64 * i, D - 1)] + add);
            }
        }
    }
#pragma unroll
    for (uint32_t u = 0; u < kPrepHeads; ++u)
#pragma unroll
        for (uint32_t i = 0; i < NI; ++i) {
            if (lane + 64 * i < D) xs[u * D + lane + 64 * i] = x[u][i];
        }
    // (LDS operations of one wave are performed in order)
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    // rotate-half over the first rotary_dim dims (math.rs:52-99)
#pragma unroll
    for (uint32_t k = 0; k < kPairs; ++k) {
        const uint32_t i = lane + 64 * k;
        if (i >= half) continue;
#pragma unroll
        for (uint32_t u = 0; u < kPrepHeads; ++u) {
            const float left = xs[u * D + i], right = xs[u * D + i + half];
            xs[u * D + i] = left * cs[k] - right * sn[k];
            xs[u * D + i + half] = right * cs[k] + left * sn[k];
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    const uint32_t group = c.heads / c.kv_heads;
    bool finite = true;
#pragma unroll
    for (uint32_t u = 0; u < kPrepHeads; ++u) {
        const uint32_t hh = h0 + u;
        if (hh >= all) break;
        const float *y = xs + u * D;
        if (hh < c.kv_heads) {
            const size_t base =
                ((((size_t)hh * c.num_pages + page) << c.log2_page) + (tok & ((1u << c.log2_page) - 1))) * D;
            // A value that is not finite would reach rows that do not see it (0 x inf in the
            // products): such a row gets a key of NaN, which its own descendants'
            // scores take up and the others' masks drop, and a value of 0.
            uint16_t kb[NI], vb[NI];
            bool fine = true;
#pragma unroll
            for (uint32_t i = 0; i < NI; ++i) {
                kb[i] = f32_to_bf16(y[min(lane + 64 * i, D - 1)]);
                vb[i] = f32_to_bf16(v[u][i]);
                fine = fine && isfinite(bf16_to_f32(kb[i])) && isfinite(bf16_to_f32(vb[i]));
            }
            const bool lost = __builtin_amdgcn_ballot_w64(!fine) != 0;
            finite = finite && !lost;
#pragma unroll
            for (uint32_t i = 0; i < NI; ++i) {
                const uint32_t d = lane + 64 * i;
                if (d >= D) continue;
                c.k_pages[base + d] = lost ? (uint16_t)0x7fc0u : kb[i];
                c.v_pages[base + d] = lost ? (uint16_t)0u : vb[i];
            }
            continue;
        }
        const uint32_t head = hh - c.kv_heads;
        if (p.parts == 0) {
            float *dst = (float *)c.q_ops + ((size_t)(row - c.meta[0].row0) * c.heads + head) * D;
#pragma unroll
            for (uint32_t i = 0; i < NI; ++i) {
                const uint32_t d = lane + 64 * i;
                if (d < D) dst[d] = y[d] * p.qscale;
            }
            continue;
        }
        // q operands: tiles of 32 query vectors (vector = row * group + head of
        // its KV head), [part][step of 16 dims][lane][8], as a lane of the
        // attention kernel holds them: vector lane & 31, dims 16 step + 8 (lane
        // >> 5) + 0..7.  The parts sum to q: bf16 keeps 8 bits of it each.
        const uint32_t kvh = head / group;
        const uint32_t vec = sr * group + head % group;
        const uint32_t tiles = (m.rows * group + 31) / 32;
        const uint32_t steps = D / 16;
        const size_t tile = m.tile0 + (size_t)kvh * tiles + vec / 32;
        if (lane < D / 8) {
            float a[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) a[j] = y[8 * lane + j] * p.qscale;
            for (uint32_t part = 0; part < p.parts; ++part) {
                u32x4 w;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    w[j] = pack_bf16x2(a[2 * j], a[2 * j + 1]);
                    a[2 * j] -= bf16lo(w[j]);
                    a[2 * j + 1] -= bf16hi(w[j]);
                }
                const size_t at = ((tile * p.parts + part) * steps + lane / 2) * 64 +
                                  ((lane & 1) * 32 + vec % 32);
                ((u32x4 *)c.q_ops)[at] = w;
            }
        }
    }
    if (__builtin_amdgcn_ballot_w64(!finite) != 0 && lane == 0) {
        atomicOr(c.err_word, kErrNonFiniteKv);
    }
}

__device__ __forceinline__ bool mask_bit(const uint4 &m, uint32_t b) {
    const uint32_t w = b < 64 ? (b < 32 ? m.x : m.y) : (b < 96 ? m.z : m.w);
    return (w >> (b & 31)) & 1u;
}

__device__ __forceinline__ void store_out(const TreeCommon &c, size_t at, float y) {
    if (c.flags & SAFETYRAISE_MI355X_OUTPUT_BF16) {
        ((uint16_t *)c.out)[at] = f32_to_bf16(y);
    } else {
        ((float *)c.out)[at] = y;
    }
}

// Any head width: one wave per (row, query head) over the visible keys in tiles
// of 64, a key per lane for the scores and a dim per lane for the sums.  Bound by its
// loads: every row and head reads its keys again, a lane's key value by value.  Four
// sequences of 24 rows behind 1024..16384 tokens, 32 heads over 8 of width 80: 9.2 ms,
// where the keys and values, read once, are 16 us.  It is there for widths that no
// configuration of this framework has.
__global__ void __launch_bounds__(64) tree_generic_kernel(const TreeCommon c) {
    extern __shared__ float sh[];
    const uint32_t D = c.head_dim, lane = threadIdx.x;
    float *qs = sh, *ps = sh + D;
    const uint32_t head = blockIdx.x, r = blockIdx.y;
    const TreeMeta m = find_meta<false>(c, r);
    const uint32_t sr = r - (m.row0 - c.meta[0].row0);
    const size_t row = (size_t)m.row0 + sr;
    const float *q = (const float *)c.q_ops + ((size_t)r * c.heads + head) * D;
    for (uint32_t d = lane; d < D; d += 64) qs[d] = q[d];
    const uint4 mask = c.masks[row];
    __syncthreads();
    const uint32_t kvh = head / (c.heads / c.kv_heads);
    const uint32_t keys = m.ctx + sr + 1;
    const int32_t *table = c.page_table + (size_t)m.slot * c.pages_per_seq;
    const uint32_t pmask = (1u << c.log2_page) - 1;
    auto base = [&](uint32_t t) {
        return ((((size_t)kvh * c.num_pages + table[t >> c.log2_page]) << c.log2_page) + (t & pmask)) * D;
    };
    float m_run = -INFINITY, l_run = 0.0f;
    float o[kPrepDims] = {};
    for (uint32_t t0 = 0; t0 < keys; t0 += 64) {
        const uint32_t j = t0 + lane;
        float score = -INFINITY;
        if (j < keys && (j < m.ctx || mask_bit(mask, j - m.ctx))) {
            const uint16_t *k = c.k_pages + base(j);
            float dot = 0.0f;
            for (uint32_t d = 0; d < D; ++d) dot = fmaf(qs[d], bf16_to_f32(k[d]), dot);
            score = dot;
        }
        const float mx = fmaxf(m_run, max64(score));
        // (no key so far: every weight is 0)
        const float ref = mx == -INFINITY ? 0.0f : mx;
        const float prior = exp2f(m_run - ref);
        const float pj = exp2f(score - ref);
        l_run = l_run * prior + sum64(pj);
        m_run = mx;
        ps[lane] = pj;
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < kPrepDims; ++i) o[i] *= prior;
        const uint32_t n = min(64u, keys - t0);
        for (uint32_t k = 0; k < n; ++k) {
            const float pk = ps[k];
            if (pk == 0.0f) continue;  // wave-uniform: a masked key's value is not read
            const uint16_t *v = c.v_pages + base(t0 + k);
#pragma unroll
            for (uint32_t i = 0; i < kPrepDims; ++i) {
                const uint32_t d = lane + 64 * i;
                if (d < D) o[i] = fmaf(pk, bf16_to_f32(v[d]), o[i]);
            }
        }
        __syncthreads();
    }
    const bool bf16_in = (c.flags & SAFETYRAISE_MI355X_INPUT_BF16) != 0;
    const bool gated = (c.flags & SAFETYRAISE_MI355X_GATED) != 0;
    const size_t gate = (row * c.heads + head) * 2 * (size_t)D + D;
    const float inv = 1.0f / l_run;
#pragma unroll
    for (uint32_t i = 0; i < kPrepDims; ++i) {
        const uint32_t d = lane + 64 * i;
        if (d >= D) continue;
        float y = o[i] * inv;
        if (gated) y *= ref_sigmoid(load_act(c.q, gate + d, bf16_in));
        store_out(c, (row * c.heads + head) * D + d, y);
    }
}


// ---------------------------------------------------------------------------
// The MFMA kernel: head widths 64, 128 and 256.
//
// S^T = K Q^T and O^T += V^T P^T with v_mfma_f32_32x32x16_bf16 on the cache's own
// bf16 values: keys (dims) are the rows of the accumulators and a lane's column
// is one query vector, so its maximum takes one exchange between the two halves
// of the wave, and the probabilities are in the layout of the next product's
// operand where they are made.  q and p are split into bf16 parts that sum to
// them: three of each (24 bits) for an f32 result; for a bf16 result two of q (its
// rounding is multiplied by the scores' size) and one of p, whose rounding is to the
// values that it weighs what the result's is to the result.  Products and sums are f32.
//
// A workgroup has up to 4 x 32 query vectors and 32 KB stages of kKeys keys: a
// wave takes one of the vector groups and 32 keys of a stage.  Stages come
// straight into LDS (global_load_lds, 16 bytes per lane), kAhead ahead, one
// barrier per stage.  K rows have their 16-byte units swapped by the row's index, so
// that the operand reads (ds_read_b128) meet no bank twice; V rows are read as they
// are, a lane the same D / 32 dims of 8 keys, and v_perm_b32 pairs the keys' values
// for the product.  The scores of stage k run beside the softmax and P V of stage
// k - 1.
//
// What bounds it: the matrix pipe.  Eight sequences of 16..32 rows behind 1024..16384
// tokens, 32 heads over 8 of width 128, f32: 122 us (median of a kernel trace, one pass
// after another), of which 89 are its products at the 1205 TFLOP/s that a large bf16
// matrix product reaches, and 79 the loads alone.  Four of 20..64 rows behind 8192..65536
// tokens at width 256, bf16: 251 us; products 184, loads 74.  (Without its loads the
// kernel takes 93 and 226 us, with the loads alone 79 and 99.)
// ---------------------------------------------------------------------------
constexpr uint32_t kStages = 4;
constexpr uint32_t kAhead = 2;  // stages on their way; one more may still be read by late waves
constexpr uint32_t kStageBytes = 32768;
constexpr float kLazy = 8.0f;  // log2 growth of the maximum before sums are rescaled

typedef __attribute__((address_space(3))) unsigned char lds_byte;

template <int D, bool kF32>
struct TreeShape {
    static constexpr int VG = (int)tree_vector_waves(D);  // waves of query vectors
    static constexpr int kKeys = 8192 / D;      // keys per stage
    static constexpr int KG = kKeys / 32;       // waves over the keys of a stage
    static constexpr int NW = VG * KG;
    static constexpr int kThreads = 64 * NW;
    static constexpr int QP = kF32 ? 3 : 2;     // bf16 parts of q
    static constexpr int PP = kF32 ? 3 : 1;     // of the probabilities
    // steps whose last part of q is kept in LDS, where the registers do not hold it: a
    // spilled register's reload would wait for the stages on their way
    static constexpr int kFarSteps = kF32 && D == 128 ? 4 : 0;
    static constexpr size_t kFarAt = kStages * kStageBytes + kTreePageSlots * 4;
    static constexpr size_t kLds = kFarAt + VG * kFarSteps * 1024;
};

__device__ __forceinline__ float half_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_int(x), __float_as_int(x), false, false);
    return fmaxf(__int_as_float(r[0]), __int_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_int(x), __float_as_int(x), false, false);
    return __int_as_float(r[0]) + __int_as_float(r[1]);
}
// The unit (16 bytes) at which logical unit u of key row r is stored.
template <int D>
__device__ __forceinline__ uint32_t k_unit(uint32_t r, uint32_t u) {
    return D == 64 ? u ^ ((r >> 1) & 7) : u ^ (r & 15);
}
// A lane's dims of one key row of V: D / 32 bf16 values, dims D / 32 i .. of lane i.
// (A vector type, read as such: the compiler takes reads through it, unlike reads of
// integers or structs, for apart from the stages on their way into LDS and does not
// wait for those.)
template <int NT>
struct VRowOf {
    typedef __bf16 type __attribute__((ext_vector_type(NT)));
};
template <int NT>
using VRow = typename VRowOf<NT>::type;
// Operand of O^T += V^T P^T for tile t (row i: dim NT i + t) from 8 keys' rows: the
// keys' values of that dim, two to a register.
template <int NT>
__device__ __forceinline__ bf16x8 v_operand(const VRow<NT> (&v)[8], int t) {
    struct Words {
        uint32_t w[NT / 2];
    };
    u32x4 x;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        x[j] = __builtin_amdgcn_perm(__builtin_bit_cast(Words, v[2 * j + 1]).w[t / 2],
                                     __builtin_bit_cast(Words, v[2 * j]).w[t / 2],
                                     (t & 1) ? 0x07060302u : 0x05040100u);
    }
    return __builtin_bit_cast(bf16x8, x);
}

template <int D, bool kF32>
__global__ __launch_bounds__((TreeShape<D, kF32>::kThreads)) void tree_attn_kernel(const TreeCommon c) {
    using T = TreeShape<D, kF32>;
    constexpr int VG = T::VG;
    constexpr int NS = D / 16, NT = D / 32;
    constexpr int CH = D / 8;             // 16-byte units per row
    constexpr int RPI = 64 / CH;          // rows per load instruction
    constexpr int kLoads = 16 / T::NW > 0 ? 16 / T::NW : 1;  // of K, and of V, per wave and stage
    static_assert(kLoads * T::NW == 16, "a stage's loads are shared out evenly");
    extern __shared__ __align__(16) unsigned char lds[];
    int32_t *pids = (int32_t *)(lds + kStages * kStageBytes);

    const uint32_t tid = threadIdx.x, lane = tid & 63;
    const uint32_t wave = (uint32_t)wave_index();
    // (wave i runs on SIMD i % 4: the waves of one vector group on different ones, so
    // that few vectors still keep all four busy)
    const uint32_t vg = wave / T::KG, kg = wave % T::KG;
    const TreeMeta m = find_meta<true>(c, blockIdx.x);
    const uint32_t group = c.heads / c.kv_heads;
    const uint32_t nvec = m.rows * group;
    const uint32_t slices = (nvec + 32 * VG - 1) / (32 * VG);
    // blocks of a sequence: groups of 8 (partition, KV head) units, slice by
    // slice, so that the slices of a unit run on one XCD (block i runs on XCD i
    // % 8) at about the same time and share its L2
    const uint32_t units = m.parts * c.kv_heads;
    const uint32_t at = blockIdx.x - m.block0;
    const uint32_t unit0 = at / (8 * slices) * 8;
    const uint32_t width = min(8u, units - unit0);
    const uint32_t unit = unit0 + (at - unit0 * slices) % width;
    const uint32_t slice = (at - unit0 * slices) / width;
    const uint32_t kvh = unit % c.kv_heads;
    const uint32_t part = unit / c.kv_heads;
    const uint32_t part_keys = tree_part_keys(m.ctx + m.rows, m.parts, D);
    const uint32_t key_begin = part * part_keys;
    const uint32_t key_end = min(key_begin + part_keys, m.ctx + m.rows);  // > key_begin
    const uint32_t steps = (key_end - key_begin + T::kKeys - 1) / T::kKeys;

    // this wave's query vectors (a wave without any only loads keys).  They are
    // requested ahead of the page ids, so that nothing of theirs is on its way when the
    // stages are: the compiler would wait for those too, in every step
    const uint32_t col = lane & 31, h = lane >> 5;
    const uint32_t tiles = (nvec + 31) / 32;
    const uint32_t tile = slice * VG + vg;
    const bool live = tile < tiles;
    const uint32_t vec = min(tile * 32 + col, nvec - 1);
    const uint32_t row = vec / group;  // of the sequence
    bf16x8 q[T::QP][NS];
    unsigned char *far = lds + T::kFarAt + vg * (T::kFarSteps * 1024) + lane * 16;
    {
        const u32x4 *src = (const u32x4 *)c.q_ops +
                           (m.tile0 + (size_t)kvh * tiles + min(tile, tiles - 1)) * T::QP * NS * 64 + lane;
#pragma unroll
        for (int p = 0; p < T::QP; ++p)
#pragma unroll
            for (int st = 0; st < NS; ++st) {
                if (p < T::QP - 1 || st < NS - T::kFarSteps) q[p][st] = __builtin_bit_cast(bf16x8, src[(p * NS + st) * 64]);
            }
        if constexpr (T::kFarSteps > 0) {
            for (int st = (int)kg; st < T::kFarSteps; st += T::KG) {
                *(u32x4 *)(far + st * 1024) = src[((T::QP - 1) * NS + NS - T::kFarSteps + st) * 64];
            }
        }
    }
    uint4 mask = c.masks[m.row0 + row];

    // page ids of the partition
    const uint32_t lpt = c.log2_page, pmask = (1u << lpt) - 1;
    const uint32_t first_page = key_begin >> lpt;
    const uint32_t npages = ((key_end - 1) >> lpt) - first_page + 1;
    const int32_t *table = c.page_table + (size_t)m.slot * c.pages_per_seq + first_page;
    for (uint32_t i = tid; i < npages; i += T::kThreads) pids[i] = table[i];
#pragma unroll
    for (int p = 0; p < T::QP; ++p)
#pragma unroll
        for (int st = 0; st < NS; ++st) {
            if (p < T::QP - 1 || st < NS - T::kFarSteps) asm volatile("" : "+v"(q[p][st]));  // arrived
        }
    asm volatile("" : "+v"(mask.x), "+v"(mask.y), "+v"(mask.z), "+v"(mask.w));
    const uint64_t mask_lo = ((uint64_t)mask.y << 32) | mask.x, mask_hi = ((uint64_t)mask.w << 32) | mask.z;
    __syncthreads();

    // stage k into its buffer: load i of a wave covers rows RPI (wave + NW i) .. of K
    // and of V.  Rows past the last key load it again: they are masked, and finite.
    const unsigned char *k_head = (const unsigned char *)c.k_pages + (((size_t)kvh * c.num_pages) << lpt) * (D * 2);
    const unsigned char *v_head = (const unsigned char *)c.v_pages + (((size_t)kvh * c.num_pages) << lpt) * (D * 2);
    const uint32_t lrow = lane / CH, lunit = lane % CH;
    // a wave's page ids of the next stage to issue, read from LDS a stage ahead
    int32_t ahead[kLoads];
    auto page_ids = [&](uint32_t k) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const uint32_t key0 = key_begin + k * T::kKeys + RPI * (wave + T::NW * i);
            ahead[i] = pids[(min(key0, key_end - 1) >> lpt) - first_page];
        }
    };
    auto to_lds = [](const unsigned char *from, unsigned char *to) __attribute__((always_inline)) {
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from,
                                         (__attribute__((address_space(3))) void *)to, 16, 0, 0);
    };
    auto issue = [&](uint32_t k) __attribute__((always_inline)) {
        unsigned char *buf = lds + (k % kStages) * kStageBytes;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const uint32_t r0 = RPI * (wave + T::NW * i);
            const uint32_t key0 = key_begin + k * T::kKeys + r0;
            const uint32_t page = (uint32_t)__builtin_amdgcn_readfirstlane(ahead[i]);
            unsigned char *to = buf + r0 * (D * 2);
            if (key0 + RPI <= key_end) {
                // (rows r0 .. are in one page: a page holds at least 16 keys)
                const size_t at = (((size_t)page << lpt) + (key0 & pmask)) * (D * 2);
                const uint32_t r = r0 + lrow;
                to_lds(k_head + at + (lrow * (D * 2) + k_unit<D>(r, lunit) * 16), to);
                to_lds(v_head + at + (lrow * (D * 2) + lunit * 16), to + kStageBytes / 2);
            } else {
                const uint32_t base = min(key0, (key_end - 1) & ~(uint32_t)(RPI - 1));
                const uint32_t tok = min(base + lrow, key_end - 1), r = r0 + lrow;
                const size_t at = (((size_t)page << lpt) + (tok & pmask)) * (D * 2);
                to_lds(k_head + at + k_unit<D>(r, lunit) * 16, to);
                to_lds(v_head + at + lunit * 16, to + kStageBytes / 2);
            }
        }
        page_ids(k + 1);
    };
    page_ids(0);
#pragma unroll 1
    for (uint32_t k = 0; k < kAhead; ++k) {
        if (k < steps) issue(k);
    }

    f32x16 o[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) o[t] = f32x16{};
    float m_run = -INFINITY, l_run = 0.0f;
    // the beginning of step k
    auto enter = [&](uint32_t k) __attribute__((always_inline)) {
        // this wave's loads of stage k have landed when at most those of the
        // stages after it are outstanding; its reads of the stages before are done (the
        // products that took them have waited for them, wherever the compiler put those)
        constexpr int kPer = 2 * kLoads < 64 ? 2 * kLoads : 63;
        if (k + 1 < steps) __builtin_amdgcn_s_waitcnt(0x0070 | (kPer & 15) | ((kPer >> 4) << 14));
        else __builtin_amdgcn_s_waitcnt(0x0070);
        // every wave's loads of stage k have landed, and the buffer of stage k - 2
        // has been read
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (k + kAhead < steps) issue(k + kAhead);
    };
    // a wave has its SIMD to itself
    constexpr bool kAlone = T::NW <= 4;
    // steps st0 .. st1 - 1 of the scores of stage k; a wave alone keeps two chains of
    // products going
    constexpr int kChains = kAlone ? 2 : 1;
    auto scores = [&](uint32_t k, int st0, int st1, f32x16 (&acc)[kChains]) __attribute__((always_inline)) {
        const unsigned char *kt = lds + (k % kStages) * kStageBytes + 32 * kg * (D * 2);
#pragma unroll
        for (int st = st0; st < st1; ++st) {
            const bf16x8 a = *(const bf16x8 *)(kt + col * (D * 2) + k_unit<D>(col, 2 * st + h) * 16);
#pragma unroll
            for (int p = 0; p < T::QP; ++p) {
                f32x16 &x = acc[(st + p) % kChains];
                const bool near = p < T::QP - 1 || st < NS - T::kFarSteps;
                const bf16x8 b = near ? q[p][st] : *(const bf16x8 *)(far + (st - (NS - T::kFarSteps)) * 1024);
                x = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, x, 0, 0, 0);
            }
        }
    };
    // One stage's softmax and P V, with the scores of the next beside them: the
    // matrix instructions run while the vector ones are issued.
    f32x16 held;  // scores of stage k - 1
    auto advance = [&](uint32_t k, auto next_of) __attribute__((always_inline)) {
        constexpr bool kNext = decltype(next_of)::value;
        const uint32_t key0 = key_begin + (k - 1) * T::kKeys + 32 * kg;
        if (key0 + 32 > m.ctx) {
            // bits of the wave's 32 keys: context keys, and the row's ancestors
            uint32_t w;
            if (key0 >= m.ctx) {
                const uint32_t b = key0 - m.ctx;  // < 128
                const uint64_t lo = b < 64 ? mask_lo : mask_hi, hi = b < 64 ? mask_hi : 0;
                const uint32_t sh = b & 63;
                w = (uint32_t)(lo >> sh) | (sh > 32 ? (uint32_t)(hi << (64 - sh)) : 0u);
            } else {
                const uint32_t n = m.ctx - key0;  // 1..31 context keys
                w = ((uint32_t)mask_lo << n) | ((1u << n) - 1);
            }
            w >>= 4 * h;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                if (!((w >> (8 * (i >> 2) + (i & 3))) & 1u)) held[i] = -INFINITY;
            }
        }
        f32x16 acc[kChains] = {};
        if constexpr (kNext) scores(k, 0, NS / 4, acc);
        // d = s - reference.  The reference only moves when the maximum outgrows it by
        // kLazy (or at the first visible key): sums and outputs are the same for any
        // common shift, and rescaling is rare.  (The maximum is of differences: of
        // the matrix products themselves it would cost a canonicalisation each.)
        const float ref = m_run == -INFINITY ? 0.0f : m_run;
        float d[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) d[i] = held[i] - ref;
        float mx = fmaxf(fmaxf(fmaxf(d[0], d[1]), d[2]), fmaxf(fmaxf(d[3], d[4]), d[5]));
        mx = fmaxf(fmaxf(mx, d[6]), fmaxf(fmaxf(d[7], d[8]), d[9]));
        mx = fmaxf(fmaxf(mx, d[10]), fmaxf(fmaxf(d[11], d[12]), d[13]));
        mx = half_max(fmaxf(fmaxf(mx, d[14]), d[15]));
        const bool move = mx > kLazy || (m_run == -INFINITY && mx > -INFINITY);
        if (__builtin_amdgcn_ballot_w64(move) != 0) {
            const float next = move ? ref + mx : m_run;
            const float scale = move ? __builtin_amdgcn_exp2f(m_run - next) : 1.0f;
            const bool summed = move && m_run > -INFINITY;  // (else there is nothing yet to rescale)
            m_run = next;
            const float moved = next == -INFINITY ? 0.0f : next - ref;
            l_run *= scale;
            if (__builtin_amdgcn_ballot_w64(summed) == 0) {
                // o is 0
            } else if constexpr (kAlone) {
                // a wave with the whole register file keeps o in accumulation registers;
                // multiplied there, or the compiler moves all of it back and forth in
                // every step.  (The wait: the last products' results, 18 cycles.)
                asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        float x;
                        asm volatile("v_accvgpr_read_b32 %1, %0\n\ts_nop 1\n\tv_mul_f32 %1, %1, %2\n\ts_nop 1\n\t"
                                     "v_accvgpr_write_b32 %0, %1\n\ts_nop 1"
                                     : "+a"(o[t][i]), "=&v"(x)
                                     : "v"(scale));
                    }
                asm volatile("s_nop 7" ::: "memory");
            } else {
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[t][i] *= scale;
            }
            // (from the differences: the scores' registers are free by now)
#pragma unroll
            for (int i = 0; i < 16; ++i) d[i] -= moved;
        }
        // V rows of the wave's keys: lane (i, h) reads its dims of keys 16 st + 4 h +
        // {0..3, 8..11}, those of its probabilities
        const unsigned char *vt = lds + ((k - 1) % kStages) * kStageBytes + kStageBytes / 2 +
                                  (32 * kg + 4 * h) * (D * 2) + col * (NT * 2);
        float sum[4] = {};
#pragma unroll
        for (int st = 0; st < 2; ++st) {
            VRow<NT> v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[j] = *(const VRow<NT> *)(vt + (16 * st + (j & 3) + 8 * (j >> 2)) * (D * 2));
            }
            if constexpr (kNext) scores(k, NS / 4 + st * 3 * NS / 8, NS / 4 + (st + 1) * 3 * NS / 8, acc);
            u32x4 w[T::PP];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float a = __builtin_amdgcn_exp2f(d[8 * st + 2 * j]);
                float b = __builtin_amdgcn_exp2f(d[8 * st + 2 * j + 1]);
                if constexpr (kF32) sum[j] += a + b;
#pragma unroll
                for (int p = 0; p < T::PP; ++p) {
                    w[p][j] = pack_bf16x2(a, b);
                    a -= bf16lo(w[p][j]);
                    b -= bf16hi(w[p][j]);
                }
                // (the sum is over the probabilities that the product uses)
                if constexpr (!kF32) sum[j] += bf16lo(w[0][j]) + bf16hi(w[0][j]);
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const bf16x8 a = v_operand<NT>(v, t);
#pragma unroll
                for (int p = 0; p < T::PP; ++p) {
                    o[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, __builtin_bit_cast(bf16x8, w[p]), o[t], 0, 0, 0);
                }
            }
        }
        l_run += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        if constexpr (kNext) held = kChains == 2 ? acc[0] + acc[kChains - 1] : acc[0];
    };
    // stage k's scores run in step k, its softmax and P V in step k + 1
    if (!live) {
        for (uint32_t k = 0; k < steps; ++k) enter(k);
    } else {
        enter(0);
        {
            f32x16 acc[kChains] = {};
            scores(0, 0, NS, acc);
            held = kChains == 2 ? acc[0] + acc[kChains - 1] : acc[0];
        }
        for (uint32_t k = 1; k < steps; ++k) {
            enter(k);
            advance(k, std::true_type{});
        }
        // (the last stage may end before the wave's keys)
        if (key_begin + (steps - 1) * T::kKeys + 32 * kg < key_end) advance(steps, std::false_type{});
    }
    // The waves over the keys are joined through LDS, a record per query vector and wave
    // in the place of the stages: {m, l, -, -, o}.  Then each of them finishes its share
    // of the vectors, a row at a time and as loops: a launch begins with no code in the
    // instruction cache, and code that runs once costs its fetch.
    constexpr uint32_t kRecord = tree_record_floats(D);
    float *joined = (float *)lds + (size_t)vg * 32 * kRecord;  // of wave (vg, kg 0)
    constexpr uint32_t kNextWave = VG * 32 * kRecord;
    static_assert(sizeof(float) * kNextWave * T::KG <= T::kLds, "records fit the stages");
    const float l = half_sum(l_run);
    __syncthreads();
    if (live) {
        float *w = joined + kg * kNextWave + col * kRecord;
        if (h == 0) *(float2 *)w = make_float2(m_run, l);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float *dst = w + 4 + NT * (8 * (i >> 2) + 4 * h + (i & 3));
            if constexpr (NT == 2) {
                *(float2 *)dst = make_float2(o[0][i], o[1][i]);
            } else {
#pragma unroll
                for (int t = 0; t < NT; t += 4) *(float4 *)(dst + t) = make_float4(o[t][i], o[t + 1][i], o[t + 2][i], o[t + 3][i]);
            }
        }
    }
    __syncthreads();
    if (!live) return;
    const bool gated = (c.flags & SAFETYRAISE_MI355X_GATED) != 0;
    const bool bf16_in = (c.flags & SAFETYRAISE_MI355X_INPUT_BF16) != 0;
    const bool out16 = (c.flags & SAFETYRAISE_MI355X_OUTPUT_BF16) != 0;
    constexpr uint32_t kRows = 256 / D;  // rows at a time: a lane has 4 dims of one
    constexpr uint32_t kShare = 32 / T::KG;
    const uint32_t d = 4 * (lane % (D / 4));
    const uint32_t left = min(32u, nvec - tile * 32);
#pragma unroll 1
    for (uint32_t i = kg * kShare + lane / (D / 4); i < min(left, (kg + 1) * kShare); i += kRows) {
        const float *w = joined + i * kRecord;
        float2 ml = *(const float2 *)w;
        f32x4 y = *(const f32x4 *)(w + 4 + d);
        if constexpr (T::KG > 1) {
            float mx = ml.x;
#pragma unroll
            for (int g = 1; g < T::KG; ++g) mx = fmaxf(mx, w[g * kNextWave]);
            const float ref = mx == -INFINITY ? 0.0f : mx;
            const float first = __builtin_amdgcn_exp2f(ml.x - ref);
            ml = make_float2(mx, ml.y * first);
            y *= first;
#pragma unroll
            for (int g = 1; g < T::KG; ++g) {
                const float2 next = *(const float2 *)(w + g * kNextWave);
                const float weight = __builtin_amdgcn_exp2f(next.x - ref);
                ml.y = fmaf(next.y, weight, ml.y);
                y += *(const f32x4 *)(w + g * kNextWave + 4 + d) * weight;
            }
        }
        const uint32_t v = tile * 32 + i, r = v / group, head = kvh * group + v % group;
        if (c.records != nullptr) {
            float *rec = c.records + ((size_t)m.record0 + ((size_t)r * c.heads + head) * m.parts + part) * kRecord;
            if (d == 0) *(float2 *)rec = ml;
            *(f32x4 *)(rec + 4 + d) = y;
            continue;
        }
        const size_t out_row = (size_t)(m.row0 + r) * c.heads + head;
        y *= 1.0f / ml.y;
        if (gated) {
            const size_t gate = out_row * 2 * D + D + d;
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] *= ref_sigmoid(load_act(c.q, gate + j, bf16_in));
        }
        if (out16) *(uint2 *)((uint16_t *)c.out + out_row * D + d) = make_uint2(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]));
        else *(f32x4 *)((float *)c.out + out_row * D + d) = y;
    }
}

// Joins the records of a (row, head): a wave each, all the loads of eight records
// in flight.  Bound by the records' bytes (32 MB in 9.6 us at width 256).
template <int D>
__global__ void __launch_bounds__(256) tree_combine_kernel(const TreeCommon c, uint32_t rows) {
    constexpr int EPL = D / 64, kBatch = 8;
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t w = blockIdx.x * 4 + (uint32_t)wave_index();
    if (w >= rows * c.heads) return;
    const uint32_t r = w / c.heads, head = w % c.heads;
    const TreeMeta m = find_meta<false>(c, r);
    const uint32_t sr = r - (m.row0 - c.meta[0].row0);
    const float *rec = c.records + ((size_t)m.record0 + ((size_t)sr * c.heads + head) * m.parts) * tree_record_floats(D);
    float mx = -INFINITY;
    for (uint32_t i = lane; i < m.parts; i += 64) mx = fmaxf(mx, rec[(size_t)i * tree_record_floats(D)]);
    mx = max64(mx);  // finite: a row sees itself
    float l = 0.0f, o[EPL] = {};
    for (uint32_t i0 = 0; i0 < m.parts; i0 += kBatch) {
        float2 ml[kBatch];
        float x[kBatch][EPL];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const float *q = rec + (size_t)min(i0 + u, m.parts - 1) * tree_record_floats(D);
            ml[u] = *(const float2 *)q;
#pragma unroll
            for (int i = 0; i < EPL; ++i) x[u][i] = q[4 + lane + 64 * i];
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const float weight = i0 + u < m.parts ? __builtin_amdgcn_exp2f(ml[u].x - mx) : 0.0f;
            l = fmaf(ml[u].y, weight, l);
#pragma unroll
            for (int i = 0; i < EPL; ++i) o[i] = fmaf(x[u][i], weight, o[i]);
        }
    }
    const bool gated = (c.flags & SAFETYRAISE_MI355X_GATED) != 0;
    const bool bf16_in = (c.flags & SAFETYRAISE_MI355X_INPUT_BF16) != 0;
    const size_t out_row = (size_t)(m.row0 + sr) * c.heads + head;
    const float inv = 1.0f / l;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
        float y = o[i] * inv;
        if (gated) y *= ref_sigmoid(load_act(c.q, out_row * 2 * D + D + lane + 64 * i, bf16_in));
        store_out(c, out_row * D + lane + 64 * i, y);
    }
}

template <int D, bool kF32>
hipError_t launch_attn(hipStream_t stream, const TreeCommon &c, uint32_t blocks) {
    using T = TreeShape<D, kF32>;
    static_assert(T::kLds <= 160 * 1024, "LDS");
    static LdsLimit limit;
    const hipError_t e = limit.allow((const void *)tree_attn_kernel<D, kF32>, T::kLds);
    if (e != hipSuccess) return e;
    SR_LAUNCH("tree_attn_kernel", (tree_attn_kernel<D, kF32>), dim3(blocks), dim3(T::kThreads),
              T::kLds, stream, c);
    return hipGetLastError();
}

template <int D>
hipError_t launch_width(hipStream_t stream, const TreeCommon &c, uint32_t blocks, uint32_t rows) {
    const hipError_t e = (c.flags & SAFETYRAISE_MI355X_OUTPUT_BF16) == 0
                             ? launch_attn<D, true>(stream, c, blocks)
                             : launch_attn<D, false>(stream, c, blocks);
    if (e != hipSuccess || c.records == nullptr) return e;
    SR_LAUNCH("tree_combine_kernel", tree_combine_kernel<D>, dim3((rows * c.heads + 3) / 4), dim3(256),
              0, stream, c, rows);
    return hipGetLastError();
}

}  // namespace

TreeScratch tree_scratch(const TreeLaunch &a, const SeqMeta *seqs, int nseq, uint64_t call_rows,
                         int num_cus) {
    TreeScratch t;
    const size_t group = a.heads / a.kv_heads;
    uint64_t rows = 0, tiles = 0;
    for (int i = 0; i < nseq; ++i) {
        rows += seqs[i].rows;
        tiles += a.kv_heads * ((seqs[i].rows * group + 31) / 32);
    }
    t.mask_bytes = call_rows * sizeof(uint4);
    if (generic_head_dim(a.head_dim)) {
        t.q_bytes = rows * a.heads * a.head_dim * sizeof(float);
        return t;
    }
    const size_t parts = (a.flags & SAFETYRAISE_MI355X_OUTPUT_BF16) ? 2 : 3;
    t.q_bytes = tiles * 32 * a.head_dim * 2 * parts;
    t.plan = tree_plan(a.heads, a.kv_heads, a.head_dim, a.pool->page_tokens, num_cus, seqs, nseq);
    t.record_bytes = t.plan.record_bytes;
    return t;
}

hipError_t launch_tree_attn(hipStream_t stream, const TreeLaunch &a, const SeqMeta *seqs, int nseq,
                            const uint8_t *parents, const TreePlan &plan) {
    PrepParams p{};
    TreeCommon &c = p.c;
    const auto *pool = a.pool;
    const bool generic = generic_head_dim(a.head_dim);
    const uint32_t D = a.head_dim;
    uint32_t rows = 0;
    for (int i = 0; i < nseq; ++i) rows += seqs[i].rows;
    if (nseq <= 0 || nseq > (int)kTreeSeqs || rows > kTreeRows || a.tbl_n > kInlineTable ||
        a.rotary_dim > D || D > kGenericMaxHeadDim) {
        return hipErrorInvalidValue;
    }
    c.k_pages = pool->k_pages;
    c.v_pages = pool->v_pages;
    c.page_table = pool->d_page_table;
    c.q = a.q;
    c.q_ops = a.q_ops;
    c.masks = (uint4 *)a.masks;
    c.out = a.out;
    c.err_word = a.err_word;
    c.num_pages = pool->num_pages;
    c.pages_per_seq = pool->pages_per_seq;
    c.log2_page = (uint32_t)__builtin_ctz(pool->page_tokens);
    c.flags = a.flags;
    c.heads = a.heads;
    c.kv_heads = a.kv_heads;
    c.head_dim = D;
    c.nseq = (uint32_t)nseq;
    if (!generic) {
        c.records = plan.direct ? nullptr : a.records;
        if (!plan.direct && a.records == nullptr) return hipErrorInvalidValue;
    }
    uint32_t blocks = 0, tiles = 0, records = 0;
    const uint32_t group = a.heads / a.kv_heads;
    for (int i = 0; i < nseq; ++i) {
        TreeMeta &m = c.meta[i];
        m.slot = seqs[i].slot;
        m.ctx = seqs[i].ctx;
        m.rows = seqs[i].rows;
        m.row0 = seqs[i].row0;
        m.tile0 = tiles;
        tiles += a.kv_heads * ((m.rows * group + 31) / 32);
        if (generic) continue;
        m.block0 = blocks;
        m.record0 = records;
        m.parts = tree_parts(plan, D, m.ctx + m.rows, m.rows * group);
        const uint32_t per = tree_vector_waves(D) * kTreeVectors;
        blocks += m.parts * a.kv_heads * ((m.rows * group + per - 1) / per);
        records += m.parts * m.rows * a.heads;
    }
    p.k = a.k;
    p.v = a.v;
    // without QK-norm the weights are not read
    p.q_norm = a.q_norm;
    p.k_norm = a.k_norm;
    p.positions = a.positions;
    p.rotary_dim = a.rotary_dim;
    for (int i = 0; i < 3; ++i) p.mrope[i] = a.mrope[i];
    p.eps = a.eps;
    p.qscale = kLog2e / sqrtf((float)D);
    p.rows = rows;
    p.parts = generic ? 0 : (a.flags & SAFETYRAISE_MI355X_OUTPUT_BF16) ? 2 : 3;
    p.tbl_n = a.tbl_n;
    for (uint32_t i = 0; i < a.tbl_n; ++i) {
        p.tbl_idx[i] = a.tbl_idx[i];
        p.tbl_val[i] = a.tbl_val[i];
    }
    for (uint32_t i = 0; i < a.rotary_dim / 2; ++i) p.denom[i] = a.rope_denom[i];
    for (uint32_t i = 0; i < rows; ++i) p.parent[i] = parents[i];
    const uint32_t groups = (a.kv_heads + a.heads + kPrepHeads - 1) / kPrepHeads;
    const dim3 grid((rows * groups + 3) / 4);
    const size_t prep_lds = (size_t)4 * kPrepHeads * D * sizeof(float);
    if (D <= 64) SR_LAUNCH("tree_prep_kernel", tree_prep_kernel<1>, grid, dim3(256), prep_lds, stream, p);
    else if (D <= 128) SR_LAUNCH("tree_prep_kernel", tree_prep_kernel<2>, grid, dim3(256), prep_lds, stream, p);
    else if (D <= 256) SR_LAUNCH("tree_prep_kernel", tree_prep_kernel<4>, grid, dim3(256), prep_lds, stream, p);
    else SR_LAUNCH("tree_prep_kernel", tree_prep_kernel<8>, grid, dim3(256), prep_lds, stream, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    switch (D) {
        case 64: return launch_width<64>(stream, c, blocks, rows);
        case 128: return launch_width<128>(stream, c, blocks, rows);
        case 256: return launch_width<256>(stream, c, blocks, rows);
        default: break;
    }
    SR_LAUNCH("tree_generic_kernel", tree_generic_kernel, dim3(a.heads, rows), dim3(64),
              (D + 64) * sizeof(float), stream, c);
    return hipGetLastError();
}

}  // namespace sr
