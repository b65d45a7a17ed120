// Attention over the 8-bit key/value caches (include/zw_gpu.h, zwg_kvq_attention_dev).
//
// With codes C and one scale per block of keys, s_j = (q . C_j) * sk and o = sum_j p_j sv C_j.  Codes of either
// format are exact in f16, so both products go to the f16 matrix units; the other operand, a query or a
// probability, is split into f16 hi + lo terms (22 significant bits) after a scaling by powers of two that puts it
// into f16's range whatever its size:
//   queries        each row by the power of two that brings its largest element to 2^14 .. 2^15
//   probabilities  p <= 2^kSlack relative to the reference maximum, times sv / ref <= 2, times 2^6, with ref a power
//                  of two at most the largest value scale met: below 2^15
// All sums are f32.
//
// Layout of a product (v_mfma_f32_16x16x32_f16: A 16 x 32, B 32 x 16): keys or value dims are the rows of A, query
// rows the columns of B.  Lane l holds A's row l % 16, B's column l % 16, both at contraction indices
// 8 (l / 16) .. + 7, and of the result rows 4 (l / 16) .. + 3 of column l % 16.  A lane's 16 bytes of keys or values are
// two A operands (kvq_at); its scores (column l % 16, keys 16 q + 4 (l / 16) + i) are the B operand of the value product
// for values stored in that order of keys, so probabilities never leave the lane that made them.
//
// Few query rows (up to 8 share a KV head: a decode step): the 16 columns are 8 rows' hi terms and the same rows' lo
// terms, and one product gives both.  More rows: 32 to a wave in two tiles, hi and lo as products of their own.
//
// The maximum is a lazy one: a column's reference rises only when some score passes it by kSlack = 8 (log2 units),
// so most tiles need no exchange between lanes and no rescaling.
//
// A workgroup's four waves take every fourth tile of 32 keys of one chunk and merge in LDS; chunks of one row
// are merged by kvq_merge_kernel.  Per wave and step 2 d / 32 KB are under way: the next step's keys are loaded once this
// step's scores are formed, its values once this step's are added, into the same registers, so that four waves fit a
// SIMD.  Bound by the reads and, in short calls, by the latency before the first product: 64 sequences of 1 .. 4096 keys
// (d = 128, two KV heads, 67 MB) take 14.4 us, 4.7 TB/s, where a large copy moves 4.8.
#include <hip/hip_runtime.h>

#include <cmath>
#include <string>

#include "attn_geometry.hpp"
#include "kv_quant.hpp"
#include "zw_ctx.hpp"

using namespace zwg_host;
using namespace zwg_planner;
using zwg::KvqView;

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kTile = zwg::kKvqTile; // keys of a wave's step
constexpr int kWaves = zwg_planner::kKvqWaves;
constexpr int kSplitTile = zwg_planner::kKvqSplitTile;
constexpr int kCompactSeqs = 1024; // sequences whose key counts a workgroup goes through to find its work
constexpr int kManyChunks = 32;
constexpr float kSlack = 8.0f;
constexpr float kProbScale = 64.0f; // 2^6: p * (sv / ref) * 2^6 <= 2^8 * 2 * 2^6

// Division of n < 2^31 by a divisor known on the host: the kernels' first instructions are a good part of a short
// call (they come from a cold instruction cache), and a general division is about 35 of them.
struct Div {
    uint32_t d, mul, shift;
    Div() = default;
    explicit Div(uint32_t x) : d(x), mul(0), shift(0) {
        if (x <= 1) return;
        uint32_t l = 32 - (uint32_t)__builtin_clz(x - 1); // ceil(log2 x)
        mul = (uint32_t)(((1ull << (31 + l)) + x - 1) / x);
        shift = l - 1;
    }
    __device__ __forceinline__ int of(int n) const { return d == 1 ? n : (int)(__umulhi((uint32_t)n, mul) >> shift); }
};

struct KvqArgs {
    KvqView view;
    int64_t unit0; // unit of (layer, seq0, head 0)
    const float *q;
    float *out;
    int64_t q_stride, q_bstride, out_stride, out_bstride;
    const int32_t *n_kv_dev;
    int32_t n_seq, n_q, n_kv, n_head, group, rows; // rows = n_q * group of a (sequence, KV head)
    int32_t row_blocks;
    int32_t causal;
    float scale_log2;
    int32_t tau, max_chunks; // split tiles of a chunk aimed at
    Div by_group, by_heads, by_per, by_seqs, by_tau, by_rows; // n_head_kv; n_head_kv * row_blocks; ...
    int32_t per;
    int32_t block_shift; // log2 of the tokens of a scale
    float *part_o;  // [row][max_chunks][d]
    float *part_ml; // [row][max_chunks][2]
    float *row_ml;  // [row][2]: the rows' final maximum and sum, for the weights; or nullptr
    float *weights;
    int64_t w_stride, w_bstride;
    float decay;
};

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ uint32_t abs_bits(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7fffffffu; }

__device__ __forceinline__ int item_kv(const KvqArgs &a, int item) {
    return a.n_kv_dev ? min(max(a.n_kv_dev[item], 0), a.n_kv) : a.n_kv;
}
// Keys that row r of a (sequence, KV head) sees.
__device__ __forceinline__ int row_limit(const KvqArgs &a, int n_kv, int r) {
    return a.causal ? max(0, n_kv - a.n_q + a.by_group.of(r) + 1) : n_kv;
}
// Keys that the last row of row block rb sees.
__device__ __forceinline__ int block_limit(const KvqArgs &a, int n_kv, int rb, int RB) {
    return row_limit(a, n_kv, min(a.rows, (rb + 1) * RB) - 1);
}
// a / b for 0 <= a < 2^22, 0 < b: the quotient of the floats is at most one off.
__device__ __forceinline__ int div_small(int a, int b) {
    int q = (int)((float)a * __builtin_amdgcn_rcpf((float)b));
    const int r = a - q * b;
    return r < 0 ? q - 1 : r >= b ? q + 1 : q;
}
// zwg::unit_split with its divisions as above: the chunks of [0, kv_hi) and the keys of each.
__device__ __forceinline__ int split_bound(const KvqArgs &a, int w) { return min(max(a.by_tau.of(w + a.tau / 2), 1), a.max_chunks); }
__device__ __forceinline__ int split(const KvqArgs &a, int kv_hi, int *chunk_keys) {
    const int w = (kv_hi + kSplitTile - 1) / kSplitTile;
    const int nc = split_bound(a, w);
    const int lt = max(1, div_small(w + nc - 1, nc));
    *chunk_keys = lt * kSplitTile;
    return max(1, div_small(w + lt - 1, lt));
}
// Row r of (item, KV head): partials and final statistics at this index.
__device__ __forceinline__ int64_t row_at(const KvqArgs &a, int item, int hk, int r) {
    return ((int64_t)item * a.view.n_head_kv + hk) * a.rows + r;
}

// 8 codes (two words) to f16.
template <int FMT> __device__ __forceinline__ f16x8 codes_f16(u32x2 w) {
    uint32_t h[4];
    if (FMT == ZWG_KVQ_I8) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            // code + 128 under the exponent byte 0x64: 1024 + code + 128
            h[2 * i] = __builtin_amdgcn_perm(0x64646464u, w[i], 0x04010400u);
            h[2 * i + 1] = __builtin_amdgcn_perm(0x64646464u, w[i], 0x04030402u);
        }
        f16x8 r;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f16x2 v = __builtin_bit_cast(f16x2, h[i]) - (f16x2){(_Float16)1152.0f, (_Float16)1152.0f};
            r[2 * i] = v[0];
            r[2 * i + 1] = v[1];
        }
        return r;
    }
    f16x8 r;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const auto lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w[i], 1.0f, false);
        const auto hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w[i], 1.0f, true);
        r[4 * i] = (_Float16)lo[0];
        r[4 * i + 1] = (_Float16)lo[1];
        r[4 * i + 2] = (_Float16)hi[0];
        r[4 * i + 3] = (_Float16)hi[1];
    }
    return r;
}

// A register's values moved between the 16 lanes of a row.
template <int CTRL> __device__ __forceinline__ float dpp_f32(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}

// x of lane `lane`, the same for the whole wave.
__device__ __forceinline__ float lane_value(float x, int lane) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), lane));
}
// x of the lane 8 columns away (l ^ 8 within its row of 16).
__device__ __forceinline__ float other_half(float x) { return dpp_f32<0x128>(x); } // row_ror 8
__device__ __forceinline__ float groups_max(float x) {
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float groups_sum(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

// Geometry of a wave: CT column tiles of 16, PACKED: one tile that holds 8 rows' hi and lo terms.
template <int D, int CT, bool PACKED> struct Geo {
    static constexpr int kRows = PACKED ? 8 : 16 * CT;
    static constexpr int kSteps = D / 32;              // score products of a key tile
    static constexpr int kDims = D / 16;               // value tiles
    static constexpr int kParts = PACKED ? 1 : 2;      // hi and lo products
};

// The queries of a wave as B operands, and what turns a product into a score in log2 units.
template <int D, int CT, bool PACKED> struct Queries {
    using G = Geo<D, CT, PACKED>;
    f16x8 frag[CT][G::kParts][G::kSteps];
    float back[CT];

    // Score step s of lane group g covers dims at_dim(s, g) .. + 7.
    static __device__ __forceinline__ int at_dim(int s, int g) {
        return D == 32 ? 8 * g : 64 * (s >> 1) + 16 * g + 8 * (s & 1);
    }

    // a lane's elements as they are: the loads, which the caller issues before the codes' (they are needed first)
    struct Raw {
        f32x4 x[CT][G::kSteps][2];
        __device__ __forceinline__ void load(const KvqArgs &a, int item, int hk, int r0, int lane) {
            const int g = lane >> 4, col = lane & 15;
#pragma unroll
            for (int t = 0; t < CT; ++t) {
                // rows behind the last repeat it: what they give is not stored
                const int r = min(r0 + (PACKED ? (col & 7) : 16 * t + col), a.rows - 1);
                const int qi = a.by_group.of(r);
                const float *q = a.q + item * a.q_bstride + qi * a.q_stride + (int64_t)(hk * a.group + (r - qi * a.group)) * D;
#pragma unroll
                for (int s = 0; s < G::kSteps; ++s)
#pragma unroll
                    for (int h = 0; h < 2; ++h) x[t][s][h] = *reinterpret_cast<const f32x4 *>(q + at_dim(s, g) + 4 * h);
            }
        }
    };

    __device__ __forceinline__ void take(const KvqArgs &a, const Raw &raw, int lane) {
#pragma unroll
        for (int t = 0; t < CT; ++t) {
            uint32_t top = 0;
#pragma unroll
            for (int s = 0; s < G::kSteps; ++s)
#pragma unroll
                for (int k = 0; k < 8; ++k) top = max(top, abs_bits(raw.x[t][s][k >> 2][k & 3]));
            top = max(top, (uint32_t)__shfl_xor((int)top, 16));
            top = max(top, (uint32_t)__shfl_xor((int)top, 32));
            // largest element 1.m * 2^(e - 127) -> times 2^(141 - e): into 2^14 .. 2^15 (e 15 at least, so that
            // both powers are normal numbers; 255, an infinity or a NaN, stays one)
            const uint32_t e = max(top >> 23, 15u);
            const float up = __builtin_bit_cast(float, (268u - e) << 23);
            back[t] = __builtin_bit_cast(float, (e - 14u) << 23) * a.scale_log2;
#pragma unroll
            for (int s = 0; s < G::kSteps; ++s)
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const float v = raw.x[t][s][k >> 2][k & 3] * up;
                    const _Float16 hi = (_Float16)v;
                    const _Float16 lo = (_Float16)(v - (float)hi);
                    if (PACKED) {
                        frag[t][0][s][k] = (lane & 15) < 8 ? hi : lo;
                    } else {
                        frag[t][0][s][k] = hi;
                        frag[t][G::kParts - 1][s][k] = lo;
                    }
                }
        }
    }
};

constexpr int kQ = kTile / 16; // key tiles of a step

// A unit's keys or values, range-checked by the hardware: a load past the end returns zeros and reads nothing, so loads
// of steps that do not exist need no branch (a branch around loads makes the waits for earlier ones too long, as the
// compiler must take the loads not to have been issued).
constexpr uint32_t kNoStep = 0x80000000u;
constexpr int kCachePolicyNT = 2; // read once a call: pass the caches without displacing lines
__device__ __forceinline__ __amdgpu_buffer_rsrc_t unit_codes(const uint8_t *codes, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(codes), 0, (int)bytes, 0x00020000);
}

// A step's keys or values: d / 32 KB, 16 bytes a lane each.
template <int D> struct Codes {
    u32x4 w[D / 32];
    // at: the step's byte offset (its first key times d), or kNoStep; in the lane's offset, which is the checked one
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t codes, uint32_t at, int lane) {
        const uint32_t off = at + 64u * (uint32_t)(lane & 15) + 16u * (uint32_t)(lane >> 4);
#pragma unroll
        for (int n = 0; n < D / 32; ++n)
            w[n] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(codes, (int)(off + 1024u * n), 0, kCachePolicyNT));
    }
    static __device__ __forceinline__ u32x2 half(u32x4 v, int h) { return h ? (u32x2){v[2], v[3]} : (u32x2){v[0], v[1]}; }
    // key tile q's operand of score product st; value tile d's operand
    __device__ __forceinline__ u32x2 key(int q, int st) const {
        return D == 32 ? half(w[0], q) : half(w[q * (D / 64) + (st >> 1)], st & 1);
    }
    __device__ __forceinline__ u32x2 value(int d) const { return half(w[d >> 1], d & 1); }
};
// The scales of a step, one per 16 tokens (wave-uniform: scalar loads).
struct Scales {
    float s[kQ];
    __device__ __forceinline__ void load(const float *scales, int k0, int shift) {
#pragma unroll
        for (int q = 0; q < kQ; ++q) s[q] = scales[(k0 + 16 * q) >> shift];
    }
};

// The products of a step's keys, unscaled: column tile t, key tile q.
template <int D, int FMT, int CT, bool PACKED>
__device__ __forceinline__ void score_tile(const Queries<D, CT, PACKED> &qs, const Codes<D> &kt, f32x4 (&s)[CT][kQ]) {
    using G = Geo<D, CT, PACKED>;
#pragma unroll
    for (int q = 0; q < kQ; ++q)
#pragma unroll
        for (int t = 0; t < CT; ++t) s[t][q] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int st = 0; st < G::kSteps; ++st)
#pragma unroll
        for (int q = 0; q < kQ; ++q) {
            const f16x8 k = codes_f16<FMT>(kt.key(q, st));
#pragma unroll
            for (int t = 0; t < CT; ++t)
#pragma unroll
                for (int p = 0; p < G::kParts; ++p)
                    s[t][q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qs.frag[t][p][st], s[t][q], 0, 0, 0);
        }
    if (PACKED) {
#pragma unroll
        for (int q = 0; q < kQ; ++q)
#pragma unroll
            for (int t = 0; t < CT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[t][q][i] += other_half(s[t][q][i]);
    }
}

// The running softmax of a wave's rows and the value products' operand.
template <int D, int CT, bool PACKED> struct Softmax {
    using G = Geo<D, CT, PACKED>;
    float m[CT], l[CT], ref; // per column: reference maximum (log2 units) and this lane's sum; ref: see above
    f32x4 o[CT][G::kDims];
    f16x8 p[CT][G::kParts];

    __device__ __forceinline__ void init() {
        ref = 0.f;
#pragma unroll
        for (int t = 0; t < CT; ++t) {
            m[t] = -INFINITY;
            l[t] = 0.f;
#pragma unroll
            for (int d = 0; d < G::kDims; ++d) o[t][d] = (f32x4){0.f, 0.f, 0.f, 0.f};
        }
    }

    // Takes the products s of the keys from k0 on, of which column tile t sees those below lim[t] (k_end: the last
    // limit of any row here; mask, the same in the whole wave: some column does not see them all): raises the references.
    // f and w get what a product and a probability are to be multiplied by, and s is changed where the mask says so.  The
    // branches are around few values: two copies of the whole would each want the accumulators in registers of their own.
    __device__ __forceinline__ void prepare(f32x4 (&s)[CT][kQ], const float (&back)[CT], const Scales &sk, const Scales &sv,
                                            const int (&lim)[CT], bool mask, int k0, int k_end, int lane, float (&f)[CT][kQ],
                                            float (&w)[CT][kQ]) {
        const int g = lane >> 4;
        // blocks behind the last visible key count for nothing, whatever they hold
        float big = ref;
#pragma unroll
        for (int q = 0; q < kQ; ++q) {
            const float v = k0 + 16 * q < k_end ? sv.s[q] : 0.f;
            big = fmaxf(big, v);
#pragma unroll
            for (int t = 0; t < CT; ++t) {
                f[t][q] = back[t] * sk.s[q];
                w[t][q] = v;
            }
        }
        if (mask) {
            // an unseen key: -infinity; its block's scales may be zero or NaN, and are then not to be multiplied with
#pragma unroll
            for (int t = 0; t < CT; ++t)
#pragma unroll
                for (int q = 0; q < kQ; ++q) {
                    const bool sees = k0 + 16 * q < lim[t], zero = f[t][q] == 0.f;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float x = zero ? 0.f : s[t][q][i];
                        s[t][q][i] = k0 + 16 * q + 4 * g + i < lim[t] ? x : -INFINITY;
                    }
                    if (zero || !sees) f[t][q] = 1.f;
                    if (!sees) w[t][q] = 0.f;
                }
        }
        // scales are not negative: the largest product is the largest score
        float top[CT];
        bool rise = false;
#pragma unroll
        for (int t = 0; t < CT; ++t) {
            top[t] = -INFINITY;
#pragma unroll
            for (int q = 0; q < kQ; ++q)
                top[t] = fmaxf(top[t], fmaxf(fmaxf(s[t][q][0], s[t][q][1]), fmaxf(s[t][q][2], s[t][q][3])) * f[t][q]);
            rise |= top[t] > m[t] + kSlack;
        }
        // the value scales relative to a power of two at most the largest met (NaNs aside)
        const float ref_new = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, big) & 0x7f800000u);
        if (__any(rise) || ref_new != ref) {
            const float down = ref > 0.f ? ref * power_inverse(ref_new) : 1.f; // powers of two: exact
            ref = ref_new;
#pragma unroll
            for (int t = 0; t < CT; ++t) {
                const float m_new = fmaxf(m[t], groups_max(top[t]));
                const float alpha = m_new == -INFINITY ? 1.f : exp2_fast(m[t] - m_new);
                m[t] = m_new;
                l[t] *= alpha;
#pragma unroll
                for (int d = 0; d < G::kDims; ++d) o[t][d] *= alpha * down;
            }
        }
        const float inv_ref = ref > 0.f ? kProbScale * power_inverse(ref) : 0.f;
#pragma unroll
        for (int t = 0; t < CT; ++t)
#pragma unroll
            for (int q = 0; q < kQ; ++q) w[t][q] *= inv_ref;
    }

    // The probabilities of what prepare left, and p.  No branches: other products may go between.
    __device__ __forceinline__ void weigh(const f32x4 (&s)[CT][kQ], const float (&f)[CT][kQ], const float (&w)[CT][kQ], int lane) {
        const int col = lane & 15;
#pragma unroll
        for (int t = 0; t < CT; ++t) {
            const float mu = m[t] == -INFINITY ? 0.f : m[t];
#pragma unroll
            for (int q = 0; q < kQ; ++q)
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    const float e0 = exp2_fast(__builtin_fmaf(s[t][q][i], f[t][q], -mu));
                    const float e1 = exp2_fast(__builtin_fmaf(s[t][q][i + 1], f[t][q], -mu));
                    l[t] += e0;
                    l[t] += e1;
                    const float x = e0 * w[t][q], y = e1 * w[t][q];
                    // hi by truncation (two in one instruction); what is left fits 11 more bits, rounded
                    const auto h = __builtin_amdgcn_cvt_pkrtz(x, y);
                    const _Float16 hx = (_Float16)h[0], hy = (_Float16)h[1];
                    const _Float16 rx = (_Float16)(x - (float)hx), ry = (_Float16)(y - (float)hy);
                    const int k = 4 * q + i;
                    if (PACKED) {
                        p[t][0][k] = col < 8 ? hx : rx;
                        p[t][0][k + 1] = col < 8 ? hy : ry;
                    } else {
                        p[t][0][k] = hx;
                        p[t][0][k + 1] = hy;
                        p[t][G::kParts - 1][k] = rx;
                        p[t][G::kParts - 1][k + 1] = ry;
                    }
                }
        }
    }

    // 1 / x of a power of two (normal, and its inverse too: scales lie between 2^-108 and 2^122)
    static __device__ __forceinline__ float power_inverse(float x) {
        return __builtin_bit_cast(float, 0x7f000000u - __builtin_bit_cast(uint32_t, x));
    }

    __device__ __forceinline__ void add(const f16x8 v, int d) {
#pragma unroll
        for (int t = 0; t < CT; ++t)
#pragma unroll
            for (int q = 0; q < G::kParts; ++q) o[t][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p[t][q], o[t][d], 0, 0, 0);
    }
};

// The work of workgroup `b`: over all (chunk, sequence, row block, KV head) with the chunk slowest, or, when the
// sequences have their own key counts, over those with keys alone, sequence by sequence, so that consecutive
// workgroups -- and so every CU -- get an even share however the counts differ.
__device__ __forceinline__ bool find_unit(const KvqArgs &a, uint32_t b, int RB, int *item, int *rb, int *hk, int *chunk) {
    const uint32_t per = (uint32_t)a.per;
    uint32_t rest;
    if (a.n_kv_dev && a.n_seq <= kCompactSeqs) {
        const int lane = (int)(threadIdx.x & 63);
        uint32_t base = 0;
        bool hit = false;
        for (int k = 0; k < a.n_seq && !hit; k += 64) {
            const int it = k + lane;
            uint32_t c = 0;
            if (it < a.n_seq) {
                const int hi = block_limit(a, item_kv(a, it), a.row_blocks - 1, RB);
                int keys;
                // fewer keys can be cut into more chunks (132 tiles into 44 of 3, 133 into 34 of 4), so with several row blocks
                // the bound that grows with the keys
                c = (uint32_t)(a.row_blocks == 1 ? split(a, hi, &keys) : split_bound(a, (hi + kSplitTile - 1) / kSplitTile)) * per;
            }
            uint32_t incl = c;
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const uint32_t v = (uint32_t)__shfl_up((int)incl, off);
                if (lane >= off) incl += v;
            }
            const unsigned long long first = __ballot(base + incl > b);
            if (first) {
                const int f = __builtin_ctzll(first);
                *item = k + f;
                rest = b - (base + (uint32_t)__builtin_amdgcn_readlane((int)(incl - c), f));
                hit = true;
            } else {
                base += (uint32_t)__builtin_amdgcn_readlane((int)incl, 63);
            }
        }
        if (!hit) return false;
        *chunk = a.by_per.of((int)rest);
        rest -= (uint32_t)*chunk * per;
    } else {
        const int c = a.by_per.of((int)b);
        rest = b - (uint32_t)c * per;
        *chunk = a.by_seqs.of(c);
        *item = c - *chunk * a.n_seq;
    }
    *rb = a.by_heads.of((int)rest);
    *hk = (int)(rest - (uint32_t)*rb * (uint32_t)a.view.n_head_kv);
    *item = __builtin_amdgcn_readfirstlane(*item);
    *rb = __builtin_amdgcn_readfirstlane(*rb);
    *hk = __builtin_amdgcn_readfirstlane(*hk);
    *chunk = __builtin_amdgcn_readfirstlane(*chunk);
    return true;
}

// A row's sums x (4 dims from c on) with maximum M and sum L: into out, or into its chunk's slot.
template <int D>
__device__ __forceinline__ void store_row(const KvqArgs &a, int item, int hk, int row, int c, int n_chunks, int chunk, float M,
                                          float L, f32x4 x) {
    const int64_t at = row_at(a, item, hk, row);
    if (n_chunks == 1) {
        const int qi = a.by_group.of(row), head = hk * a.group + row - qi * a.group;
        const float inv = L != 0.f ? 1.f / L : 0.f; // a NaN stays one
        *reinterpret_cast<f32x4 *>(a.out + item * a.out_bstride + qi * a.out_stride + (int64_t)head * D + c) = x * inv;
        if (a.row_ml && c == 0) *reinterpret_cast<float2 *>(a.row_ml + 2 * at) = make_float2(M, L);
    } else {
        const int64_t slot = at * a.max_chunks + chunk;
        *reinterpret_cast<f32x4 *>(a.part_o + slot * D + c) = x;
        if (c == 0) *reinterpret_cast<float2 *>(a.part_ml + 2 * slot) = make_float2(M, L);
    }
}

template <int D, int FMT, int CT, bool PACKED>
__global__ __launch_bounds__(64 * kWaves) void kvq_attn_kernel(KvqArgs a) {
    using G = Geo<D, CT, PACKED>;
    constexpr int RB = G::kRows;
    __shared__ __align__(16) float o_s[kWaves][RB][D + 4];
    __shared__ float m_s[kWaves][RB], l_s[kWaves][RB];

    const KvqView &v = a.view;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, col = lane & 15;
    int item, rb, hk, chunk;
    if (!find_unit(a, blockIdx.x, RB, &item, &rb, &hk, &chunk)) return;

    const int n_kv = item_kv(a, item);
    const int hi = block_limit(a, n_kv, rb, RB);
    int chunk_keys;
    const int n_chunks = split(a, hi, &chunk_keys);
    if (chunk >= n_chunks) return;
    const int k_begin = chunk * chunk_keys, k_end = min(hi, k_begin + chunk_keys);

    const int64_t u = a.unit0 + (int64_t)item * v.n_head_kv + hk;
    const __amdgpu_buffer_rsrc_t keys = unit_codes(v.codes[0] + u * v.unit_bytes, v.unit_bytes);
    const __amdgpu_buffer_rsrc_t vals = unit_codes(v.codes[1] + u * v.unit_bytes, v.unit_bytes);
    const float *ks = v.scales[0] + u * v.n_blocks, *vs = v.scales[1] + u * v.n_blocks;

    typename Queries<D, CT, PACKED>::Raw raw;
    raw.load(a, item, hk, rb * RB, lane);
    int k0 = k_begin + wave * kTile;
    Codes<D> kt, vt;
    Scales sk, sv;
    kt.load(keys, k0 < k_end ? (uint32_t)k0 * D : kNoStep, lane);
    vt.load(vals, k0 < k_end ? (uint32_t)k0 * D : kNoStep, lane);
    sk.load(ks, k0 < k_end ? k0 : k_begin, a.block_shift);
    sv.load(vs, k0 < k_end ? k0 : k_begin, a.block_shift);
    Queries<D, CT, PACKED> qs;
    qs.take(a, raw, lane);
    int lim[CT];
#pragma unroll
    for (int t = 0; t < CT; ++t) {
        const int r = rb * RB + (PACKED ? (col & 7) : 16 * t + col);
        lim[t] = r < a.rows ? min(k_end, row_limit(a, n_kv, r)) : 0;
    }
    // the smallest limit of the block's rows: tiles below it need no mask
    const int lim_all = min(k_end, row_limit(a, n_kv, rb * RB));

    Softmax<D, CT, PACKED> sm;
    sm.init();
#pragma unroll 1
    while (k0 < k_end) {
        f32x4 s[CT][kQ];
        score_tile<D, FMT, CT, PACKED>(qs, kt, s);
        // the next tile's keys on their way over this one's softmax and value products, its values over the next one's
        // score products
        const int next = k0 + kSplitTile;
        const bool more = next < k_end;
        const uint32_t at = more ? (uint32_t)next * D : kNoStep;
        Scales sk_next, sv_next;
        kt.load(keys, at, lane);
        sk_next.load(ks, more ? next : k0, a.block_shift);
        sv_next.load(vs, more ? next : k0, a.block_shift);
        __builtin_amdgcn_sched_barrier(0);
        float f[CT][kQ], w[CT][kQ];
        sm.prepare(s, qs.back, sk, sv, lim, k0 + kTile > lim_all, k0, k_end, lane, f, w);
        sm.weigh(s, f, w, lane);
#pragma unroll
        for (int d = 0; d < G::kDims; ++d) sm.add(codes_f16<FMT>(vt.value(d)), d);
        vt.load(vals, at, lane);
        __builtin_amdgcn_sched_barrier(0);
        sk = sk_next;
        sv = sv_next;
        k0 = next;
    }

    // ---- the waves' results merged in LDS
    const float unit = sm.ref * (1.0f / kProbScale);
#pragma unroll
    for (int t = 0; t < CT; ++t) {
        const float lt = groups_sum(sm.l[t]);
        const int r = PACKED ? (col & 7) : 16 * t + col;
        const bool writes = !PACKED || col < 8;
        if (writes && g == 0) {
            m_s[wave][r] = sm.m[t];
            l_s[wave][r] = lt;
        }
#pragma unroll
        for (int d = 0; d < G::kDims; ++d) {
            f32x4 x = sm.o[t][d];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = (PACKED ? x[i] + other_half(x[i]) : x[i]) * unit;
            if (writes) *reinterpret_cast<f32x4 *>(&o_s[wave][r][16 * d + 4 * g]) = x;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < RB * (D / 4); i += 64 * kWaves) {
        const int r = i / (D / 4), c = 4 * (i % (D / 4));
        const int row = rb * RB + r;
        if (row >= a.rows) break;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) M = fmaxf(M, m_s[w][r]);
        float L = 0.f;
        f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            // 0 for a wave that saw no key of this row; with no key seen by any, sums of zeros, or of NaNs where the
            // scores are no numbers
            const float f = M == -INFINITY ? 1.f : exp2_fast(m_s[w][r] - M);
            L += f * l_s[w][r];
            x += f * *reinterpret_cast<const f32x4 *>(&o_s[w][r][c]);
        }
        store_row<D>(a, item, hk, row, c, n_chunks, chunk, M, L, x);
    }
}

// Prompts: 128 rows of a (sequence, KV head) to a workgroup, 16 to each of 8 waves, over the same keys.  A step's codes are
// read once, a KB a wave, turned into f16 operands and put into LDS, from where all waves feed their products (turning
// codes into f16 takes a wave as many instructions as its softmax, so it is shared); the next step's are put into the other
// half of LDS behind this step's products, and those of the one after that are on their way.
//
// Bound by the sum of matrix and vector instructions, which do not overlap here: 1024 queries of 12 heads over 8000 keys (d =
// 128) take 123 us, of which the products alone, 94 GFLOP with their hi and lo terms, take 64 (1.47 PFLOP/s, what a large
// library product reaches on this card) and everything else alone 55.  For that reason none of these measured faster: the next
// step's score products between this step's softmax instructions (124 us), 32 rows to each of 4 waves (124), 64 keys between
// two barriers (127).
constexpr int kPromptRows = 128;
constexpr int kPromptWaves = 8;

template <int D, int FMT> __global__ __launch_bounds__(64 * kPromptWaves, 4) void kvq_prompt_kernel(KvqArgs a) {
    constexpr int CT = 1;
    using G = Geo<D, CT, false>;
    constexpr int kKB = D / 32; // KBs of a step's keys, and of its values: at most one a wave
    static_assert(2 * kKB <= kPromptWaves, "a KB a wave");
    __shared__ __align__(16) f16x8 stage[2][4 * kKB][64]; // operands: [key tile][step] of keys, then value tiles
    const KvqView &v = a.view;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, col = lane & 15;
    int item, rb, hk, chunk;
    if (!find_unit(a, blockIdx.x, kPromptRows, &item, &rb, &hk, &chunk)) return;
    if (a.causal) rb = a.row_blocks - 1 - rb; // the longest first

    const int n_kv = item_kv(a, item);
    const int hi = block_limit(a, n_kv, rb, kPromptRows);
    int chunk_keys;
    const int n_chunks = split(a, hi, &chunk_keys);
    if (chunk >= n_chunks) return;
    const int k_begin = chunk * chunk_keys, k_end = min(hi, k_begin + chunk_keys);

    const int64_t u = a.unit0 + (int64_t)item * v.n_head_kv + hk;
    const int of_val = wave >= kKB; // this wave's KB is of the values
    const __amdgpu_buffer_rsrc_t codes = unit_codes((of_val ? v.codes[1] : v.codes[0]) + u * v.unit_bytes, v.unit_bytes);
    // A step's scales are vector loads of their own, a lane to a key tile, a step ahead: scalar loads beside the LDS reads
    // would have the products wait for both.
    const __amdgpu_buffer_rsrc_t scales[2] = {
        unit_codes(reinterpret_cast<const uint8_t *>(v.scales[0] + u * v.n_blocks), (int64_t)v.n_blocks * 4),
        unit_codes(reinterpret_cast<const uint8_t *>(v.scales[1] + u * v.n_blocks), (int64_t)v.n_blocks * 4)};

    const int row0 = rb * kPromptRows + 16 * CT * wave;
    typename Queries<D, CT, false>::Raw raw;
    raw.load(a, item, hk, row0, lane);

    u32x4 held;
    uint32_t next_scale[2];
    const auto load = [&](int k0) { // steps that do not exist read nothing and come out as zeros
        const bool is = k0 < k_end;
        const uint32_t scale_at = is ? 4u * ((uint32_t)(k0 + 16 * (lane & (kQ - 1))) >> a.block_shift) : kNoStep;
#pragma unroll
        for (int i = 0; i < 2; ++i) next_scale[i] = __builtin_amdgcn_raw_buffer_load_b32(scales[i], (int)scale_at, 0, 0);
        const uint32_t at = is && wave < 2 * kKB ? (uint32_t)k0 * D + 1024u * (uint32_t)(of_val ? wave - kKB : wave) : kNoStep;
        held = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(codes, (int)(at + 64u * col + 16u * g), 0, 0));
    };
    const auto put = [&](int half) {
        if (wave >= 2 * kKB) return;
        // a KB is two operands: of keys (d = 128) steps 2 (n % 2) and 2 (n % 2) + 1 of key tile n / 2; (64) both steps of tile n;
        // (32) both key tiles' one step -- in every case 2 n and 2 n + 1 of [key tile][step] -- of values tiles 2 n and 2 n + 1
        stage[half][2 * wave][lane] = codes_f16<FMT>((u32x2){held[0], held[1]});
        stage[half][2 * wave + 1][lane] = codes_f16<FMT>((u32x2){held[2], held[3]});
    };
    Scales sk, sv; // of the step at hand
    const auto take_scales = [&] {
#pragma unroll
        for (int q = 0; q < kQ; ++q) {
            sk.s[q] = lane_value(__builtin_bit_cast(float, next_scale[0]), q);
            sv.s[q] = lane_value(__builtin_bit_cast(float, next_scale[1]), q);
        }
    };
    load(k_begin);
    Queries<D, CT, false> qs;
    qs.take(a, raw, lane);
    const int row = row0 + col;
    const int lim[CT] = {row < a.rows ? min(k_end, row_limit(a, n_kv, row)) : 0};
    // the smallest and the largest limit of this wave's rows
    const int lim_all = row0 < a.rows ? min(k_end, row_limit(a, n_kv, row0)) : 0;
    const int lim_any = row0 < a.rows ? min(k_end, row_limit(a, n_kv, min(a.rows, row0 + 16 * CT) - 1)) : 0;

    Softmax<D, CT, false> sm;
    sm.init();
    put(0);
    take_scales();
    load(k_begin + kTile);
    __syncthreads();
    int half = 0;
#pragma unroll 1
    for (int k0 = k_begin; k0 < k_end; k0 += kTile) {
        if (k0 < lim_any) {
            f32x4 s[CT][kQ];
#pragma unroll
            for (int q = 0; q < kQ; ++q) s[0][q] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int st = 0; st < G::kSteps; ++st)
#pragma unroll
                for (int p = 0; p < 2; ++p)
#pragma unroll
                    for (int q = 0; q < kQ; ++q)
                        s[0][q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(stage[half][q * G::kSteps + st][lane], qs.frag[0][p][st], s[0][q], 0, 0, 0);
            float f[CT][kQ], w[CT][kQ];
            sm.prepare(s, qs.back, sk, sv, lim, k0 + kTile > lim_all, k0, k_end, lane, f, w);
            sm.weigh(s, f, w, lane);
            // two value tiles in turn: no product waits for the one before it
#pragma unroll
            for (int d = 0; d < G::kDims; d += 2)
#pragma unroll
                for (int p = 0; p < 2; ++p)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        sm.o[0][d + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(stage[half][2 * kKB + d + e][lane], sm.p[0][p], sm.o[0][d + e], 0, 0, 0);
        }
        // every wave left the other half at the last barrier
        half ^= 1;
        put(half);
        take_scales();
        load(k0 + 2 * kTile);
        __syncthreads();
    }

    const float unit = sm.ref * (1.0f / kProbScale);
    const float L = groups_sum(sm.l[0]);
    if (row >= a.rows) return;
#pragma unroll
    for (int d = 0; d < G::kDims; ++d) store_row<D>(a, item, hk, row, 16 * d + 4 * g, n_chunks, chunk, sm.m[0], L, sm.o[0][d] * unit);
}

// The chunks of each row, added in an order of their own: W dims of a row to a workgroup, W / 4 threads over them in
// kGroups groups over the chunks, whose sums are added at the end.  W is d where the chunks are few; with many, a
// narrow W brings more workgroups to a row (one CU takes in 30 to 40 GB/s).
template <int D, int W, int RB> __global__ __launch_bounds__(256) void kvq_merge_kernel(KvqArgs a) {
    constexpr int kGroups = 256 / (W / 4);
    __shared__ __align__(16) f32x4 x_s[kGroups][W / 4];
    __shared__ float red[4], l_s[kGroups];
    const uint32_t at = blockIdx.x / (uint32_t)(D / W), first = blockIdx.x % (uint32_t)(D / W) * W;
    const int ih = a.by_rows.of((int)at);
    const int row = (int)at - ih * a.rows;
    const int item = a.by_heads.of(ih), hk = ih - item * a.view.n_head_kv;
    int chunk_keys;
    const int n_chunks = split(a, block_limit(a, item_kv(a, item), row / RB, RB), &chunk_keys);
    if (n_chunks == 1) return; // written by the attention kernel
    const int tid = threadIdx.x, grp = tid / (W / 4), c = tid % (W / 4);
    const float *ml = a.part_ml + 2 * (int64_t)at * a.max_chunks;
    const f32x4 *po = reinterpret_cast<const f32x4 *>(a.part_o + (int64_t)at * a.max_chunks * D + first) + c;
    float M = -INFINITY;
    for (int k = tid; k < n_chunks; k += 256) M = fmaxf(M, ml[2 * k]);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) M = fmaxf(M, __shfl_xor(M, off));
    if ((tid & 63) == 0) red[tid >> 6] = M;
    __syncthreads();
    M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    float L = 0.f;
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int k = grp; k < n_chunks; k += kGroups) {
        const float f = M == -INFINITY ? 1.f : exp2_fast(ml[2 * k] - M);
        L += f * ml[2 * k + 1];
        x += f * po[(int64_t)k * (D / 4)];
    }
    x_s[grp][c] = x;
    if (c == 0) l_s[grp] = L;
    __syncthreads();
    if (tid >= W / 4) return;
    L = 0.f;
    x = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < kGroups; ++k) {
        L += l_s[k];
        x += x_s[k][c];
    }
    store_row<D>(a, item, hk, row, (int)first + 4 * c, 1, 0, M, L, x);
}

// The same for up to MAXC chunks: a thread per (row, 4 dims), all of its loads on their way at once (those of slots past
// the row's chunks repeat the last).
template <int D, int MAXC, int RB> __device__ __forceinline__ void merge_few(const KvqArgs &a, int n_rows, int i) {
    const int at = i / (D / 4), c = i % (D / 4);
    if (at >= n_rows) return;
    const int last = a.max_chunks - 1;
    const float2 *ml = reinterpret_cast<const float2 *>(a.part_ml) + (int64_t)at * a.max_chunks;
    const f32x4 *po = reinterpret_cast<const f32x4 *>(a.part_o + (int64_t)at * a.max_chunks * D) + c;
    float2 s[MAXC];
    f32x4 x[MAXC];
#pragma unroll
    for (int k = 0; k < MAXC; ++k) {
        s[k] = ml[min(k, last)];
        x[k] = po[min(k, last) * (D / 4)];
    }
    const int ih = a.by_rows.of(at);
    const int row = at - ih * a.rows;
    const int item = a.by_heads.of(ih), hk = ih - item * a.view.n_head_kv;
    int chunk_keys;
    const int n_chunks = split(a, block_limit(a, item_kv(a, item), row / RB, RB), &chunk_keys);
    if (n_chunks == 1) return; // written by the attention kernel
    float M = -INFINITY, L = 0.f;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < MAXC; ++k)
        if (k < n_chunks) M = fmaxf(M, s[k].x);
#pragma unroll
    for (int k = 0; k < MAXC; ++k) {
        if (k >= n_chunks) continue; // the slots of other calls may hold anything
        const float f = M == -INFINITY ? 1.f : exp2_fast(s[k].x - M);
        L += f * s[k].y;
        sum += f * x[k];
    }
    store_row<D>(a, item, hk, row, 4 * c, 1, 0, M, L, sum);
}
template <int D, int MAXC, int RB> __global__ __launch_bounds__(256) void kvq_merge_few_kernel(KvqArgs a, int n_rows) {
    merge_few<D, MAXC, RB>(a, n_rows, (int)(blockIdx.x * 256 + threadIdx.x));
}

// Each key's probability summed over the rows that see it: a wave per 128 keys of a (sequence, KV head) keeps their codes in
// registers, goes over all row blocks in order, forms the scores again and adds exp2(s - M) / L in its lanes; the columns are
// added at the end.  Turning a row block into operands costs about what scoring 32 keys does, so it is done for 128.
constexpr int kWeightTiles = 4;
constexpr int kWeightKeys = kWeightTiles * kTile;

// JOIN: the rows' statistics are not there yet: they are formed from those of their chunks, at most kJoinChunks.
constexpr int kJoinChunks = 16;
template <int D, int FMT, bool PACKED, bool JOIN> __device__ __forceinline__ void weigh_keys(const KvqArgs &a, int unit, int piece) {
    constexpr int CT = 1;
    using G = Geo<D, CT, PACKED>;
    constexpr int RB = G::kRows;
    const KvqView &v = a.view;
    const int lane = threadIdx.x, g = lane >> 4, col = lane & 15;
    const int item = a.by_heads.of(unit), hk = unit - item * v.n_head_kv;
    const int k0 = piece * kWeightKeys;
    const int n_kv = item_kv(a, item);
    if (k0 >= n_kv) return;
    const int row_blocks = (a.rows + RB - 1) / RB;
    // causal rows from here on see a key of this wave
    int rb = 0;
    while (rb < row_blocks - 1 && block_limit(a, n_kv, rb, RB) <= k0) ++rb;
    typename Queries<D, CT, PACKED>::Raw raw;
    raw.load(a, item, hk, rb * RB, lane);
    const int64_t u = a.unit0 + (int64_t)item * v.n_head_kv + hk;
    const __amdgpu_buffer_rsrc_t keys = unit_codes(v.codes[0] + u * v.unit_bytes, v.unit_bytes);
    Codes<D> kt[kWeightTiles];
    Scales sk[kWeightTiles];
#pragma unroll
    for (int n = 0; n < kWeightTiles; ++n) {
        const int k = k0 + n * kTile;
        kt[n].load(keys, k < n_kv ? (uint32_t)k * D : kNoStep, lane);
        sk[n].load(v.scales[0] + u * v.n_blocks, k < n_kv ? k : k0, a.block_shift);
    }
    // the old weights, in the lanes that will write the keys' new ones
    float *w = a.weights + item * a.w_bstride + hk * a.w_stride;
    float old[kWeightTiles];
#pragma unroll
    for (int n = 0; n < kWeightTiles; ++n) {
        const int key = k0 + n * kTile + 16 * (col >> 2) + 4 * g + (col & 3);
        old[n] = a.decay != 0.f && col < 4 * kQ && key < n_kv ? w[key] : 0.f;
    }
    f32x4 acc[kWeightTiles][kQ];
#pragma unroll
    for (int n = 0; n < kWeightTiles; ++n)
#pragma unroll
        for (int q = 0; q < kQ; ++q) acc[n][q] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (; rb < row_blocks; ++rb) {
        const int r = rb * RB + (PACKED ? (col & 7) : col);
        const int lim = r < a.rows && (!PACKED || col < 8) ? row_limit(a, n_kv, r) : 0;
        float M = 0.f, inv = 0.f;
        if (lim > k0) {
            const int64_t at = row_at(a, item, hk, r);
            float2 ml;
            int chunk_keys, n_chunks = 1;
            if (JOIN) n_chunks = split(a, block_limit(a, n_kv, rb, RB), &chunk_keys); // RB: the attention kernel's too
            if (n_chunks == 1) {
                ml = *reinterpret_cast<const float2 *>(a.row_ml + 2 * at);
            } else {
                const float2 *part = reinterpret_cast<const float2 *>(a.part_ml) + at * a.max_chunks;
                float2 s[kJoinChunks];
#pragma unroll
                for (int k = 0; k < kJoinChunks; ++k) s[k] = part[min(k, n_chunks - 1)];
                ml = make_float2(-INFINITY, 0.f);
#pragma unroll
                for (int k = 0; k < kJoinChunks; ++k) ml.x = fmaxf(ml.x, s[k].x);
#pragma unroll
                for (int k = 0; k < kJoinChunks; ++k)
                    if (k < n_chunks) ml.y += (ml.x == -INFINITY ? 1.f : exp2_fast(s[k].x - ml.x)) * s[k].y;
            }
            M = ml.x;
            inv = ml.y != 0.f ? 1.f / ml.y : 0.f;
        }
        Queries<D, CT, PACKED> qs;
        qs.take(a, raw, lane);
        if (rb + 1 < row_blocks) raw.load(a, item, hk, (rb + 1) * RB, lane);
#pragma unroll
        for (int n = 0; n < kWeightTiles; ++n) {
            f32x4 s[CT][kQ];
            score_tile<D, FMT, CT, PACKED>(qs, kt[n], s);
#pragma unroll
            for (int q = 0; q < kQ; ++q) {
                const float f = qs.back[0] * sk[n].s[q];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float p = exp2_fast(__builtin_fmaf(s[0][q][i], f, -M)) * inv;
                    acc[n][q][i] += k0 + n * kTile + 16 * q + 4 * g + i < lim ? p : 0.f;
                }
            }
        }
    }
    // over the columns (8 rows: the first 8), all of which then have the sum: column 4 q + i writes key 16 q + 4 g + i
    static_assert(4 * kQ <= 8);
#pragma unroll
    for (int n = 0; n < kWeightTiles; ++n) {
        float mine = 0.f;
#pragma unroll
        for (int q = 0; q < kQ; ++q)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float x = acc[n][q][i];
                x += dpp_f32<0xb1>(x);  // quad_perm [1, 0, 3, 2]
                x += dpp_f32<0x4e>(x);  // quad_perm [2, 3, 0, 1]
                x += dpp_f32<0x141>(x); // row_half_mirror
                if (!PACKED) x += dpp_f32<0x140>(x); // row_mirror
                if (col == 4 * q + i) mine = x;
            }
        const int key = k0 + n * kTile + 16 * (col >> 2) + 4 * g + (col & 3);
        if (col < 4 * kQ && key < n_kv) w[key] = (a.decay != 0.f ? a.decay * old[n] : 0.f) + mine;
    }
}

template <int D, int FMT, bool PACKED> __global__ __launch_bounds__(64) void kvq_weights_kernel(KvqArgs a) {
    weigh_keys<D, FMT, PACKED, false>(a, blockIdx.x, blockIdx.y);
}
// Decode steps: merge and weights in one launch, the merge's workgroups first (merge_y rows of the grid), the weights' with
// statistics of their own.  One launch less and side by side: 32 sequences of 1 .. 4096 keys (d = 64) 18.9 -> 16.1 us a
// call.  With more rows the statistics would be joined again by each wave for each row block.
template <int D, int FMT> __global__ __launch_bounds__(64) void kvq_merge_weights_kernel(KvqArgs a, int n_rows, int merge_y) {
    if ((int)blockIdx.y < merge_y)
        merge_few<D, kJoinChunks, kKvqPackedRows>(a, n_rows, (int)((blockIdx.y * gridDim.x + blockIdx.x) * 64 + threadIdx.x));
    else
        weigh_keys<D, FMT, true, true>(a, blockIdx.x, (int)blockIdx.y - merge_y);
}

template <int D, int FMT, int CT, bool PACKED> hipError_t launch(const KvqArgs &a, bool prompt, hipStream_t stream) {
    constexpr int RB = Geo<D, CT, PACKED>::kRows;
    const uint64_t blocks = (uint64_t)a.per * a.n_seq * a.max_chunks;
    if (blocks * 64 * (prompt ? kPromptWaves : kWaves) > 0xffffffffull) return hipErrorInvalidValue; // a launch's threads
    if (prompt)
        kvq_prompt_kernel<D, FMT><<<(unsigned)blocks, 64 * kPromptWaves, 0, stream>>>(a);
    else
        kvq_attn_kernel<D, FMT, CT, PACKED><<<(unsigned)blocks, 64 * kWaves, 0, stream>>>(a);
    hipError_t e = hipGetLastError();
    const uint64_t rows = (uint64_t)a.n_seq * a.view.n_head_kv * a.rows;
    const uint64_t units = (uint64_t)a.view.n_head_kv * a.n_seq, pieces = ((uint64_t)a.n_kv + kWeightKeys - 1) / kWeightKeys;
    if constexpr (PACKED) {
        const uint64_t merge_y = (rows * (D / 4) + 64 * units - 1) / (64 * units); // at most 4
        if (e == hipSuccess && a.weights && a.max_chunks > 1 && a.max_chunks <= kJoinChunks && merge_y + pieces <= 65535) {
            kvq_merge_weights_kernel<D, FMT><<<dim3((unsigned)units, (unsigned)(merge_y + pieces)), 64, 0, stream>>>(a, (int)rows, (int)merge_y);
            return hipGetLastError();
        }
    }
    if (e == hipSuccess && a.max_chunks > 1) {
        const unsigned few = (unsigned)((rows * (D / 4) + 255) / 256);
#define ZWG_KVQ_MERGE(RB_)                                                                                         \
    if (a.max_chunks <= 4)                                                                                        \
        kvq_merge_few_kernel<D, 4, RB_><<<few, 256, 0, stream>>>(a, (int)rows);                                   \
    else if (a.max_chunks <= 8)                                                                                   \
        kvq_merge_few_kernel<D, 8, RB_><<<few, 256, 0, stream>>>(a, (int)rows);                                   \
    else if (a.max_chunks <= 16)                                                                                  \
        kvq_merge_few_kernel<D, 16, RB_><<<few, 256, 0, stream>>>(a, (int)rows);                                  \
    else if (a.max_chunks <= kManyChunks)                                                                         \
        kvq_merge_kernel<D, D, RB_><<<(unsigned)rows, 256, 0, stream>>>(a);                                       \
    else                                                                                                          \
        kvq_merge_kernel<D, 16, RB_><<<(unsigned)(rows * (D / 16)), 256, 0, stream>>>(a);
        if (prompt) {
            ZWG_KVQ_MERGE(kPromptRows)
        } else {
            ZWG_KVQ_MERGE(RB)
        }
#undef ZWG_KVQ_MERGE
        e = hipGetLastError();
    }
    if (e == hipSuccess && a.weights && a.n_kv > 0) {
        const dim3 grid((unsigned)units, (unsigned)pieces);
        kvq_weights_kernel<D, FMT, PACKED><<<grid, 64, 0, stream>>>(a);
        e = hipGetLastError();
    }
    return e;
}

template <int D, int FMT> hipError_t launch_rows(const KvqArgs &a, bool prompt, hipStream_t stream) {
    return a.rows <= kKvqPackedRows ? launch<D, FMT, 1, true>(a, false, stream) : launch<D, FMT, 2, false>(a, prompt, stream);
}

int attention(zwg_kvq *kv, uint64_t layer, uint64_t seq0, uint64_t n_seq, const float *q, const zwg_kvq_attn &s,
              float *out, float *weights) {
    zwg_ctx *ctx = kv->ctx;
    const zwg_kvq_desc &d = kv->desc;
    const std::string msg = check_kvq_attn(d, layer, seq0, n_seq, q, s, out, weights);
    if (!msg.empty()) return fail(ctx, msg);
    if (n_seq == 0 || s.n_q == 0) return ZWG_OK;
    if (out == q || (weights && (weights == out || weights == q))) return fail(ctx, "q, out and weights must not be the same memory");
    const uint64_t group = s.n_head / d.n_head_kv, rows = s.n_q * group;
    hipError_t e = hipSetDevice(ctx->device);
    if (e != hipSuccess) return fail_hip(ctx, "hipSetDevice", e);

    const bool prompt = rows > kKvqPackedRows && kvq_prompt(rows, n_seq * d.n_head_kv, s.n_kv);
    const uint64_t RB = rows <= kKvqPackedRows ? 8 : prompt ? kPromptRows : 32;
    const uint64_t n_rows = n_seq * d.n_head_kv * rows, row_blocks = (rows + RB - 1) / RB;
    const KvqSplit sp = kvq_split(n_seq * d.n_head_kv * row_blocks, s.n_kv, n_rows, d.d, weights != nullptr, ctx->workspace_bytes, prompt);
    const KvqWorkspace ws = kvq_workspace(n_rows, (uint64_t)sp.max_chunks, d.d, weights != nullptr);
    if (ws.total * sizeof(float) > ctx->workspace_bytes)
        return fail(ctx, "the context's workspace is smaller than the rows' statistics (weights)");

    KvqArgs a{};
    a.view = kv->view;
    a.unit0 = (int64_t)((layer * d.n_seq + seq0) * d.n_head_kv);
    a.q = q;
    a.out = out;
    a.q_stride = (int64_t)s.q_stride;
    a.q_bstride = (int64_t)s.q_bstride;
    a.out_stride = (int64_t)s.out_stride;
    a.out_bstride = (int64_t)s.out_bstride;
    a.n_kv_dev = s.n_kv_dev;
    a.n_seq = (int32_t)n_seq;
    a.n_q = (int32_t)s.n_q;
    a.n_kv = (int32_t)s.n_kv;
    a.n_head = (int32_t)s.n_head;
    a.group = (int32_t)group;
    a.rows = (int32_t)rows;
    a.row_blocks = (int32_t)row_blocks;
    a.causal = (int32_t)s.causal;
    a.scale_log2 = (1.0f / std::sqrt((float)d.d)) * 1.4426950408889634f;
    a.tau = sp.chunk_len / kSplitTile;
    a.per = (int32_t)(d.n_head_kv * row_blocks);
    a.by_group = Div((uint32_t)group);
    a.by_heads = Div((uint32_t)d.n_head_kv);
    a.by_per = Div((uint32_t)a.per);
    a.by_seqs = Div((uint32_t)n_seq);
    a.by_tau = Div((uint32_t)a.tau);
    a.by_rows = Div((uint32_t)rows);
    a.max_chunks = sp.max_chunks;
    a.block_shift = d.block == 16 ? 4 : d.block == 32 ? 5 : 6;
    a.row_ml = weights ? ctx->workspace : nullptr;
    a.part_ml = ctx->workspace + ws.part_ml;
    a.part_o = ctx->workspace + ws.part_o;
    a.weights = weights;
    a.w_stride = (int64_t)s.weights_stride;
    a.w_bstride = (int64_t)s.weights_bstride;
    a.decay = s.decay;
    switch (d.d) {
    case 32: e = d.format == ZWG_KVQ_I8 ? launch_rows<32, 0>(a, prompt, ctx->stream) : launch_rows<32, 1>(a, prompt, ctx->stream); break;
    case 64: e = d.format == ZWG_KVQ_I8 ? launch_rows<64, 0>(a, prompt, ctx->stream) : launch_rows<64, 1>(a, prompt, ctx->stream); break;
    default: e = d.format == ZWG_KVQ_I8 ? launch_rows<128, 0>(a, prompt, ctx->stream) : launch_rows<128, 1>(a, prompt, ctx->stream); break;
    }
    return e == hipSuccess ? ZWG_OK : fail_hip(ctx, "kvq attention launch", e);
}

} // namespace

extern "C" int zwg_kvq_attention_dev(zwg_kvq *kv, uint64_t layer, uint64_t seq0, uint64_t n_seq, const float *q,
                                     const zwg_kvq_attn *attn, float *out, float *weights) {
    if (!kv) return fail(nullptr, "null kvq");
    if (!kv->ctx) return fail(nullptr, "the kvq cache's context is closed");
    if (!attn) return fail(kv->ctx, "null attention shape");
    return guarded(kv->ctx, [&] { return attention(kv, layer, seq0, n_seq, q, *attn, out, weights); });
}
