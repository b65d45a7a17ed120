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
// 8 (l / 16) .. + 7, and of the result rows 4 (l / 16) .. + 3 of column l % 16.  A lane's 16 bytes of a key row are
// two A operands; its scores (column l % 16, keys 16 q + 4 (l / 16) + i) are the B operand of the value product for
// values stored in that order of keys (kvq_v_slot), so probabilities never leave the lane that made them.
//
// Few query rows (up to 8 share a KV head: a decode step): the 16 columns are 8 rows' hi terms and the same rows' lo
// terms, and one product gives both.  More rows: 32 to a wave in two tiles, hi and lo as products of their own.
//
// The maximum is a lazy one: a column's reference rises only when some score passes it by kSlack = 8 (log2 units),
// so most tiles need no exchange between lanes and no rescaling.
//
// A workgroup's four waves take every fourth tile of 64 keys of one chunk and merge in LDS; chunks of one row
// are merged by kvq_merge_kernel in their order.
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
constexpr float kSlack = 8.0f;
constexpr float kProbScale = 64.0f; // 2^6: p * (sv / ref) * 2^6 <= 2^8 * 2 * 2^6

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
    int32_t chunk_len, max_chunks;
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
    return a.causal ? max(0, n_kv - a.n_q + r / a.group + 1) : n_kv;
}
// Keys that the last row of row block rb sees.
__device__ __forceinline__ int block_limit(const KvqArgs &a, int n_kv, int rb, int RB) {
    return row_limit(a, n_kv, min(a.rows, (rb + 1) * RB) - 1);
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

// x of the lane 8 columns away (l ^ 8 within its row of 16).
__device__ __forceinline__ float other_half(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x128, 0xf, 0xf, true));
}
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

    __device__ __forceinline__ void load(const KvqArgs &a, int item, int hk, int r0, int lane) {
        const int g = lane >> 4, col = lane & 15;
#pragma unroll
        for (int t = 0; t < CT; ++t) {
            const int r = r0 + (PACKED ? (col & 7) : 16 * t + col);
            float x[G::kSteps][8];
            uint32_t top = 0;
            const bool live = r < a.rows;
            const int qi = live ? r / a.group : 0;
            const float *q = a.q + item * a.q_bstride + qi * a.q_stride + (int64_t)(hk * a.group + (live ? r - qi * a.group : 0)) * D;
#pragma unroll
            for (int s = 0; s < G::kSteps; ++s)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const f32x4 v = live ? *reinterpret_cast<const f32x4 *>(q + at_dim(s, g) + 4 * h) : (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x[s][4 * h + e] = v[e];
                        top = max(top, abs_bits(v[e]));
                    }
                }
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
                    const float v = x[s][k] * up;
                    const _Float16 hi = (_Float16)v;
                    const _Float16 lo = (_Float16)(v - (float)hi);
                    if (PACKED) {
                        frag[t][0][s][k] = col < 8 ? hi : lo;
                    } else {
                        frag[t][0][s][k] = hi;
                        frag[t][G::kParts - 1][s][k] = lo;
                    }
                }
        }
    }
};

// 64 keys' codes: of the key tile q (16 keys) step s's operand.
template <int D> struct KeyTile {
    u32x4 w[4][D == 32 ? 1 : D / 64];
    __device__ __forceinline__ void load(const uint8_t *keys, int lane) {
        const int g = lane >> 4, row = lane & 15;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const uint8_t *p = keys + (16 * q + row) * D;
            if (D == 32) {
                const u32x2 v = __builtin_nontemporal_load(reinterpret_cast<const u32x2 *>(p + 8 * g));
                w[q][0] = (u32x4){v[0], v[1], 0u, 0u};
            } else {
#pragma unroll
                for (int h = 0; h < (D == 32 ? 1 : D / 64); ++h)
                    w[q][h] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p + 64 * h + 16 * g));
            }
        }
    }
    __device__ __forceinline__ u32x2 step(int q, int s) const {
        const u32x4 v = w[q][D == 32 ? 0 : s >> 1];
        return s & 1 ? (u32x2){v[2], v[3]} : (u32x2){v[0], v[1]};
    }
};

// The scores of 64 keys, log2 units, unmasked: column tile t, key tile q.
template <int D, int FMT, int CT, bool PACKED>
__device__ __forceinline__ void score_tile(const Queries<D, CT, PACKED> &qs, const KeyTile<D> &kt, const float *ks, int block,
                                           int k0, f32x4 (&s)[CT][4]) {
    using G = Geo<D, CT, PACKED>;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        f32x4 acc[CT];
#pragma unroll
        for (int t = 0; t < CT; ++t) acc[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < G::kSteps; ++st) {
            const f16x8 k = codes_f16<FMT>(kt.step(q, st));
#pragma unroll
            for (int t = 0; t < CT; ++t)
#pragma unroll
                for (int p = 0; p < G::kParts; ++p)
                    acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qs.frag[t][p][st], acc[t], 0, 0, 0);
        }
        const float sk = ks[(k0 + 16 * q) / block];
#pragma unroll
        for (int t = 0; t < CT; ++t) {
            const float f = qs.back[t] * sk;
#pragma unroll
            for (int i = 0; i < 4; ++i) s[t][q][i] = (PACKED ? acc[t][i] + other_half(acc[t][i]) : acc[t][i]) * f;
        }
    }
}

template <int D, int FMT, int CT, bool PACKED>
__global__ __launch_bounds__(64 * kWaves) void kvq_attn_kernel(KvqArgs a) {
    using G = Geo<D, CT, PACKED>;
    constexpr int RB = G::kRows;
    __shared__ __align__(16) float o_s[kWaves][RB][D + 4];
    __shared__ float m_s[kWaves][RB], l_s[kWaves][RB];

    const KvqView &v = a.view;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int g = lane >> 4, col = lane & 15;
    // chunk slowest, so that the long sequences' work starts everywhere at once
    int64_t b = blockIdx.x;
    const int hk = (int)(b % v.n_head_kv);
    b /= v.n_head_kv;
    const int rb = (int)(b % a.row_blocks);
    b /= a.row_blocks;
    const int item = (int)(b % a.n_seq);
    const int chunk = (int)(b / a.n_seq);

    const int n_kv = item_kv(a, item);
    const int hi = block_limit(a, n_kv, rb, RB);
    int chunk_keys;
    const int n_chunks = zwg::unit_split(hi, kSplitTile, a.chunk_len, a.max_chunks, &chunk_keys);
    if (chunk >= n_chunks) return;
    const int k_begin = chunk * chunk_keys, k_end = min(hi, k_begin + chunk_keys);

    const int64_t u = a.unit0 + (int64_t)item * v.n_head_kv + hk;
    const uint8_t *keys = v.codes[0] + u * v.unit_bytes;
    const uint8_t *vals = v.codes[1] + u * v.unit_bytes;
    const float *ks = v.scales[0] + u * v.n_blocks, *vs = v.scales[1] + u * v.n_blocks;

    Queries<D, CT, PACKED> qs;
    qs.load(a, item, hk, rb * RB, lane);
    int lim[CT];
#pragma unroll
    for (int t = 0; t < CT; ++t) {
        const int r = rb * RB + (PACKED ? (col & 7) : 16 * t + col);
        lim[t] = r < a.rows ? min(k_end, row_limit(a, n_kv, r)) : 0;
    }
    // the smallest limit of the block's rows: tiles below it need no mask (a block's rows behind the last have
    // zero queries: what they compute is not stored)
    const int lim_all = min(k_end, row_limit(a, n_kv, rb * RB));

    float m[CT], l[CT], ref = 0.f;
    f32x4 o[CT][G::kDims];
#pragma unroll
    for (int t = 0; t < CT; ++t) {
        m[t] = -INFINITY;
        l[t] = 0.f;
#pragma unroll
        for (int d = 0; d < G::kDims; ++d) o[t][d] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }

#pragma unroll 1
    for (int k0 = k_begin + wave * kTile; k0 < k_end; k0 += kSplitTile) {
        KeyTile<D> kt;
        kt.load(keys + (int64_t)k0 * D, lane);
        u32x4 vt[G::kDims];
#pragma unroll
        for (int d = 0; d < G::kDims; ++d)
            vt[d] = __builtin_nontemporal_load(
                reinterpret_cast<const u32x4 *>(vals + (int64_t)k0 * D + (16 * d + col) * 64 + 16 * g));
        f32x4 s[CT][4];
        score_tile<D, FMT, CT, PACKED>(qs, kt, ks, v.block, k0, s);
        const bool mask = k0 + kTile > lim_all;
        if (mask) {
#pragma unroll
            for (int t = 0; t < CT; ++t)
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (k0 + 16 * q + 4 * g + i >= lim[t]) s[t][q][i] = -INFINITY;
        }
        // the reference maxima, raised when a score passes one by kSlack
        float top[CT];
        bool rise = false;
#pragma unroll
        for (int t = 0; t < CT; ++t) {
            top[t] = -INFINITY;
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int i = 0; i < 4; ++i) top[t] = fmaxf(top[t], s[t][q][i]);
            rise |= top[t] > m[t] + kSlack;
        }
        if (__any(rise)) {
#pragma unroll
            for (int t = 0; t < CT; ++t) {
                const float m_new = fmaxf(m[t], groups_max(top[t]));
                const float alpha = m_new == -INFINITY ? 1.f : exp2_fast(m[t] - m_new);
                m[t] = m_new;
                l[t] *= alpha;
#pragma unroll
                for (int d = 0; d < G::kDims; ++d) o[t][d] *= alpha;
            }
        }
        // the value scales relative to a power of two at most the largest met (NaNs aside)
        float sv[4], big = ref;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            // blocks behind the last visible key count for nothing, whatever they hold
            sv[q] = k0 + 16 * q < k_end ? vs[(k0 + 16 * q) / v.block] : 0.f;
            big = fmaxf(big, sv[q]);
        }
        const float ref_new = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, big) & 0x7f800000u);
        if (ref_new != ref) {
            const float down = ref / ref_new; // powers of two: exact
#pragma unroll
            for (int t = 0; t < CT; ++t)
#pragma unroll
                for (int d = 0; d < G::kDims; ++d) o[t][d] *= down;
            ref = ref_new;
        }
        const float inv_ref = ref > 0.f ? kProbScale / ref : 0.f;
#pragma unroll
        for (int q = 0; q < 4; ++q) sv[q] *= inv_ref;

        f16x8 pf[CT][G::kParts][2];
#pragma unroll
        for (int t = 0; t < CT; ++t) {
            const float mu = m[t] == -INFINITY ? 0.f : m[t];
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float p = exp2_fast(s[t][q][i] - mu);
                    l[t] += p;
                    float w = p * sv[q];
                    // a masked key's block may have a NaN scale
                    if (mask && k0 + 16 * q + 4 * g + i >= lim[t]) w = 0.f;
                    const _Float16 h = (_Float16)w;
                    const _Float16 r = (_Float16)(w - (float)h);
                    const int j = q >> 1, e = 4 * (q & 1) + i;
                    if (PACKED) {
                        pf[t][0][j][e] = col < 8 ? h : r;
                    } else {
                        pf[t][0][j][e] = h;
                        pf[t][G::kParts - 1][j][e] = r;
                    }
                }
        }
#pragma unroll
        for (int d = 0; d < G::kDims; ++d)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const f16x8 vf = codes_f16<FMT>(j ? (u32x2){vt[d][2], vt[d][3]} : (u32x2){vt[d][0], vt[d][1]});
#pragma unroll
                for (int t = 0; t < CT; ++t)
#pragma unroll
                    for (int p = 0; p < G::kParts; ++p)
                        o[t][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[t][p][j], o[t][d], 0, 0, 0);
            }
    }

    // ---- the waves' results merged in LDS
    const float unit = ref * (1.0f / kProbScale);
#pragma unroll
    for (int t = 0; t < CT; ++t) {
        const float lt = groups_sum(l[t]);
        const int r = PACKED ? (col & 7) : 16 * t + col;
        const bool writes = !PACKED || col < 8;
        if (writes && g == 0) {
            m_s[wave][r] = m[t];
            l_s[wave][r] = lt;
        }
#pragma unroll
        for (int d = 0; d < G::kDims; ++d) {
            f32x4 x = o[t][d];
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
        if (M != -INFINITY) {
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const float f = exp2_fast(m_s[w][r] - M); // 0 for a wave that saw no key of this row
                L += f * l_s[w][r];
                x += f * *reinterpret_cast<const f32x4 *>(&o_s[w][r][c]);
            }
        } else {
#pragma unroll
            for (int w = 0; w < kWaves; ++w) L += l_s[w][r]; // no key seen: 0; scores that are no numbers: NaN
        }
        const int64_t at = row_at(a, item, hk, row);
        if (n_chunks == 1) {
            const int qi = row / a.group, head = hk * a.group + row - qi * a.group;
            const float inv = L != 0.f ? 1.f / L : 0.f; // a NaN stays one
            *reinterpret_cast<f32x4 *>(a.out + item * a.out_bstride + qi * a.out_stride + (int64_t)head * D + c) = x * inv;
            if (a.row_ml && c == 0) {
                a.row_ml[2 * at] = M;
                a.row_ml[2 * at + 1] = L;
            }
        } else {
            const int64_t slot = at * a.max_chunks + chunk;
            *reinterpret_cast<f32x4 *>(a.part_o + slot * D + c) = x;
            if (c == 0) {
                a.part_ml[2 * slot] = M;
                a.part_ml[2 * slot + 1] = L;
            }
        }
    }
}

// The chunks of each row, in their order: a thread per (row, 4 dims).
template <int D, int RB> __global__ __launch_bounds__(256) void kvq_merge_kernel(KvqArgs a, int64_t n_rows) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t at = i / (D / 4);
    const int c = 4 * (int)(i % (D / 4));
    if (at >= n_rows) return;
    const int row = (int)(at % a.rows);
    const int64_t ih = at / a.rows;
    const int hk = (int)(ih % a.view.n_head_kv), item = (int)(ih / a.view.n_head_kv);
    int chunk_keys;
    const int n_chunks = zwg::unit_split(block_limit(a, item_kv(a, item), row / RB, RB), kSplitTile, a.chunk_len, a.max_chunks, &chunk_keys);
    if (n_chunks == 1) return; // written by the attention kernel
    const float *ml = a.part_ml + 2 * at * a.max_chunks;
    float M = -INFINITY;
    for (int k = 0; k < n_chunks; ++k) M = fmaxf(M, ml[2 * k]);
    float L = 0.f;
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < n_chunks; ++k) {
        const float f = M == -INFINITY ? 1.f : exp2_fast(ml[2 * k] - M);
        L += f * ml[2 * k + 1];
        x += f * *reinterpret_cast<const f32x4 *>(a.part_o + (at * a.max_chunks + k) * D + c);
    }
    const int qi = row / a.group, head = hk * a.group + row - qi * a.group;
    const float inv = L != 0.f ? 1.f / L : 0.f;
    *reinterpret_cast<f32x4 *>(a.out + item * a.out_bstride + qi * a.out_stride + (int64_t)head * D + c) = x * inv;
    if (a.row_ml && c == 0) {
        a.row_ml[2 * at] = M;
        a.row_ml[2 * at + 1] = L;
    }
}

// Each key's probability summed over the rows that see it: a wave per 64 keys of a (sequence, KV head) goes over all
// row blocks in order, forms the scores again and adds exp2(s - M) / L in its lanes; the columns are added at the end.
template <int D, int FMT, int CT, bool PACKED>
__global__ __launch_bounds__(64) void kvq_weights_kernel(KvqArgs a) {
    using G = Geo<D, CT, PACKED>;
    constexpr int RB = G::kRows;
    const KvqView &v = a.view;
    const int lane = threadIdx.x, g = lane >> 4, col = lane & 15;
    const int hk = blockIdx.x % v.n_head_kv, item = blockIdx.x / v.n_head_kv;
    const int k0 = blockIdx.y * kTile;
    const int n_kv = item_kv(a, item);
    if (k0 >= n_kv) return;
    const int64_t u = a.unit0 + (int64_t)item * v.n_head_kv + hk;
    KeyTile<D> kt;
    kt.load(v.codes[0] + u * v.unit_bytes + (int64_t)k0 * D, lane);
    const float *ks = v.scales[0] + u * v.n_blocks;
    f32x4 acc[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) acc[q] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int rb = 0; rb < a.row_blocks; ++rb) {
        if (block_limit(a, n_kv, rb, RB) <= k0) continue;
        Queries<D, CT, PACKED> qs;
        qs.load(a, item, hk, rb * RB, lane);
        f32x4 s[CT][4];
        score_tile<D, FMT, CT, PACKED>(qs, kt, ks, v.block, k0, s);
#pragma unroll
        for (int t = 0; t < CT; ++t) {
            const int r = rb * RB + (PACKED ? (col & 7) : 16 * t + col);
            const int lim = r < a.rows && (!PACKED || col < 8) ? row_limit(a, n_kv, r) : 0;
            float M = 0.f, inv = 0.f;
            if (lim > k0) {
                const float *ml = a.row_ml + 2 * row_at(a, item, hk, r);
                M = ml[0];
                inv = ml[1] != 0.f ? 1.f / ml[1] : 0.f;
            }
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (k0 + 16 * q + 4 * g + i < lim) acc[q][i] += exp2_fast(s[t][q][i] - M) * inv;
        }
    }
    // over the 16 columns
    float *w = a.weights + item * a.w_bstride + hk * a.w_stride;
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float x = acc[q][i];
#pragma unroll
            for (int off = 1; off < 16; off <<= 1) x += __shfl_xor(x, off);
            const int key = k0 + 16 * q + 4 * g + i;
            // column 4 q + i of the group writes this key
            if (col == 4 * q + i && key < n_kv) w[key] = (a.decay != 0.f ? a.decay * w[key] : 0.f) + x;
        }
}

template <int D, int FMT, int CT, bool PACKED> hipError_t launch(const KvqArgs &a, hipStream_t stream) {
    constexpr int RB = Geo<D, CT, PACKED>::kRows;
    const uint64_t blocks = (uint64_t)a.view.n_head_kv * a.row_blocks * a.n_seq * a.max_chunks;
    if (blocks > 0x7fffffffull) return hipErrorInvalidValue;
    kvq_attn_kernel<D, FMT, CT, PACKED><<<(unsigned)blocks, 64 * kWaves, 0, stream>>>(a);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && a.max_chunks > 1) {
        const int64_t rows = (int64_t)a.n_seq * a.view.n_head_kv * a.rows;
        kvq_merge_kernel<D, RB><<<(unsigned)((rows * (D / 4) + 255) / 256), 256, 0, stream>>>(a, rows);
        e = hipGetLastError();
    }
    if (e == hipSuccess && a.weights && a.n_kv > 0) {
        const dim3 grid((unsigned)(a.view.n_head_kv * a.n_seq), (unsigned)((a.n_kv + kTile - 1) / kTile));
        kvq_weights_kernel<D, FMT, CT, PACKED><<<grid, 64, 0, stream>>>(a);
        e = hipGetLastError();
    }
    return e;
}

template <int D, int FMT> hipError_t launch_rows(const KvqArgs &a, hipStream_t stream) {
    return a.rows <= kKvqPackedRows ? launch<D, FMT, 1, true>(a, stream) : launch<D, FMT, 2, false>(a, stream);
}

int attention(zwg_kvq *kv, uint64_t layer, uint64_t seq0, uint64_t n_seq, const float *q, const zwg_kvq_attn &s,
              float *out, float *weights) {
    zwg_ctx *ctx = kv->ctx;
    const zwg_kvq_desc &d = kv->desc;
    const std::string msg = check_kvq_attn(d, layer, seq0, n_seq, q, s, out, weights);
    if (!msg.empty()) return fail(ctx, msg);
    if (n_seq == 0 || s.n_q == 0) return ZWG_OK;
    const uint64_t group = s.n_head / d.n_head_kv, rows = s.n_q * group;
    hipError_t e = hipSetDevice(ctx->device);
    if (e != hipSuccess) return fail_hip(ctx, "hipSetDevice", e);

    const uint64_t RB = rows <= kKvqPackedRows ? 8 : 32;
    const uint64_t n_rows = n_seq * d.n_head_kv * rows, row_blocks = (rows + RB - 1) / RB;
    const KvqSplit sp = kvq_split(n_seq * d.n_head_kv * row_blocks, s.n_kv, n_rows, d.d, weights != nullptr, ctx->workspace_bytes);
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
    a.chunk_len = sp.chunk_len;
    a.max_chunks = sp.max_chunks;
    a.row_ml = weights ? ctx->workspace : nullptr;
    a.part_ml = ctx->workspace + ws.part_ml;
    a.part_o = ctx->workspace + ws.part_o;
    a.weights = weights;
    a.w_stride = (int64_t)s.weights_stride;
    a.w_bstride = (int64_t)s.weights_bstride;
    a.decay = s.decay;
    switch (d.d) {
    case 32: e = d.format == ZWG_KVQ_I8 ? launch_rows<32, 0>(a, ctx->stream) : launch_rows<32, 1>(a, ctx->stream); break;
    case 64: e = d.format == ZWG_KVQ_I8 ? launch_rows<64, 0>(a, ctx->stream) : launch_rows<64, 1>(a, ctx->stream); break;
    default: e = d.format == ZWG_KVQ_I8 ? launch_rows<128, 0>(a, ctx->stream) : launch_rows<128, 1>(a, ctx->stream); break;
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
