// Host side of the rotary positions and the 8-bit caches (include/zw_gpu.h, zwg_rope_*, zwg_kvq_*): the argument
// rules, the layout in memory and the key splits.  Plain C++ (no HIP headers), so it is also built on its own, under
// the address / undefined-behaviour sanitizers (tests/cpp/test_kvq_plan.cpp).
#pragma once

#include <stdint.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <string>
#include <vector>

#include "attn_geometry.hpp"
#include "zw_gpu.h"

#ifdef __HIPCC__
#define ZWG_KVQ_HD __host__ __device__
#else
#define ZWG_KVQ_HD
#endif

namespace zwg {

constexpr int kKvqTile = 32; // keys of a wave's step
constexpr int kKvqPad = 64;  // a unit's tokens are padded to whole scale blocks of any size
constexpr int kKvqMaxBlock = 64;

// Byte offset of (token, dim) in a unit's keys or values: KBs that a wave's 64 lanes read together, 16 bytes a lane, two
// operands of 8 codes each.  Lane 16 g + c reads, at 64 c + 16 g,
//   keys    of 16 tokens and 64 dims (d 64 and 128): token c's dims 16 g .. 16 g + 15; at d = 32, of 32 tokens: dims
//           8 g .. 8 g + 7 of tokens c and 16 + c
//   values  of 32 tokens and 32 dims: dims c and 16 + c of tokens 4 g .. 4 g + 3 and 16 + 4 g .. 16 + 4 g + 3 (the keys
//           whose scores the lane holds after the score products)
ZWG_KVQ_HD constexpr int64_t kvq_at(int is_v, int64_t token, int dim, int d) {
    const int t = (int)(token & 31);
    if (is_v)
        return (token >> 5) * 32 * d + (dim >> 5) * 1024 + (dim & 15) * 64 + ((t >> 2) & 3) * 16 + ((dim >> 4) & 1) * 8 +
               (t >> 4) * 4 + (t & 3);
    if (d == 32) return (token >> 5) * 1024 + (dim >> 3) * 16 + (t & 15) * 64 + (t >> 4) * 8 + (dim & 7);
    return (token >> 4) * 16 * d + (dim >> 6) * 1024 + (t & 15) * 64 + (dim & 63);
}

// What of an open block is held, keys and values each (they are written by different workgroups).
struct KvqOpen {
    int32_t block;           // its index, -1: none
    int32_t filled;          // rows 0 .. filled - 1 are held
    float top[kKvqMaxBlock]; // each held row's largest magnitude
};

} // namespace zwg

namespace zwg_planner {

constexpr uint64_t kMaxStride = 1ull << 40;

inline bool off(const void *p, uintptr_t mask) { return (reinterpret_cast<uintptr_t>(p) & mask) != 0; }

// ---- rotary positions

inline std::string check_rope_desc(const zwg_rope_desc &d) {
    if (d.layout > ZWG_ROPE_INTERLEAVED) return "rope layout must be ZWG_ROPE_HALF or ZWG_ROPE_INTERLEAVED";
    if (d.scaling > ZWG_ROPE_YARN) return "unknown rope scaling";
    if (d.d == 0 || d.d % 4 || d.d > 1024) return "rope head dim d must be a multiple of 4 up to 1024";
    if (d.n_rot < 2 || d.n_rot % 2 || d.n_rot > d.d) return "n_rot must be even, 2 .. d";
    if (d.n_ctx == 0 || d.n_ctx > 0x7fffffffull / d.n_rot) return "rope n_ctx must be positive and below 2^31 / n_rot";
    if (!(d.base > 0.0) || !std::isfinite(d.base)) return "rope base must be positive and finite";
    if (!(d.factor >= 1.0) || !std::isfinite(d.factor)) return "rope factor must be at least 1 and finite";
    if (d.scaling == ZWG_ROPE_NONE && d.factor != 1.0) return "an unscaled rope has factor 1";
    if (d.scaling == ZWG_ROPE_NTK && d.n_rot < 4) return "NTK scaling needs n_rot of at least 4";
    if (!(d.mscale >= 0.0) || !std::isfinite(d.mscale)) return "mscale must be finite and >= 0";
    if (d.scaling == ZWG_ROPE_YARN) {
        if (d.n_orig == 0) return "YARN scaling needs n_orig, the trained positions";
        const double fast = d.beta_fast != 0.0 ? d.beta_fast : 32.0, slow = d.beta_slow != 0.0 ? d.beta_slow : 1.0;
        if (!(slow > 0.0) || !(fast > slow) || !std::isfinite(fast)) return "YARN needs 0 < beta_slow < beta_fast";
    }
    return "";
}

// The pairs' frequencies, in f64, and the factor on cos and sin.
inline std::vector<double> rope_frequencies(const zwg_rope_desc &d) {
    std::vector<double> w(d.n_rot / 2);
    const double n = (double)d.n_rot;
    const double base = d.scaling == ZWG_ROPE_NTK ? d.base * std::pow(d.factor, n / (n - 2.0)) : d.base;
    const double fast = d.beta_fast != 0.0 ? d.beta_fast : 32.0, slow = d.beta_slow != 0.0 ? d.beta_slow : 1.0;
    for (size_t j = 0; j < w.size(); ++j) {
        // as the f32 cache's tables (src/llm.zig:131-137): 1 / base^(2j / n_rot)
        w[j] = 1.0 / std::pow(base, (double)(2 * j) / n);
        if (d.scaling == ZWG_ROPE_LINEAR) w[j] /= d.factor;
        if (d.scaling == ZWG_ROPE_YARN) {
            const double turns = (double)d.n_orig * w[j] / (2.0 * 3.14159265358979323846);
            const double g = std::min(1.0, std::max(0.0, (turns - slow) / (fast - slow)));
            w[j] = g * w[j] + (1.0 - g) * (w[j] / d.factor);
        }
    }
    return w;
}
inline double rope_mscale(const zwg_rope_desc &d) {
    if (d.mscale != 0.0) return d.mscale;
    return d.scaling == ZWG_ROPE_YARN && d.factor > 1.0 ? 0.1 * std::log(d.factor) + 1.0 : 1.0;
}

inline std::string check_rope_apply(const zwg_rope_desc &d, const float *x, uint64_t n, uint64_t n_head, uint64_t x_stride,
                                    const int32_t *pos_dev, uint64_t pos0, const float *out, uint64_t out_stride,
                                    uint32_t flags) {
    if (flags & ~ZWG_ROPE_INVERSE) return "unknown rope flags";
    if (n == 0) return "";
    if (!x || !out) return "null x or out";
    if (off(x, 15) || off(out, 15)) return "x and out must be 16-byte aligned";
    if (off(pos_dev, 3)) return "pos_dev must be 4-byte aligned";
    if (n_head == 0 || n_head > 65535) return "n_head must be in 1 .. 65535";
    if (n > 0x7fffffffull) return "too many rows";
    if (x_stride % 4 || out_stride % 4) return "x_stride and out_stride must be multiples of 4 floats";
    if (n > 1 && (x_stride < n_head * d.d || out_stride < n_head * d.d)) return "a row stride is smaller than n_head * d";
    if (x_stride > kMaxStride || out_stride > kMaxStride) return "a row stride is out of range";
    if (!pos_dev && (pos0 > d.n_ctx || n > d.n_ctx - pos0)) return "pos0 + n is past the rope's n_ctx";
    if (x == out) return n > 1 && x_stride != out_stride ? "in place, x_stride and out_stride must be equal" : "";
    // rows may interleave (queries and keys of one buffer), so of the overlaps only one of the first rows is
    // certain to be wrong
    const uintptr_t xb = reinterpret_cast<uintptr_t>(x), ob = reinterpret_cast<uintptr_t>(out);
    const uint64_t row = n_head * d.d * sizeof(float);
    return (ob > xb && ob - xb < row) || (xb > ob && xb - ob < row) ? "x and out overlap" : "";
}

// ---- 8-bit caches

inline std::string check_kvq_desc(const zwg_kvq_desc &d) {
    if (d.reserved != 0) return "kvq desc.reserved must be 0";
    if (d.format != ZWG_KVQ_I8 && d.format != ZWG_KVQ_E4M3) return "kvq format must be ZWG_KVQ_I8 or ZWG_KVQ_E4M3";
    if (d.d != 32 && d.d != 64 && d.d != 128) return "kvq head dim d must be 32, 64 or 128";
    if (d.block != 16 && d.block != 32 && d.block != 64) return "kvq block must be 16, 32 or 64 tokens";
    if (d.n_layer == 0 || d.n_seq == 0 || d.n_ctx == 0 || d.n_head_kv == 0)
        return "kvq n_layer, n_seq, n_ctx and n_head_kv must be positive";
    if (d.n_layer > 65535 || d.n_seq > 65535 || d.n_head_kv > 4096) return "kvq sizes out of range";
    if (d.n_layer * d.n_seq * d.n_head_kv > 0x7fffffffull) return "kvq n_layer * n_seq * n_head_kv must be below 2^31";
    if (d.n_ctx >= (0x7fffffffull - (1ull << 20)) / d.d) return "kvq n_ctx * d must be below 2^31 - 2^20";
    return "";
}

// One allocation: codes, scales and open rows (keys then values each), then the open blocks' states.  Bytes.
struct KvqLayout {
    uint64_t units, n_pad, codes, scales, rows, open, total;
};

inline KvqLayout kvq_layout(const zwg_kvq_desc &d) {
    const auto up256 = [](uint64_t x) { return (x + 255) / 256 * 256; };
    KvqLayout l{};
    l.units = d.n_layer * d.n_seq * d.n_head_kv;
    l.n_pad = (d.n_ctx + zwg::kKvqPad - 1) / zwg::kKvqPad * zwg::kKvqPad;
    l.codes = up256(l.units * l.n_pad * d.d);
    l.scales = up256(l.units * (l.n_pad / d.block) * sizeof(float));
    l.rows = up256(l.units * d.block * d.d * sizeof(float));
    l.open = up256(l.units * 2 * sizeof(zwg::KvqOpen));
    l.total = 2 * (l.codes + l.scales + l.rows) + l.open;
    return l;
}

inline std::string check_kvq_range(const zwg_kvq_desc &d, uint64_t layer0, uint64_t n_layer, uint64_t seq0, uint64_t n_seq) {
    if (layer0 > d.n_layer || n_layer > d.n_layer - layer0) return "kvq layers out of range";
    if (seq0 > d.n_seq || n_seq > d.n_seq - seq0) return "kvq sequences out of range";
    return "";
}

struct KvqAppend {
    uint64_t layer, seq0, pos, n, rope_pos;
    bool batch; // one row per sequence, at pos_dev
    const int32_t *pos_dev, *rope_pos_dev;
    const float *k, *v, *q, *q_out;
    uint64_t n_head, q_stride;
};

inline std::string check_kvq_append(const zwg_kvq_desc &d, const zwg_rope_desc *rope, const KvqAppend &a) {
    if (a.layer >= d.n_layer) return "kvq layer out of range";
    if (a.n == 0) return "";
    if (!a.k || !a.v) return "null k or v rows";
    if (off(a.k, 15) || off(a.v, 15)) return "k and v rows must be 16-byte aligned";
    if (a.batch) {
        if (!a.pos_dev) return "null position array";
        if (off(a.pos_dev, 3) || off(a.rope_pos_dev, 3)) return "position arrays must be 4-byte aligned";
        if (a.seq0 > d.n_seq || a.n > d.n_seq - a.seq0) return "kvq sequences out of range";
    } else {
        if (a.seq0 >= d.n_seq) return "kvq sequence out of range";
        if (a.pos > d.n_ctx || a.n > d.n_ctx - a.pos) return "append past the end of the cache (pos + n > n_ctx)";
        if (rope && (a.rope_pos > rope->n_ctx || a.n > rope->n_ctx - a.rope_pos))
            return "rotary positions past the end of the rope (rope_pos + n > its n_ctx)";
        if (a.n > (1ull << 27)) return "at most 2^27 rows in one call"; // a launch has fewer than 2^32 threads
    }
    if (!a.q && !a.q_out) return "";
    if (!rope) return "q is rotated only when the cache has a rope";
    if (!a.q || !a.q_out) return "null q or q_out";
    if (off(a.q, 15) || off(a.q_out, 15)) return "q and q_out must be 16-byte aligned";
    if (a.n_head == 0 || a.n_head % d.n_head_kv) return "n_head must be a positive multiple of n_head_kv";
    if (a.n_head > 65535 - 2 * d.n_head_kv) return "n_head out of range";
    if (a.q_stride % 4) return "q_stride must be a multiple of 4 floats";
    if (a.q_stride < a.n_head * d.d || a.q_stride > kMaxStride) return "q_stride is smaller than n_head * d, or out of range";
    return "";
}

inline std::string check_kvq_rows(const zwg_kvq_desc &d, uint64_t layer0, uint64_t n_layer, uint64_t seq0, uint64_t n_seq,
                                  const int32_t *pos_dev, uint64_t pos0, uint64_t n, const float *k, const float *v) {
    const std::string msg = check_kvq_range(d, layer0, n_layer, seq0, n_seq);
    if (!msg.empty()) return msg;
    if (off(k, 15) || off(v, 15)) return "k_out and v_out must be 16-byte aligned";
    if (off(pos_dev, 3)) return "position arrays must be 4-byte aligned";
    if (n > (1ull << 27) || pos0 > 0x7fffffffull) return "positions out of range (at most 2^27 in one call)";
    if (n_layer * n_seq > 65535) return "n_layer * n_seq must be below 65536 in one call";
    return "";
}

// New tokens of a workgroup of an eviction: as many codes of d = 128 as two workgroups' LDS hold; a quarter of that many
// tokens at d = 64 and 32, where more workgroups gain (32 units of 1001 kept tokens: groups of 1024, 512, 256: 16.4, 16.0,
// 12.1 us; 56 units of 2048 at d = 128, groups of 512, 256: 25.8, 27.8 us).
constexpr uint64_t kvq_move_group(uint64_t d) { return d == 128 ? 512 : 256; }
// The workspace of an eviction: each unit's new positions of its tokens (rows of whole tiles), all kept tokens' old ones, a
// ticket and a flag to each group of its keys, the same of its values (lines of their own, for the tickets' sake), its tokens.
struct KvqCutPlan {
    uint64_t row, kept, flags, groups, bytes;
};
inline KvqCutPlan kvq_cut_plan(uint64_t units, const zwg_kvq_desc &d, const zwg_kvq_cut &c) {
    KvqCutPlan p{0, 0, 0, 1, 0};
    if (c.n_keep < c.n_kv) {
        p.row = (c.n_kv + 31) / 32 * 32;
        p.kept = (units * c.n_keep + 31) / 32 * 32;
        p.groups = (c.n_keep + kvq_move_group(d.d) - 1) / kvq_move_group(d.d);
        p.flags = (1 + p.groups + 31) / 32 * 32;
    }
    p.bytes = 4 * (units * p.row + p.kept + 2 * units * p.flags + units);
    return p;
}

inline std::string check_kvq_cut(const zwg_kvq_desc &d, uint64_t layer0, uint64_t n_layer, uint64_t seq0, uint64_t n_seq,
                                 const zwg_kvq_cut &c, const float *weights, const float *weights_out) {
    const std::string msg = check_kvq_range(d, layer0, n_layer, seq0, n_seq);
    if (!msg.empty()) return msg;
    if (c.n_kv > d.n_ctx) return "n_kv is more than the cache has (n_ctx)";
    if (c.n_keep == 0 || c.n_keep > (1ull << 24)) return "n_keep must be in 1 .. 2^24";
    if (c.n_first > c.n_keep || c.n_recent > c.n_keep - c.n_first) return "n_first + n_recent must be at most n_keep";
    if (n_layer == 0 || n_seq == 0) return "";
    if (!weights && c.n_kv) return "null weights";
    if (off(weights, 3) || off(weights_out, 3) || off(c.kept, 3) || off(c.n_kv_dev, 3) || off(c.n_kv_out, 3))
        return "weights, kept and counts must be 4-byte aligned";
    if (c.weights_stride < c.n_kv || c.weights_stride > kMaxStride) return "weights_stride is smaller than n_kv, or out of range";
    if (c.n_kv > (1ull << 24)) return "n_kv is above 2^24";
    // the kernels' grids: a launch has fewer than 2^32 threads
    const uint64_t units = n_layer * n_seq * d.n_head_kv;
    if (units > (1ull << 21) || 2 * units * kvq_cut_plan(units, d, c).groups > (1ull << 21))
        return "too many (layer, sequence, head) units of this many tokens in one call";
    return "";
}

// ---- attention over them

constexpr int kKvqWaves = 4; // waves of a workgroup, over the keys
constexpr int kKvqSplitTile = zwg::kKvqTile * kKvqWaves;
constexpr int kKvqPackedRows = 8;
// Which calls of more than 8 rows (queries x heads of a KV head) take the prompt kernel (128 rows to a workgroup that share
// operands in LDS) and not the one that splits the keys over a workgroup's waves (32 rows): those with rows for most of a
// workgroup and enough products to fill the card with such workgroups, fewer where the keys are many.  Measured, split keys
// against prompt, us a call, d = 128, two KV heads: 6144 rows x 8000 keys 186 : 123, 2400 x 4000 41.7 : 42.3, 1152 x 4000
// 29.7 : 32.8, 576 x 4000 21.3 : 30.3, 192 x 30,000 64.9 : 48.1, 144 x 30,000 54.9 : 48.2, 96 x 30,000 38.4 : 44.9.
inline bool kvq_prompt(uint64_t rows, uint64_t units, uint64_t n_kv) {
    const uint64_t pairs = rows * units * n_kv; // below 2^31 * 2^31
    return rows >= 112 && pairs >= (n_kv >= 16384 ? 1ull << 23 : 1ull << 24);
}
constexpr uint64_t kKvqMaxChunks = 4096;

inline std::string check_kvq_attn(const zwg_kvq_desc &d, uint64_t layer, uint64_t seq0, uint64_t n_seq, const float *q,
                                  const zwg_kvq_attn &s, const float *out, const float *weights) {
    if (layer >= d.n_layer) return "kvq layer out of range";
    if (seq0 > d.n_seq || n_seq > d.n_seq - seq0) return "kvq sequences out of range";
    if (s.n_head == 0 || s.n_head % d.n_head_kv) return "n_head must be a positive multiple of n_head_kv";
    if (s.n_head > 65535 || s.n_q > (1ull << 24)) return "n_head or n_q out of range";
    if (s.n_kv > d.n_ctx) return "n_kv is more than the cache has (n_ctx)";
    if (s.causal > 1) return "causal must be 0 or 1";
    if (n_seq == 0 || s.n_q == 0) return "";
    if (!q || !out) return "null q or out";
    if (off(q, 15) || off(out, 15)) return "q and out must be 16-byte aligned";
    if (off(s.n_kv_dev, 3)) return "n_kv_dev must be 4-byte aligned";
    if (s.q_stride % 4 || s.out_stride % 4 || s.q_bstride % 4 || s.out_bstride % 4)
        return "q and out strides must be multiples of 4 floats";
    if (s.q_stride > kMaxStride || s.out_stride > kMaxStride || s.q_bstride > kMaxStride || s.out_bstride > kMaxStride)
        return "strides out of range";
    if (s.n_q > 1 && (s.q_stride < s.n_head * d.d || s.out_stride < s.n_head * d.d))
        return "q_stride or out_stride is smaller than n_head * d";
    if (weights) {
        if (off(weights, 3)) return "weights must be 4-byte aligned";
        if (!(s.decay >= 0.f) || std::isinf(s.decay)) return "decay must be finite and >= 0";
        if (s.weights_stride > kMaxStride || s.weights_bstride > kMaxStride) return "strides out of range";
        if (d.n_head_kv > 1 && s.weights_stride < s.n_kv) return "weights_stride is smaller than n_kv";
        if (n_seq > 1 && s.weights_bstride < (d.n_head_kv - 1) * s.weights_stride + s.n_kv)
            return "weights_bstride is smaller than a sequence's weights";
        if (s.n_kv > 65535ull * 128) return "weights: n_kv must be below 65535 * 128";
    }
    if (s.n_q * s.n_head * n_seq > 0x7fffffffull) return "n_q * n_head * sequences must be below 2^31";
    return "";
}

// The workspace of an attention call, in floats, each part on a 256-byte boundary: the rows' final statistics (with
// weights), the chunks' statistics, the chunks' sums.
struct KvqWorkspace {
    uint64_t part_ml, part_o, total;
};
inline KvqWorkspace kvq_workspace(uint64_t rows, uint64_t chunks, uint64_t d, bool weights) {
    const auto up64 = [](uint64_t x) { return (x + 63) / 64 * 64; };
    KvqWorkspace w{};
    w.part_ml = weights ? up64(2 * rows) : 0;
    w.part_o = w.part_ml + (chunks > 1 ? up64(2 * rows * chunks) : 0);
    w.total = w.part_o + (chunks > 1 ? rows * chunks * d : 0);
    return w;
}

struct KvqSplit {
    int chunk_len, max_chunks;
};

// Keys of a chunk (unit_split's), so that units * chunks come to about two workgroups a CU, or to four where chunks stay
// at least kKvqLongChunk tiles long: each workgroup costs about 5 us before its first product and after its last, a tile
// 0.9 us.  Measured, kernel and merge: 64 sequences of 1 .. 4096 keys, d = 128, 17.4 + 4.0 us at two a CU and 14.4 + 4.0 at
// four (512 keys a chunk); one of 131,001 keys 13.3 + 5.5 at two (512 keys) and 15.2 + 7.6 at four (256 keys).
// Partials have to fit the workspace.
constexpr uint64_t kKvqLongChunk = 4;
constexpr uint64_t kKvqUnsplit = 6;

//
// Prompts (workgroups of 128 rows, two to a CU, a tile of 128 keys 5.8 us when both are there, about a tile more at a
// workgroup's ends): the chunk count of the least time over whole rounds of 512 workgroups and the merge, which reads
// the partials at 3.3 TB/s.  Measured, 1024 queries over 8000 keys (96 units): 10 chunks 126 + 20 us, 5 chunks 124 + 11.
inline KvqSplit kvq_split(uint64_t units, uint64_t n_kv, uint64_t rows, uint64_t d, bool weights, uint64_t ws_bytes, bool prompt) {
    const uint64_t w = std::max<uint64_t>(1, (n_kv + kKvqSplitTile - 1) / kKvqSplitTile);
    const auto tiles = [&](uint64_t blocks) {
        const uint64_t want = std::min<uint64_t>(w, std::max<uint64_t>(1, (blocks + units - 1) / units));
        return (w + want - 1) / want;
    };
    uint64_t tau = tiles(512);
    if (tau > kKvqLongChunk) tau = std::max(kKvqLongChunk, tiles(1024));
    if (prompt) {
        double best = 0;
        for (uint64_t c = 1; c <= std::min<uint64_t>(w, 32); ++c) {
            const double rounds = (double)((units * c + 511) / 512), merge = c > 1 ? (3.0 + (double)(rows * c * d) * 4 / 3.3e6) / 5.8 : 0.0;
            const double cost = rounds * (double)((w + c - 1) / c + 1) + merge;
            if (c == 1 || cost < best) {
                best = cost;
                tau = (w + c - 1) / c;
            }
        }
    } else if (w <= kKvqUnsplit) tau = w; // up to 6 steps a wave: less than a merge's launch
    const auto bound = [&](uint64_t t) { return std::max<uint64_t>(1, (w + t / 2) / t); };
    while (bound(tau) > 1 && (bound(tau) > kKvqMaxChunks || kvq_workspace(rows, bound(tau), d, weights).total * sizeof(float) > ws_bytes))
        ++tau;
    return {(int)(tau * kKvqSplitTile), (int)bound(tau)};
}

} // namespace zwg_planner
