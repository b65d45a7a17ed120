// Writing and reading the 8-bit key/value caches (include/zw_gpu.h, zwg_kvq_*): appends, reads as values, eviction.
//
// A block's scale is shared by all its tokens, so a token that outgrows it changes the codes of every token
// before it in the block.  The rows of the block being filled are therefore also held in f32: the codes are always
// those of the block's rows, never codes of codes.  An appended token whose block keeps its largest
// magnitude (most do: token r of a block brings a new largest one time in r + 1) writes its own codes alone.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "kv_quant.hpp"
#include "zw_ctx.hpp"

using namespace zwg_host;
using namespace zwg_planner;
using zwg::KvqOpen;
using zwg::KvqView;

namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kAppendThreads = 256;
constexpr int kPad = 4; // floats between the staged rows' ends and the next row: 16-byte rows on other banks

__device__ __forceinline__ uint32_t abs_bits(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7fffffffu; }

struct AppendArgs {
    KvqView view;
    zwg::RopeView rope;
    int64_t unit0; // unit of (layer, seq0, head 0)
    const float *src[2]; // [n][n_head_kv * d]
    const float *q;
    float *q_out;
    int64_t q_stride;
    const int32_t *pos_dev, *rope_pos_dev; // one token per sequence; nullptr: n tokens of one, at pos0 and rope_pos0
    int64_t pos0, rope_pos0;
    int32_t n, n_head;
};

// Codes of rows [r0, r1) of the staged block in `rows`, written to the unit's codes.  16 rows of a value
// tile's dim are four runs of four bytes, so both tensors are written in words of four codes; the rows of a
// word outside [r0, r1) are written only where the whole block is (r0 = 0, r1 = block).
template <int D, int FMT, int IS_V>
__device__ __forceinline__ void write_codes(uint8_t *codes, const float (*rows)[D + kPad], int block_size, int64_t first,
                                            int r0, int r1, float mul) {
    if (!IS_V) {
        for (int i = threadIdx.x; i < (r1 - r0) * (D / 4); i += kAppendThreads) {
            const int r = r0 + i / (D / 4), c = 4 * (i % (D / 4));
            const float4 x = *reinterpret_cast<const float4 *>(&rows[r][c]);
            *reinterpret_cast<uint32_t *>(codes + zwg::kvq_at(0, first + r, c, D)) = zwg::kvq_encode4<FMT>(x.x, x.y, x.z, x.w, mul);
        }
    } else if (r0 == 0 && r1 == block_size) {
        for (int i = threadIdx.x; i < block_size / 4 * D; i += kAppendThreads) {
            const int c = i % D, r = 4 * (i / D);
            *reinterpret_cast<uint32_t *>(codes + zwg::kvq_at(1, first + r, c, D)) =
                zwg::kvq_encode4<FMT>(rows[r][c], rows[r + 1][c], rows[r + 2][c], rows[r + 3][c], mul);
        }
    } else {
        for (int i = threadIdx.x; i < (r1 - r0) * D; i += kAppendThreads) {
            const int r = r0 + i / D, c = i % D;
            codes[zwg::kvq_at(1, first + r, c, D)] = (uint8_t)zwg::kvq_encode4<FMT>(rows[r][c], 0.f, 0.f, 0.f, mul);
        }
    }
}

// Rows [r0, r1) of a block, token `tok` on, into LDS, keys rotated, and their largest magnitudes.  Begins and ends without a
// barrier; what was written to `top` before is there after it for all.
template <int D, int IS_V>
__device__ __forceinline__ void new_rows(const AppendArgs &a, int head, int r0, int r1, int64_t tok, int64_t rope_pos,
                                         float (*rows)[D + kPad], uint32_t *top) {
    const int tid = threadIdx.x, kvw = a.view.n_head_kv * D;
    for (int i = tid; i < (r1 - r0) * (D / 4); i += kAppendThreads) {
        const int r = i / (D / 4), c = 4 * (i % (D / 4));
        *reinterpret_cast<float4 *>(&rows[r0 + r][c]) =
            *reinterpret_cast<const float4 *>(a.src[IS_V] + (tok + r) * kvw + head * D + c);
    }
    __syncthreads();
    if (!IS_V && a.rope.cos) {
        const int turned = zwg::rope_turned(a.rope);
        for (int i = tid; i < (r1 - r0) * turned; i += kAppendThreads) {
            const int r = i / turned;
            zwg::rope_piece(a.rope, rope_pos + r, i - r * turned, rows[r0 + r], rows[r0 + r]);
        }
        __syncthreads();
    }
    // each row's largest magnitude: D / 4 lanes a row (8, 16 or 32, in one wave)
    for (int i = tid; i < (r1 - r0) * (D / 4); i += kAppendThreads) {
        const int r = r0 + i / (D / 4), c = 4 * (i % (D / 4));
        const float4 x = *reinterpret_cast<const float4 *>(&rows[r][c]);
        uint32_t m = max(max(abs_bits(x.x), abs_bits(x.y)), max(abs_bits(x.z), abs_bits(x.w)));
#pragma unroll
        for (int off = D / 8; off >= 1; off >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, off));
        if (i % (D / 4) == 0) top[r] = m;
    }
}

// Rows [from, r1) of block b, and the magnitudes of all before r1, become the unit's open block.
template <int D, int IS_V>
__device__ __forceinline__ void hold_rows(const AppendArgs &a, int64_t u, int b, int from, int r1, const float (*rows)[D + kPad],
                                          const uint32_t *top) {
    const int tid = threadIdx.x;
    float *held = a.view.rows[IS_V] + u * a.view.block * D;
    KvqOpen *open = a.view.open + 2 * u + IS_V;
    for (int i = tid; i < (r1 - from) * (D / 4); i += kAppendThreads) {
        const int r = from + i / (D / 4), c = 4 * (i % (D / 4));
        *reinterpret_cast<float4 *>(held + r * D + c) = *reinterpret_cast<const float4 *>(&rows[r][c]);
    }
    if (tid < r1) open->top[tid] = __builtin_bit_cast(float, top[tid]);
    if (tid == 0) {
        open->block = b;
        open->filled = r1;
    }
}

// One block of a unit: rows [r0, r1) are new (token `tok` on), those before r0 are held in the open block or
// count as the values of their codes, those from r1 on become zeros.  keep: the block stays open (it is the last
// that the call touches, and no other workgroup holds its rows for it).
template <int D, int FMT, int IS_V>
__device__ void append_block(const AppendArgs &a, int64_t u, int head, int b, int r0, int r1, int64_t tok,
                             int64_t rope_pos, bool keep, float (*rows)[D + kPad], uint32_t *top, uint32_t *shared_top) {
    const KvqView &v = a.view;
    const int B = v.block, tid = threadIdx.x;
    uint8_t *codes = v.codes[IS_V] + u * v.unit_bytes;
    float *scale_at = v.scales[IS_V] + u * v.n_blocks + b;
    const float *held = v.rows[IS_V] + u * B * D;
    const KvqOpen *open = v.open + 2 * u + IS_V;
    const int64_t first = (int64_t)b * B;

    // a block with no rows before the new ones has no use for what is held (which another workgroup may be replacing)
    const bool is_open = r0 > 0 && open->block == b;
    const int filled = is_open ? open->filled : 0;
    const float old_scale = *scale_at;
    if (tid < B) top[tid] = tid < r0 && tid < filled ? abs_bits(open->top[tid]) : 0u;
    new_rows<D, IS_V>(a, head, r0, r1, tok, rope_pos, rows, top);
    __syncthreads();
    if (tid < 64) {
        uint32_t m = tid < r1 ? top[tid] : 0u, was = tid < filled ? abs_bits(open->top[tid]) : 0u;
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) {
            m = max(m, (uint32_t)__shfl_xor((int)m, off));
            was = max(was, (uint32_t)__shfl_xor((int)was, off));
        }
        if (tid == 0) {
            shared_top[0] = m;
            shared_top[1] = was;
        }
    }
    __syncthreads();
    float scale, mul;
    zwg::kvq_scale<FMT>(shared_top[0], &scale, &mul);
    // an open block whose largest magnitude stays, with no row behind r1 to clear, needs the new rows' codes
    // alone (rows between the filled ones and r0 are zeros already)
    const bool same = is_open && filled <= r1 && shared_top[0] == shared_top[1];
    if (same) {
        write_codes<D, FMT, IS_V>(codes, rows, B, first, r0, r1, mul);
    } else {
        // the whole block: the rows before r0, then zeros behind r1
        for (int i = tid; i < r0 * (D / 4); i += kAppendThreads) {
            const int r = i / (D / 4), c = 4 * (i % (D / 4));
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            if (is_open) {
                if (r < filled) x = *reinterpret_cast<const float4 *>(held + r * D + c);
            } else {
                x.x = zwg::kvq_decode_byte<FMT>(codes[zwg::kvq_at(IS_V, first + r, c, D)]) * old_scale;
                x.y = zwg::kvq_decode_byte<FMT>(codes[zwg::kvq_at(IS_V, first + r, c + 1, D)]) * old_scale;
                x.z = zwg::kvq_decode_byte<FMT>(codes[zwg::kvq_at(IS_V, first + r, c + 2, D)]) * old_scale;
                x.w = zwg::kvq_decode_byte<FMT>(codes[zwg::kvq_at(IS_V, first + r, c + 3, D)]) * old_scale;
            }
            *reinterpret_cast<float4 *>(&rows[r][c]) = x;
        }
        for (int i = tid; i < (B - r1) * (D / 4); i += kAppendThreads) {
            const int r = r1 + i / (D / 4), c = 4 * (i % (D / 4));
            *reinterpret_cast<float4 *>(&rows[r][c]) = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        __syncthreads(); // also: every old code is read before any is written
        if (!is_open && r0 > 0) {
            // the reopened rows take part in the block's largest magnitude
            for (int i = tid; i < r0 * (D / 4); i += kAppendThreads) {
                const int r = i / (D / 4), c = 4 * (i % (D / 4));
                const float4 x = *reinterpret_cast<const float4 *>(&rows[r][c]);
                uint32_t m = max(max(abs_bits(x.x), abs_bits(x.y)), max(abs_bits(x.z), abs_bits(x.w)));
#pragma unroll
                for (int off = D / 8; off >= 1; off >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, off));
                if (i % (D / 4) == 0) top[r] = m;
            }
            __syncthreads();
            if (tid < 64) {
                uint32_t m = tid < r1 ? top[tid] : 0u;
#pragma unroll
                for (int off = 32; off >= 1; off >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, off));
                if (tid == 0) shared_top[0] = m;
            }
            __syncthreads();
            zwg::kvq_scale<FMT>(shared_top[0], &scale, &mul);
        }
        write_codes<D, FMT, IS_V>(codes, rows, B, first, 0, B, mul);
        if (tid == 0) *scale_at = scale;
    }
    if (keep) {
        // rows of an open block that was held already stay where they are; gap rows (filled .. r0) are zeros
        const int from = is_open ? min(filled, r0) : 0;
        if (same && from < r0) {
            for (int i = tid; i < (r0 - from) * (D / 4); i += kAppendThreads)
                *reinterpret_cast<float4 *>(&rows[from + i / (D / 4)][4 * (i % (D / 4))]) = make_float4(0.f, 0.f, 0.f, 0.f);
            __syncthreads();
        }
        hold_rows<D, IS_V>(a, u, b, from, r1, rows, top);
    }
}

// Workgroups (x, y): y < 2 n_head_kv: head y / 2's keys (y even) or values of the x-th touched block (tokens of one
// sequence) or of sequence x (one token each); from there on query head y - 2 n_head_kv of the same tokens.
// A call's first block b0 may need the unit's open block, which its last one, b1, replaces: where b0 has rows before the new
// ones, its workgroup also puts b1's rows in their place, after its own use of it, and b1's writes codes alone.
//
// Bound by the chain of a block (rows, rotation, largest, codes), not by bytes: 64 sequences' tokens at d = 128 take 5.6 us,
// 2048 that begin and end inside blocks 10.1, and 11.5 with all of b1 behind b0, where the bytes take 4.
template <int D, int FMT> __global__ __launch_bounds__(kAppendThreads) void kvq_append_kernel(AppendArgs a) {
    __shared__ __align__(16) float rows[zwg::kKvqMaxBlock][D + kPad];
    __shared__ uint32_t top[zwg::kKvqMaxBlock];
    __shared__ uint32_t shared_top[2];
    const KvqView &v = a.view;
    const int B = v.block, x = blockIdx.x, y = blockIdx.y;

    int64_t pos = a.pos0, rp = a.rope_pos0, n = a.n, tok = 0, u = a.unit0;
    if (a.pos_dev) {
        pos = a.pos_dev[x];
        rp = a.rope_pos_dev ? a.rope_pos_dev[x] : pos;
        if (pos < 0 || pos >= v.n_ctx || (a.rope.cos && (rp < 0 || rp >= a.rope.n_ctx))) return;
        n = 1;
        tok = x;
        u += (int64_t)x * v.n_head_kv;
    }
    const int64_t b0 = pos / B, b1 = (pos + n - 1) / B;

    const int64_t b = b0 + (a.pos_dev ? 0 : x);
    const int64_t t0 = max(pos, b * B) - pos, t1 = min(pos + n, (b + 1) * B) - pos;
    if (y >= 2 * v.n_head_kv) {
        // query rows: those of the block's tokens
        const int h = y - 2 * v.n_head_kv;
        const int pieces = a.q == a.q_out ? zwg::rope_turned(a.rope) : zwg::rope_pieces(a.rope);
        for (int i = threadIdx.x; i < (int)(t1 - t0) * pieces; i += kAppendThreads) {
            const int t = i / pieces, c = i - t * pieces;
            const int64_t row = (tok + t0 + t) * a.q_stride + (int64_t)h * D;
            zwg::rope_piece(a.rope, rp + t0 + t, c, a.q + row, a.q_out + row);
        }
        return;
    }
    const int head = y >> 1;
    u += head;
    const int r0 = (int)(pos + t0 - b * B), r1 = (int)(pos + t1 - b * B);
    const bool first_holds = b0 < b1 && pos > b0 * B, keep = b == b1 && !first_holds;
    const int64_t tl = b1 * B - pos; // b1's first token
    const auto block = [&](auto is_v) {
        append_block<D, FMT, is_v.value>(a, u, head, (int)b, r0, r1, tok + t0, rp + t0, keep, rows, top, shared_top);
        if (first_holds && b == b0) {
            __syncthreads();
            new_rows<D, is_v.value>(a, head, 0, (int)(n - tl), tok + tl, rp + tl, rows, top);
            __syncthreads();
            hold_rows<D, is_v.value>(a, u, (int)b1, 0, (int)(n - tl), rows, top);
        }
    };
    if (y & 1)
        block(std::integral_constant<int, 1>{});
    else
        block(std::integral_constant<int, 0>{});
}

// ---------------------------------------------------------------------------------------------- reads

struct RowsArgs {
    KvqView view;
    int64_t layer0, seq0;
    const int32_t *pos_dev;
    int64_t pos0;
    int64_t n; // positions of a sequence
    int32_t n_seq;
    float *out[2]; // [n_layer][n_seq][n][n_head_kv * d]
};

// The i-th code of a lane's 16 bytes.
template <int FMT> __device__ __forceinline__ float code_of(const u32x4 &w, int i) {
    return zwg::kvq_decode_byte<FMT>((uint8_t)(w[i >> 2] >> (8 * (i & 3))));
}

// A wave per KB of codes of one unit's keys or values (32 positions have d / 32), read as the attention reads them: 16 bytes
// a lane.  Workgroups (x, y, z): four such from 4 x on of (layer, sequence) y; z: KV head and keys or values.  Bound by its
// stores, four times the bytes it reads: 56 units of 2048 positions, d = 128, 147 MB in 32 us, 4.5 TB/s.
template <int D, int FMT> __global__ __launch_bounds__(256) void kvq_rows_kernel(RowsArgs a) {
    const KvqView &v = a.view;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, col = lane & 15;
    const int is_v = blockIdx.z & 1, head = blockIdx.z >> 1;
    float *out = a.out[is_v];
    if (!out) return;
    const int64_t layer = a.layer0 + blockIdx.y / a.n_seq, i = blockIdx.y % a.n_seq;
    const int64_t u = (layer * v.n_seq + a.seq0 + i) * v.n_head_kv + head;
    const int64_t start = a.pos_dev ? (int64_t)a.pos_dev[i] : a.pos0;
    // the positions start .. start + n - 1 that the cache has, and this wave's tile of them
    const int64_t lo = max(start, (int64_t)0), hi = min(start + a.n, (int64_t)v.n_ctx);
    const int64_t kb = (int64_t)blockIdx.x * 4 + wave;
    const int64_t p0 = (lo / 32 + kb / (D / 32)) * 32;
    const int n = (int)(kb % (D / 32));
    if (p0 >= hi) return;
    const uint8_t *codes = v.codes[is_v] + u * v.unit_bytes + p0 * D + 64 * col + 16 * g;
    const float *scales = v.scales[is_v] + u * v.n_blocks;
    const float s[2] = {scales[p0 / v.block], scales[(p0 + 16) / v.block]};
    const int64_t kvw = (int64_t)v.n_head_kv * D;
    out += ((int64_t)blockIdx.y * a.n - start) * kvw + head * D;
    const u32x4 w = *reinterpret_cast<const u32x4 *>(codes + 1024 * n);
    if (is_v) {
        // dims 32 n + col and 16 on, of tokens 16 q + 4 g + e
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const int h = k >> 3, q = (k >> 2) & 1, e = k & 3;
            const int64_t p = p0 + 16 * q + 4 * g + e;
            if (p >= lo && p < hi) out[p * kvw + 32 * n + 16 * h + col] = code_of<FMT>(w, k) * s[q];
        }
    } else {
        // dims 64 (n % (d / 64)) + 16 g .. of token 16 (n / (d / 64)) + col; at d = 32 dims 8 g .. of col and 16 + col
        constexpr int kHalves = D == 128 ? 2 : 1;
#pragma unroll
        for (int k = 0; k < 16; k += 4) {
            const int q = D == 32 ? k >> 3 : n / kHalves;
            const int c = D == 32 ? 8 * g + (k & 7) : 64 * (n % kHalves) + 16 * g + k;
            const int64_t p = p0 + 16 * q + col;
            const float f = q ? s[1] : s[0];
            if (p >= lo && p < hi)
                *reinterpret_cast<float4 *>(out + p * kvw + c) = make_float4(code_of<FMT>(w, k) * f, code_of<FMT>(w, k + 1) * f,
                                                                            code_of<FMT>(w, k + 2) * f, code_of<FMT>(w, k + 3) * f);
        }
    }
}

// ---------------------------------------------------------------------------------------------- eviction

constexpr int kSelectThreads = 1024;
constexpr int kSelectWaves = kSelectThreads / 64;

struct CutArgs {
    KvqView view;
    int64_t layer0, seq0;
    int32_t n_seq;
    int32_t n_kv, n_keep, n_first, n_recent;
    int64_t w_stride;
    const int32_t *n_kv_dev;
    int32_t *n_kv_out, *kept;
    const float *w;
    float *w_out;
    int32_t *src;   // [unit of the call][n_keep]: the kept tokens' old positions
    int32_t *dst;   // [unit of the call][n_kv rounded up to 32]: each token's new position, or -1
    int64_t dst_stride;
    int32_t *count; // [unit of the call]: the tokens before the cut (the counts may be overwritten after it)
    int32_t *flags; // [unit of the call][keys, values][flag_stride]: a ticket, then for each group: its codes are out of the cache
    int32_t n_groups, flag_stride;
};

// A weight as an unsigned number in the order of the selection: negative below positive, the zeros equal, a NaN
// above everything.
__device__ __forceinline__ uint32_t rank_bits(float w) {
    if (w != w) return 0xffffffffu;
    const uint32_t b = __builtin_bit_cast(uint32_t, w + 0.0f); // -0 + 0 = 0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// One workgroup per (layer, sequence, head): the threshold weight by up to four passes over 8 bits each (counts in LDS,
// whole numbers, so their order does not matter), as many as decide, then an ordered pass that writes the kept positions and
// weights.  Equal weights
// at the threshold go to the lowest positions.  Of 8192 weights each thread holds 8 in registers over all passes; what is
// left is launch, loads and barriers (measured: 56 units of 2304 weights 10.6 us, 32 of 4096 10.9; with two barriers to each
// 1024 weights 10.9 and 13.3, with 512 threads and 16 weights each 13.4 and 13.7).
constexpr int kHeld = 8;
__global__ __launch_bounds__(kSelectThreads) void kvq_select_kernel(CutArgs a) {
    __shared__ uint32_t hist[2][256];
    __shared__ uint32_t found_prefix, found_left, found_all;
    __shared__ uint2 counts[kHeld][kSelectWaves]; // weights above the threshold, and at it: first a wave's, then those before it
    __shared__ uint2 all;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t cu = blockIdx.x; // unit of the call
    const uint32_t seq = blockIdx.x / (uint32_t)a.view.n_head_kv % (uint32_t)a.n_seq;
    const int n = a.n_kv_dev ? min(max(a.n_kv_dev[seq], 0), a.n_kv) : a.n_kv;
    const float *w = a.w + cu * a.w_stride;
    float *w_out = a.w_out ? a.w_out + cu * a.w_stride : nullptr;
    int32_t *src = a.src + cu * a.n_keep, *dst = a.dst + cu * a.dst_stride;
    int32_t *kept = a.kept ? a.kept + cu * a.n_keep : nullptr;
    if (tid == 0) a.count[cu] = n;
    for (int i = tid; i < 2 * a.flag_stride; i += kSelectThreads) a.flags[2 * cu * a.flag_stride + i] = 0;
    if (n <= a.n_keep) {
        for (int i = tid; i < a.n_keep; i += kSelectThreads)
            if (kept) kept[i] = i < n ? i : -1;
        if (w_out)
            for (int i = tid; i < a.n_kv; i += kSelectThreads) w_out[i] = i < n ? w[i] : 0.0f;
        return;
    }
    const int lo = a.n_first, hi = n - a.n_recent; // the contested positions
    constexpr int kSpan = kHeld * kSelectThreads;
    float held[kHeld]; // of positions base + tid + kSelectThreads k
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
        const int i = tid + k * kSelectThreads;
        held[k] = i < n ? w[i] : 0.0f;
    }
    if (tid < 256) hist[0][tid] = 0;
    __syncthreads();
    int low = 0; // bits below the threshold's
    uint32_t prefix = 0, left = (uint32_t)(a.n_keep - a.n_first - a.n_recent); // < hi - lo
#pragma unroll 1
    for (int shift = 24; shift >= 0 && left > 0; shift -= 8) {
        uint32_t *h = hist[(shift >> 3) & 1 ? 0 : 1];
        const auto count = [&](int i, float x) {
            const uint32_t r = rank_bits(x);
            if (i >= lo && i < hi && (shift == 24 || (r >> (shift + 8)) == prefix)) atomicAdd(&h[(r >> shift) & 255u], 1u);
        };
#pragma unroll
        for (int k = 0; k < kHeld; ++k)
            if (k * kSelectThreads < n) count(tid + k * kSelectThreads, held[k]);
        for (int i = kSpan + tid; i < hi; i += kSelectThreads) count(i, w[i]);
        __syncthreads();
        if (wave == 0) {
            // the digit at which the counts from the top reach `left`: four digits a lane, lane 0 the highest
            uint32_t c[4], s = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                c[k] = h[255 - 4 * lane - k];
                s += c[k];
            }
            uint32_t incl = s;
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const uint32_t o = (uint32_t)__shfl_up((int)incl, off);
                if (lane >= off) incl += o;
            }
            uint32_t before = incl - s;
            if (before < left && incl >= left) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if (before < left && before + c[k] >= left) {
                        found_prefix = (prefix << 8) | (uint32_t)(255 - 4 * lane - k);
                        found_left = left - before;
                        found_all = c[k];
                    }
                    before += c[k];
                }
            }
        } else if (tid >= 256 && tid < 512) {
            hist[(shift >> 3) & 1][tid - 256] = 0; // the next pass's
        }
        __syncthreads();
        prefix = found_prefix;
        left = found_left;
        if (left == found_all) { // all weights of these digits stay: the lower ones decide nothing
            low = shift;
            break;
        }
    }
    // now `prefix` is the threshold and `left` of its equals stay (none contested: nothing stays between)
    const bool any = a.n_keep > a.n_first + a.n_recent;
    uint32_t more_before = 0, ties_before = 0; // in the spans so far
    for (int base = 0; base < n; base += kSpan) {
        if (base > 0) {
            __syncthreads(); // the counts are free
#pragma unroll
            for (int k = 0; k < kHeld; ++k) {
                const int i = base + tid + k * kSelectThreads;
                held[k] = i < n ? w[i] : 0.0f;
            }
        }
        const auto is_more = [&](int i, uint32_t r) { return i < n && (i < lo || i >= hi || (any && (r >> low) > prefix)); };
        const auto is_tie = [&](int i, uint32_t r) { return i >= lo && i < hi && any && (r >> low) == prefix; };
#pragma unroll
        for (int k = 0; k < kHeld; ++k) {
            const int i = base + tid + k * kSelectThreads;
            const uint32_t r = rank_bits(held[k]);
            const uint2 c = make_uint2((uint32_t)__popcll(__ballot(is_more(i, r))), (uint32_t)__popcll(__ballot(is_tie(i, r))));
            if (lane == 0) counts[k][wave] = c;
        }
        __syncthreads();
        if (wave == 0) {
            // 128 counts in order, two to a lane
            uint2 *at = &counts[0][0] + 2 * lane;
            static_assert(kHeld * kSelectWaves == 128);
            const uint2 c0 = at[0], c1 = at[1];
            uint32_t x = c0.x + c1.x, y = c0.y + c1.y;
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const uint32_t ox = (uint32_t)__shfl_up((int)x, off), oy = (uint32_t)__shfl_up((int)y, off);
                if (lane >= off) {
                    x += ox;
                    y += oy;
                }
            }
            at[0] = make_uint2(x - c0.x - c1.x, y - c0.y - c1.y);
            at[1] = make_uint2(x - c1.x, y - c1.y);
            if (lane == 63) all = make_uint2(x, y);
        }
        __syncthreads();
        // every weight of the span is in registers, and new positions never lie above old ones: the weights may be compacted in place
#pragma unroll
        for (int k = 0; k < kHeld; ++k) {
            const int i = base + tid + k * kSelectThreads;
            const uint32_t r = rank_bits(held[k]);
            const bool more = is_more(i, r), tie = is_tie(i, r);
            const unsigned long long below = (1ull << lane) - 1;
            const uint2 c = counts[k][wave];
            const uint32_t ties = ties_before + c.y + __popcll(__ballot(tie) & below);
            const bool stays = more || (tie && ties < left);
            const int at = (int)(more_before + c.x + __popcll(__ballot(more) & below) + min(ties, left));
            if (i < (int)a.dst_stride) dst[i] = stays ? at : -1;
            if (stays) {
                src[at] = i;
                if (kept) kept[at] = i;
                if (w_out) w_out[at] = held[k];
            }
        }
        more_before += all.x;
        ties_before += all.y;
    }
    if (w_out)
        for (int i = a.n_keep + tid; i < a.n_kv; i += kSelectThreads) w_out[i] = 0.0f;
}

template <int D> constexpr int kMoveGroup = (int)kvq_move_group(D); // new tokens of a workgroup
template <int D> constexpr int kMoveThreads = 2 * kMoveGroup<D>;

// Groups of a unit in parallel, in place.  A kept token never moves up, so the old codes under a group's new positions are
// read by that group and lower ones only: a group takes its own codes out of the cache (into registers, or LDS), says so,
// and waits for all lower groups of its keys or values to have said so before it writes.  The unit's workgroups take their
// groups by tickets, in ascending order: what one waits for has a lower ticket and runs already, and the lowest waits for
// nothing, so every wait ends; the bound on it (seconds) is for a workspace that something else overwrites.  Nothing is
// passed through the cache from group to group, only the loads' completion, so the flags need no release of the caches.
//
// Measured, 56 units of four groups, d = 128: 26 us for 33 MB read and 29 MB written, 2.4 TB/s; with one workgroup taking
// a unit's groups in turn 34, with the groups gathered into a staging buffer and copied back 32, with one ticket counter for
// all units 30.6 (its atomics queue up).  What is left is the chain of a group: positions, gather, largest, wait, store.
constexpr int kMaxPolls = 1 << 22;
// Behind a barrier: every load of the workgroup from the cache has returned (its value was used before the barrier).
__device__ __forceinline__ void group_read(const CutArgs &a, int64_t unit2, int group) {
    if (a.n_groups > 1 && threadIdx.x == 0)
        __hip_atomic_store(a.flags + unit2 * a.flag_stride + 1 + group, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <int D> __device__ __forceinline__ void await_lower_groups(const CutArgs &a, int64_t unit2, int group) {
    if (group == 0) return;
    const int32_t *flags = a.flags + unit2 * a.flag_stride + 1;
    for (int g = threadIdx.x; g < group; g += kMoveThreads<D>)
        for (int i = 0; i < kMaxPolls && !__hip_atomic_load(flags + g, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); ++i)
            __builtin_amdgcn_s_sleep(1);
    __syncthreads();
}

// New tokens [t0, t0 + kMoveGroup) of a (layer, sequence, head)'s keys or values.
//
// Keys: a token's codes are runs of 16 bytes (8 at d = 32), gathered run by run.  Values: a token's codes lie one or two to a
// 64-byte line, so the old tiles are read whole and in order, each wave one at a time, and their kept tokens' bytes are put into
// LDS by new position, [d][group].  Both are taken twice: for the new blocks' largest magnitudes, and for the new codes.
template <int D, int FMT, int IS_V> __device__ __forceinline__ void move_group(const CutArgs &a, int64_t cu, int group) {
    constexpr int kGroup = kMoveGroup<D>, kMoveWaves = kMoveThreads<D> / 64;
    constexpr int kRow = kGroup + 16;                 // bytes of a dim's row in LDS: 4 words beyond a multiple of the banks
    constexpr int kRun = D == 32 ? 8 : 16;            // bytes of a key run
    constexpr int kRuns = kGroup * D / kRun / kMoveThreads<D>; // runs of a thread: 4, at d = 64 and 32 2
    __shared__ uint32_t tops[kGroup / 16];
    __shared__ float scale_s[kGroup];
    __shared__ __align__(16) uint8_t vals[IS_V ? D * kRow : 16];
    const KvqView &v = a.view;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int shift = v.block == 16 ? 4 : v.block == 32 ? 5 : 6;
    const uint32_t H = v.n_head_kv, ls = (uint32_t)cu / H, layer = ls / (uint32_t)a.n_seq; // 32 bits: short divisions
    const uint32_t seq = ls - layer * a.n_seq, head = (uint32_t)cu - ls * H;
    const int n = a.count[cu];
    // the counts may be overwritten now: the kernel before this one read them
    if (IS_V && group == 0 && layer == 0 && head == 0 && a.n_kv_out && tid == 0) a.n_kv_out[seq] = min(n, a.n_keep);
    if (n <= a.n_keep) return;
    const int64_t u = ((a.layer0 + layer) * v.n_seq + a.seq0 + seq) * H + head;
    if (group == 0 && tid == 0) v.open[2 * u + IS_V].block = -1; // the open block's rows are others now
    const int t0 = group * kGroup;
    uint8_t *codes = v.codes[IS_V] + u * v.unit_bytes;
    float *scales = v.scales[IS_V] + u * v.n_blocks;
    const int32_t *src = a.src + cu * a.n_keep;
    const int32_t *dst = a.dst + cu * a.dst_stride;
    const int end = ((a.n_keep + v.block - 1) >> shift) << shift;
    const int live = min(a.n_keep - t0, kGroup); // tokens of the group; the rest up to `end` becomes zeros
    if (tid < kGroup / 16) tops[tid] = 0; // fewer than threads
    for (int t = tid; t < kGroup; t += kMoveThreads<D>) {
        const int p = t < live ? src[t0 + t] : 0;
        scale_s[t] = t < live ? scales[p >> shift] : 0.f;
    }
    u32x4 run[IS_V ? 1 : kRuns];
    if (!IS_V) {
#pragma unroll
        for (int k = 0; k < kRuns; ++k) {
            const int w = k * kMoveThreads<D> + tid, t = w / (D / kRun), c = kRun * (w % (D / kRun));
            run[k] = (u32x4){0u, 0u, 0u, 0u};
            if (t < live) {
                const uint8_t *at = codes + zwg::kvq_at(0, src[t0 + t], c, D);
                if (kRun == 16) {
                    run[k] = *reinterpret_cast<const u32x4 *>(at);
                } else {
                    const u32x2 x = *reinterpret_cast<const u32x2 *>(at);
                    run[k] = (u32x4){x[0], x[1], 0u, 0u};
                }
            }
        }
        __syncthreads();
        // a wave's 64 runs are of at most 16 aligned tokens: of one block
#pragma unroll
        for (int k = 0; k < kRuns; ++k) {
            const int t = (k * kMoveThreads<D> + tid) / (D / kRun);
            // the largest code's value is the largest (one factor for all, and rounding keeps the order)
            float m = 0.f;
#pragma unroll
            for (int i = 0; i < kRun; ++i) m = fmaxf(m, fabsf(code_of<FMT>(run[k], i)));
            uint32_t top = t < live ? abs_bits(m * scale_s[t]) : 0u;
#pragma unroll
            for (int off = 32; off >= 1; off >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, off));
            if (lane == 0) atomicMax(&tops[t >> shift], top);
        }
        __syncthreads();
        group_read(a, 2 * cu + IS_V, group);
        float scale[kRuns];
#pragma unroll
        for (int k = 0; k < kRuns; ++k) {
            const int t = (k * kMoveThreads<D> + tid) / (D / kRun);
            float mul;
            zwg::kvq_scale<FMT>(tops[t >> shift], &scale[k], &mul);
            const float s = scale_s[t];
#pragma unroll
            for (int i = 0; i < kRun / 4; ++i) {
                const bool on = t < live;
                run[k][i] = zwg::kvq_encode4<FMT>(on ? code_of<FMT>(run[k], 4 * i) * s : 0.f, on ? code_of<FMT>(run[k], 4 * i + 1) * s : 0.f,
                                                  on ? code_of<FMT>(run[k], 4 * i + 2) * s : 0.f,
                                                  on ? code_of<FMT>(run[k], 4 * i + 3) * s : 0.f, mul);
            }
        }
        await_lower_groups<D>(a, 2 * cu + IS_V, group);
#pragma unroll
        for (int k = 0; k < kRuns; ++k) {
            const int w = k * kMoveThreads<D> + tid, t = w / (D / kRun), c = kRun * (w % (D / kRun));
            if (t0 + t >= end) continue;
            uint8_t *at = codes + zwg::kvq_at(0, t0 + t, c, D);
            if (kRun == 16)
                *reinterpret_cast<u32x4 *>(at) = run[k];
            else
                *reinterpret_cast<u32x2 *>(at) = (u32x2){run[k][0], run[k][1]};
            if (c == 0 && ((t0 + t) & (v.block - 1)) == 0) scales[(t0 + t) >> shift] = scale[k];
        }
    } else {
        // the old tiles that hold the group's tokens
        const int first = src[t0] >> 5, last = src[t0 + live - 1] >> 5;
        const int g = lane >> 4, col = lane & 15;
        for (int tile = first + wave; tile <= last; tile += kMoveWaves) {
            int32_t to[8];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int4 x = *reinterpret_cast<const int4 *>(dst + 32 * tile + 16 * q + 4 * g);
                to[4 * q] = x.x - t0;
                to[4 * q + 1] = x.y - t0;
                to[4 * q + 2] = x.z - t0;
                to[4 * q + 3] = x.w - t0;
            }
            u32x4 w[D / 32];
#pragma unroll
            for (int k = 0; k < D / 32; ++k)
                w[k] = *reinterpret_cast<const u32x4 *>(codes + (int64_t)tile * 32 * D + 1024 * k + 64 * col + 16 * g);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (to[e] >= 0 && to[e] < live) // -1, a token of another group: not here
#pragma unroll
                    for (int k = 0; k < D / 32; ++k)
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            vals[(32 * k + 16 * h + col) * kRow + to[e]] = (uint8_t)(w[k][2 * h + (e >> 2)] >> (8 * (e & 3)));
        }
        __syncthreads();
        group_read(a, 2 * cu + IS_V, group);
        // new tiles, a wave to 32 tokens: lane (g, col) takes the 16 bytes of each KB that it would read there, from rows 4
        // words (mod 64) apart at words g apart: all banks.  Word 2 h + q: dim 32 i + 16 h + col of tokens 16 q + 4 g ..
        static_assert(kGroup == 32 * kMoveWaves);
        const int t = 32 * wave;
        constexpr int kN = D / 32;
        u32x4 code[kN];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const int tq = t + 16 * q + 4 * g;
            float m[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < kN; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    code[i][2 * h + q] = *reinterpret_cast<const uint32_t *>(&vals[(32 * i + 16 * h + col) * kRow + tq]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) m[e] = fmaxf(m[e], fabsf(code_of<FMT>(code[i], 4 * (2 * h + q) + e)));
                }
            const float4 s = *reinterpret_cast<const float4 *>(&scale_s[tq]);
            uint32_t top = tq < live ? abs_bits(m[0] * s.x) : 0u;
            top = max(top, tq + 1 < live ? abs_bits(m[1] * s.y) : 0u);
            top = max(top, tq + 2 < live ? abs_bits(m[2] * s.z) : 0u);
            top = max(top, tq + 3 < live ? abs_bits(m[3] * s.w) : 0u);
#pragma unroll
            for (int off = 32; off >= 1; off >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, off));
            if (lane == 0) atomicMax(&tops[(t + 16 * q) >> shift], top);
        }
        __syncthreads();
        float scale[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const int tq = t + 16 * q + 4 * g;
            float mul;
            zwg::kvq_scale<FMT>(tops[(t + 16 * q) >> shift], &scale[q], &mul);
            const float4 s4 = *reinterpret_cast<const float4 *>(&scale_s[tq]);
            const float s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
            for (int i = 0; i < kN; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float x[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        x[e] = tq + e < live ? code_of<FMT>(code[i], 4 * (2 * h + q) + e) * s[e] : 0.f;
                    code[i][2 * h + q] = zwg::kvq_encode4<FMT>(x[0], x[1], x[2], x[3], mul);
                }
        }
        await_lower_groups<D>(a, 2 * cu + IS_V, group);
        if (lane == 0)
#pragma unroll
            for (int q = 0; q < 2; ++q)
                if (((t + 16 * q) & (v.block - 1)) == 0 && t0 + t + 16 * q < end) scales[(t0 + t + 16 * q) >> shift] = scale[q];
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            // a last block of 16 may end in the middle of a tile: what lies behind it stays
            uint8_t *to = codes + (int64_t)(t0 + t) * D + 1024 * i + 64 * col + 16 * g;
            if (t0 + t + 16 < end) {
                *reinterpret_cast<u32x4 *>(to) = code[i];
            } else if (t0 + t < end) {
                *reinterpret_cast<uint32_t *>(to) = code[i][0];
                *reinterpret_cast<uint32_t *>(to + 8) = code[i][2];
            }
        }
    }
}

template <int D, int FMT> __global__ __launch_bounds__(kMoveThreads<D>) void kvq_move_kernel(CutArgs a) {
    __shared__ int ticket;
    const int64_t unit2 = blockIdx.x / (unsigned)a.n_groups;
    int group = 0;
    if (a.n_groups > 1) { // else nothing waits
        if (threadIdx.x == 0) ticket = atomicAdd(a.flags + unit2 * a.flag_stride, 1);
        __syncthreads();
        group = ticket;
    }
    if (unit2 & 1)
        move_group<D, FMT, 1>(a, unit2 >> 1, group);
    else
        move_group<D, FMT, 0>(a, unit2 >> 1, group);
}

// ---------------------------------------------------------------------------------------------- host

const char *const kKvqClosed = "the kvq cache's context is closed";

void release(zwg_kvq *kv) {
    if (kv->ctx) {
        (void)hipSetDevice(kv->ctx->device);
        (void)hipStreamSynchronize(kv->ctx->stream);
    }
    if (kv->mem) (void)hipFree(kv->mem);
    kv->mem = nullptr;
    kv->tables.reset();
}

void detach_kvq(void *obj) {
    auto *kv = static_cast<zwg_kvq *>(obj);
    release(kv);
    kv->ctx = nullptr;
}

int create(zwg_ctx *ctx, const zwg_kvq_desc *desc, const zwg_rope *rope, zwg_kvq **out) {
    const std::string msg = check_kvq_desc(*desc);
    if (!msg.empty()) return fail(ctx, msg);
    if (rope) {
        if (rope->ctx != ctx) return fail(ctx, "the rope belongs to another context (or its context is closed)");
        if (rope->desc.d != desc->d) return fail(ctx, "the rope's head dim differs from the cache's");
    }
    hipError_t e = hipSetDevice(ctx->device);
    if (e != hipSuccess) return fail_hip(ctx, "hipSetDevice", e);
    const KvqLayout l = kvq_layout(*desc);
    auto kv = std::make_unique<zwg_kvq>();
    kv->ctx = ctx;
    kv->desc = *desc;
    kv->n_pad = l.n_pad;
    e = hipMalloc(&kv->mem, l.total);
    if (e != hipSuccess) {
        kv->mem = nullptr;
        return fail_hip(ctx, "kvq cache allocation", e);
    }
    uint8_t *p = static_cast<uint8_t *>(kv->mem);
    KvqView &v = kv->view;
    for (int i = 0; i < 2; ++i) {
        v.codes[i] = p;
        p += l.codes;
    }
    for (int i = 0; i < 2; ++i) {
        v.scales[i] = reinterpret_cast<float *>(p);
        p += l.scales;
    }
    for (int i = 0; i < 2; ++i) {
        v.rows[i] = reinterpret_cast<float *>(p);
        p += l.rows;
    }
    v.open = reinterpret_cast<KvqOpen *>(p);
    v.unit_bytes = (int64_t)(l.n_pad * desc->d);
    v.n_blocks = (int32_t)(l.n_pad / desc->block);
    v.block = (int32_t)desc->block;
    v.n_ctx = (int32_t)desc->n_ctx;
    v.d = (int32_t)desc->d;
    v.n_head_kv = (int32_t)desc->n_head_kv;
    v.n_seq = (int32_t)desc->n_seq;
    // zeros: the code of zero, zero scales, no open block (-1)
    e = hipMemsetAsync(v.codes[0], desc->format == ZWG_KVQ_I8 ? 0x80 : 0, 2 * l.codes, ctx->stream);
    if (e == hipSuccess) e = hipMemsetAsync(v.scales[0], 0, 2 * (l.scales + l.rows), ctx->stream);
    if (e == hipSuccess) e = hipMemsetAsync(v.open, 0xff, l.open, ctx->stream);
    const hipError_t es = hipStreamSynchronize(ctx->stream);
    if (e == hipSuccess) e = es;
    if (e != hipSuccess) {
        release(kv.get());
        return fail_hip(ctx, "kvq cache", e);
    }
    if (rope) {
        kv->has_rope = true;
        kv->rope = rope->desc;
        kv->tables = rope->tables;
    }
    add_child(ctx, kv.get(), detach_kvq);
    *out = kv.release();
    return ZWG_OK;
}

#define ZWG_KVQ_DISPATCH(KERNEL, D_, FMT_, ...)                                                                   \
    switch (D_) {                                                                                                \
    case 32: if (FMT_ == ZWG_KVQ_I8) KERNEL<32, 0> __VA_ARGS__; else KERNEL<32, 1> __VA_ARGS__; break;            \
    case 64: if (FMT_ == ZWG_KVQ_I8) KERNEL<64, 0> __VA_ARGS__; else KERNEL<64, 1> __VA_ARGS__; break;            \
    default: if (FMT_ == ZWG_KVQ_I8) KERNEL<128, 0> __VA_ARGS__; else KERNEL<128, 1> __VA_ARGS__; break;          \
    }

int append(zwg_kvq *kv, const KvqAppend &c, float *q_out) {
    zwg_ctx *ctx = kv->ctx;
    const zwg_kvq_desc &d = kv->desc;
    const std::string msg = check_kvq_append(d, kv->has_rope ? &kv->rope : nullptr, c);
    if (!msg.empty()) return fail(ctx, msg);
    if (c.n == 0) return ZWG_OK;
    hipError_t e = hipSetDevice(ctx->device);
    if (e != hipSuccess) return fail_hip(ctx, "hipSetDevice", e);
    AppendArgs a{};
    a.view = kv->view;
    if (kv->has_rope) a.rope = zwg::rope_view(kv->rope, *kv->tables, false);
    a.unit0 = (int64_t)((c.layer * d.n_seq + c.seq0) * d.n_head_kv);
    a.src[0] = c.k;
    a.src[1] = c.v;
    a.q = c.q;
    a.q_out = q_out;
    a.q_stride = (int64_t)c.q_stride;
    a.pos_dev = c.batch ? c.pos_dev : nullptr;
    a.rope_pos_dev = c.batch ? c.rope_pos_dev : nullptr;
    a.pos0 = (int64_t)c.pos;
    a.rope_pos0 = (int64_t)c.rope_pos;
    a.n = (int32_t)c.n;
    a.n_head = (int32_t)c.n_head;
    const uint64_t blocks = c.batch ? c.n : (c.pos + c.n - 1) / d.block - c.pos / d.block + 1;
    const dim3 grid((unsigned)blocks, (unsigned)(2 * d.n_head_kv + (c.q ? c.n_head : 0)));
    ZWG_KVQ_DISPATCH(kvq_append_kernel, d.d, d.format, <<<grid, kAppendThreads, 0, ctx->stream>>>(a))
    e = hipGetLastError();
    return e == hipSuccess ? ZWG_OK : fail_hip(ctx, "kvq append launch", e);
}

int rows(zwg_kvq *kv, uint64_t layer0, uint64_t n_layer, uint64_t seq0, uint64_t n_seq, const int32_t *pos_dev,
         uint64_t pos0, uint64_t n, float *k_out, float *v_out) {
    zwg_ctx *ctx = kv->ctx;
    const zwg_kvq_desc &d = kv->desc;
    const std::string msg = check_kvq_rows(d, layer0, n_layer, seq0, n_seq, pos_dev, pos0, n, k_out, v_out);
    if (!msg.empty()) return fail(ctx, msg);
    if (n_layer == 0 || n_seq == 0 || n == 0 || (!k_out && !v_out)) return ZWG_OK;
    hipError_t e = hipSetDevice(ctx->device);
    if (e != hipSuccess) return fail_hip(ctx, "hipSetDevice", e);
    RowsArgs a{};
    a.view = kv->view;
    a.layer0 = (int64_t)layer0;
    a.seq0 = (int64_t)seq0;
    a.pos_dev = pos_dev;
    a.pos0 = (int64_t)pos0;
    a.n = (int64_t)n;
    a.n_seq = (int32_t)n_seq;
    a.out[0] = k_out;
    a.out[1] = v_out;
    // up to 31 positions of the first tile may lie before the first one asked for
    const uint64_t kbs = (std::min(n, d.n_ctx) + 31 + 31) / 32 * (d.d / 32);
    const dim3 grid((unsigned)((kbs + 3) / 4), (unsigned)(n_layer * n_seq), (unsigned)(2 * d.n_head_kv));
    ZWG_KVQ_DISPATCH(kvq_rows_kernel, d.d, d.format, <<<grid, 256, 0, ctx->stream>>>(a))
    e = hipGetLastError();
    return e == hipSuccess ? ZWG_OK : fail_hip(ctx, "kvq rows launch", e);
}

int evict(zwg_kvq *kv, uint64_t layer0, uint64_t n_layer, uint64_t seq0, uint64_t n_seq, const zwg_kvq_cut *c,
          const float *weights, float *weights_out) {
    zwg_ctx *ctx = kv->ctx;
    const zwg_kvq_desc &d = kv->desc;
    const std::string msg = check_kvq_cut(d, layer0, n_layer, seq0, n_seq, *c, weights, weights_out);
    if (!msg.empty()) return fail(ctx, msg);
    if (n_layer == 0 || n_seq == 0) return ZWG_OK;
    const uint64_t units = n_layer * n_seq * d.n_head_kv;
    const KvqCutPlan plan = kvq_cut_plan(units, d, *c);
    if (plan.bytes > ctx->workspace_bytes) {
        char buf[200];
        snprintf(buf, sizeof buf, "this eviction needs %llu bytes of workspace, more than the context's (%llu): fewer layers or sequences a call",
                 (unsigned long long)plan.bytes, (unsigned long long)ctx->workspace_bytes);
        return fail(ctx, buf);
    }
    hipError_t e = hipSetDevice(ctx->device);
    if (e != hipSuccess) return fail_hip(ctx, "hipSetDevice", e);
    CutArgs a{};
    a.view = kv->view;
    a.layer0 = (int64_t)layer0;
    a.seq0 = (int64_t)seq0;
    a.n_seq = (int32_t)n_seq;
    a.n_kv = (int32_t)c->n_kv;
    a.n_keep = (int32_t)c->n_keep;
    a.n_first = (int32_t)c->n_first;
    a.n_recent = (int32_t)c->n_recent;
    a.w_stride = (int64_t)c->weights_stride;
    a.n_kv_dev = c->n_kv_dev;
    a.n_kv_out = c->n_kv_out;
    a.kept = c->kept;
    a.w = weights;
    a.w_out = weights_out;
    a.dst_stride = (int64_t)plan.row;
    a.n_groups = (int32_t)plan.groups;
    a.flag_stride = (int32_t)plan.flags;
    a.dst = reinterpret_cast<int32_t *>(ctx->workspace); // the new positions first: the kernel reads them 16 bytes at a time
    a.src = a.dst + units * plan.row;
    a.flags = a.src + plan.kept;
    a.count = a.flags + 2 * units * plan.flags;
    kvq_select_kernel<<<(unsigned)units, kSelectThreads, 0, ctx->stream>>>(a);
    e = hipGetLastError();
    if (e != hipSuccess) return fail_hip(ctx, "kvq select launch", e);
    if (c->n_keep >= c->n_kv && !c->n_kv_out) return ZWG_OK; // nothing goes
    ZWG_KVQ_DISPATCH(kvq_move_kernel, d.d, d.format, <<<(unsigned)(2 * units * plan.groups), (unsigned)(2 * kvq_move_group(d.d)), 0, ctx->stream>>>(a))
    e = hipGetLastError();
    return e == hipSuccess ? ZWG_OK : fail_hip(ctx, "kvq move launch", e);
}

} // namespace

extern "C" {

int zwg_kvq_create(zwg_ctx *ctx, const zwg_kvq_desc *desc, const zwg_rope *rope, zwg_kvq **out) {
    if (!out) return fail(ctx, "null output pointer");
    *out = nullptr;
    if (!ctx || !desc) return fail(ctx, "null context or kvq desc");
    return guarded(ctx, [&] { return create(ctx, desc, rope, out); });
}

void zwg_kvq_destroy(zwg_kvq *kv) {
    if (!kv) return;
    if (kv->ctx) remove_child(kv->ctx, kv);
    release(kv);
    delete kv;
}

uint64_t zwg_kvq_bytes(const zwg_kvq_desc *desc) {
    if (!desc) return 0;
    try {
        return check_kvq_desc(*desc).empty() ? kvq_layout(*desc).total : 0;
    } catch (...) {
        return 0;
    }
}

int zwg_kvq_append(zwg_kvq *kv, uint64_t layer, uint64_t seq, uint64_t pos, uint64_t n, uint64_t rope_pos,
                   const float *k_rows, const float *v_rows, const float *q, float *q_out, uint64_t n_head,
                   uint64_t q_stride) {
    if (!kv) return fail(nullptr, "null kvq");
    if (!kv->ctx) return fail(nullptr, kKvqClosed);
    return guarded(kv->ctx, [&] {
        return append(kv, {layer, seq, pos, n, rope_pos, false, nullptr, nullptr, k_rows, v_rows, q, q_out, n_head, q_stride}, q_out);
    });
}

int zwg_kvq_append_batch(zwg_kvq *kv, uint64_t layer, uint64_t seq0, uint64_t n_seq, const int32_t *pos_dev,
                         const int32_t *rope_pos_dev, const float *k_rows, const float *v_rows, const float *q,
                         float *q_out, uint64_t n_head, uint64_t q_stride) {
    if (!kv) return fail(nullptr, "null kvq");
    if (!kv->ctx) return fail(nullptr, kKvqClosed);
    return guarded(kv->ctx, [&] {
        return append(kv, {layer, seq0, 0, n_seq, 0, true, pos_dev, rope_pos_dev, k_rows, v_rows, q, q_out, n_head, q_stride}, q_out);
    });
}

int zwg_kvq_rows_dev(zwg_kvq *kv, uint64_t layer0, uint64_t n_layer, uint64_t seq0, uint64_t n_seq,
                     const int32_t *pos_dev, uint64_t pos0, uint64_t n, float *k_out, float *v_out) {
    if (!kv) return fail(nullptr, "null kvq");
    if (!kv->ctx) return fail(nullptr, kKvqClosed);
    return guarded(kv->ctx, [&] { return rows(kv, layer0, n_layer, seq0, n_seq, pos_dev, pos0, n, k_out, v_out); });
}

int zwg_kvq_evict_dev(zwg_kvq *kv, uint64_t layer0, uint64_t n_layer, uint64_t seq0, uint64_t n_seq,
                      const zwg_kvq_cut *cut, const float *weights, float *weights_out) {
    if (!kv) return fail(nullptr, "null kvq");
    if (!kv->ctx) return fail(nullptr, kKvqClosed);
    if (!cut) return fail(kv->ctx, "null cut");
    return guarded(kv->ctx, [&] { return evict(kv, layer0, n_layer, seq0, n_seq, cut, weights, weights_out); });
}

} // extern "C"
