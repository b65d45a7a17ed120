// The host side of the rotary positions and the 8-bit caches (zwhisper_amd/csrc/kvq_plan.hpp) built on its own, with no
// GPU, under the address and undefined-behaviour sanitizers: the argument rules on calls that break them one by one, the
// layout of codes (every byte of a unit once), the key splits and workspaces.  Built and run by tests/test_kvq_host.py.
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <limits>
#include <random>
#include <vector>

#include "kvq_plan.hpp"

using namespace zwg_planner;

static int g_fail = 0;
#define CHECK(cond, ...)                                                                                           \
    do {                                                                                                           \
        if (!(cond)) {                                                                                             \
            std::fprintf(stderr, "FAIL %s:%d: %s | ", __FILE__, __LINE__, #cond);                                \
            std::fprintf(stderr, __VA_ARGS__);                                                                     \
            std::fprintf(stderr, "\n");                                                                            \
            if (++g_fail > 20) std::exit(1);                                                                       \
        }                                                                                                          \
    } while (0)

static const uint64_t kMax = std::numeric_limits<uint64_t>::max();
static float *at(uint64_t a) { return reinterpret_cast<float *>(a); }
static int32_t *iat(uint64_t a) { return reinterpret_cast<int32_t *>(a); }
static bool says(const std::string &msg, const char *part) { return msg.find(part) != std::string::npos; }

static void layout() {
    for (int d : {32, 64, 128})
        for (int is_v = 0; is_v < 2; ++is_v) {
            std::vector<int> hit(192 * d);
            for (int t = 0; t < 192; ++t)
                for (int c = 0; c < d; ++c) {
                    const int64_t a = zwg::kvq_at(is_v, t, c, d);
                    CHECK(a >= 0 && a < 192 * d, "byte %lld", (long long)a);
                    if (a >= 0 && a < 192 * d) ++hit[a];
                    // what the lanes of a wave expect at 16 bytes each
                    const int kb = (int)(a / 1024), l = (int)(a % 1024) / 64, g = (int)(a % 64) / 16, e = (int)(a % 16);
                    if (is_v) {
                        CHECK(t == 32 * (kb / (d / 32)) + 16 * (e / 4 % 2) + 4 * g + e % 4, "token %d", t);
                        CHECK(c == 32 * (kb % (d / 32)) + 16 * (e / 8) + l, "dim %d", c);
                    } else if (d == 32) {
                        CHECK(t == 32 * kb + 16 * (e / 8) + l && c == 8 * g + e % 8, "token %d dim %d", t, c);
                    } else {
                        CHECK(t == 16 * (kb / (d / 64)) + l && c == 64 * (kb % (d / 64)) + 16 * g + e, "token %d dim %d", t, c);
                    }
                }
            for (int h : hit) CHECK(h == 1, "a byte is used %d times", h);
        }
    zwg_kvq_desc k{2, 3, 100, 2, 64, 32, ZWG_KVQ_I8, 0};
    const KvqLayout l = kvq_layout(k);
    CHECK(l.units == 12 && l.n_pad == 128 && l.codes >= 12 * 128 * 64 && l.scales >= 12 * 4 * 4, "sizes");
    CHECK(l.codes % 256 == 0 && l.scales % 256 == 0 && l.rows % 256 == 0, "alignment");
    CHECK(l.open >= 24 * sizeof(zwg::KvqOpen), "open");
}

static void descs() {
    const zwg_kvq_desc good{1, 1, 64, 2, 64, 32, ZWG_KVQ_I8, 0};
    CHECK(check_kvq_desc(good).empty(), "good");
    auto bad = [&](auto change, const char *part) {
        zwg_kvq_desc d = good;
        change(d);
        CHECK(says(check_kvq_desc(d), part), "%s: %s", part, check_kvq_desc(d).c_str());
    };
    bad([](auto &d) { d.d = 96; }, "head dim");
    bad([](auto &d) { d.block = 0; }, "block");
    bad([](auto &d) { d.block = 128; }, "block");
    bad([](auto &d) { d.format = 2; }, "format");
    bad([](auto &d) { d.reserved = 1; }, "reserved");
    bad([](auto &d) { d.n_ctx = 0; }, "positive");
    bad([](auto &d) { d.n_ctx = 1ull << 25; }, "below 2^31");
    bad([](auto &d) { d.n_ctx = kMax; }, "below 2^31");
    bad([](auto &d) { d.n_layer = kMax; }, "out of range");
    bad([](auto &d) { d.n_seq = 65535, d.n_layer = 65535; }, "below 2^31");
    const zwg_rope_desc rope{100, 64, 64, 0, 0, 1e6, 1.0, 0, 0, 0, 0};
    CHECK(check_rope_desc(rope).empty(), "good rope");
    auto badr = [&](auto change, const char *part) {
        zwg_rope_desc d = rope;
        change(d);
        CHECK(says(check_rope_desc(d), part), "%s: %s", part, check_rope_desc(d).c_str());
    };
    badr([](auto &d) { d.d = 0; }, "head dim");
    badr([](auto &d) { d.n_rot = 63; }, "even");
    badr([](auto &d) { d.n_rot = 128; }, "even");
    badr([](auto &d) { d.n_ctx = kMax; }, "n_ctx");
    badr([](auto &d) { d.base = -1; }, "base");
    badr([](auto &d) { d.base = NAN; }, "base");
    badr([](auto &d) { d.factor = INFINITY; }, "factor");
    badr([](auto &d) { d.mscale = NAN; }, "mscale");
    badr([](auto &d) { d.scaling = ZWG_ROPE_YARN; }, "n_orig");
    badr([](auto &d) { d.scaling = ZWG_ROPE_YARN, d.n_orig = 10, d.beta_fast = 1, d.beta_slow = 2; }, "beta");
    badr([](auto &d) { d.scaling = ZWG_ROPE_NTK, d.n_rot = 2; }, "NTK");
    // scalings by 1 change nothing
    for (uint32_t s : {ZWG_ROPE_NONE, ZWG_ROPE_LINEAR, ZWG_ROPE_NTK, ZWG_ROPE_YARN}) {
        zwg_rope_desc d = rope;
        d.scaling = s;
        d.n_orig = 10;
        CHECK(rope_frequencies(d) == rope_frequencies(rope) || s == ZWG_ROPE_YARN, "scaling %u", s);
        for (size_t j = 0; j < 32; ++j)
            CHECK(std::fabs(rope_frequencies(d)[j] / rope_frequencies(rope)[j] - 1) < 1e-15, "scaling %u pair %zu", s, j);
        CHECK(rope_mscale(d) == 1.0, "mscale %u", s);
    }
    // rope calls
    const auto x = at(0x10000), far = at(0x90000);
    CHECK(check_rope_apply(rope, x, 100, 2, 128, nullptr, 0, x, 128, 0).empty(), "in place");
    CHECK(check_rope_apply(rope, x, 100, 2, 128, nullptr, 0, far, 132, 1).empty(), "apart");
    CHECK(check_rope_apply(rope, nullptr, 0, 0, 0, nullptr, kMax, nullptr, 0, 0).empty(), "no rows");
    CHECK(says(check_rope_apply(rope, x, 100, 2, 128, nullptr, 1, x, 128, 0), "past"), "pos0");
    CHECK(says(check_rope_apply(rope, x, 1, 2, 128, nullptr, kMax, x, 128, 0), "past"), "pos0 wraps");
    CHECK(says(check_rope_apply(rope, x, 2, 2, 128, nullptr, 0, x, 132, 0), "in place"), "strides in place");
    CHECK(says(check_rope_apply(rope, x, 2, 2, 128, nullptr, 0, x + 4, 128, 0), "overlap"), "overlap");
    CHECK(says(check_rope_apply(rope, x, 2, 2, 124, nullptr, 0, far, 128, 0), "smaller"), "stride");
    CHECK(says(check_rope_apply(rope, x, 2, 2, kMax - 3, nullptr, 0, far, 128, 0), "out of range"), "stride");
    CHECK(says(check_rope_apply(rope, at(0x10004), 2, 2, 128, nullptr, 0, far, 128, 0), "16-byte"), "alignment");
    CHECK(says(check_rope_apply(rope, x, 2, 2, 128, iat(0x10002), 0, far, 128, 0), "4-byte"), "alignment");
    CHECK(says(check_rope_apply(rope, x, 2, 70000, 1 << 24, nullptr, 0, far, 1 << 24, 0), "n_head"), "heads");
    CHECK(says(check_rope_apply(rope, x, 2, 2, 128, nullptr, 0, far, 128, 2), "flags"), "flags");
}

static void calls() {
    const zwg_kvq_desc d{2, 4, 100, 2, 64, 32, ZWG_KVQ_I8, 0};
    const zwg_rope_desc rope{50, 64, 64, 0, 0, 1e6, 1.0, 0, 0, 0, 0};
    const auto x = at(0x10000);
    const KvqAppend good{0, 0, 0, 10, 0, false, nullptr, nullptr, x, x, x, x, 4, 256};
    CHECK(check_kvq_append(d, &rope, good).empty(), "good");
    auto bad = [&](auto change, const char *part, bool with_rope = true) {
        KvqAppend a = good;
        change(a);
        const std::string m = check_kvq_append(d, with_rope ? &rope : nullptr, a);
        CHECK(says(m, part), "%s: %s", part, m.c_str());
    };
    bad([](auto &a) { a.layer = 2; }, "layer");
    bad([](auto &a) { a.seq0 = kMax; }, "sequence");
    bad([](auto &a) { a.pos = 91; }, "end of the cache");
    bad([](auto &a) { a.pos = kMax - 5; }, "end of the cache");
    bad([](auto &a) { a.n = kMax; }, "end of the cache");
    bad([](auto &a) { a.rope_pos = 41; }, "end of the rope");
    bad([](auto &a) { a.rope_pos = kMax; }, "end of the rope");
    bad([](auto &) {}, "has a rope", false);
    bad([](auto &a) { a.k = nullptr; }, "null k");
    bad([](auto &a) { a.v = at(0x10008); }, "16-byte");
    bad([](auto &a) { a.q_out = nullptr; }, "null q");
    bad([](auto &a) { a.q = at(0x10004); }, "16-byte");
    bad([](auto &a) { a.n_head = 3; }, "multiple");
    bad([](auto &a) { a.n_head = 0; }, "multiple");
    bad([](auto &a) { a.n_head = kMax - 1; }, "out of range");
    bad([](auto &a) { a.q_stride = 252; }, "smaller");
    bad([](auto &a) { a.q_stride = 257; }, "multiple of 4");
    bad([](auto &a) { a.batch = true; }, "null position");
    bad([](auto &a) { a.batch = true, a.pos_dev = iat(0x10001); }, "4-byte");
    bad([](auto &a) { a.batch = true, a.pos_dev = iat(0x10000), a.n = 5; }, "sequences");
    bad([](auto &a) { a.batch = true, a.pos_dev = iat(0x10000), a.seq0 = kMax; }, "sequences");

    CHECK(check_kvq_rows(d, 0, 2, 0, 4, nullptr, 0, 100, x, nullptr).empty(), "rows");
    CHECK(says(check_kvq_rows(d, 1, 2, 0, 4, nullptr, 0, 100, x, x), "layers"), "rows");
    CHECK(says(check_kvq_rows(d, kMax, 2, 0, 4, nullptr, 0, 100, x, x), "layers"), "rows");
    CHECK(says(check_kvq_rows(d, 0, 2, 1, kMax, nullptr, 0, 100, x, x), "sequences"), "rows");
    CHECK(says(check_kvq_rows(d, 0, 2, 0, 4, nullptr, kMax, 100, x, x), "positions"), "rows");
    CHECK(says(check_kvq_rows(d, 0, 2, 0, 4, nullptr, 0, 1, at(4), x), "16-byte"), "rows");

    const zwg_kvq_cut cut{100, 50, 10, 40, 100, nullptr, nullptr, nullptr};
    CHECK(check_kvq_cut(d, 0, 2, 0, 4, cut, x, x).empty(), "cut");
    auto badc = [&](auto change, const char *part, const float *w = at(0x10000)) {
        zwg_kvq_cut c = cut;
        change(c);
        CHECK(says(check_kvq_cut(d, 0, 2, 0, 4, c, w, nullptr), part), "%s", part);
    };
    badc([](auto &c) { c.n_kv = 101; }, "n_ctx");
    badc([](auto &c) { c.n_keep = 0; }, "n_keep");
    badc([](auto &c) { c.n_keep = (1u << 24) + 1; }, "n_keep");
    badc([](auto &c) { c.n_keep = 0x7fffffff; }, "n_keep");
    badc([](auto &c) { c.n_first = 11; }, "n_first");
    badc([](auto &c) { c.n_first = 2, c.n_recent = kMax; }, "n_first");
    badc([](auto &c) { c.weights_stride = 99; }, "weights_stride");
    badc([](auto &) {}, "null weights", nullptr);
    badc([](auto &c) { c.kept = iat(2); }, "4-byte");

    const zwg_kvq_attn at0{3, 100, 4, 256, 256, 768, 768, 100, 200, nullptr, 1.0f, 1};
    CHECK(check_kvq_attn(d, 0, 0, 4, x, at0, x, x).empty(), "attention");
    auto bada = [&](auto change, const char *part) {
        zwg_kvq_attn a = at0;
        change(a);
        CHECK(says(check_kvq_attn(d, 0, 0, 4, x, a, x, x), part), "%s: %s", part, check_kvq_attn(d, 0, 0, 4, x, a, x, x).c_str());
    };
    bada([](auto &a) { a.n_head = 5; }, "multiple");
    bada([](auto &a) { a.n_head = 0; }, "multiple");
    bada([](auto &a) { a.n_kv = 101; }, "n_ctx");
    bada([](auto &a) { a.n_q = kMax; }, "out of range");
    bada([](auto &a) { a.causal = 2; }, "causal");
    bada([](auto &a) { a.q_stride = 252; }, "smaller");
    bada([](auto &a) { a.out_bstride = 6; }, "multiples of 4");
    bada([](auto &a) { a.q_bstride = kMax - 3; }, "out of range");
    bada([](auto &a) { a.decay = -0.5f; }, "decay");
    bada([](auto &a) { a.decay = NAN; }, "decay");
    bada([](auto &a) { a.weights_stride = 50; }, "weights_stride");
    bada([](auto &a) { a.weights_bstride = 150; }, "weights_bstride");
    bada([](auto &a) { a.n_kv_dev = iat(3); }, "4-byte");
    CHECK(says(check_kvq_attn(d, 2, 0, 4, x, at0, x, x), "layer"), "layer");
    CHECK(says(check_kvq_attn(d, 0, 1, 4, x, at0, x, x), "sequences"), "sequences");
    CHECK(says(check_kvq_attn(d, 0, 0, 4, nullptr, at0, x, x), "null"), "null");
}

// Every row's keys are covered by its chunks, and the partials fit.
static void splits() {
    std::mt19937_64 rng(5);
    for (int it = 0; it < 20000; ++it) {
        const uint64_t n_kv = rng() % (it % 2 ? 300 : 200000), units = 1 + rng() % (it % 3 ? 64 : 5000), RB = rng() % 2 ? 8 : 32;
        const uint64_t rows = units * (1 + rng() % RB), d = 32u << (rng() % 3);
        const bool weights = rng() % 2;
        const uint64_t ws = rng() % 4 ? 256ull << 20 : 1 + rng() % (1 << 20);
        const KvqSplit s = kvq_split(units, n_kv, rows, d, weights, ws, it % 5 == 0);
        CHECK(s.chunk_len > 0 && s.chunk_len % kKvqSplitTile == 0 && s.max_chunks >= 1 && s.max_chunks <= (int)kKvqMaxChunks, "split");
        const KvqWorkspace w = kvq_workspace(rows, (uint64_t)s.max_chunks, d, weights);
        CHECK(s.max_chunks == 1 || w.total * 4 <= ws, "workspace %llu of %llu", (unsigned long long)w.total * 4, (unsigned long long)ws);
        CHECK(w.part_ml % 64 == 0 && w.part_o % 64 == 0 && w.part_ml >= (weights ? 2 * rows : 0), "layout");
        for (int k = 0; k < 8; ++k) {
            const int hi = k == 0 ? (int)n_kv : (int)(rng() % (n_kv + 1));
            int keys = 0;
            const int n = zwg::unit_split(hi, kKvqSplitTile, s.chunk_len, s.max_chunks, &keys);
            CHECK(n >= 1 && n <= s.max_chunks && keys % kKvqSplitTile == 0 && (int64_t)n * keys >= hi &&
                      (hi == 0 || (int64_t)(n - 1) * keys < hi), "cover %d: %d of %d", hi, n, keys);
        }
    }
}

// An eviction's groups cover the kept tokens; its lists, flags and ticket are counted; its grid stays in range.
static void cuts() {
    std::mt19937_64 rng(6);
    for (int it = 0; it < 20000; ++it) {
        const zwg_kvq_desc d{1, 1, 1 << 24, 1, 32u << (rng() % 3), 16u << (rng() % 3), ZWG_KVQ_I8, 0};
        const uint64_t units = 1 + rng() % 300;
        zwg_kvq_cut c{};
        c.n_kv = rng() % (it % 2 ? 5000 : 1 << 24);
        c.n_keep = 1 + rng() % (c.n_kv + 10);
        const KvqCutPlan p = kvq_cut_plan(units, d, c);
        const uint64_t group = kvq_move_group(d.d);
        if (c.n_keep < c.n_kv) {
            CHECK(p.groups * group >= c.n_keep && (p.groups - 1) * group < c.n_keep, "groups");
            CHECK(p.row % 32 == 0 && p.row >= c.n_kv && p.kept % 32 == 0 && p.kept >= units * c.n_keep, "rows");
            CHECK(p.flags % 32 == 0 && p.flags > p.groups, "flags");
        } else {
            CHECK(p.groups == 1 && p.row == 0 && p.kept == 0 && p.flags == 0, "nothing to cut");
        }
        CHECK(p.bytes == 4 * (units * (p.row + 2 * p.flags + 1) + p.kept), "bytes");
    }
    // 2^21 workgroups at most
    const float *w = reinterpret_cast<const float *>(256);
    const uint64_t group = kvq_move_group(128);
    zwg_kvq_desc d{1u << 21, 1, 4096, 1, 128, 16, ZWG_KVQ_I8, 0};
    zwg_kvq_cut c{};
    c.n_kv = 4096;
    c.n_keep = group;
    c.weights_stride = 4096;
    CHECK(check_kvq_cut(d, 0, 1u << 20, 0, 1, c, w, nullptr).empty(), "in range");
    CHECK(!check_kvq_cut(d, 0, (1u << 20) + 1, 0, 1, c, w, nullptr).empty(), "out of range");
    c.n_keep = group + 1;
    CHECK(!check_kvq_cut(d, 0, (1u << 19) + 1, 0, 1, c, w, nullptr).empty(), "two groups");
}

int main() {
    cuts();
    layout();
    descs();
    calls();
    splits();
    if (g_fail) return 1;
    std::puts("ok");
    return 0;
}
