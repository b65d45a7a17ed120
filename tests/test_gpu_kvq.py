"""The 8-bit caches (zwg_kvq_*) against the plain restatement in _kvq_ref.py: stored values and kept positions equal
to the bit, attention and weights within bounds derived from the arithmetic (_kvq_ref.tolerance)."""
from __future__ import annotations

import re

import numpy as np
import pytest

import _kvq_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no GPU on this machine")
    return torch


@pytest.fixture(scope="module")
def z():
    import zwhisper_amd as z

    return z


@pytest.fixture(scope="module")
def ctx(torch, z):
    c = z.Context(0)
    yield c
    c.close()


FMT = ["i8", "e4m3"]


def fmt_of(z, name):
    return {"i8": z.KVQ_I8, "e4m3": z.KVQ_E4M3}[name]


def dev(torch, a, dtype=np.float32):
    return torch.from_numpy(np.ascontiguousarray(a, dtype)).cuda()


def values(torch, kv, layer, seq, n):
    k = torch.full((n, kv.n_head_kv, kv.d), 99.0, device="cuda")
    v = torch.full_like(k, 99.0)
    kv.rows(layer, 1, seq, 1, n, k, v)
    return k.cpu().numpy(), v.cpu().numpy()


def same(a, b):
    return np.array_equal(a, b, equal_nan=True)


# ---------------------------------------------------------------------------------------------- appends


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("d,heads,block", [(128, 2, 32), (64, 3, 16), (32, 1, 64), (64, 2, 64)])
def test_appends(torch, z, ctx, d, heads, block, fmt):
    """Prompts and tokens in every position of a block, rewound and skipped positions, the last position, another
    layer and sequence: the stored values are the definition's, and nothing else changes."""
    n_ctx = 300  # ends inside a block and inside a tile
    rng = np.random.default_rng(d + block)
    with z.KVQCache(ctx, 2, 2, n_ctx, heads, d, block, fmt_of(z, fmt)) as kv:
        want = {(l, s): ref.Cache(n_ctx, heads, d, block, fmt) for l in range(2) for s in range(2)}
        calls = [(0, 0, 0, 1), (0, 0, 1, 1), (0, 0, 2, 5), (0, 0, 7, block + 3), (0, 0, block + 10, 1), (0, 0, block + 11, 3 * block - 11),
                 (0, 0, 4 * block, 1), (0, 0, block + 5, 1), (0, 0, block + 3, 2), (0, 0, block + 9, 1), (1, 1, 3, 2), (1, 1, 5, 90),
                 (0, 1, 0, 299), (0, 1, 299, 1), (1, 0, 290, 10), (1, 0, 17, 200), (0, 1, 40, 1), (0, 1, 41, 2 * block)]
        for i, (layer, seq, pos, n) in enumerate(calls):
            if pos + n > n_ctx:
                n = n_ctx - pos
            k, v = (rng.standard_normal((n, heads, d)) * 10.0 ** rng.integers(-2, 3) for _ in range(2))
            k, v = k.astype(np.float32), v.astype(np.float32)
            kv.append(layer, seq, pos, dev(torch, k), dev(torch, v))
            want[layer, seq].append(pos, k, v)
            for (a, b), c in want.items():
                got = values(torch, kv, a, b, n_ctx)
                for j in range(2):
                    assert same(got[j], c.vals[j][:n_ctx]), (i, (layer, seq, pos, n), (a, b), "kv"[j])


@pytest.mark.parametrize("fmt", FMT)
def test_token_by_token_equals_at_once(torch, z, ctx, fmt):
    """A block filled token by token holds what one append of all its rows gives, and batches of one token in several
    sequences what appends one by one give."""
    n, heads, d, S = 75, 2, 128, 5
    rng = np.random.default_rng(1)
    k, v = (dev(torch, rng.standard_normal((S, n, heads, d))) for _ in range(2))
    with z.KVQCache(ctx, 1, S, 128, heads, d, 32, fmt_of(z, fmt)) as a, z.KVQCache(ctx, 1, S, 128, heads, d, 32, fmt_of(z, fmt)) as b:
        for s in range(S):
            a.append(0, s, 0, k[s], v[s])
        for i in range(n):
            b.append_batch(0, 0, torch.full((S,), i, dtype=torch.int32, device="cuda"), k[:, i].contiguous(), v[:, i].contiguous())
        for s in range(S):
            for x, y in zip(values(torch, a, 0, s, 128), values(torch, b, 0, s, 128)):
                assert np.array_equal(x, y)


@pytest.mark.parametrize("fmt", FMT)
def test_extreme_values(torch, z, ctx, fmt):
    """Zeros, tiny and huge rows, infinities and NaNs: a block with a number that is none reads as NaN and no other
    block does; once its rows are appended again it is as if they had never been."""
    heads, d, B = 2, 64, 16
    rng = np.random.default_rng(2)
    with z.KVQCache(ctx, 1, 1, 96, heads, d, B, fmt_of(z, fmt)) as kv:
        c = ref.Cache(96, heads, d, B, fmt)
        k = rng.standard_normal((96, heads, d)).astype(np.float32)
        v = rng.standard_normal((96, heads, d)).astype(np.float32)
        k[0:16] = 0
        k[16:32] *= 1e-35
        v[0:16] *= 2.0 ** -98
        v[16:32] = 3.3e38
        k[40, 1, 3] = np.inf
        v[50, 0, 63] = np.nan
        v[70, 1, 0] = -np.inf
        v[80:96] *= 1e-37
        v[81, 0, 5] = 1.0
        kv.append(0, 0, 0, dev(torch, k), dev(torch, v))
        c.append(0, k, v)
        for g, w in zip(values(torch, kv, 0, 0, 96), c.vals):
            assert same(g, w[:96])
        assert np.isnan(c.vals[0][32:48, 1]).all() and np.isfinite(c.vals[0][32:48, 0]).all()
        for pos, n in ((40, 1), (40, 8), (50, 14)):
            a, b = (rng.standard_normal((n, heads, d)).astype(np.float32) for _ in range(2))
            kv.append(0, 0, pos, dev(torch, a), dev(torch, b))
            c.append(pos, a, b)
            for g, w in zip(values(torch, kv, 0, 0, 96), c.vals):
                assert same(g, w[:96]), pos


@pytest.mark.parametrize("layout,n_rot,scaling,factor", [("half", 64, "none", 1.0), ("interleaved", 64, "yarn", 4.0),
                                                         ("half", 32, "linear", 2.0), ("interleaved", 18, "none", 1.0)])
def test_rotated_appends(torch, z, ctx, layout, n_rot, scaling, factor):
    """Keys and queries rotated at positions of their own, queries in place and beside; skipped sequences stay."""
    heads, n_head, d, B, S = 2, 6, 64, 32, 4
    rng = np.random.default_rng(n_rot)
    w, m = ref.rope_freqs(n_rot, 1e6, scaling, factor, 64)
    rope = z.Rope(ctx, 500, d, n_rot, {"half": z.ROPE_HALF, "interleaved": z.ROPE_INTERLEAVED}[layout], 1e6,
                  {"none": z.ROPE_NONE, "linear": z.ROPE_LINEAR, "yarn": z.ROPE_YARN}[scaling], factor, n_orig=64)
    turn = lambda x, pos: ref.rotate(x, pos, n_rot, layout, w, m, rounded=True).astype(np.float32)  # noqa: E731
    kv = z.KVQCache(ctx, 1, S, 200, heads, d, B, z.KVQ_I8, rope)
    rope.close()  # the cache keeps the tables
    want = [ref.Cache(200, heads, d, B, "i8") for _ in range(S)]
    off = 0
    for pos, n, rp in ((0, 45, 0), (45, 100, 300), (145, 1, 499)):
        k, v, q = (rng.standard_normal((n, h, d)).astype(np.float32) for h in (heads, heads, n_head))
        qd = dev(torch, q)
        out = torch.zeros_like(qd)
        kv.append(0, 1, pos, dev(torch, k), dev(torch, v), q=qd, n_head=n_head, q_out=out, rope_pos=rp)
        want[1].append(pos, turn(k, rp + np.arange(n)), v)
        off += np.count_nonzero(out.cpu().numpy() != turn(q, rp + np.arange(n)))
        kv.append(0, 1, pos, dev(torch, k), dev(torch, v), q=qd, n_head=n_head, rope_pos=rp)
        want[1].append(pos, turn(k, rp + np.arange(n)), v)
        assert torch.equal(qd, out)
    slots, rps = np.array([199, 3, -1, 200], np.int32), np.array([7, 500, 3, 4], np.int32)
    k, v, q = (rng.standard_normal((S, h, d)).astype(np.float32) for h in (heads, heads, n_head))
    out = torch.full((S, n_head + 1, d), 5.0, device="cuda")
    qd = torch.zeros(S, n_head + 1, d, device="cuda")
    qd[:, :n_head] = dev(torch, q)
    kv.append_batch(0, 0, dev(torch, slots, np.int32), dev(torch, k), dev(torch, v), q=qd, n_head=n_head,
                    q_stride=(n_head + 1) * d, q_out=out, rope_pos_dev=dev(torch, rps, np.int32))
    want[0].append(199, turn(k[:1], [7]), v[:1])
    off += np.count_nonzero(out[0, :n_head].cpu().numpy() != turn(q[:1], [7])[0])
    assert (out[1:] == 5.0).all() and (out[:, n_head:] == 5.0).all()
    assert off < 5  # a sine of another library may round the other way
    for s in range(S):
        for g, c in zip(values(torch, kv, 0, s, 200), want[s].vals):
            # a key that rounds the other way may move by a step of its block
            assert np.mean(g != c[:200]) < 1e-3, s
    kv.close()


def test_rows(torch, z, ctx):
    """Ranges of layers, sequences and positions of their own; positions outside the cache are not written."""
    L, S, N, H, d = 3, 3, 70, 2, 32
    rng = np.random.default_rng(5)
    with z.KVQCache(ctx, L, S, N, H, d, 16) as kv:
        whole = np.zeros((2, L, S, N, H, d), np.float32)
        for layer in range(L):
            for s in range(S):
                k, v = (rng.standard_normal((N, H, d)).astype(np.float32) for _ in range(2))
                kv.append(layer, s, 0, dev(torch, k), dev(torch, v))
                c = ref.Cache(N, H, d, 16, "i8")
                c.append(0, k, v)
                whole[0, layer, s], whole[1, layer, s] = c.vals[0][:N], c.vals[1][:N]
        k, v = torch.full((2, 2, 50, H, d), 4.0, device="cuda"), torch.full((2, 2, 50, H, d), 4.0, device="cuda")
        kv.rows(1, 2, 1, 2, 50, k, v, pos=torch.tensor([33, -7], dtype=torch.int32, device="cuda"))
        for t, got in enumerate((k.cpu().numpy(), v.cpu().numpy())):
            assert np.array_equal(got[:, 0, :37], whole[t, 1:, 1, 33:]) and (got[:, 0, 37:] == 4.0).all()
            assert np.array_equal(got[:, 1, 7:], whole[t, 1:, 2, :43]) and (got[:, 1, :7] == 4.0).all()
        only = torch.zeros(1, 1, 5, H, d, device="cuda")
        kv.rows(0, 1, 2, 1, 5, None, only, pos=65)
        assert np.array_equal(only.cpu().numpy()[0, 0], whole[1, 0, 2, 65:])


# ---------------------------------------------------------------------------------------------- attention


def filled(torch, z, ctx, S, n_ctx, H, d, block, fmt, lens, rng, spread=1.0):
    kv = z.KVQCache(ctx, 1, S, n_ctx, H, d, block, fmt_of(z, fmt))
    stored = []
    for s in range(S):
        c = ref.Cache(n_ctx, H, d, block, fmt)
        if lens[s]:
            chan = np.exp(0.7 * rng.standard_normal(d))
            k, v = ((rng.standard_normal((lens[s], H, d)) * chan * spread).astype(np.float32) for _ in range(2))
            kv.append(0, s, 0, dev(torch, k), dev(torch, v))
            c.append(0, k, v)
        stored.append(c)
    return kv, stored


ATTEND = [  # lens, n_q, n_head, H, d, block, causal
    ([1], 1, 6, 6, 64, 16, True), ([0, 5, 64, 65, 187], 1, 12, 2, 128, 32, True), ([300], 1, 7, 1, 64, 64, False),
    ([513, 31], 1, 8, 1, 32, 16, True), ([200], 3, 4, 2, 128, 32, True), ([64, 80], 2, 4, 1, 64, 16, False),
    ([130], 130, 2, 1, 64, 32, True), ([257, 40, 33], 33, 6, 2, 128, 32, True), ([300], 9, 24, 2, 64, 64, False),
    ([1500], 5, 6, 6, 32, 32, False), ([40, 3], 9, 2, 1, 128, 16, True), ([1000], 40, 3, 1, 32, 16, True),
    ([2100], 1, 12, 2, 128, 64, True),
    # calls of the prompt kernel: rows that fill no workgroup, sequences of unlike lengths, keys in many chunks
    ([1500, 1490, 700], 560, 14, 2, 128, 32, True), ([3000], 1111, 6, 1, 64, 64, True), ([2900, 17], 700, 12, 2, 32, 16, False),
    ([17000], 130, 2, 1, 128, 64, True),
]


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("case", ATTEND, ids=lambda c: f"{c[0]}-{c[1:]}".replace(" ", ""))
def test_attention(torch, z, ctx, case, fmt):
    """Decode, several queries and prompts; ragged lengths (some rows see nothing); head groups of every size; with and
    without weights; strided queries and outputs whose gaps stay."""
    lens, n_q, n_head, H, d, block, causal = case
    rng = np.random.default_rng(sum(lens) + n_q + d)
    S, N = len(lens), max(lens)
    kv, stored = filled(torch, z, ctx, S, N + 70, H, d, block, fmt, lens, rng)
    q = rng.standard_normal((S, n_q, n_head, d)).astype(np.float32) * 2
    qs, os_ = n_head * d + 4, n_head * d + 12
    qd = torch.zeros(S, n_q, qs, device="cuda")
    qd[..., : n_head * d] = dev(torch, q).flatten(2)
    out = torch.full((S, n_q, os_), 9.0, device="cuda")
    w0 = rng.random((S, H, N + 3)).astype(np.float32)
    w = dev(torch, w0)
    n_dev = dev(torch, lens, np.int32)
    kw = dict(n_q=n_q, n_head=n_head, n_kv=N, causal=causal, n_kv_dev=n_dev, q_stride=qs, out_stride=os_)
    kv.attention(0, 0, S, qd, out, weights=w, decay=0.5, weights_stride=N + 3, **kw)
    plain = torch.full_like(out, 9.0)
    kv.attention(0, 0, S, qd, plain, **kw)
    assert torch.equal(out, plain)  # the weights change nothing of the output
    got, gw = out.cpu().numpy(), w.cpu().numpy()
    assert (got[..., n_head * d:] == 9.0).all()
    for s in range(S):
        k, v = stored[s].vals
        want, wsum, size = ref.attend(q[s], k, v, lens[s], causal)
        tol, rel = ref.tolerance(size, np.abs(v).max())
        assert np.abs(got[s, :, : n_head * d].reshape(n_q, n_head, d) - want).max() <= tol, s
        n = lens[s]
        # the old weights' halves and up to n_q n_head sums round too
        bound = (rel + n_q * n_head * 2.0 ** -24) * wsum + 2.0 ** -23 * (w0[s, :, :n] + wsum) + 1e-30
        assert (np.abs(gw[s, :, :n] - (0.5 * w0[s, :, :n].astype(np.float64) + wsum)) <= bound).all(), s
        assert np.array_equal(gw[s, :, n:], w0[s, :, n:])
    kv.close()


SPLIT_STEPS = [  # decode steps whose keys are split: up to 16 chunks beside whole and empty sequences, and more than 16
    ([6000, 1, 0, 900, 300], 1, 12, 2, 128, 32, True), ([5200, 3000], 2, 6, 2, 64, 16, True), ([7000], 4, 2, 1, 32, 32, False),
    ([12000], 1, 8, 1, 32, 64, True),
]


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("case", SPLIT_STEPS, ids=lambda c: f"{c[0]}-{c[1:]}".replace(" ", ""))
def test_weights_of_split_steps(torch, z, ctx, case, fmt):
    """As test_attention, where the weights form the rows' statistics from those of their chunks, and where they do not."""
    test_attention(torch, z, ctx, case, fmt)


@pytest.mark.parametrize("n_q", [1, 40])
def test_split_keys_and_small_workspaces(torch, z, ctx, n_q):
    """One long sequence over many chunks, in contexts whose workspaces hold fewer chunks, down to none: within the bounds
    each, and calls without weights need no workspace at all."""
    H, n_head, d, N = 1, 4, 64, 20000
    rng = np.random.default_rng(8)
    k, v = (rng.standard_normal((N, H, d)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((n_q, n_head, d)).astype(np.float32)
    c = ref.Cache(N, H, d, 32, "i8")
    c.append(0, k, v)
    want, wsum, size = ref.attend(q, c.vals[0], c.vals[1], N, True)
    tol, rel = ref.tolerance(size, np.abs(v).max())
    for ws in (0, 1 << 20, 1 << 16, 1 << 12, 64):
        with z.Context(0, workspace_bytes=ws) as cx, z.KVQCache(cx, 1, 1, N, H, d) as kv:
            kv.append(0, 0, 0, dev(torch, k), dev(torch, v))
            out = torch.empty(n_q, n_head, d, device="cuda")
            kv.attention(0, 0, 1, dev(torch, q), out, n_q=n_q, n_head=n_head, n_kv=N)
            assert np.abs(out.cpu().numpy() - want).max() <= tol, ws
            w = torch.zeros(H, N, device="cuda")
            if ws == 64 and n_q > 1:
                with pytest.raises(z.ZwgError, match="workspace"):
                    kv.attention(0, 0, 1, dev(torch, q), out, n_q=n_q, n_head=n_head, n_kv=N, weights=w)
            elif ws != 64:
                kv.attention(0, 0, 1, dev(torch, q), out, n_q=n_q, n_head=n_head, n_kv=N, weights=w, decay=0.0)
                assert (np.abs(w.cpu().numpy() - wsum) <= (rel + 2.0 ** -17) * wsum + 1e-30).all()


@pytest.mark.parametrize("n_q", [1, 12])
def test_values_that_are_none_stay_where_they_are(torch, z, ctx, n_q):
    """A block that holds NaNs is NaN for the queries that see it, and nothing to those whose keys end before it;
    likewise a query row that is no number, huge and tiny queries and values."""
    H, n_head, d, N = 2, 4, 64, 300
    rng = np.random.default_rng(9)
    k, v = (rng.standard_normal((N, H, d)).astype(np.float32) for _ in range(2))
    k[150, 0, 0] = np.nan
    v[150, 1, 5] = np.inf
    q = rng.standard_normal((n_q, n_head, d)).astype(np.float32)
    with z.KVQCache(ctx, 1, 1, N, H, d, 16) as kv:
        kv.append(0, 0, 0, dev(torch, k), dev(torch, v))
        out = torch.empty(n_q, n_head, d, device="cuda")
        c = ref.Cache(N, H, d, 16, "i8")
        c.append(0, k, v)
        for n in (144, 145, 200, 300) if n_q == 1 else (144, 150, 300):
            w = torch.zeros(H, N, device="cuda")
            kv.attention(0, 0, 1, dev(torch, q), out, n_q=n_q, n_head=n_head, n_kv=n, weights=w, weights_stride=N)
            got = out.cpu().numpy()
            for i in range(n_q):
                lim = n - n_q + i + 1
                want, _, size = ref.attend(q[i: i + 1], c.vals[0], c.vals[1], min(lim, 144), True)
                tol, _ = ref.tolerance(size, np.abs(v[:144]).max())
                if lim <= 144:
                    assert np.abs(got[i] - want[0]).max() <= tol
                else:
                    assert np.isnan(got[i]).all()
        # numbers of any size
        k, v = (rng.standard_normal((N, H, d)).astype(np.float32) for _ in range(2))
        for ks, vs, qs in ((1e30, 1e30, 1e-30), (1e-25, 1e-25, 1e25), (1e-12, 1e35, 1e12), (1.0, 1e-28, 1.0)):
            kk, vv, qq = (k * np.float32(ks)), (v * np.float32(vs)), (q * np.float32(qs))
            kv.append(0, 0, 0, dev(torch, kk), dev(torch, vv))
            c.append(0, kk, vv)
            kv.attention(0, 0, 1, dev(torch, qq), out, n_q=n_q, n_head=n_head, n_kv=N)
            want, _, size = ref.attend(qq, c.vals[0], c.vals[1], N, True)
            tol, _ = ref.tolerance(size, np.abs(vv).max())
            assert np.abs(out.cpu().numpy() - want).max() <= tol, (ks, vs, qs)
        qq = q.copy()
        qq[-1, 1, 7] = np.inf
        kv.attention(0, 0, 1, dev(torch, qq), out, n_q=n_q, n_head=n_head, n_kv=N)
        bad = np.isnan(out.cpu().numpy()).all(-1)
        assert bad[-1, 1] and bad.sum() == 1


def test_value_scales_that_differ(torch, z, ctx):
    """Blocks of values of very unlike sizes, growing and falling along the keys: the running power of two follows."""
    H, n_head, d, N = 1, 2, 128, 640
    rng = np.random.default_rng(10)
    k, v = (rng.standard_normal((N, H, d)).astype(np.float32) for _ in range(2))
    size = 2.0 ** rng.integers(-60, 60, N // 32)
    q = rng.standard_normal((1, n_head, d)).astype(np.float32)
    with z.KVQCache(ctx, 1, 1, N, H, d, 32) as kv:
        for order in (np.arange(20), np.argsort(size), np.argsort(-size)):
            vv = (v.reshape(20, 32, H, d) * size[order][:, None, None, None]).astype(np.float32).reshape(N, H, d)
            kv.append(0, 0, 0, dev(torch, k), dev(torch, vv))
            c = ref.Cache(N, H, d, 32, "i8")
            c.append(0, k, vv)
            out = torch.empty(1, n_head, d, device="cuda")
            for n in (33, 257, N):
                kv.attention(0, 0, 1, dev(torch, q), out, n_q=1, n_head=n_head, n_kv=n)
                want, _, sz = ref.attend(q, c.vals[0], c.vals[1], n, True)
                tol, _ = ref.tolerance(sz, np.abs(vv[:n]).max())
                assert np.abs(out.cpu().numpy() - want).max() <= tol, n


def test_caches_beyond_32_bits(torch, z, ctx):
    """A cache whose codes pass 4 GiB: its last unit is written, read and attended to, and the first is not touched."""
    L, S, N, H, d = 2, 3, 3_000_000, 2, 128  # 4.6 GB each of keys and values
    rng = np.random.default_rng(11)
    with z.KVQCache(ctx, L, S, N, H, d, 64) as kv:
        assert kv.nbytes > 8 << 30  # keys and values 4 GiB each
        c = ref.Cache(300, H, d, 64, "i8")
        k, v = (rng.standard_normal((100, H, d)).astype(np.float32) for _ in range(2))
        at = N - 128 - N % 64  # a block's start near the end
        kv.append(L - 1, S - 1, at + 3, dev(torch, k), dev(torch, v))
        c.append(3, k, v)
        gk, gv = torch.empty(103, H, d, device="cuda"), torch.empty(103, H, d, device="cuda")
        kv.rows(L - 1, 1, S - 1, 1, 103, gk, gv, pos=at)
        assert np.array_equal(gk.cpu().numpy(), c.vals[0][:103]) and np.array_equal(gv.cpu().numpy(), c.vals[1][:103])
        kv.rows(0, 1, 0, 1, 103, gk, gv, pos=at)
        assert not gk.any() and not gv.any()
        # every key but those is zero: scores 0, so zeros weigh e^0 each
        q = np.zeros((1, H, d), np.float32)
        out = torch.empty(1, H, d, device="cuda")
        kv.attention(L - 1, S - 1, 1, dev(torch, q), out, n_q=1, n_head=H, n_kv=at + 103)
        want = c.vals[1][:103].astype(np.float64).sum(0) / (at + 103)
        assert np.abs(out.cpu().numpy()[0] - want).max() < 1e-5 * np.abs(want).max()


# ---------------------------------------------------------------------------------------------- eviction


CUT = [  # L, S, n_ctx, H, d, block, n_kv, keep, first, recent
    (1, 1, 100, 2, 64, 16, 100, 50, 4, 20), (2, 3, 300, 2, 32, 32, 257, 100, 0, 0), (1, 2, 200, 1, 128, 64, 200, 199, 1, 198),
    (1, 1, 3000, 2, 64, 16, 2900, 1001, 4, 256), (1, 1, 2100, 1, 128, 32, 2048, 1500, 0, 700), (1, 1, 64, 3, 64, 16, 20, 1, 0, 0),
    (1, 2, 100, 1, 32, 16, 60, 60, 4, 4), (1, 2, 100, 1, 32, 16, 60, 90, 4, 4), (1, 1, 5000, 1, 32, 64, 5000, 4096, 0, 5),
]


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("case", CUT, ids=lambda c: "-".join(map(str, c)))
def test_eviction(torch, z, ctx, case, fmt):
    """Ragged sequences, ties, zeros, negative and NaN weights; weights in place or apart; the cut cache goes on: rows are
    appended behind it as to any other."""
    L, S, n_ctx, H, d, block, n_kv, keep, first, recent = case
    rng = np.random.default_rng(keep + d)
    lens = [n_kv - int(i * n_kv * 0.3) for i in range(S)]
    with z.KVQCache(ctx, L, S, n_ctx, H, d, block, fmt_of(z, fmt)) as kv:
        want = {}
        for layer in range(L):
            for s in range(S):
                k, v = (rng.standard_normal((lens[s], H, d)).astype(np.float32) * 3 for _ in range(2))
                kv.append(layer, s, 0, dev(torch, k), dev(torch, v))
                want[layer, s] = ref.Cache(n_ctx, H, d, block, fmt)
                want[layer, s].append(0, k, v)
        stride = n_kv + 5
        w = rng.random((L, S, H, stride)).astype(np.float32)
        w[..., ::3] = 0.0
        w[..., 1::5] = 0.25
        if n_kv > 50:
            w[..., 33], w[..., 34], w[..., 35] = -1.0, np.nan, np.inf
            w[..., 36] = -0.0
        n_dev = dev(torch, lens, np.int32)
        kept = torch.full((L, S, H, keep), 77, dtype=torch.int32, device="cuda")
        wd = dev(torch, w)
        in_place = block == 16
        wo = wd if in_place else torch.full((L, S, H, stride), 8.0, device="cuda")
        n_out = n_dev if in_place else torch.zeros(S, dtype=torch.int32, device="cuda")
        kv.evict(0, L, 0, S, n_kv, keep, wd, wo, first, recent, n_dev, n_out, kept, weights_stride=stride)
        gk, gw = kept.cpu().numpy(), wo.cpu().numpy()
        assert n_out.tolist() == [min(n, keep) for n in lens]
        for layer in range(L):
            for s in range(S):
                idx = [ref.choose(w[layer, s, h], lens[s], keep, first, recent) for h in range(H)]
                m = len(idx[0])
                for h in range(H):
                    assert gk[layer, s, h].tolist() == idx[h] + [-1] * (keep - m), (layer, s, h)
                    assert same(gw[layer, s, h, :m], w[layer, s, h][idx[h]]) and (gw[layer, s, h, m:n_kv] == 0).all()
                    assert same(gw[layer, s, h, n_kv:], w[layer, s, h, n_kv:] if in_place else np.full(5, 8.0, np.float32))
                if lens[s] > keep:
                    want[layer, s].evict(idx)
                k, v = (rng.standard_normal((3, H, d)).astype(np.float32) for _ in range(2))
                for step in range(2):
                    for g, c in zip(values(torch, kv, layer, s, n_ctx), want[layer, s].vals):
                        assert same(g, c[:n_ctx]), (layer, s, step)
                    if step == 0 and m + 3 <= n_ctx:
                        kv.append(layer, s, m, dev(torch, k), dev(torch, v))
                        want[layer, s].append(m, k, v)


@pytest.mark.parametrize("d,block,keep", [(32, 16, 4400), (64, 64, 3001), (128, 32, 1300), (128, 16, 2000), (128, 64, 4999)])
def test_eviction_of_many_groups(torch, z, d, block, keep):
    """Groups of one unit that move in parallel into each other's old places, with exactly the workspace they need."""
    H, N = 2, 5000
    rng = np.random.default_rng(keep)
    k, v = (rng.standard_normal((N, H, d)).astype(np.float32) for _ in range(2))
    w = rng.random((1, 1, H, N)).astype(np.float32)
    with z.Context(0, workspace_bytes=4096) as cx, z.KVQCache(cx, 1, 1, N, H, d, block) as kv:
        with pytest.raises(z.ZwgError, match="workspace") as e:
            kv.evict(0, 1, 0, 1, N, keep, dev(torch, w))
    need = int(re.search(r"needs (\d+) bytes", str(e.value)).group(1))
    idx = [ref.choose(w[0, 0, h], N, keep, 3, 100) for h in range(H)]
    c = ref.Cache(N, H, d, block, "i8")
    c.append(0, k, v)
    c.evict(idx)
    with z.Context(0, workspace_bytes=need) as cx, z.KVQCache(cx, 1, 1, N, H, d, block) as kv:
        for _ in range(3):  # its flags and ticket start over in each call
            kv.append(0, 0, 0, dev(torch, k), dev(torch, v))
            kept = torch.empty(1, 1, H, keep, dtype=torch.int32, device="cuda")
            kv.evict(0, 1, 0, 1, N, keep, dev(torch, w), None, 3, 100, kept=kept)
            assert kept[0, 0].tolist() == [list(i) for i in idx]
            for g, x in zip(values(torch, kv, 0, 0, N), c.vals):
                assert np.array_equal(g, x[:N])
    with z.Context(0, workspace_bytes=need - 1) as cx, z.KVQCache(cx, 1, 1, N, H, d, block) as kv:
        with pytest.raises(z.ZwgError, match="workspace"):
            kv.evict(0, 1, 0, 1, N, keep, dev(torch, w))


def test_evictions_of_many_groups_side_by_side(torch, z):
    """Two contexts' evictions on streams of their own, eager and as graphs replayed with eager work between: every
    workgroup that waits for lower groups gets on, and the results are those of one at a time."""
    H, N, d, keep = 3, 6000, 64, 5001
    rng = np.random.default_rng(8)
    k, v = (dev(torch, rng.standard_normal((N, H, d)).astype(np.float32)) for _ in range(2))
    w = dev(torch, rng.random((2, 1, H, N)).astype(np.float32))

    def step(kv):
        for layer in range(2):
            kv.append(layer, 0, 0, k, v)
        kv.evict(0, 2, 0, 1, N, keep, w, None, 4, 500)

    with z.Context(0) as c0, z.Context(0) as c1, z.Context(0) as c2:
        with z.KVQCache(c0, 2, 1, N, H, d, 16) as want, z.KVQCache(c1, 2, 1, N, H, d, 16) as a, z.KVQCache(c2, 2, 1, N, H, d, 16) as b:
            step(want)
            torch.cuda.synchronize()
            expected = [values(torch, want, layer, 0, N) for layer in range(2)]

            def check():
                torch.cuda.synchronize()
                for kv in (a, b):
                    for layer in range(2):
                        for got, x in zip(values(torch, kv, layer, 0, N), expected[layer]):
                            assert np.array_equal(got, x)

            streams = torch.cuda.Stream(), torch.cuda.Stream()
            for s, kv in zip(streams, (a, b)):
                with torch.cuda.stream(s):
                    for _ in range(3):
                        step(kv)
            check()
            graphs = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
            for g, kv in zip(graphs, (a, b)):
                with torch.cuda.graph(g):
                    step(kv)
            for _ in range(3):
                for s, g in zip(streams, graphs):
                    with torch.cuda.stream(s):
                        g.replay()
                check()
                for kv in (a, b):
                    kv.append(1, 0, 100, k[:77].contiguous(), v[:77].contiguous())


def test_eviction_without_extras(torch, z, ctx):
    """No kept list, no new weights, no counts; one count for all; twice (the second cuts nothing); no sequence at all."""
    H, d, N = 2, 64, 90
    rng = np.random.default_rng(12)
    k, v = (rng.standard_normal((N, H, d)).astype(np.float32) for _ in range(2))
    w = rng.random((1, 1, H, N)).astype(np.float32)
    with z.KVQCache(ctx, 1, 1, N, H, d, 32) as kv:
        kv.append(0, 0, 0, dev(torch, k), dev(torch, v))
        c = ref.Cache(N, H, d, 32, "i8")
        c.append(0, k, v)
        kv.evict(0, 1, 0, 0, N, 40, dev(torch, w))
        kv.evict(0, 1, 0, 1, N, N, dev(torch, w))
        for g, x in zip(values(torch, kv, 0, 0, N), c.vals):
            assert np.array_equal(g, x[:N])
        kv.evict(0, 1, 0, 1, N, 40, dev(torch, w))
        c.evict([ref.choose(w[0, 0, h], N, 40, 0, 0) for h in range(H)])
        kv.evict(0, 1, 0, 1, 40, 40, dev(torch, w))
        for g, x in zip(values(torch, kv, 0, 0, N), c.vals):
            assert np.array_equal(g, x[:N])


# ---------------------------------------------------------------------------------------------- together


def test_a_long_generation(torch, z, ctx):
    """The operators as a program uses them: a prompt in batches, then token steps whose weights accumulate, with an
    eviction whenever the budget is passed; rotary positions go on counting while slots are reused.  Against the plain
    restatement step by step, fed with the library's own stored values and choices so that roundings do not add up."""
    S, H, n_head, d, B, budget = 2, 2, 6, 64, 16, 48
    n_ctx = budget + 16
    rng = np.random.default_rng(13)
    w, m = ref.rope_freqs(d, 1e6, "yarn", 4.0, 32)
    turn = lambda x, pos: ref.rotate(x, pos, d, "half", w, m, rounded=True).astype(np.float32)  # noqa: E731
    rope = z.Rope(ctx, 1000, d, scaling=z.ROPE_YARN, factor=4.0, n_orig=32)
    kv = z.KVQCache(ctx, 1, S, n_ctx, H, d, B, z.KVQ_I8, rope)
    acc = torch.zeros(S, H, n_ctx, device="cuda")
    out = torch.empty(S, 20, n_head, d, device="cuda")
    lens, true = [0] * S, [0] * S

    def check(s, q, got, n, causal):
        k, v = values(torch, kv, 0, s, n)
        want, wsum, size = ref.attend(q, k, v, n, causal)
        tol, rel = ref.tolerance(size, np.abs(v).max())
        assert np.abs(got - want).max() <= tol
        return wsum, rel

    for s in range(S):
        for n in (20, 13 + s):
            k, v, q = (rng.standard_normal((n, h, d)).astype(np.float32) for h in (H, H, n_head))
            qd = dev(torch, q)
            kv.append(0, s, lens[s], dev(torch, k), dev(torch, v), q=qd, n_head=n_head, rope_pos=true[s])
            assert np.mean(qd.cpu().numpy() != turn(q, true[s] + np.arange(n))) < 1e-3
            lens[s] += n
            true[s] += n
            kv.attention(0, s, 1, qd, out[s], n_q=n, n_head=n_head, n_kv=lens[s], weights=acc[s], weights_stride=n_ctx)
            check(s, qd.cpu().numpy(), out[s, :n].cpu().numpy(), lens[s], True)
    cuts = 0
    for step in range(55):
        k, v, q = (rng.standard_normal((S, h, d)).astype(np.float32) for h in (H, H, n_head))
        qd = dev(torch, q)
        kv.append_batch(0, 0, dev(torch, lens, np.int32), dev(torch, k), dev(torch, v), q=qd, n_head=n_head,
                        rope_pos_dev=dev(torch, true, np.int32))
        lens, true = [n + 1 for n in lens], [n + 1 for n in true]
        n_dev = dev(torch, lens, np.int32)
        before = acc.cpu().numpy().astype(np.float64)
        kv.attention(0, 0, S, qd, out, n_q=1, n_head=n_head, n_kv=n_ctx, n_kv_dev=n_dev, weights=acc, out_bstride=n_head * d)
        rows = out.view(-1)[: S * n_head * d].view(S, 1, n_head, d).cpu().numpy()
        after = acc.cpu().numpy()
        for s in range(S):
            wsum, rel = check(s, qd[s: s + 1].cpu().numpy(), rows[s], lens[s], True)
            n = lens[s]
            assert (np.abs(after[s, :, :n] - before[s, :, :n] - wsum) <= (rel + 2.0 ** -20) * (wsum + before[s, :, :n])).all()
            assert (after[s, :, n:] == 0).all()
        if max(lens) == n_ctx:
            kept = torch.empty(1, S, H, budget, dtype=torch.int32, device="cuda")
            held = [values(torch, kv, 0, s, n_ctx) for s in range(S)]
            kv.evict(0, 1, 0, S, n_ctx, budget, acc, acc, 2, 16, n_dev, n_dev, kept)
            for s in range(S):
                idx = [ref.choose(after[s, h], lens[s], budget, 2, 16) for h in range(H)]
                assert [list(map(int, r)) for r in kept[0, s].cpu().numpy()] == idx
                for was, now in zip(held[s], values(torch, kv, 0, s, budget)):
                    for h in range(H):
                        rows_ = np.zeros((budget, d), np.float32)
                        rows_[:] = was[idx[h], h]
                        want = np.concatenate([ref.quantise(rows_[b: b + B], "i8") for b in range(0, budget, B)])
                        assert np.array_equal(now[:, h], want)
            lens = n_dev.tolist()
            cuts += 1
    assert cuts >= 2
    kv.close()
    rope.close()


def test_graph_replays(torch, z, ctx):
    """A token step (append, attention with weights) and an eviction captured, replayed with other inputs and eager work
    between: each replay equals the eager calls on a cache of its own."""
    S, H, n_head, d, N = 3, 2, 8, 64, 128
    rng = np.random.default_rng(14)
    rope = z.Rope(ctx, 4 * N, d)
    caches = [z.KVQCache(ctx, 1, S, N, H, d, 16, z.KVQ_E4M3, rope) for _ in range(2)]
    k, v = torch.randn(S, H, d, device="cuda"), torch.randn(S, H, d, device="cuda")
    q = torch.randn(S, n_head, d, device="cuda")
    pos = torch.zeros(S, dtype=torch.int32, device="cuda")
    n_kv = torch.ones(S, dtype=torch.int32, device="cuda")
    qr = [torch.empty_like(q) for _ in range(2)]
    out = [torch.empty_like(q) for _ in range(2)]
    acc = [torch.zeros(S, H, N, device="cuda") for _ in range(2)]
    kept = [torch.zeros(1, S, H, 24, dtype=torch.int32, device="cuda") for _ in range(2)]

    def step(i):
        caches[i].append_batch(0, 0, pos, k, v, q=q, n_head=n_head, q_out=qr[i])
        caches[i].attention(0, 0, S, qr[i], out[i], n_q=1, n_head=n_head, n_kv=N, n_kv_dev=n_kv, weights=acc[i])

    def cut(i):
        caches[i].evict(0, 1, 0, S, N, 24, acc[i], acc[i], 1, 8, n_kv, None, kept[i])

    rows = [dev(torch, rng.standard_normal((40, H, d))) for _ in range(2)]
    for c in caches:
        for s in range(S):
            c.append(0, s, 0, rows[0], rows[1])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(s):
        ctx._bind_torch_stream()
        s.synchronize()
        for f in (step, cut):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                f(0)
            graphs.append(g)
    torch.cuda.synchronize()
    for t in range(6):
        pos.fill_(40 + t - (16 if t >= 3 else 0))
        n_kv.copy_(pos + 1)
        n_kv[1] = t  # a shorter sequence
        for x in (k, v, q):
            x.normal_()
        torch.cuda.synchronize()
        for g, f in zip(graphs[: 2 if t % 3 == 2 else 1], (step, cut)):
            g.replay()
            torch.cuda.synchronize()
            f(1)
            torch.cuda.synchronize()
        assert torch.equal(out[0], out[1]) and torch.equal(acc[0], acc[1]) and torch.equal(kept[0], kept[1]), t
        for i in range(S):
            for a, b in zip(values(torch, caches[0], 0, i, N), values(torch, caches[1], 0, i, N)):
                assert np.array_equal(a, b), t
    for c in caches:
        c.close()
    rope.close()


def test_streams(torch, z, ctx):
    """Calls issued from several streams in turn run in the order of issue (the context orders its streams)."""
    H, d, N = 2, 64, 200
    k, v, q = (torch.randn(N, H, d, device="cuda") for _ in range(3))
    with z.KVQCache(ctx, 1, 1, N, H, d) as kv:
        kv.append(0, 0, 0, k, v)
        want, out = torch.empty(1, H, d, device="cuda"), torch.empty(1, H, d, device="cuda")
        kv.attention(0, 0, 1, q[:1].contiguous(), want, n_q=1, n_head=H, n_kv=N)
        torch.cuda.synchronize()
        a, b = torch.cuda.Stream(), torch.cuda.Stream()
        zero = torch.zeros_like(k)
        torch.cuda.synchronize()
        for _ in range(5):
            with torch.cuda.stream(a):
                kv.append(0, 0, 0, zero, zero)
                kv.append(0, 0, 0, k, v)
            with torch.cuda.stream(b):
                kv.attention(0, 0, 1, q, out, n_q=1, n_head=H, n_kv=N)
            torch.cuda.synchronize()
            assert torch.equal(out, want)


def test_refusals(torch, z, ctx):
    for kw, msg in [(dict(d=48), "head dim"), (dict(block=8), "block"), (dict(block=33), "block"), (dict(n_ctx=0), "positive"),
                    (dict(n_ctx=2 ** 27), "below 2"), (dict(fmt=2), "format"), (dict(n_seq=70000), "out of range"),
                    (dict(rope=z.Rope(ctx, 64, 32)), "head dim")]:
        with pytest.raises(z.ZwgError, match=msg):
            z.KVQCache(ctx, **{"n_layer": 1, "n_seq": 1, "n_ctx": 64, "n_head_kv": 2, "d": 64, **kw})
    x = torch.zeros(4, 2, 64, device="cuda")
    i = torch.zeros(4, dtype=torch.int32, device="cuda")
    with z.KVQCache(ctx, 2, 4, 64, 2, 64, rope=z.Rope(ctx, 16, 64)) as kv:
        bad = [
            (kv.append, (2, 0, 0, x, x), {}, "layer"), (kv.append, (0, 4, 0, x, x), {}, "sequence"),
            (kv.append, (0, 0, 61, x, x), dict(rope_pos=0), "past the end of the cache"), (kv.append, (0, 0, 13, x, x), {}, "past the end of the rope"),
            (kv.append, (0, 0, 0, x, x[:3]), {}, "elements"), (kv.append, (0, 0, 0, x.half(), x), {}, "float32"),
            (kv.append, (0, 0, 0, x.view(-1)[1:129], x), {}, "16-byte"), (kv.append, (0, 0, 0, x.view(-1)[:100], x), {}, "whole rows"),
            (kv.append, (0, 0, 0, x, x), dict(q=x, n_head=3), "elements|multiple"), (kv.append, (0, 0, 0, x, x), dict(q_out=x), "without q"),
            (kv.append, (0, 0, -1, x, x), {}, "whole number"),
            (kv.append_batch, (0, 1, i, x, x), {}, "sequences"), (kv.append_batch, (0, 0, i.long(), x, x), {}, "int32"),
            (kv.append_batch, (0, 0, i, x, x), dict(rope_pos_dev=i[:2]), "elements"),
            (kv.rows, (0, 3, 0, 1, 4, x, x), {}, "layers|elements"), (kv.rows, (0, 1, 0, 1, 5, x, x), {}, "elements"),
            (kv.attention, (0, 0, 1, x, x.clone(), 1, 3, 4), {}, "multiple"), (kv.attention, (0, 0, 1, x, x.clone(), 1, 2, 65), {}, "n_ctx"),
            (kv.attention, (0, 0, 5, x, x.clone(), 1, 2, 4), {}, "sequences|elements"), (kv.attention, (0, 0, 1, x, x.clone(), 5, 2, 4), {}, "elements"),
            (kv.attention, (0, 0, 1, x, x.clone(), 2, 2, 4), dict(q_stride=130), "multiples of 4"),
            (kv.attention, (0, 0, 1, x, x.clone(), 1, 2, 64), dict(weights=x.view(-1)[:100]), "elements"),
            (kv.attention, (0, 0, 1, x, x.clone(), 1, 2, 64), dict(weights=x, decay=-1.0), "decay"),
            (kv.evict, (0, 1, 0, 1, 64, 0, x), {}, "n_keep"), (kv.evict, (0, 1, 0, 1, 64, 10, x, None, 6, 5), {}, "n_first"),
            (kv.evict, (0, 1, 0, 1, 65, 10, x), {}, "n_ctx"), (kv.evict, (0, 1, 0, 1, 64, 10, x), dict(weights_stride=32), "weights_stride|elements"),
            (kv.evict, (0, 1, 0, 4, 64, 10, x.view(-1)[:256]), {}, "elements"), (kv.evict, (1, 2, 0, 1, 32, 10, x), {}, "layers"),
        ]
        for f, args, kw, msg in bad:
            with pytest.raises(z.ZwgError, match=msg):
                f(*args, **kw)
    with pytest.raises(z.ZwgError, match="closed"):
        kv.append(0, 0, 0, x, x)
    with z.KVQCache(ctx, 1, 1, 64, 2, 64) as kv, pytest.raises(z.ZwgError, match="rope"):
        kv.append(0, 0, 0, x, x, q=x, n_head=2)
    with z.Context(0) as other, pytest.raises(z.ZwgError, match="another context"):
        z.KVQCache(other, 1, 1, 64, 2, 64, rope=z.Rope(ctx, 16, 64))


def test_refusals_of_shared_memory_and_missing_tensors(torch, z, ctx):
    x = torch.zeros(4, 2, 64, device="cuda")
    o = torch.zeros_like(x)
    i = torch.zeros(4, dtype=torch.int32, device="cuda")
    with z.KVQCache(ctx, 1, 4, 64, 2, 64) as kv:
        for f, args, kw, msg in [(kv.attention, (0, 0, 4, x, x, 1, 2, 4), {}, "same memory"),
                                 (kv.attention, (0, 0, 1, x, o, 1, 2, 4), dict(weights=o), "same memory"),
                                 (kv.attention, (0, 0, 1, x, o, 1, 2, 4), dict(weights=x), "same memory"),
                                 (kv.append, (0, 0, 0, None, x), {}, "k_rows"), (kv.append, (0, 0, 0, x, None), {}, "null k or v"),
                                 (kv.append, (0, 0, 2 ** 64, x, x), {}, "whole number"), (kv.append_batch, (0, 0, None, x, x), {}, "pos_dev"),
                                 (kv.append_batch, (0, 0, [0, 1, 2, 3], x, x), {}, "pos_dev"), (kv.append_batch, (0, 0, i, x, None), {}, "null k or v"),
                                 (kv.attention, (0, 0, 1, None, o, 1, 2, 4), {}, "null q"),
                                 (kv.evict, (0, 1, 0, 1, 64, 10, None), {}, "null weights"),
                                 (kv.evict, (0, 1, 0, 1, 64, 2 ** 31 - 1, x), {}, "n_keep")]:
            with pytest.raises(z.ZwgError, match=msg):
                f(*args, **kw)


def test_the_context_closes_first(torch, z):
    """Caches and ropes that outlive their context refuse calls; closing them afterwards is safe, in either order."""
    import ctypes

    from zwhisper_amd import _lib

    L = _lib.lib()
    h = ctypes.c_void_p()
    assert L.zwg_open(0, None, ctypes.byref(h)) == 0
    r, kv = ctypes.c_void_p(), ctypes.c_void_p()
    rd = _lib.RopeDescC(64, 64, 64, 0, 0, 1e6, 1.0, 0, 0.0, 0.0, 0.0)
    kd = _lib.KVQDescC(1, 1, 64, 2, 64, 32, 0, 0)
    assert L.zwg_rope_create(h, ctypes.byref(rd), ctypes.byref(r)) == 0
    assert L.zwg_kvq_create(h, ctypes.byref(kd), r, ctypes.byref(kv)) == 0
    L.zwg_close(h)
    x = torch.zeros(128, device="cuda")
    assert L.zwg_kvq_append(kv, 0, 0, 0, 1, 0, x.data_ptr(), x.data_ptr(), None, None, 0, 0) == _lib.ZWG_ERROR
    assert "closed" in _lib.last_error(None)
    assert L.zwg_rope_apply_dev(r, x.data_ptr(), 1, 1, 64, None, 0, x.data_ptr(), 64, 0) == _lib.ZWG_ERROR
    L.zwg_rope_destroy(r)
    L.zwg_kvq_destroy(kv)
