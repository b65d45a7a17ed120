"""Rotary positions (zwg_rope_*) against the rotation in f64 and against its definition rounding by rounding."""
from __future__ import annotations

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


def scaling_of(z, name):
    return {"none": z.ROPE_NONE, "linear": z.ROPE_LINEAR, "ntk": z.ROPE_NTK, "yarn": z.ROPE_YARN}[name]


def layout_of(z, name):
    return {"half": z.ROPE_HALF, "interleaved": z.ROPE_INTERLEAVED}[name]


CASES = [  # n, heads, d, n_rot, layout, scaling, factor
    (1, 14, 128, 128, "half", "none", 1.0), (7, 3, 64, 64, "interleaved", "none", 1.0),
    (33, 2, 64, 32, "half", "linear", 4.0), (5, 16, 128, 96, "interleaved", "yarn", 8.0),
    (129, 1, 32, 24, "half", "ntk", 2.5), (3, 5, 4, 2, "half", "none", 1.0), (3, 5, 4, 2, "interleaved", "linear", 2.0),
    (9, 2, 20, 14, "half", "yarn", 4.0), (9, 2, 20, 14, "interleaved", "ntk", 3.0), (2, 1, 1024, 1024, "half", "yarn", 1.0),
    (1000, 14, 64, 64, "half", "yarn", 4.0),
]


@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_rotation(torch, z, ctx, case, inverse):
    """Every product and sum rounds to f32 by itself: the result is the definition's bit for bit wherever the f32
    tables are (a sine formed by another library may round the other way once in 2^29), and within a product's
    and a sum's rounding of f64: three halves of a step of the larger term, under 2^-22 of the pair's size."""
    n, heads, d, n_rot, layout, scaling, factor = case
    n_ctx = 200000 if n_rot >= 64 else 4096
    rng = np.random.default_rng(n * d + n_rot)
    x = rng.standard_normal((n, heads, d)).astype(np.float32)
    pos = rng.integers(0, n_ctx, n).astype(np.int32)
    pos[-1] = n_ctx - 1
    w, m = ref.rope_freqs(n_rot, 1e6, scaling, factor, n_orig=32768)
    with z.Rope(ctx, n_ctx, d, n_rot, layout_of(z, layout), 1e6, scaling_of(z, scaling), factor, n_orig=32768) as r:
        xd, out = torch.from_numpy(x).cuda(), torch.full((n, heads, d), 7.0, device="cuda")
        r.apply(xd, n, heads, pos=torch.from_numpy(pos).cuda(), out=out, inverse=inverse)
        assert torch.equal(xd.cpu(), torch.from_numpy(x))
        got = out.cpu().numpy()
        want = ref.rotate(x, pos, n_rot, layout, w, m, inverse, rounded=True)
        assert np.mean(got != want) < 1e-3
        exact = ref.rotate(x, pos, n_rot, layout, w, m, inverse)
        assert np.abs(got - exact).max() <= 2.0 ** -22 * m * 2 * np.abs(x).max()
        assert np.array_equal(got[..., n_rot:], x[..., n_rot:])
        # in place, and at consecutive positions
        r.apply(xd, n, heads, pos=torch.from_numpy(pos).cuda(), inverse=inverse)
        assert torch.equal(xd, out)
        xd = torch.from_numpy(x).cuda()
        r.apply(xd, n, heads, pos=n_ctx - n, inverse=inverse)
        want = ref.rotate(x, np.arange(n_ctx - n, n_ctx), n_rot, layout, w, m, inverse)
        assert np.abs(xd.cpu().numpy() - want).max() <= 2.0 ** -22 * m * 2 * np.abs(x).max()


def test_matches_the_f32_cache(torch, z, ctx):
    """The plain half rotation equals the one that KVCache.append applies to q, bit for bit."""
    n, heads, d = 17, 12, 128
    q = torch.randn(n, heads, d, device="cuda")
    k = torch.randn(n, 2 * d, device="cuda")
    with z.KVCache(ctx, 1, 1, 256, 2, d, z.KV_KT, rope_base=1e6) as kv, z.Rope(ctx, 256, d, base=1e6) as r:
        a, b = q.clone(), q.clone()
        kv.append(0, 0, 100, k, k.clone(), a, heads, heads * d)
        r.apply(b, n, heads, pos=100)
        assert torch.equal(a, b)


def test_strides_and_skipped_rows(torch, z, ctx):
    """Rows of an interleaved q/k/v buffer; positions outside the tables leave their rows alone, and columns
    behind the heads are never written."""
    n, heads, d, row = 6, 3, 64, 5 * 64
    x = torch.randn(n, row, device="cuda")
    pos = torch.tensor([0, -1, 5, 64, 63, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    with z.Rope(ctx, 64, d, layout=z.ROPE_INTERLEAVED) as r:
        y = x.clone()
        r.apply(y, n, heads, pos=pos, x_stride=row)
        assert torch.equal(y[:, heads * d:], x[:, heads * d:])
        assert torch.equal(y[[1, 3, 5]], x[[1, 3, 5]])
        out = torch.full((n, row + 8), 3.0, device="cuda")
        r.apply(x, n, heads, pos=pos, out=out, x_stride=row, out_stride=row + 8)
        assert (out[[1, 3, 5]] == 3.0).all() and (out[:, heads * d:] == 3.0).all()
        assert torch.equal(out[[0, 2, 4], : heads * d], y[[0, 2, 4], : heads * d])
        w, m = ref.rope_freqs(d, 1e6)
        want = ref.rotate(x[[0, 2, 4], : heads * d].reshape(3, heads, d).cpu().numpy(), [0, 5, 63], d, "interleaved", w)
        assert np.abs(y[[0, 2, 4], : heads * d].cpu().numpy().reshape(3, heads, d) - want).max() < 2.0 ** -20 * 5
        r.apply(x, 0, heads)  # no rows


@pytest.mark.parametrize("layout,n_rot", [("half", 32), ("interleaved", 20), ("half", 14)])
def test_gradient(torch, z, ctx, layout, n_rot):
    """inverse is the gradient: against the formula (the transposed rotation) and against differences of the forward
    pass, which is linear, so that a central difference has no error but rounding (2^-24 of values about 8, over a step
    of 1: 1e-5 with the sum over a head)."""
    n, heads, d = 5, 2, 32
    rng = np.random.default_rng(3)
    x, g = (rng.standard_normal((n, heads, d)).astype(np.float32) for _ in range(2))
    with z.Rope(ctx, 512, d, n_rot, layout_of(z, layout), 1e4, z.ROPE_YARN, 4.0, n_orig=128) as r:
        def forward(a):
            t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
            r.apply(t, n, heads, pos=300)
            return t.cpu().numpy().astype(np.float64)

        gd = torch.from_numpy(g).cuda()
        r.apply(gd, n, heads, pos=300, inverse=True)
        got = gd.cpu().numpy()
        w, m = ref.rope_freqs(n_rot, 1e4, "yarn", 4.0, 128)
        assert np.abs(got - ref.rotate(g, np.arange(300, 300 + n), n_rot, layout, w, m, inverse=True)).max() < 1e-5
        for j in (0, 1, n_rot // 2, n_rot - 1, d - 1):
            up, down = x.copy(), x.copy()
            up[2, 1, j] += 0.5
            down[2, 1, j] -= 0.5
            step = float(up[2, 1, j]) - float(down[2, 1, j])
            diff = ((forward(up) - forward(down)) * g.astype(np.float64)).sum() / step
            assert abs(diff - got[2, 1, j]) < 1e-5 * 8


def test_graph_and_streams(torch, z, ctx):
    """On a stream of the caller's, captured and replayed with the caller's eager work between the replays."""
    n, heads, d = 40, 14, 128
    x, pos = torch.randn(n, heads, d, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda")
    out, want = torch.empty_like(x), torch.empty_like(x)
    with z.Rope(ctx, 1000, d, scaling=z.ROPE_LINEAR, factor=2.0) as r:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            r.apply(x, n, heads, pos=pos, out=out)
            s.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                r.apply(x, n, heads, pos=pos, out=out)
        torch.cuda.synchronize()
        for k in range(4):
            pos.copy_(torch.randint(0, 1000, (n,), device="cuda", dtype=torch.int32))
            x.normal_()
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            r.apply(x, n, heads, pos=pos, out=want)
            assert torch.equal(out, want), k


def test_refusals(torch, z, ctx):
    x = torch.zeros(4, 2, 64, device="cuda")
    for kw, msg in [(dict(d=62), "multiple of 4"), (dict(n_rot=33), "even"), (dict(n_rot=66), "even"), (dict(n_rot=0), "even"),
                    (dict(base=0.0), "base"), (dict(factor=0.5, scaling=z.ROPE_LINEAR), "factor"), (dict(factor=2.0), "factor 1"),
                    (dict(scaling=z.ROPE_YARN, factor=2.0), "n_orig"), (dict(scaling=7), "scaling"), (dict(layout=2), "layout"),
                    (dict(n_ctx=0), "n_ctx"), (dict(n_ctx=2 ** 31), "n_ctx"), (dict(mscale=-1.0), "mscale"),
                    (dict(scaling=z.ROPE_NTK, n_rot=2, factor=2.0), "NTK")]:
        with pytest.raises(z.ZwgError, match=msg):
            z.Rope(ctx, **{"n_ctx": 16, "d": 64, **kw})
    with z.Rope(ctx, 16, 64) as r:
        for args, kw, msg in [((x, 4, 2), dict(pos=13), "past"), ((x, 5, 2), {}, "elements"), ((x, 4, 2), dict(x_stride=64), "stride"),
                              ((x, 2, 2), dict(x_stride=130), "multiples of 4"), ((x.double(), 4, 2), {}, "float32"),
                              ((x.cpu(), 4, 2), {}, "CUDA"), ((x[:, :, ::2], 1, 1), {}, "contiguous"), ((x, 4, 0), {}, "n_head"),
                              ((x.view(-1)[1:], 1, 2), {}, "16-byte"), ((x, 4, 2), dict(pos=-1), "whole number"),
                              ((x, 4, 2), dict(out=x.view(-1)[64:].view(-1, 64), out_stride=128), "elements|overlap"),
                              ((x, 4, 2), dict(pos=torch.zeros(4, device="cuda")), "int32"),
                              ((x, 4, 2), dict(pos=torch.zeros(3, dtype=torch.int32, device="cuda")), "elements")]:
            with pytest.raises(z.ZwgError, match=msg):
                r.apply(*args, **kw)
        with pytest.raises(z.ZwgError, match="overlap"):
            r.apply(x, 1, 2, out=x.view(-1)[64:])
    with pytest.raises(z.ZwgError, match="closed"):
        r.apply(x, 4, 2)
