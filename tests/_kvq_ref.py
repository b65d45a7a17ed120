"""Plain restatement of the rotary positions and the 8-bit caches -- TEST INFRASTRUCTURE ONLY.

numpy on the CPU, written from the definitions in include/zw_gpu.h: the stored values with every f32 rounding that
the definition makes (formed in f64 and rounded, which for one product, quotient or sum is the f32 operation), the
attention, the weights and the rotation by themselves in f64.
"""
from __future__ import annotations

import math

import numpy as np

F32, F64 = np.float32, np.float64
QMAX = {"i8": 127.0, "e4m3": 448.0}


def rope_freqs(n_rot, base, scaling="none", factor=1.0, n_orig=0, fast=32.0, slow=1.0, mscale=0.0):
    if scaling == "ntk":
        base = base * factor ** (n_rot / (n_rot - 2))
    w = np.array([base ** (-2.0 * j / n_rot) for j in range(n_rot // 2)])
    m = 1.0
    if scaling == "linear":
        w = w / factor
    if scaling == "yarn":
        g = np.clip((n_orig * w / (2 * math.pi) - slow) / (fast - slow), 0.0, 1.0)
        w = g * w + (1 - g) * w / factor
        m = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    return w, mscale or m


def rotate(x, pos, n_rot, layout, w, m=1.0, inverse=False, rounded=False):
    """x [n][heads][d] f32 at positions pos[n], in f64; rounded: each product and sum to f32, as the library does."""
    step = (lambda v: v.astype(F32).astype(F64)) if rounded else (lambda v: v)
    y = x.astype(F64).copy()
    a = np.asarray(pos, F64)[:, None] * w
    c, s = (m * np.cos(a)).astype(F32).astype(F64)[:, None], (m * np.sin(a)).astype(F32).astype(F64)[:, None]
    s = -s if inverse else s
    h = n_rot // 2
    i0, i1 = (slice(0, h), slice(h, n_rot)) if layout == "half" else (slice(0, n_rot, 2), slice(1, n_rot, 2))
    p, q = x[..., i0].astype(F64), x[..., i1].astype(F64)
    y[..., i0] = step(step(p * c) - step(q * s))
    y[..., i1] = step(step(p * s) + step(q * c))
    return y


def quantise(rows, fmt):
    """The values that one block of one head, [block][d] f32, stands for (f32)."""
    rows = np.asarray(rows, F32)
    if not np.isfinite(rows).all():
        return np.full(rows.shape, np.nan, F32)
    amax = F64(np.abs(rows).max())
    if amax < 2.0 ** -100:
        return np.zeros(rows.shape, F32)
    scale, mul = F64(F32(amax / QMAX[fmt])), F64(F32(QMAX[fmt] / amax))
    n = (rows.astype(F64) * mul).astype(F32).astype(F64)
    if fmt == "i8":
        n = np.rint(n)
    else:
        mant, e = np.frexp(np.maximum(np.abs(n), 2.0 ** -6))  # |n| = mant 2^e, mant in [1/2, 1): 4 bits kept
        ulp = np.ldexp(1.0, e - 4)
        n = np.rint(n / ulp) * ulp
    return (n * scale).astype(F32)


class Cache:
    """One (layer, sequence) of a zwg_kvq: values [n_ctx][heads][d] of keys and values."""

    def __init__(self, n_ctx, heads, d, block, fmt):
        self.n_pad = -(-n_ctx // 64) * 64
        self.vals = [np.zeros((self.n_pad, heads, d), F32) for _ in range(2)]
        self.open, self.rows = None, [np.zeros((block, heads, d), F32) for _ in range(2)]
        self.n_ctx, self.heads, self.block, self.fmt = n_ctx, heads, block, fmt

    def append(self, pos, k, v):
        B, n = self.block, len(k)
        first, last = pos // B, (pos + n - 1) // B
        held = self.open
        keep = None
        for b in range(first, last + 1):
            r0, r1 = max(pos, b * B) - b * B, min(pos + n, (b + 1) * B) - b * B
            new = []
            for x, vals, rows in zip((k, v), self.vals, self.rows):
                blk = np.zeros_like(rows)
                if held is not None and held[0] == b:
                    blk[: min(r0, held[1])] = rows[: min(r0, held[1])]
                else:
                    blk[:r0] = vals[b * B: b * B + r0]
                blk[r0:r1] = x[b * B + r0 - pos: b * B + r1 - pos]
                for h in range(self.heads):
                    vals[b * B: (b + 1) * B, h] = quantise(blk[:, h], self.fmt)
                new.append(blk)
            keep = (b, r1, new)
        self.open, self.rows = keep[:2], keep[2]

    def evict(self, kept):
        """kept: per head the positions that stay."""
        B, K = self.block, len(kept[0])
        end = -(-K // B) * B
        for vals in self.vals:
            new = np.zeros((end,) + vals.shape[1:], F32)
            for h, idx in enumerate(kept):
                new[:K, h] = vals[idx, h]
            for b in range(0, end, B):
                for h in range(self.heads):
                    vals[b: b + B, h] = quantise(new[b: b + B, h], self.fmt)
        self.open = None


def choose(w, n, keep, first, recent):
    """The positions of one head that an eviction keeps."""
    if n <= keep:
        return list(range(n))
    mid = list(range(first, n - recent))
    key = lambda j: (0 if math.isnan(w[j]) else 1, 0.0 if math.isnan(w[j]) else -float(w[j]), j)  # noqa: E731
    return sorted([*range(first), *sorted(mid, key=key)[: keep - first - recent], *range(n - recent, n)])


def attend(q, k, v, n_kv, causal):
    """q [n_q][n_head][d], k, v [>= n_kv][heads][d]: (out [n_q][n_head][d], weights [heads][n_kv], the scores' scale), f64."""
    n_q, H, d = q.shape
    G = H // k.shape[1]
    out, w = np.zeros((n_q, H, d)), np.zeros((k.shape[1], n_kv))
    size = 0.0
    for h in range(H):
        kk, vv = k[:n_kv, h // G].astype(F64), v[:n_kv, h // G].astype(F64)
        x = q[:, h].astype(F64) @ kk.T / math.sqrt(d)
        if n_kv:
            size = max(size, float((np.abs(q[:, h].astype(F64)) @ np.abs(kk).T).max()) / math.sqrt(d))
        for i in range(n_q):
            lim = min(n_kv, max(0, n_kv - n_q + i + 1)) if causal else n_kv
            if lim == 0:
                continue
            p = np.exp(x[i, :lim] - x[i, :lim].max())
            p /= p.sum()
            out[i, h] = p @ vv[:lim]
            w[h // G, :lim] += p
    return out, w, size


def tolerance(size, vmax):
    """Absolute bounds on an output and on a probability's relative error.

    A score is a sum of products whose second factors carry 22 significant bits (half a step: 2^-23), times factors
    rounded to f32 (four of them, 2^-24 each), summed in f32: d / 32 partial sums and the unit's own additions, taken as 16
    roundings of 2^-24 relative to the sum of magnitudes, `size`.  So |error| <= size (2^-23 + 20 2^-24) < size 2^-19.4;
    the bound uses 2^-19.  A probability's relative error is twice that (its own and the largest's share in the sum) and
    2^-21 for the exponential and the rounding of the product with the value scale; outputs are means of values below vmax
    under those probabilities, with the 22-bit split and the f32 sums adding 2^-20."""
    rel = 2 * size * 2.0 ** -19 + 2.0 ** -21
    return vmax * (2 * rel + 2.0 ** -20), rel
