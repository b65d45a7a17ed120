"""Operators of a token step over long contexts, as measurable cases: rotary positions, appends to a key/value
cache held in 8 bits, attention over that cache, and eviction from it by accumulated attention weight.

Sizes are those of the framework's tests and benchmark (Qwen2.5-0.5B and 1.5B, Whisper tiny.en and small.en
decoders) and sizes between and around them.

Kinds of case:
  rope    Rope.apply: rotary positions on rows of heads, out of place
  append  KVQCache.append / append_batch: rows rotated, quantised per block of tokens and head, and the
          touched blocks read back as the values they stand for (KVQCache.rows)
  attend  KVQCache.attention: queries of one or many tokens over the cache, with or without the keys'
          accumulated weights
  evict   KVQCache.evict: the first, the last and the heaviest tokens of every head kept, in order

The cache's arithmetic is part of its definition, so both forms give the same stored values: a rotated key is
rounded to f32 after each product and sum, a block's scale is f32(amax / Q), and a code is
round(f32(x * f32(Q / amax))), ties to even, with Q = 127 (int8) or 448 (e4m3).
"""
import math

import torch

own = False

DEVICE = "cuda:0"
QMAX = {"i8": 127.0, "e4m3": 448.0}
ROPE_BASE = 1e6
TRAINED = 32768  # positions the unscaled rotary frequencies are meant for


def listed():
    return [
        # One token of one sequence: the query and key heads of a Qwen2.5-1.5B layer. Latency is all there is to it.
        {"name": "rope_token_1", "kind": "rope", "n": 1, "heads": 14, "d": 128, "n_rot": 128, "layout": "half",
         "scaling": "none", "factor": 1.0, "ctx": 4096, "inverse": False},
        # A long document's rows at positions far past the trained ones.
        {"name": "rope_prompt_8192", "kind": "rope", "n": 8192, "heads": 14, "d": 128, "n_rot": 128, "layout": "half",
         "scaling": "yarn", "factor": 4.0, "ctx": 131072, "inverse": False},
        # Half of each head rotated in neighbouring pairs, rotated back as a gradient or a re-positioned key is.
        {"name": "rope_partial_777", "kind": "rope", "n": 777, "heads": 16, "d": 64, "n_rot": 32,
         "layout": "interleaved", "scaling": "linear", "factor": 2.0, "ctx": 8192, "inverse": True},
        # A chat server's token step: one new token in each of 64 sequences of a Qwen2.5-1.5B layer.
        {"name": "append_token_64", "kind": "append", "mode": "tokens", "seqs": 64, "n": 1, "pos": 0, "ctx": 4096,
         "heads": 12, "kv_heads": 2, "d": 128, "block": 32, "format": "i8", "rope": True},
        # A prompt batch that continues a sequence inside a block (Qwen2.5-0.5B heads).
        {"name": "append_prompt_2048", "kind": "append", "mode": "rows", "seqs": 1, "n": 2048, "pos": 777, "ctx": 4096,
         "heads": 14, "kv_heads": 2, "d": 64, "block": 64, "format": "e4m3", "rope": True},
        # The smallest attention: one token in the middle of one window of a tiny.en-sized decoder.
        {"name": "attend_token_1", "kind": "attend", "seqs": 1, "n_q": 1, "n_kv": 187, "ragged": False, "heads": 6,
         "kv_heads": 6, "d": 64, "block": 16, "format": "i8", "causal": True, "weights": False},
        # The chat server's step: 64 sequences of unlike lengths, one of them idle. Bound by reading the cache.
        {"name": "attend_token_64", "kind": "attend", "seqs": 64, "n_q": 1, "n_kv": 4096, "ragged": True, "heads": 12,
         "kv_heads": 2, "d": 128, "block": 32, "format": "i8", "causal": True, "weights": False},
        # One very long sequence: the keys have to be split over the whole card.
        {"name": "attend_long_1", "kind": "attend", "seqs": 1, "n_q": 1, "n_kv": 131001, "ragged": False, "heads": 12,
         "kv_heads": 2, "d": 128, "block": 64, "format": "e4m3", "causal": True, "weights": False},
        # A batch of a long prompt over the cache so far: bound by the products.
        {"name": "attend_prompt_1024", "kind": "attend", "seqs": 1, "n_q": 1024, "n_kv": 8000, "ragged": False,
         "heads": 12, "kv_heads": 2, "d": 128, "block": 32, "format": "i8", "causal": True, "weights": False},
        # A step that also keeps each key's accumulated weight, for the eviction below.
        {"name": "attend_weights_32", "kind": "attend", "seqs": 32, "n_q": 1, "n_kv": 4096, "ragged": True, "heads": 14,
         "kv_heads": 2, "d": 64, "block": 32, "format": "i8", "causal": True, "weights": True},
        # One sequence over its budget in all 28 layers of Qwen2.5-1.5B.
        {"name": "evict_layers_28", "kind": "evict", "layers": 28, "seqs": 1, "n_kv": 2304, "keep": 2048, "first": 4,
         "recent": 512, "kv_heads": 2, "d": 128, "block": 32, "format": "i8"},
        # A batch cut to a quarter in one layer, sequences of unlike lengths (Qwen2.5-0.5B heads).
        {"name": "evict_batch_16", "kind": "evict", "layers": 1, "seqs": 16, "n_kv": 4096, "keep": 1001, "first": 4,
         "recent": 256, "kv_heads": 2, "d": 64, "block": 16, "format": "e4m3"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rope", "append", "attend", "attend", "evict"])
    d = rng.choice([32, 64, 128])
    kv_heads, group = rng.choice([(2, 6), (2, 7), (6, 1), (12, 1), (4, 8), (1, 3), (2, 12)])
    block, fmt = rng.choice([16, 32, 64]), rng.choice(["i8", "e4m3"])
    if kind == "rope":
        scaling = rng.choice(["none", "linear", "ntk", "yarn"])
        n = _log(rng, 1, 8000)
        return {"kind": "rope", "n": n, "heads": min(16, kv_heads * (group + 1)), "d": d,
                "n_rot": rng.choice([d, d // 2, d - 8]), "layout": rng.choice(["half", "interleaved"]), "scaling": scaling,
                "factor": 1.0 if scaling == "none" else rng.choice([2.0, 3.5, 8.0]),
                "ctx": max(n, rng.choice([2001, 8192, 100000])), "inverse": rng.random() < 0.3}
    if kind == "append":
        tokens = rng.random() < 0.5
        n, pos = (1, 0) if tokens else (_log(rng, 1, 2000), _log(rng, 1, 2000) - 1)
        return {"kind": "append", "mode": "tokens" if tokens else "rows", "seqs": _log(rng, 1, 64) if tokens else 1, "n": n,
                "pos": pos, "ctx": rng.choice([4096, 4444]), "heads": kv_heads * group, "kv_heads": kv_heads, "d": d,
                "block": block, "format": fmt, "rope": rng.random() < 0.7}
    if kind == "attend":
        n_q = 1 if rng.random() < 0.5 else _log(rng, 2, 700)
        seqs = _log(rng, 1, 64) if n_q == 1 else _log(rng, 1, 4) if n_q < 100 else 1
        n_kv = _log(rng, n_q + 1, 60000 if seqs == 1 and n_q < 16 else 4096)
        return {"kind": "attend", "seqs": seqs, "n_q": n_q, "n_kv": n_kv, "ragged": seqs > 1, "heads": kv_heads * group,
                "kv_heads": kv_heads, "d": d, "block": block, "format": fmt, "causal": n_q == 1 or rng.random() < 0.7,
                "weights": rng.random() < 0.3}
    layers, seqs = (rng.randint(2, 28), 1) if rng.random() < 0.5 else (1, _log(rng, 1, 16))
    n_kv = _log(rng, 100, 4096 if layers == 1 else 2304)
    keep = rng.randint(n_kv // 4, n_kv - 1)
    return {"kind": "evict", "layers": layers, "seqs": seqs, "n_kv": n_kv, "keep": keep, "first": min(4, keep // 4),
            "recent": keep // rng.randint(2, 8), "kv_heads": min(kv_heads, 4), "d": d, "block": block, "format": fmt}


# ---------------------------------------------------------------------------------------------- inputs


def _rows(g, *shape):
    """Rows of heads as projections give them: channels of unlike spread, a few of them much wider."""
    spread = torch.exp(0.5 * torch.randn(shape[-1], device=DEVICE, generator=g))
    return torch.randn(*shape, device=DEVICE, generator=g) * spread


def _inputs(case, seed):
    """What both forms and the exact one start from."""
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    c, t = case, {}
    if c["kind"] == "rope":
        t["x"] = _rows(g, c["n"], c["heads"], c["d"])
        if c["n"] == 1:
            t["pos"] = torch.randint(0, c["ctx"], (1,), device=DEVICE, generator=g, dtype=torch.int32)
        else:  # consecutive positions that end at the longest
            t["pos"] = torch.arange(c["ctx"] - c["n"], c["ctx"], device=DEVICE, dtype=torch.int32)
    elif c["kind"] == "append":
        S, n, H, d, B = c["seqs"], c["n"], c["kv_heads"], c["d"], c["block"]
        if c["mode"] == "tokens":
            t["pos"] = torch.randint(0, c["ctx"], (S,), device=DEVICE, generator=g, dtype=torch.int32)
        else:
            t["pos"] = torch.full((1,), c["pos"], device=DEVICE, dtype=torch.int32)
        t["start"] = t["pos"] // B * B  # where the first touched block begins
        t["old_k"], t["old_v"] = _rows(g, S, B, H, d), _rows(g, S, B, H, d)  # its rows before pos are in the cache
        t["k"], t["v"] = _rows(g, S, n, H, d), _rows(g, S, n, H, d)
        t["q"] = _rows(g, S, n, c["heads"], d)
    elif c["kind"] == "attend":
        S, N, H, d = c["seqs"], c["n_kv"], c["kv_heads"], c["d"]
        t["k"], t["v"] = _rows(g, S, N, H, d), _rows(g, S, N, H, d)
        t["q"] = torch.randn(S, c["n_q"], c["heads"], d, device=DEVICE, generator=g)
        t["n_kv"] = torch.full((S,), N, device=DEVICE, dtype=torch.int32)
        if c["ragged"]:
            t["n_kv"] = torch.randint(c["n_q"], N + 1, (S,), device=DEVICE, generator=g, dtype=torch.int32)
            if S > 4:
                t["n_kv"][S // 2] = 0 if c["n_q"] == 1 else c["n_q"]  # an idle place in the batch
        if c["weights"]:
            t["w"] = torch.rand(S, H, N, device=DEVICE, generator=g)
    else:
        L, S, N, H, d = c["layers"], c["seqs"], c["n_kv"], c["kv_heads"], c["d"]
        t["k"], t["v"] = _rows(g, L, S, N, H, d), _rows(g, L, S, N, H, d)
        # attention weights: most keys are hardly looked at; sums that no step has reached yet tie at zero
        w = torch.rand(L, S, H, N, device=DEVICE, generator=g).pow(8)
        t["w"] = torch.where(w < 1e-6, torch.zeros_like(w), w)
        t["n_kv"] = torch.full((S,), N, device=DEVICE, dtype=torch.int32)
        if S > 1:
            t["n_kv"] = torch.randint(max(1, N // 2), N + 1, (S,), device=DEVICE, generator=g, dtype=torch.int32)
    return t


def _freqs(n_rot, scaling, factor):
    """Rotary frequencies per pair, in 64 bits, and the factor on cos and sin."""
    j = torch.arange(n_rot // 2, device=DEVICE, dtype=torch.float64)
    base = ROPE_BASE * factor ** (n_rot / (n_rot - 2)) if scaling == "ntk" else ROPE_BASE
    w = 1.0 / torch.pow(torch.tensor(base, device=DEVICE, dtype=torch.float64), 2 * j / n_rot)
    if scaling == "linear":
        return w / factor, 1.0
    if scaling == "yarn":  # frequencies of under 1 turn over the trained length slow down, over 32 turns stay
        keep = ((TRAINED * w / (2 * math.pi) - 1) / (32 - 1)).clamp(0, 1)
        return keep * w + (1 - keep) * (w / factor), 0.1 * math.log(factor) + 1
    return w, 1.0


def _tables(ctx, n_rot, scaling, factor):
    w, m = _freqs(n_rot, scaling, factor)
    a = torch.arange(ctx, device=DEVICE, dtype=torch.float64)[:, None] * w
    return (m * torch.cos(a)).float(), (m * torch.sin(a)).float()


# ---------------------------------------------------------------------------------------------- plain forms


def _rotate(x, cos, sin, n_rot, layout, inverse=False):
    """x [..., heads, d] with cos, sin [..., n_rot / 2] broadcast over the heads."""
    cos, sin = cos.unsqueeze(-2), (-sin if inverse else sin).unsqueeze(-2)
    r = x[..., :n_rot]
    a, b = (r[..., : n_rot // 2], r[..., n_rot // 2:]) if layout == "half" else (r[..., 0::2], r[..., 1::2])
    ya, yb = a * cos - b * sin, a * sin + b * cos
    y = torch.cat([ya, yb], -1) if layout == "half" else torch.stack([ya, yb], -1).flatten(-2)
    return torch.cat([y, x[..., n_rot:]], -1)


def _quantise(x, block, fmt):
    """x [..., tokens (whole blocks), heads, d] -> codes of the same shape, scales [..., blocks, heads]."""
    b = x.unflatten(-3, (-1, block))
    amax = b.abs().amax((-3, -1))
    ok = amax >= 2.0 ** -100
    top = torch.full_like(amax, QMAX[fmt])  # a tensor: a quotient with a number would be a product with its reciprocal
    inv = torch.where(ok, top / amax, 0.0)
    scaled = b * inv[..., None, :, None]
    codes = scaled.round().clamp(-127, 127).to(torch.int8) if fmt == "i8" else scaled.to(torch.float8_e4m3fn)
    return codes.flatten(-4, -3), torch.where(ok, amax / top, 0.0)


def _values(codes, scales, block):
    return codes.float() * scales.repeat_interleave(block, -2)[..., : codes.shape[-3], :, None]


def _whole(x, block):
    """x [..., tokens, heads, d] with zero rows up to whole blocks."""
    return torch.nn.functional.pad(x, (0, 0, 0, 0, 0, -x.shape[-3] % block))


def _plain_rope(s):
    c, at = s["case"], s["pos"].long()
    return _rotate(s["x"], s["cos"][at], s["sin"][at], c["n_rot"], c["layout"], c["inverse"])


def _plain_append(s):
    c, B = s["case"], s["case"]["block"]
    S, n = c["seqs"], c["n"]
    at = s["pos"].long()[:, None] + torch.arange(n, device=DEVICE)
    k, q = s["k"], s["q"]
    if c["rope"]:
        k = _rotate(k, s["cos"][at], s["sin"][at], c["d"], "half")
        q = _rotate(q, s["cos"][at], s["sin"][at], c["d"], "half")
    place = at - s["start"].long()[:, None]
    held = torch.arange(B, device=DEVICE) < (s["pos"] - s["start"])[:, None]
    out = []
    for new, old in ((k, s["open_k"]), (s["v"], s["open_v"])):
        rows = torch.zeros(S, s["touched"], *new.shape[2:], device=DEVICE)
        rows[:, :B] = torch.where(held[..., None, None], old, 0.0)
        rows[torch.arange(S, device=DEVICE)[:, None], place] = new
        out.append(_values(*_quantise(rows, B, c["format"]), B).flatten(-2))
    return {"k": out[0], "v": out[1], "q": q}


def _plain_attend(s):
    c = s["case"]
    S, n_q, N, H, d = c["seqs"], c["n_q"], c["n_kv"], c["kv_heads"], c["d"]
    G = c["heads"] // H
    k = _values(s["kc"], s["ks"], c["block"]).permute(0, 2, 3, 1).contiguous()  # [S][H][d][N]
    v = _values(s["vc"], s["vs"], c["block"]).permute(0, 2, 1, 3).contiguous()
    q = s["q"].view(S, n_q, H, G, d).permute(0, 2, 1, 3, 4).reshape(S, H, n_q * G, d)
    x = torch.matmul(q, k) * (1.0 / math.sqrt(d))
    last = s["n_kv"].long()[:, None] + (torch.arange(n_q, device=DEVICE) - n_q + 1 if c["causal"] else
                                        torch.zeros(n_q, device=DEVICE, dtype=torch.long))
    seen = torch.arange(N, device=DEVICE) < last.repeat_interleave(G, 1)[:, None, :, None]
    x = x.masked_fill(~seen, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top > -math.inf, top, 0.0))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    out = torch.matmul(p, v).view(S, H, n_q, G, d).permute(0, 2, 1, 3, 4).reshape(S, n_q, c["heads"], d)
    if not c["weights"]:
        return {"out": out}
    s["w"] += p.sum(2)
    return {"out": out, "w": s["w"]}


def _plain_evict(s):
    c, B, K = s["case"], s["case"]["block"], s["case"]["keep"]
    L, S, N, H = c["layers"], c["seqs"], c["n_kv"], c["kv_heads"]
    n = s["n_kv"].long()[:, None, None]
    at = torch.arange(N, device=DEVICE)
    rank = torch.where((at < c["first"]) | (at >= n - c["recent"]), math.inf, s["w"])
    rank = torch.where(at < n, rank, -1.0)  # weights are never negative
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :K]
    kept = torch.sort(torch.where(order < n, order, N), -1).values
    some = kept < N
    src = torch.where(some, kept, 0)
    w = torch.zeros_like(s["w"])
    w[..., :K] = torch.where(some, s["w"].gather(-1, src), 0.0)
    out, cut = {}, (n > K)[..., None]  # only longer sequences are rewritten
    rows = src.permute(0, 1, 3, 2)[..., None]
    for t, codes, scales in (("k", "kc", "ks"), ("v", "vc", "vs")):
        held = _values(s[codes], s[scales], B)
        got = held.gather(2, rows.expand(*rows.shape[:-1], c["d"]))
        qc, qs = _quantise(_whole(got, B), B, c["format"])
        nb = qs.shape[-2]
        s[scales][:, :, :nb] = torch.where(cut[..., 0], qs, s[scales][:, :, :nb])
        m = min(nb * B, s[codes].shape[2])
        old = s[codes][:, :, :m]
        s[codes][:, :, :m] = torch.where(cut, qc[:, :, :m].float(), old.float()).to(old.dtype)
        out[t] = _values(s[codes][:, :, :K], s[scales], B).flatten(-2)
    return {"kept": torch.where(some, kept, -1).int(), "w": w, "n_kv": s["n_kv"].clamp(max=K), **out}


# ---------------------------------------------------------------------------------------------- the framework's


_context = None


def _ctx():
    global _context
    import zwhisper_amd as z

    if _context is None:
        _context = z.Context(0)
    return z, _context


def _handles(case, s):
    """The rotary tables and the filled cache that a program keeps."""
    z, ctx = _ctx()
    c = case
    scaling = {"none": z.ROPE_NONE, "linear": z.ROPE_LINEAR, "ntk": z.ROPE_NTK, "yarn": z.ROPE_YARN}
    if c["kind"] == "rope":
        s["rope"] = z.Rope(ctx, c["ctx"], c["d"], n_rot=c["n_rot"], base=ROPE_BASE, scaling=scaling[c["scaling"]],
                           layout=z.ROPE_INTERLEAVED if c["layout"] == "interleaved" else z.ROPE_HALF,
                           factor=c["factor"], n_orig=TRAINED)
        s["out"] = torch.empty_like(s["x"])
        return
    fmt = {"i8": z.KVQ_I8, "e4m3": z.KVQ_E4M3}[c["format"]]
    kvw = c["kv_heads"] * c["d"]
    if c["kind"] == "append":
        s["rope"] = z.Rope(ctx, c["ctx"], c["d"], base=ROPE_BASE) if c["rope"] else None
        s["kv"] = z.KVQCache(ctx, 1, c["seqs"], c["ctx"], c["kv_heads"], c["d"], block=c["block"], fmt=fmt, rope=s["rope"])
        for i, (a, b) in enumerate(zip(s["start"].tolist(), s["pos"].tolist())):
            if b > a:  # the open block's earlier rows
                s["kv"].append(0, i, a, s["old_k"][i, : b - a].contiguous(), s["old_v"][i, : b - a].contiguous())
        s["k_out"] = torch.zeros(c["seqs"], s["touched"], kvw, device=DEVICE)
        s["v_out"], s["q_out"] = torch.zeros_like(s["k_out"]), torch.empty_like(s["q"])
        return
    layers, rows = (c["layers"], s["k"]) if c["kind"] == "evict" else (1, s["k"][None])
    vals = s["v"] if c["kind"] == "evict" else s["v"][None]
    s["kv"] = z.KVQCache(ctx, layers, c["seqs"], c["n_kv"], c["kv_heads"], c["d"], block=c["block"], fmt=fmt)
    for layer in range(layers):
        for i in range(c["seqs"]):
            s["kv"].append(layer, i, 0, rows[layer, i], vals[layer, i])
    if c["kind"] == "attend":
        s["out"] = torch.empty_like(s["q"])
    else:
        s["k_out"] = torch.zeros(layers, c["seqs"], c["keep"], kvw, device=DEVICE)
        s["v_out"], s["w_out"] = torch.zeros_like(s["k_out"]), torch.zeros_like(s["w"])
        s["kept"] = torch.empty(layers, c["seqs"], c["kv_heads"], c["keep"], device=DEVICE, dtype=torch.int32)
        s["n_out"] = torch.empty_like(s["n_kv"])


def _own(s):
    c = s["case"]
    if c["kind"] == "rope":
        s["rope"].apply(s["x"], c["n"], c["heads"], pos=s["pos"], out=s["out"], inverse=c["inverse"])
        return s["out"]
    kv = s["kv"]
    if c["kind"] == "append":
        q = {"q": s["q"], "n_head": c["heads"], "q_out": s["q_out"]} if c["rope"] else {}
        if c["mode"] == "tokens":
            kv.append_batch(0, 0, s["pos"], s["k"], s["v"], **q)
        else:
            kv.append(0, 0, c["pos"], s["k"], s["v"], **q)
        kv.rows(0, 1, 0, c["seqs"], s["touched"], s["k_out"], s["v_out"], pos=s["start"])
        return {"k": s["k_out"], "v": s["v_out"], "q": s["q_out"] if c["rope"] else s["q"]}
    if c["kind"] == "attend":
        kv.attention(0, 0, c["seqs"], s["q"], s["out"], n_q=c["n_q"], n_head=c["heads"], n_kv=c["n_kv"],
                     causal=c["causal"], n_kv_dev=s["n_kv"] if c["ragged"] else None, weights=s.get("w"))
        return {"out": s["out"], "w": s["w"]} if c["weights"] else {"out": s["out"]}
    kv.evict(0, c["layers"], 0, c["seqs"], c["n_kv"], c["keep"], s["w"], s["w_out"], n_first=c["first"],
             n_recent=c["recent"], n_kv_dev=s["n_kv"], n_kv_out=s["n_out"], kept=s["kept"])
    kv.rows(0, c["layers"], 0, c["seqs"], c["keep"], s["k_out"], s["v_out"])
    return {"kept": s["kept"], "w": s["w_out"], "n_kv": s["n_out"], "k": s["k_out"], "v": s["v_out"]}


# ---------------------------------------------------------------------------------------------- the interface


def prepare(case, seed):
    s = {"case": case, **_inputs(case, seed)}
    c = case
    if c["kind"] == "append":
        B = c["block"]
        n = c["n"] + (c["pos"] % B if c["mode"] == "rows" else 0)
        s["touched"] = -(-n // B) * B  # rows of the touched blocks
    if own:
        _handles(c, s)
        return s
    if c["kind"] == "rope":
        s["cos"], s["sin"] = _tables(c["ctx"], c["n_rot"], c["scaling"], c["factor"])
    elif c["kind"] == "append":
        s["open_k"], s["open_v"] = s.pop("old_k"), s.pop("old_v")
        if c["rope"]:
            s["cos"], s["sin"] = _tables(c["ctx"] + c["block"], c["d"], "none", 1.0)
            at = s["start"].long()[:, None] + torch.arange(c["block"], device=DEVICE)
            s["open_k"] = _rotate(s["open_k"], s["cos"][at], s["sin"][at], c["d"], "half")
    else:
        for t in ("k", "v"):
            codes, s[t + "s"] = _quantise(_whole(s.pop(t), c["block"]), c["block"], c["format"])
            s[t + "c"] = codes[..., : c["n_kv"], :, :].contiguous()
    return s


def run(s):
    if own:
        return _own(s)
    return {"rope": _plain_rope, "append": _plain_append, "attend": _plain_attend, "evict": _plain_evict}[s["case"]["kind"]](s)


def work(case):
    c = case
    if c["kind"] == "rope":
        return {"bytes": c["n"] * (c["heads"] * c["d"] * 8 + c["n_rot"] * 4), "flops": c["n"] * c["heads"] * c["n_rot"] * 3}
    if c["kind"] == "append":
        rows, kvw = c["seqs"] * c["n"], c["kv_heads"] * c["d"]
        touched = rows if c["mode"] == "rows" else c["seqs"] * c["block"]
        q = 8 * c["heads"] * c["d"] if c["rope"] else 0
        return {"bytes": rows * (2 * kvw * 4 + 2 * kvw + q) + touched * 2 * kvw * 5, "flops": rows * kvw * 8}
    if c["kind"] == "attend":
        n = c["seqs"] * (c["n_q"] + c["n_kv"]) / 2 if c["ragged"] else c["seqs"] * c["n_kv"]
        pairs = c["n_q"] * n - (c["seqs"] * c["n_q"] * (c["n_q"] - 1) / 2 if c["causal"] else 0)
        b = n * c["kv_heads"] * (2 * c["d"] + 8 / c["block"] + (8 if c["weights"] else 0))
        return {"bytes": b + 8 * c["seqs"] * c["n_q"] * c["heads"] * c["d"], "flops": 4 * c["d"] * c["heads"] * pairs}
    units = c["layers"] * c["seqs"] * c["kv_heads"]
    n = c["n_kv"] if c["seqs"] == 1 else 0.75 * c["n_kv"]
    kept = min(n, c["keep"])
    return {"bytes": units * (n * 4 + c["n_kv"] * 4 + kept * (4 + 2 * c["d"] * (1 + 1 + 1 + 4))), "flops": units * kept * c["d"] * 6}


# ---------------------------------------------------------------------------------------------- in 64 bits


def _f32(x):
    """A 64-bit result rounded to the f32 that the definition stores, back in 64 bits."""
    return x.to(torch.float32).to(torch.float64)


def _angles64(pos, n_rot, scaling, factor):
    lists = []
    for j in range(n_rot // 2):
        base = ROPE_BASE * factor ** (n_rot / (n_rot - 2)) if scaling == "ntk" else ROPE_BASE
        w = base ** (-2.0 * j / n_rot)
        if scaling == "linear":
            w /= factor
        elif scaling == "yarn":
            turns = TRAINED * w / (2 * math.pi)
            stay = min(1.0, max(0.0, (turns - 1.0) / 31.0))
            w = w * stay + w / factor * (1.0 - stay)
        lists.append(w)
    m = 0.1 * math.log(factor) + 1.0 if scaling == "yarn" else 1.0
    a = pos.double().cpu().unsqueeze(-1) * torch.tensor(lists, dtype=torch.float64)
    return _f32(m * torch.cos(a)).to(DEVICE), _f32(m * torch.sin(a)).to(DEVICE)


def _turned64(x, pos, n_rot, layout, scaling, factor, inverse, step=lambda v: v):
    """Pair by pair; `step` rounds each product and sum where the definition does."""
    cos, sin = _angles64(pos, n_rot, scaling, factor)
    y = x.double().clone()
    for j in range(n_rot // 2):
        i0, i1 = (j, j + n_rot // 2) if layout == "half" else (2 * j, 2 * j + 1)
        a, b = x[..., i0].double(), x[..., i1].double()
        co, si = cos[..., j, None], sin[..., j, None]
        si = -si if inverse else si
        y[..., i0] = step(step(a * co) - step(b * si))
        y[..., i1] = step(step(a * si) + step(b * co))
    return y


def _stored64(x, block, fmt):
    """What a cache holding x [tokens, heads, d] gives back, in 64 bits (each rounding of the definition made)."""
    T, H, d = x.shape
    full = torch.zeros(-(-T // block) * block, H, d, dtype=torch.float64, device=x.device)
    full[:T] = x
    b = full.reshape(-1, block, H, d).transpose(1, 2)  # [blocks][heads][block][d]
    amax = b.abs().reshape(b.shape[0], H, -1).max(-1).values[..., None, None]
    ok = amax >= 2.0 ** -100
    safe = torch.where(ok, amax, torch.ones_like(amax))
    scale, inv = _f32(safe / QMAX[fmt]), _f32(QMAX[fmt] / safe)
    n = _f32(b * inv)
    if fmt == "i8":
        n = torch.round(n).clamp(-127, 127)
    else:  # 3 bits after the leading one, steps no finer than 2^-9
        power = n.abs().clamp(min=2.0 ** -6).view(torch.int64) >> 52 << 52  # the power of two at or below
        ulp = power.view(torch.float64) / 8
        n = (torch.round(n / ulp) * ulp).clamp(-448, 448)
    got = torch.where(ok, _f32(n * scale), torch.zeros_like(n))
    return got.transpose(1, 2).reshape(-1, H, d)[:T]


def exact(case, seed):
    c, t = case, _inputs(case, seed)
    if c["kind"] == "rope":
        return _turned64(t["x"], t["pos"], c["n_rot"], c["layout"], c["scaling"], c["factor"], c["inverse"])
    if c["kind"] == "append":
        B, ks, vs = c["block"], [], []
        n = c["n"] + (c["pos"] % B if c["mode"] == "rows" else 0)
        touched = -(-n // B) * B
        turn = lambda x, p, step: _turned64(x, p, c["d"], "half", "none", 1.0, False, step)  # noqa: E731
        at = t["pos"].long()[:, None] + torch.arange(c["n"], device=DEVICE)
        q, k = t["q"].double(), t["k"].double()
        old = t["old_k"].double()
        if c["rope"]:
            q, k = turn(t["q"], at, lambda v: v), turn(t["k"], at, _f32)
            old = turn(t["old_k"], t["start"].long()[:, None] + torch.arange(B, device=DEVICE), _f32)
        for i in range(c["seqs"]):
            r = int(t["pos"][i] - t["start"][i])
            for new, before, to in ((k[i], old[i], ks), (t["v"][i].double(), t["old_v"][i].double(), vs)):
                rows = torch.zeros(touched, *new.shape[1:], dtype=torch.float64, device=DEVICE)
                rows[:r], rows[r: r + c["n"]] = before[:r], new
                to.append(_stored64(rows, B, c["format"]).flatten(-2))
        return {"k": torch.stack(ks), "v": torch.stack(vs), "q": q}
    if c["kind"] == "attend":
        S, n_q, H, d = c["seqs"], c["n_q"], c["kv_heads"], c["d"]
        G = c["heads"] // H
        out = torch.zeros(S, n_q, c["heads"], d, dtype=torch.float64, device=DEVICE)
        w = t["w"].double() if c["weights"] else None
        for i in range(S):
            n = int(t["n_kv"][i])
            k, v = (_stored64(t[x][i].double(), c["block"], c["format"])[:n] for x in ("k", "v"))
            for h in range(c["heads"] if n else 0):
                x = t["q"][i, :, h].double() @ k[:, h // G].T / math.sqrt(d)
                if c["causal"]:
                    x += torch.full_like(x, -math.inf).triu(n - n_q + 1)
                p = torch.softmax(x, -1)
                out[i, :, h] = p @ v[:, h // G]
                if w is not None:
                    w[i, h // G, :n] += p.sum(0)
        return {"out": out, "w": w} if c["weights"] else {"out": out}
    L, S, N, H, K = c["layers"], c["seqs"], c["n_kv"], c["kv_heads"], c["keep"]
    w = t["w"].cpu()
    kept = torch.full((L, S, H, K), -1, dtype=torch.int64)
    wo = torch.zeros(L, S, H, N, dtype=torch.float64)
    ko = torch.zeros(L, S, K, H, c["d"], dtype=torch.float64, device=DEVICE)
    vo = torch.zeros_like(ko)
    for a in range(L):
        for i in range(S):
            n = int(t["n_kv"][i])
            held = [_stored64(t[x][a, i].double(), c["block"], c["format"]) for x in ("k", "v")]
            if n <= K:  # nothing is cut: the rows stay, those past n as they were
                ko[a, i], vo[a, i] = held[0][:K], held[1][:K]
            for h in range(H):
                if n <= K:
                    idx = list(range(n))
                else:
                    middle = w[a, i, h, c["first"]: n - c["recent"]].tolist()
                    best = sorted(range(len(middle)), key=lambda j: (-middle[j], j))[: K - c["first"] - c["recent"]]
                    idx = sorted([*range(c["first"]), *(c["first"] + j for j in best), *range(n - c["recent"], n)])
                kept[a, i, h, : len(idx)] = torch.tensor(idx)
                wo[a, i, h, : len(idx)] = w[a, i, h, idx].double()
                if n > K:
                    rows = torch.tensor(idx, device=DEVICE)
                    for x, to in ((held[0], ko), (held[1], vo)):
                        to[a, i, :, h] = _stored64(x[rows, h: h + 1], c["block"], c["format"])[:, 0]
    return {"kept": kept, "w": wo, "n_kv": t["n_kv"].clamp(max=K).long().cpu(), "k": ko.flatten(-2), "v": vo.flatten(-2)}
