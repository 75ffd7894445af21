"""A decode step on a bounded cache as a program calls it: cases, their plain form in torch operations, and their
values in 64 bits.

The paged cache is the one of operators.py's cases: page p of `page` tokens is one run of bytes, kv head after kv head,
each K [page][dim], V [page / 16][dim][16] and, with 8-bit elements, a float32 scale per token for K and for V.

  rope      q's and k's heads are normed and rotated by their positions; k and v go into the cache on the way. From an
            8-bit cache the rows are read back, as the values that it stands for
  weights   attention over the cache, which also adds up the weight that every cached position gets
  evict     of each sequence and kv head the first `sinks` positions, the last `recent` and the heaviest of the others
            are kept, `keep` in all, and move to new pages in their order (read back from an 8-bit cache)
  logprobs  log probabilities of given tokens, entropy, and the `top` most likely tokens, from rows of logits
"""
import math
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda:0"
IO = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS, THETA = 1e-6, 1e6
own = False


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def _cache_case(name, op, cache, io, seqs, new, ctx, heads=64, kv_heads=8, dim=128, page=64, ragged=False, **more):
    c = {"op": op, "cache": cache, "io": io, "seqs": seqs, "new": new, "ctx": ctx, "heads": heads, "kv_heads": kv_heads,
         "dim": dim, "page": page, "ragged": ragged}
    c.update(more)
    return dict(c, name=name) if name else c


def _rope(name, cache, io, seqs, new, ctx, rotated=1, pairs="halves", norm=True, moved=0, **more):
    return _cache_case(name, "rope", cache, io, seqs, new, ctx, rotated=rotated, pairs=pairs, norm=norm, moved=moved, **more)


def _weights(name, cache, io, seqs, new, ctx, window=0, sinks=0, fresh=False, **more):
    return _cache_case(name, "weights", cache, io, seqs, new, ctx, window=window, sinks=sinks, fresh=fresh, **more)


def _evict(name, cache, seqs, ctx, keep, recent, sinks, **more):
    return _cache_case(name, "evict", cache, "f32", seqs, 1, ctx, keep=keep, recent=recent, sinks=sinks, **more)


def _logprobs(name, io, rows, vocab, given, top, masked=False):
    c = {"op": "logprobs", "io": io, "rows": rows, "vocab": vocab, "given": given, "top": top, "masked": masked}
    return dict(c, name=name) if name else c


def listed():
    # 64 heads over 8 kv heads of 128 channels and a vocabulary of 151936: the decoder layer and the head that the linear
    # benchmarks run
    return [
        # a decode step of 16 branches whose cache has been thinned: true positions lie behind the cache's
        _rope("rope_16_branches", "f16", "f32", 16, 1, 1569, moved=977),
        # packed chunks of unequal length of a 16-bit model that rotates half of its channels by neighbours, without norms
        _rope("rope_chunks_bf16", "f16", "bf16", 9, 701, 1999, rotated=2, pairs="neighbours", norm=False, heads=20,
              kv_heads=4, dim=64, page=16, ragged=True),
        # a prompt's rows of one layer
        _rope("rope_prompt_2048", "f16", "f32", 1, 2048, 2048),
        # the smallest step: one token of one conversation
        _weights("weights_1x1025", "f16", "f32", 1, 1, 1025),
        # a decode step of a serving batch over 8-bit caches of unequal length; the sums start with this step
        _weights("weights_24x2100_q8", "q8", "f32", 24, 1, 2100, page=32, ragged=True, fresh=True),
        # a full serving batch over long contexts: the most bytes
        _weights("weights_64x8192_bf16", "f16", "bf16", 64, 1, 8192),
        # a prompt: every position's weight over the whole prompt, the most operations
        _weights("weights_prompt_2048", "f16", "f32", 1, 2048, 2048),
        # conversations past their budget, 8-bit caches of unequal length
        _evict("evict_24x3001_q8", "q8", 24, 3001, 1024, 128, 4, page=32, ragged=True),
        # a full batch is halved
        _evict("evict_64x8192", "f16", 64, 8192, 4096, 512, 16),
        # the next token of one conversation with its alternatives
        _logprobs("logprobs_1", "f32", 1, 151936, 1, 20),
        # branches with a constrained vocabulary, each scored for a handful of answers
        _logprobs("logprobs_16_masked", "f32", 16, 151936, 8, 5, masked=True),
        # a prompt's tokens scored, 16-bit logits of an odd vocabulary
        _logprobs("logprobs_2047_bf16", "bf16", 2047, 151937, 1, 8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Another case of the same ranges, no more work than the largest listed ones."""
    op = rng.choice(["rope", "rope", "weights", "weights", "evict", "logprobs", "logprobs"])
    if op == "logprobs":
        vocab = rng.choice([_log(rng, 1000, 200000), 151936])
        rows = _log(rng, 1, max(2, 2047 * 151937 // (2 * vocab)))
        rows = min(rows, 8192)
        return _logprobs("", rng.choice(["f32", "bf16", "f16"]), rows, vocab, _log(rng, 1, 64), rng.choice([0, 1, 5, 20, 33, 64]),
                         masked=rng.random() < 0.3)
    cache, dim, page = rng.choice(["f16", "q8"]), rng.choice([64, 128, 128]), rng.choice([16, 32, 64, 128])
    kv_heads = rng.choice([1, 2, 4, 6, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 5, 8, 8, 16])
    row = kv_heads * dim
    shape = {"heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page}
    if op == "rope":
        io = "bf16" if cache == "q8" else rng.choice(["f32", "f32", "bf16", "f16"])
        tokens = _log(rng, 1, max(1, 2048 * 64 * 128 // (heads * dim + 2 * row)))
        seqs = min(tokens, _log(rng, 1, 32))
        new = -(-tokens // seqs)
        return _rope("", cache, io, seqs, new, new + _log(rng, 1, 600), rotated=rng.choice([1, 1, 2, 4]),
                     pairs=rng.choice(["halves", "neighbours"]), norm=rng.random() < 0.7, moved=rng.choice([0, 0, 5000, 3000017]),
                     ragged=seqs > 1, **shape)
    if op == "evict":
        ctx = _log(rng, 64, 30000)
        most = 64 * 8192 * 1024 // (2 * ctx * row) // (2 if cache == "q8" else 1)      # those are read back, in 32 bits
        seqs = _log(rng, 1, min(64, max(1, most)))
        keep = max(8, int(ctx * rng.uniform(0.1, 1.0)))
        sinks = rng.choice([0, 1, 4])
        return _evict("", cache, seqs, ctx, keep, int((keep - sinks) * rng.uniform(0, 0.6)), sinks, ragged=seqs > 1, **shape)
    io = rng.choice(["f32", "f32", "bf16", "f16"])
    if rng.random() < 0.6:       # decode: one token, or a few
        new = rng.choice([1, 1, 1, 2, 4])
        ctx = _log(rng, 64, 20000)
        most = min(64, max(1, 64 * 8192 * 1024 // (ctx * row * 2)), max(1, 64 * 2048 * 1024 // (heads * new * ctx)))
        seqs = _log(rng, 1, most)
    else:                        # chunks
        new = _log(rng, 5, 1500)
        ctx = new + _log(rng, 1, 6000)
        seqs = _log(rng, 1, min(16, max(1, 64 * 2048 * 1024 // (2 * heads * new * ctx))))
        while seqs * heads * new * ctx > 64 * 2048 * 1024:
            new = max(1, new // 2)
            ctx = max(new, ctx // 2)
    window, sinks = (_log(rng, 16, 2000), rng.choice([0, 1, 4, 21])) if rng.random() < 0.25 else (0, 0)
    return _weights("", cache, io, seqs, new, ctx, window=window, sinks=sinks, ragged=seqs > 1,
                    fresh=rng.random() < 0.4, **shape)


def _lengths(c):
    """(new rows, context length) of each sequence: the first has the most, ragged ones spread down to about half."""
    new, ctx = [], []
    for b in range(c["seqs"]):
        down = (b * 7 % c["seqs"]) / (2.0 * c["seqs"]) if c["ragged"] else 0.0
        new.append(max(1, c["new"] - int(down * c["new"])))
        ctx.append(max(new[-1], c["ctx"] - int(down * c["ctx"])))
    return new, ctx


def work(case):
    c = case
    size = 4 if c["io"] == "f32" else 2
    if c["op"] == "logprobs":
        n = c["rows"] * c["vocab"]
        return {"bytes": n * size + c["rows"] * (8 * c["given"] + 4 + 8 * c["top"]), "flops": 5 * n}
    new, ctx = _lengths(c)
    rows, row, wide = sum(new), c["kv_heads"] * c["dim"], c["heads"] * c["dim"]
    held = 2 * row * (2 if c["cache"] == "f16" else 1) + (8 * c["kv_heads"] if c["cache"] == "q8" else 0)
    if c["op"] == "rope":
        read_back = (held + 2 * row * size) if c["cache"] == "q8" else 0
        return {"bytes": rows * (2 * wide * size + 2 * row * size + held + read_back), "flops": 10 * rows * (wide + row)}
    if c["op"] == "evict":
        kept = sum(min(n, c["keep"]) for n in ctx)
        read_back = kept * (held + 2 * row * size) if c["cache"] == "q8" else 0
        return {"bytes": kept * (2 * held + 8 * c["kv_heads"]) + sum(ctx) * 4 * c["kv_heads"] + read_back,
                "flops": sum(ctx) * c["kv_heads"]}
    pairs = tokens = 0
    w, s = c["window"], c["sinks"]
    for n, length in zip(new, ctx):
        for p in (range(length - n, length) if w else ()):
            pairs += min(p + 1, w) + min(s, max(0, p + 1 - w))
        if w:
            low = max(0, length - n - w + 1)
            tokens += length - low + min(s, low)
        else:
            pairs += n * (length - n) + n * (n + 1) // 2
            tokens += length
    sums = sum(ctx) * (4 if c["fresh"] else 8) * c["kv_heads"]
    return {"bytes": tokens * held + sums + 2 * rows * wide * size, "flops": 4 * pairs * wide}


# ---------------------------------------------------------------------------
# what a program has in hand
# ---------------------------------------------------------------------------

def _regions(pool, c):
    """(K, V, K scale, V scale) as views into the cache's bytes."""
    pages, heads, page, dim = pool.shape[0], c["kv_heads"], c["page"], c["dim"]
    t, e = (torch.float16, 2) if c["cache"] == "f16" else (torch.int8, 1)
    n = page * dim * e
    k = pool[:, :, :n].view(t).view(pages, heads, page, dim)
    v = pool[:, :, n:2 * n].view(t).view(pages, heads, page // 16, dim, 16)
    if c["cache"] == "f16":
        return k, v, None, None
    return k, v, pool[:, :, 2 * n:2 * n + 4 * page].view(torch.float32), pool[:, :, 2 * n + 4 * page:].view(torch.float32)


def _pool(c, pages, g):
    e = 2 if c["cache"] == "f16" else 1
    chunk = 2 * c["page"] * c["dim"] * e + (8 * c["page"] if e == 1 else 0)
    pool = torch.empty((pages, c["kv_heads"], chunk), dtype=torch.uint8, device=DEV)
    k, v, ks, vs = _regions(pool, c)
    # keys have a few channels that stand out, values have none; every token's vectors have a size of their own
    channel = torch.where(torch.rand(c["dim"], generator=g, device=DEV) < 0.03, 4.0, 1.0)
    per = max(1, (1 << 27) // (c["kv_heads"] * c["page"] * c["dim"]))
    for p in range(0, pages, per):
        kk, vv = k[p:p + per], v[p:p + per]
        rk = torch.randn(kk.shape, generator=g, device=DEV, dtype=torch.float16)
        rv = torch.randn(vv.shape, generator=g, device=DEV, dtype=torch.float16)
        if e == 2:
            kk.copy_(rk * channel.half())
            vv.copy_(rv)
        else:
            kk.copy_((rk * 36).round_().clamp_(-127, 127))
            vv.copy_((rv * 38).round_().clamp_(-127, 127))
    if e == 1:
        ks.copy_(torch.exp(0.25 * torch.randn(ks.shape, generator=g, device=DEV)) / 36)
        vs.copy_(torch.exp(0.5 * torch.randn(vs.shape, generator=g, device=DEV)) / 38)
    return pool, channel


def _ints(a):
    return torch.tensor(a, dtype=torch.int32, device=DEV)


def _starts(new):
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    return starts


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEV).manual_seed(seed)
    if c["op"] == "logprobs":
        return _prepare_logprobs(c, g)
    t, dim = IO[c["io"]], c["dim"]
    new, ctx = _lengths(c)
    starts, width = _starts(new), -(-max(ctx) // c["page"])
    more = -(-c["keep"] // c["page"]) if c["op"] == "evict" else 0
    old = c["seqs"] * width
    pool, channel = _pool(c, old + c["seqs"] * more, g)
    # pages are handed out as sequences grow, so a table's entries are in no order
    table = torch.randperm(old, generator=g, device=DEV).to(torch.int32).view(c["seqs"], width)
    rows, row = starts[-1], c["kv_heads"] * dim
    s = {"case": c, "pool": pool, "table": table, "max_new": max(new), "max_kv": max(ctx), "rows": rows, "pages": old,
         "row_start": _ints(starts), "kv_len": _ints(ctx)}
    if c["op"] != "rope":        # what some steps leave: most positions have little, many nothing
        shape = (c["seqs"], c["kv_heads"], max(ctx) + 3)
        s["before"] = torch.exp(2.5 * torch.randn(shape, generator=g, device=DEV)).sub_(0.2).clamp_(min=0.0).mul_(0.01)
    if c["op"] == "rope":
        channels = dim // c["rotated"]
        s["inv_freq"] = (THETA ** (-torch.arange(0, channels, 2, device=DEV, dtype=torch.float64) / channels)).float()
        s["gamma"] = [1 + 0.2 * torch.randn(dim, generator=g, device=DEV) if c["norm"] else None for _ in "qk"]
        s["positions"] = None
        if c["moved"]:
            at = torch.cat([torch.arange(n - m, n) for m, n in zip(new, ctx)]) + c["moved"]
            s["positions"] = at.to(torch.int32).to(DEV)
        s["q"] = (torch.randn((rows, c["heads"] * dim), generator=g, device=DEV) * 1.5).to(t)
        s["k"] = (torch.randn((rows, row), generator=g, device=DEV) * channel.repeat(c["kv_heads"])).to(t)
        s["v"] = torch.randn((rows, row), generator=g, device=DEV).to(t)
        s["q_out"], s["k_out"], s["v_out"] = (torch.empty_like(s[x]) for x in "qkv")
    elif c["op"] == "weights":
        s["q"] = (torch.randn((rows, c["heads"] * dim), generator=g, device=DEV) * 1.5).to(t)
        s["out"], s["weights"] = torch.empty_like(s["q"]), torch.zeros_like(s["before"])
    else:
        s["new_table"] = (old + torch.randperm(c["seqs"] * more, generator=g, device=DEV)).to(torch.int32).view(c["seqs"], more)
        s["new_len"] = torch.empty(c["seqs"], dtype=torch.int32, device=DEV)
        s["kept"] = torch.empty((c["seqs"], c["kv_heads"], c["keep"]), dtype=torch.int32, device=DEV)
        s["weights"] = torch.zeros_like(s["before"])
        left = _starts([min(n, c["keep"]) for n in ctx])
        s["left"], s["left_start"] = left[-1], _ints(left)
        s["k_out"] = torch.empty((left[-1], row), device=DEV)
        s["v_out"] = torch.empty_like(s["k_out"])
    if own:   # the handles that a program keeps beside its tensors
        q3q4 = _library()
        s["cache"] = q3q4.KVCache(q3q4.KV_F16 if c["cache"] == "f16" else q3q4.KV_Q8, pool.shape[0], c["page"],
                                  c["kv_heads"], dim, pool)
        s["batch"] = q3q4.KVBatch(s["row_start"], s["kv_len"], table, rows, s["max_new"], s["max_kv"])
        if c["op"] == "rope":
            s["rope"] = q3q4.Rope(s["inv_freq"], s["gamma"][0], s["gamma"][1], EPS,
                                  q3q4.ROPE_HALVES if c["pairs"] == "halves" else q3q4.ROPE_NEIGHBOURS)
        elif c["op"] == "weights":
            s["workspace"] = q3q4.attention_weights_workspace(s["cache"], s["batch"], c["heads"])
        else:
            s["left_batch"] = q3q4.KVBatch(s["left_start"], s["new_len"], s["new_table"], s["left"],
                                           min(max(ctx), c["keep"]), min(max(ctx), c["keep"]))
    return s


def _prepare_logprobs(c, g):
    rows, vocab = c["rows"], c["vocab"]
    x = torch.empty((rows, vocab), dtype=IO[c["io"]], device=DEV)
    for r in range(0, rows, 256):
        y = torch.randn((min(256, rows - r), vocab), generator=g, device=DEV).mul_(2.2)
        if c["masked"]:
            y.masked_fill_(torch.rand(y.shape, generator=g, device=DEV) < 0.6, -math.inf)
        x[r:r + 256] = y
    # a few tokens stand out, by more or by less
    peaks = torch.randint(0, vocab, (rows, 4), generator=g, device=DEV)
    x.scatter_(1, peaks, (6 + 5 * torch.randn((rows, 4), generator=g, device=DEV)).to(x.dtype))
    tokens = torch.randint(0, vocab, (rows, c["given"]), generator=g, device=DEV)
    tokens[:, 0] = peaks[:, 0]
    s = {"case": c, "logits": x, "tokens": tokens.to(torch.int32),
         "given": torch.empty((rows, c["given"]), device=DEV), "entropy": torch.empty(rows, device=DEV),
         "ids": torch.empty((rows, c["top"]), dtype=torch.int32, device=DEV), "top": torch.empty((rows, c["top"]), device=DEV)}
    if own:
        s["workspace"] = _library().logprobs_workspace(x, c["top"])
    return s


def _library():
    if os.path.join(ROOT, "sera.c_amd") not in sys.path:
        sys.path.insert(0, os.path.join(ROOT, "sera.c_amd"))
    import q3q4
    return q3q4


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    s = state
    c = s["case"]
    op, q8 = c["op"], c.get("cache") == "q8"
    if op == "logprobs":
        if own:
            import q3q4
            q3q4.logprobs(s["logits"], s["tokens"], s["given"], s["entropy"], s["ids"], s["top"], workspace=s["workspace"])
            return s["given"], s["entropy"], s["ids"], s["top"]
        return _score(s)
    if op == "rope":
        if own:
            import q3q4
            q3q4.kv_write_rope(s["cache"], s["batch"], s["rope"], s["q"], s["q_out"], s["k"], s["v"], s["positions"])
            if q8:
                q3q4.kv_read(s["cache"], s["batch"], s["k_out"], s["v_out"])
                return s["q_out"], s["k_out"], s["v_out"]
            return (s["q_out"],) + _regions(s["pool"], c)[:2]
        q = _rotate(s)
        return (q,) + (_read(s, s["row_start"], s["kv_len"], s["table"], s["rows"], s["k"].dtype) if q8
                       else _regions(s["pool"], c)[:2])
    if op == "weights":
        if own:
            import q3q4
            q3q4.attention_weights(s["cache"], s["batch"], s["q"], s["out"], c["dim"] ** -0.5, s["weights"],
                                   None if c["fresh"] else s["before"], window=c["window"], sinks=c["sinks"],
                                   workspace=s["workspace"])
            return s["out"], s["weights"]
        return _attend(s)
    if own:
        import q3q4
        q3q4.kv_evict(s["cache"], s["batch"], c["keep"], s["before"], s["new_table"], s["new_len"], s["weights"], s["kept"],
                      recent=c["recent"], sinks=c["sinks"])
        if q8:
            q3q4.kv_read(s["cache"], s["left_batch"], s["k_out"], s["v_out"])
            held = s["k_out"], s["v_out"]
        else:
            held = _regions(s["pool"][s["pages"]:], c)[:2]
        return held + (s["weights"], s["kept"], s["new_len"])
    kept, length, weights = _evict_plain(s)
    held = (_read(s, s["left_start"], length, s["new_table"], s["left"], torch.float32) if q8
            else _regions(s["pool"][s["pages"]:], c)[:2])
    return held + (weights, kept, length)


def _places(s, row_start, kv_len, table, rows):
    """Sequence, position, page and offset of every packed row."""
    r = torch.arange(rows, device=DEV)
    b = torch.searchsorted(row_start[1:].contiguous(), r.to(torch.int32), right=True)
    at = kv_len.long()[b] - row_start.long()[b + 1] + r
    page = s["case"]["page"]
    return b, at, table.long()[b, at // page], at % page


def _quantise(x):
    """int8 codes and the scale of each vector (last axis) of x; the quotient is in 64 bits."""
    d = x.abs().amax(-1, keepdim=True) / 127
    q = torch.where(d > 0, torch.round(x.double() / d.double()), 0.0).clamp(-127, 127)
    return q.to(torch.int8), d[..., 0]


def _normed(x, gamma, s, at):
    """Heads x [rows, heads, dim] in 32 bits, normed and rotated."""
    c = s["case"]
    if gamma is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * gamma
    angle = at.double()[:, None] * s["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    n = c["dim"] // c["rotated"]
    turned = x.clone()
    a, b = (x[..., :n // 2], x[..., n // 2:n]) if c["pairs"] == "halves" else (x[..., 0:n:2], x[..., 1:n:2])
    first, second = a * cos - b * sin, a * sin + b * cos
    if c["pairs"] == "halves":
        turned[..., :n // 2], turned[..., n // 2:n] = first, second
    else:
        turned[..., 0:n:2], turned[..., 1:n:2] = first, second
    return turned


def _rotate(s):
    """Rotated q; k and v into the cache."""
    c = s["case"]
    k, v, ks, vs = _regions(s["pool"], c)
    _, at, p, o = _places(s, s["row_start"], s["kv_len"], s["table"], s["rows"])
    true = at if s["positions"] is None else s["positions"]
    q = _normed(s["q"].float().unflatten(1, (c["heads"], c["dim"])), s["gamma"][0], s, true)
    kx = _normed(s["k"].float().unflatten(1, (c["kv_heads"], c["dim"])), s["gamma"][1], s, true)
    vx = s["v"].float().unflatten(1, (c["kv_heads"], c["dim"]))
    if ks is None:
        k[p, :, o] = kx.half()
        v[p, :, o // 16, :, o % 16] = vx.half()
    else:
        (kq, kd), (vq, vd) = _quantise(kx), _quantise(vx)
        k[p, :, o] = kq
        v[p, :, o // 16, :, o % 16] = vq
        ks[p, :, o] = kd
        vs[p, :, o] = vd
    return q.flatten(1).to(s["q"].dtype)


def _read(s, row_start, kv_len, table, rows, t):
    k, v, ks, vs = _regions(s["pool"], s["case"])
    _, _, p, o = _places(s, row_start, kv_len, table, rows)
    kx, vx = k[p, :, o].float() * ks[p, :, o][..., None], v[p, :, o // 16, :, o % 16].float() * vs[p, :, o][..., None]
    return kx.flatten(1).to(t), vx.flatten(1).to(t)


def _attend(s):
    """Softmax attention in 32 bits, every sequence padded to the longest, and the columns' sums."""
    c = s["case"]
    seqs, hk, dim, page = c["seqs"], c["kv_heads"], c["dim"], c["page"]
    g, new, width = c["heads"] // hk, s["max_new"], s["table"].shape[1]
    k, v, ks, vs = _regions(s["pool"], c)
    at = s["table"].long()
    kx, vx = k[at].float(), v[at].float()                  # [seqs, width, hk, page, dim], [.., page/16, dim, 16]
    if ks is not None:
        kx *= ks[at][..., None]
        vx *= vs[at].view(seqs, width, hk, page // 16, 1, 16)
    n = width * page
    kx = kx.permute(0, 2, 1, 3, 4).reshape(seqs, hk, n, dim)
    vx = vx.permute(0, 2, 1, 3, 5, 4).reshape(seqs, hk, n, dim)
    length, start = s["kv_len"].long(), s["row_start"].long()
    count = start[1:] - start[:-1]
    i = torch.arange(new, device=DEV)
    row = (start[:-1, None] + i).clamp_(max=s["rows"] - 1)
    q = s["q"].float()[row].view(seqs, new, hk, g, dim).permute(0, 2, 3, 1, 4).reshape(seqs, hk, g * new, dim)
    score = torch.matmul(q, kx.transpose(-1, -2).contiguous()).mul_(dim ** -0.5).view(seqs, hk, g, new, n)
    p = (length - count)[:, None] + i                      # [seqs, new]: each row's position
    j = torch.arange(n, device=DEV)
    see = j <= p[..., None]
    if c["window"]:
        see &= (j > p[..., None] - c["window"]) | (j < c["sinks"])
    score.masked_fill_(~see[:, None, None], -math.inf)
    score = score.sub_(score.amax(-1, keepdim=True)).exp_()
    score /= score.sum(-1, keepdim=True)
    vx = vx.masked_fill_((j >= length[:, None])[:, None, :, None], 0.0)
    o = torch.matmul(score.view(seqs, hk, g * new, n), vx)
    o = o.view(seqs, hk, g, new, dim).permute(0, 3, 1, 2, 4).reshape(seqs, new, hk * g * dim)
    score.masked_fill_((i >= count[:, None])[:, None, None, :, None], 0.0)
    m = s["max_kv"]
    got = score.sum((2, 3))[..., :m]
    j = j[:m]
    if not c["fresh"]:
        got += torch.where(j < (length - count)[:, None, None], s["before"][..., :m], 0.0)
    weights = s["weights"]
    weights[..., :m] = torch.where(j < length[:, None, None], got, weights[..., :m])
    return o[i < count[:, None]].to(s["q"].dtype), weights


def _ordered(x):
    """Whole numbers in the order of x's float32 values (no NaN)."""
    i = (x + 0.0).view(torch.int32).long()
    return torch.where(i < 0, -(i & 0x7fffffff), i)


def _evict_plain(s):
    """The kept positions, the new lengths and weights; what is kept goes to the new pages."""
    c = s["case"]
    keep, page, m = c["keep"], c["page"], s["max_kv"]
    length = s["kv_len"].long()[:, None, None]
    j = torch.arange(m, device=DEV)
    key = _ordered(s["before"][..., :m].contiguous())
    key = torch.where((j < c["sinks"]) | (j >= length - c["recent"]), 1 << 31, key)
    key = torch.where(j < length, key, -(1 << 31)) * (1 << 31) + (m - j)      # no two alike, the lower position before
    pos = torch.topk(key, keep, -1).indices
    pos = torch.where(pos < length, pos, m).sort(-1).values
    there = pos < m
    kept = torch.where(there, pos, -1).to(torch.int32)
    weights = s["weights"]
    weights[..., :keep] = torch.where(there, s["before"].gather(-1, pos), weights[..., :keep])
    b, h, t = there.nonzero(as_tuple=True)
    pos = pos[b, h, t]
    p, o = s["table"].long()[b, pos // page], pos % page
    to, at = s["new_table"].long()[b, t // page], t % page
    k, v, ks, vs = _regions(s["pool"], c)
    k[to, h, at] = k[p, h, o]
    v[to, h, at // 16, :, at % 16] = v[p, h, o // 16, :, o % 16]
    if ks is not None:
        ks[to, h, at] = ks[p, h, o]
        vs[to, h, at] = vs[p, h, o]
    return kept, s["kv_len"].clamp(max=keep), weights


def _score(s):
    c = s["case"]
    x = s["logits"].float()
    shifted = x - x.amax(-1, keepdim=True)
    e = shifted.exp()
    total = e.sum(-1, keepdim=True)
    lse = total.log()
    entropy = (lse - torch.where(e > 0, e * shifted, 0.0).sum(-1, keepdim=True) / total)[:, 0]
    given = shifted.gather(1, s["tokens"].long()) - lse
    key = _ordered(x) * (1 << 20) + (c["vocab"] - torch.arange(c["vocab"], device=DEV))      # the lower token first
    ids = torch.topk(key, c["top"], -1).indices
    return given, entropy, ids.to(torch.int32), shifted.gather(1, ids) - lse


# ---------------------------------------------------------------------------
# the same values from the definition, in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "logprobs":
        given, entropy, top = [], [], []
        for r in range(0, c["rows"], 128):
            x = s["logits"][r:r + 128].double()
            lp = torch.log_softmax(x, -1)
            given.append(lp.gather(1, s["tokens"][r:r + 128].long()))
            entropy.append(-torch.where(lp > -math.inf, lp.exp() * lp, 0.0).sum(-1))
            top.append(lp.topk(c["top"], -1).values)
        return torch.cat(given), torch.cat(entropy), None, torch.cat(top)
    hk, dim, page, wide = c["kv_heads"], c["dim"], c["page"], 2 * c["page"] * c["dim"]
    new, ctx = _lengths(c)
    table = s["table"].cpu().tolist()

    def codes(x):
        """What an 8-bit cache makes of vectors x."""
        d = (x.abs().amax(-1) / 127).float().double()      # the scale is held in 32 bits
        return torch.where(d[..., None] > 0, torch.round(x / d[..., None]), 0.0) * d[..., None]

    def cached(b, h, n):
        """Keys and values of positions 0 .. n of sequence b, kv head h."""
        raw = s["pool"][torch.tensor(table[b][:-(-n // page)], device=DEV), h]
        if c["cache"] == "f16":
            x = raw.contiguous().view(torch.float16).double()
        else:
            x = raw[:, :wide].contiguous().view(torch.int8).double()
        kk = x[:, :page * dim].unflatten(1, (page, dim))
        vv = x[:, page * dim:].unflatten(1, (page // 16, dim, 16)).transpose(2, 3).flatten(1, 2)
        if c["cache"] == "q8":
            d = raw[:, wide:].contiguous().view(torch.float32).double()
            kk, vv = kk * d[:, :page, None], vv * d[:, page:, None]
        return kk.flatten(0, 1)[:n], vv.flatten(0, 1)[:n]

    if c["op"] == "rope":
        at = torch.cat([torch.arange(n - m, n, device=DEV) for m, n in zip(new, ctx)]).double() + c["moved"]
        z = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), at[:, None, None] * s["inv_freq"].double())
        n = dim // c["rotated"]

        def turned(x, gamma):
            y = x.double().unflatten(1, (-1, dim))
            if gamma is not None:
                y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS) * gamma.double()
            apart = c["pairs"] == "halves"
            pair = y[..., :n].unflatten(-1, (2, n // 2)).transpose(-1, -2) if apart else y[..., :n].unflatten(-1, (n // 2, 2))
            w = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * z)
            w = w.transpose(-1, -2).flatten(-2) if apart else w.flatten(-2)
            return torch.cat([w, y[..., n:]], -1)

        q, k, v = turned(s["q"], s["gamma"][0]), turned(s["k"], s["gamma"][1]), s["v"].double().unflatten(1, (hk, dim))
        if c["cache"] == "q8":
            return q.flatten(1), codes(k).flatten(1), codes(v).flatten(1)
        held = [a.double() for a in _regions(s["pool"], c)[:2]]
        row = 0
        for b in range(c["seqs"]):
            for j in range(ctx[b] - new[b], ctx[b]):
                to = table[b][j // page]
                held[0][to, :, j % page] = k[row].half().double()
                held[1][to, :, (j % page) // 16, :, j % 16] = v[row].half().double()
                row += 1
        return (q.flatten(1),) + tuple(held)
    if c["op"] == "evict":
        weights, rows = s["weights"].double(), []
        held = [a.double() for a in _regions(s["pool"][s["pages"]:], c)[:2]] if c["cache"] == "f16" else None
        to = (s["new_table"].long() - s["pages"]).cpu().tolist()
        before = s["before"].cpu().numpy()
        for b in range(c["seqs"]):
            length, ks, vs = ctx[b], [], []
            for h in range(hk):
                kk, vv = cached(b, h, length)
                middle = range(c["sinks"], length - c["recent"])
                room = c["keep"] - c["sinks"] - c["recent"]
                pos = list(range(length))
                if length > c["keep"]:
                    best = sorted(middle, key=lambda j: (-before[b, h, j], j))[:room]
                    pos = sorted(list(range(c["sinks"])) + best + list(range(length - c["recent"], length)))
                i = torch.tensor(pos, device=DEV)
                weights[b, h, :len(pos)] = s["before"][b, h, i].double()
                ks.append(kk[i])
                vs.append(vv[i])
                if held is not None:
                    for z in range(0, len(pos), page):
                        n = min(page, len(pos) - z)
                        held[0][to[b][z // page], h, :n] = kk[i[z:z + n]]
                        flat = held[1][to[b][z // page], h].transpose(1, 2).flatten(0, 1).clone()
                        flat[:n] = vv[i[z:z + n]]
                        held[1][to[b][z // page], h] = flat.unflatten(0, (-1, 16)).transpose(1, 2)
            rows.append((torch.cat(ks, 1), torch.cat(vs, 1)))
        if held is None:
            held = [torch.cat([r[a] for r in rows]) for a in (0, 1)]
        return tuple(held) + (weights, None, None)
    g, outs, at = c["heads"] // hk, [], 0
    weights = s["weights"].double()
    for b in range(c["seqs"]):
        n, length = new[b], ctx[b]
        q = s["q"][at:at + n].double().unflatten(1, (hk, g, dim))
        pos = torch.arange(length - n, length, device=DEV)[:, None]
        j = torch.arange(length, device=DEV)
        hidden = j > pos
        if c["window"]:
            hidden = hidden | ((j <= pos - c["window"]) & (j >= c["sinks"]))
        o = torch.empty((n, hk, g, dim), dtype=torch.float64, device=DEV)
        for h in range(hk):
            kk, vv = cached(b, h, length)
            weights[b, h, :length] = 0
            if not c["fresh"]:
                weights[b, h, :length - n] = s["before"][b, h, :length - n].double()
            for x in range(g) if n > 16 else (slice(None),):
                qq = q[:, h, x]
                z = (qq @ kk.T) / math.sqrt(dim)
                hid = hidden if z.dim() == 2 else hidden[:, None]
                p = torch.softmax(z.masked_fill(hid, -math.inf), -1)
                o[:, h, x] = p @ vv
                weights[b, h, :length] += p.flatten(0, -2).sum(0)
        outs.append(o.flatten(1))
        at += n
    return torch.cat(outs), weights
