"""The key/value cache and its attention as a program calls them: cases, their plain
form in torch operations, and their values in 64 bits.

A paged key/value cache holds the keys and values of many sequences. Page p of
`page` tokens is one run of bytes, kv head after kv head; a head's run is

    K        [page][dim]              elements
    V        [page / 16][dim][16]     elements: 16 tokens of one channel side by side
    K scale  [page] float32           only with 8-bit elements
    V scale  [page] float32           only with 8-bit elements

Elements are fp16, or int8 with one scale for each token and kv head. A batch
is `seqs` sequences whose new rows are packed one after the other: sequence b
has the rows row_start[b] .. row_start[b+1], which are the last positions of
its kv_len[b] positions; position j is in page table[b][j / page].

  write      the new rows' keys and values go into the cache
  roundtrip  the same, and are read back as the values that the cache stands for
  read       cached positions come back as dense rows
  attention  each new row attends to the positions up to its own, or to the
             last `window` of them and the first `sinks`
"""
import math
import os
import random
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda:0"
IO = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
own = False


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def _case(name, op, cache, io, seqs, new, ctx, heads=64, kv_heads=8, dim=128, page=64, ragged=False, shared=0,
          window=0, sinks=0):
    c = {"op": op, "cache": cache, "io": io, "seqs": seqs, "new": new, "ctx": ctx, "heads": heads,
         "kv_heads": kv_heads, "dim": dim, "page": page, "ragged": ragged, "shared": shared, "window": window,
         "sinks": sinks}
    return dict(c, name=name) if name else c


def listed():
    # 64 heads over 8 kv heads of 128 channels: the q (8192) and k/v (1024) rows of the decoder layer that the linear
    # benchmarks run
    return [
        # a decode step of 16 branches appends one token each, behind the shared 1536-token prefix
        _case("append_16_branches", "write", "f16", "f32", 16, 1, 1569, shared=1536),
        # packed chunks of unequal length from a 16-bit model and other head counts
        _case("write_chunks_bf16", "write", "f16", "bf16", 9, 701, 1999, heads=24, kv_heads=6, dim=64, page=16,
              ragged=True),
        # prefill writes an 8-bit cache; what the model will see of it is read back
        _case("write_read_2048_q8", "roundtrip", "q8", "f32", 1, 2048, 2048),
        # whole contexts leave the 8-bit cache as dense rows (moved to another layout or host)
        _case("read_contexts_q8", "read", "q8", "f32", 12, 4099, 4099, ragged=True),
        # the smallest call: one token of one short conversation
        _case("decode_1x513", "attention", "f16", "f32", 1, 1, 513),
        # a decode step of a serving batch, 8-bit cache, unequal lengths
        _case("decode_24x2100_q8", "attention", "q8", "f32", 24, 1, 2100, page=32, ragged=True),
        # a full serving batch over long contexts: the most bytes
        _case("decode_64x8192_bf16", "attention", "f16", "bf16", 64, 1, 8192),
        # shared-prefix branches: 16 suffixes of 32 tokens over one 1536-token prefix
        _case("branches_16x32_over_1536", "attention", "f16", "f32", 16, 32, 1568, shared=1536),
        # prefill of one prompt
        _case("prefill_2048", "attention", "f16", "f32", 1, 2048, 2048),
        # a chunk of a long prompt against what the cache holds already: the most operations
        _case("chunk_512_of_32768_q8", "attention", "q8", "f32", 1, 512, 32768, page=128),
        # decode with a window and sinks: the middle of the context is not read
        _case("decode_window_32x20000", "attention", "f16", "f32", 32, 1, 20000, window=1024, sinks=4, ragged=True),
        # a ragged prefill with a window of 16-bit rows and other head counts
        _case("prefill_window_3x1501_f16", "attention", "f16", "f16", 3, 1501, 2503, heads=20, kv_heads=4, dim=64,
              page=16, ragged=True, window=500, sinks=16),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Another case of the same ranges, no more work than the largest listed ones."""
    op = rng.choice(["write", "roundtrip", "read", "attention", "attention", "attention", "attention"])
    cache, io = rng.choice(["f16", "q8"]), rng.choice(["f32", "f32", "bf16", "f16"])
    dim, page = rng.choice([64, 128, 128]), rng.choice([16, 32, 64, 128])
    kv_heads = rng.choice([1, 2, 4, 6, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 5, 8, 8, 16])
    row = kv_heads * dim
    if op != "attention":
        cache = "f16" if op == "write" else cache
        tokens = _log(rng, 1, max(1, 2048 * 1024 // row))
        seqs = min(tokens, _log(rng, 1, 16))
        new = -(-tokens // seqs)
        ctx = new if op == "read" else new + _log(rng, 1, 600)
        return _case("", op, cache, io, seqs, new, ctx, heads, kv_heads, dim, page, ragged=seqs > 1)
    if rng.random() < 0.5:       # decode: one token, or a few
        new = rng.choice([1, 1, 1, 2, 4])
        ctx = _log(rng, 64, 20000)
        most = min(64, max(1, 64 * 8192 * 1024 // (ctx * row * 2)), max(1, 64 * 512 * 32768 // (heads * new * ctx)))
        seqs = _log(rng, 1, most)
    else:                        # chunks
        new = _log(rng, 5, 2048)
        ctx = new + _log(rng, 1, 16000)
        seqs = _log(rng, 1, min(16, max(1, 64 * 512 * 32768 // (2 * heads * new * ctx))))
        while seqs * heads * new * ctx > 64 * 512 * 32768:
            new = max(1, new // 2)
            ctx = max(new, ctx // 2)
    window, sinks = (_log(rng, 16, 2000), rng.choice([0, 1, 4, 21])) if rng.random() < 0.35 else (0, 0)
    return _case("", "attention", cache, io, seqs, new, ctx, heads, kv_heads, dim, page, ragged=seqs > 1,
                 window=window, sinks=sinks)


def _lengths(c):
    """(new rows, context length) of each sequence: the first has the most, ragged ones spread down to about half."""
    new, ctx = [], []
    for b in range(c["seqs"]):
        down = (b * 7 % c["seqs"]) / (2.0 * c["seqs"]) if c["ragged"] else 0.0
        new.append(max(1, c["new"] - int(down * c["new"])))
        ctx.append(new[-1] if c["op"] == "read" else max(new[-1], c["ctx"] - int(down * c["ctx"])))
    return new, ctx


def work(case):
    c = case
    new, ctx = _lengths(c)
    rows, row = sum(new), c["kv_heads"] * c["dim"]
    io = 4 if c["io"] == "f32" else 2
    held = 2 * row * (2 if c["cache"] == "f16" else 1) + (8 * c["kv_heads"] if c["cache"] == "q8" else 0)
    if c["op"] != "attention":
        return {"bytes": rows * (2 * row * io + held) if c["op"] != "roundtrip" else rows * (4 * row * io + held),
                "flops": rows * row * 4}
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
            tokens += length - c["shared"]
    return {"bytes": (tokens + c["shared"]) * held + 2 * rows * c["heads"] * c["dim"] * io,
            "flops": 4 * pairs * c["heads"] * c["dim"]}


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


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEV).manual_seed(seed)
    new, ctx = _lengths(c)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    width = -(-max(ctx) // c["page"])
    shared = c["shared"] // c["page"]
    pages = shared + c["seqs"] * (width - shared)
    # pages are handed out as sequences grow, so a table's entries are in no order
    order = torch.randperm(pages, generator=g, device=DEV)
    table = torch.empty((c["seqs"], width), dtype=torch.int32, device=DEV)
    table[:, :shared] = order[:shared].to(torch.int32)
    table[:, shared:] = order[shared:].view(c["seqs"], width - shared).to(torch.int32)

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

    t, rows, row = IO[c["io"]], starts[-1], c["kv_heads"] * c["dim"]
    s = {"case": c, "pool": pool, "table": table, "max_new": max(new), "max_kv": max(ctx), "rows": rows,
         "row_start": torch.tensor(starts, dtype=torch.int32, device=DEV),
         "kv_len": torch.tensor(ctx, dtype=torch.int32, device=DEV)}
    if c["op"] == "attention":
        s["q"] = (torch.randn((rows, c["heads"] * c["dim"]), generator=g, device=DEV) * 1.5).to(t)
        s["out"] = torch.empty_like(s["q"])
    else:
        s["k"] = (torch.randn((rows, row), generator=g, device=DEV) * channel.repeat(c["kv_heads"])).to(t)
        s["v"] = torch.randn((rows, row), generator=g, device=DEV).to(t)
        s["k_out"], s["v_out"] = torch.empty_like(s["k"]), torch.empty_like(s["v"])
    if own:   # the handles that a program keeps beside its tensors
        if os.path.join(ROOT, "sera.c_amd") not in sys.path:
            sys.path.insert(0, os.path.join(ROOT, "sera.c_amd"))
        import q3q4
        s["cache"] = q3q4.KVCache(q3q4.KV_F16 if e == 2 else q3q4.KV_Q8, pages, c["page"], c["kv_heads"], c["dim"],
                                  pool)
        s["batch"] = q3q4.KVBatch(s["row_start"], s["kv_len"], table, rows, s["max_new"], s["max_kv"])
        if c["op"] == "attention":
            s["workspace"] = q3q4.attention_workspace(s["cache"], s["batch"], c["heads"])
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    s = state
    op = s["case"]["op"]
    if own:
        import q3q4
        if op == "attention":
            c = s["case"]
            q3q4.attention(s["cache"], s["batch"], s["q"], s["out"], c["dim"] ** -0.5, window=c["window"],
                           sinks=c["sinks"], workspace=s["workspace"])
            return s["out"]
        if op != "read":
            q3q4.kv_write(s["cache"], s["batch"], s["k"], s["v"])
            if op == "write":
                return _held(s)
        q3q4.kv_read(s["cache"], s["batch"], s["k_out"], s["v_out"])
        return s["k_out"], s["v_out"]
    if op == "attention":
        return _attend(s)
    if op != "read":
        _write(s)
        if op == "write":
            return _held(s)
    return _read(s)


def _held(s):
    """The keys and values that an fp16 cache holds after a write."""
    return _regions(s["pool"], s["case"])[:2]


def _places(s):
    """The page and the offset of every packed row's position."""
    r = torch.arange(s["rows"], device=DEV)
    b = torch.searchsorted(s["row_start"][1:].contiguous(), r.to(torch.int32), right=True)
    at = s["kv_len"].long()[b] - s["row_start"].long()[b + 1] + r
    page = s["case"]["page"]
    return s["table"].long()[b, at // page], at % page


def _quantise(x):
    """int8 codes and the scale of each vector (last axis) of x. The quotient is in 64 bits: a code lies next to a
    border where 32 bits round the quotient onto a half."""
    amax = x.abs().amax(-1, keepdim=True)
    d = amax / torch.full_like(amax, 127)
    q = torch.where(d > 0, torch.round(x.double() / d.double()), 0.0).clamp(-127, 127)
    return q.to(torch.int8), d[..., 0]


def _write(s):
    c = s["case"]
    k, v, ks, vs = _regions(s["pool"], c)
    p, o = _places(s)
    rows = (s["rows"], c["kv_heads"], c["dim"])
    kx, vx = s["k"].float().view(rows), s["v"].float().view(rows)
    if ks is None:
        k[p, :, o] = kx.half()
        v[p, :, o // 16, :, o % 16] = vx.half()
        return
    kq, kd = _quantise(kx)
    vq, vd = _quantise(vx)
    k[p, :, o] = kq
    v[p, :, o // 16, :, o % 16] = vq
    ks[p, :, o] = kd
    vs[p, :, o] = vd


def _read(s):
    c = s["case"]
    k, v, ks, vs = _regions(s["pool"], c)
    p, o = _places(s)
    kx, vx = k[p, :, o].float(), v[p, :, o // 16, :, o % 16].float()
    if ks is not None:
        kx, vx = kx * ks[p, :, o][..., None], vx * vs[p, :, o][..., None]
    t = IO[c["io"]]
    return kx.reshape(s["rows"], -1).to(t), vx.reshape(s["rows"], -1).to(t)


def _attend(s):
    """Softmax attention in 32 bits, every sequence padded to the longest."""
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
    return o[i < count[:, None]].to(s["q"].dtype)


# ---------------------------------------------------------------------------
# the same values from the definition, in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    op, hk, dim, page, wide = c["op"], c["kv_heads"], c["dim"], c["page"], 2 * c["page"] * c["dim"]
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

    if op in ("roundtrip", "write"):
        x, y = (s[a].double().unflatten(1, (hk, dim)) for a in ("k", "v"))
        x, y = (codes(a) if c["cache"] == "q8" else a.half().double() for a in (x, y))
    if op == "roundtrip":
        return x.flatten(1), y.flatten(1)
    if op == "write":
        held = [a.double() for a in _held(s)]
        at = 0
        for b in range(c["seqs"]):
            for i in range(new[b]):
                j = ctx[b] - new[b] + i
                to = table[b][j // page]
                held[0][to, :, j % page] = x[at + i]
                held[1][to, :, (j % page) // 16, :, j % 16] = y[at + i]
            at += new[b]
        return tuple(held)
    if op == "read":
        got = [[cached(b, h, ctx[b]) for h in range(hk)] for b in range(c["seqs"])]
        return tuple(torch.cat([torch.cat([got[b][h][a][ctx[b] - new[b]:] for h in range(hk)], 1)
                                for b in range(c["seqs"])]) for a in (0, 1))
    g, outs, at = c["heads"] // hk, [], 0
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
            for x in range(g) if n > 16 else (slice(None),):
                qq = q[:, h, x]
                z = (qq @ kk.T) / math.sqrt(dim)
                hid = hidden if z.dim() == 2 else hidden[:, None]
                o[:, h, x] = torch.softmax(z.masked_fill(hid, -math.inf), -1) @ vv
        outs.append(o.flatten(1))
        at += n
    return torch.cat(outs)
