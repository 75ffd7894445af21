"""A layer and a head whose cache stays within a budget: a prompt, then tokens one by one.

Rows of the residual stream go through RMSNorm and the q/k/v products (Q4_K); q's and k's heads are normed and rotated
on the way into the paged cache; attention adds up the weight that every cached position gets; the o product adds to
the residual. A conversation that reaches `limit` positions is thinned to `keep`: the first four, the last eight and the
heaviest of the others move to new pages, and the old ones are free again. From then on a token's true position, which it
is rotated by, is not its place in the cache. The head's logits give the log probability of a token, the entropy and the
most likely tokens. Every stage is compared with the same in 64 bits over what the stage before it left.

    python examples/bounded_cache.py [f16|q8]
"""
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if os.path.join(ROOT, "sera.c_amd") not in sys.path:
    sys.path.insert(0, os.path.join(ROOT, "sera.c_amd"))
import q3q4  # noqa: E402

HIDDEN, HEADS, KV_HEADS, DIM, PAGE, VOCAB, TOP = 1024, 16, 4, 128, 16, 4096, 5
SINKS, RECENT, EPS = 4, 8, 1e-6


def _weight(rows, k, gen, dev):
    x = torch.randn((rows, k), generator=gen, device=dev) * k ** -0.5
    w = torch.empty((rows, k // 256 * 144), dtype=torch.uint8, device=dev)
    q3q4.quantize_weights(x, w)
    return q3q4.bind_geometry(q3q4.QTYPE_Q4_K, k, rows), w


def _off(got, want):
    """Largest difference, relative to the largest value."""
    return float((got.double() - want).abs().max() / want.abs().max())


class Model:
    def __init__(self, gen, dev):
        self.dev = dev
        self.qkv = [_weight(n * DIM, HIDDEN, gen, dev) for n in (HEADS, KV_HEADS, KV_HEADS)]
        self.o, self.head = _weight(HIDDEN, HEADS * DIM, gen, dev), _weight(VOCAB, HIDDEN, gen, dev)
        self.gamma = 1 + 0.1 * torch.randn(HIDDEN, generator=gen, device=dev)
        self.q_gamma, self.k_gamma = (1 + 0.1 * torch.randn(DIM, generator=gen, device=dev) for _ in "qk")
        self.inv_freq = (1e6 ** (-torch.arange(0, DIM, 2, device=dev, dtype=torch.float64) / DIM)).float()
        self.rope = q3q4.Rope(self.inv_freq, self.q_gamma, self.k_gamma, EPS)

    def turned(self, x, gamma, at):
        """Heads of rows x in 64 bits."""
        y = x.double().unflatten(1, (-1, DIM))
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS) * gamma.double()
        a = at.double()[:, None, None] * self.inv_freq.double()
        i, j = y[..., :DIM // 2], y[..., DIM // 2:]
        return torch.cat([i * a.cos() - j * a.sin(), i * a.sin() + j * a.cos()], -1).flatten(1)


def run(kind=q3q4.KV_Q8, prompts=(70, 33), limit=72, keep=48, steps=12, device=0, seed=0):
    """The largest error of each stage, and how often a conversation was thinned."""
    dev = f"cuda:{device}"
    gen = torch.Generator(device=dev).manual_seed(seed)
    ints = lambda a: torch.tensor(a, dtype=torch.int32, device=dev)  # noqa: E731
    n, width = len(prompts), -(-(max(max(prompts), limit) + 1) // PAGE)
    products = q3q4.Linear(device=device, max_tokens=sum(prompts), max_features=max(VOCAB, HEADS * DIM), max_k=HEADS * DIM)
    model = Model(gen, dev)
    cache = q3q4.KVCache(kind, 2 * n * width, PAGE, KV_HEADS, DIM, device=device)
    cache.data.zero_()
    tables = [ints(range(n * width)).view(n, width), ints(range(n * width, 2 * n * width)).view(n, width)]
    weights = [torch.zeros((n, KV_HEADS, width * PAGE), device=dev) for _ in "ab"]
    now, lens, seen = 0, [0] * n, [0] * n               # tables in use; places taken; tokens so far
    worst, thinned = {"rope": 0.0, "attention": 0.0, "weights": 0.0, "logprobs": 0.0}, 0

    def note(stage, off):
        worst[stage] = off if not off <= worst[stage] else worst[stage]         # a NaN stays

    for step in range(steps + 1):
        news = list(prompts) if step == 0 else [1] * n
        lens, seen = [a + b for a, b in zip(lens, news)], [a + b for a, b in zip(seen, news)]
        starts = [0]
        for m in news:
            starts.append(starts[-1] + m)
        rows = starts[-1]
        at = torch.cat([torch.arange(s - m, s, device=dev) for s, m in zip(seen, news)]).to(torch.int32)
        batch = q3q4.KVBatch(ints(starts), ints(lens), tables[now], rows, max(news), width * PAGE)
        hidden = torch.randn((rows, HIDDEN), generator=gen, device=dev)
        q, k, v = (torch.empty((rows, h * DIM), device=dev) for h in (HEADS, KV_HEADS, KV_HEADS))
        turned, out, old = torch.empty_like(q), torch.empty_like(q), weights[now].clone()
        q3q4.linear_group([g for g, _ in model.qkv], [w for _, w in model.qkv], [q, k, v], hidden, gamma=model.gamma, eps=EPS,
                          flags=q3q4.LIN_RMSNORM)
        q3q4.kv_write_rope(cache, batch, model.rope, q, turned, k, v, at)
        q3q4.attention_weights(cache, batch, turned, out, DIM ** -0.5, weights[now], weights[now],
                               workspace=q3q4.attention_weights_workspace(cache, batch, HEADS))
        q3q4.linear_group([model.o[0]], [model.o[1]], [hidden], out, flags=q3q4.LIN_ACCUMULATE)
        logits = torch.empty((rows, VOCAB), device=dev)
        q3q4.linear_group([model.head[0]], [model.head[1]], [logits], hidden, gamma=model.gamma, eps=EPS, flags=q3q4.LIN_RMSNORM)
        tokens = torch.randint(0, VOCAB, (rows, 1), generator=gen, device=dev).to(torch.int32)
        given, entropy = torch.empty((rows, 1), device=dev), torch.empty(rows, device=dev)
        ids, top = torch.empty((rows, TOP), dtype=torch.int32, device=dev), torch.empty((rows, TOP), device=dev)
        q3q4.logprobs(logits, tokens, given, entropy, ids, top, workspace=q3q4.logprobs_workspace(logits, TOP))

        # the same in 64 bits
        note("rope", _off(turned, model.turned(q, model.q_gamma, at)))
        whole = [0]
        for length in lens:
            whole.append(whole[-1] + length)
        kk, vv = (torch.empty((whole[-1], KV_HEADS * DIM), device=dev) for _ in "kv")
        q3q4.kv_read(cache, q3q4.KVBatch(ints(whole), ints(lens), tables[now], whole[-1], max(lens), max(lens)), kk, vv)
        if kind == q3q4.KV_F16:        # fp16 holds keys within 2^-11
            new = torch.cat([kk[e - m:e] for e, m in zip(whole[1:], news)])
            note("rope", max(0.0, _off(new, model.turned(k, model.k_gamma, at)) - 2.0 ** -11))
        for s in range(n):
            own = slice(starts[s], starts[s + 1])
            keys, values = (t[whole[s]:whole[s + 1]].double().view(-1, KV_HEADS, DIM) for t in (kk, vv))
            hid = torch.arange(lens[s], device=dev) > torch.arange(lens[s] - news[s], lens[s], device=dev)[:, None]
            sums = torch.zeros((KV_HEADS, lens[s]), dtype=torch.float64, device=dev)
            sums[:, :lens[s] - news[s]] = old[s, :, :lens[s] - news[s]].double()
            for h in range(HEADS):
                g, cols = h * KV_HEADS // HEADS, slice(h * DIM, (h + 1) * DIM)
                z = turned[own, cols].double() @ keys[:, g].t().contiguous() * DIM ** -0.5
                p = torch.softmax(z.masked_fill(hid, -torch.inf), -1)
                sums[g] += p.sum(0)
                note("attention", _off(out[own, cols], p @ values[:, g].contiguous()))
            note("weights", _off(weights[now][s, :, :lens[s]], sums))
        lp = torch.log_softmax(logits.double(), -1)
        best = lp.topk(TOP, -1)
        note("logprobs", max(_off(given, lp.gather(1, tokens.long())), _off(top, best.values), _off(entropy, -(lp.exp() * lp).sum(-1)),
                             float((ids != best.indices).any())))

        if max(lens) >= limit:          # thin those; the others go along to the new pages as they are
            new_len, kept = ints([0] * n), torch.empty((n, KV_HEADS, keep), dtype=torch.int32, device=dev)
            short = [length if length < limit else keep for length in lens]
            q3q4.kv_evict(cache, batch, keep, weights[now], tables[1 - now], new_len, weights[1 - now], kept, RECENT, SINKS)
            lens, now = new_len.tolist(), 1 - now
            if lens != [min(a, keep) for a in short]:
                raise RuntimeError(f"lengths {lens} after thinning {short}")
            thinned += 1
    del products
    return worst, thinned


if __name__ == "__main__":
    kinds = {"f16": q3q4.KV_F16, "q8": q3q4.KV_Q8}
    for name in sys.argv[1:] or list(kinds):
        e, times = run(kinds[name])
        print(f"{name}: thinned {times} times; " + ", ".join(f"{k} {x:.2e}" for k, x in e.items()), flush=True)
