"""The attention half of a decoder layer over a paged cache: a prompt, then branches of it.

A prompt's hidden states go through RMSNorm, the q/k/v products (Q4_K), the cache
write, attention and the o product with its residual; then `branches`
continuations share the prompt's pages and decode some tokens each, one step
captured in a graph and replayed while lengths and inputs change on the device. After every call the result is
compared with attention in 64 bits over the keys and values that sera_kv_read gives back.

    python examples/cached_attention.py [f16|q8]
"""
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if os.path.join(ROOT, "sera.c_amd") not in sys.path:
    sys.path.insert(0, os.path.join(ROOT, "sera.c_amd"))
import q3q4  # noqa: E402

HIDDEN, HEADS, KV_HEADS, DIM, PAGE = 5120, 64, 8, 128, 64


def _weight(rows, k, gen, dev):
    x = torch.randn((rows, k), generator=gen, device=dev) * k ** -0.5
    w = torch.empty((rows, k // 256 * 144), dtype=torch.uint8, device=dev)
    q3q4.quantize_weights(x, w)
    return q3q4.bind_geometry(q3q4.QTYPE_Q4_K, k, rows), w


class Layer:
    """Norm, q/k/v, cache, attention, o: what one call of a layer does with rows of the residual stream."""

    def __init__(self, cache, gen, dev):
        self.cache, self.scale = cache, DIM ** -0.5
        self.qkv = [_weight(n, HIDDEN, gen, dev) for n in (HEADS * DIM, KV_HEADS * DIM, KV_HEADS * DIM)]
        self.o = _weight(HIDDEN, HEADS * DIM, gen, dev)
        self.gamma = 1 + 0.1 * torch.randn(HIDDEN, generator=gen, device=dev)

    def buffers(self, batch):
        def rows(n):
            return torch.empty((batch.rows, n), device=self.gamma.device)
        return {"q": rows(HEADS * DIM), "k": rows(KV_HEADS * DIM), "v": rows(KV_HEADS * DIM), "out": rows(HEADS * DIM),
                "workspace": q3q4.attention_workspace(self.cache, batch, HEADS)}

    def __call__(self, batch, hidden, b):
        q3q4.linear_group([g for g, _ in self.qkv], [w for _, w in self.qkv], [b["q"], b["k"], b["v"]], hidden,
                          gamma=self.gamma, eps=1e-6, flags=q3q4.LIN_RMSNORM)
        q3q4.kv_write(self.cache, batch, b["k"], b["v"])
        q3q4.attention(self.cache, batch, b["q"], b["out"], self.scale, workspace=b["workspace"])
        q3q4.linear_group([self.o[0]], [self.o[1]], [hidden], b["out"], flags=q3q4.LIN_ACCUMULATE)


def check(layer, batch, b, news, lens):
    """Largest difference from attention in 64 bits over what the cache holds, relative to the largest result."""
    dev = layer.gamma.device
    ints = lambda a: torch.tensor(a, dtype=torch.int32, device=dev)  # noqa: E731
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    whole = q3q4.KVBatch(ints(starts), ints(lens), batch.page_table, starts[-1], max(lens), max(lens))
    k = torch.empty((starts[-1], KV_HEADS * DIM), device=dev)
    v = torch.empty_like(k)
    q3q4.kv_read(layer.cache, whole, k, v)
    worst, at = 0.0, 0
    for s, (n, length) in enumerate(zip(news, lens)):
        kk, vv = (t[starts[s]:starts[s + 1]].double().view(length, KV_HEADS, DIM) for t in (k, v))
        hidden = torch.arange(length, device=dev) > torch.arange(length - n, length, device=dev)[:, None]
        for h in range(HEADS):
            cols = slice(h * DIM, (h + 1) * DIM)
            z = b["q"][at:at + n, cols].double() @ kk[:, h * KV_HEADS // HEADS].t().contiguous() * layer.scale
            want = torch.softmax(z.masked_fill(hidden, -torch.inf), -1) @ vv[:, h * KV_HEADS // HEADS].contiguous()
            off = float((b["out"][at:at + n, cols] - want).abs().max() / want.abs().max())
            worst = off if not off <= worst else worst          # a NaN stays
        at += n
    return worst


def run(kind=q3q4.KV_Q8, prompt=200, branches=4, steps=3, device=0, seed=0):
    """Errors of the prompt's call and of every step's replay."""
    dev = f"cuda:{device}"
    gen = torch.Generator(device=dev).manual_seed(seed)
    ints = lambda a: torch.tensor(a, dtype=torch.int32, device=dev)  # noqa: E731
    products = q3q4.Linear(device=device, max_tokens=max(prompt, branches), max_features=HEADS * DIM, max_k=HEADS * DIM)   # holds the products' workspace
    # the prompt's whole pages are shared; each branch has the page that it goes on in, and more, to itself
    width = -(-(prompt + steps) // PAGE)
    shared = prompt // PAGE
    cache = q3q4.KVCache(kind, shared + branches * (width - shared), PAGE, KV_HEADS, DIM, device=device)
    layer = Layer(cache, gen, dev)
    table = torch.empty((branches, width), dtype=torch.int32)
    for s in range(branches):
        table[s] = torch.tensor(list(range(shared)) + [shared + s * (width - shared) + j for j in range(width - shared)])
    table = table.to(dev)

    first = q3q4.KVBatch(ints([0, prompt]), ints([prompt]), table[:1].contiguous(), prompt, prompt, prompt)
    b = layer.buffers(first)
    layer(first, torch.randn((prompt, HIDDEN), generator=gen, device=dev), b)
    errors = [check(layer, first, b, [prompt], [prompt])]
    if width > shared and prompt % PAGE:      # the prompt's last, partial page goes to every branch as bytes
        pages = cache.data.view(cache.pages, cache.page_bytes)
        for s in range(1, branches):
            pages[table[s, shared]] = pages[table[0, shared]]

    lens = ints([prompt] * branches)
    batch = q3q4.KVBatch(ints(list(range(branches + 1))), lens, table, branches, 1, prompt + steps)
    hidden, b = torch.zeros((branches, HIDDEN), device=dev), layer.buffers(batch)
    lens += 1
    layer(batch, hidden, b)                   # what a graph needs loaded, is
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer(batch, hidden, b)
    for t in range(1, steps + 1):
        hidden.copy_(torch.randn((branches, HIDDEN), generator=gen, device=dev))
        lens.fill_(prompt + t)
        graph.replay()
        torch.cuda.synchronize()
        errors.append(check(layer, batch, b, [1] * branches, [prompt + t] * branches))
    del products, graph
    return errors


if __name__ == "__main__":
    kinds = {"f16": q3q4.KV_F16, "q8": q3q4.KV_Q8}
    for name in sys.argv[1:] or list(kinds):
        e = run(kinds[name])
        print(f"{name}: prompt {e[0]:.2e}, steps " + " ".join(f"{x:.2e}" for x in e[1:]), flush=True)
