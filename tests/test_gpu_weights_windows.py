"""sera_attention_weights with a window on the GPU: how its work is shared out, and what it does not read."""
import numpy as np
import pytest

import attn_oracle as ao
import q3q4
from test_gpu_attention import torch  # noqa: F401  (torch: the fixture)

pytestmark = pytest.mark.gpu
TILE = 512                                  # positions of a unit of the sums of many rows, of 32 columns


def setup(torch, news, lens, heads, kv_heads, page=64):  # noqa: F811
    ints = lambda a: torch.tensor(np.asarray(a, np.int32), device="cuda")  # noqa: E731
    width = -(-max(lens) // page)
    cache = q3q4.KVCache(ao.F16, width, page, kv_heads, 128)
    cache.data.zero_()
    batch = q3q4.KVBatch(ints([0] + list(np.cumsum(news))), ints(lens), ints(np.tile(np.arange(width), (len(news), 1))), sum(news),
                         max(news), max(lens))
    return cache, batch, torch.randn(sum(news), heads * 128, device="cuda")


def units(new, length, group, window, sinks):
    """Blocks of 32 columns over the tiles that a row of theirs sees any of."""
    first, n = length - new, 0
    for j in range(0, length, TILE):
        end = new if not window or j < sinks else min(new, max(j + TILE - 1 + window - first, 0))
        n += max(-(-end * group // 32) - max(j - first, 0) * group // 32, 0)
    return n


@pytest.mark.parametrize("news,lens,window,sinks", [([1024], [16384], 512, 4), ([512], [32768], 1024, 0), ([1024], [16384], 0, 0),
                                                    ([300, 200], [9000, 7000], 300, 70), ([2048], [2048], 256, 0)])
def test_the_work_of_a_window_is_shared_by_all(torch, news, lens, window, sinks):  # noqa: F811
    """Every workgroup leaves the sums of its part of a tile in a place of its own behind the rows' norms: the places that
    are written tell how many had work. They are to be at least half of as many as an equal share for every compute unit
    gives (shares are of the longest sequence, and of 8 units at least)."""
    heads, kv_heads = 64, 8
    print(f"case {news} of {lens} window={window} sinks={sinks}", flush=True)
    cache, batch, q = setup(torch, news, lens, heads, kv_heads)
    out, weights = torch.empty_like(q), torch.empty(len(news), kv_heads, max(lens), device="cuda")
    ws = q3q4.attention_weights_workspace(cache, batch, heads)
    plain = q3q4.attention_workspace(cache, batch, heads)
    ws.fill_(0xA5)
    q3q4.attention_weights(cache, batch, q, out, 0.1, weights, None, window, sinks, workspace=ws)
    torch.cuda.synchronize()
    at = -(-(0 if plain is None else plain.numel()) // 16) * 16 + batch.rows * heads * 8
    written = (ws[at:].view(-1, 4 * TILE) != 0xA5).any(1).view(len(news) * kv_heads, -1).sum(1).tolist()
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    each = [units(n, length, heads // kv_heads, window, sinks) for n, length in zip(news, lens)]
    share = max(8, -(-sum(each) * kv_heads // cus))
    for b, n in enumerate(each):
        print(f"  sequence {b}: {n} units, {written[b * kv_heads]} places of sums", flush=True)
        assert min(written[b * kv_heads:(b + 1) * kv_heads]) >= n / (2 * share)


def test_steps_with_a_window_do_not_read_the_scores_of_the_whole_context(torch):  # noqa: F811
    """64 single tokens over 8192 positions of which 16 are seen: the sums may take some times the attention itself, but not
    the time of the whole context's scores (268 MB, some 50 us; the attention some 10)."""
    cache, batch, q = setup(torch, [1] * 64, [8192] * 64, 128, 8)
    out, weights = torch.empty_like(q), torch.zeros(64, 8, 8192, device="cuda")
    ws, ws2 = q3q4.attention_weights_workspace(cache, batch, 128), q3q4.attention_workspace(cache, batch, 128)

    def time_of(step):
        step()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            for _ in range(20):
                step()
        best = 1e9
        for _ in range(7):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            g.replay()
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b) * 50)
        return best

    whole = time_of(lambda: q3q4.attention_weights(cache, batch, q, out, 0.1, weights, None, workspace=ws))
    both = time_of(lambda: q3q4.attention_weights(cache, batch, q, out, 0.1, weights, None, 16, workspace=ws))
    alone = time_of(lambda: q3q4.attention(cache, batch, q, out, 0.1, 16, workspace=ws2))
    print(f"  whole {whole:.1f} us, with a window {both:.1f}, its attention alone {alone:.1f}", flush=True)
    assert both < 4 * alone
