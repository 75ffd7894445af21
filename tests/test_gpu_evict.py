"""sera_kv_evict on the GPU: what stays is exactly what the oracle keeps, and arrives byte for byte."""
import numpy as np
import pytest

import attn_oracle as ao
import q3q4
import step_oracle as so
from test_gpu_attention import F32, Setup, spoil, torch  # noqa: F401  (torch: the fixture)

pytestmark = pytest.mark.gpu


def run(torch, s, weights, keep, recent=0, sinks=0, new_table=None, max_kv=None, spare=3):  # noqa: F811
    """One call; (new_len, kept, new_weights, pool) of it. New pages lie behind the old ones."""
    n, kv = len(s.lens), s.kv_heads
    entries = -(-min(keep, max_kv or max(s.lens)) // s.page)
    old = s.pool.shape[0]
    if new_table is None:
        s.pool = np.concatenate([s.pool, np.full((n * entries + spare,) + s.pool.shape[1:], 0x5A, np.uint8)])
        new_table = (old + s.rng.permutation(n * entries + spare)[:n * entries]).reshape(n, entries).astype(np.int32)
    s.new_table = new_table
    cache, batch = s.device(max_kv=max_kv)
    w = torch.from_numpy(weights).cuda()
    to = torch.full_like(w, 9.0)
    new_len = torch.full((n,), 77, dtype=torch.int32, device="cuda")
    kept = torch.full((n, kv, keep), 77, dtype=torch.int32, device="cuda")
    table = torch.from_numpy(np.ascontiguousarray(new_table)).cuda()
    q3q4.kv_evict(cache, batch, keep, w, table, new_len, to, kept, recent=recent, sinks=sinks)
    torch.cuda.synchronize()
    assert np.array_equal(w.cpu().numpy(), weights, equal_nan=True)
    return new_len.cpu().numpy(), kept.cpu().numpy(), to.cpu().numpy(), s.data.cpu().numpy().reshape(s.pool.shape)


def check(torch, s, weights, keep, recent=0, sinks=0, ok=None, **more):  # noqa: F811
    new_len, kept, to, pool = run(torch, s, weights, keep, recent, sinks, **more)
    want = s.pool.copy()
    parts = ao.views(want, s.kind, s.page, s.kv_heads, s.dim)
    old = ao.views(s.pool, s.kind, s.page, s.kv_heads, s.dim)
    for b, length in enumerate(s.lens):
        if ok is not None and not ok[b]:
            assert new_len[b] == -1 and (kept[b] == -1).all() and (to[b] == 9.0).all()
            continue
        assert new_len[b] == min(length, keep)
        for h in range(s.kv_heads):
            pos = so.kept_of(weights[b, h], length, keep, recent, sinks)
            assert kept[b, h, :len(pos)].tolist() == pos, f"sequence {b} head {h}"
            assert (kept[b, h, len(pos):] == -1).all()
            assert np.array_equal(to[b, h, :len(pos)], weights[b, h, pos], equal_nan=True) and (to[b, h, len(pos):] == 9.0).all()
            for t, j in enumerate(pos):
                p, o, f, g = s.new_table[b][t // s.page], t % s.page, s.table[b][j // s.page], j % s.page
                if not 0 <= p < pool.shape[0]:
                    continue
                lost = not 0 <= f < pool.shape[0]
                x = [np.nan] * 4 if lost else [old[0][f, h, g], old[1][f, h, g // 16, :, g % 16],
                                               *(a[f, h, g] if a is not None else None for a in old[2:])]
                if lost and s.kind == ao.Q8:
                    x[:2] = [0, 0]
                parts[0][p, h, o], parts[1][p, h, o // 16, :, o % 16] = x[0], x[1]
                if s.kind == ao.Q8:
                    parts[2][p, h, o], parts[3][p, h, o] = x[2], x[3]
    for a, b in zip(ao.views(pool, s.kind, s.page, s.kv_heads, s.dim), parts):
        assert a is None or np.array_equal(a, b, equal_nan=a.dtype != np.int8)


def weights_of(s, rng, kind="spread", stride=None):
    shape = (len(s.lens), s.kv_heads, stride or max(s.lens) + 3)
    w = np.exp(3 * rng.standard_normal(shape)).astype(np.float32)
    if kind == "ties":
        w = np.floor(w)                            # most are 0 or the same few
    if kind == "equal":
        w[:] = 0.25
    if kind == "signs":
        w = rng.integers(-3, 4, shape).astype(np.float32) * np.float32(0.5)
        w[rng.random(shape) < 0.2] = -0.0
    if kind == "odd":
        w[rng.random(shape) < 0.1] = np.nan
        w[rng.random(shape) < 0.1] = np.inf
        w[rng.random(shape) < 0.1] = -np.inf
        w[rng.random(shape) < 0.1] = 1e-42
    return w


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 16), (128, 64), (64, 128)])
@pytest.mark.parametrize("keep,recent,sinks", [(64, 16, 4), (33, 0, 0), (70, 70, 0), (20, 3, 17), (1, 0, 0), (600, 100, 2)])
def test_sizes(torch, kind, dim, page, keep, recent, sinks):  # noqa: F811
    print(f"case kind={kind} dim={dim} page={page} keep={keep} recent={recent} sinks={sinks}", flush=True)
    lens = [300, 1, 64, 65, 0, 33, 34, 1027, 16]
    s = Setup(torch, kind, F32, [0] * len(lens), lens, kv_heads=3, dim=dim, page=page)
    check(torch, s, weights_of(s, s.rng), keep, recent, sinks)


@pytest.mark.parametrize("spread", ["spread", "ties", "equal", "signs", "odd"])
@pytest.mark.parametrize("keep,recent,sinks", [(500, 64, 4), (100, 0, 0), (1999, 10, 1)])
def test_ties_signs_and_odd_weights(torch, spread, keep, recent, sinks):  # noqa: F811
    print(f"case {spread} keep={keep} recent={recent} sinks={sinks}", flush=True)
    s = Setup(torch, ao.F16, F32, [0, 0], [2000, 1501], kv_heads=2, dim=64, page=32)
    check(torch, s, weights_of(s, s.rng, spread), keep, recent, sinks)


@pytest.mark.parametrize("length,keep", [(20000, 700), (40001, 40000), (70000, 16)])
def test_long_contexts(torch, length, keep):  # noqa: F811
    s = Setup(torch, ao.Q8, F32, [0], [length], kv_heads=1, dim=64, page=128)
    check(torch, s, weights_of(s, s.rng, "ties"), keep, keep // 4, 4)


@pytest.mark.parametrize("length", [4096, 4097, 8192, 8193, 16384, 16385, 24576, 24577])
@pytest.mark.parametrize("spread", ["spread", "equal", "signs"])
def test_lengths_around_what_registers_hold(torch, length, spread):  # noqa: F811
    print(f"case {length} {spread}", flush=True)
    s = Setup(torch, ao.Q8, F32, [0, 0], [length, length // 3], kv_heads=1, dim=64, page=128)
    check(torch, s, weights_of(s, s.rng, spread), length // 2, 100, 3)


def test_shared_pages_stay(torch):  # noqa: F811
    """Branches that share a prefix are thinned each to pages of its own; the shared ones stay as they were."""
    s = Setup(torch, ao.F16, F32, [0] * 5, [300] * 5, kv_heads=2, page=16, shared=15)
    check(torch, s, weights_of(s, s.rng), 128, 20, 4)


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
def test_short_sequences_keep_their_pages(torch, kind):  # noqa: F811
    """A sequence of up to `keep` positions that names its own pages again: nothing moves; the others do."""
    s = Setup(torch, kind, F32, [0, 0, 0], [40, 200, 64], kv_heads=2, page=16)
    entries, old = 4, s.pool.shape[0]
    s.pool = np.concatenate([s.pool, np.full((entries,) + s.pool.shape[1:], 0x5A, np.uint8)])
    table = s.table[:, :entries].copy()
    table[1] = old + np.arange(entries)
    check(torch, s, weights_of(s, s.rng), 64, 8, 2, new_table=table)


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("entry", [-1, 1 << 20, -(1 << 31)])
def test_bad_pages_are_not_followed(torch, kind, entry):  # noqa: F811
    """Tokens of an old page outside the pool arrive as NaN; to a new one nothing is written."""
    s = Setup(torch, kind, F32, [0, 0], [300, 300], kv_heads=2, page=16)
    s.table[0, 5] = entry
    old = s.pool.shape[0]
    s.pool = np.concatenate([s.pool, np.full((16,) + s.pool.shape[1:], 0x5A, np.uint8)])
    table = (old + np.arange(16)).reshape(2, 8).astype(np.int32)
    table[1, 3] = entry
    check(torch, s, weights_of(s, s.rng), 128, 20, 4, new_table=table)


@pytest.mark.parametrize("lens", [[301, 100], [-1, 100], [100, -(1 << 31)], [2 ** 31 - 1, 250]])
def test_lengths_outside_the_bounds(torch, lens):  # noqa: F811
    s = Setup(torch, ao.F16, F32, [0, 0], [300, 300], kv_heads=2, page=16)
    s.lens = lens
    check(torch, s, weights_of(s, s.rng, stride=301), 64, 8, 2, ok=[0 <= n <= 300 for n in lens], max_kv=300)


def test_nothing_behind_the_end_matters(torch):  # noqa: F811
    s = Setup(torch, ao.F16, F32, [0], [75], kv_heads=2, page=64)
    spoil(s, 0, range(75, 128), np.nan)
    w = weights_of(s, s.rng, stride=128)
    w[:, :, 75:] = 1e30
    check(torch, s, w, 50, 5, 5)


def test_graph_replays_take_the_lengths_and_weights_of_their_time(torch):  # noqa: F811
    s = Setup(torch, ao.F16, F32, [0, 0], [300, 200], kv_heads=2, page=16)
    old = s.pool.shape[0]
    s.pool = np.concatenate([s.pool, np.zeros((8,) + s.pool.shape[1:], np.uint8)])
    cache, batch = s.device(max_kv=304)
    w = torch.rand(2, 2, 304, device="cuda")
    to, new_len = torch.zeros_like(w), torch.zeros(2, dtype=torch.int32, device="cuda")
    kept = torch.zeros(2, 2, 64, dtype=torch.int32, device="cuda")
    table = torch.arange(old, old + 8, dtype=torch.int32, device="cuda").view(2, 4)

    def step():
        q3q4.kv_evict(cache, batch, 64, w, table, new_len, to, kept, recent=8, sinks=2)

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for lens in ([300, 200], [299, 64], [65, 0]):
        w.copy_(torch.rand_like(w))
        batch.kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
        for t in (to, kept, new_len):
            t.fill_(5)
        cache.data.view(-1, cache.page_bytes)[old:] = 0
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (to, kept, new_len, cache.data)]
        for b, n in enumerate(lens):
            for h in range(2):
                pos = so.kept_of(w[b, h].cpu().numpy(), n, 64, 8, 2)
                assert kept[b, h, :len(pos)].tolist() == pos
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        q3q4.kv_evict(cache, batch, 64, w, table, new_len, to, kept, recent=8, sinks=2, stream=side)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (to, kept, new_len, cache.data)))


def test_no_sequences(torch):  # noqa: F811
    s = Setup(torch, ao.F16, F32, [0], [20], kv_heads=2)
    cache, batch = s.device()
    i = lambda *a: torch.zeros(a, dtype=torch.int32, device="cuda")  # noqa: E731
    e = torch.empty(0, 2, 20, device="cuda")
    none = q3q4.KVBatch(batch.row_start[:1], batch.kv_len[:0], batch.page_table[:0], 0, 1, 1)
    q3q4.kv_evict(cache, none, 8, e, i(0, 1), i(0), e.clone(), i(0, 2, 8))


def test_offsets_past_32_bits(torch):  # noqa: F811
    """Pages at the end of a pool of more than 4 GiB, moved to its first ones."""
    page, kv_heads = 64, 8
    page_bytes = q3q4.kv_page_bytes(ao.F16, page, kv_heads, 128)
    pages = (9 << 29) // page_bytes
    cache = q3q4.KVCache(ao.F16, pages, page, kv_heads, 128)
    i = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    table = torch.arange(pages - 4, pages, dtype=torch.int32, device="cuda")[None]
    k = torch.randn(200, 1024, device="cuda").half().float()
    q3q4.kv_write(cache, q3q4.KVBatch(i([0, 200]), i([200]), table, 200, 200, 200), k, -k)
    w = torch.rand(1, 8, 200, device="cuda")
    new, kept, new_len, to = i([[0, 1]]), torch.zeros(1, 8, 100, dtype=torch.int32, device="cuda"), i([0]), torch.zeros_like(w)
    q3q4.kv_evict(cache, q3q4.KVBatch(i([0, 0]), i([200]), table, 0, 1, 200), 100, w, new, new_len, to, kept, recent=9)
    ko, vo = torch.empty(100, 1024, device="cuda"), torch.empty(100, 1024, device="cuda")
    q3q4.kv_read(cache, q3q4.KVBatch(i([0, 100]), new_len, new, 100, 100, 100), ko, vo)
    for h in range(8):
        want = k[kept[0, h].long(), h * 128:(h + 1) * 128]
        assert torch.equal(ko[:, h * 128:(h + 1) * 128], want) and torch.equal(vo[:, h * 128:(h + 1) * 128], -want)
        assert kept[0, h].tolist() == so.kept_of(w[0, h].cpu().numpy(), 200, 100, 9, 0)
