"""sera_attention_weights on the GPU: its result is sera_attention's, bit for bit, and the sums are those of the 64-bit
oracle (tolerance: step_oracle.weights_of).
"""
import numpy as np
import pytest

import attn_oracle as ao
import q3q4
import step_oracle as so
from test_gpu_attention import BF16, F16, F32, Setup, spoil, torch  # noqa: F401  (torch: the fixture)

pytestmark = pytest.mark.gpu


def expect(s, q, scale, window, sinks, before):
    """(sums, tolerance) [sequences, kv heads, max length]; before is None or an array of at least that."""
    most = max(max(s.lens), 1)
    want, tol = np.zeros((len(s.lens), s.kv_heads, most)), np.zeros((len(s.lens), s.kv_heads, most))
    q = q.reshape(s.rows, s.heads, s.dim)
    for b, n in enumerate(s.news):
        length = s.lens[b]
        if length == 0:
            continue
        K, _ = ao.values(s.pool, s.kind, s.page, s.kv_heads, s.dim, s.table, b, length)
        want[b, :, :length], tol[b, :, :length] = so.weights_of(K, q[s.starts[b]:s.starts[b] + n], length, scale, window, sinks)
        old = max(length - n, 0)
        if before is not None:
            x = before[b, :, :old].astype(np.float64)
            want[b, :, :old] += x
            tol[b, :, :old] += np.abs(x) * 2.0 ** -22
    return want, tol


def call(torch, s, q, scale, window=0, sinks=0, before=None, weights=None, stride=None, **bounds):  # noqa: F811
    s.device(**bounds)
    out = torch.full_like(q, 7.0)
    if weights is None:
        weights = torch.full((len(s.lens), s.kv_heads, stride or s.batch.max_kv + 5), 9.0, device="cuda")
    ws = q3q4.attention_weights_workspace(s.cache, s.batch, s.heads)
    if ws is not None:
        ws.fill_(0xFF)           # NaN everywhere: its content does not matter
    q3q4.attention_weights(s.cache, s.batch, q, out, scale, weights, before, window, sinks, workspace=ws)
    torch.cuda.synchronize()
    return out, weights


def compare(weights, want, tol, lens, what=""):
    got = weights.double().cpu().numpy()
    worst = 0.0
    for b, n in enumerate(lens):
        g, w, t = got[b, :, :n], want[b, :, :n], tol[b, :, :n]
        off = np.abs(g - w)
        bad = ~(off <= t) & ~(np.isnan(g) & np.isnan(w))
        worst = max(worst, np.nanmax(off / np.where(t > 0, t, np.inf), initial=0))
        assert not bad.any(), f"{what} sequence {b}: {bad.sum()} of {bad.size}, first at {np.argwhere(bad)[0]}: {g[bad][:4]} for {w[bad][:4]}"
        assert (got[b, :, n:] == 9.0).all(), f"{what} sequence {b}: places behind the end"
    print(f"  {what} worst {worst:.3f} of the tolerance", flush=True)


def check(torch, s, scale=None, window=0, sinks=0, q_scale=1.5, with_before=True, **bounds):  # noqa: F811
    scale = s.dim ** -0.5 if scale is None else scale
    q, qv = s.rows_of(s.heads * s.dim, q_scale)
    stride = max(s.lens + [bounds.get("max_kv") or 1]) + 5
    before = np.exp(2 * s.rng.standard_normal((len(s.lens), s.kv_heads, stride))).astype(np.float32) if with_before else None
    want, tol = expect(s, qv, scale, window, sinks, before)
    dev = None if before is None else torch.from_numpy(before).cuda()
    out, weights = call(torch, s, q, scale, window, sinks, dev, stride=stride, **bounds)
    compare(weights, want, tol, s.lens, f"{s.io} {s.news} of {s.lens}")
    plain = s.attend(q, scale, window, sinks, **bounds)
    assert torch.equal(out.isnan(), plain.isnan()) and torch.equal(out.nan_to_num(), plain.nan_to_num())
    return q, out, weights


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("io", [F32, F16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
def test_decode_ragged(torch, kind, io, dim):  # noqa: F811
    print(f"case decode kind={kind} io={io} dim={dim}", flush=True)
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 127, 300, 513, 1000]
    check(torch, Setup(torch, kind, io, [1] * len(lens), lens, heads=16, kv_heads=2, dim=dim, page=32, seed=dim))


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("io", [F32, BF16])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (5, 1), (12, 4), (16, 1), (40, 2), (70, 2)])
def test_head_layouts(torch, kind, io, heads, kv_heads):  # noqa: F811
    print(f"case heads={heads} kv_heads={kv_heads} kind={kind} io={io}", flush=True)
    check(torch, Setup(torch, kind, io, [1, 2], [70, 201], heads=heads, kv_heads=kv_heads, seed=heads), with_before=False)


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("io", [F32, F16, BF16])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 16), (128, 64), (128, 128)])
def test_chunks_ragged(torch, kind, io, dim, page):  # noqa: F811
    print(f"case chunks kind={kind} io={io} dim={dim} page={page}", flush=True)
    check(torch, Setup(torch, kind, io, [1, 5, 0, 33, 64, 100, 17], [90, 5, 7, 200, 64, 131, 17], heads=8, kv_heads=2, dim=dim,
                       page=page, seed=page))


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("group", [1, 3, 5, 8, 20])
def test_chunk_groups(torch, kind, group):  # noqa: F811
    print(f"case chunk group={group} kind={kind}", flush=True)
    check(torch, Setup(torch, kind, F32, [37, 70], [37, 150], heads=2 * group, kv_heads=2, page=16, seed=group))


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("news,lens", [([1], [5000]), ([3], [4999]), ([40], [3001]), ([1, 1], [9001, 20]), ([300, 1, 1], [900, 3000, 7])])
def test_split_contexts_and_mixed_batches(torch, kind, news, lens):  # noqa: F811
    print(f"case split {news} of {lens} kind={kind}", flush=True)
    check(torch, Setup(torch, kind, F32, news, lens, heads=8, kv_heads=1, page=64, seed=sum(lens)))


@pytest.mark.parametrize("max_kv", [301, 4096, 100000])
def test_loose_bounds(torch, max_kv):  # noqa: F811
    s = Setup(torch, ao.F16, F32, [1, 2, 1], [300, 17, 301], heads=8, kv_heads=2, page=16)
    wide = np.full((3, -(-max_kv // 16)), -5, np.int32)
    wide[:, :s.table.shape[1]] = s.table
    s.table = wide
    check(torch, s, max_kv=max_kv, max_new=4)


def test_many_sequences(torch):  # noqa: F811
    rng = np.random.default_rng(1)
    news = [int(n) for n in rng.integers(0, 4, 300)]
    lens = [n + int(x) for n, x in zip(news, rng.integers(0, 40, 300))]
    check(torch, Setup(torch, ao.F16, F32, news, lens, heads=2, kv_heads=1, dim=64))


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 0), (50, 4), (64, 64), (100, 33), (7, 1000), (5000, 3), (2 ** 31 - 1, 0)])
@pytest.mark.parametrize("news,lens", [([1, 1, 2], [700, 31, 90]), ([70, 9], [300, 400])])
def test_window_and_sinks(torch, kind, window, sinks, news, lens):  # noqa: F811
    print(f"case window={window} sinks={sinks} {news} of {lens} kind={kind}", flush=True)
    check(torch, Setup(torch, kind, F32, news, lens, heads=8, kv_heads=2, page=16, seed=(window + sinks) % 1000), window=window,
          sinks=sinks)


def test_windows_over_long_contexts(torch):  # noqa: F811
    check(torch, Setup(torch, ao.F16, F32, [1, 2], [9000, 8000], heads=8, kv_heads=1, page=64), window=5000, sinks=70)
    check(torch, Setup(torch, ao.Q8, BF16, [1], [12000], heads=4, kv_heads=1, page=64), window=64, sinks=4)
    check(torch, Setup(torch, ao.F16, F32, [200], [3000], heads=4, kv_heads=1, page=64), window=300, sinks=10)


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("news,lens", [([3, 2], [1, 0]), ([50, 20], [7, 40]), ([0, 4, 0], [33, 20, 0])])
def test_rows_in_front_of_the_start_and_sequences_without_rows(torch, kind, news, lens):  # noqa: F811
    """Rows that see nothing add nothing; a sequence without rows has its sums taken over."""
    check(torch, Setup(torch, kind, F32, news, lens, heads=8, kv_heads=2))


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("news,lens", [([1], [200]), ([64], [200])])
def test_peaked_and_flat_scores(torch, kind, news, lens):  # noqa: F811
    check(torch, Setup(torch, kind, F32, news, lens, heads=8, kv_heads=2), scale=3.0, q_scale=4.0, with_before=False)
    s = Setup(torch, kind, F32, news, lens, heads=8, kv_heads=2)
    check(torch, s, q_scale=0.0)
    check(torch, s, scale=0.0)
    check(torch, s, scale=-0.2)
    check(torch, s, q_scale=1e-20, scale=1e19)
    check(torch, s, q_scale=1e15, scale=1e-16)


@pytest.mark.parametrize("new", [1, 50])
def test_value_scales_do_not_matter(torch, new):  # noqa: F811
    """8-bit values whose scales span 24 binades, or are zero or not finite: the sums are those of the keys alone."""
    for e in (np.linspace(-12, 12, 700), np.full(700, -80.0), np.full(700, 90.0)):
        s = Setup(torch, ao.Q8, F32, [new], [700], heads=8, kv_heads=1, page=64)
        _, _, _, vs = s.views()
        for j in range(700):
            vs[s.table[0][j // 64], :, j % 64] = np.float32(2.0 ** e[j])
        # the maximum that the sums are held around follows the values' scales: log2 of the sum is of their size, one of up to 128,
        # and its rounding 2^-17 (ln 2 of it in a weight)
        q, qv = s.rows_of(1024)
        want, tol = expect(s, qv, 0.1, 0, 0, None)
        _, weights = call(torch, s, q, 0.1, stride=705)
        compare(weights, want, tol + 2.0 ** -16 * want, s.lens, f"scales {e[0]} to {e[-1]}")
    s = Setup(torch, ao.Q8, F32, [new], [700], heads=8, kv_heads=1, page=64)
    _, _, _, vs = s.views()
    vs[s.table[0][2], :, 5:9] = [0.0, np.nan, np.inf, -np.inf]
    q, qv = s.rows_of(1024)
    want, tol = expect(s, qv, 0.1, 0, 0, None)
    _, weights = call(torch, s, q, 0.1, stride=705)
    compare(weights, want, tol + 2.0 ** -16 * want, s.lens, "odd scales")


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("new", [1, 40])
def test_nothing_behind_the_end_matters(torch, kind, value, new):  # noqa: F811
    s = Setup(torch, kind, F32, [new], [75], heads=8, kv_heads=2, page=64)
    spoil(s, 0, range(75, 128), value)
    check(torch, s)


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("new,at", [(60, 97), (1, 50)])
def test_a_key_that_is_not_finite_spoils_what_its_rows_see(torch, kind, new, at):  # noqa: F811
    """NaN at position `at`: the rows that see it give NaN to all that they see, which is the whole context here; out of
    every window it does nothing."""
    s = Setup(torch, kind, F32, [new], [100], heads=8, kv_heads=2, page=16)
    spoil(s, 0, [at], np.nan)
    q, qv = s.rows_of(1024)
    _, weights = call(torch, s, q, 0.1, stride=105)
    assert torch.isnan(weights[..., :100]).all() and (weights[..., 100:] == 9.0).all()
    s = Setup(torch, kind, F32, [new], [100], heads=8, kv_heads=2, page=16)
    spoil(s, 0, [20], np.nan)
    want, tol = expect(s, qv, 0.1, 12, 3, None)
    _, weights = call(torch, s, q, 0.1, 12, 3, stride=105)
    compare(weights, want, tol, s.lens, "out of the windows")


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("new", [1, 40])
def test_bad_pages_are_not_followed(torch, kind, new):  # noqa: F811
    s = Setup(torch, kind, F32, [new, new], [150, 150], heads=8, kv_heads=2, page=16)
    s.table[0, 4] = -1                                       # positions 64 .. 79
    q, qv = s.rows_of(1024)
    want, tol = expect(s, qv, 0.1, 0, 0, None)
    _, weights = call(torch, s, q, 0.1, stride=155)
    assert torch.isnan(weights[0, :, :150]).all()
    compare(weights[1:], want[1:], tol[1:], s.lens[1:], "the other sequence")
    want, tol = expect(s, qv, 0.1, 5, 0, None)               # out of every window
    _, weights = call(torch, s, q, 0.1, 5, 0, stride=155)
    compare(weights, want, tol, s.lens, "out of the windows")


@pytest.mark.parametrize("starts,lens", [([0, 2, 4], [20, 301]), ([0, 2, 4], [-1, 20]), ([0, 4, 2], [20, 20]), ([0, -3, 4], [20, 20]),
                                         ([1, 2, 900], [20, 20]), ([0, 4, 4], [20, 20])])
def test_batches_outside_the_bounds(torch, starts, lens):  # noqa: F811
    """Sequences that break the host's bounds leave their places as they were."""
    s = Setup(torch, ao.F16, F32, [2, 2], [300, 300], heads=16, kv_heads=2, page=16)
    cache, _ = s.device()
    i = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    batch = q3q4.KVBatch(i(starts), i(lens), i(s.table), 4, 3, 300)
    ok = [0 <= starts[b] <= starts[b + 1] <= 4 and starts[b + 1] - starts[b] <= 3 and 0 <= lens[b] <= 300 for b in (0, 1)]
    q = torch.randn(4, 2048, device="cuda")
    out, weights = torch.full_like(q, 7.0), torch.full((2, 2, 300), 9.0, device="cuda")
    need = q3q4.attention_weights_workspace(cache, batch, 16).numel()
    ws = torch.full((need + (1 << 20),), 0xA5, dtype=torch.uint8, device="cuda")
    q3q4.attention_weights(cache, batch, q, out, 0.1, weights, workspace=ws)
    torch.cuda.synchronize()
    assert (ws[need:] == 0xA5).all()
    for b in (0, 1):
        if not ok[b]:
            assert (weights[b] == 9.0).all()
        else:
            assert (weights[b, :, lens[b]:] == 9.0).all()
            if starts == sorted(starts):
                n = starts[b + 1] - starts[b]
                K, _ = ao.values(s.pool, ao.F16, 16, 2, 128, s.table, b, lens[b])
                rows = q[starts[b]:starts[b + 1]].double().cpu().numpy().reshape(n, 16, 128)
                want, tol = so.weights_of(K, rows, lens[b], 0.1, 0, 0)
                compare(weights[b:b + 1], want[None], tol[None], [lens[b]], "the other sequence")


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("sequences", [300, 70, 40])
def test_overlapping_sequences_end(torch, kind, sequences):  # noqa: F811
    """row_start that decreases: the call ends, and nothing but rows, sums and the workspace is written."""
    print(f"case overlapping kind={kind} sequences={sequences}", flush=True)
    rows, page, heads = 100, 64, 8
    ints = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    cache = q3q4.KVCache(kind, 40, page, 1, 128)
    cache.data.zero_()
    starts = [(0, 90, 30, 100, 29)[b % 5] for b in range(sequences + 1)]
    batch = q3q4.KVBatch(ints(starts), ints([4000 - b for b in range(sequences)]), ints(np.resize(np.arange(3, 23), (sequences, 64))),
                         rows, 95, 4096)
    need = q3q4.attention_weights_workspace(cache, batch, heads).numel()
    ws = torch.full((need + (32 << 20),), 0xA5, dtype=torch.uint8, device="cuda")
    q, out = torch.randn(rows, heads * 128, device="cuda"), torch.full((rows + 16, heads * 128), 7.0, device="cuda")
    weights = torch.full((sequences, 1, 4100), 9.0, device="cuda")
    q3q4.attention_weights(cache, batch, q, out[:rows], 0.1, weights, workspace=ws)
    torch.cuda.synchronize()
    assert (ws[need:] == 0xA5).all() and (out[rows:] == 7.0).all() and (weights[..., 4000:] == 9.0).all()
    assert not cache.data.any()


def test_sums_go_on_in_place_and_repeat(torch):  # noqa: F811
    """A prompt's sums, then steps that add to them in place: those of all rows at once. Bit for bit the same on a second
    run, on other page ids and on another stream."""
    for kind in (ao.F16, ao.Q8):
        s = Setup(torch, kind, F32, [60], [60], heads=8, kv_heads=2, page=16)
        q, qv = s.rows_of(1024)
        want, tol = expect(s, qv, 0.1, 0, 0, None)
        runs = []
        for again in range(3):
            if again == 2:
                perm = np.random.default_rng(5).permutation(s.pool.shape[0])
                s.pool, s.table = s.pool[perm], np.argsort(perm)[s.table].astype(np.int32)
            weights = torch.full((1, 2, 65), 9.0, device="cuda")
            at = 0
            side = torch.cuda.Stream()
            for n in (40, 1, 1, 3, 15):
                s.device()
                i = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
                batch = q3q4.KVBatch(i(0, n), i(at + n), s.batch.page_table, n, n, 64)
                out = torch.empty(n, 1024, device="cuda")
                ws = q3q4.attention_weights_workspace(s.cache, batch, 8)
                torch.cuda.synchronize()
                q3q4.attention_weights(s.cache, batch, q[at:at + n], out, 0.1, weights, weights if at else None, workspace=ws,
                                       stream=side if again == 1 else None)
                torch.cuda.synchronize()
                at += n
            runs.append(weights)
            compare(weights, want, tol * 2 + want * 2.0 ** -20, [60], f"kind {kind} run {again}")
        assert torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("new", [1, 30])
def test_graph_replays(torch, kind, new):  # noqa: F811
    s = Setup(torch, kind, F32, [new, new], [40, 2000], heads=8, kv_heads=2, page=16)
    cache, batch = s.device()
    q = torch.randn(s.rows, 1024, device="cuda")
    out, weights = torch.zeros_like(q), torch.zeros(2, 2, 2005, device="cuda")
    before = torch.rand_like(weights)
    ws = q3q4.attention_weights_workspace(cache, batch, 8)

    def step():
        q3q4.attention_weights(cache, batch, q, out, 0.1, weights, before, workspace=ws)

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for lens in ([40, 2000], [41, 1999], [33, 700], [1500, 64]):
        q.copy_(torch.randn_like(q))
        s.lens = lens
        batch.kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
        weights.fill_(9.0)
        g.replay()
        torch.cuda.synchronize()
        want, tol = expect(s, q.double().cpu().numpy(), 0.1, 0, 0, before.cpu().numpy())
        compare(weights, want, tol, lens, f"replay at {lens}")
        replayed = weights.clone()
        weights.fill_(9.0)
        step()
        assert torch.equal(replayed, weights)


def test_large_calls_against_torch(torch):  # noqa: F811
    for kind, new, length, window, sinks in ((ao.F16, 700, 1900, 0, 0), (ao.Q8, 333, 2777, 400, 9), (ao.F16, 1, 40000, 0, 0)):
        s = Setup(torch, kind, F32, [new], [length], heads=16, kv_heads=2, page=32)
        q, _ = s.rows_of(2048, 1.5)
        _, weights = call(torch, s, q, 0.09, window, sinks)
        K, _ = ao.values(s.pool, kind, 32, 2, 128, s.table, 0, length)
        K = torch.from_numpy(K).cuda()
        p = torch.arange(length - new, length, device="cuda")[:, None]
        j = torch.arange(length, device="cuda")
        hid = j > p
        if window:
            hid = hid | ((j <= p - window) & (j >= sinks))
        want, tol = (torch.zeros(2, length, dtype=torch.float64, device="cuda") for _ in "wt")
        for h in range(16):
            qq = q.double()[:, h * 128:(h + 1) * 128]
            w = torch.softmax((qq @ K[h // 8].T * 0.09).masked_fill(hid, -torch.inf), -1)
            a = (qq.abs() @ K[h // 8].abs().T).max(1, keepdim=True).values * 0.09
            want[h // 8] += w.sum(0)
            tol[h // 8] += (w * (2 * 2.0 ** -19 * (a + 1))).sum(0)
        tol += want * (8 * new + 8) * 2.0 ** -24
        off = (weights[0, :, :length].double() - want).abs()
        print(f"  {new} of {length} worst {float((off / tol).max()):.3f} of the tolerance", flush=True)
        assert (off <= tol).all()


def test_offsets_past_32_bits(torch):  # noqa: F811
    """Sums whose places lie more than 2^31 elements from the first, keys at the end of a pool of more than 4 GiB."""
    page, kv_heads = 64, 2
    page_bytes = q3q4.kv_page_bytes(ao.F16, page, kv_heads, 128)
    pages = (9 << 29) // page_bytes
    cache = q3q4.KVCache(ao.F16, pages, page, kv_heads, 128)
    last = torch.arange(pages - 4, pages, dtype=torch.int32, device="cuda")
    i = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    k = torch.randn(200, 256, device="cuda")
    q3q4.kv_write(cache, q3q4.KVBatch(i(0, 200), i(200), last[None], 200, 200, 200), k, k)
    weights = torch.empty(2, 2, 3 << 28, device="cuda")      # the last array starts at 9 * 2^28
    K = k.half().double().cpu().numpy().reshape(200, 2, 128).transpose(1, 0, 2)
    for rows in (60, 1):
        q = torch.randn(2 * rows, 512, device="cuda")
        batch = q3q4.KVBatch(i(0, rows, 2 * rows), i(200, 200), torch.stack([last, last]), 2 * rows, rows, 200)
        out = torch.empty_like(q)
        q3q4.attention_weights(cache, batch, q, out, 0.1, weights, workspace=q3q4.attention_weights_workspace(cache, batch, 4))
        for b in (0, 1):
            want, tol = so.weights_of(K, q[b * rows:(b + 1) * rows].double().cpu().numpy().reshape(rows, 4, 128), 200, 0.1, 0, 0)
            got = weights[b, :, :200].double().cpu().numpy()
            assert (np.abs(got - want) <= tol).all()
