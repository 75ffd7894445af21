"""sera_kv_write_rope on the GPU against the 64-bit oracle: row and cache types, head layouts, how many channels turn and
which together, norms, positions near and far, and what must not matter. Tolerances: step_oracle.heads_turned, and half a
step of the type that a value is held in.
"""
import numpy as np
import pytest

import attn_oracle as ao
import q3q4
import step_oracle as so
from test_gpu_attention import BF16, F16, F32, IDS, Setup, torch  # noqa: F401  (torch: the fixture)

pytestmark = pytest.mark.gpu


def freqs(n, base=10000.0):
    return (base ** (-np.arange(n, dtype=np.float64) / max(n, 1))).astype(np.float32)


def places(s, moved=None):
    """The position of every row: its place in the sequence, or another."""
    at = np.concatenate([np.arange(n - m, n) for m, n in zip(s.news, s.lens)] + [np.zeros(0)]).astype(np.int64)
    return at if moved is None else at + moved


def make(torch, s, rotated, pairing, norm_q=True, norm_k=True, eps=1e-6, seed=3):  # noqa: F811
    rng = np.random.default_rng(seed)
    f = freqs(rotated // 2) if rotated else None
    gq, gk = ((1 + 0.3 * rng.standard_normal(s.dim)).astype(np.float32) if x else None for x in (norm_q, norm_k))
    dev = lambda a: None if a is None else torch.from_numpy(a).cuda()  # noqa: E731
    return q3q4.Rope(dev(f), dev(gq), dev(gk), eps, pairing), (f, gq, gk, eps, pairing)


def close(got, want, tol, what):
    got = np.asarray(got, np.float64)
    off = np.abs(got - want)
    bad = ~(off <= tol) & ~(np.isnan(got) & np.isnan(want))
    print(f"  {what} worst {np.nanmax(off / np.where(tol > 0, tol, np.inf), initial=0):.3f} of the tolerance", flush=True)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size}, first at {np.argwhere(bad)[0]}: {got[bad][:4]} for {want[bad][:4]}"


def rounded(want, tol, io):
    return tol + (np.abs(want) + tol) * ao.HALF_STEP[IDS[io]] + (2.0 ** -25 if io == F16 else 0)


def check(torch, s, spec, q, q_out, k, v, before, positions=None):  # noqa: F811
    """q_out and the cache after a call against the oracle; k, v, q are the values given (float64)."""
    f, gq, gk, eps, pairing = spec
    at = places(s) if positions is None else np.asarray(positions)
    with np.errstate(all="ignore"):
        want, tol = so.heads_turned(q.reshape(s.rows, s.heads, s.dim), gq, eps, f, pairing, at)
        kw, kt = so.heads_turned(k.reshape(s.rows, s.kv_heads, s.dim), gk, eps, f, pairing, at)
    for b, n in enumerate(s.news):
        gone = max(n - s.lens[b], 0)                 # rows in front of the start
        want[s.starts[b]:s.starts[b] + gone] = tol[s.starts[b]:s.starts[b] + gone] = 0
    got = q_out.double().cpu().numpy().reshape(want.shape)
    close(got, want, rounded(want, tol, s.io), f"q {s.io}")
    pool = s.data.cpu().numpy().reshape(s.pool.shape)
    s.pool = before.copy()
    # V, and which bytes change, are those of a plain write
    ao.write(s.pool, s.kind, s.page, s.kv_heads, s.dim, s.table, s.starts, s.lens, np.zeros_like(k, np.float32), v.astype(np.float32))
    K, V, KS, VS = ao.views(pool, s.kind, s.page, s.kv_heads, s.dim)
    wk, wv, wks, wvs = s.views()
    assert np.array_equal(V, wv) and (VS is None or np.array_equal(VS, wvs, equal_nan=True)), "V differs from a plain write's"
    K64, tolerance, other = K.astype(np.float64), np.zeros(K.shape), wk.astype(np.float64)
    if KS is not None:
        K64, other = K64 * KS.astype(np.float64)[..., None], other * wks.astype(np.float64)[..., None]
    for b, n in enumerate(s.news):
        for i in range(n):
            j = s.lens[b] - n + i
            p = s.table[b][j // s.page] if j >= 0 else -1
            if 0 <= p < pool.shape[0]:
                r = s.starts[b] + i
                other[p, :, j % s.page] = kw[r]
                t = kt[r]
                if KS is None:
                    t = t + np.abs(kw[r]) * 2.0 ** -11 + 2.0 ** -25
                else:                               # half a step of the scale, which is the largest's 1 / 127
                    t = t + 0.5001 * (np.abs(kw[r]).max(-1) + t.max(-1))[:, None] / 127
                tolerance[p, :, j % s.page] = t
    close(K64, other, tolerance, f"K of cache {s.kind}")


def run(torch, s, rope, positions=None, q_scale=1.5):  # noqa: F811
    """One call; (q values, q_out, k values, v values, the pool before)."""
    cache, batch = s.device()
    before = s.pool.copy()
    (q, qv), (k, kv), (v, vv) = s.rows_of(s.heads * s.dim, q_scale), s.rows_of(s.kv_heads * s.dim, 3.0), s.rows_of(s.kv_heads * s.dim)
    out = torch.full_like(q, 7.0)
    at = None if positions is None else torch.tensor(np.asarray(positions), dtype=torch.int32, device="cuda")
    q3q4.kv_write_rope(cache, batch, rope, q, out, k, v, at)
    torch.cuda.synchronize()
    return qv, out, kv, vv, before


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("io", [F32, F16, BF16])
@pytest.mark.parametrize("dim,page", [(64, 32), (128, 16), (128, 64)])
@pytest.mark.parametrize("share", [1, 2, 4])
@pytest.mark.parametrize("pairing", [so.HALVES, so.NEIGHBOURS])
def test_types_and_turns(torch, kind, io, dim, page, share, pairing):  # noqa: F811
    print(f"case kind={kind} io={io} dim={dim} page={page} 1/{share} pairing={pairing}", flush=True)
    s = Setup(torch, kind, io, [1, 37, 0, 16, 5, 64, 2], [1, 50, 9, 48, 3, 64, 700], heads=6, kv_heads=2, dim=dim, page=page)
    rope, spec = make(torch, s, dim // share, pairing)
    check(torch, s, spec, *run(torch, s, rope))


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (5, 1), (64, 8), (40, 4)])
@pytest.mark.parametrize("norm_q,norm_k", [(True, False), (False, True), (False, False)])
def test_heads_and_norms(torch, heads, kv_heads, norm_q, norm_k):  # noqa: F811
    print(f"case heads={heads} kv_heads={kv_heads} norms {norm_q} {norm_k}", flush=True)
    s = Setup(torch, ao.F16, F32, [1, 1, 20], [33, 16, 21], heads=heads, kv_heads=kv_heads)
    rope, spec = make(torch, s, 128, so.HALVES, norm_q, norm_k)
    check(torch, s, spec, *run(torch, s, rope))


@pytest.mark.parametrize("moved", [0, 5000, 3000017, (1 << 28) - 100, -60])
def test_positions_apart_from_the_cache_s(torch, moved):  # noqa: F811
    """Rows that are rotated by other positions than their places in the cache, far ones and negative ones among them."""
    s = Setup(torch, ao.F16, F32, [3, 30], [80, 30], heads=4, kv_heads=2)
    rope, spec = make(torch, s, 128, so.HALVES, norm_q=False)
    at = places(s, moved)
    check(torch, s, spec, *run(torch, s, rope, at), positions=at)


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("io", [F32, BF16])
def test_nothing_to_do_is_a_plain_write(torch, kind, io):  # noqa: F811
    s = Setup(torch, kind, io, [9, 1], [40, 17], heads=4, kv_heads=2)
    cache, batch = s.device()
    (q, _), (k, _), (v, _) = s.rows_of(512), s.rows_of(256), s.rows_of(256)
    out = torch.empty_like(q)
    q3q4.kv_write_rope(cache, batch, q3q4.Rope(), q, out, k, v)
    data = cache.data.clone()
    assert torch.equal(out, q)
    q3q4.kv_write(cache, batch, k, v)
    assert torch.equal(cache.data, data)


def test_values_without_a_size(torch):  # noqa: F811
    """Zero heads stay zero (eps keeps the norm finite), heads with an infinity or NaN come out not finite, alone."""
    s = Setup(torch, ao.F16, F32, [6], [6], heads=2, kv_heads=1)
    rope, _ = make(torch, s, 128, so.HALVES)
    cache, batch = s.device()
    q, k = torch.randn(6, 256, device="cuda"), torch.randn(6, 128, device="cuda")
    q[0, :128] = 0
    q[1, 5], q[2, 130] = float("inf"), float("nan")
    k[3] = 0
    out = torch.empty_like(q)
    q3q4.kv_write_rope(cache, batch, rope, q, out, k, k)
    ko, vo = torch.empty_like(k), torch.empty_like(k)
    q3q4.kv_read(cache, batch, ko, vo)
    assert (out[0, :128] == 0).all() and (ko[3] == 0).all() and torch.isfinite(ko).all()
    odd = ~torch.isfinite(out).view(6, 2, 128).all(-1)
    assert odd.nonzero().tolist() == [[1, 0], [2, 1]]


def test_in_place_and_out_of_a_fused_buffer(torch):  # noqa: F811
    """q, k and v as columns of one buffer, q turned where it stands: the other columns stay."""
    for pairing in (so.HALVES, so.NEIGHBOURS):
        s = Setup(torch, ao.F16, F32, [7, 30], [40, 30], heads=6, kv_heads=3, dim=64, page=32)
        rope, spec = make(torch, s, 64, pairing)
        cache, batch = s.device()
        before = s.pool.copy()
        buf = torch.randn(s.rows, (6 + 3 + 3) * 64 + 20, device="cuda")
        was = buf.clone()
        q3q4.kv_write_rope(cache, batch, rope, buf[:, :384], buf[:, :384], buf[:, 384:576], buf[:, 576:768])
        torch.cuda.synchronize()
        assert torch.equal(buf[:, 384:], was[:, 384:])
        w = was.double().cpu().numpy()
        check(torch, s, spec, w[:, :384], buf[:, :384], w[:, 384:576], w[:, 576:768], before)


@pytest.mark.parametrize("rows,heads,kv_heads", [(3000, 24, 8), (1777, 40, 10)])
def test_several_heads_a_workgroup(torch, rows, heads, kv_heads):  # noqa: F811
    """Enough rows that a wave turns several heads, the last workgroup of a block fewer, and some q's heads and k's."""
    print(f"case {rows} rows {heads} over {kv_heads} heads", flush=True)
    s = Setup(torch, ao.F16, BF16, [rows, 5], [rows + 30, 5], heads=heads, kv_heads=kv_heads, dim=64, page=64)
    rope, spec = make(torch, s, 64, so.HALVES)
    check(torch, s, spec, *run(torch, s, rope))


def test_many_sequences(torch):  # noqa: F811
    rng = np.random.default_rng(1)
    news = [int(n) for n in rng.integers(0, 4, 300)]
    lens = [n + int(x) for n, x in zip(news, rng.integers(0, 40, 300))]
    s = Setup(torch, ao.Q8, F32, news, lens, heads=2, kv_heads=1, dim=64)
    rope, spec = make(torch, s, 32, so.HALVES)
    check(torch, s, spec, *run(torch, s, rope))


def test_rows_behind_the_last_sequence_stay(torch):  # noqa: F811
    s = Setup(torch, ao.F16, F32, [4, 3], [20, 3], heads=2, kv_heads=1)
    cache, _ = s.device()
    i = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    batch = q3q4.KVBatch(i(1, 5, 8), i(20, 3), i(*s.table[0], *s.table[1]).view(2, -1), 12, 4, 20)
    rope, spec = make(torch, s, 128, so.HALVES)
    q, k = torch.randn(12, 256, device="cuda"), torch.randn(12, 128, device="cuda")
    out = torch.full_like(q, 7.0)
    q3q4.kv_write_rope(cache, batch, rope, q, out, k, k)
    assert (out[0] == 7.0).all() and (out[8:] == 7.0).all() and not (out[1:8] == 7.0).any()


@pytest.mark.parametrize("starts,lens", [([0, 2, 4], [20, 301]), ([0, 2, 4], [-1, 20]), ([0, 4, 4], [20, 20]), ([1, 2, 900], [20, 20]),
                                         ([0, 4, 2], [20, 20])])
def test_batches_outside_the_bounds(torch, starts, lens):  # noqa: F811
    """Sequences that break the host's bounds (4 rows, 3 at most each, 300 positions) write nothing, their q rows are NaN."""
    s = Setup(torch, ao.F16, F32, [2, 2], [300, 300], heads=4, kv_heads=2)
    cache, _ = s.device()
    i = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    batch = q3q4.KVBatch(i(starts), i(lens), i(s.table), 4, 3, 300)
    ok = [0 <= starts[b] <= starts[b + 1] <= 4 and starts[b + 1] - starts[b] <= 3 and 0 <= lens[b] <= 300 for b in (0, 1)]
    rope, _ = make(torch, s, 128, so.HALVES)
    q, k = torch.randn(4, 512, device="cuda"), torch.randn(4, 256, device="cuda")
    out = torch.full((8, 512), 7.0, device="cuda")
    q3q4.kv_write_rope(cache, batch, rope, q, out[:4], k, k)
    torch.cuda.synchronize()
    assert (out[4:] == 7.0).all()
    changed = (s.data.cpu().numpy().reshape(s.pool.shape) != s.pool).any((1, 2))
    for b in (0, 1):
        if not ok[b]:
            assert not changed[s.table[b]].any()
            if starts[b] <= starts[b + 1]:
                assert torch.isnan(out[max(starts[b], 0):min(starts[b + 1], 4)]).all()
        elif starts == sorted(starts):
            assert torch.isfinite(out[starts[b]:starts[b + 1]]).all()


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("entry", [-1, 1 << 20])
def test_bad_pages_are_not_written(torch, kind, entry):  # noqa: F811
    """Tokens of a page outside the pool are not written; q is turned all the same."""
    s = Setup(torch, kind, F32, [40], [150], heads=4, kv_heads=2)
    s.table[0, 8] = entry
    rope, spec = make(torch, s, 128, so.HALVES)
    check(torch, s, spec, *run(torch, s, rope))


def test_graph_replays_and_streams(torch):  # noqa: F811
    """Captured once; lengths, positions and rows change between replays. The same on another stream, bit for bit."""
    s = Setup(torch, ao.F16, F32, [1, 1], [40, 200], heads=4, kv_heads=2)
    cache, batch = s.device(max_kv=208)
    rope, spec = make(torch, s, 128, so.HALVES)
    q, k, v = (torch.randn(2, n, device="cuda") for n in (512, 256, 256))
    at, out = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros_like(q)

    def step():
        q3q4.kv_write_rope(cache, batch, rope, q, out, k, v, at)

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for lens in ([40, 200], [41, 199], [1, 16]):
        for t in (q, k, v):
            t.copy_(torch.randn_like(t))
        at.copy_(torch.tensor([n * 7 for n in lens]))
        s.lens = lens
        batch.kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
        before = s.data.cpu().numpy().reshape(s.pool.shape).copy()
        out.fill_(5.0)
        g.replay()
        torch.cuda.synchronize()
        check(torch, s, spec, *(t.double().cpu().numpy() if t is not out else t for t in (q, out, k, v)), before,
              positions=[n * 7 for n in lens])
        first, data = out.clone(), cache.data.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        q3q4.kv_write_rope(cache, batch, rope, q, out, k, v, at, stream=side)
        side.synchronize()
        assert torch.equal(out, first) and torch.equal(cache.data, data)


def test_rows_more_than_two_to_the_31_elements_apart(torch):  # noqa: F811
    """Four rows 3 * 2^28 elements apart, the last 2.4e9 from the first, as q in and out, keys and values."""
    stride, width = 3 << 28, 256
    buf = torch.empty(3 * stride + 4 * width, device="cuda")
    far = [buf.as_strided((4, width), (stride, 1), width * i) for i in range(4)]
    for f in far:
        f.copy_(torch.randn(4, width, device="cuda"))
    near = [f.clone() for f in far]
    out = torch.empty_like(near[0])
    s = Setup(torch, ao.F16, F32, [4], [4], heads=2, kv_heads=2)
    rope, _ = make(torch, s, 128, so.HALVES)
    cache, batch = s.device()
    q3q4.kv_write_rope(cache, batch, rope, far[0], far[1], far[2], far[3])
    data = cache.data.clone()
    q3q4.kv_write_rope(cache, batch, rope, near[0], out, near[2], near[3])
    assert torch.equal(far[1], out) and torch.equal(cache.data, data) and torch.equal(far[2], near[2])
