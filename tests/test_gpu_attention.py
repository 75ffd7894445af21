"""Paged cache and attention on the GPU against the 64-bit oracle: cache
types, row types, head layouts, lengths from one token to thousands, pages
that end inside a tile, windows and sinks, and what must not matter: values in
places that a row does not see, order, strides, streams, graphs.

Writes are bit-exact (codes, scales and fp16 bits), reads are the product in
fp32 rounded to the row type. Attention's tolerance is derived in attn_oracle.attend.
"""
import numpy as np
import pytest

import attn_oracle as ao
import q3q4

pytestmark = pytest.mark.gpu
F32, F16, BF16 = "float32", "float16", "bfloat16"
IDS = {F32: ao.F32T, F16: ao.F16T, BF16: ao.BF16T}


@pytest.fixture(scope="module")
def torch():
    import torch as _t
    if not _t.cuda.is_available():
        pytest.fail("gpu test without a visible HIP device")
    q3q4.load()
    return _t


class Setup:
    """A cache whose pages hold random values, and a batch over it, on both sides."""

    def __init__(self, torch, kind, io, news, lens, heads=8, kv_heads=2, dim=128, page=16, seed=0, spare=2, shared=0):
        rng = self.rng = np.random.default_rng(seed)
        self.torch, self.kind, self.io, self.news, self.lens = torch, kind, io, news, lens
        self.heads, self.kv_heads, self.dim, self.page = heads, kv_heads, dim, page
        self.starts = [0] + list(np.cumsum(news))
        self.rows, width = self.starts[-1], max(1, -(-max(lens) // page))
        own = width - shared
        pages = shared + own * len(news) + spare
        order = rng.permutation(pages)
        self.table = np.empty((len(news), width), np.int32)
        self.table[:, :shared] = order[:shared]
        self.table[:, shared:] = order[shared:shared + own * len(news)].reshape(len(news), own)
        self.pool = np.zeros((pages, kv_heads, ao.head_bytes(kind, page, dim)), np.uint8)
        k, v, ks, vs = self.views()
        if kind == ao.F16:
            k[:] = rng.standard_normal(k.shape).astype(np.float16)
            v[:] = rng.standard_normal(v.shape).astype(np.float16)
        else:
            k[:] = rng.integers(-127, 128, k.shape)
            v[:] = rng.integers(-127, 128, v.shape)
            ks[:] = np.exp(rng.standard_normal(ks.shape)) / 80
            vs[:] = np.exp(2 * rng.standard_normal(vs.shape)) / 80

    def views(self):
        return ao.views(self.pool, self.kind, self.page, self.kv_heads, self.dim)

    def rows_of(self, width, scale=1.0):
        """(device rows of the io type, the values they hold in float64)"""
        x = self.torch.from_numpy((self.rng.standard_normal((self.rows, width)) * scale).astype(np.float32))
        x = x.to(getattr(self.torch, self.io)).cuda()
        return x, x.double().cpu().numpy()

    def device(self, max_new=None, max_kv=None):
        t = self.torch
        i = lambda a: t.tensor(np.asarray(a, dtype=np.int32), device="cuda")  # noqa: E731
        self.data = t.from_numpy(self.pool.reshape(-1)).cuda()
        self.cache = q3q4.KVCache(self.kind, self.pool.shape[0], self.page, self.kv_heads, self.dim, self.data)
        self.batch = q3q4.KVBatch(i(self.starts), i(self.lens), i(self.table), self.rows, max_new or max(self.news),
                                  max_kv or max(max(self.lens), 1))
        return self.cache, self.batch

    def expect(self, q, scale, window=0, sinks=0):
        q = q.reshape(self.rows, self.heads, self.dim)
        o, tol = np.zeros(q.shape), np.zeros(q.shape)
        for b, n in enumerate(self.news):
            if n:
                K, V = ao.values(self.pool, self.kind, self.page, self.kv_heads, self.dim, self.table, b,
                                 self.lens[b])
                at = slice(self.starts[b], self.starts[b] + n)
                o[at], tol[at] = ao.attend(K, V, q[at], self.lens[b], scale, window, sinks, IDS[self.io])
        return o.reshape(self.rows, -1), tol.reshape(self.rows, -1)

    def attend(self, q, scale, window=0, sinks=0, **bounds):
        self.device(**bounds)
        out = self.torch.full_like(q, 7.0)
        ws = q3q4.attention_workspace(self.cache, self.batch, self.heads)
        if ws is not None:
            ws.fill_(0xFF)           # NaN everywhere: its content does not matter
        q3q4.attention(self.cache, self.batch, q, out, scale, window, sinks, workspace=ws)
        self.torch.cuda.synchronize()
        return out


def close(out, want, tol, what=""):
    got = out.double().cpu().numpy()
    bad = ~(np.abs(got - want) <= tol) & ~(np.isnan(got) & np.isnan(want))
    worst = np.nanmax(np.where(tol > 0, np.abs(got - want) / np.where(tol > 0, tol, 1), 0)) if got.size else 0
    print(f"  {what} worst {worst:.3f} of the tolerance", flush=True)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, first at {np.argwhere(bad)[0]}: " \
        f"{got[bad][:4]} for {want[bad][:4]}"


def check(s, scale=None, window=0, sinks=0, q_scale=1.5, **bounds):
    scale = s.dim ** -0.5 if scale is None else scale
    q, qv = s.rows_of(s.heads * s.dim, q_scale)
    want, tol = s.expect(qv, scale, window, sinks)
    out = s.attend(q, scale, window, sinks, **bounds)
    close(out, want, tol, f"{s.io} {s.news} of {s.lens}")
    return q, out


# ---- write and read ---------------------------------------------------------

@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("io", [F32, F16, BF16])
@pytest.mark.parametrize("kv_heads,dim,page", [(2, 128, 16), (5, 64, 32), (1, 128, 64)])
def test_write_and_read_back(torch, kind, io, kv_heads, dim, page):
    print(f"case write kind={kind} io={io} kv_heads={kv_heads} dim={dim} page={page}", flush=True)
    s = Setup(torch, kind, io, [1, 37, 0, 16, 5, 64], [1, 50, 9, 48, 3, 64], kv_heads=kv_heads, dim=dim, page=page)
    cache, batch = s.device()
    (k, kv), (v, vv) = s.rows_of(kv_heads * dim), s.rows_of(kv_heads * dim, 30.0)
    q3q4.kv_write(cache, batch, k, v)
    ko, vo = torch.full_like(k, 7.0), torch.full_like(v, 7.0)
    q3q4.kv_read(cache, batch, ko, vo)
    torch.cuda.synchronize()
    ao.write(s.pool, kind, page, kv_heads, dim, s.table, s.starts, s.lens, kv.astype(np.float32),
             vv.astype(np.float32))
    assert np.array_equal(s.data.cpu().numpy(), s.pool.reshape(-1)), "cache bytes differ from the oracle's"
    for b, n in enumerate(s.news):
        got = ao.values(s.pool, kind, page, kv_heads, dim, s.table, b, s.lens[b])
        for x, o in zip(got, (ko, vo)):
            m = min(n, s.lens[b])                     # rows in front of the start read as zeros
            want = np.zeros((n, kv_heads * dim), np.float32)
            want[n - m:] = x[:, s.lens[b] - m:].transpose(1, 0, 2).reshape(m, kv_heads * dim)
            w = torch.from_numpy(want).to(getattr(torch, io))
            assert torch.equal(o[s.starts[b]:s.starts[b + 1]].cpu(), w), f"sequence {b}"


def test_quantizer_borders(torch):
    """Vectors whose elements lie on and next to half steps, tiny, zero, huge and non-finite vectors."""
    rng = np.random.default_rng(9)
    n, dim = 96, 128
    k = np.zeros((n, dim), np.float32)
    for r in range(n):
        d = np.float32(rng.uniform(0.5, 2) * 2.0 ** rng.integers(-20, 20))
        x = (rng.integers(-127, 127, dim) + 0.5).astype(np.float64) * np.float64(d)
        x = x.astype(np.float32)
        x = np.where(rng.random(dim) < 0.3, np.nextafter(x, np.float32(0)), x)
        x[rng.integers(dim)] = np.float32(127) * d
        k[r] = x
    k[0], k[1, 1:], k[2], k[3] = 0, 0, 1e-44, k[3] * np.float32(1e-30)
    k[4, 5], k[5, 6], k[6, 0] = np.inf, np.nan, 3.4e38
    k[7] = (rng.integers(-300, 300, dim) * np.float64(2.0 ** -149)).astype(np.float32)   # denormals
    k[8] = (rng.standard_normal(dim) * 1e-36).astype(np.float32)
    s = Setup(torch, ao.Q8, F32, [n], [n], kv_heads=1)
    cache, batch = s.device()
    kd = torch.from_numpy(k).cuda()
    q3q4.kv_write(cache, batch, kd, kd.flip(0))
    torch.cuda.synchronize()
    ao.write(s.pool, ao.Q8, 16, 1, dim, s.table, [0, n], [n], k, k[::-1])
    got = ao.views(s.data.cpu().numpy().reshape(s.pool.shape), ao.Q8, 16, 1, dim)
    for g, w, name in zip(got, s.views(), ("K", "V", "K scale", "V scale")):
        assert np.array_equal(g, w, equal_nan=g.dtype == np.float32), name
    ko, vo = torch.empty_like(kd), torch.empty_like(kd)
    q3q4.kv_read(cache, batch, ko, vo)
    assert torch.isnan(ko[4:6]).all() and torch.isnan(vo[n - 6:n - 4]).all()
    assert torch.isfinite(ko[6]).all() and (ko[0] == 0).all()


def test_fp16_cache_keeps_infinities_and_rounds_over_its_range(torch):
    s = Setup(torch, ao.F16, F32, [16], [16], kv_heads=1)
    cache, batch = s.device()
    k = torch.zeros(16, 128, device="cuda")
    k[0, :4] = torch.tensor([65519.0, 65520.0, -1e9, float("inf")])
    k[1, 0] = float("nan")
    q3q4.kv_write(cache, batch, k, k)
    ko, vo = torch.empty_like(k), torch.empty_like(k)
    q3q4.kv_read(cache, batch, ko, vo)
    for o in (ko, vo):
        assert o[0, :4].tolist() == [65504.0, float("inf"), float("-inf"), float("inf")] and torch.isnan(o[1, 0])


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
def test_strided_rows_out_of_a_fused_buffer(torch, kind):
    """k, v and q as columns of one buffer, out as columns of another."""
    s = Setup(torch, kind, F32, [7, 30], [40, 30], heads=6, kv_heads=3, dim=64, page=32)
    cache, batch = s.device()
    buf = torch.randn(s.rows, (6 + 3 + 3) * 64 + 20, device="cuda")
    q, k, v = buf[:, :384], buf[:, 384:576], buf[:, 576:768]
    q3q4.kv_write(cache, batch, k, v)
    big = torch.full((s.rows, 384 + 64), 7.0, device="cuda")
    ws = q3q4.attention_workspace(cache, batch, 6)
    q3q4.attention(cache, batch, q, big[:, 32:416], 0.125, workspace=ws)
    back = torch.full((s.rows, 2 * 192 + 8), 7.0, device="cuda")
    q3q4.kv_read(cache, batch, back[:, :192], back[:, 196:388])
    torch.cuda.synchronize()
    ao.write(s.pool, kind, 32, 3, 64, s.table, s.starts, s.lens, k.cpu().numpy(), v.cpu().numpy())
    assert np.array_equal(s.data.cpu().numpy(), s.pool.reshape(-1))
    want, tol = s.expect(q.double().cpu().numpy(), 0.125)
    close(big[:, 32:416], want, tol, "strided")
    for t, cols in ((big, (slice(0, 32), slice(416, 448))), (back, (slice(192, 196), slice(388, 392)))):
        for c in cols:
            assert (t[:, c] == 7.0).all(), "columns beside the operand were written"


# ---- attention: sizes -------------------------------------------------------

@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("io", [F32, F16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
def test_decode_ragged(torch, kind, io, dim):
    print(f"case decode kind={kind} io={io} dim={dim}", flush=True)
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 127, 300, 513, 1000]
    check(Setup(torch, kind, io, [1] * len(lens), lens, heads=16, kv_heads=2, dim=dim, page=32, seed=dim))


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("io", [F32, BF16])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (5, 1), (12, 4), (16, 1), (40, 2)])
def test_decode_head_layouts(torch, kind, io, heads, kv_heads):
    print(f"case heads={heads} kv_heads={kv_heads} kind={kind} io={io}", flush=True)
    check(Setup(torch, kind, io, [1, 2], [70, 201], heads=heads, kv_heads=kv_heads, seed=heads))


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("io", [F32, F16, BF16])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 16), (128, 64), (128, 128)])
def test_chunks_ragged(torch, kind, io, dim, page):
    print(f"case chunks kind={kind} io={io} dim={dim} page={page}", flush=True)
    check(Setup(torch, kind, io, [1, 5, 0, 33, 64, 100, 17], [90, 5, 7, 200, 64, 131, 17], heads=8, kv_heads=2, dim=dim,
                page=page, seed=page))


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("group", [1, 3, 5, 8, 20])
def test_chunk_groups(torch, kind, group):
    print(f"case chunk group={group} kind={kind}", flush=True)
    check(Setup(torch, kind, F32, [37, 70], [37, 150], heads=2 * group, kv_heads=2, page=16, seed=group))


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("news,lens", [([1], [5000]), ([3], [4999]), ([40], [3001]), ([1, 1], [9001, 20])])
def test_long_contexts_are_split(torch, kind, news, lens):
    print(f"case split {news} of {lens} kind={kind}", flush=True)
    check(Setup(torch, kind, F32, news, lens, heads=8, kv_heads=1, page=64, seed=sum(lens)))


@pytest.mark.parametrize("max_kv", [301, 4096, 100000])
def test_loose_bounds(torch, max_kv):
    """The host's bounds may be far above the lengths that the device has (a graph captured for later lengths)."""
    s = Setup(torch, ao.F16, F32, [1, 2, 1], [300, 17, 301], heads=8, kv_heads=2, page=16)
    wide = np.full((3, -(-max_kv // 16)), -5, np.int32)
    wide[:, :s.table.shape[1]] = s.table
    s.table = wide
    check(s, max_kv=max_kv, max_new=4)


def test_many_sequences(torch):
    """More sequences than one level of the lookup holds, empty ones among them."""
    rng = np.random.default_rng(1)
    news = [int(n) for n in rng.integers(0, 4, 300)]
    lens = [n + int(x) for n, x in zip(news, rng.integers(0, 40, 300))]
    check(Setup(torch, ao.F16, F32, news, lens, heads=2, kv_heads=1, dim=64))
    news[150] = 60
    lens[150] += 60
    check(Setup(torch, ao.Q8, F32, news, lens, heads=2, kv_heads=1, dim=64))


def test_shared_prefix(torch):
    check(Setup(torch, ao.F16, F32, [9, 3, 1, 20], [73, 67, 65, 84], heads=16, kv_heads=2, page=16, shared=4))


# ---- windows, sinks, empty rows ---------------------------------------------

@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 0), (50, 4), (64, 64), (100, 33), (7, 1000), (5000, 3)])
@pytest.mark.parametrize("news,lens", [([1, 1, 2], [700, 31, 90]), ([70, 9], [300, 400])])
def test_window_and_sinks(torch, kind, window, sinks, news, lens):
    print(f"case window={window} sinks={sinks} {news} of {lens} kind={kind}", flush=True)
    check(Setup(torch, kind, F32, news, lens, heads=8, kv_heads=2, page=16, seed=window + sinks), window=window,
          sinks=sinks)


def test_window_over_a_split_context(torch):
    check(Setup(torch, ao.F16, F32, [1, 2], [9000, 8000], heads=8, kv_heads=1, page=64), window=5000, sinks=70)
    check(Setup(torch, ao.Q8, BF16, [1], [12000], heads=4, kv_heads=1, page=64), window=64, sinks=4)


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("news,lens", [([3, 2], [1, 0]), ([50, 20], [7, 40])])
def test_rows_that_see_nothing_are_zero(torch, kind, news, lens):
    """More rows than positions: the first ones lie in front of the sequence."""
    s = Setup(torch, kind, F32, news, lens, heads=8, kv_heads=2)
    q, out = check(s)
    gone = news[0] - lens[0]
    assert (out[:gone] == 0).all() and not (out[gone] == 0).all()


def test_no_sequence_has_rows(torch):
    """rows = 0 launches nothing; sequences without rows leave the others alone."""
    s = Setup(torch, ao.F16, F32, [0, 4, 0], [33, 20, 0], heads=8, kv_heads=2)
    check(s)
    b = q3q4.KVBatch(s.batch.row_start[:1], s.batch.kv_len[:0], s.batch.page_table[:0], 0, 1, 1)
    e = torch.empty(0, 1024, device="cuda")
    q3q4.attention(s.cache, b, e, e, 0.1)
    q3q4.kv_write(s.cache, b, e[:, :256], e[:, :256])


# ---- what must not matter ----------------------------------------------------

def spoil(s, b, positions, value):
    """`value` in every K, V and scale of these positions of sequence b."""
    k, v, ks, vs = s.views()
    for j in positions:
        p, o = s.table[b][j // s.page], j % s.page
        if s.kind == ao.F16:
            k[p, :, o], v[p, :, o // 16, :, o % 16] = value, value
        else:
            ks[p, :, o], vs[p, :, o] = value, value


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("new", [1, 40])
def test_nothing_behind_the_end_matters(torch, kind, value, new):
    s = Setup(torch, kind, F32, [new], [75], heads=8, kv_heads=2, page=64)
    spoil(s, 0, range(75, 128), value)
    _, out = check(s)
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("value", [np.nan, np.inf])
@pytest.mark.parametrize("io", [F32, BF16])
def test_masked_positions_do_not_matter(torch, kind, value, io):
    """Non-finite keys and values at positions that some rows see and others do not: the first stay finite."""
    s = Setup(torch, kind, io, [60], [100], heads=8, kv_heads=2, page=16)
    spoil(s, 0, [97], value)                       # seen by the last three rows only
    q, qv = s.rows_of(s.heads * s.dim)
    want, tol = s.expect(qv, 0.1)
    out = s.attend(q, 0.1)
    close(out[:57], want[:57], tol[:57], "rows in front")
    assert torch.isnan(out[57:]).any(1).all()
    s = Setup(torch, kind, io, [60], [100], heads=8, kv_heads=2, page=16)
    spoil(s, 0, [30, 62], value)                   # out of every window, and in those of rows 22 .. 31
    want, tol = s.expect(qv, 0.1, 10, 3)
    out = s.attend(q, 0.1, 10, 3)
    seen = np.zeros(60, bool)
    seen[22:32] = True
    close(out[torch.from_numpy(~seen).cuda()], want[~seen], tol[~seen], "windows")
    assert torch.isnan(out[torch.from_numpy(seen).cuda()]).any(1).all()


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("new", [1, 2])
def test_masked_positions_of_a_split_decode(torch, kind, new):
    s = Setup(torch, kind, F32, [new, new], [6000, 5000], heads=8, kv_heads=1, page=64)
    spoil(s, 0, [100, 5000, 5898], np.nan)
    _, out = check(s, window=100, sinks=70)
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("news,lens", [([1], [200]), ([64], [200])])
def test_peaked_and_flat_scores(torch, kind, news, lens):
    """Scores far apart (one weight of 1, the rest nothing), and all equal."""
    check(Setup(torch, kind, F32, news, lens, heads=8, kv_heads=2), scale=3.0, q_scale=4.0)
    s = Setup(torch, kind, F32, news, lens, heads=8, kv_heads=2)
    check(s, q_scale=0.0)
    check(s, scale=0.0)
    check(s, scale=-0.2)
    check(s, q_scale=1e-20, scale=1e19)
    check(s, q_scale=1e15, scale=1e-16)


@pytest.mark.parametrize("new", [1, 50])
def test_growing_scores(torch, new):
    """Every tile raises the running maximum, by little and by much."""
    for step in (0.01, 0.3, 20.0):
        s = Setup(torch, ao.F16, F32, [new], [900], heads=8, kv_heads=1, page=64)
        k, _, _, _ = s.views()
        for j in range(900):
            k[s.table[0][j // 64], :, j % 64] = np.float16(step * j / 128)
        q = torch.full((new, 1024), 0.25, device="cuda")
        want, tol = s.expect(q.double().cpu().numpy(), 0.3)
        close(s.attend(q, 0.3), want, tol, f"step {step}")


@pytest.mark.parametrize("new", [1, 50])
def test_value_scales_far_apart(torch, new):
    """8-bit values whose scales span 24 binades up, down and mixed."""
    for order in (1, -1, 0):
        s = Setup(torch, ao.Q8, F32, [new], [700], heads=8, kv_heads=1, page=64)
        _, _, _, vs = s.views()
        e = np.linspace(-12, 12, 700)[::order] if order else s.rng.uniform(-12, 12, 700)
        for j in range(700):
            vs[s.table[0][j // 64], :, j % 64] = np.float32(2.0 ** e[j])
        check(s)


def test_results_repeat_and_follow_no_order(torch):
    """Bit-identical on a second run, on other page ids and on another stream."""
    for kind, news, lens in ((ao.F16, [1, 1], [3000, 200]), (ao.Q8, [40, 3], [600, 64])):
        s = Setup(torch, kind, F32, news, lens, heads=8, kv_heads=2, page=32)
        q, first = check(s)
        assert torch.equal(s.attend(q, s.dim ** -0.5), first)
        perm = np.random.default_rng(5).permutation(s.pool.shape[0])
        s.pool, s.table = s.pool[perm], np.argsort(perm)[s.table].astype(np.int32)
        assert torch.equal(s.attend(q, s.dim ** -0.5), first)
        side, out = torch.cuda.Stream(), torch.zeros_like(q)
        ws = q3q4.attention_workspace(s.cache, s.batch, s.heads)
        torch.cuda.synchronize()
        q3q4.attention(s.cache, s.batch, q, out, s.dim ** -0.5, workspace=ws, stream=side)
        side.synchronize()
        assert torch.equal(out, first)


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("new", [1, 30])
def test_graph_replays_take_the_lengths_of_their_time(torch, kind, new):
    """Write, attention and read captured once; lengths, tables and rows change between replays."""
    s = Setup(torch, kind, F32, [new, new], [40, 2000], heads=8, kv_heads=2, page=16)
    cache, batch = s.device(max_kv=2048 if s.table.shape[1] * 16 >= 2048 else s.table.shape[1] * 16)
    k, v = (torch.randn(s.rows, 256, device="cuda") for _ in "kv")
    q = torch.randn(s.rows, 1024, device="cuda")
    out, ko, vo = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    ws = q3q4.attention_workspace(cache, batch, 8)

    def step():
        q3q4.kv_write(cache, batch, k, v)
        q3q4.attention(cache, batch, q, out, 0.1, workspace=ws)
        q3q4.kv_read(cache, batch, ko, vo)

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for lens in ([40, 2000], [41, 1999], [33, 700], [1500, 64]):
        for t in (k, v, q):
            t.copy_(torch.randn_like(t))
        s.lens = lens
        batch.kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
        out.fill_(5.0)
        g.replay()
        torch.cuda.synchronize()
        s.pool = s.data.cpu().numpy().reshape(s.pool.shape)
        want, tol = s.expect(q.double().cpu().numpy(), 0.1)
        close(out, want, tol, f"replay at {lens}")
        replayed = [t.clone() for t in (out, ko, vo)]
        step()
        for a, b in zip(replayed, (out, ko, vo)):
            assert torch.equal(a, b)


def test_offsets_past_32_bits(torch):
    """Pages at the end of a pool of more than 4 GiB, rows more than 2^31 elements from the first."""
    page, kv_heads = 64, 8
    page_bytes = q3q4.kv_page_bytes(ao.F16, page, kv_heads, 128)
    pages = (9 << 29) // page_bytes
    cache = q3q4.KVCache(ao.F16, pages, page, kv_heads, 128)
    last = torch.arange(pages - 4, pages, dtype=torch.int32, device="cuda")
    i = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    k, v, q = torch.randn(200, 1024, device="cuda"), torch.randn(200, 1024, device="cuda"), None
    for rows in (200, 1):
        batch = q3q4.KVBatch(i(0, rows), i(200), last[None], rows, rows, 200)
        if rows == 200:
            q3q4.kv_write(cache, batch, k, v)
        q = torch.randn(rows, 1024, device="cuda")
        out = torch.empty_like(q)
        q3q4.attention(cache, batch, q, out, 0.1, workspace=q3q4.attention_workspace(cache, batch, 8))
        K, V = (t.half().double().cpu().numpy().reshape(200, 8, 128).transpose(1, 0, 2) for t in (k, v))
        want, tol = ao.attend(K, V, q.double().cpu().numpy().reshape(rows, 8, 128), 200, 0.1, 0, 0, ao.F32T)
        close(out, want.reshape(rows, -1), tol.reshape(rows, -1), f"{rows} rows")
    del cache
    far = torch.empty(5 << 29, device="cuda")          # 5 * 2^29 elements: rows 2^29 + 2^27 apart
    stride = (1 << 29) + (1 << 27)
    rows = far.as_strided((4, 1024), (stride, 1), 0)
    rows.copy_(torch.randn(4, 1024, device="cuda"))
    cache = q3q4.KVCache(ao.F16, 1, 16, 8, 128)
    batch = q3q4.KVBatch(i(0, 4), i(4), i(0)[None], 4, 4, 16)
    q3q4.kv_write(cache, batch, rows, rows)
    ko, vo = torch.empty(4, 1024, device="cuda"), torch.empty(4, 1024, device="cuda")
    q3q4.kv_read(cache, batch, ko, vo)
    assert torch.equal(ko, rows.half().float()) and torch.equal(vo, ko)


# ---- what the host cannot check ----------------------------------------------

@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("entry", [-1, 1 << 20, -(1 << 31)])
def test_bad_pages_are_not_followed(torch, kind, new, entry):
    """A page id outside the pool: rows that see its tokens are NaN, others are right, nothing is written."""
    s = Setup(torch, kind, F32, [new, new], [150, 150], heads=8, kv_heads=2, page=16)
    s.table[0, 4] = entry                                    # positions 64 .. 79
    s.table[1, 8] = entry                                    # 128 .. 143
    q, qv = s.rows_of(1024)
    want, tol = s.expect(qv, 0.1)
    out = s.attend(q, 0.1)
    close(out, want, tol, "bad pages")
    assert torch.isnan(out[:new]).all()
    want, tol = s.expect(qv, 0.1, 5, 0)                      # out of every window of sequence 0
    out = s.attend(q, 0.1, 5, 0)
    close(out, want, tol, "bad pages out of the window")
    assert torch.isfinite(out[:new]).all()
    before = s.data.clone()
    k, kvl = s.rows_of(256)
    q3q4.kv_write(s.cache, s.batch, k, k)
    ko, vo = torch.empty_like(k), torch.empty_like(k)
    q3q4.kv_read(s.cache, s.batch, ko, vo)
    torch.cuda.synchronize()
    s.pool = before.cpu().numpy().reshape(s.pool.shape)
    ao.write(s.pool, kind, 16, 2, 128, s.table, s.starts, s.lens, kvl.astype(np.float32), kvl.astype(np.float32))
    assert np.array_equal(s.data.cpu().numpy(), s.pool.reshape(-1))
    lost = torch.tensor([s.table[b][(150 - new + i) // 16] == entry for b in (0, 1) for i in range(new)])
    assert torch.isnan(ko[lost.cuda()]).all() and torch.isfinite(ko[~lost.cuda()]).all()


@pytest.mark.parametrize("starts,lens", [([0, 2, 4], [20, 301]), ([0, 2, 4], [-1, 20]), ([0, 4, 2], [20, 20]),
                                         ([0, -3, 4], [20, 20]), ([1, 2, 900], [20, 20]), ([0, 4, 4], [20, 20])])
def test_batches_outside_the_bounds(torch, starts, lens):
    """Sequences whose rows or length break the host's bounds (4 rows, 3 at most each, 300 positions) give NaN in
    their rows and write nothing; rows of no sequence stay as they are; the others are right."""
    s = Setup(torch, ao.F16, F32, [2, 2], [300, 300], heads=16, kv_heads=2, page=16)
    cache, _ = s.device()
    i = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    batch = q3q4.KVBatch(i(starts), i(lens), i(s.table), 4, 3, 300)
    ok = [0 <= starts[b] <= starts[b + 1] <= 4 and starts[b + 1] - starts[b] <= 3 and 0 <= lens[b] <= 300
          for b in (0, 1)]
    q = torch.randn(4, 2048, device="cuda")
    out = torch.full_like(q, 7.0)
    q3q4.attention(cache, batch, q, out, 0.1, workspace=q3q4.attention_workspace(cache, batch, 16))
    k = torch.randn(4, 256, device="cuda")
    ko, vo = torch.full_like(k, 7.0), torch.full_like(k, 7.0)
    q3q4.kv_read(cache, batch, ko, vo)
    q3q4.kv_write(cache, batch, k, k)
    torch.cuda.synchronize()
    if not all(starts[b] <= starts[b + 1] for b in (0, 1)):
        return                                # rows of unordered sequences are anybody's; it ended
    for b in (0, 1):
        rows = slice(max(starts[b], 0), min(starts[b + 1], 4))
        if ok[b]:
            K, V = ao.values(s.pool, ao.F16, 16, 2, 128, s.table, b, lens[b])
            n = starts[b + 1] - starts[b]
            if n:
                want, tol = ao.attend(K, V, q[rows].double().cpu().numpy().reshape(n, 16, 128), lens[b], 0.1, 0, 0,
                                      ao.F32T)
                close(out[rows], want.reshape(n, -1), tol.reshape(n, -1), f"sequence {b}")
        else:
            assert torch.isnan(out[rows]).all() and torch.isnan(ko[rows]).all() and torch.isnan(vo[rows]).all()
    changed = (s.data.cpu().numpy().reshape(s.pool.shape) != s.pool).any((1, 2))
    for b in (0, 1):
        if not ok[b]:
            assert not changed[s.table[b]].any()


def test_large_prefill_against_torch(torch):
    """A chunk over several tiles and splits against float64 in torch, row by row to the last."""
    for kind, new, length, window, sinks in ((ao.F16, 700, 1900, 0, 0), (ao.Q8, 333, 2777, 400, 9)):
        s = Setup(torch, kind, F32, [new], [length], heads=16, kv_heads=2, page=32)
        q, qv = s.rows_of(2048, 1.5)
        out = s.attend(q, 0.09, window, sinks)
        K, V = ao.values(s.pool, kind, 32, 2, 128, s.table, 0, length)
        K, V = torch.from_numpy(K).cuda(), torch.from_numpy(V).cuda()
        p = torch.arange(length - new, length, device="cuda")[:, None]
        j = torch.arange(length, device="cuda")
        hid = j > p
        if window:
            hid = hid | ((j <= p - window) & (j >= sinks))
        for h in range(16):
            qq = q.double()[:, h * 128:(h + 1) * 128]
            w = torch.softmax((qq @ K[h // 8].T * 0.09).masked_fill(hid, -torch.inf), -1)
            want = w @ V[h // 8]
            a = (qq.abs() @ K[h // 8].abs().T).max(1, keepdim=True).values * 0.09
            tol = V[h // 8].abs().max() * (2 * 2.0 ** -19 * (a + 1) + 2.0 ** -20)
            assert ((out[:, h * 128:(h + 1) * 128].double() - want).abs() <= tol + want.abs() * 2.0 ** -24).all(), h
