"""Attention at the limits of what a caller may pass: arrays on the device that break the rules, the largest arguments,
offsets. Tolerances as in test_gpu_attention.
"""
import numpy as np
import pytest

import attn_oracle as ao
import q3q4
from test_gpu_attention import BF16, F16, F32, Setup, check, close, torch  # noqa: F401  (torch: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("starts,rows,max_new,max_kv", [
    ([0, 64, 0, 64, 0, 64], 64, 64, 4096),
    ([0, 200, 0, 200, 0, 200, 0, 200], 200, 200, 4096),
    ([0, 900, 100, 1000], 1000, 900, 16384),
    ([0, 1, 0, 200, 1, 2, 0, 200, 3, 4, 5, 6, 7, 8, 9, 10], 200, 200, 4096),
])
def test_overlapping_sequences_stay_inside_the_workspace(torch, kind, starts, rows, max_new, max_kv):  # noqa: F811
    """row_start that decreases: sequences that lie inside the bounds one by one and have more row tiles together than
    the batch has rows for. Nothing behind the workspace is written, and an ordered batch in the same workspace is
    right afterwards."""
    print(f"case overlapping kind={kind} {starts}", flush=True)
    n = len(starts) - 1
    s = Setup(torch, kind, F32, [40, 3], [1000, 700], heads=8, kv_heads=1, page=64)
    cache, _ = s.device()
    ints = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    # every entry is a page of the pool
    table = ints(np.resize(s.table[0, :8], (n, max_kv // 64)))
    batch = q3q4.KVBatch(ints(starts), ints([max_kv - 7 * b for b in range(n)]), table, rows, max_new, max_kv)
    need = q3q4.load().sera_attention_workspace_bytes(cache.ref, batch.ref, 8)
    assert need > 0, "the case is meant to leave partial sums"
    ws = torch.full((need + (64 << 20),), 0xA5, dtype=torch.uint8, device="cuda")
    q = torch.randn(rows, 1024, device="cuda")
    out = torch.full((rows + 64, 1024), 7.0, device="cuda")
    q3q4.attention(cache, batch, q, out[:rows], 0.1, workspace=ws)
    torch.cuda.synchronize()
    assert (ws[need:] == 0xA5).all(), "written behind the workspace"
    assert (out[rows:] == 7.0).all(), "written behind the rows"
    q, qv = s.rows_of(1024)
    want, tol = s.expect(qv, 0.1)
    o = torch.full_like(q, 7.0)
    assert q3q4.load().sera_attention_workspace_bytes(cache.ref, s.batch.ref, 8) <= ws.numel()
    q3q4.attention(cache, s.batch, q, o, 0.1, workspace=ws)
    close(o, want, tol, "ordered")


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 40, 2 ** 30, 129, 128])
@pytest.mark.parametrize("news,lens", [([50, 33], [7, 40]), ([2, 1], [1, 128]), ([300], [128])])
def test_windows_as_wide_as_the_context_are_none(torch, kind, window, news, lens):  # noqa: F811
    """A window of every position or more, up to the largest int: the result is that of no window, bit for bit, also
    where a sequence has rows in front of its start."""
    s = Setup(torch, kind, F32, news, lens, heads=8, kv_heads=2, page=16)
    print(f"case wide window kind={kind} window={window} {news} of {lens}", flush=True)
    q, first = check(s)
    for sinks in (0, 5, 2 ** 31 - 1):
        assert torch.equal(s.attend(q, s.dim ** -0.5, window, sinks), first)


@pytest.mark.parametrize("new", [40, 1])
def test_long_runs_of_zero_values(torch, new):  # noqa: F811
    """An 8-bit context whose values are zero vectors (scale 0) but for the last 128, with scores that rise by 7.9
    binades (less than the running maximum follows) behind the first 256: a sum of 56000 weights whose values hold
    none of them down. The result is the sum of the last values over all weights."""
    sequences, heads, kv_heads, dim, page, length = 32, 64, 8, 128, 128, 56064
    rng = np.random.default_rng(2)
    pages = length // page
    pool = np.zeros((pages, kv_heads, ao.head_bytes(ao.Q8, page, dim)), np.uint8)
    k, v, ks, vs = ao.views(pool, ao.Q8, page, kv_heads, dim)
    k[2:], ks[2:] = 100, 1e-4                  # 0.01 in each channel
    v[-1], vs[-1] = rng.integers(60, 128, v[-1].shape), 1 / 80
    ints = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    cache = q3q4.KVCache(ao.Q8, pages, page, kv_heads, dim, torch.from_numpy(pool.reshape(-1)).cuda())
    table = ints(range(pages))[None].expand(sequences, -1).contiguous()
    batch = q3q4.KVBatch(ints([new * b for b in range(sequences + 1)]), ints([length] * sequences), table,
                         new * sequences, new, length)
    scale = 7.9 * np.log(2) / (0.01 * dim)
    out = torch.full((new * sequences, heads * dim), 7.0, device="cuda")
    q3q4.attention(cache, batch, torch.ones_like(out), out, scale,
                   workspace=q3q4.attention_workspace(cache, batch, heads))
    K, V = ao.values(pool, ao.Q8, page, kv_heads, dim, [list(range(pages))], 0, length)
    n = min(new, 4)                            # the last rows, of the first and the last head
    want, tol = ao.attend(K[[0, -1]], V[[0, -1]], np.ones((n, 2, dim)), length, scale, 0, 0, ao.F32T)
    assert want.min() > 20 * tol.max()
    for b in (0, sequences - 1):
        got = out[(b + 1) * new - n:(b + 1) * new].view(n, heads, dim)[:, [0, -1]]
        close(got, want, tol, f"sequence {b}")


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
def test_rows_more_than_two_to_the_31_elements_apart(torch, kind):  # noqa: F811
    """Four rows 3 * 2^28 elements apart, the last 2.4e9 from the first, as keys and values in and out, q and result."""
    stride, width = 3 << 28, 1024
    buf = torch.empty(3 * stride + 4 * width, device="cuda")
    far = [buf.as_strided((4, width), (stride, 1), width * i) for i in range(4)]
    i = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    cache = q3q4.KVCache(kind, 1, 16, 8, 128)
    cache.data.zero_()
    batch = q3q4.KVBatch(i(0, 4), i(4), i(0)[None], 4, 4, 16)
    for f in far:
        f.copy_(torch.randn(4, width, device="cuda"))
    near = [f.clone() for f in far]
    q3q4.kv_write(cache, batch, far[0], far[1])
    pool = np.zeros((1, 8, ao.head_bytes(kind, 16, 128)), np.uint8)
    ao.write(pool, kind, 16, 8, 128, [[0]], [0, 4], [4], *(t.cpu().numpy() for t in near[:2]))
    assert np.array_equal(cache.data.cpu().numpy(), pool.reshape(-1))
    q3q4.kv_read(cache, batch, far[0], far[1])
    K, V = ao.values(pool, kind, 16, 8, 128, [[0]], 0, 4)
    for f, x in ((far[0], K), (far[1], V)):
        assert np.array_equal(f.cpu().numpy(), x.transpose(1, 0, 2).reshape(4, width).astype(np.float32))
    assert torch.equal(far[2], near[2]) and torch.equal(far[3], near[3])
    q3q4.attention(cache, batch, far[2], far[3], 0.1, workspace=q3q4.attention_workspace(cache, batch, 8))
    want, tol = ao.attend(K, V, near[2].double().cpu().numpy().reshape(4, 8, 128), 4, 0.1, 0, 0, ao.F32T)
    close(far[3], want.reshape(4, -1), tol.reshape(4, -1), "far rows")


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("sequences", [300, 70, 40])
def test_overlapping_sequences_in_every_search(torch, kind, sequences):  # noqa: F811
    """The same for as many sequences as take each of the searches over row_start, and for writes and reads: they end,
    and nothing but the batch's rows, the workspace and the tables' pages is written."""
    print(f"case overlapping kind={kind} sequences={sequences}", flush=True)
    rows, pages, page, heads, width, pad = 100, 40, 64, 8, 128, 16
    ints = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    cache = q3q4.KVCache(kind, pages, page, 1, 128)
    cache.data.zero_()
    starts = [(0, 90, 30, 100, 29)[b % 5] for b in range(sequences + 1)]
    table = ints(np.resize(np.arange(3, 23), (sequences, 64)))
    batch = q3q4.KVBatch(ints(starts), ints([4000 - b for b in range(sequences)]), table, rows, 95, 4096)
    need = q3q4.load().sera_attention_workspace_bytes(cache.ref, batch.ref, heads)
    ws = torch.full((need + (32 << 20),), 0xA5, dtype=torch.uint8, device="cuda")
    k, q = torch.randn(rows, width, device="cuda"), torch.randn(rows, heads * width, device="cuda")
    out, ko, vo = (torch.full((rows + pad, w), 7.0, device="cuda") for w in (heads * width, width, width))
    q3q4.kv_write(cache, batch, k, k)
    q3q4.kv_read(cache, batch, ko[:rows], vo[:rows])
    q3q4.attention(cache, batch, q, out[:rows], 0.1, workspace=ws)
    torch.cuda.synchronize()
    assert (ws[need:] == 0xA5).all() and all((t[rows:] == 7.0).all() for t in (out, ko, vo))
    held = cache.data.view(pages, -1)
    assert not held[:3].any() and not held[23:].any() and held[3:23].any()
