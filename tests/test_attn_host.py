"""Cache and attention without a GPU: layout and sizes, refusals of every
argument the host can check, and the oracle against a second statement."""
import ctypes

import numpy as np
import pytest

import attn_oracle as ao
import q3q4


@pytest.fixture(scope="module")
def L():
    return q3q4.load()


def structs(**over):
    c = dict(type=ao.F16, page_tokens=64, kv_heads=8, head_dim=128, pages=10, data=4096)
    b = dict(sequences=2, rows=5, max_new=3, max_kv=100, table_stride=2, row_start=64, kv_len=128, page_table=256)
    for n, v in over.items():
        (c if n in c else b)[n] = v
    return q3q4.KVCacheArgs(**c), q3q4.KVBatchArgs(**b)


def call(L, what, type=0, x=4096, xs=1024, y=8192, ys=1024, heads=64, scale=0.1, window=0, sinks=0, ws=4096,
         wb=1 << 40, cache=True, batch=True, **over):
    c, b = structs(**over)
    cp, bp = (ctypes.byref(c) if cache else None), (ctypes.byref(b) if batch else None)
    if what == "attention":
        xs = 8192 if xs == 1024 else xs
        ys = 8192 if ys == 1024 else ys
        rc = L.sera_attention(cp, bp, type, x, xs, y, ys, heads, scale, window, sinks, ws, wb, None)
    else:
        rc = getattr(L, "sera_kv_" + what)(cp, bp, type, x, xs, y, ys, None)
    return rc, L.sera_q4k_last_error().decode()


def test_struct_sizes():
    assert ctypes.sizeof(q3q4.KVCacheArgs) == 32 and q3q4.KVCacheArgs.data.offset == 24
    assert ctypes.sizeof(q3q4.KVBatchArgs) == 48 and q3q4.KVBatchArgs.row_start.offset == 24


@pytest.mark.parametrize("kind,page,heads,dim,want", [
    (ao.F16, 64, 8, 128, 64 * 8 * 128 * 4), (ao.F16, 16, 1, 64, 16 * 64 * 4),
    (ao.Q8, 32, 6, 128, 6 * (32 * 128 * 2 + 32 * 8)), (ao.Q8, 1024, 3, 64, 3 * (1024 * 64 * 2 + 8192)),
    (ao.F16, 48, 8, 128, 0), (ao.F16, 8, 8, 128, 0), (ao.F16, 2048, 8, 128, 0), (ao.F16, 64, 0, 128, 0),
    (ao.F16, 64, 8, 96, 0), (8, 64, 8, 128, 0), (ao.Q8, -16, 8, 128, 0),
])
def test_page_bytes(L, kind, page, heads, dim, want):
    assert L.sera_kv_page_bytes(kind, page, heads, dim) == want
    if want:
        assert want == heads * ao.head_bytes(kind, page, dim)


BOTH = [
    (dict(cache=False), "null"), (dict(batch=False), "null"), (dict(type=8), "row type"),
    (dict(page_tokens=48), "power of two"), (dict(head_dim=80), "64 or 128"), (dict(kv_heads=0), "heads"),
    (dict(pages=0), "pages"), (dict(pages=1 << 31), "pages"), (dict(data=None), "aligned"), (dict(data=4104), "aligned"),
    (dict(sequences=0), "no sequence"), (dict(sequences=-1), "outside"), (dict(rows=-1), "outside"),
    (dict(rows=(1 << 22) + 1), "outside"), (dict(max_new=0), "max_new"), (dict(max_new=6), "max_new"),
    (dict(max_kv=0), "max_kv"), (dict(max_kv=129), "max_kv"), (dict(table_stride=0), "max_kv"),
    (dict(max_kv=(1 << 28) + 1, table_stride=1 << 30), "max_kv"),
    (dict(row_start=None), "null"), (dict(kv_len=None), "null"), (dict(page_table=None), "null"),
    (dict(kv_len=130), "4-byte"), (dict(x=None), "null"), (dict(y=None), "null"), (dict(x=4104), "16-byte"),
    (dict(ys=8198), "16-byte"), (dict(xs=512), "apart"), (dict(ys=1 << 41), "apart"), (dict(type=1, xs=8196), "16-byte"),
]


@pytest.mark.parametrize("what", ["write", "read", "attention"])
@pytest.mark.parametrize("bad,msg", BOTH, ids=[",".join(f"{k}={v}" for k, v in b[0].items()) for b in BOTH])
def test_refusals(L, what, bad, msg):
    rc, err = call(L, what, **bad)
    assert rc == -1 and msg in err, (rc, err)
    assert ("sera_attention" if what == "attention" else "sera_kv_" + what) in err


@pytest.mark.parametrize("bad,msg", [
    (dict(heads=0), "query heads"), (dict(heads=12), "query heads"), (dict(heads=16392), "query heads"),
    (dict(window=-1), "below zero"), (dict(sinks=-1), "below zero"), (dict(scale=float("nan")), "finite"),
    (dict(scale=float("inf")), "finite"), (dict(rows=1 << 20, max_new=1, heads=16384, kv_heads=1024), "2^31"),
])
def test_attention_refusals(L, bad, msg):
    rc, err = call(L, "attention", **bad)
    assert rc == -1 and msg in err, (rc, err)


def test_workspace_of_refused_arguments_is_zero(L):
    for over, heads in ((dict(head_dim=80), 64), (dict(rows=0), 64), (dict(max_kv=0), 64), ({}, 12), ({}, 0)):
        c, b = structs(**over)
        assert L.sera_attention_workspace_bytes(ctypes.byref(c), ctypes.byref(b), heads) == 0
    assert L.sera_attention_workspace_bytes(None, None, 64) == 0


def test_no_rows_is_no_work(L):
    for what in ("write", "read", "attention"):
        assert call(L, what, rows=0, x=None, y=None, data=None)[0] == 0
        assert call(L, what, rows=0, sequences=0, row_start=None)[0] == 0


def test_python_refusals():
    import torch
    with pytest.raises(q3q4.Q3Q4Error, match="no cache"):
        q3q4.KVCache(ao.F16, 4, 48, 8, 128, data=torch.empty(1, dtype=torch.uint8))
    with pytest.raises(q3q4.Q3Q4Error, match="contiguous uint8"):
        q3q4.KVCache(ao.F16, 4, 64, 8, 128, data=torch.empty(100, dtype=torch.uint8))
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(q3q4.Q3Q4Error, match="int32"):
        q3q4.KVBatch(i(3).long(), i(2), i(2, 4), 2, 1, 10)
    with pytest.raises(q3q4.Q3Q4Error, match="int32"):
        q3q4.KVBatch(i(2), i(2), i(2, 4), 2, 1, 10)
    with pytest.raises(q3q4.Q3Q4Error, match="hold"):
        q3q4.KVBatch(i(3), i(2), i(2, 4), 2, 1, 5000)
    c = q3q4.KVCache(ao.F16, 1, 16, 1, 64, data=torch.empty(4096, dtype=torch.uint8))
    b = q3q4.KVBatch(i(3), i(2), i(2, 4), 2, 1, 64)
    with pytest.raises(q3q4.Q3Q4Error, match="device tensor"):
        q3q4.kv_write(c, b, torch.zeros(2, 64), torch.zeros(2, 64))
    with pytest.raises(q3q4.Q3Q4Error, match="hold"):
        q3q4.kv_write(c, q3q4.KVBatch(i(3), i(2), i(2, 4), 2, 1, 65), torch.zeros(2, 64), torch.zeros(2, 64))


def test_oracle_layout_and_codes():
    """The oracle's cache read back equals what was written; codes round the exact quotient half to even."""
    rng = np.random.default_rng(3)
    for kind in (ao.F16, ao.Q8):
        page, heads, dim = 16, 2, 64
        pool = np.zeros((5, heads, ao.head_bytes(kind, page, dim)), np.uint8)
        k, v = (rng.standard_normal((21, heads * dim)).astype(np.float32) for _ in "kv")
        ao.write(pool, kind, page, heads, dim, [[3, 1]], [0, 21], [21], k, v)
        K, V = ao.values(pool, kind, page, heads, dim, [[3, 1]], 0, 21)
        for got, x in ((K, k), (V, v)):
            x = x.reshape(21, heads, dim).transpose(1, 0, 2)
            if kind == ao.F16:
                assert np.array_equal(got, x.astype(np.float16))
            else:
                assert np.all(np.abs(got - x) <= 0.5001 * np.abs(x).max(-1, keepdims=True) / 127)
    q, d = ao.codes(np.array([127, 0.5, 1.5, 2.5, -0.5, -63.5], np.float32))
    assert d == 1 and list(q) == [127, 0, 2, 2, 0, -64]
    assert np.isnan(ao.codes([1, np.inf])[1]) and ao.codes([0, 0])[1] == 0


def test_oracle_attention_against_softmax():
    rng = np.random.default_rng(4)
    K, V, q = rng.standard_normal((2, 9, 64)), rng.standard_normal((2, 9, 64)), rng.standard_normal((4, 6, 64))
    o, _ = ao.attend(K, V, q, 9, 0.2, 3, 2, ao.F32T)
    for i in range(4):
        p = 5 + i
        see = sorted(set(range(max(0, p - 2), p + 1)) | {0, 1})
        for h in range(6):
            s = np.exp(0.2 * K[h // 3][see] @ q[i, h])
            assert np.allclose(o[i, h], (s[:, None] * V[h // 3][see]).sum(0) / s.sum(), rtol=1e-12)
    o, _ = ao.attend(K[:, :2], V[:, :2], q, 2, 0.2, 0, 0, ao.F32T)
    assert np.all(o[:2] == 0) and np.allclose(o[2], np.repeat(V[:, 0], 3, 0))
