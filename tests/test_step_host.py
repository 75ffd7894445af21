"""Normed and rotated writes, attention weights, eviction and log probabilities without a GPU: refusals of every argument
that the host can check, sizes, and the oracle against second statements."""
import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest
import torch

import attn_oracle as ao
import q3q4
import step_oracle as so
from test_attn_devices import OnDevice, cache_and_batch, ints

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def L():
    return q3q4.load()


def structs(over):
    c = dict(type=ao.F16, page_tokens=64, kv_heads=8, head_dim=128, pages=10, data=4096)
    b = dict(sequences=2, rows=5, max_new=3, max_kv=100, table_stride=2, row_start=64, kv_len=128, page_table=256)
    for n in list(over):
        if n in c:
            c[n] = over.pop(n)
        elif n in b:
            b[n] = over.pop(n)
    return q3q4.KVCacheArgs(**c), q3q4.KVBatchArgs(**b)


def call(L, what, **over):
    c, b = structs(over)
    cp = ctypes.byref(c) if over.pop("cache", True) else None
    bp = ctypes.byref(b) if over.pop("batch", True) else None
    a = dict(type=0, heads=64, q=4096, qs=8192, out=8192, os=8192, k=4096, ks=1024, v=4096, vs=1024, positions=64, inv_freq=64,
             q_gamma=64, k_gamma=128, eps=1e-6, rotated=128, pairing=0, rope=True, scale=0.1, window=0, sinks=0, before=1 << 30,
             weights=1 << 20, stride=100, ws=4096, wb=1 << 40, keep=50, recent=10, new_weights=1 << 30, new_table=64, new_stride=1,
             new_len=64, kept=64)
    assert not set(over) - set(a), over
    a.update(over)
    if what == "rope":
        r = q3q4.QKRopeArgs(a["inv_freq"], a["q_gamma"], a["k_gamma"], a["eps"], a["rotated"], a["pairing"])
        rc = L.sera_kv_write_rope(cp, bp, ctypes.byref(r) if a["rope"] else None, a["type"], a["q"], a["qs"], a["out"], a["os"],
                                  a["heads"], a["k"], a["ks"], a["v"], a["vs"], a["positions"], None)
    elif what == "weights":
        rc = L.sera_attention_weights(cp, bp, a["type"], a["q"], a["qs"], a["out"], a["os"], a["heads"], a["scale"], a["window"],
                                      a["sinks"], a["before"], a["weights"], a["stride"], a["ws"], a["wb"], None)
    else:
        rc = L.sera_kv_evict(cp, bp, a["keep"], a["recent"], a["sinks"], a["weights"], a["new_weights"], a["stride"], a["new_table"],
                             a["new_stride"], a["new_len"], a["kept"], None)
    return rc, L.sera_q4k_last_error().decode()


BOTH = [(dict(cache=False), "null"), (dict(batch=False), "null"), (dict(type_=8), "type"), (dict(page_tokens=48), "power of two"),
        (dict(head_dim=80), "64 or 128"), (dict(kv_heads=0), "heads"), (dict(pages=0), "pages"), (dict(pages=1 << 31), "pages"),
        (dict(data=None), "aligned"), (dict(data=4104), "aligned"), (dict(sequences=-1), "outside"),
        (dict(sequences=(1 << 20) + 1), "outside"), (dict(max_kv=0), "max_kv"), (dict(max_kv=129), "max_kv"),
        (dict(table_stride=0), "max_kv"), (dict(max_kv=(1 << 28) + 1, table_stride=1 << 30), "max_kv"), (dict(kv_len=None), "null"),
        (dict(page_table=None), "null"), (dict(kv_len=130), "4-byte")]
NAMES = {"rope": "sera_kv_write_rope", "weights": "sera_attention_weights", "evict": "sera_kv_evict"}


@pytest.mark.parametrize("what", NAMES)
@pytest.mark.parametrize("bad,msg", BOTH, ids=[",".join(f"{k}={v}" for k, v in b[0].items()) for b in BOTH])
def test_refusals_of_cache_and_batch(L, what, bad, msg):
    bad = dict(bad)
    if "type_" in bad:
        if what == "evict":
            pytest.skip("eviction has no row type")
        bad = {"type": bad.pop("type_")}
        c, b = structs({})
        r = q3q4.QKRopeArgs(64, 64, 64, 0.0, 128, 0)
        rc = (L.sera_kv_write_rope(ctypes.byref(c), ctypes.byref(b), ctypes.byref(r), 8, 4096, 8192, 4096, 8192, 64, 4096, 1024, 4096, 1024, None, None)
              if what == "rope" else
              L.sera_attention_weights(ctypes.byref(c), ctypes.byref(b), 8, 4096, 8192, 8192, 8192, 64, 0.1, 0, 0, None, 4096, 100, 4096, 1 << 40, None))
        err = L.sera_q4k_last_error().decode()
    else:
        rc, err = call(L, what, **bad)
    assert rc == -1 and msg in err and NAMES[what] in err, (rc, err)


ROWS = [(dict(sequences=0), "no sequence"), (dict(rows=-1), "outside"), (dict(rows=(1 << 22) + 1), "outside"), (dict(max_new=0), "max_new"),
        (dict(max_new=6), "max_new"), (dict(row_start=None), "null"), (dict(row_start=66), "4-byte"), (dict(heads=0), "query heads"),
        (dict(heads=12), "query heads"), (dict(heads=16392), "query heads"), (dict(q=None), "null q"), (dict(out=None), "null"),
        (dict(q=4104), "16-byte"), (dict(os=8198), "16-byte"), (dict(qs=512), "apart"), (dict(os=1 << 41), "apart")]


@pytest.mark.parametrize("what", ["rope", "weights"])
@pytest.mark.parametrize("bad,msg", ROWS, ids=[",".join(f"{k}={v}" for k, v in b[0].items()) for b in ROWS])
def test_refusals_of_rows(L, what, bad, msg):
    rc, err = call(L, what, **bad)
    assert rc == -1 and msg in err and NAMES[what] in err, (rc, err)


@pytest.mark.parametrize("bad,msg", [
    (dict(rope=False), "null rope"), (dict(rotated=100), "rotate"), (dict(rotated=-128), "rotate"), (dict(rotated=256), "rotate"),
    (dict(pairing=2), "pairing"), (dict(pairing=-1), "pairing"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(eps=float("inf")), "eps"), (dict(inv_freq=None), "inv_freq"), (dict(inv_freq=66), "inv_freq"), (dict(q_gamma=68), "gamma"),
    (dict(k_gamma=68), "gamma"), (dict(positions=66), "positions"), (dict(k=None), "null k"), (dict(v=None), "null v"),
    (dict(k=4104), "16-byte"), (dict(ks=512), "apart"), (dict(vs=1026), "16-byte"), (dict(q=8192, os=8256), "another stride"),
])
def test_rope_refusals(L, bad, msg):
    rc, err = call(L, "rope", **bad)
    assert rc == -1 and msg in err, (rc, err)


@pytest.mark.parametrize("bad,msg", [
    (dict(window=-1), "below zero"), (dict(sinks=-1), "below zero"), (dict(scale=float("nan")), "finite"),
    (dict(rows=1 << 20, max_new=1, heads=16384, kv_heads=1024), "2^31"), (dict(weights=None), "weights"), (dict(weights=(1 << 20) + 2), "weights"),
    (dict(before=(1 << 20) + 4), "overlap"), (dict(before=(1 << 20) - 4), "overlap"), (dict(stride=99), "apart"), (dict(stride=1 << 40), "apart"),
    (dict(ws=None), "workspace"), (dict(ws=4100), "workspace"), (dict(wb=5 * 64 * 4 - 1), "workspace"),
])
def test_weights_refusals(L, bad, msg):
    rc, err = call(L, "weights", **bad)
    assert rc == -1 and msg in err, (rc, err)


@pytest.mark.parametrize("bad,msg", [
    (dict(keep=0, recent=0), "keep"), (dict(keep=-1, recent=0), "keep"), (dict(keep=(1 << 28) + 1), "keep"), (dict(recent=-1), "recent"),
    (dict(sinks=-1), "sinks"), (dict(recent=40, sinks=11), "no more"), (dict(recent=2 ** 31 - 1, sinks=2 ** 31 - 1), "no more"),
    (dict(new_stride=0), "new positions"), (dict(keep=65, new_stride=1), "new positions"), (dict(new_table=None), "new_table"),
    (dict(new_len=None), "new_len"), (dict(kept=None), "kept"), (dict(kept=66), "aligned"), (dict(new_len=128), "kv_len"),
    (dict(weights=None), "weights"), (dict(new_weights=None), "weights"), (dict(new_weights=1 << 20), "overlap"),
    (dict(new_len=132), "kv_len"), (dict(new_len=124), "kv_len"),
    (dict(new_weights=(1 << 20) + 4 * 1599), "overlap"), (dict(stride=99), "apart"),
])
def test_evict_refusals(L, bad, msg):
    rc, err = call(L, "evict", **bad)
    assert rc == -1 and msg in err, (rc, err)


def test_no_rows_or_sequences_is_no_work(L):
    for what in ("rope", "weights"):
        assert call(L, what, rows=0, q=None, out=None, data=None, weights=None, inv_freq=None)[0] == 0
    assert call(L, "evict", sequences=0, weights=None, kept=None, data=None)[0] == 0


def test_weights_workspace(L):
    """Room for a number of every row and head at least; 0 where the call refuses the bounds."""
    c, b = structs({})
    plain = L.sera_attention_workspace_bytes(ctypes.byref(c), ctypes.byref(b), 64)
    assert L.sera_attention_weights_workspace_bytes(ctypes.byref(c), ctypes.byref(b), 64) >= plain + 5 * 64 * 4
    for over, heads in ((dict(head_dim=80), 64), (dict(rows=0), 64), (dict(max_kv=0), 64), ({}, 12), ({}, 0)):
        c, b = structs(dict(over))
        assert L.sera_attention_weights_workspace_bytes(ctypes.byref(c), ctypes.byref(b), heads) == 0
    assert L.sera_attention_weights_workspace_bytes(None, None, 64) == 0


def logprobs(L, **over):
    a = dict(type=0, x=4096, stride=1000, rows=2, vocab=1000, tokens=64, n=3, given=64, entropy=64, top=5, ids=64, lp=64, ws=4096,
             wb=1 << 40)
    assert not set(over) - set(a)
    a.update(over)
    rc = L.sera_logprobs(a["type"], a["x"], a["stride"], a["rows"], a["vocab"], a["tokens"], a["n"], a["given"], a["entropy"], a["top"],
                         a["ids"], a["lp"], a["ws"], a["wb"], None)
    return rc, L.sera_q4k_last_error().decode()


@pytest.mark.parametrize("bad,msg", [
    (dict(type=8), "row type"), (dict(rows=-1), "rows"), (dict(rows=(1 << 22) + 1), "rows"), (dict(vocab=0), "rows"),
    (dict(vocab=(1 << 28) + 1, stride=1 << 30), "rows"), (dict(top=-1), "top"), (dict(top=65), "top"), (dict(top=6, vocab=5), "top"),
    (dict(n=-1), "per_row"), (dict(n=1 << 30), "per_row"), (dict(stride=999), "apart"), (dict(stride=1 << 41), "apart"),
    (dict(x=None), "logits"), (dict(x=4098), "aligned"), (dict(type=1, x=4097), "aligned"), (dict(tokens=None), "tokens"),
    (dict(given=None), "token_logprobs"), (dict(tokens=66), "tokens"), (dict(ids=None), "top_ids"), (dict(lp=None), "top_logprobs"),
    (dict(lp=66), "top_ids"), (dict(entropy=66), "entropy"), (dict(vocab=151936, stride=151936, ws=None), "workspace"),
    (dict(vocab=151936, stride=151936, wb=100), "workspace"), (dict(vocab=151936, stride=151936, ws=4100), "workspace"),
])
def test_logprobs_refusals(L, bad, msg):
    rc, err = logprobs(L, **bad)
    assert rc == -1 and msg in err and "sera_logprobs" in err, (rc, err)


def test_logprobs_of_nothing(L):
    assert logprobs(L, rows=0, x=None, tokens=None, ids=None)[0] == 0
    assert logprobs(L, n=0, top=0, entropy=None, x=None)[0] == 0


def test_logprobs_workspace_is_bounded(L):
    rng = np.random.default_rng(3)
    log = lambda hi: int(np.exp(rng.uniform(0, np.log(hi + 0.5))))  # noqa: E731
    seen = 0
    for _ in range(3000):
        vocab = log(1 << 22)
        n = L.sera_logprobs_workspace_bytes(log(1 << 14), vocab, min(int(rng.integers(0, 65)), vocab))
        assert n <= 3e5
        seen += n > 0
    assert seen > 300
    for rows, vocab, top in ((0, 10, 1), (1, 0, 0), (1, 10, 11), (1, 100, 65), (-1, 10, 1)):
        assert L.sera_logprobs_workspace_bytes(rows, vocab, top) == 0


# ---- the Python calls ---------------------------------------------------------

def rope_call(c, b, q=None, q_out=None, k=None, rope=None, positions=None, v=None):
    q, q_out, k, v = (OnDevice(2, 64) if t is None else t for t in (q, q_out, k, v))
    q3q4.kv_write_rope(c, b, rope or q3q4.Rope(), q, q_out, k, v, positions)


def test_python_rope_refusals():
    c, b = cache_and_batch(0, 0)
    for host in ("q", "q_out", "k", "v"):
        with pytest.raises(q3q4.Q3Q4Error, match="cache's device"):
            rope_call(c, b, **{host: torch.zeros(2, 64)})
    with pytest.raises(q3q4.Q3Q4Error, match="no heads"):
        rope_call(c, b, q=OnDevice(2, 72), q_out=OnDevice(2, 72))
    with pytest.raises(q3q4.Q3Q4Error, match="one type"):
        rope_call(c, b, k=OnDevice(2, 64, torch.float16), v=OnDevice(2, 64, torch.float16))
    with pytest.raises(q3q4.Q3Q4Error, match="positions"):
        rope_call(c, b, positions=ints(2))
    with pytest.raises(q3q4.Q3Q4Error, match="on device 0"):
        rope_call(c, b, rope=q3q4.Rope(torch.ones(32)))
    with pytest.raises(q3q4.Q3Q4Error, match="q_gamma"):
        q3q4.Rope(None, torch.ones(64, dtype=torch.float16))
    with pytest.raises(q3q4.Q3Q4Error, match="inv_freq"):
        q3q4.Rope(torch.ones(64)[::2])
    r = q3q4.Rope(None, torch.ones(32))
    r.device = 0
    with pytest.raises(q3q4.Q3Q4Error, match="gamma of 32"):
        rope_call(c, b, rope=r)
    c, b = cache_and_batch()
    with pytest.raises(q3q4.Q3Q4Error, match="one device"):
        rope_call(c, b)


def test_python_weights_and_evict_refusals():
    r = OnDevice(2, 64)
    c, b = cache_and_batch(0, 0)
    for w in (torch.zeros(2, 1, 16), torch.zeros(2, 1, 16, dtype=torch.float16)):
        with pytest.raises(q3q4.Q3Q4Error, match="weights must be"):
            q3q4.attention_weights(c, b, r, r, 0.1, w)
    c, b = cache_and_batch()
    with pytest.raises(q3q4.Q3Q4Error, match="one device"):
        q3q4.attention_weights(c, b, r, r, 0.1, torch.zeros(2, 1, 16))
    with pytest.raises(q3q4.Q3Q4Error, match="device tensor"):
        q3q4.attention_weights_workspace(c, b, 1)
    new = (ints(2, 1), ints(2), torch.zeros(2, 1, 16), ints(2, 1, 8))
    with pytest.raises(q3q4.Q3Q4Error, match="one device"):
        q3q4.kv_evict(c, b, 8, torch.zeros(2, 1, 16), *new)
    c, b = cache_and_batch(0, 0)
    with pytest.raises(q3q4.Q3Q4Error, match="weights must be"):
        q3q4.kv_evict(c, b, 8, torch.zeros(2, 1, 16), *new)


def test_python_logprobs_refusals():
    with pytest.raises(q3q4.Q3Q4Error, match="rows, vocab"):
        q3q4.logprobs(torch.zeros(5))
    with pytest.raises(q3q4.Q3Q4Error, match="device tensor"):
        q3q4.logprobs(torch.zeros(2, 5))
    with pytest.raises(q3q4.Q3Q4Error, match="rows, vocab"):
        q3q4.logprobs_workspace(torch.zeros(5))
    with pytest.raises(q3q4.Q3Q4Error, match="device tensor"):
        q3q4.logprobs_workspace(torch.zeros(2, 5))


# ---- the oracle ---------------------------------------------------------------

def test_oracle_of_heads():
    """As complex numbers; a turn keeps a pair's length, and scores depend on the difference of positions alone."""
    rng = np.random.default_rng(0)
    x, f = rng.standard_normal((3, 2, 8)), np.array([1.0, 0.1, 0.01], np.float32)
    for pairing in (so.HALVES, so.NEIGHBOURS):
        y, _ = so.heads_turned(x, None, 0.0, f, pairing, [0, 5, 7])
        pick = (lambda a: a[..., :3] + 1j * a[..., 3:6]) if pairing == so.HALVES else (lambda a: a[..., 0:6:2] + 1j * a[..., 1:6:2])
        turn = np.exp(1j * np.array([0, 5, 7])[:, None, None] * f.astype(np.float64))
        assert np.allclose(pick(y), pick(x) * turn, rtol=1e-12) and np.array_equal(y[..., 6:], x[..., 6:])
        a, _ = so.heads_turned(x[:1], None, 0.0, f, pairing, [11])
        b, _ = so.heads_turned(x[1:2], None, 0.0, f, pairing, [8])
        c, _ = so.heads_turned(x[:1], None, 0.0, f, pairing, [103])
        d, _ = so.heads_turned(x[1:2], None, 0.0, f, pairing, [100])
        assert np.allclose((a * b).sum(-1), (c * d).sum(-1))
    g = np.arange(8, dtype=np.float32)
    y, _ = so.heads_turned(x, g, 0.5, None, 0, [0, 0, 0])
    assert np.allclose(y, x / np.sqrt((x ** 2).mean(-1, keepdims=True) + 0.5) * g)


def test_oracle_of_weights_and_kept():
    rng = np.random.default_rng(4)
    K, q = rng.standard_normal((2, 9, 64)), rng.standard_normal((4, 6, 64))
    w, _ = so.weights_of(K, q, 9, 0.2, 3, 2)
    assert np.allclose(w.sum(), 24) and w[0, 8] < w[0].sum()
    o, _ = ao.attend(K, np.broadcast_to(np.eye(9, 64), (2, 9, 64)), q, 9, 0.2, 3, 2, ao.F32T)      # values that say their position
    assert np.allclose(o.sum(0).reshape(2, 3, 64).sum(1)[:, :9], w)
    assert so.kept_of([5, 1, 2, 2, 9, 0], 6, 4, 1, 1) == [0, 2, 4, 5]
    assert so.kept_of([0, 0, 0, 0, 0], 5, 3, 0, 0) == [0, 1, 2]
    assert so.kept_of([np.nan, -np.inf, -5], 3, 2, 0, 0) == [1, 2] and so.kept_of([1, 2], 2, 3, 0, 0) == [0, 1]


def test_oracle_of_scores():
    x = np.random.default_rng(5).standard_normal(50)
    x[7] = -np.inf
    given, entropy, ids, lp = so.scores(x, [3, 7, 50, -1], 4)
    t = torch.log_softmax(torch.from_numpy(x), -1).numpy()
    assert np.allclose(given[:2], t[[3, 7]]) and np.isnan(given[2:]).all() and np.allclose(lp, np.sort(t)[::-1][:4])
    p = np.exp(t)
    assert np.allclose(entropy, -np.sum(p[p > 0] * t[p > 0])) and ids.tolist() == np.argsort(-x)[:4].tolist()
    assert np.isnan(so.scores(np.full(3, -np.inf), [0], 1)[1]) and so.scores(np.zeros(5), [], 3)[2].tolist() == [0, 1, 2]


# ---- C ------------------------------------------------------------------------

SOURCE = r"""
#include "sera_attn.h"
#include "sera_logprobs.h"
#include "sera_q4k.h"
#include <stdio.h>

int main(void) {
    static int32_t ints[64];
    static float floats[64];
    sera_kv_cache cache = {SERA_KV_F16, 16, 1, 64, 4, floats};
    sera_kv_batch batch = {1, 1, 1, 16, 1, ints, ints, ints};
    sera_qk_rope rope = {floats, floats, 0, 1e-6f, 64, SERA_ROPE_NEIGHBOURS};
    printf("sizes %zu %zu %zu\n", sizeof rope, offsetof(sera_qk_rope, eps), offsetof(sera_qk_rope, pairing));
    printf("workspace %zu %zu\n", sera_attention_weights_workspace_bytes(&cache, &batch, 2), sera_logprobs_workspace_bytes(1, 151936, 20));
    printf("rope %d\n", sera_kv_write_rope(&cache, &batch, &rope, SERA_TYPE_F32, 0, 64, 0, 64, 1, 0, 64, 0, 64, 0, 0));
    printf("weights %d\n", sera_attention_weights(&cache, &batch, SERA_TYPE_F32, 0, 64, 0, 64, 1, 0.1f, 0, 0, 0, 0, 16, 0, 0, 0));
    printf("evict %d\n", sera_kv_evict(&cache, &batch, 8, 9, 0, floats, floats, 16, ints, 1, ints, ints, 0));
    printf("logprobs %d\n", sera_logprobs(SERA_TYPE_BF16, 0, 10, 1, 10, 0, 0, 0, floats, SERA_LOGPROBS_MAX_TOP, ints, floats, 0, 0, 0));
    return 0;
}
"""


def test_c99_caller(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    assert cc, "no C compiler in PATH"
    flags = [cc, "-std=c99", "-Wall", "-Wextra", "-Werror", "-pedantic", "-I", os.path.join(ROOT, "include")]
    alone = tmp_path / "alone.c"
    alone.write_text('#include "sera_logprobs.h"\n#include "sera_logprobs.h"\nint unused;\n')
    r = subprocess.run(flags + ["-c", str(alone), "-o", str(tmp_path / "alone.o")], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    src, exe, libdir = tmp_path / "caller.c", tmp_path / "caller", os.path.dirname(q3q4.LIB_PATH)
    src.write_text(SOURCE)
    r = subprocess.run(flags + [str(src), "-L", libdir, "-lsera_q4k", f"-Wl,-rpath,{libdir}", "-o", str(exe)], capture_output=True,
                       text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr
    out = dict(line.split(" ", 1) for line in r.stdout.strip().splitlines())
    R = q3q4.QKRopeArgs
    assert out["sizes"] == f"{ctypes.sizeof(R)} {R.eps.offset} {R.pairing.offset}"
    L = q3q4.load()
    c, b = q3q4.KVCacheArgs(ao.F16, 16, 1, 64, 4, 16), q3q4.KVBatchArgs(1, 1, 1, 16, 1, 4, 4, 4)
    assert out["workspace"] == (f"{L.sera_attention_weights_workspace_bytes(ctypes.byref(c), ctypes.byref(b), 2)} "
                                f"{L.sera_logprobs_workspace_bytes(1, 151936, 20)}")
    assert [out[k] for k in ("rope", "weights", "evict", "logprobs")] == ["-1"] * 4
