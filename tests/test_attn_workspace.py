"""Bytes of the attention's workspace: enough for what is split, and bounded whatever the batch. No GPU (256 compute
units are assumed without one; tests run on cards of 256).

Contexts are split into at most cus / (row tiles * kv heads) parts of tiles of 256 rows, (dim + 2) floats a row:
256 * 256 * 130 * 4 bytes. The few-row kernel splits into cus / (sequences * kv heads) parts of 32 rows: 256 * 32 * 130 * 4.
"""
import ctypes

import numpy as np
import pytest

import attn_oracle as ao
import q3q4

MOST = 256 * (256 + 32) * 130 * 4


def bytes_of(sequences, rows, max_new, max_kv, heads, kv_heads, dim=128):
    c = q3q4.KVCacheArgs(ao.F16, 64, kv_heads, dim, 10, 4096)
    b = q3q4.KVBatchArgs(sequences, rows, max_new, max_kv, 1 << 24, 64, 128, 256)
    return q3q4.load().sera_attention_workspace_bytes(ctypes.byref(c), ctypes.byref(b), heads)


@pytest.mark.parametrize("sequences,rows,max_new,max_kv,heads,kv_heads", [
    (64, 63 + 64, 64, 32768, 64, 8), (256, 255 + 64, 64, 16384, 64, 8), (4000, 4000 + 63, 64, 32768, 8, 1),
    (300, 299 + 200, 200, 32768, 8, 1), (1 << 20, 64, 64, 65536, 8, 1), (1 << 20, 1 << 20, 100, 4096, 1, 1),
    (1, 512, 512, 32768, 64, 8), (1, 40, 40, 1 << 20, 1, 1), (40, 1000, 34, 9000, 34, 1),
])
def test_batches_of_all_kinds_stay_bounded(sequences, rows, max_new, max_kv, heads, kv_heads):
    assert bytes_of(sequences, rows, max_new, max_kv, heads, kv_heads) <= MOST <= 39e6


def test_drawn_batches_stay_bounded():
    rng = np.random.default_rng(11)
    log = lambda hi: int(np.exp(rng.uniform(0, np.log(hi + 0.5))))  # noqa: E731
    seen = 0
    for _ in range(5000):
        rows = log(1 << 17)
        kv_heads = log(16)
        n = bytes_of(log(1 << 13), rows, log(rows), log(1 << 20), kv_heads * log(40), kv_heads, int(rng.choice([64, 128])))
        assert n <= MOST
        seen += n > 0
    assert seen > 500


@pytest.mark.parametrize("new,max_kv,heads,kv_heads,splits", [(512, 32768, 64, 8, 2), (64, 4096, 8, 1, 16)])
def test_every_row_of_a_split_chunk_has_room(new, max_kv, heads, kv_heads, splits):
    assert bytes_of(1, new, new, max_kv, heads, kv_heads) == splits * new * heads * 130 * 4
