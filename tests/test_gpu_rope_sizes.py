"""sera_kv_write_rope on the GPU: very many sequences, nearly all of them without rows."""
import numpy as np
import pytest

import attn_oracle as ao
import q3q4
from test_gpu_attention import torch  # noqa: F401  (torch: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sequences,owner", [(1 << 20, 0), (1 << 20, (1 << 20) - 1), (1 << 20, 777777), (300000, 5)])
def test_a_row_among_very_many_sequences(torch, sequences, owner):  # noqa: F811
    """One row of 64 and 8 heads: with a workgroup for each of its 24 parts in every slot, 2^20 sequences would be 10^10
    threads. The result is that of a batch of its sequence alone."""
    print(f"case {sequences} sequences, row of {owner}", flush=True)
    ints = lambda a: torch.tensor(np.asarray(a, np.int32), device="cuda")  # noqa: E731
    rope = q3q4.Rope(torch.rand(64, device="cuda"), torch.rand(128, device="cuda"), torch.rand(128, device="cuda"))
    q, k, v = (torch.randn(1, n, device="cuda") for n in (8192, 1024, 1024))
    got = []
    for n in (1, sequences):
        at = owner if n > 1 else 0
        cache = q3q4.KVCache(ao.F16, 1, 16, 8, 128)
        cache.data.zero_()
        starts, lens = np.zeros(n + 1), np.full(n, 9)
        starts[at + 1:] = 1
        batch = q3q4.KVBatch(ints(starts), ints(lens), torch.zeros(n, 1, dtype=torch.int32, device="cuda"), 1, 1, 16)
        out = torch.full_like(q, 7.0)
        q3q4.kv_write_rope(cache, batch, rope, q, out, k, v)
        torch.cuda.synchronize()
        got.append((out, cache.data))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1]) and got[0][1].any()
