"""sera_attention_weights on the GPU: rows that see positions whose scores are all -inf have no softmax. They come out as
NaN, and so do the sums of all that they see; rows in front of a sequence's start, whose scores are as empty, add nothing.
"""
import numpy as np
import pytest

import attn_oracle as ao
import q3q4
from test_gpu_attention import BF16, F32, Setup, torch  # noqa: F401  (torch: the fixture)

pytestmark = pytest.mark.gpu


def call(torch, s, q, scale, window=0, sinks=0):  # noqa: F811
    s.device()
    out, weights = torch.full_like(q, 7.0), torch.full((len(s.lens), s.kv_heads, max(s.lens) + 5), 9.0, device="cuda")
    ws = q3q4.attention_weights_workspace(s.cache, s.batch, s.heads)
    ws.fill_(0xFF)
    q3q4.attention_weights(s.cache, s.batch, q, out, scale, weights, None, window, sinks, workspace=ws)
    torch.cuda.synchronize()
    return out, weights


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("io", [F32, BF16])
@pytest.mark.parametrize("news,lens", [([1], [1]), ([1], [300]), ([2], [5000]), ([40], [40]), ([70], [3000]), ([50, 3], [7, 1]),
                                       ([60, 1, 1], [900, 2000, 1])])
def test_rows_whose_scores_are_all_minus_infinity(torch, kind, io, news, lens):  # noqa: F811
    """Scores of -128 times a scale near fp32's largest number."""
    print(f"case kind={kind} io={io} {news} of {lens}", flush=True)
    s = Setup(torch, kind, io, news, lens, heads=8, kv_heads=1, page=16)
    k, _, ks, _ = s.views()
    k[:] = -1
    if ks is not None:
        ks[:] = 1
    q = torch.ones(s.rows, s.heads * s.dim, dtype=getattr(torch, io), device="cuda")
    out, weights = call(torch, s, q, 2e38)
    for b, (n, length) in enumerate(zip(news, lens)):
        rows = out[s.starts[b]:s.starts[b] + n]
        front = max(n - length, 0)
        assert (rows[:front] == 0).all() and torch.isnan(rows[front:]).all(), f"rows of sequence {b}"
        assert torch.isnan(weights[b, :, :length]).all(), f"sums of sequence {b}"
        assert (weights[b, :, length:] == 9.0).all()


@pytest.mark.parametrize("new", [1, 40])
def test_keys_of_minus_infinity(torch, new):  # noqa: F811
    """Infinite keys in the first positions, rows of one sign in 16 bits: the rows that see nothing else are NaN, and with
    them all that they see; over finite keys as well such a position has no weight, and where no row is without a finite
    one, the sums are finite."""
    s = Setup(torch, ao.F16, BF16, [new], [new], heads=8, kv_heads=1, page=16)
    k, _, _, _ = s.views()
    k[:] = np.abs(k)
    for j in range(min(new, 5)):
        k[s.table[0][j // 16], :, j % 16, 3] = -np.inf
    q = (torch.rand(new, 1024, device="cuda") + 0.5).bfloat16()
    out, weights = call(torch, s, q, 0.1)
    empty = min(new, 5)
    assert torch.isnan(out[:empty]).all() and torch.isfinite(out[empty:]).all()
    assert torch.isnan(weights[..., :empty]).all() and torch.isfinite(weights[..., empty:new]).all()
    if new > 5:                     # a window that ends before them, and one that only late rows have: sinks of 5
        s = Setup(torch, ao.F16, BF16, [new - 10], [new], heads=8, kv_heads=1, page=16)
        k, _, _, _ = s.views()
        k[:] = np.abs(k)
        for j in range(5):
            k[s.table[0][j // 16], :, j % 16, 3] = -np.inf
        out, weights = call(torch, s, q[10:], 0.1, 4, 5)
        assert torch.isfinite(out).all() and (weights[..., :5] == 0).all() and torch.isfinite(weights[..., :new]).all()
