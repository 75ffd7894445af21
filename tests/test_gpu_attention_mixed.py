"""Batches that two kernels share (a few long chunks among many single tokens), and contexts longer than the page list
that a workgroup holds at a time (16384 positions), against the 64-bit oracle. Tolerances as in test_gpu_attention.
"""
import numpy as np
import pytest

import attn_oracle as ao
import q3q4
from test_gpu_attention import BF16, F16, F32, Setup, check, close, spoil, torch  # noqa: F401  (torch: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("io", [F32, F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 2, 128), (6, 2, 64), (40, 2, 128), (34, 1, 64)])
def test_chunks_among_single_tokens(torch, kind, io, heads, kv_heads, dim):  # noqa: F811
    """Groups of 8, 3, 20 and 34 query heads (the last: no rows are few)."""
    print(f"case mixed kind={kind} io={io} heads={heads} kv_heads={kv_heads} dim={dim}", flush=True)
    news, lens = [1, 1, 90, 1, 2, 0, 1, 3, 50, 1], [300, 1, 200, 77, 64, 9, 33, 500, 50, 130]
    check(Setup(torch, kind, io, news, lens, heads=heads, kv_heads=kv_heads, dim=dim, page=32, seed=heads))


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
def test_mixed_batches_split_both_ways(torch, kind):  # noqa: F811
    """Long contexts, few workgroups: both kernels leave partial sums, in one workspace."""
    print(f"case mixed splits kind={kind}", flush=True)
    s = Setup(torch, kind, F32, [1, 70, 1, 2, 1], [4000, 3000, 20, 3500, 1], heads=8, kv_heads=1, page=64, seed=3)
    q, first = check(s)
    assert torch.equal(s.attend(q, s.dim ** -0.5), first)
    check(Setup(torch, kind, F32, [1, 70, 1, 1], [4000, 3000, 700, 90], heads=8, kv_heads=1, page=64, seed=4),
          window=600, sinks=40)


def test_mixed_rows_that_see_nothing_and_odd_values(torch):  # noqa: F811
    s = Setup(torch, ao.F16, F32, [2, 40, 1, 1], [1, 30, 0, 60], heads=8, kv_heads=2)
    q, out = check(s)
    assert (out[0] == 0).all() and (out[2:12] == 0).all() and (out[42] == 0).all()
    s = Setup(torch, ao.F16, F32, [1, 40, 1, 1], [90, 75, 33, 60], heads=8, kv_heads=2, page=64)
    for b, length in enumerate(s.lens):
        spoil(s, b, range(length, -(-length // 64) * 64), np.nan)
    _, out = check(s)
    assert torch.isfinite(out).all()


def test_mixed_sequences_outside_the_bounds(torch):  # noqa: F811
    """One sequence of each kind is longer than the host said: NaN in its rows, the others are right."""
    s = Setup(torch, ao.F16, F32, [1, 50, 1, 50, 1], [90, 80, 400, 401, 20], heads=8, kv_heads=2)
    q, qv = s.rows_of(1024)
    want, tol = s.expect(qv, 0.1)
    out = s.attend(q, 0.1, max_kv=100)
    bad = torch.zeros(103, dtype=torch.bool)
    bad[51:102] = True
    assert torch.isnan(out[bad.cuda()]).all()
    close(out[~bad.cuda()], want[~bad.numpy()], tol[~bad.numpy()], "others")


def long_case(torch, kind, sequences, new, length, window=0, sinks=0, io="float32"):  # noqa: F811
    """Sequences over the same pages; 64 bits in torch for the first and last sequence and four heads."""
    heads, kv_heads, dim, page = 64, 8, 128, 128
    s = Setup(torch, kind, io, [new], [length], heads=heads, kv_heads=kv_heads, dim=dim, page=page, seed=length)
    s.device()
    ints = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    table = s.batch.page_table.expand(sequences, -1).contiguous()
    batch = q3q4.KVBatch(ints([new * b for b in range(sequences + 1)]), ints([length] * sequences), table,
                         new * sequences, new, length)
    q = torch.randn(new * sequences, heads * dim, device="cuda").to(getattr(torch, io))
    out = torch.full_like(q, 7.0)
    q3q4.attention(s.cache, batch, q, out, 0.09, window, sinks, workspace=q3q4.attention_workspace(s.cache, batch, heads))
    K, V = (torch.from_numpy(a).cuda() for a in ao.values(s.pool, kind, page, kv_heads, dim, s.table, 0, length))
    p = torch.arange(length - new, length, device="cuda")[:, None]
    j = torch.arange(length, device="cuda")
    hid = j > p
    if window:
        hid = hid | ((j <= p - window) & (j >= sinks))
    for b in {0, sequences - 1}:
        for h in (0, 9, 40, 63):
            rows, cols = slice(new * b, new * b + new), slice(h * dim, (h + 1) * dim)
            qq = q[rows, cols].double()
            w = torch.softmax((qq @ K[h // 8].T * 0.09).masked_fill(hid, -torch.inf), -1)
            want = w @ V[h // 8]
            a = (qq.abs() @ K[h // 8].abs().T).max(1, keepdim=True).values * 0.09
            tol = V[h // 8].abs().max() * (2 * 2.0 ** -19 * (a + 1) + 2.0 ** -20) + want.abs() * 2.0 ** -24
            assert ((out[rows, cols].double() - want).abs() <= tol).all(), (b, h)


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
def test_decode_past_one_page_list(torch, kind):  # noqa: F811
    """256 workgroups of whole contexts: each lists its pages in parts."""
    long_case(torch, kind, 32, 1, 17000)
    long_case(torch, kind, 32, 1, 20001, window=16900, sinks=100)


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
def test_chunks_past_one_page_list(torch, kind):  # noqa: F811
    long_case(torch, kind, 1, 1030, 17501)


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("new,group", [(5, 8), (8, 8), (16, 8), (33, 1), (9, 5)])
def test_rows_of_the_smaller_tiles(torch, kind, new, group):  # noqa: F811
    """33 to 128 rows of a group: tiles of 64 and 128 rows, ragged ends."""
    print(f"case small tiles new={new} group={group} kind={kind}", flush=True)
    check(Setup(torch, kind, F32, [new, new - 2], [300, 41], heads=2 * group, kv_heads=2, page=16, seed=new))
    check(Setup(torch, kind, BF16, [new, new - 1], [77, 260], heads=2 * group, kv_heads=2, dim=64, page=16, seed=new))


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("io,heads", [(F32, 8), (F32, 13), (BF16, 16), (F16, 3)])
def test_many_whole_contexts(torch, kind, io, heads):  # noqa: F811
    """A workgroup for each of 150 sequences: contexts are not split, an 8-bit cache's workgroups have eight waves."""
    print(f"case whole contexts kind={kind} io={io} heads={heads}", flush=True)
    lens = [1 + (b * 37) % 600 for b in range(150)]
    check(Setup(torch, kind, io, [1] * 150, lens, heads=heads, kv_heads=1, page=64, seed=heads))
    check(Setup(torch, kind, io, [1] * 150, lens, heads=heads, kv_heads=1, dim=64, page=16, seed=heads), window=90,
          sinks=5)
