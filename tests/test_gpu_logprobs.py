"""sera_logprobs on the GPU against the 64-bit oracle.

Tolerances. A lane sums at most m = vocab / 256 + 64 exponentials (a wave has a quarter of a row or less), and
joins some ten times: in fp32 throughout the sum would be off by (m + 20) 2^-24 of itself (16 elements' are, and those are
added up in 64 bits), and each exponential by (2 |x - max| + 2) 2^-24, which for
the weights that count is below 2^-19. Their logarithm is as far off absolutely; a log probability adds the rounding of x - max and of
the result. The entropy is the difference of such a logarithm and a mean of x - max, whose terms are off as the weights are.
The top's ids are exact.
"""
import numpy as np
import pytest

import q3q4
import step_oracle as so
from test_gpu_attention import BF16, F16, F32, torch  # noqa: F401  (torch: the fixture)

pytestmark = pytest.mark.gpu


def run(torch, x, tokens=None, top=0, entropy=True, stream=None):  # noqa: F811
    rows, _ = x.shape
    dev = "cuda"
    n = 0 if tokens is None else tokens.shape[1]
    given = torch.full((rows, n), 9.0, device=dev) if n else None
    ent = torch.full((rows,), 9.0, device=dev) if entropy else None
    ids = torch.full((rows, top), 77, dtype=torch.int32, device=dev) if top else None
    lp = torch.full((rows, top), 9.0, device=dev) if top else None
    ws = q3q4.logprobs_workspace(x, top)
    if ws is not None:
        ws.fill_(0xFF)
    q3q4.logprobs(x, tokens if n else None, given, ent, ids, lp, workspace=ws, stream=stream)
    torch.cuda.synchronize()
    return tuple(None if t is None else t.cpu().numpy() for t in (given, ent, ids, lp))


def check(torch, x, tokens=None, top=0, what=""):  # noqa: F811
    got = run(torch, x, None if tokens is None else torch.from_numpy(tokens).cuda(), top)
    v = x.double().cpu().numpy()
    vocab = v.shape[1]
    eps = (vocab / 256 + 64 + 20) * 2.0 ** -24 + 2.0 ** -19
    worst = 0.0
    for r in range(len(v)):
        given, ent, ids, lp = so.scores(v[r], [] if tokens is None else tokens[r], top)
        pairs = [(np.atleast_1d(got[1][r]), np.atleast_1d(ent), np.full(1, 3 * eps * (1 + np.abs(np.nan_to_num(ent)))))]
        if tokens is not None:
            pairs.append((got[0][r], given, eps + np.abs(given) * 2.0 ** -22))
        if top:
            assert np.array_equal(got[2][r], ids), f"{what} row {r}: {got[2][r]} for {ids}"
            pairs.append((got[3][r], lp, eps + np.abs(lp) * 2.0 ** -22))
        for g, w, t in pairs:
            g = g.astype(np.float64)
            # results are fp32: from 2^128 - 2^103 on, half a step over the largest, a value rounds to an infinity
            w = np.where(np.abs(w) >= 2.0 ** 128 - 2.0 ** 103, np.copysign(np.inf, w), w)
            same = (g == w) | (np.isnan(g) & np.isnan(w))
            with np.errstate(invalid="ignore"):
                off = np.where(same, 0, np.abs(g - w))
            assert (same | (off <= t)).all(), f"{what} row {r}: {g} for {w}"
            worst = max(worst, np.nanmax(np.where(same, 0, off / t), initial=0))
    print(f"  {what} worst {worst:.3f} of the tolerance", flush=True)
    return got


def logits(torch, rows, vocab, io, seed=0, scale=2.5):  # noqa: F811
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, vocab, generator=g) * scale).to(getattr(torch, io)).cuda()


def some(rows, vocab, n, seed=1):
    return np.random.default_rng(seed).integers(0, vocab, (rows, n)).astype(np.int32)


@pytest.mark.parametrize("io", [F32, F16, BF16])
@pytest.mark.parametrize("vocab", [1, 2, 5, 63, 64, 257, 1000, 4099, 32001])
@pytest.mark.parametrize("rows", [1, 3])
def test_sizes(torch, io, vocab, rows):  # noqa: F811
    for top in (0, 1, 5, 64):
        if top <= vocab:
            check(torch, logits(torch, rows, vocab, io, vocab), some(rows, vocab, 3), top, f"{io} {rows}x{vocab} top {top}")


@pytest.mark.parametrize("io", [F32, BF16])
@pytest.mark.parametrize("rows", [1, 7, 40, 300, 700])
def test_rows_whole_and_split(torch, io, rows):  # noqa: F811
    check(torch, logits(torch, rows, 20011, io, rows), some(rows, 20011, 2), 20, f"{io} {rows} rows")


@pytest.mark.parametrize("rows", [1, 16])
def test_the_head_s_vocabulary(torch, rows):  # noqa: F811
    check(torch, logits(torch, rows, 151936, F32), some(rows, 151936, 100), 64, f"{rows} rows")
    check(torch, logits(torch, rows, 151937, F16), some(rows, 151937, 1), 10, f"{rows} rows, fp16")


@pytest.mark.parametrize("io", [F32, F16, BF16])
@pytest.mark.parametrize("first", [0, 1, 2, 3, 5, 7])
def test_strides_and_alignment(torch, io, first):  # noqa: F811
    """Rows of a wider buffer that start anywhere; what lies beside them is large and does not matter."""
    for width in (3001, 3008):
        buf = torch.full((4, width), 60000.0, dtype=getattr(torch, io), device="cuda")
        x = buf[:, first:first + 2990]
        x.copy_(logits(torch, 4, 2990, io, first))
        check(torch, x, some(4, 2990, 4), 7, f"{io} from {first} of {width}")


def test_equal_logits_come_in_the_order_of_their_ids(torch):  # noqa: F811
    for io in (F32, BF16):
        x = torch.full((2, 30000), 1.5, dtype=getattr(torch, io), device="cuda")
        x[1] = 0.0
        x[1, ::2] = -0.0
        got = check(torch, x, some(2, 30000, 2), 64, f"{io} equal")
        assert (got[2] == np.arange(64)).all()
        check(torch, logits(torch, 3, 30000, io).round(), some(3, 30000, 2), 50, f"{io} few values")


@pytest.mark.parametrize("io", [F32, BF16])
@pytest.mark.parametrize("rows", [1, 600])
def test_a_token_that_stands_out(torch, io, rows):  # noqa: F811
    """Nearly all of a row's sum in one token: the entropy is what the many small weights beside it add up to."""
    x = logits(torch, rows, 20000, io, rows, 1.0)
    at = torch.arange(rows, device="cuda") * 31 % 20000
    for height in (14.0, 20.0, 30.0):
        x[torch.arange(rows, device="cuda"), at] = height
        check(torch, x, at[:, None].int().cpu().numpy(), 3, f"{io} {rows} rows, {height}")


@pytest.mark.parametrize("vocab", [9000, 151936])
def test_orders(torch, vocab):  # noqa: F811
    """Rising and falling rows (every element, or none after the first, is a candidate), the largest at the ends."""
    up = torch.linspace(-9, 9, vocab).float()
    ends = torch.randn(vocab)
    ends[:70], ends[-70:] = 20 + torch.rand(70), 20 + torch.rand(70)
    x = torch.stack([up, up.flip(0), ends]).cuda()
    check(torch, x, some(3, vocab, 3), 64, f"orders of {vocab}")
    check(torch, x.bfloat16(), some(3, vocab, 3), 33, f"orders of {vocab}, bf16")


@pytest.mark.parametrize("io", [F32, F16, BF16])
@pytest.mark.parametrize("vocab", [900, 40000])
def test_masks(torch, io, vocab):  # noqa: F811
    """-inf and the type's lowest value as masks: most of a row, all but fewer than `top`, all but one, all."""
    lowest = torch.finfo(getattr(torch, io)).min
    x = logits(torch, 9, vocab, io)
    keep = torch.zeros(9, vocab, dtype=torch.bool)
    for r, n in enumerate((vocab // 3, 7, 1, 0, vocab // 3, 7, 1, 0, 300)):
        keep[r, torch.randperm(vocab, generator=torch.Generator().manual_seed(r))[:n]] = True
    keep = keep.cuda()
    x[:4].masked_fill_(~keep[:4], float("-inf"))
    x[4:8].masked_fill_(~keep[4:8], lowest)
    x[8].masked_fill_(~keep[8], float("-inf"))
    x[8, :40] = lowest
    got = check(torch, x, some(9, vocab, 5), 20, f"{io} masks of {vocab}")
    assert np.isnan(got[1][3]) and (got[2][3] == -1).all() and np.isfinite(got[1][7])


@pytest.mark.parametrize("vocab", [900, 40000])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_rows_without_a_distribution(torch, vocab, value):  # noqa: F811
    """A NaN or +inf anywhere: that row is NaN with ids of -1, the others are right."""
    x = logits(torch, 5, vocab, F32)
    x[1, 0], x[2, vocab - 1], x[3, vocab // 2] = value, value, value
    got = check(torch, x, some(5, vocab, 2), 9, f"{value} in {vocab}")
    assert (got[2][1:4] == -1).all() and np.isnan(got[0][1:4]).all() and np.isnan(got[3][1:4]).all() and (got[2][4] >= 0).all()


@pytest.mark.parametrize("size", [1e-30, 1e4, 1e30, 3e38])
def test_sizes_of_logits(torch, size):  # noqa: F811
    x = logits(torch, 3, 5000, F32, 2, 1.0)
    x = x.clamp(-0.999, 0.999) * size
    check(torch, x, some(3, 5000, 3), 20, f"size {size}")


def test_tokens_outside_the_vocabulary(torch):  # noqa: F811
    tokens = np.array([[-1, 0, 999, 1000], [2 ** 31 - 1, -(2 ** 31), -100, 5]], np.int32)
    got = check(torch, logits(torch, 2, 1000, F32), tokens, 3, "tokens")
    assert np.isnan(got[0]).tolist() == [[True, False, False, True], [True, True, True, False]]


def test_parts_of_the_answer(torch):  # noqa: F811
    """Each result alone is what it is among all."""
    for rows in (2, 600):
        x = logits(torch, rows, 9001, F32)
        tokens = torch.from_numpy(some(rows, 9001, 3)).cuda()
        given, ent, ids, lp = run(torch, x, tokens, 12)
        assert np.array_equal(run(torch, x, tokens, 0, False)[0], given)
        assert np.array_equal(run(torch, x, None, 0)[1], ent)
        a = run(torch, x, None, 12, False)
        assert np.array_equal(a[2], ids) and np.array_equal(a[3], lp)
        assert run(torch, x, None, 0, False) == (None,) * 4


def test_no_rows(torch):  # noqa: F811
    x = torch.empty(0, 100, device="cuda")
    q3q4.logprobs(x, torch.empty(0, 2, dtype=torch.int32, device="cuda"), torch.empty(0, 2, device="cuda"))


@pytest.mark.parametrize("rows", [2, 600])
def test_repeats_graphs_and_streams(torch, rows):  # noqa: F811
    x, tokens = logits(torch, rows, 30011, BF16), torch.from_numpy(some(rows, 30011, 2)).cuda()
    first = run(torch, x, tokens, 30)
    side = torch.cuda.Stream()
    for got in (run(torch, x, tokens, 30), run(torch, x, tokens, 30, stream=side)):
        assert all(np.array_equal(a, b) for a, b in zip(first, got))
    given, ent = torch.zeros(rows, 2, device="cuda"), torch.zeros(rows, device="cuda")
    ids, lp = torch.zeros(rows, 30, dtype=torch.int32, device="cuda"), torch.zeros(rows, 30, device="cuda")
    ws = q3q4.logprobs_workspace(x, 30)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        q3q4.logprobs(x, tokens, given, ent, ids, lp, workspace=ws)
    for seed in (3, 4, 5):
        x.copy_(logits(torch, rows, 30011, BF16, seed))
        g.replay()
        torch.cuda.synchronize()
        want = run(torch, x, tokens, 30)
        assert all(np.array_equal(t.cpu().numpy(), w) for t, w in zip((given, ent, ids, lp), want))


def test_rows_more_than_two_to_the_31_elements_apart(torch):  # noqa: F811
    stride = 3 << 28
    buf = torch.empty(3 * stride + 5000, dtype=torch.bfloat16, device="cuda")
    x = buf.as_strided((4, 5000), (stride, 1), 0)
    x.copy_(logits(torch, 4, 5000, BF16))
    check(torch, x, some(4, 5000, 3), 20, "far rows")
