"""Single precision steps on the GPU, held to the bounds of step_precision (which test_step_precision shows to be broken
without them): the angle of a rotation, the norm of attention weights, the sums of log probabilities."""
import numpy as np
import pytest

import attn_oracle as ao
import q3q4
import step_precision as sp
from test_gpu_attention import Setup, torch  # noqa: F401  (torch: the fixture)

pytestmark = pytest.mark.gpu


def held(got, want, bound, what):
    off = np.abs(np.asarray(got, np.float64) - np.asarray(want, np.float64))
    print(f"  {what} worst {np.max(off / bound):.3f} of the bound", flush=True)
    assert (off <= bound).all(), f"{what}: first at {np.argwhere(off > bound)[0]}"


@pytest.mark.parametrize("pairing", [q3q4.ROPE_HALVES, q3q4.ROPE_NEIGHBOURS])
def test_sines_and_cosines(torch, pairing):  # noqa: F811
    """Pairs of (1, 0) turn into the cosine and the sine."""
    at, f, c, s = sp.angle_cases()
    n = len(at)
    cache = q3q4.KVCache(ao.F16, -(-n // 16), 16, 1, 128)
    ints = lambda a: torch.tensor(np.asarray(a, np.int32), device="cuda")  # noqa: E731
    batch = q3q4.KVBatch(ints([0, n]), ints([n]), ints(np.arange(-(-n // 16)))[None], n, n, n)
    pick = (slice(0, 64), slice(64, 128)) if pairing == q3q4.ROPE_HALVES else (slice(0, 128, 2), slice(1, 128, 2))
    q, k = torch.zeros(n, 128, device="cuda"), torch.zeros(n, 128, device="cuda")
    q[:, pick[0]] = 1
    q3q4.kv_write_rope(cache, batch, q3q4.Rope(torch.from_numpy(f).cuda(), pairing=pairing), q, q, k, k, ints(at))
    out = q.cpu().numpy()
    for name, p, want in zip(("cosine", "sine"), pick, (c, s)):
        want = want.astype(np.float64)
        held(out[:, p], want, sp.angle_bound(want, at, f), name)


@pytest.mark.parametrize("new,length", [(1, 16), (2, 12), (12, 12), (16, 16)])
def test_weights_of_equal_scores(torch, new, length):  # noqa: F811
    """q of 0 over 8-bit caches whose values' scales are near 2^90, the same for all positions: few rows and many."""
    want = sp.equal_weights(new, length, 8)
    for scale in sp.SCALES:
        s = Setup(torch, ao.Q8, "float32", [new], [length], heads=8, kv_heads=1)
        s.views()[3][:] = scale
        cache, batch = s.device()
        q, weights = torch.zeros(new, 1024, device="cuda"), torch.empty(1, 1, length, device="cuda")
        q3q4.attention_weights(cache, batch, q, torch.empty_like(q), 0.1, weights,
                               workspace=q3q4.attention_weights_workspace(cache, batch, 8))
        held(weights[0, 0].cpu().numpy(), want, sp.weights_bound(want), f"{new} of {length}, scale {scale:.4g}")


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("new,length", [(1, 11), (1, 12), (2, 13)])
def test_weights_of_equal_scores_far_from_zero(torch, kind, new, length):  # noqa: F811
    """Few rows: the norm keeps all bits of scores of 10^5."""
    want = sp.equal_weights(new, length, 8)
    s = Setup(torch, kind, "float32", [new], [length], heads=8, kv_heads=1)
    k, _, ks, _ = s.views()
    k[:] = 1
    if ks is not None:
        ks[:] = 1
    cache, batch = s.device()
    for size in sp.SIZES:
        q, weights = torch.full((new, 1024), size, device="cuda"), torch.empty(1, 1, length, device="cuda")
        q3q4.attention_weights(cache, batch, q, torch.empty_like(q), 1.0, weights,
                               workspace=q3q4.attention_weights_workspace(cache, batch, 8))
        held(weights[0, 0].cpu().numpy(), want, sp.weights_bound(want), f"{new} of {length}, q of {size}")


def peaked_on_gpu(torch, x, at, io, wide):  # noqa: F811
    """(the logits as they are held, entropy, log probability of the token that stands out) of rows `wide` apart."""
    rows, vocab = x.shape
    y = torch.zeros(rows, wide, dtype=getattr(torch, io), device="cuda")[:, :vocab]
    y.copy_(torch.from_numpy(x))
    given, entropy = torch.empty(rows, 1, device="cuda"), torch.empty(rows, device="cuda")
    q3q4.logprobs(y, torch.from_numpy(at.astype(np.int32))[:, None].cuda(), given, entropy, workspace=q3q4.logprobs_workspace(y))
    return y.float().cpu().numpy(), entropy.cpu().numpy(), given[:, 0].cpu().numpy()


@pytest.mark.parametrize("io", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows", [1, 600])
@pytest.mark.parametrize("height", [14.0, 20.0, 30.0])
def test_entropy_beside_a_token_that_stands_out(torch, io, rows, height):  # noqa: F811
    x, at = sp.peaked(rows, 20000, height, rows)
    v, *got = peaked_on_gpu(torch, x, at, io, 20000)
    bound = sp.peaked_bound(v, at)
    for name, g, want, lost in zip(("entropy", "log probability"), got, sp.peaked_exact(v, at), sp.peaked_among_16(v, at)):
        held(g, want, bound * np.abs(want) + lost, f"{name} {io} {rows} rows {height}")


@pytest.mark.parametrize("io", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows", [1, 600])
@pytest.mark.parametrize("height", [14.0, 20.0, 30.0])
def test_entropy_beside_a_token_that_stands_out_alone(torch, io, rows, height):  # noqa: F811
    """The last token of rows that start at 16-byte borders and have one more than whole 16-byte units: it is added up with
    no other in 32 bits."""
    x, at = sp.peaked(rows, 20001, 1.0, rows)
    at[:] = 20000
    x[:, 20000] = height
    v, *got = peaked_on_gpu(torch, x, at, io, 20008)
    bound = sp.peaked_bound(v, at)
    for name, g, want in zip(("entropy", "log probability"), got, sp.peaked_exact(v, at)):
        held(g, want, bound * np.abs(want), f"{name} {io} {rows} rows {height}")
