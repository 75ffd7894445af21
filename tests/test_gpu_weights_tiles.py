"""sera_attention_weights on the GPU: chunks over several 512-position tiles of the sums of many rows, in every row and cache
type, both head sizes and groups that divide 32 or do not, so that workgroups begin in the middle of a tile, and with a window
in the middle of what it leaves. Tolerance: step_oracle.weights_of.
"""
import pytest

import attn_oracle as ao
from test_gpu_attention import BF16, F16, F32, Setup, torch  # noqa: F401  (torch: the fixture)
from test_gpu_attention_weights import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [ao.F16, ao.Q8])
@pytest.mark.parametrize("io", [F32, F16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("group,window,sinks", [(3, 0, 0), (5, 600, 70), (8, 0, 0), (8, 200, 0)])
def test_chunks_over_several_tiles(torch, kind, io, dim, group, window, sinks):  # noqa: F811
    print(f"case kind={kind} io={io} dim={dim} group={group} window={window} sinks={sinks}", flush=True)
    s = Setup(torch, kind, io, [150, 40], [1700, 1100], heads=2 * group, kv_heads=2, dim=dim, page=64, seed=group + dim)
    check(torch, s, window=window, sinks=sinks)


@pytest.mark.parametrize("io", [F32, BF16])
def test_a_prompt_over_several_tiles(torch, io):  # noqa: F811
    """All rows from the first on: blocks in front of a tile's positions, and some on its diagonal."""
    check(torch, Setup(torch, ao.F16, io, [1100, 700], [1100, 701], heads=3, kv_heads=1, dim=64, page=64))
