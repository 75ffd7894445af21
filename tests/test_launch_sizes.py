"""Batches whose bounds need a launch of 2^32 threads or more in a dimension, which no launch has: they are refused before
anything is launched. No GPU, and nothing here gets as far as a launch."""
import pytest

from test_step_host import L, call  # noqa: F401  (L: the fixture)

FAR = dict(max_kv=1 << 28, table_stride=1 << 30, new_stride=1 << 30, stride=1 << 28, new_weights=1 << 44)


@pytest.mark.parametrize("kv_heads,keep,fits", [(64, 1 << 28, False), (2, 1 << 28, False), (1, 1 << 28, True), (1024, 1 << 19, False),
                                                (1024, (1 << 19) - 32, True), (64, 1 << 20, True)])
def test_evictions_of_more_positions_than_a_launch_moves(L, kv_heads, keep, fits):  # noqa: F811
    """A workgroup of 256 threads for 32 positions of a kv head. What fits is refused for what is missing besides."""
    rc, err = call(L, "evict", kv_heads=kv_heads, keep=keep, kept=None, **FAR)
    assert rc == -1 and ("kept must be" if fits else "one launch") in err, (rc, err)


@pytest.mark.parametrize("kv_heads,max_kv,fits", [(64, 1 << 28, False), (1024, 1 << 24, False), (1024, (1 << 24) - 1024, True),
                                                  (63, 1 << 28, True)])
def test_sums_of_more_positions_than_a_launch_has(L, kv_heads, max_kv, fits):  # noqa: F811
    """A workgroup of 256 threads for 1024 positions of a kv head."""
    rc, err = call(L, "weights", kv_heads=kv_heads, heads=kv_heads, max_kv=max_kv, table_stride=1 << 30, qs=1 << 20, os=1 << 20,
                   stride=max_kv, before=1 << 50, ws=None)
    assert rc == -1 and ("workspace must be" if fits else "one launch") in err, (rc, err)
