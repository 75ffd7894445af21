"""The example that runs normed and rotated writes, attention weights, eviction and log probabilities together.

Its errors are relative to the largest value of a row's stage. Rotation: 2^-19 of a pair (step_oracle.heads_turned), 2^-18
of the largest. Attention and its weights: 2 * 2^-19 (sum|q k| scale + 1), where sum|q k| scale is at most sqrt(128) 1.3 *
1.3 (normed heads) and a half more for their turn: 2^-19 * 2 * 30 < 2^-13. Log probabilities of 4096 tokens: 2^-16.
"""
import os
import sys

import pytest

import q3q4

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


@pytest.mark.parametrize("kind", [q3q4.KV_F16, q3q4.KV_Q8])
@pytest.mark.parametrize("prompts,limit,keep,steps", [((70, 33), 72, 48, 12), ((90,), 80, 20, 3), ((1, 40, 17), 42, 41, 5)])
def test_a_prompt_and_steps(kind, prompts, limit, keep, steps):
    import bounded_cache
    worst, thinned = bounded_cache.run(kind, prompts, limit, keep, steps)
    print(worst, thinned, flush=True)
    assert thinned > 0 and all(e == e for e in worst.values())
    assert worst["rope"] < 2.0 ** -18 and worst["attention"] < 2.0 ** -13 and worst["weights"] < 2.0 ** -13
    assert worst["logprobs"] < 2.0 ** -16
