"""The example that runs norm, products, cache and attention together: a prompt and branches of it, steps from a graph.

Its errors are relative to the largest result of a head. The attention kernel's own bound (attn_oracle.attend) is 2 *
2^-19 (sum|q k| scale + 1) + 2^-20 of the largest value; scores here have sum|q k| scale of at most a few tens and
results are means of values of size 1 over up to 203 positions, a quarter of the largest or more: 2^-11 covers both.
"""
import os
import sys

import pytest

import q3q4

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


@pytest.mark.parametrize("kind", [q3q4.KV_F16, q3q4.KV_Q8])
@pytest.mark.parametrize("prompt,branches,steps", [(200, 4, 3), (64, 2, 2), (1, 1, 1)])
def test_prompt_and_branches(kind, prompt, branches, steps):
    import cached_attention
    errors = cached_attention.run(kind, prompt, branches, steps)
    print(errors, flush=True)
    assert len(errors) == 1 + steps and all(0 < e < 2.0 ** -11 for e in errors)
