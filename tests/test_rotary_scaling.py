"""The frequencies scaled by ``yarn``, pair by pair from what a pair's turns say (CPU)."""
import math

import pytest
import torch

import hmx


def _turns(rotary_dim, base, start, i):
    return start * base ** (-2 * i / rotary_dim) / (2 * math.pi)


@pytest.mark.parametrize("rotary_dim,base,start,fast,slow", [
    (128, 1e6, 32768, None, None), (64, 1e4, 4096, 32.0, 1.0), (128, 1.5e5, 4096, 32, 1), (64, 5e5, 8192, 8.0, 4.0),
    (32, 1e4, 2048, 64.0, 0.5), (128, 1e4, 4096, 100.0, 100.0), (64, 1e4, 512, 1000.0, 1.0), (16, 100.0, 4096, 2.0, 1.0),
    (64, 1e4, 4096, 4000.0, 1000.0)])
def test_yarn_pair_by_pair(rotary_dim, base, start, fast, slow):
    """Kept where a pair turns `fast` times, over s where it turns less than `slow`, and on a
    straight line in i between the last kept and the first whole one."""
    s, R = 6.0, rotary_dim // 2
    scaling = dict(rope_type="yarn", factor=s, original_max_position_embeddings=start, beta_fast=fast, beta_slow=slow)
    got, factor = hmx.rotary_frequencies(rotary_dim, base, scaling, device="cpu")
    fast, slow = fast or 32.0, slow or 1.0
    plain = [base ** (-2 * i / rotary_dim) for i in range(R)]
    turns = [_turns(rotary_dim, base, start, i) for i in range(R)]
    # the last i that turns `fast` times, or 0, and the first that turns at most `slow` times
    low = max([i for i in range(rotary_dim) if _turns(rotary_dim, base, start, i) >= fast], default=0)
    high = next((i for i in range(rotary_dim) if _turns(rotary_dim, base, start, i) <= slow), rotary_dim - 1)
    for i in range(R):
        if turns[i] >= fast:
            mix = 0.0
        elif turns[i] < slow:
            mix = 1.0
        else:
            mix = (i - low) / (high - low) if high > low else 1.0
        want = plain[i] * (1 - mix) + plain[i] / s * mix
        assert abs(got[i].item() - want) <= 1e-12 * want, (i, turns[i], got[i].item() / plain[i], want / plain[i])
    assert abs(factor - (0.1 * math.log(s) + 1)) < 1e-15
