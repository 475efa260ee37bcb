"""The registered ops of 8-bit caches and the rotation refuse what the functions refuse (CPU)."""
import pytest
import torch

import hmx.library as lib

BF, F8 = torch.bfloat16, torch.float8_e4m3fn


def test_frequencies_that_need_a_gradient_are_refused():
    m = torch.device("meta")
    pos = torch.empty(5, dtype=torch.int32, device=m)
    inv = torch.empty(32, dtype=torch.float64, device=m, requires_grad=True)
    for grad in (False, True):
        q = torch.empty(1, 5, 4, 64, dtype=BF, device=m, requires_grad=grad)
        for call in (lambda: lib.rotary_embedding(q, None, pos, inv),
                     lambda: torch.ops.hmx.rotary_embedding(q, q, pos, inv, 1.0, False, True)):
            with pytest.raises(NotImplementedError, match="frequencies"):
                call()
            with torch.no_grad():
                assert not call()[0].requires_grad
        assert lib.rotary_embedding(q, None, pos, inv.detach())[0].requires_grad == grad
