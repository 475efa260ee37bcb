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


def test_one_of_two_scales_is_refused():
    """Never taken for a cache of 16 bits, nor dropped beside one."""
    m = torch.device("meta")
    q, k = torch.empty(5, 4, 64, dtype=BF, device=m), torch.empty(5, 2, 64, dtype=BF, device=m)
    sc = torch.empty(3, 2, 16, dtype=torch.uint8, device=m)
    tab, n = torch.empty(5, 2, dtype=torch.int32, device=m), torch.empty(5, dtype=torch.int32, device=m)
    for kv in (torch.empty(3, 16, 2, 64, dtype=t, device=m) for t in (BF, F8)):
        for one in (dict(k_scales=sc), dict(v_scales=sc)):
            for call in (lambda: lib.append_paged_kv(k, k, kv, kv.clone(), n, **one),
                         lambda: lib.paged_attention_decode(q, kv, kv, tab, n, **one),
                         lambda: lib.paged_causal_attention(q, kv, kv, tab, n, n, **one),
                         lambda: lib.shared_prefix_attention_decode(q, kv, kv, tab, n, tab[:1], n[:1], **one)):
                with pytest.raises(ValueError, match="k_scales and v_scales"):
                    call()
