"""Calls at the edges of what the attention ops accept, against the float64 definitions.

Tolerances are elementwise and derived in attn_util.o_tolerance."""
import pytest
import torch

import hmx
from attn_util import bounds_of, check_o, paged, randn, ref

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


@pytest.mark.parametrize("page,at", [(16, 32), (16, 48), (32, 32), (8, 40), (16, 0), (8, 24)])
@pytest.mark.parametrize("H,HKV,D", [(4, 1, 128), (14, 2, 64)])
def test_missing_pages_beside_every_cut_of_the_keys(dev, page, at, H, HKV, D):
    """Few rows behind long contexts, whose keys are split at multiples of 64; in each 64 keys
    one page lies outside the cache, so one does right behind (or before) every cut."""
    gen = torch.Generator().manual_seed(page + at)
    lens, news = [9000, 5003, 700], [3, 1, 5]
    kc, vc, table, ks, vs = paged(gen, lens, page, HKV, D, BF)
    keep = []
    for n, L in enumerate(lens):
        key = torch.arange(L)
        gone = (key % 64 // page == at // page) & (key < L - 64)
        table[n, key[gone] // page] = torch.where(key[gone] // 64 % 2 == 0, -1, kc.shape[0]).to(torch.int32)
        keep.append((table[n, key // page] >= 0) & (table[n, key // page] < kc.shape[0]))
    cu = [0, 3, 4, 9]
    q = randn(gen, cu[-1], H, D)
    out = hmx.paged_causal_attention(q.to(dev), kc.to(dev), vc.to(dev), table.to(dev),
                                     torch.tensor(lens, dtype=torch.int32, device=dev),
                                     torch.tensor(cu, dtype=torch.int32, device=dev))
    for n, (b, e) in enumerate(bounds_of(cu)):
        # the new tokens are past the missing pages, so the last keys stay the last
        k, v = ks[n][keep[n]], vs[n][keep[n]]
        o, a = ref.rows(q[b:e], k, v, D ** -0.5, len(k) - (e - b))
        check_o(out[b:e], o, a, v, f"sequence {n}")
