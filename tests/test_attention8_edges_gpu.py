"""Ends of what the ops over caches of 8 bits, shared prefixes and the rotation take: the longest
table rows, and outputs that graphs have saved."""
import pytest
import torch

import hmx

pytestmark = pytest.mark.gpu
BF, F16, F8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


@pytest.mark.parametrize("eight", [True, False])
def test_the_longest_table_rows(dev, eight):
    """2^31 - 320 keys of one page of 64, listed over and over: rows asked for ahead of a share's end
    pass 2^31.  Scores of 0 and whole values up to 8, so a wave's sums (2^20 keys) are exact, and
    the mean is off by the joining of at most 512 workers' shares in fp32 and one rounding."""
    page, D = 64, 64
    keys = (1 << 31) - 320
    gen = torch.Generator().manual_seed(0)
    k, v = (torch.randint(0, 9, (1, page, 1, D), generator=gen).float() for _ in range(2))
    kc, vc = (x.to(F8 if eight else BF).to(dev) for x in (k, v))
    sc = {n: torch.full((1, 1, page), 127, dtype=torch.uint8, device=dev) for n in ("k_scales", "v_scales")} if eight else {}
    table = torch.zeros(1, keys // page, dtype=torch.int32, device=dev)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)
    n, q = i32(keys), torch.zeros(2, 4, D, dtype=BF, device=dev)
    outs = [hmx.shared_prefix_attention_decode(q, kc, vc, table[:, :1].expand(2, 1), i32(0, 0), table, n, **sc)]
    if eight:
        outs += [hmx.paged_attention_decode(q[:1], kc, vc, table, n, **sc),
                 hmx.paged_causal_attention(q, kc, vc, table, n, i32(0, 2), **sc)]
    want = v[0, :, 0].double().mean(0)
    for o in outs:
        assert ((o.double().cpu() - want).abs() <= (2.0 ** -8 + 520 * 2.0 ** -24) * want).all()


def test_rotating_in_place_beside_graphs(dev):
    """A graph that has saved what q_out or k_out writes over refuses its backward, as torch's own
    operations in place make it; tensors that need a gradient themselves are no outputs."""
    pos, (inv, _) = torch.arange(5, device=dev), hmx.rotary_frequencies(64, device=dev)
    x = torch.randn(1, 5, 2, 64, device=dev, dtype=BF).requires_grad_()
    for name in ("q_out", "k_out"):
        y = x * 2
        z = (y * y).sum()                                                # saves y
        other, mine = torch.zeros_like(x), y.detach()
        q, k = (mine, other) if name == "q_out" else (other, mine)
        hmx.rotary_embedding(q, k, pos, inv, **{name: mine})
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            z.backward()
        with pytest.raises(ValueError, match="gradient"):
            hmx.rotary_embedding(other, other, pos, inv, **{name: x})
        with torch.no_grad():
            assert hmx.rotary_embedding(other, other, pos, inv, **{name: x})[name == "k_out"] is x
    with torch.inference_mode():
        t = torch.ones(5, 2, 64, device=dev, dtype=BF)
        assert hmx.rotary_embedding(t, None, pos, inv, q_out=t)[0].shape == t.shape


@pytest.mark.parametrize("eight", [True, False])
def test_an_append_that_rotates_in_place_beside_graphs(dev, eight):
    """q_out that a graph has saved counts as written."""
    kc, vc = (torch.zeros(1, 16, 2, 64, dtype=torch.uint8 if eight else BF, device=dev) for _ in range(2))
    sc = {n: torch.ones(1, 2, 16, dtype=torch.uint8, device=dev) for n in ("k_scales", "v_scales")} if eight else {}
    kc, vc = (x.view(F8) if eight else x for x in (kc, vc))
    x = torch.randn(5, 2, 64, device=dev, dtype=BF).requires_grad_()
    at, table = torch.arange(5, device=dev), torch.rand(9, 64, device=dev)
    y = x * 2
    z = (y * y).sum()
    mine = y.detach()
    got = hmx.append_paged_kv(torch.ones_like(mine), torch.ones_like(mine), kc, vc, at, q=mine, positions=at, cos_sin=table, q_out=mine, **sc)
    assert got is mine
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()


def test_outputs_of_attention_beside_graphs(dev):
    """``out`` that a graph has saved counts as written, whichever op writes it."""
    kc, vc = (torch.zeros(2, 16, 2, 64, dtype=BF, device=dev) for _ in range(2))
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)
    q, table, lens = torch.ones(2, 4, 64, dtype=BF, device=dev), i32(0, 1)[:, None], i32(9, 3)
    kv = torch.ones(1, 2, 2, 64, dtype=BF, device=dev)
    calls = [lambda out: hmx.paged_attention_decode(q, kc, vc, table, lens, out=out),
             lambda out: hmx.paged_causal_attention(q, kc, vc, table, lens, i32(0, 1, 2), out=out),
             lambda out: hmx.shared_prefix_attention_decode(q, kc, vc, table, lens, table[:1], lens[:1], out=out),
             lambda out: hmx.causal_attention(q[None], kv, kv, out=out[None])]
    x = torch.randn(2, 4, 64, device=dev, dtype=BF).requires_grad_()
    for call in calls:
        y = x * 2
        z = (y * y).sum()
        call(y.detach())
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            z.backward()
        with torch.inference_mode():
            call(torch.empty_like(q))
