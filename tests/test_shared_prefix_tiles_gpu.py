"""Shared prefixes with many rows behind them (more than 64 a prefix, which go in tiles) against
float64: both types and caches, odd pages, groups, gaps, empty prefixes, missing pages, many
prefixes, and values that are not finite.  Then few rows of several tokens over missing pages."""
import pytest
import torch

import hmx
from attn_util import check_o, half_step, paged, paged8, randn, ref
from test_attention8_gpu import _extend, _shared

pytestmark = pytest.mark.gpu
BF, F16, F8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def _tiles(dev, pre, cu, lens, G, *args, **kw):
    assert len(lens) * G > 64 * len(pre)
    _shared(dev, pre, cu, lens, G, *args, **kw)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("D,dtype,page", [(64, BF, 16), (64, F16, 7), (128, BF, 24), (128, F16, 16), (64, F16, 48), (128, BF, 7),
                                          (128, F16, 64)])
def test_lengths_and_gaps(dev, D, dtype, page, eight):
    """One prefix; five of no keys, of one, of whole and cut tiles, and of no sequences, with
    sequences behind none before, between and after."""
    own = lambda n: [(0, 1, 3, 17, 16, 65)[i % 6] for i in range(n)]
    _tiles(dev, [100], None, own(20), 4, 2, D, page, dtype, eight)
    for n in (1, 63, 64, 65):
        _tiles(dev, [n], None, own(9), 8, 1, D, page, dtype, eight, seed=n)
    _tiles(dev, [70, 0, 1, 129, 5], [2, 9, 14, 20, 27, 27], own(31), 11, 1, D, page, dtype, eight, seed=1)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("G,HKV,N", [(1, 2, 131), (5, 3, 27), (17, 1, 9), (128, 1, 2), (130, 1, 3)])
def test_groups(dev, G, HKV, N, eight):
    _tiles(dev, [150], None, [1 + 7 * i % 40 for i in range(N)], G, HKV, 128, 16, F16 if G % 2 else BF, eight, seed=G)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("page,dtype", [(16, BF), (24, F16), (64, F16)])
def test_missing_pages(dev, page, dtype, eight):
    """Pages outside the cache in the prefix (its first, one in the middle, its last) and among own
    keys; and a prefix of missing pages alone."""
    last = 299 // page
    _tiles(dev, [300, page], [0, 21, 30], [5 + 9 * i % 60 for i in range(32)], 6, 1, 64, page, dtype, eight, seed=2,
           holes=((0, 0), (0, 2), (0, last), (1, 0), (2, 0), (9, 0), (30, 0)))


@pytest.mark.parametrize("host", [False, True])
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("M", [62, 63, 64, 100])
def test_many_prefixes(dev, M, eight, host):
    """As many prefixes as a wave's lanes weigh, and more, which lie in their order."""
    cu = [2 + i * 2 + i // 5 for i in range(M + 1)]
    N = cu[-1] + 3
    _tiles(dev, [1 + 37 * i % 150 for i in range(M)], cu, [i % 5 for i in range(N)], 30, 1, 64, 16, BF if host else F16, eight,
           seed=M, host=host)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("D,dtype", [(64, F16), (128, F16), (128, BF)])
def test_prefixes_cut_over_workgroups(dev, D, dtype, eight):
    _tiles(dev, [3000, 1111], [0, 60, 70], [1 + 7 * i % 50 for i in range(72)], 4, 1, D, 48, dtype, eight, seed=3)
    _tiles(dev, [2500], None, [0] * 33, 2, 2, D, 16, dtype, eight, seed=4, pwidth=400)


def test_outputs_in_place_of_a_wider_one(dev):
    """Written where ``out`` lies and nowhere else, rows behind no prefix and without keys too."""
    gen = torch.Generator().manual_seed(5)
    lens, N = [200] + [i % 4 for i in range(40)], 40
    kc, vc, ks, vs, table, _, _ = paged8(gen, lens, 16, 2, 64)
    q, t, n = randn(gen, N, 8, 64).to(dev), table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev)
    args = (q, kc.to(dev), vc.to(dev), t[1:], n[1:], t[:1], n[:1], torch.tensor([3, 37]))
    sc = dict(k_scales=ks.to(dev), v_scales=vs.to(dev))
    want = hmx.shared_prefix_attention_decode(*args, **sc)
    wide = torch.full((N + 1, 9, 64), 3.0, dtype=BF, device=dev)
    out = wide[:N, 1:]
    assert hmx.shared_prefix_attention_decode(*args, out=out, **sc) is out and torch.equal(out, want)
    assert (wide[N] == 3).all() and (wide[:, 0] == 3).all() and (want[0] == 0).all()


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("prefix", [10, 64, 100, 700])
def test_values_that_are_not_finite(dev, prefix, eight):
    """In a prefix's values they reach their columns of the rows behind it, in its keys all columns of
    their key/value head, in own values that sequence's column; nobody else is touched."""
    gen = torch.Generator().manual_seed(prefix)
    N, G, HKV, D, page = 24, 8, 2, 64, 16
    lens = [prefix, prefix + 3] + [i % 5 for i in range(N)]
    if eight:
        kc, vc, ks, vs, table, kl, vl = paged8(gen, lens, page, HKV, D)
        sc = dict(k_scales=ks.to(dev), v_scales=vs.to(dev))
        put = lambda c, n, j, h, d, x: c.view(torch.uint8)[table[n, j // page], j % page, h].__setitem__(d, 0x7f)
    else:
        (kc, vc, table, kl, vl), sc = paged(gen, lens, page, HKV, D, BF), {}
        put = lambda c, n, j, h, d, x: c[table[n, j // page], j % page, h].__setitem__(d, x)
    q = randn(gen, N, G * HKV, D, scale=0.5)
    inf, nan = float("inf"), float("nan")
    bad = torch.zeros(N, G * HKV, D, dtype=torch.bool)
    a, b = slice(1, 13), slice(13, 22)                       # sequences 0, 22 and 23 are behind none
    for j, d, x in ((0, 3, inf), (prefix - 1, 5, -inf), (prefix - 1, 6, nan), (prefix // 2, 63, nan)):
        put(vc, 0, j, 0, d, x)
        bad[a, :G, d] = True
    put(kc, 1, prefix + 2, 1, 9, nan)
    bad[b, G:] = True
    for n in (4, 9, 23):                                     # own keys: (n % 5) of them
        put(vc, 2 + n, n % 5 - 1, 1, 7, nan)
        bad[n, G:, 7] = True
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    t, n = table.to(dev), i32(lens)
    assert N * G > 64 * 2
    o = hmx.shared_prefix_attention_decode(q.to(dev), kc.to(dev), vc.to(dev), t[2:], n[2:], t[:2], n[:2], i32([1, 13, 22]), **sc).cpu()
    assert torch.equal(~torch.isfinite(o), bad)
    none = torch.zeros(0, HKV, D, dtype=kl[0].dtype)
    for i in range(N):
        m = 0 if 1 <= i < 13 else 1 if 13 <= i < 22 else None
        pk, pv = (none, none) if m is None else (kl[m], vl[m])
        want, mag = ref.behind_prefix(q[i], pk, pv, kl[2 + i], vl[2 + i], D ** -0.5)
        keep = ~bad[i]
        check_o(o[i][keep], want[keep], mag[keep], torch.cat([pv, vl[2 + i]]), f"sequence {i}")


def test_half_precision_past_its_range(dev):
    """fp16 rows behind a prefix whose values pass that type's range: in tiles they count as its
    largest, few rows take them as they are; below its range both give the same."""
    page = torch.ones(2, 16, 1, 64)
    kc, vc = page.to(F8).to(dev), (page * 448).to(F8).to(dev)
    ks = torch.full((2, 1, 16), 127, dtype=torch.uint8, device=dev)
    vs = torch.full((2, 1, 16), 127 + 8, dtype=torch.uint8, device=dev)   # 448 * 2^8 = 114688
    vs[1] = 127                                                          # own values: 448
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)
    table = i32(0, 1)[:, None].expand(2, 3).contiguous()
    for N, large in ((40, 65504.0), (4, 114688.0)):
        q = torch.zeros(N, 2, 64, dtype=F16, device=dev)
        run = lambda own: hmx.shared_prefix_attention_decode(q, kc, vc, table[1:].expand(N, 3).contiguous(), i32(*[own] * N), table[:1],
                                                             i32(3), k_scales=ks, v_scales=vs).float()
        assert (N * 2 > 64) == (large == 65504.0)
        # one prefix key's weight of 3 beside 13 own: equal probabilities, exact in fp16
        want = (3 * large + 13 * 448) / 16
        assert ((run(13) - want).abs() <= 2 * half_step(F16) * want).all()
        vs[0] = 127 + 7                                                  # 57344
        assert ((run(0) - 57344).abs() <= 32).all()
        vs[0] = 127 + 8


@pytest.mark.parametrize("width", [None, 120])
@pytest.mark.parametrize("page,D,dtype", [(16, 64, BF), (20, 128, F16), (48, 128, BF), (7, 64, F16)])
def test_few_rows_of_several_tokens_over_missing_pages(dev, page, D, dtype, width):
    news, lens = [4, 1, 0, 6, 2, 3, 1], [150, 90, 33, 61, 2, 700, 1]
    assert sum(news) * 2 <= 16 * len(news)                               # those go row block by row block
    holes = ((0, 0), (0, 149 // page), (1, 1), (3, 60 // page), (3, 0), (4, 0), (5, 2), (5, 699 // page), (6, 0))
    _extend(dev, news, lens, 2, 2, D, page, dtype, seed=page, holes=holes, gap=(1, 2), width=width)
