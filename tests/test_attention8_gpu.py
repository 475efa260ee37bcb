"""The ops over a cache of 8 bits: the append against the operations it is made of, bit by bit,
and against float64; decode and new tokens over it against float64 of what the cache stands for."""
import pytest
import torch

import hmx
from attn_util import bounds_of, check_o, half_step, paged8, randn, ref

pytestmark = pytest.mark.gpu
BF, F16, F8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def _turn32(x, cos_sin, inter):
    """The rotation in fp32, every product and sum rounded."""
    x = x.float()
    R = cos_sin.shape[1]
    c, s = cos_sin[:, None, :R // 2].float(), cos_sin[:, None, R // 2:].float()
    a, b = (slice(0, R, 2), slice(1, R, 2)) if inter else (slice(0, R // 2), slice(R // 2, R))
    y = x.clone()
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    return y


def _empty8(pages, page, HKV, D, dev, split=False):
    if split:                                   # both halves of one allocation, heads first
        both = torch.zeros(pages, 2, HKV, page, D, dtype=torch.uint8, device=dev).view(F8)
        kc, vc = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
        sc = torch.zeros(2, pages, HKV, page + 5, dtype=torch.uint8, device=dev)
        return kc, vc, sc[0, ..., :page], sc[1, ..., :page]
    kv = torch.zeros(2, pages, page, HKV, D, dtype=torch.uint8, device=dev).view(F8)
    sc = torch.zeros(2, pages, HKV, page, dtype=torch.uint8, device=dev)
    return kv[0], kv[1], sc[0], sc[1]


@pytest.mark.parametrize("T,H,HKV,D,R,inter,page,dtype,split", [
    (1, 4, 2, 64, 64, False, 16, BF, False), (37, 6, 3, 128, 128, False, 16, BF, True),
    (200, 2, 2, 128, 64, True, 7, F16, False), (65, 8, 1, 64, 16, False, 528, F16, True),
    (1000, 3, 3, 128, 0, False, 48, BF, False)])
def test_append_to_8_bits(dev, T, H, HKV, D, R, inter, page, dtype, split):
    gen = torch.Generator().manual_seed(T)
    q, k, v = (randn(gen, T, h, D, dtype=dtype) for h in (H, HKV, HKV))
    k *= torch.exp2(torch.randint(-9, 9, (T, HKV, 1), generator=gen).float()).to(dtype)
    pages = -(-T // page) + 2
    slots = torch.randperm(pages * page, generator=gen)[:T]
    if T > 4:
        slots[3], slots[4] = -1, pages * page   # padding
    pos = torch.randint(0, 99, (T,), generator=gen)
    ang = torch.rand(99, max(R, 2) // 2, generator=gen) * 7
    cs = torch.cat([ang.cos(), ang.sin()], 1)
    kc, vc, ks, vs = _empty8(pages, page, HKV, D, dev, split)
    rope = dict(q=q.to(dev), positions=pos.to(dev), cos_sin=cs.to(dev), interleaved=inter) if R else {}
    got = hmx.append_paged_kv(k.to(dev), v.to(dev), kc, vc, slots.to(dev), k_scales=ks, v_scales=vs, **rope)
    keep = (slots >= 0) & (slots < pages * page)
    at = slots[keep]
    kf = _turn32(k, cs[pos], inter) if R else k.float()
    for x, cache, scales in ((kf, kc, ks), (v.float(), vc, vs)):
        values, e = ref.quantise(x[keep])
        cache, scales = cache.float().cpu(), scales.cpu().long()
        want = torch.zeros(pages, page, HKV, D, dtype=torch.float64)
        want[at // page, at % page] = values
        assert torch.equal(cache.double(), want)
        codes = torch.zeros(pages, page, HKV, dtype=torch.long)
        codes[at // page, at % page] = (e + 127).long()
        assert torch.equal(scales, codes.transpose(1, 2))
    if R:
        want = ref.rotate(q, cs, pos, inter)
        # one rounding, beside three of fp32 for each of two terms of at most |x1| + |x2| < 16
        assert ((got.cpu().double() - want).abs() <= half_step(dtype) * want.abs() + 2.0 ** -18).all()


def test_rows_at_the_ends_of_the_scales(dev):
    """Zeros, subnormals, the types' largest values, magnitudes at and just past a scale's, and
    what is not finite."""
    rows = []
    for x in (0.0, 1e-39, 2.0 ** -133, 2.0 ** -126 * 1.5, 448.0, 450.0, 1.75 * 2.0 ** 40, 1.7578125 * 2.0 ** 40, 3.3e38):
        r = torch.full((64,), x * 0.37)
        r[5] = -x
        rows.append(r)
    bad = torch.linspace(-3, 3, 64)
    bad[7], bad[9], bad[11] = float("inf"), float("nan"), float("-inf")
    rows += [bad, torch.full((64,), float("nan"))]
    for dtype in (BF, F16):
        k = torch.stack(rows).to(dtype)[:, None]
        T = len(k)
        kc, vc, ks, vs = _empty8(2, 16, 1, 64, dev)
        hmx.append_paged_kv(k.to(dev), k.flip(0).to(dev), kc, vc, torch.arange(T, device=dev), k_scales=ks, v_scales=vs)
        for x, c, s in ((k, kc, ks), (k.flip(0), vc, vs)):
            values, e = ref.quantise(x)
            got = c.flatten(0, 1)[:T].cpu().double()
            assert torch.equal(torch.isnan(got), torch.isnan(values)) and torch.equal(got.nan_to_num(), values.nan_to_num())
            assert torch.equal(s.cpu().transpose(1, 2).reshape(-1, 1)[:T].long(), (e + 127).long())


def _take_out(table, kl, vl, page, holes, pages):
    """Pages (sequence, page of its row) put outside the cache, where they hold no keys."""
    for n in {n for n, _ in holes}:
        out = [p for m, p in holes if m == n]
        for p in out:
            table[n, p] = -1 if p % 2 else pages
        j = torch.tensor([x // page not in out for x in range(kl[n].shape[0])])
        kl[n], vl[n] = kl[n][j], vl[n][j]


def _decode(dev, lens, G, HKV, D, page, dtype, seed=0, holes=(), width=None, grow=1.0):
    gen = torch.Generator().manual_seed(seed)
    kc, vc, ks, vs, table, kl, vl = paged8(gen, lens, page, HKV, D, grow=grow, width=width)
    q = randn(gen, len(lens), G * HKV, D, dtype=dtype, scale=0.5)
    _take_out(table, kl, vl, page, holes, kc.shape[0])
    o = hmx.paged_attention_decode(q.to(dev), kc.to(dev), vc.to(dev), table.to(dev),
                                   torch.tensor(lens, dtype=torch.int32, device=dev), k_scales=ks.to(dev),
                                   v_scales=vs.to(dev))
    for n in range(len(lens)):
        want, a = ref.rows(q[n:n + 1], kl[n], vl[n], D ** -0.5, kl[n].shape[0] - 1)
        check_o(o[n:n + 1].cpu(), want, a, vl[n], f"sequence {n} of {lens[n]}")


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [16, 7, 48])
def test_decode_lengths(dev, D, page, dtype):
    _decode(dev, [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 0, 300], 4, 2, D, page, dtype)


@pytest.mark.parametrize("G,HKV", [(1, 3), (7, 2), (16, 1), (17, 1), (40, 2)])
def test_decode_groups(dev, G, HKV):
    _decode(dev, [130, 1, 77], G, HKV, 128, 16, BF, seed=G)


@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF)])
def test_decode_cut_over_workers(dev, D, dtype):
    _decode(dev, [5003, 0, 3, 2049, 1, 64, 1999], 2, 2, D, 16, dtype, seed=5)
    _decode(dev, [9000], 3, 1, D, 528, dtype, seed=6, width=40)


@pytest.mark.parametrize("page", [16, 24])
def test_decode_missing_pages(dev, page):
    _decode(dev, [200, 90, 1500], 4, 2, 128, page, BF, seed=7, holes=((0, 0), (0, 3), (1, 3), (2, 5), (2, 40)))
    _decode(dev, [page], 4, 2, 64, page, BF, seed=8, holes=((0, 0),))


def test_decode_far_scales(dev):
    """Rows whose scales lie 2^12 apart: large values of little weight, and the other way round."""
    _decode(dev, [777, 33], 4, 2, 128, 16, BF, seed=9, grow=0.0)
    gen = torch.Generator().manual_seed(1)
    kc, vc, ks, vs, table, kl, vl = paged8(gen, [500], 16, 1, 64, grow=0.0)
    up = torch.randint(-6, 7, vs.shape, generator=gen)
    keep = vs != 255
    vs = torch.where(keep, vs.long() + up, 255).to(torch.uint8)
    up = torch.where(keep, up, 0).transpose(1, 2)
    v = vl[0] * torch.exp2(ref.gather(up[..., None].double(), table[0], 500))
    q = randn(gen, 1, 4, 64, dtype=BF, scale=0.5)
    o = hmx.paged_attention_decode(q.to(dev), kc.to(dev), vc.to(dev), table.to(dev),
                                   torch.tensor([500], dtype=torch.int32, device=dev), k_scales=ks.to(dev), v_scales=vs.to(dev))
    want, a = ref.rows(q, kl[0], v, 0.125, 499)
    check_o(o.cpu(), want, a, v, "far scales")


def test_decode_values_that_are_nan(dev):
    """A NaN in v reaches its column of its sequence, one in k every column; no other row."""
    gen = torch.Generator().manual_seed(3)
    lens = [50, 70, 300]
    kc, vc, ks, vs, table, kl, vl = paged8(gen, lens, 16, 2, 64)
    bad = lambda c, n, j, h, d: c.view(torch.uint8)[table[n, j // 16], j % 16, h].__setitem__(d, 0x7f)
    bad(vc, 0, 49, 0, 3)
    bad(kc, 2, 7, 1, 5)
    q = randn(gen, 3, 8, 64, dtype=BF)
    o = hmx.paged_attention_decode(q.to(dev), kc.to(dev), vc.to(dev), table.to(dev),
                                   torch.tensor(lens, dtype=torch.int32, device=dev), k_scales=ks.to(dev), v_scales=vs.to(dev)).cpu()
    want = torch.zeros(3, 8, 64, dtype=torch.bool)
    want[0, :4, 3] = True
    want[2, 4:] = True
    assert torch.equal(torch.isnan(o), want)


def _extend(dev, news, lens, G, HKV, D, page, dtype, seed=0, holes=(), gap=(0, 0), width=None):
    gen = torch.Generator().manual_seed(seed)
    kc, vc, ks, vs, table, kl, vl = paged8(gen, lens, page, HKV, D, width=width)
    cu = [gap[0]]
    for n in news:
        cu.append(cu[-1] + n)
    T = cu[-1] + gap[1]
    q = randn(gen, T, G * HKV, D, dtype=dtype, scale=0.5)
    live = [torch.ones(n, dtype=torch.bool) for n in lens]
    for n, p in holes:
        table[n, p] = -1 if p % 2 else kc.shape[0]
        live[n][p * page:(p + 1) * page] = False
    args = (q.to(dev), kc.to(dev), vc.to(dev), table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev),
            torch.tensor(cu, dtype=torch.int32, device=dev))
    sc = dict(k_scales=ks.to(dev), v_scales=vs.to(dev))
    o = hmx.paged_causal_attention(*args, **sc)
    left = torch.full_like(o, 7.0)
    assert hmx.paged_causal_attention(*args, out=left, **sc) is left
    o, left = o.cpu(), left.cpu()
    for n, (a, b) in enumerate(bounds_of(cu)):
        assert torch.equal(o[a:b], left[a:b])
        for i in range(a, b):
            m = max(lens[n] - (b - a) + (i - a) + 1, 0)
            k, v = kl[n][:m][live[n][:m]], vl[n][:m][live[n][:m]]
            want, mag = ref.rows(q[i:i + 1], k, v, D ** -0.5, k.shape[0] - 1)
            check_o(o[i:i + 1], want, mag, v, f"sequence {n}, token {i - a} of {b - a} behind {lens[n]}")
    for a, b in ((0, gap[0]), (T - gap[1], T)):
        assert (o[a:b] == 0).all() and (left[a:b] == 7).all()


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [16, 9, 64])
def test_new_tokens(dev, D, page, dtype):
    _extend(dev, [1, 5, 33, 0, 70, 3], [1, 64, 33, 10, 200, 2], 2, 2, D, page, dtype, gap=(2, 3))


@pytest.mark.parametrize("G,HKV", [(1, 1), (7, 2), (32, 1)])
def test_new_tokens_of_groups(dev, G, HKV):
    _extend(dev, [40, 2], [97, 63], G, HKV, 128, 16, BF, seed=G)


@pytest.mark.parametrize("D,dtype", [(64, BF), (128, F16)])
def test_new_tokens_behind_long_contexts(dev, D, dtype):
    _extend(dev, [4, 2, 1], [3001, 700, 1], 2, 1, D, 16, dtype, seed=2, width=300)


@pytest.mark.parametrize("page", [16, 20])
def test_new_tokens_missing_pages(dev, page):
    _extend(dev, [9, 30], [300, 150], 2, 2, 128, page, BF, seed=3, holes=((0, 0), (0, 4), (1, 7), (1, 2)))


@pytest.mark.parametrize("tokens,far", [(5, 0), (200, 0), (3, 2000)])
def test_new_tokens_values_that_are_nan(dev, tokens, far):
    """A NaN in v reaches the rows that attend it and no others, wherever it lies."""
    gen = torch.Generator().manual_seed(tokens)
    n = tokens + far
    kc, vc, ks, vs, table, kl, vl = paged8(gen, [n], 16, 1, 64, width=-(-n // 16) + 100 * bool(far))
    places = sorted({0, far, far + tokens // 2, n - 2, n - 1})
    for i, j in enumerate(places):
        vc.view(torch.uint8)[table[0, j // 16], j % 16, 0, 3 + i] = 0xff
    q = randn(gen, tokens, 2, 64, dtype=BF)
    o = hmx.paged_causal_attention(q.to(dev), kc.to(dev), vc.to(dev), table.to(dev),
                                   torch.tensor([n], dtype=torch.int32, device=dev),
                                   torch.tensor([0, tokens], dtype=torch.int32, device=dev),
                                   k_scales=ks.to(dev), v_scales=vs.to(dev)).cpu()
    want = torch.zeros(tokens, 2, 64, dtype=torch.bool)
    for i, j in enumerate(places):
        want[max(j - far, 0):, :, 3 + i] = True
    assert torch.equal(torch.isnan(o), want)


def test_half_precision_past_its_range(dev):
    """Values past fp16's range, which a cache written in bf16 may hold, count as its largest
    where prompts form them in fp16."""
    page = torch.ones(1, 16, 1, 64)
    kc, vc = page.to(F8).to(dev), (page * 448).to(F8).to(dev)
    ks = torch.full((1, 1, 16), 127, dtype=torch.uint8, device=dev)
    vs = torch.full((1, 1, 16), 127 + 8, dtype=torch.uint8, device=dev)   # 448 * 2^8 = 114688
    q = torch.zeros(20, 2, 64, dtype=F16, device=dev)
    table, lens = (torch.tensor(x, dtype=torch.int32, device=dev) for x in ([[0]], [3]))
    cu = torch.tensor([0, 20], dtype=torch.int32, device=dev)            # tokens 17 .. 19 have keys
    o = hmx.paged_causal_attention(q, kc, vc, table, lens, cu, k_scales=ks, v_scales=vs)
    # up to three probabilities of 1, exact in fp16, times 65504, over their sum by its fp32 reciprocal
    assert (o[:17] == 0).all() and ((o[17:].float() - 65504).abs() <= 32).all()
    vs -= 1                                                              # 57344
    for o in (hmx.paged_causal_attention(q, kc, vc, table, lens, cu, k_scales=ks, v_scales=vs)[17:],
              hmx.paged_attention_decode(q[:1], kc, vc, table, lens, k_scales=ks, v_scales=vs)):
        assert ((o.float() - 57344).abs() <= 32).all()


def _shared(dev, pre, cu, lens, G, HKV, D, page, dtype, eight, seed=0, holes=(), host=False, width=None, pwidth=None):
    gen = torch.Generator().manual_seed(seed)
    M, N = len(pre), len(lens)
    if eight:
        kc, vc, ks, vs, table, kl, vl = paged8(gen, pre + lens, page, HKV, D, width=max(
            [1, *(-(-n // page) for n in pre + lens), width or 0, pwidth or 0]))
        sc = dict(k_scales=ks.to(dev), v_scales=vs.to(dev))
    else:
        from attn_util import paged
        kc, vc, table, kl, vl = paged(gen, pre + lens, page, HKV, D, dtype, width=max(
            [1, *(-(-n // page) for n in pre + lens), width or 0, pwidth or 0]))
        sc = {}
    _take_out(table, kl, vl, page, holes, kc.shape[0])
    need = lambda xs: max([1, *(-(-n // page) for n in xs)])
    q = randn(gen, N, G * HKV, D, dtype=dtype, scale=0.5)
    off = None if cu is None else torch.tensor(cu, dtype=torch.int64 if host else torch.int32)
    if off is not None and not host:
        off = off.to(dev)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    tab = table.to(dev)
    o = hmx.shared_prefix_attention_decode(q.to(dev), kc.to(dev), vc.to(dev), tab[M:, :width or need(lens)], i32(lens),
                                           tab[:M, :pwidth or need(pre)], i32(pre), off, **sc).cpu()
    none = torch.zeros(0, HKV, D, dtype=kl[0].dtype)
    for n in range(N):
        m = 0 if cu is None else next((m for m in range(M) if cu[m] <= n < cu[m + 1]), None)
        pk, pv = (none, none) if m is None else (kl[m], vl[m])
        want, a = ref.behind_prefix(q[n], pk, pv, kl[M + n], vl[M + n], D ** -0.5)
        v = torch.cat([pv, vl[M + n]])
        check_o(o[n:n + 1], want[None], a[None], v, f"sequence {n}, {lens[n]} behind prefix {m}")


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("D,dtype,page", [(64, BF, 16), (128, F16, 24), (128, BF, 64), (64, F16, 7)])
def test_shared_prefixes(dev, D, dtype, page, eight):
    _shared(dev, [100], None, [1, 0, 33, 64, 65], 4, 2, D, page, dtype, eight)
    # sequences behind none before, between and after; prefixes of no keys, of one, and of no sequences
    _shared(dev, [70, 0, 1, 129, 5], [1, 4, 6, 7, 9, 9], [3, 1, 0, 17, 0, 2, 5, 40, 130, 0, 8], 2, 2, D, page, dtype, eight, seed=1)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("G,HKV", [(1, 2), (7, 1), (17, 1), (40, 2)])
def test_shared_prefix_of_groups(dev, G, HKV, eight):
    _shared(dev, [300], None, [5, 200, 31], G, HKV, 128, 16, BF, eight, seed=G)


@pytest.mark.parametrize("eight", [False, True])
def test_long_shared_prefixes(dev, eight):
    """Prefixes split over workgroups, own keys over workers, one and many sequences behind them."""
    _shared(dev, [4000], None, [1], 4, 1, 128, 16, BF, eight, seed=2)
    _shared(dev, [3000, 1000], [0, 60, 70], [1 + 7 * (i % 5) for i in range(70)], 4, 1, 64, 16, BF, eight, seed=3)
    _shared(dev, [2000], None, [3000, 5, 1500], 2, 2, 128, 48, F16, eight, seed=4)


@pytest.mark.parametrize("eight", [False, True])
def test_many_groups_and_host_offsets(dev, eight):
    pre = [1 + 13 * i % 90 for i in range(70)]
    cu = [i + i // 9 for i in range(71)]
    _shared(dev, pre, cu, [1 + i % 20 for i in range(cu[-1] + 2)], 2, 1, 64, 16, BF, eight, seed=5, host=True)


@pytest.mark.parametrize("eight", [False, True])
def test_shared_missing_pages_and_wide_tables(dev, eight):
    _shared(dev, [100], None, [50, 20], 4, 2, 128, 16, BF, eight, seed=6, holes=((0, 0), (0, 6), (1, 1), (2, 0)))
    _shared(dev, [1], None, [2], 4, 2, 128, 16, BF, eight, seed=7, width=100, pwidth=200)


def test_no_prefixes(dev):
    """Tables of no prefixes: every sequence by itself."""
    gen = torch.Generator().manual_seed(0)
    kc, vc, ks, vs, table, kl, vl = paged8(gen, [20, 0, 300], 16, 2, 64)
    q = randn(gen, 3, 4, 64).to(dev)
    args = (q, kc.to(dev), vc.to(dev), table.to(dev), torch.tensor([20, 0, 300], dtype=torch.int32, device=dev))
    sc = dict(k_scales=ks.to(dev), v_scales=vs.to(dev))
    none = torch.zeros(0, 3, dtype=torch.int32, device=dev)
    want = hmx.paged_attention_decode(*args, **sc)
    for cu in (torch.zeros(1, dtype=torch.int32, device=dev), torch.tensor([2])):
        got = hmx.shared_prefix_attention_decode(*args, none, none[:, 0], cu, **sc)
        # the join rounds once more in fp32
        assert ((got.float() - want.float()).abs() <= 2 * half_step(BF) * want.float().abs() + 1e-6).all()
