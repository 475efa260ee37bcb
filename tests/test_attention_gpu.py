"""Attention ops on the GPU against the float64 definitions (oracle/attention.py).

Tolerances are elementwise and derived in attn_util.o_tolerance."""
import pytest
import torch

import hmx
from attn_util import bounds_of, check_o, paged, randn, ref

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def _case(seed, T, H, HKV, D, dtype, B=1):
    gen = torch.Generator().manual_seed(seed)
    return (randn(gen, B, T, H, D, dtype=dtype), randn(gen, B, T, HKV, D, dtype=dtype),
            randn(gen, B, T, HKV, D, dtype=dtype))


@pytest.mark.parametrize("T,H,HKV,D,dtype", [
    (1, 4, 4, 128, BF), (2, 4, 1, 128, BF), (31, 6, 2, 64, FP), (32, 4, 2, 128, BF),
    (33, 8, 1, 64, BF), (63, 3, 3, 128, FP), (64, 4, 4, 64, BF), (65, 14, 2, 128, BF),
    (128, 2, 2, 128, BF), (129, 5, 1, 128, BF), (257, 4, 2, 64, FP), (700, 8, 2, 128, BF),
    (1000, 7, 1, 128, FP), (300, 40, 1, 64, BF),
])
def test_causal_attention_one_sequence(dev, T, H, HKV, D, dtype):
    q, k, v = _case(T, T, H, HKV, D, dtype)
    out = hmx.causal_attention(q.to(dev), k.to(dev), v.to(dev))
    o, a = ref.causal(q[0], k[0], v[0], D ** -0.5, [(0, T)])
    check_o(out[0], o, a, v[0], f"T={T}")


def test_causal_attention_batch_and_scale(dev):
    B, T, H, HKV, D = 3, 77, 4, 2, 128
    q, k, v = _case(5, T, H, HKV, D, BF, B)
    out = hmx.causal_attention(q.to(dev), k.to(dev), v.to(dev), 0.05)
    for b in range(B):
        o, a = ref.causal(q[b], k[b], v[b], 0.05, [(0, T)])
        check_o(out[b], o, a, v[b], f"b={b}")


@pytest.mark.parametrize("cu", [[0, 5, 5, 70, 200], [0, 1, 2, 3, 130], [0, 200], [0, 64, 128, 192, 200],
                                [0, 0, 0, 150], [0, *range(1, 71), 200]])
@pytest.mark.parametrize("where", ["device", "host", "int64"])
def test_causal_attention_packed(dev, cu, where):
    """Empty sequences, lengths of one, and tokens behind the last sequence."""
    T, H, HKV, D = 200, 6, 2, 64
    q, k, v = _case(len(cu), T, H, HKV, D, BF)
    k[0, cu[-1]:], v[0, cu[-1]:] = float("nan"), float("nan")
    c = torch.tensor(cu, dtype=torch.int64 if where == "int64" else torch.int32)
    c = c if where == "host" else c.to(dev)
    args = [x.to(dev) for x in (q, k, v)]
    out = hmx.causal_attention(*args, cu_seqlens=c)
    o, a = ref.causal(q[0], k[0], v[0], D ** -0.5, bounds_of(cu))
    check_o(out[0, :cu[-1]], o[:cu[-1]], a[:cu[-1]], v[0, :cu[-1]], str(cu))
    assert (out[0, cu[-1]:] == 0).all()
    mine = torch.full_like(args[0], 7.0)
    got = hmx.causal_attention(*args, cu_seqlens=c, out=mine)
    assert got is mine and torch.equal(mine[0, :cu[-1]], out[0, :cu[-1]])
    assert (mine[0, cu[-1]:] == 7).all()


def test_causal_attention_first_offset(dev):
    """Offsets that start past 0 leave the rows before them."""
    q, k, v = _case(3, 300, 4, 2, 128, BF)
    cu = [130, 140, 290]
    out = hmx.causal_attention(q.to(dev), k.to(dev), v.to(dev),
                               cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=dev))
    o, a = ref.causal(q[0], k[0], v[0], 128 ** -0.5, bounds_of(cu))
    check_o(out[0, 130:290], o[130:290], a[130:290], v[0], "offsets")
    assert (out[0, :130] == 0).all() and (out[0, 290:] == 0).all()


def test_causal_attention_strides(dev):
    """Slices of one projection, head-major tensors, and views that need a copy."""
    T, H, HKV, D = 150, 4, 2, 128
    gen = torch.Generator().manual_seed(2)
    qkv = randn(gen, T, (H + 2 * HKV) * D).to(dev)
    q = qkv[:, :H * D].view(1, T, H, D)
    k = qkv[:, H * D:(H + HKV) * D].view(1, T, HKV, D)
    v = qkv[:, (H + HKV) * D:].view(1, T, HKV, D)
    want = hmx.causal_attention(q.contiguous(), k.contiguous(), v.contiguous())
    assert torch.equal(hmx.causal_attention(q, k, v), want)
    qt, kt, vt = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v))
    assert torch.equal(hmx.causal_attention(qt, kt, vt), want)
    odd = torch.empty(1, T, H, D + 1, dtype=BF, device=dev)[..., 1:]
    odd.copy_(q)
    assert torch.equal(hmx.causal_attention(odd, k, v), want)
    out = torch.empty(1, H, T, D, dtype=BF, device=dev).transpose(1, 2)
    assert torch.equal(hmx.causal_attention(q, k, v, out=out), want)


def test_causal_attention_peaked_and_growing_scores(dev):
    """Scores that grow along the keys by far more than the lag of the running maximum, and
    rows that one key dominates."""
    T, H, D = 600, 2, 128
    gen = torch.Generator().manual_seed(9)
    q = torch.ones(1, T, H, D)
    k = torch.linspace(-1, 1, T)[None, :, None, None].expand(1, T, H, D).clone()
    k[0, 100] = -1.5
    v = torch.randn(1, T, H, D, generator=gen)
    q, k, v = (x.to(BF) for x in (q, k, v))
    for s in (0.02, 0.1):
        out = hmx.causal_attention(q.to(dev), k.to(dev), v.to(dev), s)
        o, a = ref.causal(q[0], k[0], v[0], s, [(0, T)])
        check_o(out[0], o, a, v[0], f"scale {s}")


@pytest.mark.parametrize("bad", [float("inf"), float("nan"), float("-inf")])
def test_causal_attention_nonfinite_values_stay_behind(dev, bad):
    """A value that is not finite reaches only the rows that attend it."""
    T, H, HKV, D, at = 200, 4, 2, 64, 150
    q, k, v = _case(8, T, H, HKV, D, BF)
    v[0, at, 1, 3] = bad
    k[0, 170] = float("nan")
    out = hmx.causal_attention(q.to(dev), k.to(dev), v.to(dev))[0].double().cpu()
    o, a = ref.causal(q[0], k[0], v[0], D ** -0.5, [(0, T)])
    fine = torch.isfinite(o)
    assert fine[:at].all() and not torch.isfinite(out[at:, 2:, 3]).any()
    assert not torch.isfinite(out[170:]).any()
    clean = fine.clone()
    clean[170:] = False
    err = (out - o).abs()[clean]
    assert (err <= 0.02 * (1 + a[clean])).all()   # finite rows are the definition's
    assert torch.isfinite(out[clean]).all()


@pytest.mark.parametrize("lens,H,HKV,D,page,dtype", [
    ([1], 4, 4, 128, 16, BF), ([64], 8, 2, 128, 16, BF), ([65], 8, 1, 64, 16, FP),
    ([700], 32, 8, 128, 16, BF), ([5, 0, 33, 1, 200], 14, 2, 64, 48, FP),
    ([0, 0], 4, 2, 128, 16, BF), ([1000, 3, 0, 2500, 257], 8, 2, 128, 528, BF),
    ([300, 31], 40, 2, 64, 1, BF), ([130, 64, 32, 31, 33], 6, 3, 128, 7, FP),
    ([4100], 4, 1, 64, 256, BF),
])
def test_paged_attention_decode(dev, lens, H, HKV, D, page, dtype):
    gen = torch.Generator().manual_seed(sum(lens) + H)
    kc, vc, table, ks, vs = paged(gen, lens, page, HKV, D, dtype)
    q = randn(gen, len(lens), H, D, dtype=dtype)
    out = hmx.paged_attention_decode(q.to(dev), kc.to(dev), vc.to(dev), table.to(dev),
                                     torch.tensor(lens, dtype=torch.int32, device=dev))
    for n, L in enumerate(lens):
        o, a = ref.rows(q[n:n + 1], ks[n], vs[n], D ** -0.5, L - 1)
        check_o(out[n:n + 1], o, a, vs[n], f"sequence {n} of {L}")
        assert L > 0 or (out[n] == 0).all()


def test_paged_attention_decode_many_sequences(dev):
    """More sequences than threads of a workgroup, empty ones among them."""
    lens = [(37 * i) % 91 if i % 5 else 0 for i in range(600)]
    gen = torch.Generator().manual_seed(4)
    kc, vc, table, ks, vs = paged(gen, lens, 16, 2, 64, BF)
    q = randn(gen, 600, 4, 64)
    out = hmx.paged_attention_decode(q.to(dev), kc.to(dev), vc.to(dev), table.to(dev),
                                     torch.tensor(lens, dtype=torch.int32, device=dev))
    for n, L in enumerate(lens):
        o, a = ref.rows(q[n:n + 1], ks[n], vs[n], 64 ** -0.5, L - 1)
        check_o(out[n:n + 1], o, a, vs[n], f"sequence {n} of {L}")


@pytest.mark.parametrize("news,lens,H,HKV,D,page,dtype", [
    ([1], [1], 4, 4, 128, 16, BF), ([4, 1, 3], [500, 64, 2000], 8, 2, 128, 16, BF),
    ([70, 200, 5], [70, 333, 640], 14, 2, 64, 48, FP), ([130], [1111], 4, 1, 128, 528, BF),
    ([0, 3, 0, 9], [20, 3, 0, 100], 8, 4, 64, 7, BF), ([2] * 70, [40 + i for i in range(70)], 4, 2, 64, 16, FP),
    ([5], [3], 2, 1, 128, 16, BF),
])
def test_paged_causal_attention(dev, news, lens, H, HKV, D, page, dtype):
    """New tokens behind a context; where a sequence has fewer keys than new tokens, its
    first rows attend none and are 0."""
    gen = torch.Generator().manual_seed(sum(lens) + H)
    kc, vc, table, ks, vs = paged(gen, lens, page, HKV, D, dtype)
    T = sum(news) + 6
    q = randn(gen, T, H, D, dtype=dtype)
    cu = [2]
    for n in news:
        cu.append(cu[-1] + n)
    out = hmx.paged_causal_attention(q.to(dev), kc.to(dev), vc.to(dev), table.to(dev),
                                     torch.tensor(lens, dtype=torch.int32, device=dev),
                                     torch.tensor(cu, dtype=torch.int32, device=dev))
    for n, (b, e) in enumerate(bounds_of(cu)):
        o, a = ref.rows(q[b:e], ks[n], vs[n], D ** -0.5, lens[n] - (e - b))
        check_o(out[b:e], o, a, vs[n], f"sequence {n}")
    assert (out[:2] == 0).all() and (out[cu[-1]:] == 0).all()


def test_pages_outside_the_cache_hold_no_keys(dev):
    lens, H, HKV, D, page = [200, 90], 4, 2, 128, 16
    gen = torch.Generator().manual_seed(1)
    kc, vc, table, ks, vs = paged(gen, lens, page, HKV, D, BF)
    table[0, 3], table[0, 9], table[1, 0] = -1, 10 ** 6, kc.shape[0]
    keep = [torch.ones(n, dtype=torch.bool) for n in lens]
    keep[0][48:64] = keep[0][144:160] = keep[1][:16] = False
    dv = [x.to(dev) for x in (kc, vc, table, torch.tensor(lens, dtype=torch.int32))]
    q = randn(gen, 2, H, D)
    out = hmx.paged_attention_decode(q.to(dev), *dv)
    new = randn(gen, 9, H, D)
    out2 = hmx.paged_causal_attention(new.to(dev), *dv, torch.tensor([0, 4, 9], dtype=torch.int32))
    for n in range(2):
        k, v = ks[n][keep[n]], vs[n][keep[n]]
        o, a = ref.rows(q[n:n + 1], k, v, D ** -0.5, len(k) - 1)
        check_o(out[n:n + 1], o, a, v, f"decode {n}")
        b, e = ((0, 4), (4, 9))[n]
        # the new tokens are past the missing pages, so the last keys stay the last
        o, a = ref.rows(new[b:e], k, v, D ** -0.5, len(k) - (e - b))
        check_o(out2[b:e], o, a, v, f"new tokens of {n}")


@pytest.mark.parametrize("T,H,HKV,D,R,inter,dtype,cdt", [
    (1, 4, 2, 128, 128, False, BF, torch.float32), (70, 6, 3, 64, 32, False, FP, torch.float32),
    (33, 8, 1, 128, 64, True, BF, BF), (200, 3, 3, 64, 64, True, FP, FP),
    (17, 2, 2, 128, 16, True, BF, torch.float32), (9, 1, 1, 64, 16, False, BF, torch.float32),
])
@pytest.mark.parametrize("idx", [torch.int32, torch.int64])
def test_append_paged_kv(dev, T, H, HKV, D, R, inter, dtype, cdt, idx):
    """Rotation within a rounding (two fp32 products and their sum, then one rounding to the
    type); stored values and everything not written bit for bit; padded slots store nothing."""
    gen = torch.Generator().manual_seed(T)
    page = 7
    qkv = randn(gen, T, (H + 2 * HKV) * D, dtype=dtype)
    q = qkv[:, :H * D].view(T, H, D)
    k = qkv[:, H * D:(H + HKV) * D].view(T, HKV, D)
    v = qkv[:, (H + HKV) * D:].view(T, HKV, D)
    pages = T // page + 3
    caches = randn(gen, 2, pages, page, HKV, D, dtype=dtype)
    slots = torch.randperm(pages * page, generator=gen)[:T]
    slots[::5] = -1
    if T > 8:
        slots[8] = pages * page
    pos = torch.randint(0, 50, (T,), generator=gen)
    ang = torch.rand(50, R // 2, generator=gen) * 6
    cs = torch.cat([ang.cos(), ang.sin()], 1).to(cdt)
    d = caches.to(dev)
    g = qkv.to(dev)
    out = hmx.append_paged_kv(g[:, H * D:(H + HKV) * D].view(T, HKV, D), g[:, (H + HKV) * D:].view(T, HKV, D),
                              d[0], d[1], slots.to(idx).to(dev), q=g[:, :H * D].view(T, H, D),
                              positions=pos.to(idx).to(dev), cos_sin=cs.to(dev), interleaved=inter)
    e = torch.finfo(dtype).eps / 2
    kc, vc = caches.clone(), caches[1].clone()
    kept = [t for t in range(T) if 0 <= slots[t] < pages * page]
    for x, got in ((q, out.cpu()), (k, None)):
        want = ref.rotate(x, cs, pos, inter)
        mag = x.double().abs() + x.double().abs().amax(-1, keepdim=True)
        if got is None:
            flat = d[0].cpu().view(-1, HKV, D)
            got, want, mag = (flat[slots[kept]], want[kept], mag[kept])
        err = (got.double() - want).abs()
        assert (err <= e * want.abs() + 2.0 ** -22 * mag).all()
        assert torch.equal(got[..., R:], (x if got.shape[0] == T and x is q else x[kept])[..., R:])
    written = torch.zeros(pages * page, dtype=torch.bool)
    written[slots[kept]] = True
    assert torch.equal(d[0].cpu().view(-1, HKV, D)[~written], kc[0].reshape(-1, HKV, D)[~written])
    vc.view(-1, HKV, D)[slots[kept]] = v[kept]
    assert torch.equal(d[1].cpu(), vc)


def test_append_without_rotation_and_in_place(dev):
    gen = torch.Generator().manual_seed(0)
    T, H, HKV, D = 5, 4, 2, 64
    q, k, v = (randn(gen, T, h, D).to(dev) for h in (H, HKV, HKV))
    both = torch.zeros(3, 2, 4, HKV, D, dtype=BF, device=dev)         # pages hold k and v side by side
    slots = torch.tensor([11, 0, 5, 6, 2], device=dev)
    assert hmx.append_paged_kv(k, v, both[:, 0], both[:, 1], slots) is None
    for t, s in enumerate(slots.tolist()):
        assert torch.equal(both[s // 4, 0, s % 4], k[t]) and torch.equal(both[s // 4, 1, s % 4], v[t])
    assert hmx.append_paged_kv(k, v, both[:, 0], both[:, 1], slots, q=q) is q
    cs = torch.randn(9, 64, generator=gen).to(dev)
    pos = torch.tensor([0, 8, 3, 3, 1], device=dev)
    kw = dict(positions=pos, cos_sin=cs)
    want = hmx.append_paged_kv(k, v, both[:, 0], both[:, 1], slots, q=q, **kw)
    got = hmx.append_paged_kv(k, v, both[:, 0], both[:, 1], slots, q=q, q_out=q, **kw)
    assert got is q and torch.equal(got, want)
    far = hmx.append_paged_kv(k, v, both[:, 0], both[:, 1], slots, q=q,
                              positions=torch.tensor([0, 9, -1, 3, 1], device=dev), cos_sin=cs)
    assert torch.isnan(far[1:3]).all() and torch.isfinite(far[[0, 3, 4]]).all()


def test_no_pages_no_keys(dev):
    """An empty cache, and a table without columns, hold no keys: rows of 0."""
    q = torch.ones(2, 4, 64, dtype=BF, device=dev)
    lens = torch.tensor([5, 0], dtype=torch.int32, device=dev)
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device=dev)
    for pages, width in ((0, 3), (4, 0)):
        kc = torch.ones(pages, 16, 2, 64, dtype=BF, device=dev)
        table = torch.zeros(2, width, dtype=torch.int32, device=dev)
        assert (hmx.paged_attention_decode(q, kc, kc, table, lens) == 0).all()
        assert (hmx.paged_causal_attention(q, kc, kc, table, lens, cu) == 0).all()
    none = torch.tensor([1], dtype=torch.int32, device=dev)       # no sequence at all
    assert (hmx.paged_causal_attention(q, kc, kc, table[:0], lens[:0], none) == 0).all()
    assert hmx.paged_attention_decode(q[:0], kc, kc, table[:0], lens[:0]).shape == (0, 4, 64)
    assert (hmx.causal_attention(q[None], q[None], q[None], cu_seqlens=none) == 0).all()
    assert hmx.causal_attention(q[None, :0], q[None, :0], q[None, :0]).shape == (1, 0, 4, 64)


@pytest.mark.parametrize("D", [64, 128])
def test_long_caches_past_32_bit_offsets(dev, D):
    """Pages more than 4 GiB into the cache, in both paged forms and the append."""
    H, HKV, page = 4, 2, 256
    pages = (5 << 30) // (page * HKV * D * 2)
    kc = torch.zeros(pages, page, HKV, D, dtype=BF, device=dev)
    vc = torch.zeros(pages, page, HKV, D, dtype=BF, device=dev)
    gen = torch.Generator().manual_seed(D)
    L = 700
    table = torch.tensor([[pages - 1, 3, pages - 2]], dtype=torch.int32)
    k, v = randn(gen, L, HKV, D), randn(gen, L, HKV, D)
    j = torch.arange(L)
    slots = table[0].long()[j // page] * page + j % page
    hmx.append_paged_kv(k.to(dev), v.to(dev), kc, vc, slots.to(dev))
    assert torch.equal(kc[pages - 1].cpu(), k[:page]) and torch.equal(vc[pages - 2, :L - 512].cpu(), v[512:])
    q = randn(gen, 3, H, D)
    dv = (kc, vc, table.to(dev), torch.tensor([L], dtype=torch.int32, device=dev))
    o, a = ref.rows(q, k, v, D ** -0.5, L - 3)
    check_o(hmx.paged_causal_attention(q.to(dev), *dv, torch.tensor([0, 3])), o, a, v, "new tokens")
    check_o(hmx.paged_attention_decode(q[2:].to(dev), *dv), o[2:], a[2:], v, "one token")


def test_many_packed_sequences(dev):
    """More sequences than a wave has lanes, and just as many, empty ones among them."""
    for N in (61, 62, 63, 64, 130):
        cu = [0]
        for i in range(N):
            cu.append(cu[-1] + (i * 29) % 37 * (i % 4 > 0))
        T, H, HKV, D = cu[-1] + 3, 4, 2, 64
        q, k, v = _case(N, T, H, HKV, D, BF)
        out = hmx.causal_attention(q.to(dev), k.to(dev), v.to(dev), cu_seqlens=torch.tensor(cu, device=dev))
        o, a = ref.causal(q[0], k[0], v[0], D ** -0.5, bounds_of(cu))
        check_o(out[0], o, a, v[0], f"{N} sequences")


def test_append_to_an_empty_cache(dev):
    """A cache of no pages stores nothing; q is rotated all the same."""
    gen = torch.Generator().manual_seed(21)
    k, q = randn(gen, 3, 2, 64).to(dev), randn(gen, 3, 4, 64).to(dev)
    cs = torch.cat([torch.zeros(4, 8), torch.ones(4, 8)], 1).to(dev)      # a quarter turn
    kc = torch.empty(0, 16, 2, 64, dtype=BF, device=dev)
    idx = torch.zeros(3, dtype=torch.int32, device=dev)
    got = hmx.append_paged_kv(k, k, kc, kc, idx, q=q, positions=idx, cos_sin=cs)
    assert torch.equal(got, torch.cat([-q[..., 8:16], q[..., :8], q[..., 16:]], -1))


@pytest.mark.parametrize("news,lens,H,HKV,D", [
    ([3, 1, 2, 40], [9000, 3, 700, 4096], 4, 1, 128), ([1, 1], [20000, 1], 14, 2, 64),
    ([2, 0, 5] * 22, [1500, 0, 40] * 22, 2, 1, 64), ([8] * 3, [8192, 8, 8191], 128, 128, 64),
])
def test_paged_causal_attention_few_rows_long_contexts(dev, news, lens, H, HKV, D):
    """Keys split over workgroups, as many to a sequence as its length asks for."""
    gen = torch.Generator().manual_seed(sum(lens))
    kc, vc, table, ks, vs = paged(gen, lens, 16, HKV, D, BF)
    cu = [1]
    for n in news:
        cu.append(cu[-1] + n)
    q = randn(gen, cu[-1] + 1, H, D)
    args = [x.to(dev) for x in (kc, vc, table)]
    args += [torch.tensor(x, dtype=torch.int32, device=dev) for x in (lens, cu)]
    out = hmx.paged_causal_attention(q.to(dev), *args)
    for n, (b, e) in enumerate(bounds_of(cu)):
        o, a = ref.rows(q[b:e], ks[n], vs[n], D ** -0.5, lens[n] - (e - b))
        check_o(out[b:e], o, a, vs[n], f"sequence {n} of {lens[n]}")
    assert (out[:1] == 0).all() and (out[cu[-1]:] == 0).all()
    # an infinite score reaches the row's output whichever share holds it
    q = q.abs()
    page, at = divmod(lens[0] // 3, 16)
    args[0][table[0, page], at] = float("inf")
    out = hmx.paged_causal_attention(q.to(dev), *args)
    assert out[cu[0]:cu[1]].isnan().all() and out[cu[1]:].isfinite().all()


@pytest.mark.parametrize("B,T,cu,H,HKV,D,dtype", [
    (1, 2048, None, 8, 2, 128, BF), (2, 1500, None, 4, 4, 64, FP), (1, 3001, None, 7, 1, 64, BF),
    (1, 3000, [4, 1800, 1800, 1803, 2900], 4, 1, 128, FP),
    (1, 1600, [0] + [1000 + 9 * i for i in range(66)], 2, 2, 64, BF),
])
def test_causal_attention_few_rows_many_keys(dev, B, T, cu, H, HKV, D, dtype):
    """Rows too few for the chip: their keys are split over workgroups and joined."""
    gen = torch.Generator().manual_seed(T + H)
    q, k, v = (randn(gen, B, T, n, D, dtype=dtype) for n in (H, HKV, HKV))
    # values that no row before them may see
    k[:, -1], v[:, -1] = float("nan"), float("inf")
    out = hmx.causal_attention(q.to(dev), k.to(dev), v.to(dev),
                               cu_seqlens=None if cu is None else torch.tensor(cu, device=dev))
    for b in range(B):
        bounds = [(0, T)] if cu is None else bounds_of(cu)
        n = bounds[-1][1] - (bounds[-1][1] == T)          # the last row sees the NaN
        o, a = ref.causal(q[b], k[b], v[b], D ** -0.5, [(x, min(y, n)) for x, y in bounds])
        check_o(out[b, :n], o[:n], a[:n], v[b, :n], f"{B} x {T}")
        assert n == T or cu is not None and cu[-1] < T or out[b, -1].isnan().all()
