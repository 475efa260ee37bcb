"""Calls at the edges of what the attention ops accept, against the float64 definitions.

Tolerances are elementwise and derived in attn_util.o_tolerance."""
from types import SimpleNamespace

import pytest
import torch

import hmx
from hmx import _lib
import hmx.serving as serving
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


def test_outputs_with_rows_far_apart(dev):
    """Token strides of 2^25 elements and more, in every op that takes an output."""
    gen = torch.Generator().manual_seed(6)
    H, HKV, D, far = 4, 2, 64, 1 << 25
    kc, vc = (randn(gen, 40, 16, HKV, D).to(dev) for _ in range(2))
    table = torch.randperm(40, generator=gen).to(torch.int32).view(4, 10).to(dev)
    lens = torch.tensor([100, 7, 33, 160], dtype=torch.int32, device=dev)
    cu = torch.tensor([0, 1, 2, 3, 4], dtype=torch.int32, device=dev)
    q, k, v = (randn(gen, 4, n, D).to(dev) for n in (H, HKV, HKV))
    cs = torch.randn(9, 32, generator=gen).to(dev)
    pos = torch.tensor([0, 8, 3, 1], device=dev)
    slots = torch.full((4,), -1, device=dev)
    room = torch.full((3 * far + H * D,), 7.0, dtype=BF, device=dev)
    out = room.as_strided((4, H, D), (far, D, 1))
    for run in (lambda **kw: hmx.paged_attention_decode(q, kc, vc, table, lens, **kw),
                lambda **kw: hmx.paged_causal_attention(q, kc, vc, table, lens, cu, **kw),
                lambda **kw: hmx.causal_attention(q[None], k[None], v[None], **{n: x[None] for n, x in kw.items()}),
                lambda **kw: hmx.append_paged_kv(k, v, kc, vc, slots, q=q, positions=pos, cos_sin=cs,
                                                 **{"q_" + n: x for n, x in kw.items()})):
        room.fill_(7.0)
        want = run()
        got = run(out=out)
        assert got.data_ptr() == room.data_ptr() and torch.equal(got.view(4, H, D), want.view(4, H, D))
        assert (room[H * D:H * D + 4 * H * D] == 7).all() and int((room != 7).sum()) <= 4 * H * D


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_paged_host_offsets_of_later_sequences(dev, dtype):
    """A slice of a batch's offsets, as the host holds them: the same as on the device."""
    gen = torch.Generator().manual_seed(8)
    kc, vc = (randn(gen, 40, 16, 2, 64).to(dev) for _ in range(2))
    table = torch.randperm(40, generator=gen).to(torch.int32).view(4, 10).to(dev)
    lens = torch.tensor([100, 7, 33, 160], dtype=torch.int32, device=dev)
    cu = torch.tensor([0, 1, 2, 9, 20], dtype=dtype)
    q = randn(gen, 23, 4, 64).to(dev)
    for n in (0, 2, 4):
        args = (q, kc, vc, table[n:], lens[n:])
        assert torch.equal(hmx.paged_causal_attention(*args, cu[n:]), hmx.paged_causal_attention(*args, cu[n:].to(dev)))


@pytest.mark.parametrize("rope", [True, False])
def test_forward_core_of_no_tokens(dev, rope):
    lay = SimpleNamespace(num_heads=4, num_kv_heads=2, head_dim=64, tp_size=1, rotary_emb=SimpleNamespace(
        cos_sin_cache=torch.zeros(9, 64, device=dev), is_neox_style=True) if rope else None)
    none = torch.zeros(0, dtype=torch.int32, device=dev)
    md = SimpleNamespace(num_actual_tokens=0, num_decodes=0, num_decode_tokens=0, num_prefills=0, query_start_loc=none,
                         seq_lens=none, block_table=none.view(0, 3), slot_mapping=none)
    kc = torch.full((3, 16, 2, 64), 2.0, dtype=BF, device=dev)
    for tokens in (0, 3):
        out = torch.full((tokens, 4, 64), 5.0, dtype=BF, device=dev)
        serving.attention_forward_core(lay, torch.zeros(tokens, 8 * 64, dtype=BF, device=dev), none, out, md, kc, kc.clone())
        assert (out == 5).all() and (kc == 2).all()


def test_forward_core_with_fewer_kv_heads_than_ranks(dev):
    """Two key/value heads over four ranks: the rank's one head serves its four q heads."""
    gen = torch.Generator().manual_seed(9)
    H, D, n, page = 4, 64, 30, 16
    qkv = randn(gen, n, (H + 2) * D)
    kc, vc = (torch.zeros(4, page, 1, D, dtype=BF, device=dev) for _ in range(2))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    md = SimpleNamespace(num_actual_tokens=n, num_decodes=0, num_decode_tokens=0, num_prefills=1,
                         query_start_loc=i32([0, n]), seq_lens=i32([n]), block_table=i32([[2, 0]]),
                         slot_mapping=torch.cat([torch.arange(32, 48), torch.arange(14)]).to(dev))
    lay = SimpleNamespace(num_heads=16, num_kv_heads=2, head_dim=D, tp_size=4)
    out = torch.zeros(n, H, D, dtype=BF, device=dev)
    serving.attention_forward_core(lay, qkv.to(dev), None, out, md, kc, vc)
    q, k, v = (x.reshape(n, -1, D) for x in qkv.split([H * D, D, D], -1))
    o, a = ref.rows(q, k, v, D ** -0.5, 0)
    check_o(out, o, a, v, "one kv head")


def test_a_backward_through_the_cache_ops_raises(dev):
    """A backward that would lose gradients in silence raises instead; the values are those
    of a call that needs none."""
    gen = torch.Generator().manual_seed(10)
    kc, vc = (randn(gen, 20, 16, 2, 64).to(dev) for _ in range(2))
    table = torch.arange(20, dtype=torch.int32, device=dev).view(2, 10)
    lens = torch.tensor([100, 33], dtype=torch.int32, device=dev)
    q, k, v = (randn(gen, 2, n, 64).to(dev) for n in (4, 2, 2))
    kw = dict(positions=torch.tensor([3, 1], device=dev), cos_sin=torch.randn(9, 32, generator=gen).to(dev))
    slots, cu = torch.full((2,), -1, device=dev), torch.tensor([0, 1, 2])
    for run in (lambda q, k: hmx.paged_attention_decode(q, kc, vc, table, lens),
                lambda q, k: hmx.paged_causal_attention(q, kc, vc, table, lens, cu),
                lambda q, k: hmx.append_paged_kv(k, v, kc, vc, slots, q=q, **kw)):
        want = run(q, k)
        assert not want.requires_grad
        got = run(q.clone().requires_grad_(), k.clone().requires_grad_())
        assert torch.equal(got, want)
        with pytest.raises(NotImplementedError, match="no backward"):
            got.float().sum().backward()
        with torch.no_grad():
            assert not run(q.clone().requires_grad_(), k).requires_grad
    x = q.clone().requires_grad_()               # without a rotation q passes through, gradient and all
    assert hmx.append_paged_kv(k, v, kc, vc, slots, q=x) is x
    out = torch.empty_like(q)
    assert hmx.paged_attention_decode(x, kc, vc, table, lens, out=out) is out and not out.requires_grad


def _like(out, o, a, what):
    """out finite where the definition o is, and within the rounding of its terms there; NaN
    and the infinities where o has them."""
    out = out.double().cpu()
    fine = torch.isfinite(o)
    assert torch.equal(torch.isfinite(out), fine), what
    assert torch.equal(out.nan_to_num(0, 1, -1)[~fine], o.nan_to_num(0, 1, -1)[~fine]), what
    # o_tolerance's terms at bf16's half step, |o| <= a, and 2^-25 of fewer than 2^9 values' sum in fp16
    assert ((out - o).abs()[fine] <= (2.0 ** -7 + 2.0 ** -11) * a[fine] + 2.0 ** -16).all(), what


@pytest.mark.parametrize("T,cu,H,HKV,D,dtype", [
    (600, None, 4, 2, 128, BF), (600, None, 3, 3, 64, BF), (500, [0, 90, 90, 333, 480], 8, 1, 128, BF),
    (2048, None, 2, 1, 128, BF), (2100, [3, 1000, 2100], 4, 4, 64, BF), (400, None, 5, 1, 128, FP),
])
def test_values_that_are_not_finite_at_every_distance(dev, T, cu, H, HKV, D, dtype):
    """Infinities of both signs and NaN among the values, in different columns and in one: rows
    that attend them have exactly them, the others none; keys split and whole, packed and not."""
    gen = torch.Generator().manual_seed(T + D)
    q, k, v = (randn(gen, 1, T, n, D, dtype=dtype) for n in (H, HKV, HKV))
    for at, col, bad in ((7, 1, "nan"), (40, 2, "inf"), (61, 3, "-inf"), (130, 2, "-inf"), (131, 5, "inf"),
                         (200, 6, "nan"), (T // 2, 9, "inf"), (T - 70, 11, "nan"), (T - 2, 12, "-inf"), (T - 1, 13, "inf")):
        v[0, at, at % HKV, col] = float(bad)
    out = hmx.causal_attention(q.to(dev), k.to(dev), v.to(dev),
                               cu_seqlens=None if cu is None else torch.tensor(cu, device=dev, dtype=torch.int32))
    o, a = ref.causal(q[0], k[0], v[0], D ** -0.5, [(0, T)] if cu is None else bounds_of(cu))
    _like(out[0], o, a, f"T={T}")


@pytest.mark.parametrize("news,lens,page", [([70, 1, 130], [300, 90, 130], 16), ([3, 2], [5000, 900], 16), ([40], [777], 7)])
def test_cached_values_that_are_not_finite(dev, news, lens, page):
    """The same over pages, where some lie outside the cache and all that is no key is NaN."""
    gen = torch.Generator().manual_seed(sum(lens))
    H, HKV, D = 4, 2, 64
    kc, vc, table, ks, vs = paged(gen, lens, page, HKV, D, BF)
    keep = []
    for n, L in enumerate(lens):
        for back, col, bad in ((0, 1, "inf"), (1, 2, "nan"), (20, 3, "-inf"), (64, 4, "inf"), (80, 4, "-inf")):
            j = L - 1 - back
            if j >= 0:
                vc[table[n, j // page].long(), j % page, 1, col] = vs[n][j, 1, col] = float(bad)
        key = torch.arange(L)
        hole = key // page == (L - max(news[n], 30) - 1) // page if L > 200 else key < 0
        table[n, key[hole] // page] = -1
        keep.append(~hole)
    cu = [0]
    for m in news:
        cu.append(cu[-1] + m)
    q = randn(gen, cu[-1], H, D)
    out = hmx.paged_causal_attention(q.to(dev), kc.to(dev), vc.to(dev), table.to(dev),
                                     torch.tensor(lens, dtype=torch.int32, device=dev), torch.tensor(cu))
    for n, (b, e) in enumerate(bounds_of(cu)):
        # row i sees the keys up to its own that there are
        for i in range(e - b):
            seen = keep[n] & (torch.arange(lens[n]) <= lens[n] - (e - b) + i)
            K, V = ks[n][seen], vs[n][seen]
            o, a = ref.rows(q[b + i:b + i + 1], K, V, D ** -0.5, len(K) - 1)
            _like(out[b + i:b + i + 1], o, a, f"sequence {n} row {i}")


def test_values_that_are_not_finite_do_not_stall_a_call(dev):
    """NaN in all values (a step that has diverged) costs a few times the call, not hundreds."""
    q, k, v = (torch.randn(1, 2048, n, 128, device=dev).bfloat16() for n in (32, 8, 8))

    def fastest(v):
        best = float("inf")
        for _ in range(6):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            hmx.causal_attention(q, k, v)
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    fine = fastest(v)
    assert fastest(torch.full_like(v, float("nan"))) < 30 * fine


def test_a_batch_of_single_tokens_far_apart(dev):
    B, H, HKV, D, far = 3, 4, 2, 64, 1 << 25
    gen = torch.Generator().manual_seed(12)
    q, k, v = (randn(gen, B, 1, n, D).to(dev) for n in (H, HKV, HKV))
    room = torch.zeros(2 * far + H * D, dtype=BF, device=dev)
    for x in (k, v):
        y = room.as_strided(x.shape, (far, 8, D, 1))
        y.copy_(x)
        got = hmx.causal_attention(q, y if x is k else k, y if x is v else v)
        assert torch.equal(got, hmx.causal_attention(q, k, v))


def test_c_calls_with_strides_that_go_back(dev):
    """Heads in reverse order by a negative stride, in q and the output's gradient, through the
    C entry points: what the reversed tensors give."""
    gen = torch.Generator().manual_seed(13)
    T, H, HKV, D = 150, 4, 2, 64
    q, k, v, do = (randn(gen, 1, T, n, D).to(dev) for n in (H, HKV, HKV, H))
    back = lambda x: (x.data_ptr() + (H - 1) * D * 2, H * D, -D)
    fore = lambda x: (x.data_ptr(), x.shape[2] * D, D)
    o, dq, dk, dv = (torch.empty_like(x) for x in (q, q, k, v))
    lse, delta = (torch.empty(T, H, device=dev) for _ in range(2))
    s = _lib.stream_of(q)
    _lib.call("hmx_causal_attention", *back(q), *fore(k), *fore(v), _lib.HMX_BF16, *fore(o), lse.data_ptr(), None,
              1, T, H, HKV, D, D ** -0.5, 1, None, 0, s)
    _lib.call("hmx_causal_attention_bwd", *back(q), *fore(k), *fore(v), _lib.HMX_BF16, *fore(o), *back(do), lse.data_ptr(),
              None, 1, T, H, HKV, D, D ** -0.5, *fore(dq), *fore(dk), *fore(dv), delta.data_ptr(), s)
    ins = [x.clone().requires_grad_() for x in (q.flip(2), k, v)]
    want = hmx.causal_attention(*ins)
    assert torch.equal(o, want)
    for x, y in zip((dq, dk, dv), torch.autograd.grad(want, ins, do.flip(2).contiguous())):
        assert torch.equal(x, y)


@pytest.mark.parametrize("T,cu", [(200, [5, 60, 60, 190]), (2500, [100, 2000, 2400])])
def test_registered_row_statistics(dev, T, cu):
    """The registered op's second output: the logarithm of every row's sum, minus infinity for
    rows of no sequence, whose sum is empty.  fp32 scores leave 2^-12 of the sum, the hardware's
    logarithm less."""
    import hmx.library  # noqa: F401
    gen = torch.Generator().manual_seed(T)
    H, HKV, D = 4, 2, 64
    q, k, v = (randn(gen, 1, T, n, D) for n in (H, HKV, HKV))
    for _ in range(3):                            # memory that other results have left
        torch.full((T, H), 3.0, device=dev)
        o, lse = torch.ops.hmx.causal_attention(q.to(dev), k.to(dev), v.to(dev), None,
                                                torch.tensor(cu, dtype=torch.int32, device=dev))
    want = torch.full((T, H), -torch.inf, dtype=torch.float64)
    for b, e in bounds_of(cu):
        kk = k[0, b:e].double().repeat_interleave(H // HKV, 1)
        s = torch.einsum("ihd,jhd->ijh", q[0, b:e].double(), kk) * D ** -0.5
        s.masked_fill_(torch.ones(e - b, e - b, dtype=torch.bool).triu(1)[..., None], -torch.inf)
        want[b:e] = torch.logsumexp(s, 1) / torch.log(torch.tensor(2.0, dtype=torch.float64))
    there = torch.isfinite(want)
    lse = lse.double().cpu()
    assert torch.equal(torch.isfinite(lse), there) and (lse[~there] == -torch.inf).all()
    assert ((lse - want).abs()[there] <= 2.0 ** -11 + 2.0 ** -20 * want[there].abs()).all()


@pytest.mark.parametrize("H,HKV,D,page", [(8, 2, 128, 16), (14, 2, 64, 48)])
def test_tables_wider_than_the_sequences(dev, H, HKV, D, page):
    """An engine's table, as wide as its longest sequence may grow: short, empty and long
    sequences beside one another, entries behind their pages outside the cache."""
    gen = torch.Generator().manual_seed(page)
    lens = [5, 0, 700, 64, 3333, 1]
    kc, vc, table, ks, vs = paged(gen, lens, page, HKV, D, BF, width=20000 // page)
    n32 = torch.tensor(lens, dtype=torch.int32, device=dev)
    args = [x.to(dev) for x in (kc, vc, table)] + [n32]
    q = randn(gen, 2 * len(lens), H, D)
    out = hmx.paged_attention_decode(q[:len(lens)].to(dev), *args)
    new = hmx.paged_causal_attention(q.to(dev), *args, torch.arange(0, 2 * len(lens) + 1, 2))
    for n, L in enumerate(lens):
        o, a = ref.rows(q[n:n + 1], ks[n], vs[n], D ** -0.5, L - 1)
        check_o(out[n:n + 1], o, a, vs[n], f"decode {L}")
        o, a = ref.rows(q[2 * n:2 * n + 2], ks[n], vs[n], D ** -0.5, L - 2)
        check_o(new[2 * n:2 * n + 2], o, a, vs[n], f"new tokens of {L}")


@pytest.mark.parametrize("width", [3, 200])
def test_lengths_outside_the_table(dev, width):
    """Lengths past the table's pages count as all of them, negative ones as none."""
    gen = torch.Generator().manual_seed(width)
    kc, vc = (randn(gen, 2 * width, 16, 2, 64).to(dev) for _ in range(2))
    table = torch.randperm(2 * width, generator=gen).to(torch.int32).view(2, width).to(dev)
    q = randn(gen, 5, 4, 64).to(dev)
    cu = torch.tensor([0, 2, 5], dtype=torch.int32, device=dev)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)
    for far, near in ((i32(10 ** 9, 2 ** 31 - 1), i32(16 * width, 16 * width)), (i32(16 * width + 1, -5), i32(16 * width, 0)),
                      (i32(-(2 ** 31), 30), i32(0, 30))):
        args = (kc, vc, table)
        want = hmx.paged_attention_decode(q[:2], *args, near)
        assert torch.equal(hmx.paged_attention_decode(q[:2], *args, far), want)
        a, b = (hmx.paged_causal_attention(q, *args, n, cu).double() for n in (far, near))
        # splits of other lengths: two roundings of terms whose magnitudes are below max |v| < 6
        assert ((a - b).abs() <= 4 * 2.0 ** -8 * 6).all() and torch.equal(a == 0, b == 0)
        assert (want[near == 0] == 0).all()
