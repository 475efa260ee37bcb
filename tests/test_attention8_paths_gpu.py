"""Caches of 8 bits and shared prefixes as they are used: a layer's steps from the append to the
attention, captured steps replayed with other lengths, two streams, layouts of caches, inputs
and outputs, caches past 32-bit offsets, lengths past the tables, unequal numbers of new
tokens, and the registered ops."""
from types import SimpleNamespace

import pytest
import torch

import hmx
import hmx.library as lib
from attn_util import check_o, half_step, paged, paged8, randn, ref

pytestmark = pytest.mark.gpu
BF, F16, F8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def _i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _case(dev, lens, G=4, HKV=2, D=64, page=16, seed=0, width=None, dtype=BF):
    gen = torch.Generator().manual_seed(seed)
    kc, vc, ks, vs, table, kl, vl = paged8(gen, lens, page, HKV, D, width=width)
    q = randn(gen, len(lens), G * HKV, D, dtype=dtype, scale=0.5)
    return SimpleNamespace(kc=kc.to(dev), vc=vc.to(dev), sc=dict(k_scales=ks.to(dev), v_scales=vs.to(dev)), table=table.to(dev),
                           kl=kl, vl=vl, q=q, qd=q.to(dev), lens=_i32(lens, dev), gen=gen)


@pytest.mark.parametrize("page,prefix_pages", [(16, 3), (48, 1)])
def test_a_layers_steps(dev, page, prefix_pages):
    """attention_forward_core over a cache of 8 bits: prompts that begin alike, then decodes, then
    decodes that share the prompts' first pages; every output against float64 over what the
    cache then stands for, the cache against its definition."""
    import hmx.serving as serving
    gen = torch.Generator().manual_seed(page)
    N, H, HKV, D = 3, 4, 2, 64
    inv, factor = hmx.rotary_frequencies(D, 1e4, dict(rope_type="yarn", factor=2.0, original_max_position_embeddings=64), device=dev)
    rope = SimpleNamespace(cos_sin_cache=hmx.rotary_table(inv, 400, factor), is_neox_style=True)
    layer = SimpleNamespace(num_heads=H, num_kv_heads=HKV, head_dim=D, tp_size=1, rotary_emb=rope)
    P = prefix_pages * page
    prompts, pages = [P + 9, P + 1, P + 30], 6 + prefix_pages
    kc, vc = (torch.zeros(N * pages, page, HKV, D, dtype=torch.uint8, device=dev).view(F8) for _ in range(2))
    ks, vs = (torch.ones(N * pages, HKV, page, dtype=torch.uint8, device=dev) for _ in range(2))
    table = torch.randperm(N * pages, generator=gen).view(N, pages)
    table[1:, :prefix_pages] = table[0, :prefix_pages]                  # the first pages are one prompt's
    first = randn(gen, P, (H + 2 * HKV) * D)
    lens, keys, values = [0] * N, [[] for _ in range(N)], [[] for _ in range(N)]
    whole = lambda cache, scales: cache.double().cpu() * torch.exp2(scales.cpu().double() - 127).transpose(1, 2)[..., None]

    def step(news, decodes, shared):
        nonlocal lens
        rows = [randn(gen, n, (H + 2 * HKV) * D) for n in news]
        if lens[0] == 0:
            rows = [torch.cat([first, r[P:]]) for r in rows]
        pos = [torch.arange(a, a + n) for a, n in zip(lens, news)]
        lens = [a + n for a, n in zip(lens, news)]
        slots = torch.cat([table[i][p // page] * page + p % page for i, p in enumerate(pos)])
        qkv, at = torch.cat(rows), torch.cat(pos)
        cu = [0]
        for n in news:
            cu.append(cu[-1] + n)
        own, own_lens = (table[:, prefix_pages:], [n - P for n in lens]) if shared else (table, lens)
        md = SimpleNamespace(num_actual_tokens=cu[-1], num_decodes=decodes, num_decode_tokens=decodes, num_prefills=N - decodes,
                             query_start_loc=_i32(cu, dev), seq_lens=_i32(own_lens, dev), block_table=own.int().to(dev),
                             slot_mapping=slots.to(dev))
        if shared:
            md.prefix_table, md.prefix_lens = table[:1, :prefix_pages].int().to(dev), _i32([P], dev)
        out = torch.full((cu[-1] + 2, H, D), 5.0, dtype=BF, device=dev)
        serving.attention_forward_core(layer, qkv.to(dev), at.to(dev), out, md, kc, vc, ks, vs)
        assert (out[cu[-1]:] == 5).all()
        K, V = whole(kc, ks), whole(vc, vs)
        q, k, v = (x.unflatten(-1, (-1, D)) for x in qkv.split([H * D, HKV * D, HKV * D], -1))
        ang = at.double()[:, None] * inv.cpu()
        qr = ref.rotate_by(q, ang, factor, False)
        kr = ref.rotate_by(k, ang, factor, False)
        for x, c in ((kr, K), (v.double(), V)):
            got = c[slots // page, slots % page]
            # half a step of e4m3, or of its smallest value's at the row's scale, beside fp32's rotation
            top = x.abs().amax(-1, keepdim=True)
            assert ((got - x).abs() <= (2.0 ** -4 + 2.0 ** -18) * x.abs() + 2.0 ** -17 * top).all()
        for i in range(N):
            for t in range(cu[i], cu[i + 1]):
                n = lens[i] - (cu[i + 1] - 1 - t)
                kk, vv = ref.gather(K, table[i], n), ref.gather(V, table[i], n)
                qq = qr[t:t + 1].to(BF)                                  # as the kernel stores it, up to its rounding
                want, a = ref.rows(qq, kk, vv, D ** -0.5, n - 1)
                # a rotated q may be rounded to the other side: half a step of q in the scores, at most
                # 2^-8 of sum |q k| / 8 < 16 each, a factor of the probabilities
                s = (qq.double().abs().unflatten(1, (HKV, -1)) * kk.abs().amax(0)[None, :, None]).sum(-1).amax() * D ** -0.5
                tol = 2 * half_step(BF) * s * a + 2 * half_step(BF) * (a + want.abs()) + 1e-6
                assert ((out[t].cpu().double() - want[0]).abs() <= tol[0]).all(), (i, t)

    step(prompts, 0, False)
    step([1, 1, 1], 3, False)
    step([1, 1, 1], 3, True)
    step([1, 1, 7], 2, False)


def _replays(dev, run, change, n=5):
    """run() captured once and replayed after every change(i), against run() itself."""
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run()
    for i in range(n):
        change(i)
        torch.cuda.synchronize()
        g.replay()
        got = out.clone()
        want = run()
        torch.cuda.synchronize()
        assert torch.equal(got, want), f"replay {i}"


@pytest.mark.parametrize("width", [40, 400])
def test_captured_decodes(dev, width):
    c = _case(dev, [600, 33, 0, 128], width=width)
    lens = [[600, 33, 0, 128], [1, 1, 1, 1], [0, 0, 0, 0], [599, 20, 0, 77], [64, 33, 0, 65]]
    _replays(dev, lambda: hmx.paged_attention_decode(c.qd, c.kc, c.vc, c.table, c.lens, **c.sc),
             lambda i: c.lens.copy_(_i32(lens[i], dev)))


@pytest.mark.parametrize("tokens", [8, 60])
def test_captured_new_tokens(dev, tokens):
    c = _case(dev, [600, 133, 40, 128], width=100)
    q = randn(c.gen, tokens, 8, 64).to(dev)
    cu = _i32([0, 2, 4, 6, 8], dev)
    news = [[0, 2, 4, 6, 8], [1, 1, 1, 7, 8], [0, 8, 8, 8, 8], [0, 0, 0, 0, 0], [3, 4, 5, 6, 7]]
    _replays(dev, lambda: hmx.paged_causal_attention(q, c.kc, c.vc, c.table, c.lens, cu, **c.sc),
             lambda i: cu.copy_(_i32([x * tokens // 8 for x in news[i]], dev)))


@pytest.mark.parametrize("N,eight", [(5, True), (5, False), (70, True), (70, False)])
def test_captured_shared_prefixes(dev, N, eight):
    pre = [700, 90]
    lens = [1 + 11 * i % 70 for i in range(N)]
    gen = torch.Generator().manual_seed(N)
    if eight:
        kc, vc, ks, vs, table, _, _ = paged8(gen, pre + lens, 16, 2, 64, width=50)
        sc = dict(k_scales=ks.to(dev), v_scales=vs.to(dev))
    else:
        (kc, vc, table, _, _), sc = paged(gen, pre + lens, 16, 2, 64, BF, width=50), {}
    q, table = randn(gen, N, 8, 64).to(dev), table.to(dev)
    kc, vc, p, n, cu = kc.to(dev), vc.to(dev), _i32(pre, dev), _i32(lens, dev), _i32([0, N - 2, N], dev)
    cus = [[0, N - 2, N], [1, 1, N - 1], [0, 0, 0], [0, N, N], [2, 3, 4]]

    def change(i):
        cu.copy_(_i32(cus[i], dev))
        p.copy_(_i32([[700, 90], [1, 0], [5, 90], [333, 1], [640, 64]][i], dev))
        n.copy_(_i32([max(x - 9 * i, 0) for x in lens], dev))

    _replays(dev, lambda: hmx.shared_prefix_attention_decode(q, kc, vc, table[2:], n, table[:2], p, cu, **sc), change)


def test_captured_append(dev):
    gen = torch.Generator().manual_seed(0)
    k, v = (randn(gen, 9, 2, 64).to(dev) for _ in range(2))
    slots = torch.arange(9, device=dev)
    kc, vc = (torch.zeros(4, 16, 2, 64, dtype=torch.uint8, device=dev).view(F8) for _ in range(2))
    ks, vs = (torch.ones(4, 2, 16, dtype=torch.uint8, device=dev) for _ in range(2))

    def run():
        hmx.append_paged_kv(k, v, kc, vc, slots, k_scales=ks, v_scales=vs)
        return torch.cat([kc.view(torch.uint8).flatten(), vc.view(torch.uint8).flatten(), ks.flatten(), vs.flatten()])

    def change(i):
        k.copy_(randn(gen, 9, 2, 64, scale=2.0 ** i))
        slots.copy_(torch.randperm(64, generator=gen)[:9])

    _replays(dev, run, change)


def test_two_streams(dev):
    """The ops on two streams at once, each with a workspace of its own."""
    cases = [_case(dev, [900, 1700, 33, 64], seed=i, width=200) for i in range(2)]
    cu = _i32([0, 1, 2, 3, 4], dev)
    pt, pl = ([c.table[1:2] for c in cases], [c.lens[1:2] for c in cases])

    def run(i):
        c = cases[i]
        return (hmx.paged_attention_decode(c.qd, c.kc, c.vc, c.table, c.lens, **c.sc),
                hmx.paged_causal_attention(c.qd, c.kc, c.vc, c.table, c.lens, cu, **c.sc),
                hmx.shared_prefix_attention_decode(c.qd, c.kc, c.vc, c.table, c.lens, pt[i], pl[i], **c.sc))

    want = [run(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run(i))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(g, want[i]))


def _layouts(c):
    """The case's cache as contiguous tensors, with heads before places in one allocation with
    scales in rows of other lengths, and as slices of more heads."""
    yield c.kc, c.vc, c.sc
    n, page, HKV, D = c.kc.shape
    both = torch.zeros(n, 2, HKV, page, D, dtype=torch.uint8, device=c.kc.device)
    sc = torch.zeros(2, n, HKV, page + 3, dtype=torch.uint8, device=c.kc.device)
    for i, (x, s) in enumerate(((c.kc, "k_scales"), (c.vc, "v_scales"))):
        both[:, i] = x.view(torch.uint8).transpose(1, 2)
        sc[i, ..., :page] = c.sc[s]
    yield both.view(F8)[:, 0].transpose(1, 2), both.view(F8)[:, 1].transpose(1, 2), dict(k_scales=sc[0, ..., :page], v_scales=sc[1, ..., :page])
    wide = [torch.zeros(n, page, HKV + 1, D, dtype=torch.uint8, device=c.kc.device) for _ in range(2)]
    scw = [torch.zeros(n, HKV + 1, page, dtype=torch.uint8, device=c.kc.device) for _ in range(2)]
    for w, s, x, t in zip(wide, scw, (c.kc, c.vc), ("k_scales", "v_scales")):
        w[:, :, 1:] = x.view(torch.uint8)
        s[:, 1:] = c.sc[t]
    yield wide[0].view(F8)[:, :, 1:], wide[1].view(F8)[:, :, 1:], dict(k_scales=scw[0][:, 1:], v_scales=scw[1][:, 1:])


@pytest.mark.parametrize("page", [16, 24])
def test_layouts_of_caches_inputs_and_outputs(dev, page):
    lens = [300, 17, 96]
    c = _case(dev, lens, page=page, D=128)
    cu3, cu60 = _i32([0, 1, 2, 3], dev), _i32([0, 50, 55, 60], dev)
    q60 = randn(c.gen, 60, 8, 128).to(dev)
    q_heads_first = c.qd.transpose(0, 1).contiguous().transpose(0, 1)
    ops = [lambda kc, vc, sc, q, **kw: hmx.paged_attention_decode(q, kc, vc, c.table, c.lens, **sc, **kw),
           lambda kc, vc, sc, q, **kw: hmx.paged_causal_attention(q, kc, vc, c.table, c.lens, cu3, **sc, **kw),
           lambda kc, vc, sc, q, **kw: hmx.paged_causal_attention(q60, kc, vc, c.table, c.lens, cu60, **sc),
           lambda kc, vc, sc, q, **kw: hmx.shared_prefix_attention_decode(q, kc, vc, c.table, c.lens, c.table[:1], c.lens[:1], **sc, **kw)]
    for i, op in enumerate(ops):
        want = None
        for kc, vc, sc in _layouts(c):
            got = op(kc, vc, sc, c.qd)
            want = got if want is None else want
            assert torch.equal(got, want), i
        assert torch.equal(op(c.kc, c.vc, c.sc, q_heads_first), want)
        wide = torch.full((4, 9, 128), 3.0, dtype=BF, device=dev)
        out = wide[:3, 1:]
        if i != 2:
            assert op(c.kc, c.vc, c.sc, c.qd, out=out) is out and torch.equal(out, want)
            assert (wide[3] == 3).all() and (wide[:, 0] == 3).all()


def test_caches_past_32_bit_offsets(dev):
    """Pages behind 2^32 bytes of the cache, and slots there."""
    page, HKV, D = 64, 8, 128
    pages = (1 << 32) // (page * HKV * D) + 40
    kc, vc = (torch.empty(pages, page, HKV, D, dtype=torch.uint8, device=dev).view(F8) for _ in range(2))
    ks, vs = (torch.empty(pages, HKV, page, dtype=torch.uint8, device=dev) for _ in range(2))
    gen = torch.Generator().manual_seed(0)
    lens = [300, 65, 1]
    table = (pages - 1 - torch.arange(15).view(3, 5)).int()
    k, v = (randn(gen, sum(lens), HKV, D) for _ in range(2))
    at = torch.cat([torch.arange(n) for n in lens])
    seq = torch.repeat_interleave(torch.arange(3), torch.tensor(lens))
    slots = table[seq, at // page].long() * page + at % page
    hmx.append_paged_kv(k.to(dev), v.to(dev), kc, vc, slots.to(dev), k_scales=ks, v_scales=vs)
    sc = dict(k_scales=ks, v_scales=vs)
    q = randn(gen, 3, 16, D, scale=0.5)
    args = (kc, vc, table.to(dev), _i32(lens, dev))
    (kv, ke), (vv, ve) = (ref.quantise(x) for x in (k, v))
    K, V = torch.ldexp(kv, ke[..., None]), torch.ldexp(vv, ve[..., None])
    outs = [hmx.paged_attention_decode(q.to(dev), *args, **sc),
            hmx.paged_causal_attention(q.to(dev), *args, _i32([0, 1, 2, 3], dev), **sc),
            hmx.shared_prefix_attention_decode(q.to(dev), *args, args[2][:0], args[3][:0], _i32([0], dev), **sc)]
    long = hmx.paged_causal_attention(q.to(dev).repeat_interleave(20, 0), *args, _i32([0, 20, 40, 60], dev), **sc)
    many = hmx.shared_prefix_attention_decode(q[:1].to(dev).repeat(80, 1, 1), kc, vc, args[2][2:].repeat(80, 1), args[3][2:].repeat(80),
                                              args[2][:1], args[3][:1], **sc)
    b = [0, 300, 365, 366]
    for n in range(3):
        kk, vv = K[b[n]:b[n + 1]], V[b[n]:b[n + 1]]
        want, a = ref.rows(q[n:n + 1], kk, vv, D ** -0.5, lens[n] - 1)
        for o in outs:
            check_o(o[n:n + 1].cpu(), want, a, vv, f"sequence {n}")
        check_o(long[20 * n + 19:20 * n + 20].cpu(), want, a, vv, f"last of 20 tokens of {n}")
    want, a = ref.behind_prefix(q[0], K[:300], V[:300], K[365:], V[365:], D ** -0.5)
    for i in (0, 79):
        check_o(many[i:i + 1].cpu(), want[None], a[None], V, "behind a prefix")
    del kc, vc
    torch.cuda.empty_cache()


def test_lengths_outside_the_tables(dev):
    """A length past a table's pages counts as all of them, a negative one as none."""
    c = _case(dev, [80, 64, 48])
    full = c.table[:, :3].contiguous()
    for lens, eq in (([100, 64, 48], [48, 48, 48]), ([-5, 1 << 30, 3], [0, 48, 3])):
        a, b = _i32(lens, dev), _i32(eq, dev)
        for op in (lambda n: hmx.paged_attention_decode(c.qd, c.kc, c.vc, full, n, **c.sc),
                   lambda n: hmx.paged_causal_attention(c.qd, c.kc, c.vc, full, n, _i32([0, 1, 2, 3], dev), **c.sc),
                   lambda n: hmx.shared_prefix_attention_decode(c.qd, c.kc, c.vc, full, n, full[:1], n[:1], **c.sc)):
            assert torch.equal(op(a), op(b))


@pytest.mark.parametrize("width", [None, 300])
def test_unequal_numbers_of_new_tokens(dev, width):
    """One sequence's many tokens among single ones: blocks of 16 rows, cut and whole, with rows of
    no sequence before and behind."""
    news = [1] * 7 + [45, 0] + [2] * 12 + [9] * 3
    lens = [n + 13 * i % 400 for i, n in enumerate(news)]
    lens[7], lens[8], lens[3] = 700, 0, 0
    c = _case(dev, lens, G=2, HKV=2, D=64, width=width)
    cu = [2]
    for n in news:
        cu.append(cu[-1] + n)
    T = cu[-1] + 3
    q = randn(c.gen, T, 4, 64, scale=0.5)
    assert T * 2 <= 16 * len(news)
    o = hmx.paged_causal_attention(q.to(dev), c.kc, c.vc, c.table, c.lens, _i32(cu, dev), **c.sc)
    left = torch.full_like(o, 7.0)
    hmx.paged_causal_attention(q.to(dev), c.kc, c.vc, c.table, c.lens, _i32(cu, dev), out=left, **c.sc)
    o, left = o.cpu(), left.cpu()
    for a, b in ((0, 2), (T - 3, T)):
        assert (o[a:b] == 0).all() and (left[a:b] == 7).all()
    assert torch.equal(o[2:T - 3], left[2:T - 3])
    for n in range(len(news)):
        a, b = cu[n], cu[n + 1]
        want, mag = ref.rows(q[a:b], c.kl[n], c.vl[n], 64 ** -0.5, lens[n] - (b - a))
        check_o(o[a:b], want, mag, c.vl[n], f"sequence {n}")


def test_a_prefix_is_the_same_as_its_pages_in_every_table(dev):
    """shared_prefix_attention_decode over tables cut behind whole pages against the decode over the
    whole tables, of rows few and many."""
    for N, eight in ((6, True), (80, True), (6, False), (80, False)):
        gen = torch.Generator().manual_seed(N)
        lens = [500 + 7 * i % 90 for i in range(N)]
        if eight:
            kc, vc, ks, vs, table, kl, vl = paged8(gen, lens, 16, 2, 128)
            sc = dict(k_scales=ks.to(dev), v_scales=vs.to(dev))
        else:
            (kc, vc, table, kl, vl), sc = paged(gen, lens, 16, 2, 128, BF), {}
        table[:, :30] = table[0, :30]
        q = randn(gen, N, 8, 128, scale=0.5)
        args = (q.to(dev), kc.to(dev), vc.to(dev))
        t, n = table.to(dev), _i32(lens, dev)
        a = hmx.paged_attention_decode(*args, t, n, **sc)
        b = hmx.shared_prefix_attention_decode(*args, t[:, 30:], n - 480, t[:1, :30], _i32([480], dev), **sc)
        vmax = max(v.double().abs().amax().item() for v in vl)
        # each is within the elementwise bound of one exact value: (half step of P + 2^-12) sum p |v| twice, and roundings
        tol = 2 * ((half_step(BF) + 2.0 ** -12) * vmax + half_step(BF) * vmax)
        assert (a.float() - b.float()).abs().max().item() <= tol


def test_registered_ops(dev):
    """torch.ops.hmx's forms give what the functions give, and refuse a backward; the rotation's is
    its own, also compiled away from Python's autograd function."""
    c = _case(dev, [70, 5, 33])
    a = (c.kc, c.vc, c.sc["k_scales"], c.sc["v_scales"])
    args = (c.qd, c.kc, c.vc, c.table, c.lens)
    cu = _i32([0, 1, 2, 3], dev)
    pairs = [(lib.paged_attention_decode(*args, **c.sc), hmx.paged_attention_decode(*args, **c.sc)),
             (lib.paged_causal_attention(*args, cu, **c.sc), hmx.paged_causal_attention(*args, cu, **c.sc)),
             (lib.shared_prefix_attention_decode(*args, c.table[:1], c.lens[:1], **c.sc),
              hmx.shared_prefix_attention_decode(*args, c.table[:1], c.lens[:1], **c.sc))]
    assert all(torch.equal(x, y) for x, y in pairs)
    k = randn(c.gen, 3, 2, 64).to(dev)
    caches = [[x.view(torch.uint8).clone() for x in a] for _ in range(2)]
    for op, (x, y, s, t) in zip((hmx.append_paged_kv, lib.append_paged_kv), caches):
        assert op(k, k, x.view(F8), y.view(F8), torch.tensor([1, 40, 20], device=dev), k_scales=s, v_scales=t) is None
    assert all(torch.equal(x, y) for x, y in zip(*caches))
    q = c.qd.clone().requires_grad_()
    for f in (hmx.paged_attention_decode, lib.paged_attention_decode):
        with pytest.raises((NotImplementedError, RuntimeError), match="no backward"):
            f(q, *args[1:], **c.sc).sum().backward()
    with pytest.raises((NotImplementedError, RuntimeError), match="no backward"):
        hmx.shared_prefix_attention_decode(q, *args[1:], c.table[:1], c.lens[:1], **c.sc).sum().backward()
    inv, _ = hmx.rotary_frequencies(64, device=dev)
    pos, q4, k4 = torch.arange(3, device=dev) + 9, c.qd[None].requires_grad_(), k[None].clone().requires_grad_()
    got, want = lib.rotary_embedding(q4, k4, pos, inv, factor=1.5), hmx.rotary_embedding(q4, k4, pos, inv, factor=1.5)
    do = [randn(c.gen, *x.shape).to(dev) for x in want]
    g, w = (torch.autograd.grad(x, (q4, k4), do) for x in (got, want))
    assert all(torch.equal(x, y) for x, y in zip((*got, *g), (*want, *w)))
