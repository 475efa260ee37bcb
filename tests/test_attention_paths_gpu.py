"""The attention ops as they are used together: prompts in pieces and token by token through
the cache against one whole prompt, the serving core against the oracle, captured graphs
replayed with other lengths, other streams, and the registered ops."""
from types import SimpleNamespace

import pytest
import torch

import hmx
import hmx.library as lib
import hmx.serving as serving
from attn_util import check_o, randn, ref

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _table(seqs, width, pages, gen):
    return torch.randperm(pages, generator=gen)[:seqs * width].view(seqs, width).to(torch.int32)


def _slots(table, seq, pos, page):
    return table[seq, pos // page].long() * page + pos % page


def test_pieces_and_tokens_through_the_cache_equal_a_whole_prompt(dev):
    """Two sequences: prompts appended and attended in pieces, then token by token; every row
    against the oracle's whole causal attention on the values the cache holds."""
    gen = torch.Generator().manual_seed(0)
    H, HKV, D, page, T = 8, 2, 128, 16, [150, 97]
    table = _table(2, 12, 30, gen)
    kc = torch.full((30, page, HKV, D), float("nan"), dtype=BF, device=dev)
    vc = kc.clone()
    q, k, v = ([randn(gen, t, h, D) for t in T] for h in (H, HKV, HKV))
    ang = torch.rand(160, D // 2, generator=gen) * 6
    cs = torch.cat([ang.cos(), ang.sin()], 1).to(dev)
    tab = table.to(dev)
    got = [torch.empty(t, H, D, dtype=BF) for t in T]
    done = [0, 0]
    for new in ([60, 33], [1, 50], [64, 0], [0, 5]):
        part = [(s, done[s] + i) for s in range(2) for i in range(new[s])]
        seq, pos = (torch.tensor(x) for x in zip(*part))
        rows = [torch.stack([x[s][p] for s, p in part]).to(dev) for x in (q, k, v)]
        rq = hmx.append_paged_kv(rows[1], rows[2], kc, vc, _slots(table, seq, pos, page).to(dev), q=rows[0],
                                 positions=pos.to(dev), cos_sin=cs)
        done = [done[s] + new[s] for s in range(2)]
        cu = torch.tensor([0, new[0], new[0] + new[1]], dtype=torch.int32, device=dev)
        o = hmx.paged_causal_attention(rq, kc, vc, tab, torch.tensor(done, dtype=torch.int32, device=dev), cu).cpu()
        for (s, p), row in zip(part, o):
            got[s][p] = row
    while any(done[s] < T[s] for s in range(2)):        # a finished sequence stays as padding
        live = [done[s] < T[s] for s in range(2)]
        pos = torch.tensor([min(done[s], T[s] - 1) for s in range(2)])
        slots = _slots(table, torch.arange(2), pos, page)
        slots[~torch.tensor(live)] = -1
        rows = [torch.stack([x[s][pos[s]] for s in range(2)]).to(dev) for x in (q, k, v)]
        rq = hmx.append_paged_kv(rows[1], rows[2], kc, vc, slots.to(dev), q=rows[0], positions=pos.to(dev), cos_sin=cs)
        done = [done[s] + live[s] for s in range(2)]
        lens = torch.tensor([done[s] if live[s] else 0 for s in range(2)], dtype=torch.int32, device=dev)
        o = hmx.paged_attention_decode(rq, kc, vc, tab, lens).cpu()
        for s in range(2):
            if live[s]:
                got[s][pos[s]] = o[s]
            else:
                assert (o[s] == 0).all()
    for s in range(2):
        rk = ref.gather(kc.cpu(), table[s], T[s])
        # the rotated q as the op rounds it (its own test compares it with the oracle)
        p = torch.arange(T[s])
        rq = hmx.append_paged_kv(k[s].to(dev), v[s].to(dev), kc.clone(), vc.clone(),
                                 torch.full((T[s],), -1, device=dev), q=q[s].to(dev), positions=p.to(dev), cos_sin=cs)
        o, a = ref.causal(rq.cpu(), rk, v[s], D ** -0.5, [(0, T[s])])
        check_o(got[s], o, a, v[s], f"sequence {s}")
        assert torch.equal(ref.gather(vc.cpu(), table[s], T[s]), v[s])
        whole = hmx.causal_attention(rq[None], rk[None].to(dev), v[s][None].to(dev))
        check_o(whole[0], o, a, v[s], f"whole prompt {s}")


@pytest.mark.parametrize("rope", [None, True, False])
@pytest.mark.parametrize("batch", ["mixed", "decode", "prefill", "drafts"])
def test_attention_forward_core(dev, rope, batch):
    gen = torch.Generator().manual_seed(3)
    H, HKV, D, page = 8, 2, 64, 16
    nd, news = {"mixed": (3, [1, 1, 1, 20, 5]), "decode": (3, [1, 1, 1]), "prefill": (0, [40, 7]),
                "drafts": (2, [3, 3, 11])}[batch]
    N, n, pad = len(news), sum(news), 4
    ctx = [int(x) for x in torch.randint(0, 90, (N,), generator=gen)]
    lens = [c + m for c, m in zip(ctx, news)]
    table = _table(N, 9, 50, gen)
    kc, vc = (randn(gen, 50, page, HKV, D) for _ in range(2))
    qkv = randn(gen, n + pad, (H + 2 * HKV) * D)
    pos = torch.cat([torch.arange(c, c + m) for c, m in zip(ctx, news)])
    seq = torch.cat([torch.full((m,), i) for i, m in enumerate(news)])
    ang = torch.rand(160, 16, generator=gen) * 6
    cs = torch.cat([ang.cos(), ang.sin()], 1)
    cu = [0]
    for m in news:
        cu.append(cu[-1] + m)
    lay = SimpleNamespace(num_heads=2 * H, num_kv_heads=2 * HKV, head_dim=D, tp_size=2, scaling=0.2,
                          rotary_emb=None if rope is None else
                          SimpleNamespace(cos_sin_cache=cs.to(dev), is_neox_style=rope))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    md = SimpleNamespace(num_actual_tokens=n, num_decodes=nd, num_decode_tokens=cu[nd], num_prefills=N - nd,
                         query_start_loc=i32(cu), seq_lens=i32(lens), block_table=table.to(dev),
                         slot_mapping=_slots(table, seq, pos, page).to(dev))
    out = torch.full((n + pad, H, D), 5.0, dtype=BF, device=dev)
    k2, v2 = kc.to(dev), vc.to(dev)
    serving.attention_forward_core(lay, qkv.to(dev), pos.to(dev), out, md, k2, v2)
    assert (out[n:] == 5).all()
    q, k, v = (x.reshape(n, -1, D) for x in qkv[:n].split([H * D, HKV * D, HKV * D], -1))
    if rope is not None:
        q = hmx.append_paged_kv(k.to(dev), v.to(dev), k2.clone(), v2.clone(), torch.full((n,), -1, device=dev),
                                q=q.to(dev), positions=pos.to(dev), cos_sin=cs.to(dev), interleaved=not rope).cpu()
        want = ref.rotate(k, cs, pos, not rope)
    for s in range(N):
        rows = slice(cu[s], cu[s + 1])
        K, V = ref.gather(k2.cpu(), table[s], lens[s]), ref.gather(v2.cpu(), table[s], lens[s])
        old = ref.gather(kc, table[s], ctx[s])
        assert torch.equal(K[:ctx[s]], old) and torch.equal(V[ctx[s]:], v[rows])
        if rope is None:
            assert torch.equal(K[ctx[s]:], k[rows])
        else:
            mag = k[rows].double().abs().amax(-1, keepdim=True)
            err = (K[ctx[s]:].double() - want[rows]).abs()
            assert (err <= 2.0 ** -8 * want[rows].abs() + 2.0 ** -21 * mag).all()
        o, a = ref.rows(q[rows], K, V, 0.2, ctx[s])
        check_o(out[rows], o, a, V, f"{batch} {s}")
    serving.attention_forward_core(lay, qkv.to(dev), pos.to(dev), out, None, k2, v2)     # profile run


def test_captured_step_replays_with_other_lengths(dev):
    """A decode step captured once: appended tokens, lengths, tables and offsets change
    between replays, eager work runs between them, and every replay equals the eager call.
    Two graphs of different batches are replayed in turn."""
    gen = torch.Generator().manual_seed(7)
    H, HKV, D, page, W = 8, 2, 128, 16, 200
    steps = []
    for N in (5, 3):
        pages = N * W + 1
        st = SimpleNamespace(N=N, kc=randn(gen, pages, page, HKV, D).to(dev), vc=randn(gen, pages, page, HKV, D).to(dev),
                             q=torch.empty(N, H, D, dtype=BF, device=dev), k=torch.empty(N, HKV, D, dtype=BF, device=dev),
                             v=torch.empty(N, HKV, D, dtype=BF, device=dev),
                             slots=torch.zeros(N, dtype=torch.int64, device=dev),
                             pos=torch.zeros(N, dtype=torch.int64, device=dev),
                             lens=torch.ones(N, dtype=torch.int32, device=dev),
                             table=torch.zeros(N, W, dtype=torch.int32, device=dev),
                             cu=torch.arange(N + 1, dtype=torch.int32, device=dev),
                             cs=torch.randn(3300, D, generator=gen).to(dev))

        def step(st=st):
            q = hmx.append_paged_kv(st.k, st.v, st.kc, st.vc, st.slots, q=st.q, positions=st.pos, cos_sin=st.cs)
            return (hmx.paged_attention_decode(q, st.kc, st.vc, st.table, st.lens),
                    hmx.paged_causal_attention(q, st.kc, st.vc, st.table, st.lens, st.cu))

        st.step = step
        steps.append(st)

    def load(st, seed):
        g = torch.Generator().manual_seed(seed)
        table = torch.randperm(st.N * W + 1, generator=g)[:st.N * W].view(st.N, W)
        lens = torch.randint(0, 3200, (st.N,), generator=g)
        lens[0], lens[-1] = 3200, 1
        pos = (lens - 1).clamp(min=0)
        slots = table[torch.arange(st.N), pos // page] * page + pos % page
        slots[lens == 0] = -1
        for t, x in ((st.table, table), (st.lens, lens), (st.pos, pos), (st.slots, slots)):
            t.copy_(x)
        for t in (st.q, st.k, st.v):
            t.copy_(randn(g, *t.shape))

    side = torch.cuda.Stream()
    for st in steps:
        load(st, 1)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            st.step()
        torch.cuda.current_stream().wait_stream(side)
        st.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(st.graph):
            st.out = st.step()
    for seed in range(2, 6):
        for st in steps:
            load(st, seed)
            st.graph.replay()
            got = [x.clone() for x in st.out]
            torch.cuda.synchronize()
            for x, y in zip(got, st.step()):
                assert torch.equal(x, y)


def test_captured_training_step(dev):
    """Forward and backward of leaves that no eager graph holds, replayed on new inputs."""
    gen = torch.Generator().manual_seed(5)
    q, k, v, do = (randn(gen, 1, 200, n, 64).to(dev) for n in (4, 2, 2, 4))
    cu = torch.tensor([0, 77, 200], dtype=torch.int32, device=dev)

    def step():
        ins = [x.detach().requires_grad_() for x in (q, k, v)]
        o = hmx.causal_attention(*ins, cu_seqlens=cu)
        return (o.detach(), *torch.autograd.grad(o, ins, do))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for cut in (77, 1, 199):
        cu[1] = cut
        for x in (q, k, v, do):
            x.copy_(randn(gen, *x.shape))
        graph.replay()
        got = [x.clone() for x in out]
        torch.cuda.synchronize()
        for x, y in zip(got, step()):
            assert torch.equal(x, y)


def test_host_offsets_refused_under_capture(dev):
    q = torch.zeros(1, 8, 2, 64, dtype=BF, device=dev)
    graph = torch.cuda.CUDAGraph()
    keep = torch.zeros(1, device=dev)
    with torch.cuda.graph(graph):
        keep.add_(1)
        with pytest.raises(RuntimeError, match="on the device"):
            hmx.causal_attention(q, q, q, cu_seqlens=torch.tensor([0, 8]))


def test_other_stream(dev):
    """Calls on a side stream use that stream; two at once do not disturb each other."""
    gen = torch.Generator().manual_seed(2)
    sets = []
    for i in range(2):
        q, k, v = (randn(gen, 1, 900, n, 64).to(dev) for n in (4, 2, 2))
        kc, vc = (randn(gen, 300, 16, 2, 64).to(dev) for _ in range(2))
        table = torch.randperm(300, generator=gen)[:200].view(2, 100).to(torch.int32).to(dev)
        lens = torch.tensor([1600, 1200 + i], dtype=torch.int32, device=dev)
        sets.append((q, k, v, kc, vc, table, lens))
    run = lambda s: (hmx.causal_attention(*s[:3]), hmx.paged_attention_decode(s[0][0, :2], *s[3:]),
                     hmx.paged_causal_attention(s[0][0, :8], *s[3:], torch.tensor([0, 3, 8], dtype=torch.int32)))
    want = [run(s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for _ in range(3):
        got = []
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(run(s))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(g, w))


def test_registered_ops(dev):
    """torch.ops.hmx.*: the same results, the gradient, and torch's own checks of schema,
    fake outputs and autograd registration."""
    gen = torch.Generator().manual_seed(4)
    q, k, v, do = (randn(gen, 1, 70, n, 64).to(dev) for n in (4, 2, 2, 4))
    cu = torch.tensor([0, 30, 70], dtype=torch.int32, device=dev)
    ins = [x.clone().requires_grad_() for x in (q, k, v)]
    o = lib.causal_attention(*ins, cu_seqlens=cu)
    want = hmx.causal_attention(*ins, cu_seqlens=cu)
    assert torch.equal(o, want)
    for a, b in zip(torch.autograd.grad(o, ins, do), torch.autograd.grad(want, ins, do)):
        assert torch.equal(a, b)
    kc, vc = (randn(gen, 20, 16, 2, 64).to(dev) for _ in range(2))
    table = torch.arange(20, dtype=torch.int32, device=dev).view(2, 10)
    lens = torch.tensor([100, 33], dtype=torch.int32, device=dev)
    assert torch.equal(lib.paged_attention_decode(q[0, :2], kc, vc, table, lens),
                       hmx.paged_attention_decode(q[0, :2], kc, vc, table, lens))
    assert torch.equal(lib.paged_causal_attention(q[0], kc, vc, table, lens, cu),
                       hmx.paged_causal_attention(q[0], kc, vc, table, lens, cu))
    slots, pos = torch.arange(70, device=dev), torch.arange(70, device=dev)
    cs = torch.randn(70, 64, generator=gen).to(dev)
    k2, v2, k3, v3 = kc.clone(), vc.clone(), kc.clone(), vc.clone()
    a = lib.append_paged_kv(k[0], v[0], k2, v2, slots, q=q[0], positions=pos, cos_sin=cs)
    b = hmx.append_paged_kv(k[0], v[0], k3, v3, slots, q=q[0], positions=pos, cos_sin=cs)
    assert torch.equal(a, b) and torch.equal(k2, k3) and torch.equal(v2, v3)
    assert lib.append_paged_kv(k[0], v[0], k2, v2, slots) is None
    checks = ("test_schema", "test_faketensor", "test_autograd_registration")
    torch.library.opcheck(torch.ops.hmx.causal_attention, (*ins, 0.1, cu), test_utils=checks)
    torch.library.opcheck(torch.ops.hmx.append_paged_kv, (k[0], v[0], k2, v2, slots, q[0], pos, cs, False),
                          test_utils=checks)
    torch.library.opcheck(torch.ops.hmx.paged_attention_decode, (q[0, :2], kc, vc, table, lens, None), test_utils=checks)
    torch.library.opcheck(torch.ops.hmx.paged_causal_attention, (q[0], kc, vc, table, lens, cu, None),
                          test_utils=checks)


def test_shared_inputs_and_leaves(dev):
    """One tensor as q, k and v: its gradient is the sum of the three."""
    x = randn(torch.Generator().manual_seed(1), 1, 80, 2, 64).to(dev)
    a, b, c = (x.clone().requires_grad_() for _ in range(3))
    sep = torch.autograd.grad(hmx.causal_attention(a, b, c).float().square().sum(), (a, b, c))
    y = x.clone().requires_grad_()
    one, = torch.autograd.grad(hmx.causal_attention(y, y, y).float().square().sum(), y)
    tol = 3 * 2.0 ** -8 * sum(s.abs().float() for s in sep) + 1e-30
    assert ((one.float() - sum(s.float() for s in sep)).abs() <= tol).all()


def test_captured_prompts_whose_keys_are_split(dev):
    """Packed prompts of few rows, whose keys are split and joined through a workspace: two
    graphs replayed in turn with other offsets and inputs, eager work between them."""
    gen = torch.Generator().manual_seed(14)
    steps = []
    for T, H, HKV, D in ((3000, 4, 1, 128), (2100, 2, 2, 64)):
        q, k, v = (randn(gen, 1, T, n, D).to(dev) for n in (H, HKV, HKV))
        cu = torch.tensor([0, 700, 700, T], dtype=torch.int32, device=dev)
        st = SimpleNamespace(T=T, ins=(q, k, v), cu=cu)
        st.step = lambda st=st: (hmx.causal_attention(*st.ins, cu_seqlens=st.cu), hmx.causal_attention(*st.ins))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            st.step()
        torch.cuda.current_stream().wait_stream(side)
        st.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(st.graph):
            st.out = st.step()
        steps.append(st)
    for cut in (1, 1000, 64, 2000):
        for st in steps:
            st.cu[1] = st.cu[2] = cut
            st.cu[2] += 7
            st.cu[3] = st.T - cut % 5
            for x in st.ins:
                x.copy_(randn(gen, *x.shape))
            st.graph.replay()
            got = [x.clone() for x in st.out]
            torch.cuda.synchronize()
            for x, y in zip(got, st.step()):
                assert torch.equal(x, y)
    for st in steps:                              # the case is one that splits
        (_, T, H, D), HKV = st.ins[0].shape, st.ins[1].shape[2]
        assert hmx._lib.load().hmx_causal_attention_workspace_bytes(3, T, H, HKV, D, 1) > 0
