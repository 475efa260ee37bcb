"""Host-side checks of the ops over caches of 8 bits, of shared prefixes and of the rotation by
frequencies (CPU): refusals before any launch, the C entry points' own checks, the frequencies
and the oracle."""
import ctypes
import math
from types import SimpleNamespace

import pytest
import torch

import hmx
from hmx import _lib
from oracle import attention as ref

BF, F8 = torch.bfloat16, torch.float8_e4m3fn


def _cache8(pages=3, page=16, HKV=2, D=64):
    kv = [torch.zeros(pages, page, HKV, D, dtype=torch.uint8).view(F8) for _ in range(2)]
    return (*kv, *(torch.ones(pages, HKV, page, dtype=torch.uint8) for _ in range(2)))


def test_oracle_e4m3_against_the_type():
    """Every value of the type, every midpoint of two, and random numbers, as torch's conversion."""
    values = torch.arange(256, dtype=torch.uint8).view(F8).double()
    values = values[torch.isfinite(values)].sort().values
    mid = (values[1:] + values[:-1]) / 2
    x = torch.cat([values, mid, mid * (1 + 2.0 ** -20), mid * (1 - 2.0 ** -20),
                   torch.randn(4000, generator=torch.Generator().manual_seed(0)).double() * 20])
    assert torch.equal(ref.to_e4m3(x), x.float().to(F8).double())


def test_oracle_quantise_by_hand():
    x = torch.tensor([[448.0, 1.0], [449.0, 0.0], [0.0, 0.0], [0.875, -0.1], [float("inf"), 7.0], [2.0 ** -140, 0.0]])
    v, e = ref.quantise(x)
    # 449 > 448 needs 2^1: 224.5 -> 224; 0.875 = 448 * 2^-9, -51.2 -> -52
    assert e.tolist() == [0, 1, -126, -9, -6, -126]
    assert v[0].tolist() == [448.0, 1.0] and v[1].tolist() == [224.0, 0.0] and v[3].tolist() == [448.0, -52.0]
    assert torch.isnan(v[4, 0]) and v[4, 1] == 448.0 and v[5, 0] == 0.0


@pytest.mark.parametrize("inter", [False, True])
def test_oracle_rotation_as_complex_products(inter):
    gen = torch.Generator().manual_seed(1)
    x, ang = torch.randn(5, 3, 64, generator=gen).double(), torch.rand(5, 8, generator=gen).double() * 9
    pairs = x[..., :16].unflatten(-1, (8, 2) if inter else (2, 8))
    re, im = pairs.unbind(-1 if inter else -2)
    z = torch.complex(re, im) * torch.polar(torch.full_like(ang, 1.5), ang)[:, None]
    want = torch.stack([z.real, z.imag], -1 if inter else -2).flatten(-2)
    got = ref.rotate_by(x, ang, 1.5, inter)
    assert (got[..., :16] - want).abs().max() <= 2.0 ** -48 and torch.equal(got[..., 16:], x[..., 16:])


def test_append_refusals():
    k = torch.zeros(5, 2, 64, dtype=BF)
    kc, vc, ks, vs = _cache8()
    call = lambda **kw: hmx.append_paged_kv(**{**dict(k=k, v=k, k_cache=kc, v_cache=vc, slot_mapping=torch.arange(5),
                                                      k_scales=ks, v_scales=vs), **kw})
    with pytest.raises(RuntimeError, match="GPU"):
        call()
    for kw in (dict(k_scales=None), dict(v_scales=None), dict(k_scales=None, v_scales=None), dict(v_cache=vc.to(BF)),
               dict(k_cache=kc.to(BF), v_cache=vc.to(BF)), dict(k_scales=ks.int()), dict(k_scales=ks.transpose(1, 2)),
               dict(v_scales=vs[:2]), dict(v_scales=torch.ones(3, 16, 2, dtype=torch.uint8).transpose(1, 2)),
               dict(k_cache=torch.zeros(3, 16, 2, 72, dtype=torch.uint8).view(F8)[..., :64]),
               dict(k_scales=ks[:1].expand(3, 2, 16)), dict(v_scales=vs[:, :1].expand(3, 2, 16))):
        with pytest.raises(ValueError):
            call(**kw)
    with pytest.raises(NotImplementedError):
        call(k=k.float(), v=k.float())


def test_attention_refusals():
    kc, vc, ks, vs = _cache8()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)
    q, table, lens = torch.zeros(2, 4, 64, dtype=BF), torch.zeros(2, 3, dtype=torch.int32), i32(1, 1)
    args = dict(q=q, k_cache=kc, v_cache=vc, block_table=table, seq_lens=lens, k_scales=ks, v_scales=vs)
    more = {hmx.paged_attention_decode: {}, hmx.paged_causal_attention: dict(cu_seqlens=i32(0, 1, 2)),
            hmx.shared_prefix_attention_decode: dict(prefix_table=table[:1], prefix_lens=lens[:1])}
    for op, m in more.items():
        with pytest.raises(RuntimeError, match="GPU"):
            op(**args, **m)
        for kw in (dict(k_scales=None), dict(v_scales=vs[:, :1]), dict(v_cache=vc.to(BF)), dict(k_scales=ks.float()),
                   dict(block_table=table.long()), dict(seq_lens=lens[:1]), dict(q=q[:, :3]), dict(scale=-1.0), dict(q=q[0]),
                   dict(out=q.half()), dict(k_scales=None, v_scales=None)):
            with pytest.raises(ValueError):
                op(**{**args, **m, **kw})
        with pytest.raises(NotImplementedError):
            op(**{**args, **m, "q": q.float()})
    m = more[hmx.shared_prefix_attention_decode]
    for kw in (dict(prefix_table=table), dict(prefix_table=table[0]), dict(prefix_lens=lens), dict(prefix_lens=lens[:1].long()),
               dict(prefix_table=table, prefix_lens=lens), dict(cu_prefix=i32(0, 1, 2)), dict(cu_prefix=torch.zeros(2, 2))):
        with pytest.raises(ValueError):
            hmx.shared_prefix_attention_decode(**{**args, **m, **kw})


def test_rotary_refusals():
    q, k = torch.zeros(2, 5, 4, 64, dtype=BF), torch.zeros(2, 5, 2, 64, dtype=BF)
    pos, inv = torch.arange(5), torch.ones(32)
    call = lambda **kw: hmx.rotary_embedding(**{**dict(q=q, k=k, positions=pos, inv_freq=inv), **kw})
    with pytest.raises(RuntimeError, match="GPU"):
        call()
    for kw in (dict(k=k[:1]), dict(k=k[:, :, :, :32]), dict(k=k.half()), dict(k=k[0]), dict(q=q[0, 0]), dict(positions=pos[:4]),
               dict(positions=pos.float()), dict(positions=torch.zeros(3, 5, dtype=torch.long)), dict(inv_freq=inv[:12]),
               dict(inv_freq=torch.ones(40)), dict(inv_freq=inv.half()), dict(inv_freq=inv[None]), dict(inv_freq=inv[:0]),
               dict(factor=float("nan")), dict(q_out=q[:1]), dict(k_out=k.half()), dict(k=None, k_out=k), dict(q=q[:, :, :0]),
               dict(q_out=q[:, :1].expand(2, 5, 4, 64)), dict(q_out=torch.zeros(q.numel() + 1, dtype=BF)[1:].view(q.shape))):
        with pytest.raises(ValueError):
            call(**kw)
    with pytest.raises(NotImplementedError, match="bf16 or fp16"):
        call(q=q.float(), k=k.float())
    with pytest.raises(NotImplementedError, match="head size"):
        call(q=torch.zeros(2, 5, 4, 96, dtype=BF), k=None)
    with pytest.raises(NotImplementedError, match="frequencies"):
        call(inv_freq=inv.clone().requires_grad_())
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(q=fwd.make_dual(q, torch.ones_like(q)))
    with pytest.raises(RuntimeError, match="GPU"):
        hmx.rotary_table(inv, 9)
    for kw in (dict(positions=-1), dict(inv_freq=inv[:0], positions=2), dict(inv_freq=inv.int(), positions=2)):
        with pytest.raises(ValueError):
            hmx.rotary_table(**{"inv_freq": inv, **kw})


def test_frequencies():
    f = lambda *a, **kw: hmx.rotary_frequencies(*a, device="cpu", **kw)
    inv, factor = f(64)
    assert inv.dtype == torch.float64 and factor == 1.0 and inv[0] == 1
    assert torch.allclose(inv, 1e4 ** (-torch.arange(32).double() / 32), rtol=1e-14, atol=0)
    assert torch.equal(f(64, scaling=dict(rope_type="default"))[0], inv)
    assert torch.equal(f(64, scaling=dict(type="linear", factor=4))[0], inv / 4)
    ntk, factor = f(64, 1e4, dict(rope_type="ntk", factor=8.0))
    assert factor == 1.0 and ntk[0] == 1 and abs(ntk[-1] * 8 / inv[-1] - 1) < 1e-12     # the last pair is stretched by s
    yarn, factor = f(128, 1e6, dict(rope_type="yarn", factor=8.0, original_max_position_embeddings=32768))
    inv, _ = f(128, 1e6)
    turns = 32768 * inv / (2 * math.pi)
    assert torch.equal(yarn[turns > 60], inv[turns > 60]) and torch.allclose(yarn[turns < 0.5], inv[turns < 0.5] / 8, rtol=1e-14)
    assert ((yarn <= inv) & (yarn >= inv / 8 * (1 - 1e-14))).all() and abs(factor - (0.1 * math.log(8) + 1)) < 1e-15
    assert f(128, 1e6, dict(rope_type="yarn", factor=8.0, original_max_position_embeddings=32768, attention_factor=1.5))[1] == 1.5
    for bad in (dict(rotary_dim=3), dict(rotary_dim=64, base=1.0), dict(rotary_dim=64, scaling=dict(rope_type="linear")),
                dict(rotary_dim=64, scaling=dict(rope_type="linear", factor=0.5)),
                dict(rotary_dim=64, scaling=dict(rope_type="linear", factor=2.0, beta_fast=3)),
                dict(rotary_dim=64, scaling=dict(rope_type="yarn", factor=2.0)),
                dict(rotary_dim=64, scaling=dict(rope_type="yarn", factor=2.0, original_max_position_embeddings=9, beta_fast=0.5))):
        with pytest.raises(ValueError):
            hmx.rotary_frequencies(device="cpu", **bad)
    with pytest.raises(NotImplementedError, match="rope_type"):
        f(64, scaling=dict(rope_type="another", factor=2.0))


def test_c_entry_points_check_before_launching():
    kv = ctypes.pointer(_lib.PagedKV(0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 4, 3, 16))
    sc = ctypes.pointer(_lib.KVScales())
    dec = lambda kv=kv, sc=sc, N=1, D=64, qp=256, ws=0: _lib.call(
        "hmx_paged_attention_decode8", qp, 0, 0, 1, qp, 0, 0, kv, sc, N, 4, 2, D, 1.0, None, ws, None)
    with pytest.raises(ValueError, match="no scales"):
        dec(sc=None)
    with pytest.raises(NotImplementedError, match="head size 96"):
        dec(D=96)
    with pytest.raises(ValueError, match="null pointer"):
        dec()
    dec(N=0)
    full = lambda **kw: ctypes.pointer(_lib.PagedKV(**{**dict(k=256, k_page_stride=2048, k_token_stride=128, k_head_stride=64,
                                                              v=256, v_page_stride=2048, v_token_stride=128, v_head_stride=64,
                                                              table=256, table_stride=4, seq_lens=256, table_width=4, num_pages=3,
                                                              page_size=16), **kw}))
    with pytest.raises(ValueError, match="null pointer"):
        dec(kv=full())                                  # no bytes of scale
    some = ctypes.pointer(_lib.KVScales(256, 32, 16, 256, 32, 16))
    with pytest.raises(ValueError, match="multiples"):
        dec(kv=full(k_token_stride=136), sc=some)       # whole units of 8 elements, but not of 16 bytes
    with pytest.raises(NotImplementedError, match="2\\^25"):
        dec(kv=full(v_token_stride=1 << 25), sc=some)
    far = full(table_width=400)
    with pytest.raises(ValueError, match="too small"):
        dec(kv=far, sc=some)
    with pytest.raises(ValueError, match="no scales"):
        _lib.call("hmx_paged_causal_attention8", None, 0, 0, 1, None, 0, 0, kv, None, None, 1, 1, 4, 2, 64, 1.0, 1, None, 0, None)
    with pytest.raises(ValueError, match="no scales"):
        _lib.call("hmx_append_paged_kv8", None, 0, 0, None, 0, 0, None, 0, 0, 1, None, 0, 0, kv, None, None, 1,
                  None, 0, None, 0, 0, 0, 0, 0, 5, 4, 2, 64, None)
    with pytest.raises(ValueError, match="null pointer"):
        _lib.call("hmx_append_paged_kv8", None, 0, 0, 256, 128, 64, 256, 128, 64, 1, None, 0, 0, full(), sc, 256, 1,
                  None, 0, None, 0, 0, 0, 0, 0, 5, 4, 2, 64, None)
    shared = lambda ws, size, M=1, cu=None, width=4, plens=256: _lib.call(
        "hmx_shared_prefix_decode", 256, 256, 64, 1, 256, 256, 64, full(), some, 256, 4, width, plens, cu, 8, M, 4, 2, 64,
        1.0, ws, size, None)
    n = _lib.load().hmx_shared_prefix_decode_workspace_bytes(8, 1, 4, 2, 64, 64, 64)
    assert n > 0
    for ws, size in ((None, n), (256, n - 1), (264, n)):
        with pytest.raises(ValueError, match="too small"):
            shared(ws, size)
    with pytest.raises(ValueError, match="without offsets"):
        shared(256, n, M=2)
    with pytest.raises(ValueError, match="null pointer"):
        shared(256, n, plens=None)
    with pytest.raises(NotImplementedError, match="a table row holds"):
        shared(256, 1 << 40, width=1 << 27)
    rot = lambda D=64, R=64, B=1, T=4, qp=256, ts=256: _lib.call(
        "hmx_rotary_embedding", qp, 1024, ts, 64, 256, 1024, 256, 64, *[None, 0, 0, 0] * 2, 1, 256, 1, 0, 256, 1, 1.0, R, 0, 0,
        B, T, 4, 0, D, None)
    for kw in (dict(D=96), dict(R=24), dict(R=128), dict(B=2, T=1 << 30)):
        with pytest.raises(NotImplementedError):
            rot(**kw)
    for kw in (dict(qp=None), dict(qp=264), dict(ts=68)):
        with pytest.raises(ValueError):
            rot(**kw)
    rot(T=0)


def test_registered_with_fakes_and_mutations():
    import hmx.library  # noqa: F401
    m = torch.device("meta")
    q, k = torch.empty(9, 4, 64, dtype=BF, device=m), torch.empty(9, 2, 64, dtype=BF, device=m)
    kc, sc = torch.empty(3, 16, 2, 64, dtype=F8, device=m), torch.empty(3, 2, 16, dtype=torch.uint8, device=m)
    tab, n = torch.empty(9, 2, dtype=torch.int32, device=m), torch.empty(9, dtype=torch.int32, device=m)
    assert torch.ops.hmx.append_paged_kv8(k, k, kc, kc.clone(), sc, sc.clone(), n, q, None, None, False).shape == (9, 4, 64)
    assert torch.ops.hmx.paged_attention_decode8(q, kc, kc, sc, sc, tab, n, None).dtype == BF
    assert torch.ops.hmx.paged_causal_attention8(q, kc, kc, sc, sc, tab, n, n, None).shape == (9, 4, 64)
    assert torch.ops.hmx.shared_prefix_attention_decode(q, kc, kc, sc, sc, tab, n, tab[:1], n[:1], None, None).shape == (9, 4, 64)
    a, b = torch.ops.hmx.rotary_embedding(q[None], None, n, n.double(), 1.0, False, False)
    assert a.shape == (1, 9, 4, 64) and b.numel() == 0
    w = {a.name for a in torch.ops.hmx.append_paged_kv8.default._schema.arguments
         if a.alias_info is not None and a.alias_info.is_write}
    assert w == {"k_cache", "v_cache", "k_scales", "v_scales"}


def test_forward_core_hands_on_scales_and_prefixes(monkeypatch):
    import hmx.serving as serving
    seen = []
    for name in ("append_paged_kv", "paged_attention_decode", "paged_causal_attention", "shared_prefix_attention_decode"):
        monkeypatch.setattr(serving.ops, name, lambda *a, _n=name, q=None, **kw: seen.append((_n, a, kw)) or q)
    kc, vc, ks, vs = _cache8()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)
    lay = SimpleNamespace(num_heads=4, num_kv_heads=2, head_dim=64, tp_size=1)
    md = SimpleNamespace(num_actual_tokens=5, num_decodes=2, num_decode_tokens=2, num_prefills=1,
                         query_start_loc=i32(0, 1, 2, 5), seq_lens=i32(4, 5, 3), block_table=torch.zeros(3, 2, dtype=torch.int32),
                         slot_mapping=i32(0, 1, 2, 3, 4))
    qkv, out = torch.zeros(5, 8 * 64, dtype=BF), torch.zeros(5, 4, 64, dtype=BF)
    core = lambda *sc: serving.attention_forward_core(lay, qkv, None, out, md, kc, vc, *sc)
    core(ks, vs)
    assert [n for n, _, _ in seen] == ["append_paged_kv", "paged_attention_decode", "paged_causal_attention"]
    assert all(kw["k_scales"] is ks and kw["v_scales"] is vs for _, _, kw in seen)
    seen.clear()
    core()
    assert all("k_scales" not in kw for _, _, kw in seen)
    seen.clear()
    md.prefix_table, md.prefix_lens, md.cu_prefix = torch.zeros(1, 2, dtype=torch.int32), i32(9), None
    core(ks, vs)
    assert [n for n, _, _ in seen] == ["append_paged_kv", "shared_prefix_attention_decode", "paged_causal_attention"]
    assert seen[1][1][0].shape[0] == 2 and seen[1][1][5] is md.prefix_table and seen[1][2]["v_scales"] is vs
    md.num_decode_tokens = 4
    with pytest.raises(NotImplementedError, match="draft"):
        core(ks, vs)
