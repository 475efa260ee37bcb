"""Host-side checks of the attention ops (CPU): refusals before any launch, the C entry
points' own checks, and the oracle's gradients against differences."""
import ctypes
from types import SimpleNamespace

import pytest
import torch

import hmx
from hmx import _lib
from oracle import attention as ref

BF = torch.bfloat16


def _qkv(B=1, T=4, H=4, HKV=2, D=64, dtype=BF):
    return (torch.zeros(B, T, H, D, dtype=dtype), torch.zeros(B, T, HKV, D, dtype=dtype),
            torch.zeros(B, T, HKV, D, dtype=dtype))


def _cache(pages=3, page=16, HKV=2, D=64, dtype=BF):
    return torch.zeros(pages, page, HKV, D, dtype=dtype), torch.zeros(pages, page, HKV, D, dtype=dtype)


def test_causal_attention_refusals():
    q, k, v = _qkv()
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU"):
        hmx.causal_attention(q, k, v)
    with pytest.raises(ValueError, match="Batch size expected to be 1"):
        hmx.causal_attention(*_qkv(B=2), cu_seqlens=cu)
    with pytest.raises(NotImplementedError, match="bf16 or fp16"):
        hmx.causal_attention(*_qkv(dtype=torch.float32))
    with pytest.raises(NotImplementedError, match="head size"):
        hmx.causal_attention(*_qkv(D=96))
    with pytest.raises(ValueError, match="differ"):
        hmx.causal_attention(q, k.half(), v)
    with pytest.raises(ValueError, match="cannot share"):
        hmx.causal_attention(*_qkv(H=3))
    for bad in ((q[0], k, v), (q, k[:, :3], v), (q, k, v[:, :, :1]), (q, k[..., :32], v[..., :32])):
        with pytest.raises(ValueError):
            hmx.causal_attention(*bad)


@pytest.mark.parametrize("cu", [[1, 4], [0, 5], [0, 3, 2], []])
def test_bad_host_offsets(cu):
    from hmx.ops.attention import _offsets
    with pytest.raises(ValueError, match="cu_seqlens"):
        _offsets(torch.tensor(cu, dtype=torch.int32), 4, torch.device("cuda", 0))
    with pytest.raises(ValueError, match="int32 or int64"):
        _offsets(torch.tensor([0.0, 4.0]), 4, torch.device("cuda", 0))


@pytest.mark.parametrize("scale", [0.0, -1.0, float("nan"), float("inf")])
def test_bad_scale(scale):
    from hmx.ops.attention import _scale
    with pytest.raises(ValueError, match="positive"):
        _scale(scale, 64)


def test_append_refusals():
    k = torch.zeros(5, 2, 64, dtype=BF)
    kc, vc = _cache()
    slots = torch.arange(5)
    cs, pos = torch.zeros(9, 64), torch.arange(5)
    call = lambda **kw: hmx.append_paged_kv(**{**dict(k=k, v=k, k_cache=kc, v_cache=vc, slot_mapping=slots), **kw})
    with pytest.raises(RuntimeError, match="GPU"):
        call()
    for kw in (dict(v=k[:4]), dict(slot_mapping=slots[:4]), dict(slot_mapping=slots.float()),
               dict(cos_sin=cs), dict(positions=pos), dict(cos_sin=cs[:, :24], positions=pos),
               dict(cos_sin=torch.zeros(9, 128), positions=pos), dict(cos_sin=cs, positions=pos[:2]),
               dict(k_cache=kc[:, :, :1]), dict(v_cache=vc[:2]), dict(q=torch.zeros(4, 4, 64, dtype=BF)),
               dict(q_out=k), dict(k_cache=kc.half(), v_cache=vc.half()),
               dict(k_cache=kc[..., ::1].transpose(2, 3).contiguous().transpose(2, 3))):
        with pytest.raises(ValueError):
            call(**kw)
    with pytest.raises(NotImplementedError):
        call(k=k.float(), v=k.float())


def test_paged_refusals():
    kc, vc = _cache()
    table, lens = torch.zeros(2, 3, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    q = torch.zeros(2, 4, 64, dtype=BF)
    cu = torch.tensor([0, 1, 2], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU"):
        hmx.paged_attention_decode(q, kc, vc, table, lens)
    with pytest.raises(RuntimeError, match="GPU"):
        hmx.paged_causal_attention(q, kc, vc, table, lens, cu)
    for kw in (dict(block_table=table.long()), dict(seq_lens=lens.long()), dict(seq_lens=lens[:1]),
               dict(block_table=table[:1]), dict(q=q[:, :3]), dict(scale=0.0), dict(q=q[0]),
               dict(out=q[:, :2]), dict(out=q.half()), dict(k_cache=kc[:, :8]),
               dict(block_table=table.t().contiguous().t())):
        args = {**dict(q=q, k_cache=kc, v_cache=vc, block_table=table, seq_lens=lens), **kw}
        with pytest.raises(ValueError):
            hmx.paged_attention_decode(**args)
        with pytest.raises(ValueError):
            hmx.paged_causal_attention(cu_seqlens=cu, **args)


def test_c_entry_points_check_before_launching():
    """Sizes, types, strides and workspaces are refused by the library itself."""
    kv = _lib.PagedKV(0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 4, 3, 16)
    p = ctypes.pointer(kv)
    dec = lambda N=1, H=4, HKV=2, D=64, dt=1, scale=1.0: _lib.call(
        "hmx_paged_attention_decode", None, 0, 0, dt, None, 0, 0, p, N, H, HKV, D, scale, None, 0, None)
    with pytest.raises(NotImplementedError, match="head size 96"):
        dec(D=96)
    with pytest.raises(NotImplementedError, match="dtype"):
        dec(dt=0)
    with pytest.raises(ValueError, match="H=3"):
        dec(H=3)
    with pytest.raises(ValueError, match="positive"):
        dec(scale=0.0)
    with pytest.raises(ValueError, match="null pointer"):
        dec()
    dec(N=0)
    with pytest.raises(ValueError, match="is not N"):
        _lib.call("hmx_causal_attention", None, 0, 0, None, 0, 0, None, 0, 0, 1, None, 0, 0, None, None,
                  2, 7, 4, 2, 64, 1.0, 1, None, 0, None)
    with pytest.raises(ValueError, match="null pointer"):
        _lib.call("hmx_causal_attention", None, 0, 0, None, 0, 0, None, 0, 0, 1, None, 0, 0, None, None,
                  1, 7, 4, 2, 64, 1.0, 1, None, 0, None)
    with pytest.raises(NotImplementedError, match="bf16 only"):
        _lib.call("hmx_causal_attention_bwd", *([None, 0, 0] * 3), 2, *([None, 0, 0] * 2), None, None, 1, 7,
                  4, 2, 64, 1.0, *([None, 0, 0] * 3), None, None)
    with pytest.raises(NotImplementedError, match="rotary_dim"):
        _lib.call("hmx_append_paged_kv", None, 0, 0, None, 0, 0, None, 0, 0, 1, None, 0, 0, p, None, 1,
                  None, 0, None, 0, 0, 0, 24, 0, 5, 4, 2, 64, None)


def test_oracle_gradients_against_differences():
    """causal_grads (formulas) against central differences of causal (definition)."""
    gen = torch.Generator().manual_seed(0)
    T, H, HKV, D = 9, 4, 2, 5
    bounds = [(0, 4), (4, 4), (5, 9)]
    xs = [torch.randn(T, n, D, generator=gen, dtype=torch.float64) for n in (H, HKV, HKV)]
    do = torch.randn(T, H, D, generator=gen, dtype=torch.float64)
    (o, *grads), _ = ref.causal_grads(*xs, 0.4, bounds, do)
    assert (o - ref.causal(*xs, 0.4, bounds)[0]).abs().max() < 1e-13
    loss = lambda ys: (ref.causal(*ys, 0.4, bounds)[0] * do).sum()
    for i in range(3):
        u = torch.randn(xs[i].shape, generator=gen, dtype=torch.float64)
        hi, lo = ([x + s * 1e-5 * u if j == i else x for j, x in enumerate(xs)] for s in (1, -1))
        diff = (loss(hi) - loss(lo)) / 2e-5
        assert abs(diff - (grads[i] * u).sum()) < 1e-8 * (1 + abs(diff))


def test_oracle_rotation_and_rows_by_hand():
    x = torch.tensor([[[1.0, 2.0, 3.0, 4.0, 5.0]]])
    cs = torch.tensor([[0.0, 1.0, 1.0, 0.0]])                    # turns pair 0 by a quarter, pair 1 not
    assert ref.rotate(x, cs, torch.tensor([0]), False)[0, 0].tolist() == [-3.0, 2.0, 1.0, 4.0, 5.0]
    assert ref.rotate(x, cs, torch.tensor([0]), True)[0, 0].tolist() == [-2.0, 1.0, 3.0, 4.0, 5.0]
    q = torch.zeros(3, 1, 2)
    k = torch.zeros(2, 1, 2)
    v = torch.tensor([[[1.0, 3.0]], [[3.0, float("inf")]]])
    o, a = ref.rows(q, k, v, 1.0, -1)                            # row 0 has no key, row 2 both
    assert o[0].tolist() == [[0.0, 0.0]] and o[1].tolist() == [[1.0, 3.0]]
    assert o[2, 0, 0] == 2.0 and o[2, 0, 1] == float("inf")


def test_registered_with_fakes_and_mutations():
    import hmx.library  # noqa: F401
    m = torch.device("meta")
    q, k = torch.empty(1, 9, 4, 64, dtype=BF, device=m), torch.empty(1, 9, 2, 64, dtype=BF, device=m)
    o, lse = torch.ops.hmx.causal_attention(q, k, k, None, None)
    assert o.shape == q.shape and o.dtype == BF and lse.shape == (9, 4) and lse.dtype == torch.float32
    g = torch.ops.hmx.causal_attention_bwd(q, k, k, o, lse, o, None, None)
    assert [x.shape for x in g] == [q.shape, k.shape, k.shape]
    kc = torch.empty(3, 16, 2, 64, dtype=BF, device=m)
    tab, n = torch.empty(9, 2, dtype=torch.int32, device=m), torch.empty(9, dtype=torch.int32, device=m)
    assert torch.ops.hmx.paged_attention_decode(q[0], kc, kc, tab, n, None).shape == (9, 4, 64)
    assert torch.ops.hmx.paged_causal_attention(q[0], kc, kc, tab, n, n, None).shape == (9, 4, 64)
    assert torch.ops.hmx.append_paged_kv(k[0], k[0], kc, kc.clone(), n, q[0], None, None, False).shape == (9, 4, 64)
    w = {a.name for a in torch.ops.hmx.append_paged_kv.default._schema.arguments
         if a.alias_info is not None and a.alias_info.is_write}
    assert w == {"k_cache", "v_cache"}


def test_out_with_rows_on_one_place_is_refused():
    from hmx.ops.attention import _out
    q = torch.zeros(1, 4, 2, 64, dtype=BF)
    assert _out(torch.zeros(1, 4, 4, 64, dtype=BF)[:, :, 1:3], q) is not None
    for bad in (torch.zeros(1, 1, 2, 64, dtype=BF).expand(1, 4, 2, 64),
                torch.zeros(1, 4, 1, 64, dtype=BF).expand(1, 4, 2, 64)):
        with pytest.raises(ValueError, match="place of its own"):
            _out(bad, q)


def test_registered_backward_refuses_other_shapes():
    import hmx.library  # noqa: F401
    q, k, v = _qkv()
    lse = torch.zeros(4, 4)
    bwd = lambda o=q, lse=lse, do=q: torch.ops.hmx.causal_attention_bwd(q, k, v, o, lse, do, None, None)
    with pytest.raises(ValueError, match="o .* must be q's"):
        bwd(o=q[:, :3])
    with pytest.raises(ValueError, match="do .* must be q's"):
        bwd(do=q.float())
    for bad in (lse[:3], lse.double(), torch.zeros(4, 8)[:, ::2]):
        with pytest.raises(ValueError, match="lse"):
            bwd(lse=bad)
    with pytest.raises(RuntimeError, match="GPU"):
        bwd()


def test_short_workspaces_are_refused():
    """Few rows with many keys need a workspace; too small a one launches nothing."""
    n = _lib.load().hmx_causal_attention_workspace_bytes(1, 2048, 8, 2, 128, 0)
    assert n > 0 and _lib.load().hmx_causal_attention_workspace_bytes(1, 197, 8, 2, 128, 0) == 0
    for ws, size in ((None, n), (256, n - 1)):
        with pytest.raises(ValueError, match="too small"):
            _lib.call("hmx_causal_attention", 256, 1024, 128, 256, 256, 128, 256, 256, 128, 1, 256, 1024, 128,
                      None, None, 1, 2048, 8, 2, 128, 1.0, 1, ws, size, None)


def test_outputs_are_written_at_their_own_strides():
    """Whatever out is accepted, its rows are addressed where they lie, far apart too; strides
    of dimensions of one, which may be anything, go as 0."""
    from hmx.ops.attention import _out, _places
    far = 1 << 25
    for shape, stride, want in (((1, 3, 2, 64), (1, far, 64, 1), (far, 64)), ((3, 2, 64), (far + 8, 64, 1), (far + 8, 64)),
                                ((2, 3, 2, 64), (3 * far, far, 128, 1), (far, 128)), ((2, 1, 2, 64), (far, 5, 64, 1), (far, 64)),
                                ((4, 2, 64), (64, 256, 1), (64, 256)), ((1, 1, 1, 64), (3, 5, 7, 1), (0, 0)),
                                ((2, 3, 1, 64), (192, 64, 7, 1), (64, 0)), ((1, 4, 64), (9, 64, 1), (0, 64))):
        out = torch.empty_strided(shape, stride, dtype=BF, device="meta")
        assert _out(out, torch.empty(shape, dtype=BF, device="meta")) is out
        assert _places(out) == want


def test_host_offsets_of_later_sequences(monkeypatch):
    """The paged form takes a slice of a batch's host offsets, whose first need not be 0."""
    from hmx.ops import attention
    seen = []
    monkeypatch.setattr(torch.Tensor, "pin_memory", lambda t: seen.append(t.tolist()) or t)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    dev = torch.device("cpu")
    for cs in ([3, 5, 9], [0, 9], [9], [4, 4, 4], [0, 0, 2]):
        for dt in (torch.int32, torch.int64):
            got = attention._offsets(torch.tensor(cs, dtype=dt), 9, dev, any_first=True)
            assert got.dtype == torch.int32 and got.tolist() == cs == seen[-1]
    for cs in ([-1, 4], [3, 10], [3, 5, 4], [10]):
        with pytest.raises(ValueError, match="cu_seqlens"):
            attention._offsets(torch.tensor(cs), 9, dev, any_first=True)


@pytest.mark.parametrize("rope", [True, False])
def test_forward_core_of_no_tokens(monkeypatch, rope):
    """A step of no tokens hands empty tensors to the append and runs no attention."""
    import hmx.serving as serving
    seen = []
    monkeypatch.setattr(serving.ops, "append_paged_kv", lambda k, v, *a, q=None, **kw: seen.append((k, v, q)) or q)
    lay = SimpleNamespace(num_heads=4, num_kv_heads=2, head_dim=64, tp_size=1,
                          rotary_emb=SimpleNamespace(cos_sin_cache=torch.zeros(9, 64), is_neox_style=True) if rope else None)
    none = torch.zeros(0, dtype=torch.int32)
    md = SimpleNamespace(num_actual_tokens=0, num_decodes=0, num_decode_tokens=0, num_prefills=0, query_start_loc=none,
                         seq_lens=none, block_table=none.view(0, 3), slot_mapping=none)
    for tokens in (0, 3):
        out = torch.full((tokens, 4, 64), 5.0, dtype=BF)
        serving.attention_forward_core(lay, torch.zeros(tokens, 8 * 64, dtype=BF), none, out, md, *_cache())
        assert (out == 5).all()
    assert [tuple(x.shape) for x in seen[0][:2]] == [(0, 2, 64)] * 2 and len(seen) == 2
    assert not rope or seen[0][2].shape == (0, 4, 64)


def test_forward_core_heads_of_a_rank(monkeypatch):
    """A rank's heads; a key/value head of its own where there are fewer than ranks; a
    projection of other sizes is refused by name."""
    import hmx.serving as serving
    seen = []
    monkeypatch.setattr(serving.ops, "append_paged_kv", lambda k, v, *a, **kw: seen.append((k, v)))
    none = torch.zeros(0, dtype=torch.int32)
    md = SimpleNamespace(num_actual_tokens=0, num_decodes=0, num_decode_tokens=0, num_prefills=0, query_start_loc=none,
                         seq_lens=none, block_table=none.view(0, 3), slot_mapping=none)
    for heads, kv, tp, H, HKV in ((8, 4, 1, 8, 4), (8, 4, 2, 4, 2), (16, 2, 4, 4, 1), (8, 1, 8, 1, 1)):
        lay = SimpleNamespace(num_heads=heads, num_kv_heads=kv, head_dim=64, tp_size=tp)
        call = lambda width: serving.attention_forward_core(lay, torch.zeros(3, width, dtype=BF), None,
                                                            torch.zeros(3, H, 64, dtype=BF), md, *_cache(HKV=HKV))
        call((H + 2 * HKV) * 64)
        assert [tuple(x.shape) for x in seen[-1]] == [(0, HKV, 64)] * 2
        with pytest.raises(ValueError, match="key/value heads"):
            call((H + 2 * HKV + 1) * 64)


def test_results_without_a_backward_say_so():
    """A result that no backward reaches keeps its place in the graph, and raises there; it is
    the op's own tensor otherwise, and may be changed in place."""
    from hmx.ops.attention import _forward_only
    x, y, o = torch.ones(3, requires_grad=True), torch.ones(3), torch.ones(3)
    assert _forward_only("op", o, None, y, None) is o and _forward_only("op", o, o, x, y) is o
    with torch.no_grad():
        assert _forward_only("op", o, None, x) is o
    got = _forward_only("op", o, None, y, None, x)
    assert got.requires_grad and got.data_ptr() == o.data_ptr()
    got.mul_(2)
    with pytest.raises(NotImplementedError, match="op: no backward"):
        got.sum().backward()


def test_tangents_are_refused():
    import torch.autograd.forward_ad as fwd
    (q, k, v), (kc, vc) = _qkv(T=2), _cache()
    table, lens = torch.zeros(2, 3, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))
        for run in (lambda: hmx.causal_attention(dual(q), k, v), lambda: hmx.causal_attention(q, k, dual(v)),
                    lambda: hmx.append_paged_kv(dual(k[0]), v[0], kc, vc, lens),
                    lambda: hmx.append_paged_kv(k[0], v[0], kc, vc, lens, q=dual(q[0])),
                    lambda: hmx.paged_attention_decode(dual(q[0]), kc, vc, table, lens),
                    lambda: hmx.paged_causal_attention(q[0], kc, dual(vc), table, lens, torch.tensor([0, 1, 2]))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                run()
        with pytest.raises(RuntimeError, match="GPU"):
            hmx.causal_attention(q, k, v)


def test_an_older_library_is_refused_by_name(tmp_path):
    """A library without an entry point of the binding names it and how to build."""
    import subprocess
    src, lib = tmp_path / "old.c", tmp_path / "old.so"
    kept = [n for n in _lib.SIGNATURES if "attention" not in n and "paged" not in n]
    src.write_text("".join(f"int {n}(void) {{ return 13; }}\n" for n in kept))
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(lib), str(src)], check=True)
    with pytest.raises(_lib.HmxLibraryMissing, match="no hmx_append_paged_kv.*build"):
        _lib.load(lib)
    assert _lib.load() is _lib.load()


def test_inputs_far_apart_are_copied():
    """Rows 2^25 elements or more apart, which the kernels' offsets do not span, are copied,
    a batch's single tokens like a sequence's."""
    from hmx.ops.attention import _rows
    far = 1 << 25
    for shape, stride in (((1, 3, 2, 64), (1, far, 64, 1)), ((2, 1, 2, 64), (far, 8, 64, 1)), ((3, 2, 64), (far, 64, 1))):
        t = torch.empty_strided(shape, stride, dtype=BF, device="meta")
        got, ts, hs = _rows(t)
        assert got is not t and got.is_contiguous() and (ts, hs) == (128, 64)
    near = torch.empty_strided((2, 1, 2, 64), (far - 8, 8, 64, 1), dtype=BF, device="meta")
    assert _rows(near) == (near, far - 8, 64)


def test_appending_to_rows_on_one_place_is_refused():
    """Caches whose pages, tokens or heads share memory may be read, not written; strides of
    dimensions of one do not matter."""
    k, slots = torch.zeros(5, 2, 64, dtype=BF), torch.arange(5)
    kc, vc = _cache()
    one = lambda *shape: torch.zeros(*shape, dtype=BF).expand(3, 16, 2, 64)
    for bad in (one(1, 16, 2, 64), one(3, 1, 2, 64), one(3, 16, 1, 64)):
        for caches in ((bad, vc), (kc, bad)):
            with pytest.raises(ValueError, match="place of their own"):
                hmx.append_paged_kv(k, k, *caches, slots)
        with pytest.raises(RuntimeError, match="GPU"):
            hmx.paged_attention_decode(k, bad, bad, torch.zeros(5, 3, dtype=torch.int32), torch.ones(5, dtype=torch.int32))
    page = torch.empty_strided((1, 16, 2, 64), (0, 128, 64, 1), dtype=BF)
    with pytest.raises(RuntimeError, match="GPU"):
        hmx.append_paged_kv(k, k, page, page.clone(), slots)
