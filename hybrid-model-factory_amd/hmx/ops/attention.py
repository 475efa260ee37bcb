"""The attention layers between a hybrid model's mixers: causal attention over whole
prompts, and over a paged key/value cache that ``append_paged_kv`` fills.

- ``causal_attention``        prompts and training sequences, packed or a batch; differentiable
- ``append_paged_kv``         position rotation of q and k, k and v stored into the cache
- ``paged_causal_attention``  several new tokens a sequence behind a cached context
- ``paged_attention_decode``  one new token a sequence

q carries H heads, k and v HKV heads that groups of H / HKV consecutive q heads share.
Head sizes 64 and 128, bf16 and fp16.  A cache is a pair of tensors
[pages, page size, HKV, D] (any strides over whole 16-byte units with D contiguous, so
both halves of one allocation pass as views); ``block_table`` [N, width] int32 lists the
pages of every sequence.  Lengths, offsets, tables and slots are read on the device only,
so a captured graph replays with other lengths.

causal_attention alone has a backward; one through another op's result raises, and what is
stored into a cache or written to ``out`` has no gradient.  There is no forward-mode
derivative: inputs with tangents are refused.
"""
from __future__ import annotations

import functools

import torch
from torch.autograd import forward_ad

from .. import _lib
from .gdn import seq_bounds

_HEAD_SIZES = (64, 128)


def _same_device(ref: torch.Tensor, *tensors: torch.Tensor | None) -> None:
    dev = ref.get_device()
    for t in tensors:
        if t is not None and t.get_device() != dev:
            _lib.require_gpu(ref, t)
            raise ValueError(f"tensors on {ref.device} and {t.device}")
    if dev < 0:
        _lib.require_gpu(ref)


def _elsewhere(t: torch.Tensor) -> bool:
    """Whether t's device is not the current one, to which launches go."""
    return t.get_device() != torch._C._cuda_getDevice()


class _NoBackward(torch.autograd.Function):
    """An op's result with its place in the graph, and a backward that says there is none."""

    @staticmethod
    def forward(ctx, result, what, *inputs):
        ctx.what = what
        return result[0]                # in a list: the result itself, not a view of an input

    @staticmethod
    def backward(ctx, *grads):
        raise NotImplementedError(f"{ctx.what}: no backward is implemented")


def _grad_of(*tensors: torch.Tensor | None) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _forward_only(what: str, result: torch.Tensor, out: torch.Tensor | None, *inputs) -> torch.Tensor:
    """The result of an op without a backward, so that one through it raises; ``out``, where
    the caller gave one, stands outside any graph."""
    return _NoBackward.apply([result], what, *inputs) if out is None and _grad_of(*inputs) else result


def _refuse_tangents(what: str, *tensors: torch.Tensor | None) -> None:
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None
                                              for t in tensors):
        raise NotImplementedError(f"{what}: no forward-mode derivative is implemented")


def _check_types(what: str, q: torch.Tensor, *others: torch.Tensor | None) -> None:
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise NotImplementedError(f"{what}: bf16 or fp16, got {q.dtype}")
    if q.shape[-1] not in _HEAD_SIZES:
        raise NotImplementedError(f"{what}: head size {q.shape[-1]} not in {_HEAD_SIZES}")
    for t in others:
        if t is not None and t.dtype != q.dtype:
            raise ValueError(f"{what}: types {q.dtype} and {t.dtype} differ")


def _aligned(t: torch.Tensor) -> bool:
    """Whether 16-byte loads reach every row of [..., heads, D] in place."""
    if t.is_contiguous():
        return t.data_ptr() % 16 == 0
    st, n = t.stride(), t.shape
    return (st[-1] == 1 and t.data_ptr() % 16 == 0
            and all(s % 8 == 0 or m == 1 for s, m in zip(st[:-1], n[:-1])))


def _rows(t: torch.Tensor) -> tuple[torch.Tensor, int, int]:
    """(t, token stride, head stride) of [tokens, heads, D], or of [B, T, heads, D] whose
    tokens lie at one stride; a contiguous copy where there is no such view."""
    if t.is_contiguous() and t.data_ptr() % 16 == 0:
        H, D = t.shape[-2:]
        return t, H * D, D
    B = t.shape[0] if t.dim() == 4 else 1
    T = t.shape[-3]
    if not _aligned(t) or (B > 1 and T > 1 and t.stride(0) != T * t.stride(1)) \
            or (B * T > 1 and t.stride(-3 if T > 1 else 0) >= 1 << 25):
        t = t.contiguous()
    ts = t.stride(-3) if T > 1 or B == 1 else t.stride(0)
    # strides of dimensions of one are never used, and may be anything
    return t, ts if B * T > 1 else 0, t.stride(-2) if t.shape[-2] > 1 else 0


def _places(t: torch.Tensor) -> tuple[int, int]:
    """(token stride, head stride) of an output that _out has looked through: its own, at any
    distance, for it is written in place and a copy may never stand for it."""
    B = t.shape[0] if t.dim() == 4 else 1
    T = t.shape[-3]
    ts = t.stride(-3) if T > 1 else t.stride(0) if B > 1 else 0
    return ts, t.stride(-2) if t.shape[-2] > 1 else 0


def _out(out: torch.Tensor | None, like: torch.Tensor) -> torch.Tensor:
    if out is None:
        return torch.empty(like.shape, dtype=like.dtype, device=like.device)
    if out.shape != like.shape or out.dtype != like.dtype:
        raise ValueError(f"out {tuple(out.shape)} {out.dtype} must be {tuple(like.shape)} {like.dtype}")
    if not _aligned(out) or (out.dim() == 4 and out.shape[0] > 1 and out.shape[1] > 1
                             and out.stride(0) != out.shape[1] * out.stride(1)):
        raise ValueError("out must have D contiguous, 16-byte aligned rows and tokens at one stride")
    if not out.is_contiguous() and any(s == 0 and m > 1 for s, m in zip(out.stride(), out.shape)):
        raise ValueError("out must have a place of its own for every row")
    return out


@functools.lru_cache(maxsize=256)
def _workspace_bytes(name: str, device: int, *sizes: int) -> int:
    """A workspace's size, which depends on the sizes and the device's compute units alone."""
    return int(getattr(_lib.load(), name)(*sizes))


def _workspace(name: str, like: torch.Tensor, *sizes: int) -> tuple[torch.Tensor | None, int]:
    n = _workspace_bytes(name, like.get_device(), *sizes)
    return (torch.empty(n, dtype=torch.uint8, device=like.device), n) if n else (None, 0)


def _scale(scale: float | None, D: int) -> float:
    scale = D ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < float("inf"):
        raise ValueError(f"scale must be positive, got {scale}")
    return scale


def _offsets(cu_seqlens: torch.Tensor, T: int, device: torch.device, any_first: bool = False) -> torch.Tensor:
    """cu_seqlens as int32 on the device.  Host offsets are checked here, and start at 0 unless
    ``any_first``; offsets on the device are never read back (the kernels clamp them into the
    tokens)."""
    if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 1:
        raise ValueError(f"cu_seqlens must be a vector of N + 1 offsets, got {tuple(cu_seqlens.shape)}")
    if cu_seqlens.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"cu_seqlens must be int32 or int64, got {cu_seqlens.dtype}")
    if cu_seqlens.is_cuda:
        if cu_seqlens.device != device:
            raise ValueError(f"tensors on {device} and {cu_seqlens.device}")
        return cu_seqlens if cu_seqlens.dtype == torch.int32 and cu_seqlens.is_contiguous() \
            else cu_seqlens.to(torch.int32).contiguous()
    if any_first:
        cs = cu_seqlens.tolist()
        if cs[0] < 0 or cs[-1] > T or any(b < a for a, b in zip(cs, cs[1:])):
            raise ValueError(f"cu_seqlens must be non-decreasing from >= 0 to <= {T}: {cs}")
    else:
        seq_bounds(cu_seqlens, 1, T)
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("cu_seqlens must be on the device where a graph is captured")
    return cu_seqlens.to(torch.int32).pin_memory().to(device, non_blocking=True)


def causal_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float | None = None,
                     cu_seqlens: torch.Tensor | None = None, *,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(scale q k^T) v of every token over itself and the tokens before it.

    q [B, T, H, D], k and v [B, T, HKV, D]; with ``cu_seqlens`` (N + 1 offsets into the
    tokens, B = 1; where they are on the host, the first is 0) each of the N packed sequences
    by itself.  ``scale`` (default D ** -0.5) must be positive.  Returns [B, T, H, D] in q's
    type; rows of no sequence are 0, or left as they were in ``out`` (which may not overlap an
    input).  A value that is not finite reaches the rows that attend it and no others; a row
    whose scores are all minus infinity counts as one without keys, 0.

    Differentiable in q, k and v for bf16 (hmx.CausalAttention)."""
    _refuse_tangents("causal_attention", q, k, v)
    if _grad_of(q, k, v):
        if out is not None:
            raise ValueError("out is not supported where a gradient is needed")
        from .attention_train import CausalAttention
        return CausalAttention.apply(q, k, v, scale, cu_seqlens)
    return attention_forward(q, k, v, scale, cu_seqlens, out, False)[0]


def check_qkv(what: str, q, k, v, cu_seqlens) -> None:
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or k.shape[:2] != q.shape[:2] \
            or k.shape[-1] != q.shape[-1]:
        raise ValueError(f"{what}: q [B, T, H, D], k and v [B, T, HKV, D], got {tuple(q.shape)}, "
                         f"{tuple(k.shape)}, {tuple(v.shape)}")
    if k.shape[2] == 0 or q.shape[2] == 0 or q.shape[2] % k.shape[2] != 0:
        raise ValueError(f"{what}: {q.shape[2]} heads cannot share {k.shape[2]}")
    if cu_seqlens is not None and q.shape[0] != 1:
        raise ValueError(f"Batch size expected to be 1 with cu_seqlens, got {q.shape[0]}")
    _check_types(what, q, k, v)
    _same_device(q, k, v)


def attention_forward(q, k, v, scale, cu_seqlens, out, want_lse):
    """(o, base-2 log-sum-exp of the scaled scores [B * T, H] fp32 or None, device offsets or None)."""
    check_qkv("causal_attention", q, k, v, cu_seqlens)
    if _elsewhere(q):
        with torch.cuda.device(q.device):
            return attention_forward(q, k, v, scale, cu_seqlens, out, want_lse)
    B, T, H, D = q.shape
    scale = _scale(scale, D)
    o = _out(out, q)
    if out is not None:
        _same_device(q, o)
    cu = None if cu_seqlens is None else _offsets(cu_seqlens, T, q.device)
    N = B if cu is None else cu.shape[0] - 1
    lse = torch.empty(B * T, H, dtype=torch.float32, device=q.device) if want_lse else None
    q, qts, qhs = _rows(q)
    k, kts, khs = _rows(k)
    v, vts, vhs = _rows(v)
    ots, ohs = _places(o)
    ws, ws_bytes = _workspace("hmx_causal_attention_workspace_bytes", q, N, B * T, H, k.shape[2], D,
                              int(cu is not None))
    _lib.call("hmx_causal_attention", q.data_ptr(), qts, qhs, k.data_ptr(), kts, khs,
              v.data_ptr(), vts, vhs, _lib.dtype_code(q), o.data_ptr(), ots, ohs,
              _lib.ptr(lse), _lib.ptr(cu), N, B * T, H, k.shape[2], D, scale,
              int(out is None), _lib.ptr(ws), ws_bytes, _lib.stream_of(q))
    return o, lse, cu


def _cache(what: str, q: torch.Tensor, k_cache, v_cache, HKV: int | None = None) -> None:
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape or k_cache.shape[-1] != q.shape[-1] \
            or k_cache.shape[1] == 0 or k_cache.shape[2] == 0 \
            or (HKV is not None and k_cache.shape[2] != HKV):
        raise ValueError(f"{what}: caches [pages, page size, HKV, D], got {tuple(k_cache.shape)} and "
                         f"{tuple(v_cache.shape)} for heads of {q.shape[-1]}")
    _check_types(what, q, k_cache, v_cache)
    # never copied: a cache is written in place and as large as memory
    if not (_aligned(k_cache) and _aligned(v_cache)):
        raise ValueError(f"{what}: caches need D contiguous and strides and bases of whole 16-byte units")


def _table(what: str, block_table: torch.Tensor, seq_lens: torch.Tensor, N: int) -> None:
    for name, t in (("block_table", block_table), ("seq_lens", seq_lens)):
        if t.dtype != torch.int32:
            raise ValueError(f"{what}: {name} must be int32, got {t.dtype}")
    if block_table.dim() != 2 or block_table.shape[0] != N or tuple(seq_lens.shape) != (N,) \
            or not seq_lens.is_contiguous() or (block_table.shape[1] > 1 and block_table.stride(1) != 1):
        raise ValueError(f"{what}: block_table [{N}, width] with contiguous rows and seq_lens [{N}], got "
                         f"{tuple(block_table.shape)} and {tuple(seq_lens.shape)}")


def append_paged_kv(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    slot_mapping: torch.Tensor, *, q: torch.Tensor | None = None,
                    positions: torch.Tensor | None = None, cos_sin: torch.Tensor | None = None,
                    interleaved: bool = False, q_out: torch.Tensor | None = None) -> torch.Tensor | None:
    """Stores k and v [T, HKV, D] into the cache, k rotated, and returns q [T, H, D] rotated.

    ``slot_mapping`` [T] (int32 or int64): page * page size + place in the page; a token
    whose slot is negative or past the cache is padding and stores nothing.  Two tokens
    with one slot leave a mix of the two there.  With ``cos_sin`` [max position, R] (fp32,
    bf16 or fp16; R a multiple of 16 up to D: R / 2 cosines, then R / 2 sines) and
    ``positions`` [T] the first R elements of every q and k head turn by their position's
    angles, in pairs (i, i + R / 2), or (2i, 2i + 1) with ``interleaved``; a position
    outside the table gives NaN.  Without them k is stored and q returned as they are.
    Rows of the caches may not share memory.  ``q_out`` (may be q itself) receives the rotated
    q.  Returns it, or None without q."""
    what = "append_paged_kv"
    _refuse_tangents(what, q, k, v)
    if k.dim() != 3 or k.shape != v.shape:
        raise ValueError(f"{what}: k and v [T, HKV, D], got {tuple(k.shape)} and {tuple(v.shape)}")
    T, HKV, D = k.shape
    _check_types(what, k, v, q)
    _cache(what, k, k_cache, v_cache, HKV)
    if any(0 in c.stride() and any(s == 0 and m > 1 for s, m in zip(c.stride(), c.shape))
           for c in (k_cache, v_cache)):
        raise ValueError(f"{what}: caches must have a place of their own for every row")
    if (cos_sin is None) != (positions is None):
        raise ValueError(f"{what}: cos_sin and positions go together")
    for name, t in (("slot_mapping", slot_mapping), ("positions", positions)):
        if t is not None and (tuple(t.shape) != (T,) or t.dtype not in (torch.int32, torch.int64)):
            raise ValueError(f"{what}: {name} must be [{T}] int32 or int64, got {tuple(t.shape)} {t.dtype}")
    if q is None and q_out is not None:
        raise ValueError(f"{what}: q_out without q")
    if q is not None and (q.dim() != 3 or q.shape[0] != T or q.shape[2] != D):
        raise ValueError(f"{what}: q [{T}, H, {D}], got {tuple(q.shape)}")
    R = 0
    if cos_sin is not None:
        R = cos_sin.shape[-1] if cos_sin.dim() == 2 else 0
        if cos_sin.dim() != 2 or cos_sin.shape[0] == 0 or R == 0 or R > D or R % 16 != 0:
            raise ValueError(f"{what}: cos_sin [positions, R] with R a multiple of 16 up to {D}, got "
                             f"{tuple(cos_sin.shape)}")
        _lib.dtype_code(cos_sin)
        if cos_sin.stride(1) != 1 or cos_sin.stride(0) % 8 or cos_sin.data_ptr() % 16:
            cos_sin = cos_sin.contiguous()
    H = 0 if q is None else q.shape[1]
    _same_device(k, v, k_cache, v_cache, slot_mapping, q, positions, cos_sin, q_out)
    if _elsewhere(k):
        with torch.cuda.device(k.device):
            return append_paged_kv(k, v, k_cache, v_cache, slot_mapping, q=q, positions=positions,
                                   cos_sin=cos_sin, interleaved=interleaved, q_out=q_out)
    ret = None
    ins = (q, k, v)
    if q is not None:
        if cos_sin is None and q_out is None:
            ret, q = q, None                    # nothing to do for q
        else:
            ret = _out(q_out, q)
    if T == 0:
        return ret if q is None else _forward_only(what, ret, q_out, *ins)
    k, kts, khs = _rows(k)
    v, vts, vhs = _rows(v)
    qts = qhs = ots = ohs = 0
    if q is not None:
        q, qts, qhs = _rows(q)
        ots, ohs = _places(ret)
    slot_mapping = slot_mapping.contiguous()
    cs = (None, 0, None, 0, 0, 0)
    if cos_sin is not None:
        positions = positions.contiguous()
        cs = (positions.data_ptr(), int(positions.dtype == torch.int64), cos_sin.data_ptr(),
              _lib.dtype_code(cos_sin), cos_sin.stride(0), cos_sin.shape[0])
    _lib.call("hmx_append_paged_kv", _lib.ptr(q), qts, qhs, k.data_ptr(), kts, khs,
              v.data_ptr(), vts, vhs, _lib.dtype_code(k), None if q is None else ret.data_ptr(),
              ots, ohs, _lib.paged_kv(k_cache, v_cache), slot_mapping.data_ptr(),
              int(slot_mapping.dtype == torch.int64), *cs, R, int(bool(interleaved)), T, H, HKV,
              D, _lib.stream_of(k))
    return ret if q is None else _forward_only(what, ret, q_out, *ins)


def paged_attention_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                           block_table: torch.Tensor, seq_lens: torch.Tensor,
                           scale: float | None = None, *, out: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(scale q k^T) v of one token a sequence over its keys in the cache.

    q [N, H, D]; ``seq_lens`` [N] int32: keys of each sequence, the new token's among them
    (append_paged_kv stores it first); 0 gives a row of 0, and a length past the table
    row's pages counts as all of them.  ``block_table`` [N, width] int32; a page outside
    the cache holds no keys.  A value that is not finite makes its column of its sequence's
    rows infinite or NaN.  Returns [N, H, D] in q's type (``out``, which may not overlap an
    input)."""
    what = "paged_attention_decode"
    _refuse_tangents(what, q, k_cache, v_cache)
    if q.dim() != 3:
        raise ValueError(f"{what}: q [N, H, D], got {tuple(q.shape)}")
    N, H, D = q.shape
    _cache(what, q, k_cache, v_cache)
    HKV = k_cache.shape[2]
    if H == 0 or H % HKV != 0:
        raise ValueError(f"{what}: {H} heads cannot share {HKV}")
    _table(what, block_table, seq_lens, N)
    scale = _scale(scale, D)
    o = _out(out, q)
    _same_device(q, k_cache, v_cache, block_table, seq_lens, o)
    ins = (q, k_cache, v_cache)
    if N == 0:
        return _forward_only(what, o, out, *ins)
    if _elsewhere(q):
        with torch.cuda.device(q.device):
            return paged_attention_decode(q, k_cache, v_cache, block_table, seq_lens, scale, out=out)
    q, qts, qhs = _rows(q)
    ots, ohs = _places(o)
    ws, ws_bytes = _workspace("hmx_paged_attention_decode_workspace_bytes", q, N, H, HKV, D,
                              block_table.shape[1] * k_cache.shape[1])
    _lib.call("hmx_paged_attention_decode", q.data_ptr(), qts, qhs, _lib.dtype_code(q),
              o.data_ptr(), ots, ohs, _lib.paged_kv(k_cache, v_cache, block_table, seq_lens),
              N, H, HKV, D, scale, _lib.ptr(ws), ws_bytes, _lib.stream_of(q))
    return _forward_only(what, o, out, *ins)


def paged_causal_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                           block_table: torch.Tensor, seq_lens: torch.Tensor,
                           cu_seqlens: torch.Tensor, scale: float | None = None, *,
                           out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of new tokens that are the last of their sequences in the cache:
    prompts in pieces, prompts behind a cached prefix, draft tokens.

    q [T, H, D] holds the new tokens of all N sequences, ``cu_seqlens`` [N + 1] their
    offsets (on the host or the device; the first need not be 0, so a batch's later
    sequences pass with its own offsets); ``seq_lens`` [N] int32 counts each sequence's
    keys, the new tokens' among them: token i of n attends keys 0 .. seq_len - n + i, and
    gives 0 where that is none.  Cache and table as in paged_attention_decode.  Returns
    [T, H, D] in q's type; rows of no sequence are 0, or left as they were in ``out`` (which
    may not overlap an input)."""
    what = "paged_causal_attention"
    _refuse_tangents(what, q, k_cache, v_cache)
    if q.dim() != 3:
        raise ValueError(f"{what}: q [T, H, D], got {tuple(q.shape)}")
    T, H, D = q.shape
    _cache(what, q, k_cache, v_cache)
    HKV = k_cache.shape[2]
    if H == 0 or H % HKV != 0:
        raise ValueError(f"{what}: {H} heads cannot share {HKV}")
    N = max(cu_seqlens.shape[0] - 1, 0) if cu_seqlens.dim() == 1 else 0
    _table(what, block_table, seq_lens, N)
    scale = _scale(scale, D)
    o = _out(out, q)
    _same_device(q, k_cache, v_cache, block_table, seq_lens, o)
    if _elsewhere(q):
        with torch.cuda.device(q.device):
            return paged_causal_attention(q, k_cache, v_cache, block_table, seq_lens, cu_seqlens,
                                          scale, out=out)
    cu = _offsets(cu_seqlens, T, q.device, any_first=True)
    ins = (q, k_cache, v_cache)
    if T == 0:
        return _forward_only(what, o, out, *ins)
    q, qts, qhs = _rows(q)
    ots, ohs = _places(o)
    ws, ws_bytes = _workspace("hmx_paged_causal_attention_workspace_bytes", q, N, T, H, HKV, D,
                              block_table.shape[1] * k_cache.shape[1])
    _lib.call("hmx_paged_causal_attention", q.data_ptr(), qts, qhs, _lib.dtype_code(q),
              o.data_ptr(), ots, ohs, _lib.paged_kv(k_cache, v_cache, block_table, seq_lens),
              _lib.ptr(cu), N, T, H, HKV, D, scale, int(out is None), _lib.ptr(ws), ws_bytes,
              _lib.stream_of(q))
    return _forward_only(what, o, out, *ins)
