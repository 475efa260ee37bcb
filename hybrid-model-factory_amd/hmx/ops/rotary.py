"""Rotary positions of q and k by frequencies, for prompts and training (differentiable), and
the table that append_paged_kv reads from the same frequencies.

- ``rotary_frequencies``  the frequencies of a head, plain or scaled for longer contexts
- ``rotary_embedding``    q and k rotated by their positions
- ``rotary_table``        cosines and sines of the first positions, append_paged_kv's cos_sin
"""
from __future__ import annotations

import math

import torch

from .. import _lib
from .attention import _HEAD_SIZES, _aligned, _elsewhere, _grad_of, _refuse_tangents, _same_device, written

_SCALINGS = {"default": set(), "linear": {"factor"}, "ntk": {"factor"},
             "yarn": {"factor", "original_max_position_embeddings", "beta_fast", "beta_slow", "attention_factor"}}


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: dict | None = None,
                       device: torch.device | str = "cuda") -> tuple[torch.Tensor, float]:
    """(inv_freq [rotary_dim / 2] fp64, factor): pair i turns by position * inv_freq[i], and the
    rotation is multiplied by factor.

    Without ``scaling`` inv_freq[i] = base ** (-2 i / rotary_dim) and factor 1.  ``scaling`` is
    a model configuration's entry, with "rope_type" (or "type"):

    - "default": as without it;
    - "linear": all frequencies over "factor" s;
    - "ntk": base * s ** (rotary_dim / (rotary_dim - 2)) in the place of base;
    - "yarn": pairs that turn at least "beta_fast" (32) times within
      "original_max_position_embeddings" positions keep their frequency, those that turn less
      than "beta_slow" (1) times have it over s, the others a mix, linear in i between the two
      (rounded outwards to whole i); factor is "attention_factor", by default 0.1 ln s + 1.

    Others, and entries that a type does not have, are refused."""
    if rotary_dim < 4 or rotary_dim % 2 or not base > 1.0 or not math.isfinite(base):
        raise ValueError(f"rotary_frequencies: an even rotary_dim from 4 on and base > 1, got {rotary_dim} and {base}")
    cfg = {k: v for k, v in (scaling or {}).items() if v is not None}
    kind = cfg.pop("rope_type", cfg.get("type", "default"))
    cfg.pop("type", None)
    if kind not in _SCALINGS:
        raise NotImplementedError(f"rotary_frequencies: rope_type {kind!r} not in {sorted(_SCALINGS)}")
    if set(cfg) - _SCALINGS[kind]:
        raise ValueError(f"rotary_frequencies: {kind} has no {sorted(set(cfg) - _SCALINGS[kind])}")
    s = 1.0
    if kind != "default":
        s = float(cfg.get("factor", math.nan))
        if not 1.0 <= s < math.inf:
            raise ValueError(f"rotary_frequencies: {kind} needs a factor >= 1, got {cfg.get('factor')}")
    if kind == "ntk":
        base = base * s ** (rotary_dim / (rotary_dim - 2))
    inv = [base ** (-2 * i / rotary_dim) for i in range(rotary_dim // 2)]
    factor = 1.0
    if kind == "linear":
        inv = [f / s for f in inv]
    elif kind == "yarn":
        start = cfg.get("original_max_position_embeddings")
        fast, slow = float(cfg.get("beta_fast", 32.0)), float(cfg.get("beta_slow", 1.0))
        if start is None or not start > 0 or not fast >= slow > 0:
            raise ValueError("rotary_frequencies: yarn needs original_max_position_embeddings > 0 and "
                             f"beta_fast >= beta_slow > 0, got {start}, {fast} and {slow}")
        # the i whose pair turns n times in `start` positions
        at = lambda n: rotary_dim * math.log(start / (n * 2 * math.pi)) / (2 * math.log(base))
        low, high = max(math.floor(at(fast)), 0), min(math.ceil(at(slow)), rotary_dim - 1)
        for i, f in enumerate(inv):
            # (a ramp that ends before pair 0 has no pair in it)
            mix = 1.0 if at(slow) < 0 else min(max((i - low) / max(high - low, 1e-3), 0.0), 1.0)
            inv[i] = f / s * mix + f * (1 - mix)
        factor = float(cfg.get("attention_factor", 0.1 * math.log(s) + 1))
    return torch.tensor(inv, dtype=torch.float64, device=device), factor


def _check_freq(what: str, inv_freq: torch.Tensor, factor: float) -> None:
    if inv_freq.dim() != 1 or inv_freq.dtype not in (torch.float32, torch.float64):
        raise ValueError(f"{what}: inv_freq [rotary_dim / 2] fp32 or fp64, got {tuple(inv_freq.shape)} {inv_freq.dtype}")
    if not math.isfinite(factor):
        raise ValueError(f"{what}: factor must be finite, got {factor}")


def rotary_table(inv_freq: torch.Tensor, positions: int, factor: float = 1.0) -> torch.Tensor:
    """[positions, rotary_dim] fp32: factor times the cosines, then the sines, of positions 0 ..
    positions - 1, which is append_paged_kv's ``cos_sin``."""
    _check_freq("rotary_table", inv_freq, factor)
    positions = int(positions)
    if positions < 0 or inv_freq.shape[0] == 0:
        raise ValueError(f"rotary_table: {positions} positions of {inv_freq.shape[0]} frequencies")
    _lib.require_gpu(inv_freq)
    with torch.cuda.device(inv_freq.device):
        inv_freq = inv_freq.contiguous()
        R = 2 * inv_freq.shape[0]
        table = torch.empty(positions, R, dtype=torch.float32, device=inv_freq.device)
        _lib.call("hmx_rotary_table", inv_freq.data_ptr(), int(inv_freq.dtype == torch.float64), float(factor),
                  positions, R, table.data_ptr(), _lib.stream_of(inv_freq))
    return table


def _strided(t: torch.Tensor | None) -> tuple[int, int, int, int]:
    """(address, batch, token and head stride) of [B, T, heads, D]; strides of dimensions of
    one, which may be anything, as 0."""
    if t is None:
        return 0, 0, 0, 0
    if t.is_contiguous():
        _, T, H, D = t.shape
        return t.data_ptr(), T * H * D, H * D, D
    return (t.data_ptr(), *(s if n > 1 else 0 for s, n in zip(t.stride()[:3], t.shape)))


def _new(t: torch.Tensor | None) -> torch.Tensor | None:
    if t is None or t.is_contiguous():
        return None if t is None else torch.empty_like(t)
    return torch.empty(t.shape, dtype=t.dtype, device=t.device)


def rotate(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, inv_freq: torch.Tensor, factor: float,
           interleaved: bool, backward: bool, q_out: torch.Tensor | None = None,
           k_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """rotary_embedding of arguments that it has checked, into q_out and k_out or new tensors;
    backward: by minus the angle."""
    if _elsewhere(q):
        with torch.cuda.device(q.device):
            return rotate(q, k, positions, inv_freq, factor, interleaved, backward, q_out, k_out)
    q_out, k_out = q_out if q_out is not None else _new(q), k_out if k_out is not None else _new(k)
    B, T, H, D = q.shape
    if q.numel() == 0:
        return q_out, k_out
    if not _aligned(q):
        q = q.clone(memory_format=torch.contiguous_format)
    if k is not None and not _aligned(k):
        k = k.clone(memory_format=torch.contiguous_format)
    inv_freq = inv_freq.contiguous()
    if T > 1 and positions.stride(-1) != 1:
        positions = positions.contiguous()
    pos_stride = positions.stride(0) if positions.dim() == 2 and positions.shape[0] > 1 else 0
    _lib.call("hmx_rotary_embedding", *_strided(q), *_strided(q_out), *_strided(k), *_strided(k_out),
              _lib.dtype_code(q), positions.data_ptr(), int(positions.dtype == torch.int64), pos_stride,
              inv_freq.data_ptr(), int(inv_freq.dtype == torch.float64), float(factor), 2 * inv_freq.shape[0],
              int(interleaved), int(backward), B, T, H, 0 if k is None else k.shape[2], D, _lib.stream_of(q))
    return q_out, k_out


class RotaryEmbedding(torch.autograd.Function):
    """rotary_embedding with its gradients: the same rotation the other way round, so they have
    gradients of their own too."""

    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, factor, interleaved, backward):
        ctx.save_for_backward(positions, inv_freq)
        ctx.set_materialize_grads(False)
        ctx.args = (factor, interleaved)
        ctx.back = backward
        return rotate(q, k, positions, inv_freq, factor, interleaved, backward)

    @staticmethod
    def backward(ctx, dq, dk):
        positions, inv_freq = ctx.saved_tensors
        # as a function of its own only where a graph of the gradients is asked for
        again = RotaryEmbedding.apply if torch.is_grad_enabled() else rotate
        needs_q, needs_k = ctx.needs_input_grad[:2]
        if dq is not None and needs_q:
            dq, dk = again(dq, dk if needs_k else None, positions, inv_freq, *ctx.args, not ctx.back)
        else:
            dq = None
            if dk is not None:
                dk = again(dk, None, positions, inv_freq, *ctx.args, not ctx.back)[0] if needs_k else None
        return dq, dk, None, None, None, None, None


def _check_out(what: str, name: str, out: torch.Tensor, like: torch.Tensor) -> None:
    if out.shape != like.shape or out.dtype != like.dtype:
        raise ValueError(f"{what}: {name} {tuple(out.shape)} {out.dtype} must be {tuple(like.shape)} {like.dtype}")
    if not _aligned(out) or any(s == 0 and n > 1 for s, n in zip(out.stride(), out.shape)):
        raise ValueError(f"{what}: {name} must have D contiguous, 16-byte aligned rows and a place of its own for "
                         "every row")


def rotary_embedding(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, inv_freq: torch.Tensor, *,
                     factor: float = 1.0, interleaved: bool = False, q_out: torch.Tensor | None = None,
                     k_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """q and k (or None) rotated by their positions: the first R = 2 len(inv_freq) elements of
    every head turn by positions * inv_freq, in pairs (i, i + R / 2), or (2i, 2i + 1) with
    ``interleaved``, and are multiplied by ``factor``; the others stay.

    q [B, T, H, D] and k [B, T, HKV, D] with ``positions`` [B, T], [1, T] or [T], or q [T, H, D]
    and k [T, HKV, D] with [T]; bf16 or fp16, D 64 or 128, any strides.  ``positions`` int32 or
    int64, any values; ``inv_freq`` fp64 or fp32 on the device (rotary_frequencies), R a
    multiple of 16 up to D.  The angle is formed in fp64.  ``q_out`` and ``k_out`` (may be q
    and k themselves, and may overlap no input otherwise) receive the results where no
    gradient is needed.  Returns both.

    Differentiable in q and k (hmx.RotaryEmbedding), not in the frequencies."""
    return turn(q, k, positions, inv_freq, factor, interleaved, False, q_out, k_out)


def turn(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, inv_freq: torch.Tensor, factor: float,
         interleaved: bool, backward: bool, q_out: torch.Tensor | None = None,
         k_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """rotary_embedding; backward: by minus the angle."""
    what = "rotary_embedding"
    _refuse_tangents(what, q, k, inv_freq)
    if q.dim() not in (3, 4) or (k is not None and (k.dim() != q.dim() or k.shape[:-2] != q.shape[:-2]
                                                    or k.shape[-1] != q.shape[-1] or k.dtype != q.dtype)):
        raise ValueError(f"{what}: q [B, T, H, D] and k [B, T, HKV, D], or without B, of one type, got "
                         f"{tuple(q.shape)} and {None if k is None else tuple(k.shape)}")
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise NotImplementedError(f"{what}: bf16 or fp16, got {q.dtype}")
    D = q.shape[-1]
    if D not in _HEAD_SIZES:
        raise NotImplementedError(f"{what}: head size {D} not in {_HEAD_SIZES}")
    if q.shape[-2] == 0 or (k is not None and k.shape[-2] == 0):
        raise ValueError(f"{what}: no heads")
    factor = float(factor)
    _check_freq(what, inv_freq, factor)
    R = 2 * inv_freq.shape[0]
    if R == 0 or R > D or R % 16:
        raise ValueError(f"{what}: {inv_freq.shape[0]} frequencies: a multiple of 8 up to {D // 2}")
    lead, at = q.shape[:-2], positions.shape
    if not (at == lead or (q.dim() == 4 and (at == lead[1:] or at == (1, lead[1])))) \
            or positions.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"{what}: positions {tuple(lead)}{', or without B,' if q.dim() == 4 else ''} int32 or int64, "
                         f"got {tuple(at)} {positions.dtype}")
    if inv_freq.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError(f"{what}: no gradient of the frequencies is implemented")
    if q_out is not None:
        _check_out(what, "q_out", q_out, q)
    if k_out is not None:
        if k is None:
            raise ValueError(f"{what}: k_out without k")
        _check_out(what, "k_out", k_out, k)
    _same_device(q, k, positions, inv_freq, q_out, k_out)
    interleaved = bool(interleaved)
    flat = q.dim() == 3
    if flat:
        q, k, q_out, k_out = (t if t is None else t.unsqueeze(0) for t in (q, k, q_out, k_out))
    outs = [t for t in (q_out, k_out) if t is not None]
    if outs and _grad_of(q, k, *outs):
        raise ValueError(f"{what}: q_out and k_out are not supported where a gradient is needed")
    if outs:
        written(*outs)
    if _grad_of(q, k):
        q, k = RotaryEmbedding.apply(q, k, positions, inv_freq, factor, interleaved, backward)
    else:
        q, k = rotate(q, k, positions, inv_freq, factor, interleaved, backward, q_out, k_out)
    return (q.squeeze(0), k if k is None else k.squeeze(0)) if flat else (q, k)
