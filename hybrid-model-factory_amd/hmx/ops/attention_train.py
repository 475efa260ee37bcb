"""Causal attention with its backward (hmx.CausalAttention).

The forward of ops/attention.py keeps, beside its inputs and output, one fp32 number a row
(the log of its sum of exponentials); the backward (csrc/attn_backward.hip) forms the
probabilities from it again.
"""
from __future__ import annotations

import torch

from .. import _lib
from .attention import _elsewhere, _offsets, _rows, _scale, attention_forward, check_qkv


class CausalAttention(torch.autograd.Function):
    """causal_attention with a backward: the gradients of q, k and v (bf16), k's and v's
    summed over the heads that share them.  Rows of no sequence have a gradient of 0.  They
    are sums in a fixed order: the same inputs give the same bits.  Gradients are defined
    for finite inputs; a value that is not finite may reach rows that do not attend it."""

    @staticmethod
    def forward(ctx, q, k, v, scale, cu_seqlens):
        check_qkv("causal_attention", q, k, v, cu_seqlens)
        if q.dtype != torch.bfloat16:
            raise NotImplementedError(f"causal_attention: a gradient needs bf16, got {q.dtype}")
        o, lse, cu = attention_forward(q, k, v, scale, cu_seqlens, None, True)
        ctx.save_for_backward(q, k, v, o, lse, cu)
        ctx.scale = _scale(scale, q.shape[-1])
        return o

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do):
        q, k, v, o, lse, cu = ctx.saved_tensors
        return (*attention_backward(q, k, v, o, lse, cu, do, ctx.scale), None, None)


def attention_backward(q, k, v, o, lse, cu_seqlens, do, scale):
    """(dq, dk, dv) of causal_attention from its inputs, output, row statistics and the
    output's gradient."""
    if q.dtype != torch.bfloat16:
        raise NotImplementedError(f"causal_attention: a gradient needs bf16, got {q.dtype}")
    if _elsewhere(q):
        with torch.cuda.device(q.device):
            return attention_backward(q, k, v, o, lse, cu_seqlens, do, scale)
    scale = _scale(scale, q.shape[-1])
    cu = None if cu_seqlens is None else _offsets(cu_seqlens, q.shape[1], q.device)
    B, T, H, D = q.shape
    dq, dk, dv = (torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in (q, k, v))
    delta = torch.empty_like(lse)
    rows = [_rows(x) for x in (q, k, v, o, do.to(torch.bfloat16))]     # held until the launch
    ins = [y for x, ts, hs in rows for y in (x.data_ptr(), ts, hs)]
    grads = [y for x in (dq, dk, dv) for y in (x.data_ptr(), *_rows(x)[1:])]
    _lib.call("hmx_causal_attention_bwd", *ins[:9], _lib.HMX_BF16, *ins[9:], lse.data_ptr(),
              _lib.ptr(cu), B if cu is None else cu.shape[0] - 1, B * T, H, k.shape[2], D, scale,
              *grads, delta.data_ptr(), _lib.stream_of(q))
    return dq, dk, dv
