"""Attention layers restated in float64: causal softmax attention with grouped heads and its
gradients, the paged cache, and the position rotation.  Written from the definitions, row by
row where that is clearest; runs on the CPU or a GPU."""
from __future__ import annotations

import torch

F64 = torch.float64


def rows(q, k, v, scale, first):
    """Attention of q [m, H, D] over k, v [L, HKV, D]; row i attends keys 0 .. first + i.
    Returns (o [m, H, D], a = sum_j p_j |v_j| [m, H, D]), the second for error bounds."""
    m, H, D = q.shape
    L, HKV, _ = k.shape
    q, k, v = q.to(F64), k.to(F64), v.to(F64)
    o, a = torch.zeros_like(q), torch.zeros_like(q)
    last = first + torch.arange(m, device=q.device)
    keys = torch.arange(L, device=q.device)
    for h in range(H):
        kv = h // (H // HKV)
        s = scale * (q[:, h] @ k[:, kv].T)
        s = torch.where(keys[None] <= last[:, None], s, torch.full_like(s, -torch.inf))
        mx = s.amax(-1, keepdim=True) if L else s.new_zeros(m, 1)
        w = torch.exp(s - torch.where(mx == -torch.inf, torch.zeros_like(mx), mx))
        w = w / w.sum(-1, keepdim=True).clamp(min=1e-300)
        # 0 times an infinity behind a row's last key is nothing, not NaN
        for y, x in ((o, v[:, kv]), (a, v[:, kv].abs())):
            if torch.isfinite(x).all():
                y[:, h] = w @ x
            else:
                for i in range(m):
                    n = max(0, min(L, int(last[i]) + 1))
                    y[i, h] = (w[i, :n, None] * x[:n]).sum(0)
    return o, a


def causal(q, k, v, scale, bounds):
    """Sequences [(bos, eos)] of packed q [T, H, D], k, v [T, HKV, D]; rows of none are 0."""
    o, a = torch.zeros_like(q, dtype=F64), torch.zeros_like(q, dtype=F64)
    for b, e in bounds:
        o[b:e], a[b:e] = rows(q[b:e], k[b:e], v[b:e], scale, 0)
    return o, a


def causal_grads(q, k, v, scale, bounds, do):
    """(o, dq, dk, dv) of causal() from the formulas, and for error bounds the sums of the
    magnitudes of the terms that dq, dk and dv are made of (formed from |dS| and P)."""
    q, k, v, do = (x.to(F64) for x in (q, k, v, do))
    H, HKV = q.shape[1], k.shape[1]
    o, dq, mq = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(q)
    dk, dv, mk, mv = (torch.zeros_like(k) for _ in range(4))
    for b, e in bounds:
        n = e - b
        tri = torch.ones(n, n, dtype=torch.bool, device=q.device).tril()
        for h in range(H):
            kv = h // (H // HKV)
            Q, K, V, dO = q[b:e, h], k[b:e, kv], v[b:e, kv], do[b:e, h]
            s = torch.where(tri, scale * (Q @ K.T), torch.tensor(-torch.inf, dtype=F64, device=q.device))
            p = torch.softmax(s, -1) if n else s
            O = p @ V
            dp = dO @ V.T
            # |dP| + |delta| bounds what the difference cancels from
            mag = p * (dO.abs() @ V.abs().T + (dO.abs() * (p @ V.abs())).sum(-1, keepdim=True))
            ds = p * (dp - (dO * O).sum(-1, keepdim=True))
            o[b:e, h] = O
            dq[b:e, h] = scale * (ds @ K)
            mq[b:e, h] = scale * (mag @ K.abs())
            dk[b:e, kv] += scale * (ds.T @ Q)
            mk[b:e, kv] += scale * (mag.T @ Q.abs())
            dv[b:e, kv] += p.T @ dO
            mv[b:e, kv] += p.T @ dO.abs()
    return (o, dq, dk, dv), (mq, mk, mv)


def gather(cache, table, n):
    """The first n rows [n, HKV, D] of a sequence whose pages ``table`` lists."""
    page = cache.shape[1]
    j = torch.arange(n, device=cache.device)
    return cache[table.long()[j // page], j % page]


def rotate(x, cos_sin, positions, interleaved):
    """x [T, heads, D] with its first R elements turned by table rows [cos | sin] of R."""
    x = x.to(F64).clone()
    R = cos_sin.shape[1]
    for t, p in enumerate(positions.tolist()):
        for i in range(R // 2):
            c, s = cos_sin[p, i].to(F64), cos_sin[p, R // 2 + i].to(F64)
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
            u, w = x[t, :, a].clone(), x[t, :, b].clone()
            x[t, :, a], x[t, :, b] = u * c - w * s, w * c + u * s
    return x


def to_e4m3(x):
    """float64 values to the nearest of e4m3's (1 sign, 4 exponent and 3 mantissa bits, bias 7,
    largest 448), ties to the even one; |x| <= 448."""
    x = x.to(F64)
    _, e = torch.frexp(x)                          # x = m 2^e, 1/2 <= |m| < 1
    step = torch.ldexp(torch.ones_like(x), e.clamp(min=-5) - 4)
    return torch.round(x / step) * step


def quantise(x):
    """(e4m3 values in float64, exponents) of rows x [..., D]: the least exponent e >= -126 with
    max |x| <= 448 * 2^e over the finite elements; what is not finite becomes NaN."""
    x = x.to(F64)
    top = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(-1)
    m, e = torch.frexp(top)
    e = torch.where(top == 0, torch.full_like(e, -126), e - 9 + (m > 0.875)).clamp(min=-126)
    y = torch.where(torch.isfinite(x), x, torch.full_like(x, torch.nan))
    return to_e4m3(torch.ldexp(y, -e[..., None])), e


def behind_prefix(q, pk, pv, k, v, scale):
    """One token's q [H, D] over a prefix pk, pv [P, HKV, D] and keys k, v of its own: (o, a) of
    rows() over both."""
    k, v = torch.cat([pk, k]), torch.cat([pv, v])
    o, a = rows(q[None], k, v, scale, k.shape[0] - 1)
    return o[0], a[0]


def rotate_by(x, angles, factor, interleaved):
    """x [..., heads, D] with its first pairs turned by angles [..., R / 2] and multiplied by factor."""
    x = x.to(F64).clone()
    h = angles.shape[-1]
    c, s = factor * torch.cos(angles)[..., None, :], factor * torch.sin(angles)[..., None, :]
    a, b = (slice(0, 2 * h, 2), slice(1, 2 * h, 2)) if interleaved else (slice(0, h), slice(h, 2 * h))
    u, w = x[..., a].clone(), x[..., b].clone()
    x[..., a], x[..., b] = u * c - w * s, w * c + u * s
    return x
