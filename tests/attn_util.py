"""Inputs and derived tolerances of the attention tests."""
import torch

from oracle import attention as ref


def randn(gen, *shape, dtype=torch.bfloat16, scale=1.0):
    return (torch.randn(*shape, generator=gen) * scale).to(dtype)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def o_tolerance(o, a, v_sum, dtype):
    """Elementwise bound of a forward output.  The probabilities are rounded to the inputs'
    type: each is off by half a step of itself, together half a step of a = sum p |v|; fp16
    values below its normal range by 2^-25 of the largest, together 2^-25 sum |v|.  A score
    summed over D <= 128 products in fp32 is off by at most 128 * 2^-24 of its terms'
    magnitudes, which these inputs keep under 16 after scaling: 2^-13 of a probability, once
    in the numerator and once in the sum.  The result is rounded once more."""
    e = half_step(dtype)
    t = (e + 2.0 ** -12) * a
    if dtype == torch.float16:
        t = t + 2.0 ** -25 * v_sum
    return t + e * (o.abs() + t) + torch.finfo(dtype).tiny * e


def check_o(out, o, a, v, what):
    """out against (o, a) of oracle.attention with v's largest column sum."""
    assert torch.isfinite(out).all(), f"{what}: non-finite values"
    tol = o_tolerance(o, a, v.double().abs().sum(0).amax().item() if v.numel() else 0.0, out.dtype)
    err = (out.double().cpu() - o).abs()
    worst = (err - tol).max().item() if err.numel() else 0.0
    assert worst <= 0, f"{what}: {worst:.3e} past its tolerance (largest error {err.max().item():.3e})"


def paged(gen, lens, page, HKV, D, dtype, spare=3, width=None, fill=float("nan")):
    """(k_cache, v_cache, table, k list, v list): random rows for every sequence in shuffled
    pages; what is no key of a sequence is ``fill`` (NaN: nothing may leak)."""
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=gen)
    width = max([1, *need]) if width is None else width
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    kc = torch.full((pages, page, HKV, D), fill).to(dtype)
    vc = kc.clone()
    ks, vs, at = [], [], 0
    for i, n in enumerate(lens):
        table[i, :need[i]] = order[at:at + need[i]].to(torch.int32)
        at += need[i]
        k, v = randn(gen, n, HKV, D, dtype=dtype), randn(gen, n, HKV, D, dtype=dtype)
        j = torch.arange(n)
        pg = table[i].long()[j // page] if n else j
        kc[pg, j % page], vc[pg, j % page] = k, v
        ks.append(k)
        vs.append(v)
    return kc, vc, table, ks, vs


def bounds_of(cu):
    return list(zip(cu, cu[1:]))


__all__ = ["ref", "randn", "half_step", "o_tolerance", "check_o", "paged", "bounds_of"]
