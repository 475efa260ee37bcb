"""The backward of causal attention on the GPU against the float64 formulas and differences.

Elementwise tolerances: dS is rounded to bf16 (half a step of itself), the row term dO . O
sees O rounded and formed from rounded probabilities (two half steps of sum |dO| p |v|),
and fp32 scores leave 2^-11 of each term's magnitude (2^-12 in P, and in the sum that
normalises it); the sums of magnitudes come from the oracle.  The gradient is rounded once
more.  The norm-wise bound is the one of the other ops' outputs."""
import pytest
import torch

import hmx
from attn_util import bounds_of, half_step, randn, ref
from util import OUT_REL, rel_err

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _check(grads, want, mags, what):
    e = half_step(BF)
    for name, g, w, m, n in zip("qkv", grads, want, mags, (3, 3, 1)):
        assert torch.isfinite(g).all(), f"{what} d{name}: non-finite"
        t = (n * e + 2.0 ** -11) * m
        tol = t + e * (w.abs() + t) + 1e-30
        worst = ((g.double().cpu() - w).abs() - tol).max().item()
        assert worst <= 0, f"{what} d{name}: {worst:.3e} past its tolerance"
        assert rel_err(g, w) <= OUT_REL, f"{what} d{name}: {rel_err(g, w):.3e}"


def _inputs(seed, B, T, H, HKV, D):
    gen = torch.Generator().manual_seed(seed)
    return [randn(gen, B, T, n, D) for n in (H, HKV, HKV, H)]


@pytest.mark.parametrize("T,H,HKV,D", [
    (1, 2, 1, 128), (2, 4, 4, 64), (31, 6, 2, 64), (33, 8, 1, 128), (64, 2, 2, 128), (65, 3, 3, 64),
    (129, 7, 1, 128), (257, 4, 2, 128), (300, 8, 2, 64), (640, 2, 1, 128),
])
def test_grads_one_sequence(dev, T, H, HKV, D):
    q, k, v, do = _inputs(T, 1, T, H, HKV, D)
    ins = [x.to(dev).requires_grad_() for x in (q, k, v)]
    o = hmx.causal_attention(*ins)
    grads = torch.autograd.grad(o, ins, do.to(dev))
    (_, *want), mags = ref.causal_grads(q[0], k[0], v[0], D ** -0.5, [(0, T)], do[0])
    _check([g[0] for g in grads], want, mags, f"T={T}")
    assert torch.equal(o.detach(), hmx.causal_attention(*[x.detach() for x in ins]))


@pytest.mark.parametrize("cu", [[0, 5, 5, 70, 200], [3, 4, 5, 130], [0, 128, 200], [0, 0, 190],
                                [0, *range(1, 71), 200]])
def test_grads_packed(dev, cu):
    T, H, HKV, D = 200, 6, 2, 64
    q, k, v, do = _inputs(len(cu), 1, T, H, HKV, D)
    ins = [x.to(dev).requires_grad_() for x in (q, k, v)]
    o = hmx.causal_attention(*ins, cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=dev))
    grads = torch.autograd.grad(o, ins, do.to(dev))
    (_, *want), mags = ref.causal_grads(q[0], k[0], v[0], D ** -0.5, bounds_of(cu), do[0])
    _check([g[0] for g in grads], want, mags, str(cu))
    for g in grads:
        assert (g[0, :cu[0]] == 0).all() and (g[0, cu[-1]:] == 0).all()


def test_grads_batch_scale_strides_and_repeat(dev):
    """A batch of slices of one projection, an expanded output gradient, and the same bits
    on a second run."""
    B, T, H, HKV, D = 3, 90, 4, 2, 128
    gen = torch.Generator().manual_seed(0)
    qkv = randn(gen, B, T, (H + 2 * HKV) * D)
    x = qkv.to(dev).requires_grad_()
    runs = []
    for _ in range(2):
        q, k, v = (y.view(B, T, -1, D) for y in x.split([H * D, HKV * D, HKV * D], -1))
        o = hmx.causal_attention(q, k, v, 0.1)
        runs.append(torch.autograd.grad(o.sum(), x)[0])
    assert torch.equal(*runs)
    got = runs[0].view(B, T, -1, D).split([H, HKV, HKV], 2)
    for b in range(B):
        q, k, v = (y.view(T, -1, D) for y in qkv[b].split([H * D, HKV * D, HKV * D], -1))
        (_, *want), mags = ref.causal_grads(q, k, v, 0.1, [(0, T)], torch.ones(T, H, D))
        _check([g[b] for g in got], want, mags, f"b={b}")


def test_gradient_against_differences(dev):
    """<gradient, direction> against the central difference of the float64 forward: the
    gradient's rounding (half a step of each product's magnitude, and 3 more as above) is
    what separates them."""
    T, H, HKV, D = 70, 4, 2, 64
    q, k, v, do = _inputs(11, 1, T, H, HKV, D)
    ins = [x.to(dev).requires_grad_() for x in (q, k, v)]
    grads = torch.autograd.grad(hmx.causal_attention(*ins), ins, do.to(dev))
    _, mags = ref.causal_grads(q[0], k[0], v[0], D ** -0.5, [(0, T)], do[0])
    gen = torch.Generator().manual_seed(12)
    base = [x[0].double() for x in (q, k, v)]
    loss = lambda xs: (ref.causal(*xs, D ** -0.5, [(0, T)])[0] * do[0].double()).sum().item()
    for i in range(3):
        u = torch.randn(base[i].shape, generator=gen, dtype=torch.float64)
        h = 1e-4
        hi, lo = ([x + s * h * u if j == i else x for j, x in enumerate(base)] for s in (1, -1))
        diff = (loss(hi) - loss(lo)) / (2 * h)
        got = (grads[i][0].double().cpu() * u).sum().item()
        # rounding errors of the elements are independent: their root sum of squares, fivefold
        tol = 5 * 4 * half_step(BF) * (mags[i] * u.abs()).square().sum().sqrt().item()
        assert abs(got - diff) <= tol + 1e-6 * abs(diff), (i, got, diff, tol)


def test_refusals(dev):
    q, k, v, _ = (x.to(dev).requires_grad_() for x in _inputs(1, 1, 8, 2, 2, 64))
    with pytest.raises(ValueError, match="out"):
        hmx.causal_attention(q, k, v, out=torch.empty_like(q))
    h = [x.detach().half().requires_grad_() for x in (q, k, v)]
    with pytest.raises(NotImplementedError, match="bf16"):
        hmx.causal_attention(*h)
    with torch.no_grad():
        hmx.causal_attention(*h)


def test_grads_of_head_major_inputs_and_an_odd_group(dev):
    """Heads outermost in memory (large head strides), and groups that do not divide a tile."""
    for H, HKV, D in ((8, 2, 64), (10, 2, 128), (48, 1, 64)):
        T = 150
        q, k, v, do = _inputs(H, 1, T, H, HKV, D)
        ins = [x.to(dev).transpose(1, 2).contiguous().transpose(1, 2).requires_grad_() for x in (q, k, v)]
        g = do.to(dev).transpose(1, 2).contiguous().transpose(1, 2)
        grads = torch.autograd.grad(hmx.causal_attention(*ins), ins, g)
        (_, *want), mags = ref.causal_grads(q[0], k[0], v[0], D ** -0.5, [(0, T)], do[0])
        _check([x[0] for x in grads], want, mags, f"H={H}")


@pytest.mark.parametrize("cu", [None, [0, 700, 700, 2000]])
def test_grads_where_the_forward_splits_its_keys(dev, cu):
    T, H, HKV, D = 2000, 2, 1, 64
    q, k, v, do = _inputs(3, 1, T, H, HKV, D)
    ins = [x.to(dev).requires_grad_() for x in (q, k, v)]
    o = hmx.causal_attention(*ins, cu_seqlens=None if cu is None else torch.tensor(cu, device=dev))
    grads = torch.autograd.grad(o, ins, do.to(dev))
    bounds = [(0, T)] if cu is None else bounds_of(cu)
    (_, *want), mags = ref.causal_grads(q[0], k[0], v[0], D ** -0.5, bounds, do[0])
    _check([g[0] for g in grads], want, mags, str(cu))


@pytest.mark.parametrize("cu,H,HKV", [([0, 5, 5, 70, 400], 6, 2), ([3, 4, 5, 330], 4, 4), ([0, 128, 256, 400], 7, 1),
                                      ([0, *range(1, 71), 400], 4, 2)])
def test_grads_packed_at_the_larger_head_size(dev, cu, H, HKV):
    T, D = 400, 128
    q, k, v, do = _inputs(len(cu), 1, T, H, HKV, D)
    ins = [x.to(dev).requires_grad_() for x in (q, k, v)]
    o = hmx.causal_attention(*ins, cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=dev))
    grads = torch.autograd.grad(o, ins, do.to(dev))
    (_, *want), mags = ref.causal_grads(q[0], k[0], v[0], D ** -0.5, bounds_of(cu), do[0])
    _check([g[0] for g in grads], want, mags, str(cu))
    for g in grads:
        assert (g[0, :cu[0]] == 0).all() and (g[0, cu[-1]:] == 0).all()


@pytest.mark.parametrize("T,cu,H,HKV,D", [(2300, None, 4, 1, 128), (2300, [0, 1500, 2301], 2, 2, 128), (1801, None, 8, 2, 64)])
def test_grads_of_long_sequences(dev, T, cu, H, HKV, D):
    """Many tiles of rows and keys, the last ones ragged."""
    T = cu[-1] if cu else T
    q, k, v, do = _inputs(T, 1, T, H, HKV, D)
    ins = [x.to(dev).requires_grad_() for x in (q, k, v)]
    o = hmx.causal_attention(*ins, cu_seqlens=None if cu is None else torch.tensor(cu, device=dev))
    grads = torch.autograd.grad(o, ins, do.to(dev))
    (_, *want), mags = ref.causal_grads(q[0], k[0], v[0], D ** -0.5, [(0, T)] if cu is None else bounds_of(cu), do[0])
    _check([g[0] for g in grads], want, mags, f"T={T}")


@pytest.mark.parametrize("B,T,H,HKV,D", [(8, 16, 8, 2, 128), (4, 33, 4, 1, 64), (2, 64, 8, 8, 64), (1, 700, 4, 2, 128)])
def test_query_gradients_of_peaked_rows(dev, B, T, H, HKV, D):
    """Heads whose rows attend few keys.  The gradient's own rounding makes an error r, dS's
    rounding another of its size, and what is left of the row term's error may be a third,
    all independent: together sqrt(3) r.  (The row term is formed from a rounded output; its
    error times P K alone would make 1.8 to 2.4 r here.)"""
    q, k, v, do = _inputs(T, B, T, H, HKV, D)
    q = (q.float() * 2.5).to(BF)
    ins = [x.to(dev).requires_grad_() for x in (q, k, v)]
    got = torch.autograd.grad(hmx.causal_attention(*ins), ins, do.to(dev))[0].double().cpu()
    want = torch.stack([ref.causal_grads(q[b], k[b], v[b], D ** -0.5, [(0, T)], do[b])[0][1] for b in range(B)])
    r = rel_err(want.to(BF), want)
    assert rel_err(got, want) <= 3 ** 0.5 * r, (rel_err(got, want), r)


def test_nan_rows_of_short_sequences(dev):
    """Gradients are defined for finite inputs; NaN in one sequence stays in it, and reads
    nothing behind it (its last row's scores are all NaN, those of no keys too)."""
    H, HKV, D = 4, 2, 64
    q, k, v, do = _inputs(2, 1, 12, H, HKV, D)
    q[0, 11] = float("nan")
    cu = torch.tensor([0, 1, 4, 10, 12], dtype=torch.int32, device=dev)
    ins = [x.to(dev).requires_grad_() for x in (q, k, v)]
    grads = torch.autograd.grad(hmx.causal_attention(*ins, cu_seqlens=cu), ins, do.to(dev))
    (_, *want), mags = ref.causal_grads(q[0, :10], k[0, :10], v[0, :10], D ** -0.5, [(0, 1), (1, 4), (4, 10)], do[0, :10])
    _check([g[0, :10] for g in grads], want, mags, "beside NaN")
    assert grads[0][0, 11].isnan().all()


@pytest.mark.parametrize("D", [64, 128])
def test_the_end_of_a_long_prompt(dev, D):
    """100003 tokens: the last rows' outputs and dQ, and dK and dV of the last keys, which no
    other rows see, from the formulas over all keys."""
    T, H, HKV, m = 100003, 4, 2, 5
    gen = torch.Generator(device=dev).manual_seed(D)
    q, k, v, do = (torch.randn(1, T, n, D, generator=gen, device=dev).to(BF).requires_grad_() for n in (H, HKV, HKV, H))
    o = hmx.causal_attention(q, k, v)
    grads = [g[0, -m:].double().cpu() for g in torch.autograd.grad(o, (q, k, v), do.detach())]
    Q, K, V, dO = (x[0].detach().double() for x in (q, k, v, do))
    scale, e = D ** -0.5, half_step(BF)
    want = [torch.zeros(m, n, D, dtype=torch.float64) for n in (H, HKV, HKV)]
    mags = [torch.zeros_like(x) for x in want]
    for h in range(H):
        kv = h // (H // HKV)
        s = scale * (Q[-m:, h] @ K[:, kv].T)
        s[:, -m:].masked_fill_(torch.ones(m, m, dtype=torch.bool, device=dev).triu(1), -torch.inf)
        p = torch.softmax(s, -1)
        O = p @ V[:, kv]
        d = dO[-m:, h]
        a = p @ V[:, kv].abs()
        # P in bf16 and its scores' 2^-12, twice, and the result's rounding
        t = (e + 2.0 ** -11) * a
        assert ((o[0, -m:, h].detach().double() - O).abs() <= t + e * (O.abs() + t)).all()
        ds = p * (d @ V[:, kv].T - (d * O).sum(-1, keepdim=True))
        mag = p * (d.abs() @ V[:, kv].abs().T + (d.abs() * a).sum(-1, keepdim=True))
        for x, ww in ((want, (scale * ds @ K[:, kv], scale * ds[:, -m:].T @ Q[-m:, h], p[:, -m:].T @ d)),
                         (mags, (scale * mag @ K[:, kv].abs(), scale * mag[:, -m:].T @ Q[-m:, h].abs(), p[:, -m:].T @ d.abs()))):
            x[0][:, h] = ww[0].cpu()
            x[1][:, kv] += ww[1].cpu()
            x[2][:, kv] += ww[2].cpu()
    for name, g, w, mg, n in zip("qkv", grads, want, mags, (3, 3, 1)):
        t = (n * e + 2.0 ** -11) * mg
        assert ((g - w).abs() <= t + e * (w.abs() + t) + 1e-30).all(), name
