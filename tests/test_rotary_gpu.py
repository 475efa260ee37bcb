"""The rotation by frequencies against float64, its gradients against the formula and against
differences, the table that the append reads, strides, positions far away, and captured steps."""
import math

import pytest
import torch

import hmx
from attn_util import half_step, randn, ref

pytestmark = pytest.mark.gpu
BF, F16 = torch.bfloat16, torch.float16


def _check(out, x, angles, factor, inter, what):
    """One rounding of the result; before it the angle's cosine and sine, off by less than 2^-21
    (the turn rounded to fp32, 2^-26 of at most half a one, and the functions' own), times the
    pair's magnitudes, beside three roundings in fp32 of the same."""
    want = ref.rotate_by(x, angles, factor, inter)
    h = angles.shape[-1]
    mag = x.double().abs()
    pair = torch.zeros_like(mag)
    a, b = (slice(0, 2 * h, 2), slice(1, 2 * h, 2)) if inter else (slice(0, h), slice(h, 2 * h))
    pair[..., a] = pair[..., b] = (mag[..., a] + mag[..., b]) * abs(factor)
    t = 2.0 ** -20 * pair
    tol = t + half_step(out.dtype) * (want.abs() + t) + torch.finfo(out.dtype).tiny * half_step(out.dtype)
    err = (out.cpu().double() - want).abs()
    assert (err <= tol).all(), f"{what}: {(err - tol).max():.2e} past its tolerance"


@pytest.mark.parametrize("B,T,H,HKV,D,R,inter,dtype,pos_shape", [
    (1, 1, 1, 1, 64, 64, False, BF, "T"), (2, 37, 4, 2, 128, 128, False, BF, "BT"),
    (3, 5, 7, 1, 128, 64, True, F16, "1T"), (1, 300, 3, 3, 64, 16, False, F16, "BT"),
    (2, 65, 33, 8, 128, 32, True, BF, "T"), (1, 1025, 5, 2, 128, 128, True, BF, "BT")])
def test_forward_and_gradients(dev, B, T, H, HKV, D, R, inter, dtype, pos_shape):
    gen = torch.Generator().manual_seed(T)
    q, k, dq, dk = (randn(gen, B, T, h, D, dtype=dtype) for h in (H, HKV, H, HKV))
    shape = {"T": (T,), "BT": (B, T), "1T": (1, T)}[pos_shape]
    pos = torch.randint(-5, 5000, shape, generator=gen, dtype=torch.int32 if B == 1 else torch.int64)
    inv, factor = hmx.rotary_frequencies(R, 5e5, dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=1024), device="cpu")
    ang = (pos.double()[..., None] * inv).expand(B, T, R // 2)
    qd, kd = (x.to(dev).requires_grad_() for x in (q, k))
    with torch.no_grad():
        plain = hmx.rotary_embedding(qd, kd, pos.to(dev), inv.to(dev), factor=factor, interleaved=inter)
    out = hmx.rotary_embedding(qd, kd, pos.to(dev), inv.to(dev), factor=factor, interleaved=inter)
    for o, p, x, n in zip(out, plain, (q, k), "qk"):
        assert torch.equal(o, p) and o.dtype == dtype
        _check(o.detach(), x, ang, factor, inter, n)
    grads = torch.autograd.grad(out, (qd, kd), (dq.to(dev), dk.to(dev)))
    for g, d, n in zip(grads, (dq, dk), "qk"):
        _check(g, d, -ang, factor, inter, "d" + n)


def test_gradients_against_differences(dev):
    """sum(out do) grows by u . dq where q grows by u: the rotation is linear, so a difference of
    any size is the derivative, up to the outputs' rounding."""
    gen = torch.Generator().manual_seed(1)
    q, do, u = (randn(gen, 1, 9, 2, 64, dtype=F16) for _ in range(3))
    pos = torch.arange(9, device=dev) * 7
    inv, _ = hmx.rotary_frequencies(64, device=dev)
    qd = q.to(dev).requires_grad_()
    g, = torch.autograd.grad(hmx.rotary_embedding(qd, None, pos, inv)[0], qd, do.to(dev))
    run = lambda x: hmx.rotary_embedding(x.to(dev), None, pos, inv)[0].double().cpu()
    diff = ((run(q + u) - run(q - u)) * do.double()).sum() / 2
    size = ((run(q + u).abs() + run(q - u).abs()) * do.double().abs()).sum()
    # q + u and q - u rounded, the outputs rounded, g rounded: each half a step of about `size`
    assert abs(diff - (g.cpu().double() * u.double()).sum()) <= 4 * half_step(F16) * size


def test_only_one_gradient_and_second_derivatives(dev):
    gen = torch.Generator().manual_seed(2)
    q, k = (randn(gen, 2, 5, 3, 64).to(dev) for _ in range(2))
    pos, (inv, _) = torch.arange(5, device=dev), hmx.rotary_frequencies(64, device=dev)
    both = hmx.rotary_embedding(q.requires_grad_(), k.requires_grad_(), pos, inv)
    do = randn(gen, 2, 5, 3, 64).to(dev)
    want = hmx.RotaryEmbedding.apply(do, None, pos, inv, 1.0, False, True)[0]
    for i, x in enumerate((q, k)):
        g, = torch.autograd.grad(both[i], x, do, retain_graph=True)
        assert torch.equal(g, want)
        assert torch.autograd.grad(both[i], (q, k)[1 - i], do, retain_graph=True, allow_unused=True)[0] is None
    k2 = k.detach().requires_grad_()
    out = hmx.rotary_embedding(q.detach(), k2, pos, inv)
    assert torch.equal(torch.autograd.grad(out[1], k2, do)[0], want)
    # the gradient is linear in do: its own gradient turns forward again
    do2 = do.clone().requires_grad_()
    g, = torch.autograd.grad(hmx.rotary_embedding(q, None, pos, inv)[0], q, do2, create_graph=True)
    assert torch.equal(torch.autograd.grad(g, do2, do)[0], hmx.rotary_embedding(do, None, pos, inv)[0])


def test_broadcast_and_strided_inputs(dev):
    """Views of one fused projection, heads before tokens, rows shared by expansion, and outputs
    in place."""
    gen = torch.Generator().manual_seed(3)
    B, T, H, HKV, D = 2, 33, 4, 2, 64
    qkv = randn(gen, B, T, (H + 2 * HKV) * D)
    q = qkv[..., :H * D].unflatten(-1, (H, D))
    k = qkv[..., H * D:(H + HKV) * D].unflatten(-1, (HKV, D))
    pos, (inv, _) = torch.randint(0, 99, (B, T), generator=gen), hmx.rotary_frequencies(64, device="cpu")
    ang = pos.double()[..., None] * inv
    dq = qkv.to(dev)
    dqq, dkk = dq[..., :H * D].unflatten(-1, (H, D)), dq[..., H * D:(H + HKV) * D].unflatten(-1, (HKV, D))
    out = hmx.rotary_embedding(dqq, dkk, pos.to(dev), inv.to(dev))
    for o, x in zip(out, (q, k)):
        _check(o, x, ang, 1.0, False, "views")
    heads_first = dqq.transpose(1, 2).contiguous().transpose(1, 2)
    late = torch.zeros(T, B, dtype=torch.long).copy_(pos.t()).t().to(dev)           # positions' tokens strided
    assert torch.equal(hmx.rotary_embedding(heads_first, None, late, inv.to(dev))[0], out[0])
    one = dqq[:1, :, :1].expand(B, T, H, D).detach()
    got = hmx.rotary_embedding(one, None, pos.to(dev), inv.to(dev))[0]
    _check(got, q[:1, :, :1].expand(B, T, H, D), ang, 1.0, False, "expanded")
    x = dqq[:, :, :1].detach().clone().requires_grad_()
    g, = torch.autograd.grad(hmx.rotary_embedding(x.expand(B, T, H, D), None, pos.to(dev), inv.to(dev))[0], x, dqq)
    parts = hmx.RotaryEmbedding.apply(dqq, None, pos.to(dev), inv.to(dev), 1.0, False, True)[0]
    assert (g.float() - parts.float().sum(2, keepdim=True)).abs().max() <= 2.0 ** -8 * 64
    odd = torch.zeros(B * T * H * D + 1, dtype=BF, device=dev)[1:].view(B, T, H, D).copy_(dqq)   # off 16 bytes
    assert torch.equal(hmx.rotary_embedding(odd, None, pos.to(dev), inv.to(dev))[0], out[0])
    v = dq.clone()
    got = hmx.rotary_embedding(dqq, dkk, pos.to(dev), inv.to(dev), q_out=dqq, k_out=dkk)
    assert got[0] is dqq and torch.equal(dqq, out[0]) and torch.equal(dkk, out[1])
    assert torch.equal(dq[..., (H + HKV) * D:], v[..., (H + HKV) * D:])


def test_far_positions_and_types(dev):
    """Positions past 2^31 and negative ones, frequencies in fp32, three dimensions."""
    gen = torch.Generator().manual_seed(4)
    q = randn(gen, 4, 2, 128)
    pos = torch.tensor([1, -7, 2 ** 33 + 5, 2 ** 20 + 1])
    inv = (1e4 ** (-torch.arange(0, 64, 2) / 64)).float()
    got, none = hmx.rotary_embedding(q.to(dev), None, pos.to(dev), inv.to(dev))
    assert none is None and got.shape == q.shape
    ang = torch.remainder(pos.double()[:, None] * inv.double(), 2 * math.pi)   # 2^33 in 53 bits: off by 2^-20 of a radian
    _check(got, q, ang, 1.0, False, "far")
    assert hmx.rotary_embedding(q.to(dev)[:0], None, pos.to(dev)[:0], inv.to(dev))[0].shape == (0, 2, 128)


def test_the_append_turns_by_the_table(dev):
    """append_paged_kv with rotary_table's rows and rotary_embedding turn alike: an attention layer
    that was trained with the one is served with the other."""
    gen = torch.Generator().manual_seed(5)
    T, D = 50, 64
    inv, factor = hmx.rotary_frequencies(D, 1e4, dict(type="linear", factor=2.0), device=dev)
    table = hmx.rotary_table(inv, 200, factor)
    ang = torch.arange(200)[:, None].double() * inv.cpu()
    want = torch.cat([ang.cos(), ang.sin()], 1) * factor
    assert table.shape == (200, D) and (table.cpu().double() - want).abs().max() <= 2.0 ** -21
    q, k = randn(gen, T, 4, D).to(dev), randn(gen, T, 2, D).to(dev)
    pos = torch.randint(0, 200, (T,), generator=gen).to(dev)
    kc, vc = (torch.zeros(4, 16, 2, D, dtype=BF, device=dev) for _ in range(2))
    a = hmx.append_paged_kv(k, k, kc, vc, torch.arange(T, device=dev), q=q, positions=pos, cos_sin=table)
    b, c = hmx.rotary_embedding(q, k, pos, inv, factor=factor)
    assert torch.equal(a, b) and torch.equal(kc.flatten(0, 1)[:T], c)


def test_captured_steps(dev):
    """A captured forward and backward replays with other inputs and positions."""
    gen = torch.Generator().manual_seed(6)
    q = randn(gen, 1, 20, 2, 64).to(dev).requires_grad_()
    do, pos = randn(gen, 1, 20, 2, 64).to(dev), torch.arange(20, device=dev)
    inv, _ = hmx.rotary_embedding, None
    inv, _ = hmx.rotary_frequencies(64, device=dev)
    step = lambda: (lambda o: (o.detach(), *torch.autograd.grad(o, q, do)))(hmx.rotary_embedding(q, None, pos, inv)[0])
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for i in range(4):
        with torch.no_grad():
            q.copy_(randn(gen, 1, 20, 2, 64))
        do.copy_(randn(gen, 1, 20, 2, 64))
        pos.add_(1000 * i)
        g.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in out]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_registered_gradient_at_the_ends_of_int32(dev):
    """The registered op's gradient turns by minus the angle at every position, the least int32
    (which minus itself is itself) among them."""
    from hmx import library
    gen = torch.Generator().manual_seed(7)
    q, do = randn(gen, 1, 3, 2, 64).to(dev).requires_grad_(), randn(gen, 1, 3, 2, 64).to(dev)
    pos = torch.tensor([-2 ** 31, 2 ** 31 - 1, -5], dtype=torch.int32, device=dev)
    inv, _ = hmx.rotary_frequencies(64, device=dev)
    a, = torch.autograd.grad(library.rotary_embedding(q, None, pos, inv)[0], q, do)
    b, = torch.autograd.grad(hmx.rotary_embedding(q, None, pos, inv)[0], q, do)
    assert torch.equal(a, b)
    ang = torch.remainder(pos.cpu().double()[:, None] * inv.cpu(), 2 * math.pi)   # off by 2^-21 of a radian
    _check(a, do.cpu(), -ang, 1.0, False, "the ends")
