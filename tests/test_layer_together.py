"""Norm, rotary positions and attention with a window and first tokens in a row, as a layer runs them: its gradient penalty
against the same layer in 64 bits, built from torch's own operations."""
from __future__ import annotations

import pytest
import torch

import fhob


def weights(dim, seed, dtype):
    g = torch.Generator().manual_seed(seed)
    w = {n: torch.randn(dim, dim, generator=g) / dim ** 0.5 for n in ("q", "k", "v", "o")}
    w["norm"], w["bias"] = 1 + 0.1 * torch.randn(dim, generator=g), 0.1 * torch.randn(dim, generator=g)
    return {n: t.to(dtype).cuda() for n, t in w.items()}


def split(t, heads):
    return t.view(t.shape[0], t.shape[1], heads, -1).transpose(1, 2)


def layer(x, w, heads, window, sinks, rope):
    h = fhob.layer_norm(x, w["norm"], w["bias"], 1e-5)
    q, k, v = (split(h @ w[n], heads) for n in ("q", "k", "v"))
    o = fhob.attention(q, k, v, is_causal=True, sliding_window=window, sink_tokens=sinks, rotary=rope)
    return x + o.transpose(1, 2).reshape(x.shape) @ w["o"]


def definition(x, w, heads, window, sinks, rope):
    mean = x.mean(-1, keepdim=True)
    h = (x - mean) / torch.sqrt((x - mean).square().mean(-1, keepdim=True) + 1e-5) * w["norm"] + w["bias"]
    q, k, v = (split(h @ w[n], heads) for n in ("q", "k", "v"))
    n = len(rope.frequencies)
    angle = (rope.positions[list(rope.axis_of_pair)].double() * rope.frequencies[:, None, None]).permute(1, 2, 0)[:, None]

    def turned(t):
        a, b = t[..., :n], t[..., n:2 * n]
        return torch.cat([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos(), t[..., 2 * n:]], -1)

    q, k = turned(q), turned(k)
    i = torch.arange(x.shape[1], device=x.device)
    back = i[:, None] - i[None]
    seen = (back >= 0) & ((back < window) | (i[None] < sinks))
    p = torch.softmax((q @ k.mT * q.shape[-1] ** -0.5).masked_fill(~seen, -float("inf")), -1)
    return x + (p @ v).transpose(1, 2).reshape(x.shape) @ w["o"]


def penalty(f, x, w, c, *a):
    """The loss and its weights' gradients: the output against c, and the squared gradient of that by the input."""
    y = f(x, w, *a)
    first = (y * c).sum()
    (dx,) = torch.autograd.grad(first, x, create_graph=True)
    loss = first / x.shape[1] + dx.square().sum()
    return [y, dx, *torch.autograd.grad(loss, (x, *w.values()))]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-4), (torch.bfloat16, 6e-2)])
def test_gradient_penalty_of_a_layer(dtype, tol):
    """2-norm errors.  fp32: split operands in the forward (1e-5) through a chain of six products and two derivatives.  16-bit: a
    rounding of 2^-9 (in the mean) at each of about forty results that the second derivatives run through, adding up like independent errors
    that the two derivatives amplify a few times: 40^0.5 * 2^-9 * 4 = 5e-2."""
    dim, heads, n, window, sinks = 256, 4, 330, 60, 5
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, n, dim, generator=g).to(dtype).cuda()
    c = torch.randn(2, n, dim, generator=g).to(dtype).cuda()
    w = weights(dim, 4, dtype)
    at = torch.arange(n, device="cuda") + 70000
    pos = torch.stack([at, at // 32 % 32, at % 32])[:, None].expand(3, 2, n)
    rope = fhob.RotaryPositions(pos, 10000.0 ** (-torch.arange(24, device="cuda", dtype=torch.float64) / 24), (0,) * 8 + (1,) * 8 + (2,) * 8)
    leaf = lambda t: t.clone().requires_grad_(True)   # noqa: E731
    got = penalty(layer, leaf(x), {k: leaf(t) for k, t in w.items()}, c, heads, window, sinks, rope)
    ref = penalty(definition, leaf(x.double()), {k: leaf(t.double()) for k, t in w.items()}, c.double(), heads, window, sinks, rope)
    for name, a, b in zip(("y", "dx", "gx", *("g" + k for k in w)), got, ref):
        err = float((a.double() - b).norm() / b.norm())
        assert err < tol, (name, err)


@pytest.mark.gpu
def test_queries_that_continue():
    """The queries take the last of the keys' positions."""
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(1, 2, n, 64, generator=g).bfloat16().cuda() for n in (3, 50, 50))
    rope = fhob.RotaryPositions(torch.arange(50, device="cuda")[None], torch.rand(32, generator=g).double().cuda())
    o = fhob.attention(q, k, v, is_causal=True, sliding_window=20, sink_tokens=2, rotary=rope)
    turned = fhob.rotary(q, rope.positions[:, 47:], rope.frequencies), fhob.rotary(k, rope.positions, rope.frequencies)
    assert torch.equal(o, fhob.attention(*turned, v, is_causal=True, sliding_window=20, sink_tokens=2))
    with pytest.raises(ValueError):
        fhob.attention(k, q, q, rotary=rope)
    with pytest.raises(ValueError):
        fhob.attention(q, k[:, :, :40], v[:, :, :40], rotary=rope)
