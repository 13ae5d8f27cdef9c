"""Tangents of forward-mode differentiation: none of the operators has a rule for them, so a tensor that carries one is refused
instead of a result that looks constant."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import fhob

REFUSED = (NotImplementedError, RuntimeError)


def tensors():
    g = torch.Generator(device="cuda").manual_seed(1)
    new = lambda *s: torch.randn(*s, generator=g, device="cuda")   # noqa: E731
    t = {n: new(1, 2, 8, 64) for n in ("q", "k", "v", "do")}
    t.update(x=new(6, 64), w=new(64), b=new(64), dy=new(6, 64))
    t.update(positions=torch.arange(8, device="cuda")[None], frequencies=0.1 + torch.rand(32, generator=g, device="cuda"))
    return t


def dual(t):
    return forward_ad.make_dual(t, torch.ones_like(t))


@pytest.mark.gpu
@pytest.mark.parametrize("grad_mode", [True, False])
@pytest.mark.parametrize("call", ["rotary", "rotary_second", "rotary_inverse", "frequencies", "norm_x", "norm_weight", "norm_bias", "attention", "attention_rotary"])
def test_arguments(call, grad_mode):
    t = tensors()
    at = (t["positions"], t["frequencies"])
    r = fhob.RotaryPositions(*at)
    calls = {
        "rotary": lambda: fhob.rotary(dual(t["q"]), *at),
        "rotary_second": lambda: fhob.rotary((t["q"], dual(t["k"])), *at),
        "rotary_inverse": lambda: fhob.rotary(dual(t["q"]), *at, inverse=True, interleaved=True),
        "frequencies": lambda: fhob.rotary(t["q"], t["positions"], dual(t["frequencies"])),
        "norm_x": lambda: fhob.layer_norm(dual(t["x"]), t["w"], t["b"]),
        "norm_weight": lambda: fhob.layer_norm(t["x"], dual(t["w"]), t["b"]),
        "norm_bias": lambda: fhob.layer_norm(t["x"], t["w"], dual(t["b"])),
        "attention": lambda: fhob.attention(dual(t["q"]), t["k"], t["v"], is_causal=True, sliding_window=3, sink_tokens=2),
        "attention_rotary": lambda: fhob.attention(dual(t["q"]), dual(t["k"]), t["v"], rotary=r),
    }
    with torch.set_grad_enabled(grad_mode), forward_ad.dual_level():
        with pytest.raises(ValueError if call == "frequencies" else REFUSED):
            calls[call]()


@pytest.mark.gpu
@pytest.mark.parametrize("create_graph", [False, True])
@pytest.mark.parametrize("call", ["rotary", "norm", "attention"])
def test_cotangents(call, create_graph):
    """Of the first backward, and of the second (with a plain first cotangent)."""
    t = tensors()
    if call == "norm":
        leaf, dy = t["x"].requires_grad_(True), t["dy"]
        y = lambda: fhob.layer_norm(leaf, t["w"], t["b"])   # noqa: E731
    else:
        leaf, dy = t["q"].requires_grad_(True), t["do"]
        if call == "rotary":
            y = lambda: fhob.rotary(leaf, t["positions"], t["frequencies"])   # noqa: E731
        else:
            y = lambda: fhob.attention(leaf, t["k"], t["v"])   # noqa: E731
    with forward_ad.dual_level():
        with pytest.raises(REFUSED):
            torch.autograd.grad(y(), leaf, dual(dy), create_graph=create_graph)
        dy = dy.clone().requires_grad_(True)
        (first,) = torch.autograd.grad(y(), leaf, dy, create_graph=True)
        with pytest.raises(REFUSED):
            torch.autograd.grad(first, dy, dual(torch.ones_like(first)), create_graph=create_graph)


@pytest.mark.gpu
def test_plain_tensors_within_a_dual_level():
    t = tensors()
    want = fhob.layer_norm(t["x"], t["w"], t["b"]), fhob.rotary(t["q"], t["positions"], t["frequencies"])
    with forward_ad.dual_level():
        got = fhob.layer_norm(t["x"], t["w"], t["b"]), fhob.rotary(t["q"], t["positions"], t["frequencies"])
        x = forward_ad.unpack_dual(dual(t["x"])).primal
        again = fhob.layer_norm(x, t["w"], t["b"])
    assert all(torch.equal(a, b) for a, b in zip((*got, again), (*want, want[0])))
