"""The layer norm's double backward where eps is not small against a row's variance, with cotangents along the row.

With h = (x - mean) rstd the mean of h^2 is var / (var + eps), not one, and mean(ddx h) and mean(dy w h) are of the size of
that, not of 1 / sqrt(cols): every term of dx2 counts.  The bounds are those of ``test_layer_norm.py``: sums of at most 26 roundings
(64 * 2^-24 of a row's scale) in fp32, four times that for dx2, and half a step for the stored result.
"""
from __future__ import annotations

import pytest
import torch

import fhob
from test_layer_norm import DTYPES, definition, make, matrix_close

EPS = (0.0, 1e-5, 1e-3, 0.1, 1.0)
DEVIATIONS = (3e-3, 0.02, 1.5)
# on and off the 16-byte grid, several rows a warp, several warps a row, vectors over the columns in registers, in shared memory
# and read again
SHAPES = [(70, 1024, "fp32"), (70, 1024, "bf16"), (200, 64, "fp32"), (33, 1001, "fp32"), (33, 1001, "bf16"), (150, 2048, "bf16"), (150, 6144, "fp32"),
          (150, 12288, "bf16"), (9, 8001, "fp32"), (40, 1000, "fp16")]


def along(rows, cols, dtype, deviation, eps, seed=0):
    """Inputs whose cotangents are half noise, half (x - mean) rstd; those of fp16 are scaled so that dx2, of the size of
    rstd^2 times two of them, stays within the type's range."""
    t = make(rows, cols, "fp32", seed=seed, offset=0.0)
    x = (t["x"] * (deviation / 1.5)).to(DTYPES[dtype])
    h = (x.double() - x.double().mean(-1, keepdim=True)) * (x.double().var(-1, unbiased=False, keepdim=True) + eps).rsqrt()
    scale = min(1.0, (deviation ** 2 + eps) ** 0.5) if dtype == "fp16" else 1.0
    t["x"] = x
    for n in ("dy", "ddx"):
        t[n] = ((t[n] + h.float()) * scale).to(DTYPES[dtype])
    return {n: v.to(DTYPES[dtype]) for n, v in t.items()}


@pytest.mark.gpu
@pytest.mark.parametrize("eps", EPS)
@pytest.mark.parametrize("deviation", DEVIATIONS)
@pytest.mark.parametrize("rows,cols,dtype", SHAPES)
def test_double_backward(rows, cols, dtype, deviation, eps):
    t = along(rows, cols, dtype, deviation, eps, seed=cols)
    ref = definition(t, eps)
    y, mean, rstd = fhob.layer_norm_forward(t["x"], t["w"], t["b"], eps)
    matrix_close(y, ref[0])
    dx, _, _ = fhob.layer_norm_backward(t["dy"], t["x"], t["w"], mean, rstd)
    matrix_close(dx, ref[3])
    ddy, dx2, _ = fhob.layer_norm_bwdbwd(t["ddx"], t["ddw"], t["ddb"], t["dy"], t["x"], t["w"], mean, rstd)
    matrix_close(ddy, ref[6])
    matrix_close(dx2, ref[7], 4.0)


@pytest.mark.gpu
@pytest.mark.parametrize("deviation,eps", [(0.1, 1e-5), (1e-2, 1e-5), (3e-3, 1e-5), (1.0, 0.1), (1.0, 1.0)])
@pytest.mark.parametrize("cols", [64, 1000])
def test_gradient_penalty(cols, deviation, eps):
    """||d(sum y^2) / dx||^2: its cotangents, 2 y and 2 dx, have parts along h by themselves.  dx is what the weight's deviations
    from one and the bias leave of 2 h, about half of it; its square is differentiated, so the bound is that of the penalty in ``test_layer_norm.py``."""
    t = along(64, cols, "fp32", deviation, eps)

    def penalty(norm, x, w, b):
        (dx,) = torch.autograd.grad((norm(x, w, b) ** 2).sum(), x, create_graph=True)
        return torch.autograd.grad((dx ** 2).sum(), (x, w))

    got = penalty(lambda x, w, b: fhob.layer_norm(x, w, b, eps), *(t[n].clone().requires_grad_(True) for n in ("x", "w", "b")))
    ref = penalty(lambda x, w, b: (x - x.mean(-1, keepdim=True)) * (x.var(-1, unbiased=False, keepdim=True) + eps).rsqrt() * w + b,
                  *(t[n].double().requires_grad_(True) for n in ("x", "w", "b")))
    for g, r in zip(got, ref):
        matrix_close(g, r, 16.0)
