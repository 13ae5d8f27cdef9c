"""Layer norm: both operands of the backwards as views, and fp32 weights beside 16-bit rows of every length.  Bounds as in ``test_layer_norm.py``."""
from __future__ import annotations

import pytest
import torch

import fhob
from test_layer_norm import columns_close, definition, make, matrix_close


@pytest.mark.gpu
@pytest.mark.parametrize("view", ["slice", "one_row", "transposed", "expanded", "expanded_rows", "one_column", "one_batch", "odd_start"])
def test_backwards_of_views(view):
    """x, dy or ddx a view: the bits of a contiguous copy's, and the values of the definition (``odd_start``: off the 16-byte grid, where
    the copy is on it, so other orders of sums)."""
    take = {"slice": lambda t: t[..., 16:144], "one_row": lambda t: t[:, 2:3, :128], "transposed": lambda t: t.transpose(0, 1),
            "expanded": lambda t: t[:1, :, :128].expand(4, 5, 128), "expanded_rows": lambda t: t[:, :1, :128].expand(3, 7, 128),
            "one_column": lambda t: t[..., 3:4], "one_batch": lambda t: t[1:2, 1:4, 8:], "odd_start": lambda t: t[..., 3:131]}[view]
    g = torch.Generator("cuda").manual_seed(11)
    views = {n: take(torch.randn(3, 5, 160, device="cuda", generator=g).bfloat16()) for n in ("x", "dy", "ddx")}
    cols = views["x"].shape[-1]
    vectors = {n: torch.randn(cols, device="cuda", generator=g) for n in ("w", "b", "ddw", "ddb")}
    plain = {n: t.contiguous() for n, t in views.items()}
    eps = 1e-5 if cols > 1 else 0.5
    ref = definition({**{n: t.reshape(-1, cols) for n, t in plain.items()}, **vectors}, eps)
    _, mean, rstd = fhob.layer_norm_forward(plain["x"], vectors["w"], vectors["b"], eps)

    def backwards(t):
        return [*fhob.layer_norm_backward(t["dy"], t["x"], vectors["w"], mean, rstd),
                *fhob.layer_norm_bwdbwd(t["ddx"], vectors["ddw"], vectors["ddb"], t["dy"], t["x"], vectors["w"], mean, rstd)]

    want = backwards(plain)
    for which in (("x",), ("dy",), ("ddx",), ("x", "dy", "ddx")):
        got = backwards({**plain, **{n: views[n] for n in which}})
        for i, (a, b) in enumerate(zip(got, want)):
            if view != "odd_start":
                assert torch.equal(a, b), (which, i)
            elif i in (0, 3, 4):
                matrix_close(a.reshape(-1, cols), ref[3 + i], 4.0)
    if cols > 1:
        for i, spread in ((0, 1.0), (3, 1.0), (4, 4.0)):
            matrix_close(want[i].reshape(-1, cols), ref[3 + i], spread)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("rows,cols", [(300, 256), (160, 1000), (160, 1001), (450, 2048), (149, 2501), (149, 5120), (149, 8192), (149, 8200), (160, 9001),
                                       (149, 12288), (149, 16384), (20, 16383)])
def test_fp32_weights_beside_16_bit_rows(rows, cols, dtype):
    t = make(rows, cols, dtype, seed=cols, wdtype="fp32")
    ref = definition(t, 1e-5)
    y, mean, rstd = fhob.layer_norm_forward(t["x"], t["w"], t["b"], 1e-5)
    matrix_close(y, ref[0])
    dx, dw, db = fhob.layer_norm_backward(t["dy"], t["x"], t["w"], mean, rstd)
    ddy, dx2, dw2 = fhob.layer_norm_bwdbwd(t["ddx"], t["ddw"], t["ddb"], t["dy"], t["x"], t["w"], mean, rstd)
    assert dw.dtype == db.dtype == dw2.dtype == torch.float32
    matrix_close(dx, ref[3])
    matrix_close(ddy, ref[6])
    matrix_close(dx2, ref[7], 4.0)
    dy, v, r = t["dy"].double(), t["ddx"].double(), ref[2][:, None]
    h = (t["x"].double() - ref[1][:, None]) * r
    p = r * (v - v.mean(-1, keepdim=True) - h * (v * h).mean(-1, keepdim=True))
    columns_close(dw, ref[4], (dy.abs() * (h.abs() + 1)).sum(0), rows)
    columns_close(db, ref[5], dy.abs().sum(0), rows)
    columns_close(dw2, ref[8], (dy.abs() * (p.abs() + 4 * r)).sum(0), rows)
