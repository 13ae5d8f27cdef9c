"""fhob.layer_norm and its derivatives against autograd of the definition in 64 bits.

Error bounds.  A row's sums have at most 16 terms one behind the other in a thread and ten additions between threads: 2^-24 * 26 of the sum of
the terms' sizes.  In the elements of the results these sums come with factors of about their own size, so 64 * 2^-24 of a
row's scale (times 1 + |mean| rstd where the mean is large against the deviation: the subtraction keeps the
absolute error of the mean) covers the fp32 arithmetic; storing rounds by at most half a step of the type.
Both are compared as 2-norms over the tensor.  The sums over rows have at most rows / 148 + 64 additions in a row, each off
by 2^-24 of the sum of sizes so far, and their terms 32 * 2^-24 of theirs.
"""
from __future__ import annotations

import ctypes as C

import pytest
import torch

import fhob
from fhob import _lib

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def make(rows, cols, dtype, seed=0, offset=0.25, wdtype=None):
    g = torch.Generator().manual_seed(seed)
    dt, wt = DTYPES[dtype], DTYPES[wdtype or dtype]
    n = lambda *s: torch.randn(s, generator=g)   # noqa: E731
    t = {"x": (1.5 * n(rows, cols) + offset).to(dt), "w": (1 + 0.2 * n(cols)).to(wt), "b": (0.2 * n(cols)).to(wt), "dy": n(rows, cols).to(dt),
         "ddx": n(rows, cols).to(dt), "ddw": (0.3 * n(cols)).to(wt), "ddb": (0.3 * n(cols)).to(wt)}
    return {k: v.cuda() for k, v in t.items()}


def definition(t, eps, weight=True, bias=True):
    """y, mean, rstd, dx, dw, db, ddy, dx2, dw2 in 64 bits."""
    x, dy = (t[k].double().requires_grad_(True) for k in ("x", "dy"))
    w = t["w"].double().requires_grad_(True) if weight else torch.ones_like(t["w"].double()).requires_grad_(True)
    b = t["b"].double().requires_grad_(True) if bias else torch.zeros_like(t["b"].double()).requires_grad_(True)
    mean = x.mean(-1, keepdim=True)
    rstd = ((x - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
    y = (x - mean) * rstd * w + b
    first = torch.autograd.grad(y, (x, w, b), dy, create_graph=True)
    ddw = t["ddw"].double() if weight else torch.zeros_like(w)
    ddb = t["ddb"].double() if bias else torch.zeros_like(b)
    second = torch.autograd.grad(first, (dy, x, w), (t["ddx"].double(), ddw, ddb))
    return [v.detach() for v in (y, mean.squeeze(-1), rstd.squeeze(-1), *first, *second)]


def matrix_close(got, ref, spread=1.0):
    tol = torch.finfo(got.dtype).eps / 2 + 64 * 2.0 ** -24 * spread
    err = float((got.double() - ref).norm() / ref.norm().clamp_min(1e-300))
    assert err <= tol, (err, tol)


def columns_close(got, ref, sizes, rows, spread=1.0):
    """`sizes`: the sum over the rows of the terms' sizes"""
    bound = (rows / 148 + 64 + 32 * spread) * 2.0 ** -24 * sizes
    bound = bound + (ref.abs() + bound) * torch.finfo(got.dtype).eps / 2 + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    assert bool(((got.double() - ref).abs() <= bound).all()), float(((got.double() - ref).abs() / bound).max())


# rows of every way to cut them up, on both sides of where it changes
EDGES = [(149, c, d) for d in ("bf16", "fp32") for c in (248, 256, 257, 264, 512, 520, 1016, 1024, 1032, 2049, 2056, 4096, 4097, 4104, 8191, 8192, 8200)]
# odd numbers of warps
EDGES += [(450, c, d) for d in ("bf16", "fp32") for c in (1280, 1301, 1536, 2501, 2560, 3584, 5120, 6001, 12288, 12289, 9001)]
EDGES += [(148, c, "fp16") for c in (256, 264, 1024, 2048, 4095, 4096, 4104, 8200)]
CASES = [(1, 1, "fp32"), (1, 16, "bf16"), (2, 3, "bf16"), (7, 1001, "fp16"), (33, 256, "fp32"), (64, 2048, "bf16"), (300, 1000, "fp16"), (5, 1026, "bf16"),
         (1500, 128, "bf16"), (2000, 2048, "bf16"), (700, 4096, "fp32"), (150, 8192, "bf16"), (150, 8192, "fp32"), (149, 16384, "bf16"), (3, 16384, "fp32"),
         (200, 16383, "bf16"), (40, 12001, "fp32"), (1000, 130, "fp32"), (4099, 514, "fp16"), (170, 6002, "bf16")]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,dtype", CASES + EDGES)
def test_all_directions(rows, cols, dtype):
    eps = 1e-5 if cols > 1 else 0.5
    t = make(rows, cols, dtype, seed=cols)
    ref = definition(t, eps)
    y, mean, rstd = fhob.layer_norm_forward(t["x"], t["w"], t["b"], eps)
    matrix_close(y, ref[0])
    matrix_close(mean, ref[1], spread=4.0)
    matrix_close(rstd, ref[2])
    dx, dw, db = fhob.layer_norm_backward(t["dy"], t["x"], t["w"], mean, rstd)
    ddy, dx2, dw2 = fhob.layer_norm_bwdbwd(t["ddx"], t["ddw"], t["ddb"], t["dy"], t["x"], t["w"], mean, rstd)
    h = (t["x"].double() - ref[1][:, None]) * ref[2][:, None]
    if cols > 1:   # a row of one element has h = 0 and gradients of rounding errors
        # what is left of dx and dx2 in short rows may be small against the terms they are made of
        spread = 1.0 if cols >= 16 else 64.0
        matrix_close(dx, ref[3], spread)
        matrix_close(dx2, ref[7], 4 * spread)
    matrix_close(ddy, ref[6])
    # (h is off by 64 * 2^-24 of its scale, one, however small it is itself)
    columns_close(dw, ref[4], (t["dy"].double().abs() * (h.abs() + 1)).sum(0), rows)
    columns_close(db, ref[5], t["dy"].double().abs().sum(0), rows)
    p = ref[2][:, None] * (t["ddx"].double() - t["ddx"].double().mean(-1, keepdim=True) - h * (t["ddx"].double() * h).mean(-1, keepdim=True))
    columns_close(dw2, ref[8], (t["dy"].double().abs() * (p.abs() + 4 * ref[2][:, None])).sum(0), rows)
    again = (*fhob.layer_norm_backward(t["dy"], t["x"], t["w"], mean, rstd), *fhob.layer_norm_bwdbwd(t["ddx"], t["ddw"], t["ddb"], t["dy"], t["x"], t["w"], mean, rstd))
    assert all(torch.equal(a, b) for a, b in zip((dx, dw, db, ddy, dx2, dw2), again))   # a fixed order of sums


@pytest.mark.gpu
@pytest.mark.parametrize("weight,bias", [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize("dtype,wdtype", [("bf16", "fp32"), ("fp16", "fp16")])
def test_autograd_with_parts_missing(dtype, wdtype, weight, bias):
    t = make(130, 384, dtype, wdtype=wdtype)
    ref = definition(t, 1e-5, weight, bias)
    leaf = {k: t[k].clone().requires_grad_(True) for k in ("x", "w", "b", "dy")}
    y = fhob.layer_norm(leaf["x"], leaf["w"] if weight else None, leaf["b"] if bias else None, 1e-5)
    matrix_close(y.detach(), ref[0])
    wrt = ["x"] + ["w"] * weight + ["b"] * bias
    first = torch.autograd.grad(y, [leaf[k] for k in wrt], leaf["dy"], create_graph=True)
    want = {"x": ref[3], "w": ref[4], "b": ref[5]}
    for k, g in zip(wrt, first):
        assert g.dtype == leaf[k].dtype
        matrix_close(g.detach(), want[k], 64.0)
    wrt2 = ["dy", "x"] + ["w"] * weight
    second = torch.autograd.grad(first, [leaf[k] for k in wrt2], [t["dd" + k] for k in wrt])
    for k, g in zip(wrt2, second):
        matrix_close(g.detach(), {"dy": ref[6], "x": ref[7], "w": ref[8]}[k], 64.0)


@pytest.mark.gpu
def test_gradient_of_a_penalty_and_no_third_derivative():
    """Only ||dx||^2 is differentiated: the cotangents of dw and db are absent."""
    t = make(64, 256, "fp32")
    x, w, b = (t[k].requires_grad_(True) for k in ("x", "w", "b"))

    def penalty(norm, x, w, b, c, **k):
        (dx,) = torch.autograd.grad((norm(x, w, b) * c).sum(), x, create_graph=True)
        return (dx ** 2).sum(), torch.autograd.grad((dx ** 2).sum(), (x, w), **k)

    got = penalty(fhob.layer_norm, x, w, b, t["dy"])[1]
    d = [v.detach().double().requires_grad_(True) for v in (x, w, b)]
    ref = penalty(lambda x, w, b: torch.nn.functional.layer_norm(x, (256,), w, b), *d, t["dy"].double())[1]
    for g, r in zip(got, ref):
        matrix_close(g, r, 16.0)
    # along one direction, against differences: the penalty is smooth, so the error is O(step^2) and rounding / step
    v = torch.randn_like(x)
    step = 2.0 ** -6
    hi, lo = (float(penalty(fhob.layer_norm, (x + s * step * v).detach().requires_grad_(True), w, b, t["dy"])[0].detach()) for s in (1, -1))
    slope = float((got[0] * v).double().sum())
    assert abs((hi - lo) / (2 * step) - slope) < 2e-2 * float(got[0].norm() * v.norm()) / 16
    _, graph = penalty(fhob.layer_norm, x, w, b, t["dy"], create_graph=True)   # may be asked for, as a helper does
    with pytest.raises(NotImplementedError):
        torch.autograd.grad(graph[0].sum(), x)


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [100.0, -1000.0])
def test_large_mean(offset):
    """The variance is summed around the mean, and the double backward's products of means do not cancel."""
    t = make(200, 1024, "fp32", offset=offset)
    t["ddx"] += 50.0
    t["dy"] += 20.0
    ref = definition(t, 1e-5)
    y, mean, rstd = fhob.layer_norm_forward(t["x"], t["w"], t["b"], 1e-5)
    spread = 1 + abs(offset) / 1.5
    matrix_close(y, ref[0], spread)
    dx, dw, db = fhob.layer_norm_backward(t["dy"], t["x"], t["w"], mean, rstd)
    ddy, dx2, dw2 = fhob.layer_norm_bwdbwd(t["ddx"], t["ddw"], t["ddb"], t["dy"], t["x"], t["w"], mean, rstd)
    matrix_close(dx, ref[3], 20 * spread)
    matrix_close(ddy, ref[6], 50 * spread)
    matrix_close(dx2, ref[7], 50 * spread)


@pytest.mark.gpu
def test_views_shapes_and_empty():
    t = make(48, 256, "bf16")
    w, b = t["w"], t["b"]
    want = fhob.layer_norm(t["x"], w, b)
    wide = torch.zeros(48, 300, device="cuda", dtype=torch.bfloat16)
    for at in (8, 3):                                                     # on and off the 16-byte grid
        wide[:, at:at + 256] = t["x"]
        view = wide[:, at:at + 256]
        y, mean, rstd = fhob.layer_norm_forward(view, w, b)
        assert torch.equal(y, want)
        a = fhob.layer_norm_backward(t["dy"], view, w, mean, rstd)
        c = fhob.layer_norm_backward(t["dy"], t["x"], w, mean, rstd)
        matrix_close(a[0], c[0].double(), 1.0)
        matrix_close(a[1], c[1].double(), 64.0)
    assert torch.equal(fhob.layer_norm(t["x"].view(2, 4, 6, 256), w, b), want.view(2, 4, 6, 256))
    assert torch.equal(fhob.layer_norm(t["x"].t().contiguous().t(), w, b), want)
    assert torch.equal(fhob.layer_norm(t["x"][:1].expand(5, 256), w, b), want[:1].expand(5, 256))
    assert torch.equal(fhob.layer_norm(t["x"][0], w, b), want[0])
    y, mean, rstd = fhob.layer_norm_forward(t["x"][:0], w, b)
    assert y.shape == (0, 256) and mean.shape == (0,)
    dx, dw, db = fhob.layer_norm_backward(y, y, w, mean, rstd)
    assert dx.shape == (0, 256) and not dw.any() and not db.any()
    x = t["x"].clone().requires_grad_(True)
    (g,) = torch.autograd.grad(fhob.layer_norm(x, w, b).sum(), x)        # the cotangent is an expanded number
    assert torch.isfinite(g).all()


@pytest.mark.gpu
def test_nan_stays_in_its_row():
    t = make(40, 512, "fp32")
    t["x"][3, 7], t["x"][5, 9] = float("nan"), float("inf")
    y, mean, rstd = fhob.layer_norm_forward(t["x"], t["w"], t["b"])
    bad = torch.isnan(y).any(1)
    assert bad.nonzero().flatten().tolist() == [3, 5]
    dx, dw, _ = fhob.layer_norm_backward(t["dy"], t["x"], t["w"], mean, rstd)
    assert torch.isnan(dx).any(1).nonzero().flatten().tolist() == [3, 5] and torch.isnan(dw).all()


@pytest.mark.gpu
def test_streams_and_graphs():
    t = make(600, 1024, "bf16")

    def step(x, w, b):
        y = fhob.layer_norm(x, w, b)
        first = torch.autograd.grad(y, (x, w, b), t["dy"], create_graph=True)
        return [r.detach() for r in (*first, *torch.autograd.grad(first, (x, w), (t["ddx"], t["ddw"], t["ddb"])))]

    leaves = lambda: [t[k].clone().requires_grad_(True) for k in ("x", "w", "b")]   # noqa: E731
    want = step(*leaves())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):   # leaves of its own: torch ties a leaf to the stream of its first graph
        x, w, b = leaves()
        got = step(x, w, b)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            captured = step(x, w, b)
        graph.replay()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    assert all(torch.equal(a, c) for a, c in zip(captured, want))
    with torch.no_grad():
        x.mul_(0.5)
    t["x"] = x.detach()
    graph.replay()
    assert all(torch.equal(a, c) for a, c in zip(captured, step(*leaves())))


def test_refusals():
    """Before anything is launched; on the CPU, so none of these reaches a device."""
    x, w = torch.zeros(3, 8), torch.zeros(8)
    m = torch.zeros(3)
    for error, call in [
        (ValueError, lambda: fhob.layer_norm(x, w, w)),                    # not on a GPU
        (TypeError, lambda: fhob.layer_norm(3)), (TypeError, lambda: fhob.layer_norm(x, 3)), (TypeError, lambda: fhob.layer_norm(x.double())),
        (ValueError, lambda: fhob.layer_norm(torch.tensor(1.0))), (ValueError, lambda: fhob.layer_norm(torch.zeros(3, 0))),
        (ValueError, lambda: fhob.layer_norm(torch.zeros(1, 16385))), (ValueError, lambda: fhob.layer_norm(x, w[:7])),
        (ValueError, lambda: fhob.layer_norm(x, torch.zeros(1, 8))), (TypeError, lambda: fhob.layer_norm(x, w.bfloat16())),
        (TypeError, lambda: fhob.layer_norm(x.bfloat16(), w.half())), (TypeError, lambda: fhob.layer_norm(x.bfloat16(), w, w.bfloat16())),
        (ValueError, lambda: fhob.layer_norm(x, w, w, -1e-5)), (ValueError, lambda: fhob.layer_norm(x, w, w, float("nan"))),
        (TypeError, lambda: fhob.layer_norm(x, w, w, "a")),
        (ValueError, lambda: fhob.layer_norm_backward(x[:2], x, w, m, m)), (TypeError, lambda: fhob.layer_norm_backward(x.half(), x, w, m, m)),
        (ValueError, lambda: fhob.layer_norm_backward(x, x, w, m[:2], m)), (TypeError, lambda: fhob.layer_norm_backward(x, x, w, m, m.double())),
        (ValueError, lambda: fhob.layer_norm_bwdbwd(None, w, None, x, x, None, m, m)),
        (ValueError, lambda: fhob.layer_norm_bwdbwd(x[:1], None, None, x, x, w, m, m)),
        (TypeError, lambda: fhob.layer_norm_bwdbwd(x, w.half(), None, x, x, w, m, m)),
    ]:
        with pytest.raises(error):
            call()


def test_c_refusals():
    lib = _lib.load()

    def problem(**over):
        n = _lib.FhobLayerNorm()
        n.rows, n.cols, n.dtype, n.w_dtype, n.x, n.x_row, n.mean, n.rstd = 4, 64, 0, 1, 256, 64, 512, 768
        for k, v in over.items():
            setattr(n, k, v)
        return C.byref(n)

    assert lib.fhob_layer_norm(None, 1024, None) == 1
    for over, status in [({"rows": 0}, 1), ({"cols": 0}, 1), ({"cols": 16385}, 2), ({"dtype": 5}, 1), ({"w_dtype": 2}, 1), ({"x": None}, 1),
                         ({"mean": None}, 1), ({"rstd": None}, 1), ({"eps": -1.0}, 1), ({"x_row": -1}, 1), ({"x": 257}, 3)]:
        assert lib.fhob_layer_norm(problem(**over), 1024, None) == status, over
    assert lib.fhob_layer_norm(problem(), None, None) == 1
    assert lib.fhob_layer_norm_backward(problem(), 1024, 64, 2048, 4096, 8192, None) == 4          # no workspace for dw, db
    assert lib.fhob_layer_norm_backward(problem(workspace=256, workspace_bytes=64), 1024, 64, 2048, 4096, 8192, None) == 4
    assert lib.fhob_layer_norm_backward(problem(), 1024, 64, None, None, None, None) == 1
    assert lib.fhob_layer_norm_bwdbwd(problem(), 1024, 64, 0, 0, 0, 0, 2048, 4096, 8192, None) == 4
    assert lib.fhob_layer_norm_bwdbwd(problem(), None, 64, 0, 0, 0, 0, 2048, 4096, None, None) == 1
    assert lib.fhob_layer_norm_workspace_bytes(0) == 0 and lib.fhob_layer_norm_workspace_bytes(10) > 0


def test_c_refuses_misplaced_vectors():
    """Vectors and statistics of 4 bytes an element at addresses of 2, next to rows that may lie there."""
    lib = _lib.load()

    def problem(**over):
        n = _lib.FhobLayerNorm()
        n.rows, n.cols, n.dtype, n.w_dtype, n.x, n.x_row, n.mean, n.rstd, n.workspace, n.workspace_bytes = 4, 63, 0, 1, 258, 63, 512, 768, 4096, 1 << 30
        for k, v in over.items():
            setattr(n, k, v)
        return C.byref(n)

    for over in ({"w": 1026}, {"b": 1026}, {"mean": 514}, {"rstd": 770}):
        assert lib.fhob_layer_norm(problem(**over), 2048, None) == 3, over
    for dw, db in ((4098, None), (None, 4098)):
        assert lib.fhob_layer_norm_backward(problem(), 1024, 63, 2048, dw, db, None) == 3
    for vw, vb, dw2 in ((1026, None, None), (None, 1026, None), (None, None, 1026)):
        assert lib.fhob_layer_norm_bwdbwd(problem(), 1024, 63, 0, 0, vw, vb, 2048, 4096, dw2, None) == 3
    # 16-bit vectors may lie at addresses of 2, not of 1
    assert lib.fhob_layer_norm(problem(w_dtype=0, w=1025), 2048, None) == 3


@pytest.mark.gpu
@pytest.mark.parametrize("view", ["slice", "one_row", "transposed", "expanded", "expanded_rows", "one_column", "one_batch"])
def test_views_of_three_dims(view):
    """The same bits as of a contiguous copy, whether the rows lie at one stride (read in place) or not (copied)."""
    base = torch.randn(3, 5, 160, device="cuda", generator=torch.Generator("cuda").manual_seed(11)).bfloat16()
    x = {"slice": base[..., 16:144], "one_row": base[:, 2:3, :128], "transposed": base.transpose(0, 1), "expanded": base[:1, :, :128].expand(4, 5, 128),
         "expanded_rows": base[:, :1, :128].expand(3, 7, 128), "one_column": base[..., 3:4], "one_batch": base[1:2, 1:4, 8:]}[view]
    cols = x.shape[-1]
    w, b = (torch.randn(cols, device="cuda") for _ in range(2))
    dy, v = (torch.randn(x.shape, device="cuda").bfloat16() for _ in range(2))
    for got, want in ((fhob.layer_norm_forward(x, w, b), fhob.layer_norm_forward(x.contiguous(), w, b)),):
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    _, mean, rstd = want
    for got, want in ((fhob.layer_norm_backward(x, dy, w, mean, rstd), fhob.layer_norm_backward(x.contiguous(), dy, w, mean, rstd)),
                      (fhob.layer_norm_bwdbwd(v, w, b, dy, x, w, mean, rstd), fhob.layer_norm_bwdbwd(v, w, b, dy, x.contiguous(), w, mean, rstd))):
        assert all(torch.equal(p, q) for p, q in zip(got, want))
