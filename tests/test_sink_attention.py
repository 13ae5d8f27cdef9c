"""Attention with a sliding window and first tokens that stay visible (sink_tokens): forward, first and second backward
against dense attention in 64 bits with that mask, differentiated by autograd."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

from conftest import make_inputs
from oracle import attn_oracle as O
import fhob
from fhob import _lib

NAMES = ("o", "lse", "dq", "dk", "dv", "dq2", "dk2", "dv2", "ddo")
# Largest error of an entry against the tensor's largest, the bounds of the other parity tests: 16-bit storage rounds P and
# its derivatives to 2^-9 of an entry before the output products and the results once more; split fp32 drops 2^-16.
TOL = {torch.bfloat16: 2e-2, torch.float16: 2e-2, torch.float32: 1e-4}


def visible(nq, nk, window, sinks, device="cpu"):
    i = torch.arange(nq, device=device)[:, None] + nk - nq
    j = torch.arange(nk, device=device)[None]
    return (j <= i) & ((i - j < window) | (j < sinks))


def dense(x, scale, window, sinks):
    """The nine results in 64 bits; a query without a visible key has zeros and L = -inf."""
    q, k, v, do = (x[n].double().requires_grad_(True) for n in ("q", "k", "v", "do"))
    seen = visible(q.shape[1], k.shape[1], window, sinks, q.device)
    dead = ~seen.any(1)
    s = (q @ k.mT * scale).masked_fill(~(seen | dead[:, None]), -float("inf"))
    o = torch.softmax(s, -1).masked_fill(dead[:, None], 0.0) @ v
    lse = torch.logsumexp(s, -1).masked_fill(dead, -float("inf"))
    first = torch.autograd.grad(o, (q, k, v), do, create_graph=True)
    second = torch.autograd.grad(first, (q, k, v, do), [x[n].double() for n in ("ddq", "ddk", "ddv")])
    return [t.detach() for t in (o, lse, *first, *second)]


def ours(x, scale, window, sinks, impl="auto", check=True, out_o=True):
    kw = dict(is_causal=True, sliding_window=window, sink_tokens=sinks, impl=impl)
    o, lse = fhob.attention_forward(x["q"], x["k"], x["v"], scale, check=check, **kw)
    first = fhob.attention_backward(x["q"], x["k"], x["v"], o, x["do"], lse, scale, **kw)
    second = fhob.flash_bwdbwd(x["q"], x["k"], x["v"], o if out_o else None, x["do"], x["ddq"], x["ddk"], x["ddv"], lse, scale, check=check, **kw)
    return [o, lse, *first, *second]


def compare(got, ref, tol, few=False):
    for n, g, r in zip(NAMES, got, ref):
        if g is None:
            continue
        if n == "lse":
            g = g.reshape(r.shape).double()
            assert torch.equal(torch.isinf(g), torch.isinf(r)), n
            assert bool(((g - r).abs()[~torch.isinf(r)] < max(1e-5, tol / 50)).all()), n
            continue
        assert torch.isfinite(g).all(), n
        if float(r.abs().max()) < 1e-12:
            # One visible key: P = 1, so dS, dS2 and ddP are differences of equal numbers, sums of 2 d products of N(0, 1) entries
            # times d^-0.5: at most 32, each way of adding off by 32 * 16 * 2^-24 = 2^-15.  They multiply entries below 8.
            assert float(g.abs().max()) < 2.0 ** -12, n
            continue
        # O is rounded by half a step, eps / 2 of an entry, so D = rowsum(dO * O) is off by about eps / 2 * sqrt(d); that enters the
        # results times scale = d^-0.5 and entries of about one: by eps / 2, which shows where the results themselves are small.
        # Where a result adds up few pairs, their roundings do not average out: P, dS, dS2, ddP (entries of about one) are off by
        # eps / 2 and multiply entries of up to 4, two of them a pair: 4 eps.
        err, size = float((g.reshape(r.shape).double() - r).abs().max()), float(r.abs().max())
        assert err < tol * size + torch.finfo(g.dtype).eps * (4 if few else 0.5), (n, err, size)


# bh, n_q, n_k, window, sinks: tiles of both kinds of key; a window inside one tile and over several; sinks that end in, at and
# behind a tile; one query; queries that continue; dead queries; few queries (split keys), few keys (split queries)
SHAPES = [(2, 300, 300, 40, 4), (2, 300, 300, 1, 1), (1, 700, 700, 128, 64), (1, 700, 700, 130, 65), (2, 513, 513, 64, 128), (1, 640, 640, 100, 200),
          (3, 1, 500, 33, 4), (1, 1, 1, 1, 1), (2, 1, 5000, 900, 4), (2, 7, 3000, 64, 130), (2, 129, 1000, 300, 16), (2, 200, 90, 20, 5),
          (1, 400, 150, 60, 100), (1, 2000, 100, 30, 4), (1, 1500, 1700, 256, 1), (5, 257, 385, 50, 7),
          (2, 3000, 3000, 64, 4), (1, 2500, 2600, 70, 200),   # far queries in many parts
          (4, 2, 3000, 700, 4), (3, 4, 20, 3, 2), (2, 8, 40, 5, 3), (1, 6, 3, 1, 1), (2, 9, 200, 20, 3), (1, 1, 70, 40, 29)]   # few queries


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d,impl", [(torch.bfloat16, 64, "auto"), (torch.float16, 128, "auto"), (torch.bfloat16, 80, "auto"), (torch.float32, 64, "auto"),
                                          (torch.float32, 128, "auto"), (torch.bfloat16, 72, "simt")])
@pytest.mark.parametrize("bh,nq,nk,window,sinks", SHAPES)
def test_all_directions(bh, nq, nk, window, sinks, dtype, d, impl):
    x = make_inputs(bh, nq, nk, d, seed=nq + nk + sinks, dtype=dtype, device="cuda")
    got = ours(x, d ** -0.5, window, sinks, impl)
    compare(got, dense(x, d ** -0.5, window, sinks), TOL[dtype], few=nk < 8)
    again = ours(x, d ** -0.5, window, sinks, impl)
    for n, a, b in zip(NAMES, got, again):
        assert torch.equal(a, b), n                                  # fixed orders of sums
    lse = fhob.produce_L(x["q"], x["k"], True, d ** -0.5, window, sinks)
    compare([got[0], lse], dense(x, d ** -0.5, window, sinks)[:2], TOL[dtype])


@pytest.mark.gpu
@pytest.mark.parametrize("d", [32, 64, 128])
def test_fp32_is_fp32(d):
    """2-norm errors of a long fp32 problem: the backwards run on the CUDA cores, whose rows of sums have up to 2000 / 2 terms in a
    part, off by 2^-24 of the running sum each: 1e-6 if they average out over a tenth of them; the forward's split operands (2^-17
    each, and their product) stay below 1e-5.  impl="tcgen05" asks for the tensor cores all the way: 4e-5."""
    x = make_inputs(2, 2000, 2300, d, seed=d, dtype=torch.float32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    x = {n: t + 1e-3 * torch.randn(t.shape, generator=g, device="cuda") for n, t in x.items()}   # values that bf16 does not hold
    ref = dense(x, d ** -0.5, 700, 20)
    for impl in ("auto", "tcgen05") if d <= 64 else ("auto",):
        for n, a, b in zip(NAMES, ours(x, d ** -0.5, 700, 20, impl), ref):
            err = float((a.reshape(b.shape).double() - b).norm() / b.norm())
            assert err < (4e-5 if impl == "tcgen05" else 1e-5), (impl, n, err)


@pytest.mark.gpu
@pytest.mark.parametrize("d,d_v", [(64, 128), (128, 64), (32, 96)])
def test_two_head_dims_and_no_o(d, d_v):
    x = make_inputs(2, 400, 450, d, seed=5, dtype=torch.bfloat16, device="cuda")
    y = make_inputs(2, 400, 450, d_v, seed=6, dtype=torch.bfloat16, device="cuda")
    x.update({n: y[n] for n in ("v", "do", "ddv")})
    ref = dense(x, 0.1, 70, 9)
    compare(ours(x, 0.1, 70, 9), ref, 2e-2)
    compare(ours(x, 0.1, 70, 9, out_o=False), ref, 2e-2)


@pytest.mark.gpu
@pytest.mark.parametrize("d,d_v", [(8, 128), (128, 16), (40, 40), (96, 64)])
@pytest.mark.parametrize("nq", [1, 2, 3, 8])
def test_few_queries_of_every_width(nq, d, d_v):
    """One or two queries have a forward of their own, in fp32 throughout; more take the tensor cores, which round P to the storage
    type.  Views, the logsumexp alone, and a NaN in a value, which reaches the queries that see it."""
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        g = torch.Generator().manual_seed(nq + d)
        new = lambda *s: torch.randn(s, generator=g).to(dtype).cuda()   # noqa: E731
        q, k, v = new(2, nq, 3, d).transpose(1, 2), new(2, 900, 3, d).transpose(1, 2), new(2, 900, 3, d_v).transpose(1, 2)
        kw = dict(is_causal=True, sliding_window=333, sink_tokens=5)
        o, lse = fhob.attention_forward(q, k, v, 0.3, check=True, **kw)
        x = {"q": q.reshape(6, nq, d).double(), "k": k.reshape(6, 900, d).double(), "v": v.reshape(6, 900, d_v).double()}
        s = (x["q"] @ x["k"].mT * 0.3).masked_fill(~visible(nq, 900, 333, 5, "cuda"), -float("inf"))
        ref = torch.softmax(s, -1) @ x["v"]
        # fp32 arithmetic throughout: sums of at most 128 and 338 terms, exponentials of arguments up to about 50 (2^-24 * 50), one rounding
        assert O.rel_err(o.reshape(6, nq, d_v).cpu(), ref.cpu()) < (torch.finfo(dtype).eps / 2 + 1e-5 if nq <= 2 else TOL[dtype])
        for got in (lse, fhob.produce_L(q, k, True, 0.3, 333, 5)):   # (with rows of d alone: other groups of keys, other orders)
            assert float((got.reshape(6, nq) - torch.logsumexp(s, -1)).abs().max()) < 2e-5
        v2 = v.clone()
        v2[:, :, 900 - 333] = float("nan")   # the first key of the last query's window
        bad = torch.isnan(fhob.attention_forward(q, k, v2, 0.3, **kw)[0]).all(-1)
        assert torch.equal(bad, torch.ones_like(bad))
        if nq > 2:
            continue   # there, as in a product with the mask's zeros, a NaN value reaches queries of its tile that do not see it
        v2 = v.clone()
        v2[:, :, 900 - nq - 333] = float("nan")   # one in front of the first query's window: seen by none
        assert torch.equal(fhob.attention_forward(q, k, v2, 0.3, **kw)[0], o)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_masks_that_are_another(dtype):
    """Sinks that reach the window leave the causal mask, a window that reaches the start leaves the sinks without effect: the
    same bits."""
    x = make_inputs(2, 300, 350, 64, seed=3, dtype=dtype, device="cuda")

    def plain(**kw):
        o, lse = fhob.attention_forward(x["q"], x["k"], x["v"], 0.125, is_causal=True, **kw)
        return (o, lse, *fhob.flash_bwdbwd(x["q"], x["k"], x["v"], o, x["do"], x["ddq"], x["ddk"], x["ddv"], lse, 0.125, is_causal=True, **kw))

    for a, b in [(dict(sliding_window=50, sink_tokens=300), {}), (dict(sliding_window=50, sink_tokens=2 ** 31 - 1), {}),
                 (dict(sliding_window=350, sink_tokens=7), dict(sliding_window=350)), (dict(sliding_window=50, sink_tokens=0), dict(sliding_window=50))]:
        assert all(torch.equal(s, t) for s, t in zip(plain(**a), plain(**b))), (a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_views_and_neighbouring_heads(dtype):
    """A head's bits depend neither on its neighbours nor on where the tensors lie."""
    x = make_inputs(6, 500, 500, 64, seed=9, dtype=dtype, device="cuda")
    whole = ours(x, 0.125, 100, 4)
    one = ours({n: t[4:5] for n, t in x.items()}, 0.125, 100, 4)
    assert all(torch.equal(w[4:5], o) for w, o in zip(whole, one))
    v = {n: t.view(2, 3, *t.shape[1:]).transpose(1, 2).contiguous().transpose(1, 2) for n, t in x.items()}   # (B, N, H, D) seen as (B, H, N, D)
    assert all(torch.equal(w, o.reshape(w.shape)) for w, o in zip(whole, ours(v, 0.125, 100, 4)))


@pytest.mark.gpu
def test_nan_and_masked_garbage():
    """Keys that no query sees may hold anything; a NaN in a first key reaches every query, one behind the window only those that see it."""
    x = make_inputs(1, 300, 600, 64, seed=2, dtype=torch.bfloat16, device="cuda")
    window, sinks = 40, 4
    clean = ours(x, 0.125, window, sinks)
    hidden = ~visible(300, 600, window, sinks).any(0)
    assert int(hidden.sum()) == 300 - window + 1 - sinks
    for bad in (float("inf"), float("nan")):
        y = dict(x)
        y["v"] = x["v"].clone()
        y["v"][:, 450] = bad
        o = fhob.attention_forward(y["q"], y["k"], y["v"], 0.125, is_causal=True, sliding_window=window, sink_tokens=sinks)[0]
        seen = visible(300, 600, window, sinks)[:, 450].cuda()
        assert bool((~torch.isfinite(o[0])).any(1)[seen].all())
    z = {n: t.clone() for n, t in x.items()}
    z["k"][:, hidden.cuda()] = 3.0e4                                       # finite, however large: masked by selection
    z["v"][:, hidden.cuda()] = 3.0e4
    got = ours(z, 0.125, window, sinks)
    assert all(torch.equal(a, b) for a, b in zip(got, clean))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,tol", [(torch.bfloat16, 2e-2), (torch.float32, 1e-4)])
def test_autograd_twice(dtype, tol):
    x = make_inputs(3, 280, 330, 64, seed=8, dtype=dtype, device="cuda")
    leaf = {n: x[n].clone().requires_grad_(True) for n in ("q", "k", "v", "do")}
    o = fhob.attention(leaf["q"], leaf["k"], leaf["v"], 0.125, is_causal=True, sliding_window=60, sink_tokens=5)
    first = torch.autograd.grad(o, (leaf["q"], leaf["k"], leaf["v"]), leaf["do"], create_graph=True)
    second = torch.autograd.grad(first, tuple(leaf.values()), (x["ddq"], x["ddk"], x["ddv"]))
    ref = dense(x, 0.125, 60, 5)
    for n, g, r in zip(NAMES[:1] + NAMES[2:], (o, *first, *second), ref[:1] + ref[2:]):
        assert O.rel_err(g.detach().cpu(), r.cpu()) < tol, n
    if dtype == torch.float32:
        # along one direction, against differences of the first order results
        v = torch.randn_like(x["k"])
        step = 2.0 ** -7

        def value(k):
            o, lse = fhob.attention_forward(x["q"], k, x["v"], 0.125, is_causal=True, sliding_window=60, sink_tokens=5)
            g = fhob.attention_backward(x["q"], k, x["v"], o, x["do"], lse, 0.125, is_causal=True, sliding_window=60, sink_tokens=5)
            return sum(float((a * b).double().sum()) for a, b in zip(g, (x["ddq"], x["ddk"], x["ddv"])))

        slope = (value(x["k"] + step * v) - value(x["k"] - step * v)) / (2 * step)
        # third derivatives times step^2 (2^-14) and the rounding of the values (about 1e-5 of their terms) over the step
        assert abs(slope - float((second[1] * v).double().sum())) < 2e-2 * float(second[1].norm() * v.norm()) / 8


@pytest.mark.gpu
def test_host_tensors_compiled_op_and_graph():
    x = make_inputs(5, 300, 300, 64, seed=4, dtype=torch.bfloat16, device="cuda")
    want = ours(x, 0.125, 50, 4)
    o, lse = want[:2]
    args = (x["q"], x["k"], x["v"], o, x["do"], x["ddq"], x["ddk"], x["ddv"], lse)
    host = fhob.flash_bwdbwd(*(t.cpu() for t in args), 0.125, is_causal=True, sliding_window=50, sink_tokens=4)
    op = torch.ops.fhob.bwdbwd(*args, 0.125, True, 50, 4)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = ours(x, 0.125, 50, 4, check=False)
    graph.replay()
    for w, h, p, c in zip(want[5:], host, op, captured[5:]):
        assert torch.equal(w.cpu(), h) and torch.equal(w, p) and torch.equal(w, c)


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """One head of 2^31 / 64 + some keys and a few queries: the window and the first keys are 2^31 elements apart."""
    nk = 2 ** 25 + 300
    x = {n: torch.randn(1, 5, 64, device="cuda", dtype=torch.bfloat16) for n in ("q", "do")}
    k = torch.zeros(1, nk, 64, device="cuda", dtype=torch.bfloat16)
    v = torch.zeros_like(k)
    small = {n: torch.randn(1, 104, 64, device="cuda", dtype=torch.bfloat16) for n in ("k", "v")}
    for big, part in ((k, small["k"]), (v, small["v"])):
        big[:, :4], big[:, -100:] = part[:, :4], part[:, 4:]
    kw = dict(is_causal=True, sliding_window=60, sink_tokens=4)
    o, lse = fhob.attention_forward(x["q"], k, v, 0.125, check=True, **kw)
    ro, rl = fhob.attention_forward(x["q"], small["k"], small["v"], 0.125, check=True, **kw)
    assert O.rel_err(o.cpu(), ro.double().cpu()) < 2e-2 and float((lse - rl).abs().max()) < 1e-4
    dq, dk, dv = fhob.attention_backward(x["q"], k, v, o, x["do"], lse, 0.125, **kw)
    rq, rk, rv = fhob.attention_backward(x["q"], small["k"], small["v"], ro, x["do"], rl, 0.125, **kw)
    assert O.rel_err(dq.cpu(), rq.double().cpu()) < 2e-2
    for big, part in ((dk, rk), (dv, rv)):
        assert O.rel_err(torch.cat([big[:, :4], big[:, -100:]], 1).cpu(), part.double().cpu()) < 2e-2 and not big[:, 4:-100].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 64), (torch.float32, 64), (torch.float32, 128)])
def test_smaller_workspace(dtype, d):
    """Without room for the sums of the far queries' parts one CTA goes through them all: the same results but for the order."""
    x = make_inputs(2, 1500, 1500, d, seed=1, dtype=dtype, device="cuda")
    kw = dict(is_causal=True, sliding_window=100, sink_tokens=5)
    o, lse = fhob.attention_forward(x["q"], x["k"], x["v"], 0.1, **kw)
    args = (x["q"], x["k"], x["v"], o, x["do"], x["ddq"], x["ddk"], x["ddv"], lse, 0.1)
    p = _lib.FhobProblem()
    p.bh, p.n_q, p.n_k, p.d, p.dtype, p.causal, p.window = 2, 1500, 1500, d, _lib.DTYPES[str(dtype)], 1, 100
    lib = _lib.load()
    plain, full = lib.fhob_workspace_bytes_problem(C.byref(p)), lib.fhob_workspace_bytes_sinks(C.byref(p), 5)
    assert plain < full
    out = [torch.empty_like(t) for t in (x["q"], x["k"], x["v"], x["do"])]
    for size in (plain, full):
        got = fhob.flash_bwdbwd(*args, **kw, out=out, workspace=torch.empty(size, dtype=torch.uint8, device="cuda"), check=True)
        compare([*[None] * 5, *got], [*[None] * 5, *dense(x, 0.1, 100, 5)[5:]], TOL[dtype])


def test_refusals():
    q = torch.zeros(1, 4, 64)
    lse = torch.zeros(1, 4)
    for kw in (dict(sink_tokens=4), dict(is_causal=True, sink_tokens=4), dict(is_causal=True, sliding_window=3, sink_tokens=-1),
               dict(is_causal=True, sliding_window=3, sink_tokens=1.5), dict(is_causal=True, sliding_window=3, sink_tokens=2 ** 31)):
        with pytest.raises(ValueError):
            fhob.attention(q, q, q, 1.0, **kw)
    from fhob.ops import _sinks
    assert _sinks(3, 0) == 0 and _sinks(0, 0) == 0 and _sinks(3, 5) == 5
    e = torch.zeros(0, 4, 64)
    with pytest.raises(ValueError):
        fhob.flash_bwdbwd(*(e,) * 8, lse[:0], 1.0, is_causal=True, sink_tokens=3)


def test_c_refusals():
    lib = _lib.load()
    p = _lib.FhobProblem()
    p.bh, p.n_q, p.n_k, p.d, p.causal, p.window = 1, 128, 128, 64, 1, 0
    for n in ("q", "k", "v", "o", "d_o", "ddq", "ddk", "ddv", "lse", "dq2", "dk2", "dv2", "ddo", "workspace"):
        setattr(p, n, 4096)
    p.workspace_bytes = 1 << 20
    for window, sinks in ((0, 4), (16, -1)):
        p.window = window
        assert lib.fhob_bwdbwd_sinks(C.byref(p), sinks, None) == 1
        assert lib.fhob_forward_sinks(C.byref(p), sinks, 4096, 4096, None) == 1
        assert lib.fhob_backward_sinks(C.byref(p), sinks, 4096, 4096, 4096, None) == 1
    assert lib.fhob_forward_sinks(None, 0, 4096, 4096, None) == 1


@pytest.mark.parametrize("tile", [32, 64, 128])
def test_tile_lists_against_the_mask(tile):
    """Every visible pair's tile is streamed: first keys once in the first list, the others once in the second; no tile is out of range."""
    lib = _lib.load()
    f, b, e = C.c_int(), C.c_int(), C.c_int()
    for nq, nk in [(1, 1), (1, 700), (200, 200), (300, 700), (700, 300), (129, 128)]:
        for window in (1, 31, 128, 300):
            for sinks in (0, 1, 4, 64, 65, 130, 250):
                if sinks >= nk:
                    continue
                seen = visible(nq, nk, window, sinks)
                for q_side in (1, 0):
                    n_stat, n_strm, rows = (nq, nk, 128) if q_side else (nk, nq, 128)
                    for m0 in range(0, n_stat, rows):
                        assert lib.fhob_visible_tiles_sinks(q_side, m0, rows, tile, nq, nk, window, sinks, C.byref(f), C.byref(b), C.byref(e)) == 0
                        first, begin, end = f.value, b.value, e.value
                        assert 0 <= first <= -(-n_strm // tile) and 0 <= begin <= end <= -(-n_strm // tile)
                        part = seen[m0:m0 + rows] if q_side else seen[:, m0:m0 + rows].T
                        lists = [(0, sinks, 0, first), (sinks, nk, begin, end)] if q_side else [(0, nq, begin, end)]
                        assert q_side or first == 0
                        for c0, c1, lo, hi in lists:
                            tiles = ((part[:, c0:c1].any(0).nonzero() + c0) // tile).unique().tolist()
                            assert all(lo <= t < hi for t in tiles), (nq, nk, window, sinks, q_side, m0, lo, hi, tiles)


@pytest.mark.parametrize("tile", [64, 128])
def test_windows_of_neighbouring_query_tiles_touch(tile):
    """Two query tiles share a walk over the key tiles in the forward: no step of it may be without both."""
    lib = _lib.load()
    f, b, e = C.c_int(), C.c_int(), C.c_int()
    for nq, nk in [(1000, 1000), (700, 2000), (900, 500)]:
        for window in (1, 2, 63, 64, 65, 200):
            for sinks in (0, 1, 63, 64, 129, 300):
                lists = []
                for m0 in range(0, nq, 128):
                    assert lib.fhob_visible_tiles_sinks(1, m0, 128, tile, nq, nk, window, sinks, C.byref(f), C.byref(b), C.byref(e)) == 0
                    lists.append((f.value, b.value, e.value))
                for (f0, b0, e0), (f1, b1, e1) in zip(lists, lists[1:]):
                    assert f0 <= f1
                    if e0 > b0:
                        assert b0 <= b1 <= e0 <= e1 and e1 > b1
