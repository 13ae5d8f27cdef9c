"""Performance cases of the operators around a twice-differentiable attention layer, and their plain forms.

* ``sinks``   attention with a sliding window and a few first tokens that stay visible: ``token`` and ``forward``
  (O and the logsumexp), ``backward`` (dQ, dK, dV), ``op`` (the double backward), ``grad2`` (all three through autograd)
* ``rotary``  rotary positions with several axes on queries and keys: ``apply``, ``step`` (and the backward pass)
* ``norm``    layer norm: ``forward``, ``step`` (and the backward pass), ``grad2`` (and the double backward)

``own`` false: elementary torch operations in 32 bits, rounded once at the end.  ``own`` true: the framework's entry points.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _fhob():
    package = os.path.join(os.getcwd(), "flash-hob_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    import fhob
    return fhob


# ---------------------------------------------------------------- cases


def _sinks(kind, dtype, batch, heads, n_q, n_k, d, window, sinks, layout="bhnd", cotangent=1.0):
    """``layout`` "bnhd": (batch, sequence, head, dim) projections seen as (batch, head, sequence, dim)."""
    return {"op": "sinks", "kind": kind, "dtype": dtype, "batch": batch, "heads": heads, "n_q": n_q, "n_k": n_k, "d": d,
            "window": window, "sinks": sinks, "layout": layout, "cotangent": cotangent}


def _rotary(kind, dtype, batch, heads, heads_k, n, d, pairs, axes, interleaved=False, layout="bhnd"):
    """``pairs`` of the d/2 pairs of a row are rotated; ``axes`` 3: the first quarter of them by time, the rest by height and width."""
    return {"op": "rotary", "kind": kind, "dtype": dtype, "batch": batch, "heads": heads, "heads_k": heads_k, "n": n, "d": d,
            "pairs": pairs, "axes": axes, "interleaved": interleaved, "layout": layout}


def _norm(kind, dtype, rows, cols):
    return {"op": "norm", "kind": kind, "dtype": dtype, "rows": rows, "cols": cols}


def listed():
    def named(name, case):
        return dict(case, name=name)

    return [
        # Generation of one token a sequence behind a long cache: only the window and the first tokens are read.
        named("sinks token bf16 128h 1x8192", _sinks("token", "bf16", 8, 16, 1, 8192, 128, 1024, 4)),
        # A streaming language-model layer in training or prefill: forward ...
        named("sinks forward bf16 32h n4096", _sinks("forward", "bf16", 2, 16, 4096, 4096, 128, 1024, 4)),
        # ... and first backward; the first tokens' keys are seen by every query.
        named("sinks backward bf16 32h n4096", _sinks("backward", "bf16", 2, 16, 4096, 4096, 128, 1024, 4, cotangent=0.1)),
        # Double backward over a long context, one GPU's share of a head split: few heads, so the first keys' long
        # column of queries is the critical path unless it is shared out.
        named("sinks op bf16 4h n32768", _sinks("op", "bf16", 1, 4, 32768, 32768, 128, 2048, 4)),
        # Head dim and length off the tile grid, read in place from projections.
        named("sinks op fp16 ragged d80", _sinks("op", "fp16", 2, 12, 3333, 3333, 80, 512, 16, layout="bnhd")),
        # A numerically careful run, or the check of a 16-bit one.
        named("sinks op fp32 8h n1024 d128", _sinks("op", "fp32", 1, 8, 1024, 1024, 128, 256, 4)),
        # A gradient-penalty step of a small model: forward, first and second backward through autograd.
        named("sinks grad2 bf16 8h n512 d64", _sinks("grad2", "bf16", 2, 4, 512, 512, 64, 128, 4)),
        # Positions of one new token a sequence.
        named("rotary token bf16 8x16h", _rotary("apply", "bf16", 8, 16, 16, 1, 128, 64, 3)),
        # A video in training: 8192 patches with a time, a row and a column each.
        named("rotary step bf16 32h n8192", _rotary("step", "bf16", 2, 16, 16, 8192, 128, 64, 3)),
        # The norm in front of the attention, a few tokens ...
        named("norm forward bf16 64x2048", _norm("forward", "bf16", 64, 2048)),
        # ... a training step of 16384 tokens of a layer of 16 heads of 128 ...
        named("norm step bf16 16384x2048", _norm("step", "bf16", 16384, 2048)),
        # ... and a gradient-penalty step with a width off the grid.
        named("norm grad2 fp16 3333x1000", _norm("grad2", "fp16", 3333, 1000)),
    ]


def _log_between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_sinks(rng):
    kind = rng.choice(["token", "forward", "backward", "op", "op", "op", "grad2"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
    d = rng.choice([32, 64, 64, 80, 96, 128, 128])
    n_q = rng.choice([1, 1, 2, 7]) if kind == "token" else _log_between(rng, 64, 32768)
    if kind == "token":
        n_k = _log_between(rng, 16, 65536)
    elif rng.random() < 0.7:
        n_k = n_q                                   # self-attention
    else:
        n_k = n_q + _log_between(rng, 1, 8192)      # queries that continue a sequence
    n_k = max(n_k, n_q)
    if kind != "token" and rng.random() < 0.5:
        n_q, n_k = max(64, n_q // 64 * 64), max(64, n_k // 64 * 64)
    window = _log_between(rng, 32, 4096)
    sinks = rng.choice([1, 2, 4, 4, 4, 16, 64, 130])
    batch, heads = rng.choice([1, 1, 2, 4, 8]), rng.choice([1, 2, 4, 8, 12, 16, 32])
    layout = "bnhd" if rng.random() < 0.25 else "bhnd"
    c = _sinks(kind, dtype, batch, heads, n_q, n_k, d, window, sinks, layout, rng.choice([1.0, 0.1]))
    while True:                                     # no more than the largest listed case of its arithmetic
        w = work(c)
        if w["flops"] <= (8e11 if dtype != "fp32" else 3e11 if d <= 64 else 1e10) and _band(c) <= 5.5e8 and w["bytes"] < 1.2e9:
            return c
        if c["batch"] * c["heads"] > 1:
            c["batch" if c["batch"] > 1 else "heads"] //= 2
        else:
            c["n_q"], c["n_k"], c["window"] = max(1, c["n_q"] * 2 // 3), max(16, c["n_k"] * 2 // 3), max(32, c["window"] * 2 // 3)
            c["n_k"] = max(c["n_k"], c["n_q"])


def _draw_rotary(rng):
    kind, dtype = rng.choice(["apply", "step"]), rng.choice(["bf16", "bf16", "fp16", "fp32"])
    d = rng.choice([32, 64, 80, 96, 128, 128])
    pairs = d // 2 if rng.random() < 0.7 else max(4, d // 8 * 2)
    axes = rng.choice([1, 3, 3])
    n = 1 if rng.random() < 0.15 else _log_between(rng, 2, 32768)
    batch, heads = rng.choice([1, 1, 2, 4, 8]), rng.choice([1, 2, 4, 8, 12, 16, 32])
    c = _rotary(kind, dtype, batch, heads, rng.choice([1, heads, heads]), n, d, pairs, axes, rng.random() < 0.4,
                "bnhd" if rng.random() < 0.4 else "bhnd")
    while work(c)["bytes"] > 5.4e8:
        c["n"] = c["n"] * 2 // 3
    return c


def _draw_norm(rng):
    c = _norm(rng.choice(["forward", "step", "step", "grad2", "grad2"]), rng.choice(["bf16", "bf16", "fp16", "fp32"]),
              _log_between(rng, 1, 65536), _log_between(rng, 16, 16384))
    if rng.random() < 0.6:
        c["cols"] = max(16, c["cols"] // 64 * 64)
    while work(c)["bytes"] > 4.1e8:
        c["rows"] = c["rows"] * 2 // 3
    return c


def draw(rng):
    return rng.choice([_draw_sinks, _draw_sinks, _draw_rotary, _draw_norm])(rng)


# ---------------------------------------------------------------- what a pass cannot do without


def _block(c):
    """Query rows of a block of the plain form: as many as the window has keys, so that its band is about two windows wide."""
    return max(1, min(c["n_q"], max(64, c["window"])))


def _band(c):
    """Scores that the plain form of a case works on."""
    rows = -(-c["n_q"] // _block(c)) * _block(c)
    return c["batch"] * c["heads"] * rows * (_block(c) + c["window"] - 1 + c["sinks"])


def _pairs(c):
    """(query, key) pairs that the mask leaves visible, per head (n_k >= n_q)."""
    off, w, s = c["n_k"] - c["n_q"], c["window"], c["sinks"]
    near = max(0, min(c["n_q"], w - off))           # queries with i + off + 1 <= w see every key up to their own
    pairs = near * off + near * (near + 1) // 2
    # the others see w keys, and of the first s those that the window has left behind
    reach = off + near + 1 - w                      # keys in front of the first such query's window
    far = c["n_q"] - near
    short = max(0, min(far, s - reach))             # queries whose window still covers some of the first s
    return pairs + far * w + short * reach + short * (short - 1) // 2 + (far - short) * min(s, c["n_k"])


def work(case):
    c, es = case, DTYPES[case["dtype"]].itemsize
    if c["op"] == "rotary":
        x = c["batch"] * (c["heads"] + c["heads_k"]) * c["n"] * c["d"]
        passes = 2 if c["kind"] == "step" else 1
        return {"bytes": passes * 2 * x * es + 8 * c["axes"] * c["batch"] * c["n"], "flops": passes * 3 * x}
    if c["op"] == "norm":
        x, w = c["rows"] * c["cols"], c["cols"]
        moved = {"forward": 2 * x + 2 * w, "step": 4 * x + 4 * w, "grad2": 7 * x + 7 * w}[c["kind"]]
        return {"bytes": moved * es + (8 * c["rows"] if c["kind"] == "forward" else 0), "flops": {"forward": 7, "step": 18, "grad2": 50}[c["kind"]] * x}
    bh = c["batch"] * c["heads"]
    rows, q = bh * c["n_q"], bh * c["n_q"] * c["d"]
    # of the keys in front of every window only the first are needed
    seen = min(c["n_k"], c["n_q"] + c["window"] - 1 + c["sinks"])
    k = bh * seen * c["d"]
    k_out = bh * c["n_k"] * c["d"]
    pairs = 2 * bh * _pairs(c) * c["d"]
    if c["kind"] in ("token", "forward"):
        return {"bytes": (2 * q + 2 * k) * es + 4 * rows, "flops": 2 * pairs}
    if c["kind"] == "backward":
        return {"bytes": (4 * q + 2 * k + 2 * k_out) * es + 4 * rows, "flops": 5 * pairs}
    if c["kind"] == "op":
        return {"bytes": (6 * q + 4 * k + 2 * k_out) * es + 4 * rows, "flops": 12 * pairs}
    return {"bytes": (7 * q + 4 * k + 4 * k_out) * es, "flops": 19 * pairs}


# ---------------------------------------------------------------- inputs


def prepare(case, seed):
    """Activations N(0, 1), cotangents scaled; O and L saved from the forward, as training saves them."""
    c, dtype = case, DTYPES[case["dtype"]]
    g = torch.Generator(device="cuda").manual_seed(seed)
    leaf = c["kind"] in ("grad2", "step")

    def normal(*shape, mul=1.0, add=0.0):
        t = torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)
        return t.mul_(mul).add_(add).to(dtype)

    if c["op"] == "norm":
        s = {"case": c, "eps": 1e-5, "x": normal(c["rows"], c["cols"], mul=1.5, add=0.25), "w": normal(c["cols"], mul=0.2, add=1.0),
             "b": normal(c["cols"], mul=0.2)}
        if leaf:
            s["dy"] = normal(c["rows"], c["cols"])
        if c["kind"] == "grad2":
            s["v"], s["vw"], s["vb"] = normal(c["rows"], c["cols"]), normal(c["cols"], mul=0.1), normal(c["cols"], mul=0.1)
            s["dy"].requires_grad_(True)
        if leaf:
            for n in ("x", "w", "b"):
                s[n].requires_grad_(True)
        return s

    def heads(h, n, mul=1.0):
        if c["layout"] == "bnhd":
            return normal(c["batch"], n, h, c["d"], mul=mul).transpose(1, 2)
        return normal(c["batch"], h, n, c["d"], mul=mul)

    if c["op"] == "rotary":
        s = {"case": c, "q": heads(c["heads"], c["n"]), "k": heads(c["heads_k"], c["n"])}
        if leaf:
            s["dq"], s["dk"] = heads(c["heads"], c["n"]), heads(c["heads_k"], c["n"])
            s["q"].requires_grad_(True)
            s["k"].requires_grad_(True)
        # sequences that start anywhere in a long stream; several axes: rows and columns of frames of 32 x 32 patches
        start = torch.randint(0, 200000, (c["batch"], 1), generator=g, device="cuda")
        at = torch.arange(c["n"], device="cuda")[None]
        s["positions"] = (start + at)[None] if c["axes"] == 1 else torch.stack([start + at // 1024, at // 32 % 32 + 0 * start, at % 32 + 0 * start])
        s["frequencies"] = 10000.0 ** (-torch.arange(c["pairs"], device="cuda", dtype=torch.float64) / c["pairs"])
        time = c["pairs"] // 4
        side = (c["pairs"] - time) // 2
        s["axis_of_pair"] = (0,) * c["pairs"] if c["axes"] == 1 else (0,) * time + (1,) * side + (2,) * (c["pairs"] - time - side)
        return s

    mul = c["cotangent"]
    s = {"case": c, "scale": c["d"] ** -0.5, "q": heads(c["heads"], c["n_q"]), "k": heads(c["heads"], c["n_k"]), "v": heads(c["heads"], c["n_k"])}
    if c["kind"] in ("token", "forward"):
        return s
    s["d_o"] = heads(c["heads"], c["n_q"], mul)
    if c["kind"] != "backward":
        s["ddq"], s["ddk"], s["ddv"] = heads(c["heads"], c["n_q"], mul), heads(c["heads"], c["n_k"], mul), heads(c["heads"], c["n_k"], mul)
    if leaf:
        for n in ("q", "k", "v", "d_o"):
            s[n].requires_grad_(True)
        return s
    s["o"], s["lse"] = _rounded(_attention(s, "forward"), s)
    return s


# ---------------------------------------------------------------- plain forms, 32 bits


def _rounded(values, s):
    """Results in their shapes and types: rows (batch * heads, n, d) back to (batch, heads, n, d); a row vector stays in 32 bits."""
    c = s["case"]
    return tuple(v.reshape(c["batch"], c["heads"], *v.shape[1:]).to(DTYPES[c["dtype"]] if v.dim() == 3 else torch.float32) for v in values)


def _attention(s, kind):
    """O, L | dQ, dK, dV | the double backward's four, of queries in blocks against the first keys and a band of keys:
    (batch * heads, block, row, key) scores, of which the mask keeps the visible ones."""
    c = s["case"]
    rows, off, n_q, n_k, w = _block(c), c["n_k"] - c["n_q"], c["n_q"], c["n_k"], c["window"]
    blocks, first = -(-n_q // rows), min(c["sinks"], n_k)
    dev = s["q"].device
    i = torch.arange(blocks * rows, device=dev).view(blocks, rows, 1) + off
    band = torch.arange(rows + w - 1, device=dev) + (torch.arange(blocks, device=dev) * rows + off - w + 1).view(blocks, 1)
    key = torch.cat([torch.arange(first, device=dev).expand(blocks, first), band], 1)
    j = key.view(blocks, 1, -1)
    in_first = torch.arange(key.shape[1], device=dev) < first
    seen = (j <= i) & (in_first | ((j >= first) & (i - j < w))) & (j >= 0) & (j < n_k) & (i < n_q + off)
    key = key.clamp(0, n_k - 1)

    def q_side(t):
        t = t.detach().reshape(-1, n_q, c["d"]).float()
        return torch.nn.functional.pad(t, (0, 0, 0, blocks * rows - n_q)).view(t.shape[0], blocks, rows, c["d"])

    def k_side(t):
        return t.detach().reshape(-1, n_k, c["d"]).float()[:, key]

    def q_rows(t):
        return t.flatten(1, 2)[:, :n_q]

    def k_rows(t):
        return torch.zeros(t.shape[0], n_k, c["d"], device=dev).index_add_(1, key.flatten(), t.flatten(1, 2))

    scale = s["scale"]
    q, k, v = q_side(s["q"]), k_side(s["k"]), k_side(s["v"])
    score = (q @ k.mT * scale).masked_fill_(~seen, float("-inf"))
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    if kind == "forward":
        return q_rows(p @ v / total), q_rows(top + torch.log(total))[..., 0]
    p = p / total.clamp_min(1e-30)
    g = q_side(s["d_o"])
    dp = g @ v.mT
    d = (p * dp).sum(-1, keepdim=True)
    ds = scale * p * (dp - d)
    first_order = lambda: (q_rows(ds @ k), k_rows(ds.mT @ q), k_rows(p.mT @ g))  # noqa: E731
    if kind == "backward":
        return first_order()
    ddq, ddk, ddv = q_side(s["ddq"]), k_side(s["ddk"]), k_side(s["ddv"])
    dds = scale * (ddq @ k.mT + q @ ddk.mT)
    x = g @ ddv.mT
    dd = (dds * p).sum(-1, keepdim=True)
    ddp = p * (dds - dd)
    dp2 = x + dp * (dds - dd) - d * dds
    b = (dp2 * p).sum(-1, keepdim=True)
    ds2 = scale * p * (dp2 - b)
    second = q_rows(ds @ ddk + ds2 @ k), k_rows(ds.mT @ ddq + ds2.mT @ q), k_rows(ddp.mT @ g), q_rows(ddp @ v + p @ ddv)
    return second if kind == "op" else (q_rows(p @ v), *first_order(), *second)


def _rotated(x, s, sign):
    c, axis = s["case"], torch.tensor(s["axis_of_pair"], device=x.device)
    angle = (s["positions"][axis].double() * s["frequencies"].view(-1, 1, 1)).permute(1, 2, 0)[:, None]
    cos, sin = angle.cos().float(), sign * angle.sin().float()
    n = c["pairs"]
    turned = x.detach()[..., :2 * n].float()
    a, b = (turned[..., 0::2], turned[..., 1::2]) if c["interleaved"] else (turned[..., :n], turned[..., n:])
    pair = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack(pair, -1).flatten(-2) if c["interleaved"] else torch.cat(pair, -1)
    return torch.cat([turned.to(x.dtype), x.detach()[..., 2 * n:]], -1)


def _layer_norm(s):
    c = s["case"]
    x, w, bias = s["x"].detach().float(), s["w"].detach().float(), s["b"].detach().float()
    mean = x.mean(-1, keepdim=True)
    r = 1.0 / torch.sqrt((x - mean).square().mean(-1, keepdim=True) + s["eps"])
    h = (x - mean) * r
    y = (h * w + bias).to(s["x"].dtype)
    if c["kind"] == "forward":
        return y, mean[:, 0], r[:, 0]

    def avg(t):
        return t.mean(-1, keepdim=True)

    dy = s["dy"].detach().float()
    g = dy * w
    first = r * (g - avg(g) - h * avg(g * h)), (dy * h).sum(0), dy.sum(0)
    if c["kind"] == "step":
        return (y, *(t.to(y.dtype) for t in first))
    v, vw, vb = s["v"].float(), s["vw"].float(), s["vb"].float()
    p = r * (v - avg(v) - h * avg(v * h))
    e = vw * dy - r * (g * avg(v * h) + v * avg(g * h))
    dx2 = r * (e - avg(e) - h * avg(e * h)) - r * r * h * (avg(v * g) - avg(v) * avg(g) - avg(g * h) * avg(v * h))
    return (y, *(t.to(y.dtype) for t in (*first, dx2, (dy * p).sum(0), w * p + vw * h + vb)))


# ---------------------------------------------------------------- one pass


def run(state):
    s, c = state, state["case"]
    if own:
        return _own(s)
    if c["op"] == "norm":
        return _layer_norm(s)
    if c["op"] == "rotary":
        out = _rotated(s["q"], s, 1.0), _rotated(s["k"], s, 1.0)
        return out if c["kind"] == "apply" else (*out, _rotated(s["dq"], s, -1.0), _rotated(s["dk"], s, -1.0))
    return _rounded(_attention(s, "forward" if c["kind"] == "token" else c["kind"]), s)


def _own(s):
    fhob, c = _fhob(), s["case"]
    if c["op"] == "norm":
        if c["kind"] == "forward":
            return fhob.layer_norm_forward(s["x"], s["w"], s["b"], s["eps"])
        y = fhob.layer_norm(s["x"], s["w"], s["b"], s["eps"])
        first = torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"], create_graph=c["kind"] == "grad2")
        if c["kind"] == "step":
            return (y, *first)
        return (y, *first, *torch.autograd.grad(first, (s["x"], s["w"], s["dy"]), (s["v"], s["vw"], s["vb"])))
    if c["op"] == "rotary":
        q, k = fhob.rotary((s["q"], s["k"]), s["positions"], s["frequencies"], s["axis_of_pair"], interleaved=c["interleaved"])
        return (q, k) if c["kind"] == "apply" else (q, k, *torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"])))
    mask = {"is_causal": True, "sliding_window": c["window"], "sink_tokens": c["sinks"]}
    if c["kind"] in ("token", "forward"):
        return fhob.attention_forward(s["q"], s["k"], s["v"], s["scale"], **mask)
    if c["kind"] == "backward":
        return fhob.attention_backward(s["q"], s["k"], s["v"], s["o"], s["d_o"], s["lse"], s["scale"], **mask)
    if c["kind"] == "op":
        return fhob.flash_bwdbwd(s["q"], s["k"], s["v"], s["o"], s["d_o"], s["ddq"], s["ddk"], s["ddv"], s["lse"], s["scale"], **mask)
    o = fhob.attention(s["q"], s["k"], s["v"], s["scale"], **mask)
    first = torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["d_o"], create_graph=True)
    return (o, *first, *torch.autograd.grad(first, (s["q"], s["k"], s["v"], s["d_o"]), (s["ddq"], s["ddk"], s["ddv"])))


# ---------------------------------------------------------------- 64 bits, from the definitions


def exact(case, seed):
    """The first and second derivatives are taken of the definition by autograd, a slab of query rows at a time: what
    every slab adds to the gradients of shared keys is summed."""
    c, s = case, prepare(case, seed)
    if c["op"] == "norm":
        x, w, bias = (s[n].detach().double().requires_grad_(True) for n in ("x", "w", "b"))
        var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
        y = (x - mean) * (var + s["eps"]).rsqrt() * w + bias
        if c["kind"] == "forward":
            return y.detach(), mean.detach()[:, 0], (var + s["eps"]).rsqrt().detach()[:, 0]
        dy = s["dy"].detach().double().requires_grad_(True)
        first = torch.autograd.grad(y, (x, w, bias), dy, create_graph=True)
        out = [y, *first]
        if c["kind"] == "grad2":
            out += torch.autograd.grad(first, (x, w, dy), (s["v"].double(), s["vw"].double(), s["vb"].double()))
        return [t.detach() for t in out]

    if c["op"] == "rotary":
        def turned(t, sign):
            z = t.detach().double().clone()
            for n, axis in enumerate(s["axis_of_pair"]):
                at = (2 * n, 2 * n + 1) if c["interleaved"] else (n, n + c["pairs"])
                angle = sign * s["positions"][axis].double()[:, None] * s["frequencies"][n]
                unit = torch.complex(z[..., at[0]], z[..., at[1]]) * torch.polar(torch.ones_like(angle), angle)
                z[..., at[0]], z[..., at[1]] = unit.real, unit.imag
            return z
        out = [turned(s["q"], 1), turned(s["k"], 1)]
        return out if c["kind"] == "apply" else out + [turned(s["dq"], -1), turned(s["dk"], -1)]

    heads = c["batch"] * c["heads"]
    t = {n: x.detach().double().reshape(heads, -1, c["d"]) for n, x in s.items() if isinstance(x, torch.Tensor) and x.dim() == 4}
    n_q, n_k, w, off = c["n_q"], c["n_k"], c["window"], c["n_k"] - c["n_q"]
    zeros = {n: torch.zeros_like(t[n]) for n in ("q", "k", "v")}
    o, lse = torch.zeros_like(t["q"]), torch.zeros(heads, n_q, dtype=torch.float64, device="cuda")
    grad, grad2, ddo = zeros, {n: torch.zeros_like(x) for n, x in zeros.items()}, torch.zeros_like(o)
    slab = max(1, min(256, int(2e8 / (heads * (w + 256 + c["sinks"])))))
    for lo in range(0, n_q, slab):
        hi = min(n_q, lo + slab)
        near = torch.arange(max(0, lo + off - w + 1), hi + off, device="cuda")
        keys = torch.cat([torch.arange(min(c["sinks"], int(near[0])), device="cuda"), near])
        back = torch.arange(lo + off, hi + off, device="cuda")[:, None] - keys[None]
        visible = (back >= 0) & ((back < w) | (keys[None] < c["sinks"]))
        q, k, v = (x.clone().requires_grad_(True) for x in (t["q"][:, lo:hi], t["k"][:, keys], t["v"][:, keys]))
        score = torch.where(visible, torch.einsum("bqd,bkd->bqk", q, k) * s["scale"], float("-inf"))
        weight = torch.softmax(score, -1)
        out = torch.einsum("bqk,bkd->bqd", weight, v)
        o[:, lo:hi], lse[:, lo:hi] = out.detach(), torch.logsumexp(score.detach(), -1)
        if c["kind"] in ("token", "forward"):
            continue
        d_o = t["d_o"][:, lo:hi].clone().requires_grad_(True)
        first = torch.autograd.grad(out, (q, k, v), d_o, create_graph=True)
        grad["q"][:, lo:hi] += first[0].detach()
        grad["k"].index_add_(1, keys, first[1].detach())
        grad["v"].index_add_(1, keys, first[2].detach())
        if c["kind"] == "backward":
            continue
        second = torch.autograd.grad(first, (q, k, v, d_o), (t["ddq"][:, lo:hi], t["ddk"][:, keys], t["ddv"][:, keys]))
        grad2["q"][:, lo:hi] += second[0]
        grad2["k"].index_add_(1, keys, second[1])
        grad2["v"].index_add_(1, keys, second[2])
        ddo[:, lo:hi] = second[3]
    first, second = [grad["q"], grad["k"], grad["v"]], [grad2["q"], grad2["k"], grad2["v"], ddo]
    out = {"token": [o, lse], "forward": [o, lse], "backward": first, "op": second, "grad2": [o, *first, *second]}[c["kind"]]
    return [x.reshape(c["batch"], c["heads"], *x.shape[1:]) for x in out]
