"""fhob.rotary against complex arithmetic in 64 bits.

Error bound of an element.  The fp32 angle is off by at most pi 2^-25 (its rounding; the integer product in front is
exact to position * frequency * 2^-52), sincospif by 2 steps of 2^-24, and the two products and their sum
round to 2^-24 each: (|x| + |y|) * 2^-21 covers them all.  Storing the result rounds by at most half a step.
"""
from __future__ import annotations

import ctypes as C

import pytest
import torch

import fhob
from fhob import _lib

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def plain(x, positions, frequencies, axes, interleaved, inverse=False):
    """(B, H, N, D) in 64 bits, and the size |x| + |y| of every element's pair."""
    x, n = x.double(), len(frequencies)
    out, size = x.clone(), x.abs()
    pos = positions if positions.dim() == 3 else positions[:, None]
    for j in range(n):
        a, b = (2 * j, 2 * j + 1) if interleaved else (j, n + j)
        angle = pos[axes[j]].double()[:, None] * float(frequencies[j]) * (-1.0 if inverse else 1.0)
        z = torch.complex(x[..., a], x[..., b]) * torch.polar(torch.ones_like(angle), angle)
        out[..., a], out[..., b] = z.real, z.imag
        size[..., a] = size[..., b] = x[..., a].abs() + x[..., b].abs()
    return out, size


def close(got, ref, size):
    half = torch.finfo(got.dtype).eps / 2
    fp32 = size * 2.0 ** -21
    bad = (got.double() - ref).abs() > fp32 + (ref.abs() + fp32) * half
    if got.dtype == torch.float16:
        bad &= (got.double() - ref).abs() > 2.0 ** -25   # below 2^-14 fp16's steps are 2^-24
    return not bool(bad.any())


def make(batch, heads, n, d, dtype, seed=0, bnhd=False):
    g = torch.Generator().manual_seed(seed)
    shape = (batch, n, heads, d) if bnhd else (batch, heads, n, d)
    t = torch.randn(shape, generator=g).to(DTYPES[dtype]).cuda()
    return t.transpose(1, 2) if bnhd else t


def places(axes, batch, n, seed=0, far=1 << 20):
    return torch.randint(0, far, (axes, batch, n), generator=torch.Generator().manual_seed(seed)).cuda()


CASES = [  # dtype, batch, heads, heads_k, n, d, pairs, axes, interleaved
    ("bf16", 2, 4, 2, 33, 128, 64, 3, False), ("bf16", 2, 4, 2, 33, 128, 64, 3, True), ("bf16", 1, 1, 1, 1, 64, 32, 1, False),
    ("fp16", 3, 17, 1, 5, 80, 20, 2, False), ("fp16", 1, 5, 5, 7, 80, 20, 2, True), ("fp32", 2, 3, 3, 65, 96, 48, 3, False),
    ("fp32", 1, 2, 1, 9, 64, 32, 1, True), ("bf16", 1, 3, 2, 11, 7, 3, 2, False), ("bf16", 1, 3, 2, 11, 7, 3, 2, True),
    ("fp32", 2, 2, 2, 3, 5, 2, 1, False), ("fp32", 1, 2, 2, 3, 5, 1, 1, True), ("bf16", 1, 2, 2, 300, 1024, 512, 3, False),
    ("fp32", 1, 2, 2, 3, 1021, 510, 3, True), ("bf16", 1, 40, 3, 700, 64, 16, 3, False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("bnhd", [False, True])
@pytest.mark.parametrize("dtype,batch,heads,heads_k,n,d,pairs,axes,interleaved", CASES)
def test_forward_and_inverse(dtype, batch, heads, heads_k, n, d, pairs, axes, interleaved, bnhd):
    q, k = make(batch, heads, n, d, dtype, 1, bnhd), make(batch, heads_k, n, d, dtype, 2, bnhd)
    pos, freq = places(axes, batch, n), 10000.0 ** (-torch.arange(pairs, device="cuda", dtype=torch.float64) / pairs)
    axis = [j % axes for j in range(pairs)]
    for inverse in (False, True):
        got = fhob.rotary((q, k), pos, freq, axis, interleaved=interleaved, inverse=inverse)
        for x, y in zip((q, k), got):
            assert y.is_contiguous() and y.dtype == x.dtype and y.shape == x.shape
            assert close(y, *plain(x, pos, freq, axis, interleaved, inverse))
            assert torch.equal(y[..., 2 * pairs:], x[..., 2 * pairs:])
        assert torch.equal(fhob.rotary(k, pos, freq, axis, interleaved=interleaved, inverse=inverse), got[1])   # alone: the same bits


@pytest.mark.gpu
@pytest.mark.parametrize("far", [2 ** 31 - 1, 2 ** 40])
def test_far_positions(far):
    """In fp32 the product of position and frequency would be off by radians here."""
    x = make(1, 2, 6, 32, "fp32")
    pos = torch.tensor([[far, far - 1, -far, 0, 1, -1]], device="cuda")
    freq = torch.tensor([1.0, 0.9, 3.0, -0.7, 7.0, 1e-3, 1e-7, 0.0] * 2, device="cuda", dtype=torch.float64)
    got = fhob.rotary(x, pos, freq)
    ref, size = plain(x, pos, freq, [0] * 16, False)
    # the angle in doubles, of the kernel and here: position * frequency * 2^-52 each
    slack = 2 * far * 7.0 * 2.0 ** -52
    assert bool(((got.double() - ref).abs() <= size * (2.0 ** -21 + slack) + ref.abs() * 2.0 ** -24).all())


@pytest.mark.gpu
def test_argument_forms():
    x, freq = make(2, 3, 8, 64, "bf16"), torch.rand(32, device="cuda", dtype=torch.float64)
    pos = places(1, 2, 8)
    want = fhob.rotary(x, pos, freq)
    assert torch.equal(fhob.rotary(x, pos.int(), freq), want)
    shared = pos[:, :1]
    assert torch.equal(fhob.rotary(x, shared, freq), fhob.rotary(x, shared[:, 0], freq))
    assert torch.equal(fhob.rotary(x[1], pos[:, 1], freq), want[1])                       # (H, N, D)
    assert torch.equal(fhob.rotary(x, pos, freq.float()), fhob.rotary(x, pos, freq.float().double()))
    assert torch.equal(fhob.rotary(x, pos.transpose(1, 2).contiguous().transpose(1, 2), freq), want)
    assert torch.equal(fhob.rotary(x, pos, torch.stack([freq, freq], 1)[:, 0]), want)
    wide = torch.zeros(2, 3, 8, 67, device="cuda", dtype=x.dtype)
    wide[..., 3:] = x
    assert torch.equal(fhob.rotary(wide[..., 3:], pos, freq), want)                       # rows off the 16-byte grid
    assert torch.equal(fhob.rotary(x.transpose(2, 3).contiguous().transpose(2, 3), pos, freq), want)   # copied first
    one = x[:, :1].expand(2, 3, 8, 64)                                                    # heads of stride 0
    assert torch.equal(fhob.rotary(one, pos, freq), fhob.rotary(one.contiguous(), pos, freq))
    assert fhob.rotary(x[:, :, :0], pos[..., :0], freq).shape == (2, 3, 0, 64)
    assert fhob.rotary((x[:0], x[:0, :0]), pos[:, :0], freq)[1].shape == (0, 0, 8, 64)


@pytest.mark.gpu
def test_nan_and_infinity_stay_in_their_pair():
    x = make(1, 1, 4, 16, "fp32")
    x[0, 0, 1, 3], x[0, 0, 2, 5] = float("nan"), float("inf")
    got = fhob.rotary(x, places(1, 1, 4), torch.rand(8, device="cuda", dtype=torch.float64))
    bad = ~torch.isfinite(got)
    want = torch.zeros_like(bad)
    want[0, 0, 1, [3, 11]] = want[0, 0, 2, [5, 13]] = True
    assert torch.equal(bad, want)


@pytest.mark.gpu
def test_derivatives():
    """The backward pass is the inverse rotation; differences of the (linear) function agree; so does the second backward."""
    q, k = (make(1, h, 20, 64, "fp32", h).requires_grad_(True) for h in (4, 2))
    pos, freq = places(2, 1, 20), torch.rand(32, device="cuda", dtype=torch.float64)
    axis = [0, 1] * 16
    rope = lambda *x: fhob.rotary(x, pos, freq, axis)   # noqa: E731
    oq, ok = rope(q, k)
    gq, gk = torch.randn_like(oq).requires_grad_(True), torch.randn_like(ok).requires_grad_(True)
    dq, dk = torch.autograd.grad((oq, ok), (q, k), (gq, gk), create_graph=True)
    for d, g in ((dq, gq), (dk, gk)):
        assert close(d, *plain(g.detach(), pos, freq, axis, False, inverse=True))
    v = torch.randn_like(q)
    difference = ((rope(q + v, k)[0] - rope(q - v, k)[0]) / 2 * gq).double().sum()
    assert abs(float((difference - (dq * v).double().sum()).detach())) <= 2.0 ** -20 * float((gq.abs() * (q.abs() + v.abs())).detach().double().sum()) * 4
    uq, uk = torch.randn_like(q), torch.randn_like(k)
    ddq, ddk = torch.autograd.grad((dq, dk), (gq, gk), (uq, uk))
    assert torch.equal(ddq, rope(uq, uk)[0]) and torch.equal(ddk, rope(uq, uk)[1])
    # one result alone, and a gradient that is a view
    (dk2,) = torch.autograd.grad(rope(q, k)[1], k, gk.detach())
    assert torch.equal(dk2, dk)
    assert torch.autograd.grad(rope(q, k)[0].sum(), q)[0].shape == q.shape
    with torch.no_grad():
        assert not rope(q, k)[0].requires_grad


@pytest.mark.gpu
def test_streams_and_graphs():
    x, freq, pos = make(2, 8, 100, 128, "bf16"), torch.rand(64, device="cuda", dtype=torch.float64), places(1, 2, 100)
    want = fhob.rotary(x, pos, freq)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = fhob.rotary(x, pos, freq)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = fhob.rotary(x, pos, freq)
    pos2 = pos + 5
    x.mul_(2.0)
    pos.copy_(pos2)
    graph.replay()
    assert torch.equal(captured, fhob.rotary(x, pos2, freq))


def test_refusals():
    """Before anything is launched; on the CPU, so none of these reaches a device."""
    x, pos, freq = torch.zeros(2, 3, 8, 64), torch.zeros(1, 2, 8, dtype=torch.long), torch.zeros(32)
    for error, args in [
        (ValueError, (x, pos, freq)),                                        # not on a GPU
        (TypeError, (3, pos, freq)), (TypeError, (x, 3, freq)), (TypeError, (x, pos, None)),
        (TypeError, (x.double(), pos, freq)), (TypeError, (x, pos.float(), freq)), (TypeError, (x, pos, freq.int())),
        (ValueError, ((x, x, x), pos, freq)), (ValueError, ((), pos, freq)), (ValueError, (x[0, 0], pos, freq)),
        (ValueError, ((x, x[..., :32]), pos, freq)), (ValueError, ((x, x[:, :, :4]), pos, freq)), (ValueError, ((x, x[:1]), pos, freq)),
        (TypeError, ((x, x.bfloat16()), pos, freq)), (ValueError, ((x, x[0]), pos, freq)),
        (ValueError, (x, pos[..., :7], freq)), (ValueError, (x, pos[0, 0], freq)), (ValueError, (x, pos.expand(1, 2, 8)[:, :0], freq)),
        (ValueError, (x, pos, torch.zeros(33))), (ValueError, (x, pos, torch.zeros(0))), (ValueError, (x, pos, torch.zeros(4, 4))),
        (ValueError, (x, pos.expand(2, 2, 8), freq)),                        # several axes and no axis_of_pair
        (ValueError, (x, pos, freq, [0] * 31)), (ValueError, (x, pos, freq, [1] * 32)), (ValueError, (x, pos, freq, [-1] * 32)),
        (TypeError, (x, pos, freq, [0.5] * 32)), (TypeError, (x, pos, freq, 0)), (ValueError, (x, pos, freq, [])),
        (ValueError, (torch.zeros(1, 2, 1026), torch.zeros(1, 2, dtype=torch.long), freq)),
        (ValueError, (x, pos, freq.clone().requires_grad_(True))),
    ]:
        with pytest.raises(error):
            fhob.rotary(*args)


def test_c_refusals():
    lib = _lib.load()
    axes = (C.c_uint8 * 512)()

    def call(**over):
        r = _lib.FhobRotary()
        r.dtype, r.tensors, r.batch, r.n, r.d, r.pairs, r.axes = 0, 1, 1, 4, 64, 32, 1
        setattr(r.tensor[0], "in", 256)
        r.tensor[0].out, r.tensor[0].heads = 512, 1
        r.positions, r.frequencies, r.axis_of_pair = 1024, 2048, axes
        for n, v in over.items():
            setattr(r, n, v)
        return lib.fhob_rotary(C.byref(r), None)

    assert lib.fhob_rotary(None, None) == 1
    for over, status in [({"tensors": 0}, 1), ({"tensors": 3}, 1), ({"tensors": 2}, 1), ({"batch": 0}, 1), ({"n": -1}, 1), ({"pairs": 0}, 1),
                         ({"pairs": 33}, 2), ({"d": 1025}, 2), ({"dtype": 7}, 1), ({"positions": None}, 1), ({"frequencies": None}, 1),
                         ({"axes": 0}, 1)]:
        assert call(**over) == status, over
    axes[5] = 1
    assert call() == 1


def test_structs_match_header():
    import re
    from conftest import ROOT
    header = (ROOT / "include" / "fhob.h").read_text()
    for cls in (_lib.FhobRotaryTensor, _lib.FhobRotary, _lib.FhobLayerNorm):
        body = header.split(f"typedef struct {cls.__name__} {{")[1].split(f"}} {cls.__name__};")[0]
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        names = [re.sub(r"\[.*?\]", "", n).replace("*", "").split()[-1] for line in body.split(";") if line.strip() for n in line.split(",")]
        assert names == [f[0] for f in cls._fields_], cls.__name__


def test_c_refuses_misplaced_vectors():
    lib = _lib.load()
    axes = (C.c_uint8 * 512)()
    for positions, frequencies, wide in ((1026, 2048, 0), (1024, 2050, 0), (1028, 2048, 1), (1024, 2052, 1)):
        r = _lib.FhobRotary()
        r.dtype, r.tensors, r.batch, r.n, r.d, r.pairs, r.axes, r.axis_of_pair = 0, 1, 1, 4, 64, 32, 1, axes
        setattr(r.tensor[0], "in", 256)
        r.tensor[0].out, r.tensor[0].heads = 512, 1
        r.positions, r.frequencies, r.positions_are_64_bit, r.frequencies_are_64_bit = positions, frequencies, wide, wide
        assert lib.fhob_rotary(C.byref(r), None) == 3
