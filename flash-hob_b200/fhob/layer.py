"""What a twice-differentiable layer runs around its attention: rotary positions and layer norm.

Both run on kernels of the library (csrc/rotary.cu, csrc/layer_norm.cu; the checks and the autograd functions are
native, csrc/host_layer.cpp).  The reference has no counterpart of either.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Sequence

import torch

from .ops import _native


class RotaryPositions(NamedTuple):
    """What ``rotary`` needs besides the tensors, for ``fhob.attention(..., rotary=...)``: ``positions`` are the keys'."""
    positions: torch.Tensor
    frequencies: torch.Tensor
    axis_of_pair: Optional[Sequence[int]] = None
    interleaved: bool = False


def rotary(x, positions, frequencies, axis_of_pair=None, *, interleaved: bool = False, inverse: bool = False):
    """Rotary positions with one or several axes (time, height, width), differentiable any number of times.

    ``x`` is a CUDA bfloat16, float16 or float32 tensor ``(B, H, N, D)`` or ``(H, N, D)``, or a tuple of one or two
    of them that differ in their heads only (queries and keys: one launch).  Returns new contiguous tensors.
    The first ``2 * len(frequencies)`` elements of a row are pairs, ``(j, len(frequencies) + j)`` or, if
    ``interleaved``, ``(2j, 2j + 1)``; pair ``j`` turns by ``positions[axis_of_pair[j]] * frequencies[j]`` radians
    (``inverse``: by the negative of that), the other elements are copied.

    ``positions`` are int32 or int64 on the same device, ``(axes, N)`` or ``(axes, B, N)``: any integers.  The angle is good to
    ``position * frequency * 2^-52`` radians, a millionth where that product is 2^32 (near 2^52 it says nothing; an fp32 product is off
    by a radian at 2^24).  ``frequencies`` is a float32 or float64 vector on the
    device, finite and regarded as constant.  ``axis_of_pair`` is a sequence with the axis of every pair; it may be left out
    when there is one axis.
    """
    several = isinstance(x, (tuple, list))
    out = _native().rotary(tuple(x) if several else (x,), positions, frequencies, axis_of_pair, interleaved, inverse)
    return out if several else out[0]


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5):
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dim, differentiable twice (``create_graph=True``).

    ``x`` is a CUDA bfloat16, float16 or float32 tensor with a last dim of up to 16384; ``weight`` and ``bias`` are
    vectors of its dtype or float32 (the same for both) or None.  Sums are fp32.  A third derivative raises.
    """
    return _native().layer_norm(x, weight, bias, eps)


def layer_norm_forward(x, weight=None, bias=None, eps: float = 1e-5):
    """Returns ``(y, mean, rstd)``: the result and the fp32 statistics that the two calls below take (no graph)."""
    return _native().layer_norm_forward(x, weight, bias, eps)


def layer_norm_backward(dy, x, weight, mean, rstd, *, need_db: bool = True):
    """First backward: ``(dx, dweight, dbias)``, ``dweight`` None without a weight, ``dbias`` None unless ``need_db``."""
    return _native().layer_norm_backward(dy, x, weight, mean, rstd, need_db)


def layer_norm_bwdbwd(ddx, ddw, ddb, dy, x, weight, mean, rstd):
    """Double backward: from the cotangents of dx, dweight and dbias (any may be None) the gradients of dy, x and weight,
    ``(ddy, dx2, dw2)``, with mean and rstd regarded as functions of x; ``dw2`` is None without a weight."""
    return _native().layer_norm_bwdbwd(ddx, ddw, ddb, dy, x, weight, mean, rstd)
