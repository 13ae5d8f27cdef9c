"""Masks of problems without any work."""
from __future__ import annotations

import pytest
import torch

import fhob


def test_empty_problems_take_any_mask():
    """Without queries or keys there is nothing that a window could hide: the zeros come whatever the mask's numbers are."""
    q, k, v = torch.ones(2, 16, 64), torch.ones(2, 0, 64), torch.ones(2, 0, 32)
    args = (q, k, v, torch.zeros(2, 16, 32), torch.ones(2, 16, 32), torch.zeros(2, 16), 0.125)
    for kw in (dict(sliding_window=3), dict(is_causal=True, sliding_window=0)):
        dq, dk, dv = fhob.attention_backward(*args, **kw)
        assert dq.shape == q.shape and dk.shape == k.shape and dv.shape == v.shape and not dq.any()
    for kw in (dict(sink_tokens=3), dict(is_causal=True, sliding_window=3, sink_tokens=-1)):   # new numbers are checked
        with pytest.raises(ValueError):
            fhob.attention_backward(*args, **kw)


@pytest.mark.gpu
def test_forward_of_empty_problems_takes_any_mask():
    q, k = torch.ones(2, 16, 64, device="cuda"), torch.ones(2, 0, 64, device="cuda")
    o, lse = fhob.attention_forward(q, k, k, 0.125, sliding_window=3)
    assert o.shape == q.shape and not o.any() and torch.isinf(lse).all()
