"""Attention with first tokens at the edges of what is allowed: refusals, long caches."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

import fhob
from fhob import _lib
from test_sink_attention import dense


def test_c_refuses_first_keys_without_a_causal_mask():
    """Whatever the lengths: also where first keys and window together reach every key."""
    lib = _lib.load()
    p = _lib.FhobProblem()
    p.bh, p.n_q, p.d, p.causal, p.window = 1, 128, 64, 0, 50
    for n in ("q", "k", "v", "o", "d_o", "ddq", "ddk", "ddv", "lse", "dq2", "dk2", "dv2", "ddo", "workspace"):
        setattr(p, n, 4096)
    p.workspace_bytes = 1 << 20
    for causal in (0, 2):
        p.causal = causal
        for n_k in (128, 150, 151, 1000):
            p.n_k = n_k
            for sinks in (1, 100, 2 ** 31 - 1):
                assert lib.fhob_forward_sinks(C.byref(p), sinks, 4096, 4096, None) == 1, (causal, n_k, sinks)
                assert lib.fhob_backward_sinks(C.byref(p), sinks, 4096, 4096, 4096, None) == 1
                assert lib.fhob_bwdbwd_sinks(C.byref(p), sinks, None) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("nq", [1, 2])
def test_one_or_two_queries_behind_32_bits(nq):
    """One head of 2^25 + 300 keys of 64: the first keys and the window are 2^31 elements apart.  The kernel for few queries goes through the
    same keys in the same order in either cache: the same bits."""
    nk, window, sinks = 2 ** 25 + 300, 60, 4
    g = torch.Generator(device="cuda").manual_seed(nq)
    q, k, v = (torch.randn(1, n, 64, generator=g, device="cuda", dtype=torch.bfloat16) for n in (nq, 104, 104))
    kw = dict(is_causal=True, sliding_window=window, sink_tokens=sinks)
    want = fhob.attention_forward(q, k, v, 0.125, check=True, **kw)
    big = [torch.zeros(1, nk, 64, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    for b, part in zip(big, (k, v)):
        b[:, :4], b[:, -100:] = part[:, :4], part[:, 4:]
    got = fhob.attention_forward(q, *big, 0.125, check=True, **kw)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del got
    ref = dense({"q": q, "k": k, "v": v, "do": q, "ddq": q, "ddk": k, "ddv": v}, 0.125, window, sinks)[0]
    assert float((want[0].double() - ref).abs().max()) < 2e-2 * float(ref.abs().max())
