"""fp32 attention with first keys keeps fp32 throughout unless the caller asks for the tensor cores."""
from __future__ import annotations

import pytest
import torch

import fhob
from conftest import make_inputs
from test_sink_attention import NAMES, dense, ours


@pytest.mark.gpu
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("nq,nk,window,sinks", [(700, 700, 100, 4), (5, 900, 300, 64), (2, 900, 300, 4), (1500, 1800, 400, 130)])
def test_errors(nq, nk, window, sinks, d):
    """2-norm errors of at most 3e-6.  Scores are sums of d <= 128 products, 16 or fewer terms one behind the other in four to eight lanes or in
    packed halves: (16 + 8) * 2^-24 = 1.4e-6 of a score's size if every rounding had the same sign, about a fifth of it as a 2-norm, and an
    exponential passes on the absolute error of scores of size one to four: 1.2e-6.  The sums over keys or queries have 2^-24 of
    their running sum for each of up to 1800 / 2 terms, of which random signs leave 30: 30 * 2^-24 = 1.8e-6 at most.  bf16 pairs (2^-17 an operand: 7.6e-6)
    exceed this."""
    x = make_inputs(2, nq, nk, d, seed=d, dtype=torch.float32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    x = {n: t + 1e-3 * torch.randn(t.shape, generator=g, device="cuda") for n, t in x.items()}   # values that bf16 does not hold
    got, ref = ours(x, d ** -0.5, window, sinks), dense(x, d ** -0.5, window, sinks)
    for n, a, b in zip(NAMES, got, ref):
        err = float((a.reshape(b.shape).double() - b).norm() / b.norm())
        assert err < 3e-6, (n, err)
    # without O: the same logsumexp; views: the same bits as of their copies
    views = [t.view(1, 2, *t.shape[1:]).transpose(1, 2).contiguous().transpose(1, 2) for t in (x["q"], x["k"], x["v"])]
    kw = dict(is_causal=True, sliding_window=window, sink_tokens=sinks)
    o, lse = fhob.attention_forward(*views, d ** -0.5, **kw)
    assert torch.equal(o.reshape(got[0].shape), got[0]) and torch.equal(lse.reshape(got[1].shape), got[1])
    err = float((fhob.produce_L(x["q"], x["k"], True, d ** -0.5, window, sinks).double() - ref[1]).norm() / ref[1].norm())
    assert err < 3e-6, err
