"""The largest windows: any number up to 2^31 - 1 that reaches the first key is the causal mask."""
from __future__ import annotations

import pytest
import torch

import fhob
from conftest import make_inputs


def all_results(x, scale, impl, **kw):
    kw = dict(is_causal=True, impl=impl, **kw)
    o, lse = fhob.attention_forward(x["q"], x["k"], x["v"], scale, **kw)
    first = fhob.attention_backward(x["q"], x["k"], x["v"], o, x["do"], lse, scale, **kw)
    second = fhob.flash_bwdbwd(x["q"], x["k"], x["v"], o, x["do"], x["ddq"], x["ddk"], x["ddv"], lse, scale, **kw)
    return (o, lse, *first, *second, fhob.produce_L(x["q"], x["k"], True, scale, kw.get("sliding_window")))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,impl", [(torch.bfloat16, "auto"), (torch.float32, "auto"), (torch.bfloat16, "simt")])
@pytest.mark.parametrize("nq,nk", [(300, 300), (200, 333), (333, 200)])
def test_windows_that_hide_nothing(nq, nk, dtype, impl):
    """Masks of the same pairs."""
    x = make_inputs(2, nq, nk, 64, seed=nq, dtype=dtype, device="cuda")
    tol = 2e-2 if dtype == torch.bfloat16 else 1e-4   # the bounds of the other parity tests
    want = all_results(x, 0.125, impl)
    for window in (max(nq, nk), 2 ** 30, 2 ** 31 - 300, 2 ** 31 - 2, 2 ** 31 - 1):
        for sinks in (0, 5):
            for i, (a, b) in enumerate(zip(all_results(x, 0.125, impl, sliding_window=window, sink_tokens=sinks), want)):
                dead = torch.isinf(b)
                assert torch.equal(torch.isinf(a), dead), (window, sinks, i)
                err = float((a.double() - b.double())[~dead].abs().max()) / float(b[~dead].abs().max())
                assert err < tol, (window, sinks, i, err)
    args = (x["q"], x["k"], x["v"])
    for window in (2 ** 31 - 1, nk):   # host tensors
        o, lse = fhob.attention_forward(*args, 0.125, is_causal=True)
        host = fhob.flash_bwdbwd(*(t.cpu() for t in (*args, o, x["do"], x["ddq"], x["ddk"], x["ddv"], lse)), 0.125, is_causal=True, sliding_window=window)
        for a, b in zip(host, want[5:9]):
            assert float((a.double() - b.double().cpu()).abs().max()) < tol * float(b.abs().max())
