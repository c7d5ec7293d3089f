"""Calls under something that rewrites, traces or differentiates them another way (torch.jit.trace, make_fx, vmap,
forward-mode AD): an op goes through its registered form, or refuses, instead of handing addresses to its kernel
behind the tracer's back. On the CPU, the library's calls replaced by a record of them."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

import titans_core as tc
from titans_core.kernels import _lib


class Record:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *args: self.calls.append(name) or 0


@pytest.fixture
def raw(monkeypatch):
    rec = Record()
    monkeypatch.setattr(_lib, "lib", lambda: rec)
    monkeypatch.setattr(_lib, "require_device", lambda *t, what: t[0].device)
    monkeypatch.setattr(_lib, "stream_ptr", lambda device: 0)
    return rec


IDS, T2, W = torch.zeros(1, 3, dtype=torch.long), torch.zeros(2, dtype=torch.long), torch.ones(5, 64).bfloat16()
OPS = {
    "token_embedding": (lambda x: tc.token_embedding(IDS, x), torch.ones(5, 64)),
    "token_logprobs": (lambda x: tc.token_logprobs(x, T2, entropy=True).logprobs, torch.ones(2, 10)),
    "token_cross_entropy": (lambda x: tc.token_cross_entropy(x, T2), torch.ones(2, 10)),
    "head_logprobs": (lambda x: tc.head_logprobs(x, W, T2).logprobs, torch.ones(2, 64).bfloat16()),
    "rmsnorm_fwd": (lambda x: tc.rms_norm(x, torch.ones(10)), torch.ones(2, 10)),
    "dwconv_causal": (lambda x: tc.causal_dwconv(x, torch.ones(10, 3)), torch.ones(1, 2, 10)),
}
ops = pytest.mark.parametrize("name", OPS)


@ops
def test_plain_calls_are_direct(name, raw):
    f, x = OPS[name]
    with torch.no_grad():
        f(x)
    assert raw.calls


@ops
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(name, grad, raw):
    f, x = OPS[name]
    with fwAD.dual_level():
        f(x)  # no tangent: nothing to lose
        del raw.calls[:]
        with pytest.raises(NotImplementedError, match="jvp"):
            f(fwAD.make_dual(x.clone().requires_grad_(grad), torch.ones_like(x)))
    with pytest.raises(NotImplementedError, match="jvp"):
        torch.func.jvp(f, (x,), (torch.ones_like(x),))
    assert not raw.calls


@ops
def test_a_trace_holds_the_op(name, raw):
    f, x = OPS[name]
    kinds = [n.kind() for n in torch.jit.trace(f, (x,), check_trace=False).graph.nodes()]
    assert f"titanmac::{name}" in kinds


@ops
def test_make_fx_holds_the_op(name, raw):
    from torch.fx.experimental.proxy_tensor import make_fx
    f, x = OPS[name]
    with torch.no_grad():
        graph = make_fx(f)(x).graph
    assert any(f"titanmac.{name}" in str(n.target) for n in graph.nodes)


@ops
def test_vmap_goes_entry_by_entry(name, raw):
    f, x = OPS[name]
    with torch.no_grad():
        one = f(x)
        assert torch.func.vmap(f)(torch.stack([x] * 3)).shape == (3, *one.shape)


def test_a_backward_with_tangents_is_refused(raw):
    """Forward over reverse: the upstream gradient carries the tangent."""
    x = torch.ones(2, 10, requires_grad=True)
    lp = tc.token_logprobs(x, T2).logprobs
    with fwAD.dual_level():
        g = fwAD.make_dual(torch.ones(2), torch.ones(2))
        with pytest.raises(NotImplementedError, match="jvp"):
            lp.backward(g)
