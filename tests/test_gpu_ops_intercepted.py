"""Ops inside traces and batches on the GPU give what plain calls give."""
import pytest
import torch

import titans_core as tc

pytestmark = pytest.mark.gpu


def ops(dev):
    g = torch.Generator().manual_seed(0)
    mk = lambda *s: torch.randn(*s, generator=g).to(dev)  # noqa: E731
    ids, t = torch.randint(0, 30, (2, 7), generator=g).to(dev), torch.randint(0, 30, (6,), generator=g).to(dev)
    w, scale, conv = mk(30, 64).bfloat16(), mk(64), mk(64, 4)
    return {
        "token_embedding": (lambda x: tc.token_embedding(ids, x), mk(30, 64)),
        "token_logprobs": (lambda x: tc.token_logprobs(x, t).logprobs, mk(6, 30)),
        "entropy": (lambda x: tc.token_logprobs(x, t, entropy=True, top_k=2).entropy, mk(6, 30).bfloat16()),
        "token_cross_entropy": (lambda x: tc.token_cross_entropy(x, t), mk(6, 30)),
        "head_logprobs": (lambda x: tc.head_logprobs(x, w, t).logprobs, mk(6, 64).bfloat16()),
        "rms_norm": (lambda x: tc.rms_norm(x, scale), mk(6, 64)),
        "causal_dwconv": (lambda x: tc.causal_dwconv(x, conv), mk(2, 9, 64)),
        "windowed_attention": (lambda x: tc.windowed_attention(x, x, x, 5, 2), mk(1, 2, 40, 64).bfloat16()),
    }


NAMES = ["token_embedding", "token_logprobs", "entropy", "token_cross_entropy", "head_logprobs", "rms_norm",
         "causal_dwconv", "windowed_attention"]


@pytest.mark.parametrize("name", NAMES)
def test_trace(dev, name):
    f, x = ops(dev)[name]
    traced = torch.jit.trace(f, (x,), check_trace=False)
    with torch.no_grad():
        for y in (x, x * 0.5 + 0.25):
            assert torch.equal(traced(y), f(y))


@pytest.mark.parametrize("name", NAMES)
def test_vmap(dev, name):
    f, x = ops(dev)[name]
    xs = torch.stack([x, x * 0.5, -x])
    with torch.no_grad():
        assert torch.equal(torch.func.vmap(f)(xs), torch.stack([f(y) for y in xs]))


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode(dev, name):
    f, x = ops(dev)[name]
    with pytest.raises(NotImplementedError, match="jvp"):
        torch.func.jvp(f, (x,), (torch.ones_like(x),))


def test_default_device(dev):
    """torch.set_default_device installs a function mode: the kernels still run directly."""
    f, x = ops(dev)["token_logprobs"]
    with torch.no_grad(), torch.device(dev):
        a = f(x)
    assert torch.equal(a, f(x))
