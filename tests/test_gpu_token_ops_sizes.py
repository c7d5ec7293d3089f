"""The token operators at sizes where their kernels take turns: more rows than workgroups, more tokens than a
wave holds, rows wider than a workgroup, many sequences."""
import math

import pytest
import torch

import titans_core as tc

pytestmark = pytest.mark.gpu


def test_head_rows_past_the_joins_workgroups(dev):
    """2^26 rows and some: rows repeat, so must their scores."""
    M, n, K, V = (1 << 26) + 5, 4099, 64, 70
    g = torch.Generator().manual_seed(0)
    h = torch.randn(n, K, generator=g).to(dev, torch.bfloat16)
    w = (torch.randn(V, K, generator=g) * 0.3).to(dev, torch.bfloat16)
    t = torch.randint(0, V, (n,), generator=g).to(dev)
    t[7] = -100
    one = tc.head_logprobs(h, w, t, entropy=True)
    logp = torch.log_softmax(h.double() @ w.double().t(), -1)
    # a logit is an fp32 sum of K products (each partial sum rounded: K u of their magnitudes); lp moves by at most
    # twice that, H by sum p |ln p + H| <= ln V + H of it; 2^-19 for the exponentials, their sum and its logarithm
    dz = K * 2.0 ** -24 * (h.double().abs() @ w.double().abs().t()).max().item()
    want = logp.gather(-1, t.clamp(min=0)[:, None])[:, 0].masked_fill(t == -100, 0.0)
    assert torch.allclose(one.logprobs.double(), want, rtol=0, atol=2 * dz + 2.0 ** -19)
    assert torch.allclose(one.entropy.double(), -(logp.exp() * logp).sum(-1), rtol=0, atol=2 * math.log(V) * dz + 2.0 ** -19)
    times = M // n + 1
    many = tc.head_logprobs(h.repeat(times, 1)[:M], w, t.repeat(times)[:M], entropy=True)
    for a, b in ((one.logprobs, many.logprobs), (one.entropy, many.entropy)):
        assert torch.equal(a.expand(times - 1, n), b[:(times - 1) * n].view(times - 1, n))
        assert torch.equal(a[:M - (times - 1) * n], b[(times - 1) * n:])
