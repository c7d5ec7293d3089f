"""The loss's gradient, formed from the upstream gradient in one launch."""
import pytest
import torch

import titans_core as tc
from titans_core.kernels import logprobs as kl

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,wide", [(torch.float32, False), (torch.bfloat16, False), (torch.float16, False),
                                        (torch.bfloat16, True), (torch.float16, True)])
@pytest.mark.parametrize("rows,V", [(5, 70), (37, 1000), (3, 70001)])
def test_gradient_is_that_of_the_rows(dev, rows, V, dtype, wide):
    """The bits of the per-row gradient for g_lp = g · (−1 / n) in fp32, in place and behind an odd row."""
    gen = torch.Generator().manual_seed(V)
    z0 = (torch.randn(rows + 1, V, generator=gen) * 3).to(dev, dtype)
    t = torch.randint(0, V, (rows,), generator=gen).to(dev)
    t[2] = -100
    for z in (z0[1:], z0[:rows]):
        z = z.detach().requires_grad_()
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=wide):
            loss = tc.token_cross_entropy(z, t)
        assert loss.dtype == (torch.float32 if wide else dtype)
        for g in (1.0, -0.3, 0.0):
            g = torch.tensor(g, device=dev, dtype=loss.dtype)
            got, = torch.autograd.grad(loss, z, g, retain_graph=True)
            _, inv, stats = kl.cross_entropy_fwd(z.detach(), t, -100, wide)
            want = kl.logprob_bwd((g.float() * inv).expand(rows), None, z.detach(), t, stats, None, -100)
            assert torch.equal(got, want)
            assert torch.all(got[2] == 0)
    p = torch.softmax(z.detach().double(), -1)
    hot = torch.zeros_like(p).scatter_(-1, t.clamp(min=0)[:, None], 1.0)
    want = (p - hot) / (rows - 1) * (t != -100)[:, None]
    got, = torch.autograd.grad(loss, z)
    u = torch.finfo(dtype).eps / 2
    assert torch.all((got.double() - want).abs() <= u * want.abs() + (V + 64) * 2.0 ** -24 / (rows - 1) + 1e-7 * u)


def test_captured_loss(dev):
    """Forward and backward in a graph, replayed with other logits, targets and upstream gradients."""
    z = torch.randn(6, 301, device=dev).requires_grad_()
    t, g = torch.randint(0, 301, (6,), device=dev), torch.ones((), device=dev)

    def step():
        loss = tc.token_cross_entropy(z, t)
        return loss.detach(), torch.autograd.grad(loss, z, g)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(3):
        gen = torch.Generator().manual_seed(seed)
        with torch.no_grad():
            z.copy_(torch.randn(6, 301, generator=gen))
        t.copy_(torch.randint(0, 301, (6,), generator=gen))
        g.fill_(0.5 + seed)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)


def test_fp16_gradients_are_not_lost_in_the_upstream_type(dev):
    """An upstream gradient in 16 bit times -1 / n of many rows in fp32: the factor is not rounded to 16 bit."""
    n = 3000
    z = torch.zeros(n, 4, device=dev, dtype=torch.float16, requires_grad=True)
    t = torch.zeros(n, dtype=torch.long, device=dev)
    loss = tc.token_cross_entropy(z, t)
    g = torch.tensor(1000.0, device=dev, dtype=torch.float16)
    got, = torch.autograd.grad(loss, z, g)
    want = torch.tensor([-0.75, 0.25, 0.25, 0.25], dtype=torch.float64, device=dev) * 1000.0 / n
    assert torch.all((got.double() - want).abs() <= (2.0 ** -11 + 2.0 ** -20) * want.abs())


@pytest.mark.parametrize("B", [1, 4])
def test_kept_tensors_away_and_back(dev, B):
    """What the loss keeps may be moved to the host in between, and is there for a second backward."""
    gen = torch.Generator().manual_seed(B)
    z = (torch.randn(B, 30, 1001, generator=gen) * 2).to(dev, torch.bfloat16)
    t = torch.randint(0, 1001, (B, 30), generator=gen, dtype=torch.int32).to(dev)
    a, b = (z[:, 3:].detach().requires_grad_() for _ in range(2))
    want, = torch.autograd.grad(tc.token_cross_entropy(a, t[:, 3:]), a)
    with torch.autograd.graph.save_on_cpu():
        loss = tc.token_cross_entropy(b, t[:, 3:])
    for _ in range(2):
        got, = torch.autograd.grad(loss, b, retain_graph=True)
        assert torch.equal(got, want)
    # recorded: the same in torch's operations, and differentiable again
    loss = tc.token_cross_entropy(b, t[:, 3:])
    first, = torch.autograd.grad(loss, b, create_graph=True)
    assert (first.double() - want.double()).norm() <= 2.0 ** -7 * want.double().norm()
    second, = torch.autograd.grad(first.float().square().sum(), b)
    assert torch.isfinite(second).all() and second.abs().sum() > 0
