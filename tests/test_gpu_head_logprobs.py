"""head_logprobs against the formula in 64 bits on the same 16-bit inputs, and its composed forms."""
import pytest
import torch
import torch.nn.functional as F

import titans_core as tc
from titans_core.kernels import logprobs as kl

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
HALF = [torch.bfloat16, torch.float16]


def inputs(dev, M, V, K, dtype, seed=0, spread=2.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(M, K, generator=g, device=dev).to(dtype)
    w = (torch.randn(V, K, generator=g, device=dev) * (spread / K ** 0.5)).to(dtype)
    t = torch.randint(0, V, (M,), generator=g, device=dev)
    return x, w, t.masked_fill(torch.rand(M, generator=g, device=dev) < 0.15, -100)


def check(x, w, t, r):
    (M, K), V = x.shape, w.shape[0]
    z = x.double() @ w.double().t()
    logp = torch.log_softmax(z, -1)
    p = logp.exp()
    lp = logp.gather(-1, t.clamp(min=0)[:, None])[:, 0].masked_fill(t == -100, 0.0)
    far = (p * (z - z.amax(-1, keepdim=True)).abs()).sum(-1)
    # each logit: an fp32 sum of K exact products; the largest error over the row moves lse by no more
    dz = (K * E * (x.double().abs() @ w.double().abs().t())).amax(-1)
    # the row's sum: 64 entries of a tile per lane and tile, tiles in a row, joins; exponentials as in the stored form
    e = (V / 64 + 120) * E
    tol = 2 * dz + e * (1 + far) + 6 * E * lp.abs()
    assert torch.all((r.logprobs.double() - lp).abs() <= tol)
    assert torch.all(r.logprobs[t == -100] == 0)
    if r.entropy is not None:
        H = -(p * logp).sum(-1)
        # dH/dz is at most max p |ln p + H|, summed: below 2 (H + 1)
        assert torch.all((r.entropy.double() - H).abs() <= 2 * dz * (H + 1) + 2 * e * (1 + far) + 8 * E * H)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("K", [64, 128, 640, 704, 1024])
@pytest.mark.parametrize("M,V", [(1, 1), (3, 65), (16, 4099), (64, 127), (65, 129), (193, 1000), (1000, 2051), (8, 50001)])
def test_values(dev, M, V, K, dtype):
    x, w, t = inputs(dev, M, V, K, dtype, seed=M + V + K)
    r = tc.head_logprobs(x, w, t, entropy=True)
    check(x, w, t, r)
    q = tc.head_logprobs(x, w, t)
    assert torch.equal(q.logprobs, r.logprobs) and q.entropy is None
    assert torch.equal(r.logprobs, tc.head_logprobs(x, w, t.int(), entropy=True).logprobs)


def test_sharp_rows_and_lead_shape(dev):
    """Rows that are nearly certain, hidden states [B, T, K] that are a slice, a weight with a wide pitch."""
    x, w, t = inputs(dev, 6 * 35, 3001, 256, torch.bfloat16, spread=30.0)
    check(x, w, t, tc.head_logprobs(x, w, t, entropy=True))
    big = torch.randn(6, 36, 256, device=dev).bfloat16()
    wide = torch.randn(3001, 320, device=dev).bfloat16() * 0.1
    h, ww, tt = big[:, 1:], wide[:, 8:264], t.view(6, 35)
    r = tc.head_logprobs(h, ww, tt, entropy=True)
    assert r.logprobs.shape == (6, 35)
    s = tc.head_logprobs(h.contiguous(), ww.contiguous(), tt, entropy=True)
    assert all(torch.equal(a, b) for a, b in zip(r[:2], s[:2]))
    for off in (1, 4):  # a start and a pitch that are not 16-byte aligned are copied
        ww = wide[:, off:off + 256]
        assert torch.equal(tc.head_logprobs(h, ww, tt).logprobs, tc.head_logprobs(h, ww.contiguous(), tt).logprobs)


def test_rows_without_a_distribution_and_targets_outside(dev):
    x, w, t = inputs(dev, 70, 500, 128, torch.bfloat16)
    t[:6] = torch.tensor([-1, 500, 2 ** 40, 3, 4, 5], device=dev)
    x[3] = float("nan")
    x[4, 0] = float("inf")
    r = tc.head_logprobs(x, w, t, entropy=True)
    assert torch.isnan(r.logprobs[:5]).all() and torch.isfinite(r.logprobs[5:]).all()
    assert torch.isfinite(r.entropy[:3]).all() and torch.isnan(r.entropy[3:5]).all()
    x, w, t = inputs(dev, 70, 500, 128, torch.bfloat16)
    w[17] = float("-inf")  # an entry of +-inf (or NaN) logits spoils only the rows where it is not -inf
    x[:, :] = x.abs()
    r = tc.head_logprobs(x, w, t.masked_fill(t == 17, 3))
    assert torch.isfinite(r.logprobs).all()


def test_composed_where_the_kernel_does_not_apply(dev):
    x, w, t = inputs(dev, 33, 700, 128, torch.bfloat16)
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    r = tc.head_logprobs(a, b, t, entropy=True)
    gx, gw = torch.autograd.grad(r.logprobs.sum() + r.entropy.sum(), (a, b))
    y, v = x.double().requires_grad_(), w.double().requires_grad_()
    logp = torch.log_softmax(y @ v.t(), -1)
    obj = logp.gather(-1, t.clamp(min=0)[:, None])[:, 0].masked_fill(t == -100, 0.0).sum() - (logp.exp() * logp).sum()
    for got, want in zip((gx, gw), torch.autograd.grad(obj, (y, v))):
        # bf16 logits (2^-8 of values up to 8 in each exponent), a bf16 gradient of them, a bf16 result
        assert (got.double() - want).norm() <= 6 * 2.0 ** -8 * want.norm()
    f = tc.head_logprobs(x.float(), w.float(), t)
    assert torch.allclose(f.logprobs, tc.token_logprobs(F.linear(x.float(), w.float()), t).logprobs)
    x, w, t = inputs(dev, 33, 700, 100, torch.float16)
    assert torch.equal(tc.head_logprobs(x, w, t).logprobs, tc.token_logprobs(F.linear(x, w), t).logprobs)
    e = tc.head_logprobs(x[:0], w, t[:0], entropy=True)
    assert e.logprobs.shape == (0,) and e.entropy.shape == (0,)


def test_dispatched_op_stream_and_graph(dev):
    x, w, t = inputs(dev, 300, 3001, 192, torch.float16)
    want = tc.head_logprobs(x, w, t, entropy=True)[:2]
    assert all(torch.equal(a, b) for a, b in zip(want, kl.head_logprobs_fwd(x, w, t, True, -100)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = tc.head_logprobs(x, w, t, entropy=True)[:2]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = tc.head_logprobs(x, w, t, entropy=True)[:2]
    for seed in range(3):
        for a, b in zip((x, w, t), inputs(dev, 300, 3001, 192, torch.float16, seed=seed + 5)):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, tc.head_logprobs(x, w, t, entropy=True)[:2]))


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("K", [256, 384, 512, 640, 768, 1024])
@pytest.mark.parametrize("M,V", [(256, 100003), (240, 104200), (6250, 4001), (500, 50001), (12500, 2017)])
def test_values_by_resident_rows(dev, M, V, K, dtype):
    """Widths and row counts whose rows stay in registers: partial row tiles, entry tiles and last strips."""
    x, w, t = inputs(dev, M, V, K, dtype, seed=M + V + K)
    t[:2] = torch.tensor([0, V - 1], device=dev)
    r = tc.head_logprobs(x, w, t, entropy=True)
    check(x, w, t, r)
    q = tc.head_logprobs(x, w, t)
    assert torch.equal(q.logprobs, r.logprobs)


@pytest.mark.parametrize("K", [512, 768, 1024])
def test_resident_rows_without_a_distribution(dev, K):
    """NaN and infinite hidden states, targets outside the vocabulary, an entry of -inf in either half of K, and one
    that is the last of a partial tile."""
    x, w, t = inputs(dev, 700, 40003, K, torch.bfloat16)
    t[:7] = torch.tensor([-1, 40003, 2 ** 40, 3, 4, 5, 40002], device=dev)
    x[3, K - 1] = float("nan")
    x[4, 0] = float("inf")
    r = tc.head_logprobs(x, w, t, entropy=True)
    assert torch.isnan(r.logprobs[:5]).all() and torch.isnan(r.entropy[3:5]).all()
    ok = torch.ones(700, dtype=torch.bool, device=dev)
    ok[:5] = False
    check(x[ok], w, t[ok], tc.TokenLogprobs(r.logprobs[ok], r.entropy[ok]))
    x, w, t = inputs(dev, 700, 40003, K, torch.bfloat16)
    x[:, 0], x[:, K - 1] = x[:, 0].abs() + 0.1, x[:, K - 1].abs() + 0.1
    w[17, 0] = w[40002, K - 1] = float("-inf")
    t = t.masked_fill((t == 17) | (t == 40002), 3)
    t[0], t[1] = 17, 40002
    r = tc.head_logprobs(x, w, t, entropy=True)
    assert torch.isneginf(r.logprobs[:2]).all()
    keep = torch.ones(40003, dtype=torch.bool, device=dev)
    keep[17] = keep[40002] = False
    rest = (t - (t > 17).long()).masked_fill(t == -100, -100)[2:]
    check(x[2:], w[keep], rest, tc.TokenLogprobs(r.logprobs[2:], r.entropy[2:]))
