"""Ways of calling the token operators that programs have: torch.compile, batched gradients, threads, a chain of
them as a training step, odd positions, in-place changes between forward and backward."""
import threading

import pytest
import torch
import torch.nn.functional as F

import titans_core as tc

pytestmark = pytest.mark.gpu


def data(dev, dtype=torch.bfloat16, B=2, T=40, V=300, d=64, Np=4, seed=0):
    g = torch.Generator().manual_seed(seed)
    mk = lambda *s: torch.randn(*s, generator=g).to(dev, dtype)  # noqa: E731
    ids = torch.randint(0, V, (B, T), generator=g).to(dev)
    return ids, mk(V, d), mk(T + 5, d), mk(Np, d)


def step(ids, w, p, f, ignore_tail=True):
    """Embedding, a head tied to its table, the loss, the scores with entropy: the operators as a program chains them."""
    y = tc.token_embedding(ids, w, p, prefix=f, scale=0.5)
    logits = F.linear(y[:, f.shape[0]:], w)
    targets = F.pad(ids[:, 1:], (0, 1), value=-100)
    loss = tc.token_cross_entropy(logits, targets)
    r = tc.token_logprobs(logits, targets, entropy=True)
    return loss.float() + 1e-2 * r.entropy.mean() - 1e-3 * r.logprobs.sum()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_chain_against_torch(dev, dtype):
    ids, *tables = data(dev, dtype)
    tables = [(t * 0.3).detach().requires_grad_() for t in tables]
    got = torch.autograd.grad(step(ids, *tables), tables)
    w, p, f = (t.detach().double().requires_grad_() for t in tables)
    y = torch.cat([f.expand(2, -1, -1), 0.5 * w[ids] + p[:40]], 1)
    logits = y[:, 4:] @ w.t()
    t = F.pad(ids[:, 1:], (0, 1), value=-100)
    logp = torch.log_softmax(logits, -1)
    lp = logp.gather(-1, t.clamp(min=0)[..., None])[..., 0].masked_fill(t == -100, 0.0)
    obj = -lp.sum() / (t != -100).sum() + 1e-2 * -(logp.exp() * logp).sum(-1).mean() - 1e-3 * lp.sum()
    want = torch.autograd.grad(obj, (w, p, f), allow_unused=True)
    u = torch.finfo(dtype).eps / 2
    for a, b in zip(got, want):
        b = torch.zeros_like(a, dtype=torch.float64) if b is None else b
        # the logits (of up to 8) and their gradient are rounded to the type on the way: 8 u in each exponent
        assert (a.double() - b).norm() <= (16 * u + 1e-5) * b.norm() + 1e-12


def test_compile(dev):
    ids, *tables = data(dev)
    tables = [(t * 0.3).detach().requires_grad_() for t in tables]
    want = step(ids, *tables)
    gw = torch.autograd.grad(want, tables)
    fn = torch.compile(step, backend="aot_eager", fullgraph=True)
    got = fn(ids, *tables)
    assert torch.allclose(got, want, rtol=1e-5, atol=1e-6)
    for a, b in zip(torch.autograd.grad(got, tables), gw):
        assert (a.double() - b.double()).norm() <= 2.0 ** -6 * b.double().norm()

    def score(h, w, t):
        return tc.head_logprobs(h, w, t, entropy=True)

    with torch.no_grad():
        h = tables[0][ids]
        a, b = score(h, tables[0], ids), torch.compile(score, backend="aot_eager")(h, tables[0], ids)
        assert torch.equal(a.logprobs, b.logprobs) and torch.equal(a.entropy, b.entropy)


def test_batched_gradients(dev):
    """Several upstream gradients at once give what one at a time gives."""
    ids, w, p, f = data(dev, torch.float32)
    w.requires_grad_()
    y = tc.token_embedding(ids, w, p, prefix=f)
    gs = torch.randn(3, *y.shape, device=dev)
    got, = torch.autograd.grad(y, w, gs, is_grads_batched=True, retain_graph=True)
    want = torch.stack([torch.autograd.grad(y, w, g, retain_graph=True)[0] for g in gs])
    assert torch.allclose(got, want, rtol=0, atol=1e-5)
    z = torch.randn(5, 70, device=dev, requires_grad=True)
    t = torch.tensor([1, 5, -100, 69, 0], device=dev)
    r = tc.token_logprobs(z, t, entropy=True)
    for out in (r.logprobs, r.entropy):
        gs = torch.randn(3, 5, device=dev)
        got, = torch.autograd.grad(out, z, gs, is_grads_batched=True, retain_graph=True)
        want = torch.stack([torch.autograd.grad(out, z, g, retain_graph=True)[0] for g in gs])
        assert torch.allclose(got, want, rtol=0, atol=1e-5)
    loss = tc.token_cross_entropy(z, t)
    got, = torch.autograd.grad(loss, z, torch.tensor([1.0, -2.0], device=dev), is_grads_batched=True,
                               retain_graph=True)
    one, = torch.autograd.grad(loss, z)
    assert torch.allclose(got, torch.stack([one, -2 * one]), rtol=0, atol=1e-6)


def test_threads_and_streams_at_once(dev):
    """Two host threads, each on its own stream, sharing nothing but the library."""
    sets = [data(dev, seed=s, T=300, V=2000) for s in (1, 2)]
    alone = []
    for ids, *tables in sets:
        tables = [t.requires_grad_() for t in tables]
        alone.append(torch.autograd.grad(step(ids, *tables), tables))
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(k):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(4):
                    ids, *tables = sets[k]
                    tables = [t.detach().requires_grad_() for t in tables]
                    got[k] = torch.autograd.grad(step(ids, *tables), tables)
            s.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors
    for a, b in zip(alone, got):
        for x, y in zip(a, b):  # the head's own products are the library's
            assert (x.double() - y.double()).norm() <= 2.0 ** -6 * x.double().norm()


def test_positions_of_any_index_type(dev):
    ids, w, p, f = data(dev)
    pos = torch.randint(0, 45, (40,), device=dev)
    a = tc.token_embedding(ids, w, p, positions=pos)
    assert torch.equal(a, tc.token_embedding(ids, w, p, positions=pos.int().expand(2, 40)))
    assert torch.equal(a, tc.token_embedding(ids.t().contiguous().t(), w, p, positions=pos.expand(2, 40)))
    p.requires_grad_()
    y = tc.token_embedding(ids, w, p, positions=pos, prefix=f)
    g, = torch.autograd.grad(y.float().sum(), p)
    n = torch.zeros(45, device=dev).index_add_(0, pos, torch.full((40,), 2.0, device=dev))
    assert torch.equal(g.float(), n[:, None].expand(45, 64))  # small whole numbers are exact


def test_changed_inputs_are_noticed(dev):
    ids, w, p, f = data(dev)
    w.requires_grad_()
    y = tc.token_embedding(ids, w, p)
    ids.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()
    z = torch.randn(4, 50, device=dev, requires_grad=True)
    zz = z * 1.0
    loss = tc.token_cross_entropy(zz, torch.zeros(4, dtype=torch.long, device=dev))
    zz.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()
    # a result may be changed
    y = tc.token_embedding(torch.zeros(1, 3, dtype=torch.long, device=dev), w, p)
    y.mul_(2).float().sum().backward()
    assert torch.equal(w.grad[0].float(), torch.full((64,), 6.0, device=dev))
