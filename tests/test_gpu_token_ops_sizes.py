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


def sums_over_sequences(g, n_prefix, n_pos):
    """(dP, dprefix) in 64 bits and the sums of magnitudes."""
    out = []
    for x in (g.double(), g.double().abs()):
        s = x.sum(0)
        dp = torch.zeros(n_pos, g.shape[-1], dtype=torch.float64, device=g.device)
        dp[:s.shape[0] - n_prefix] = s[n_prefix:]
        out.append((dp, s[:n_prefix]))
    return out


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,T,Np,d,n_pos", [(5000, 3, 4, 640, 64), (20000, 1, 0, 64, 16), (4096, 16, 16, 640, 40),
                                            (1003, 2, 3, 641, 2), (16, 5, 1, 64, 9), (17, 1, 2, 8, 1), (70, 300, 0, 96, 301)])
def test_many_sequences(dev, B, T, Np, d, n_pos, dtype):
    """Default positions and the prefix: sums over the sequences."""
    g = torch.Generator().manual_seed(B)
    ids = torch.randint(0, 50, (B, T), generator=g).to(dev)
    w, p, f = (torch.randn(n, d, generator=g).to(dev, dtype).requires_grad_() for n in (50, n_pos, max(Np, 1)))
    up = (torch.randn(B, Np + T, d, generator=g) + 0.5).to(dev, dtype)
    y = tc.token_embedding(ids, w, p, prefix=f if Np else None)
    tables = (p, f) if Np else (p,)
    got = torch.autograd.grad(y, tables, up, retain_graph=True)
    for upstream in (up, torch.stack([up, up], 2)[:, :, 0]):  # rows one after the other, and in steps of two
        again = torch.autograd.grad(y, tables, upstream, retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(got, again))
    want, size = sums_over_sequences(up, Np, n_pos)
    u = torch.finfo(dtype).eps / 2
    for a, b, s in zip(got, want, size):
        # B additions, each rounded, in whatever order, and the result's rounding
        assert torch.all((a.double() - b).abs() <= B * 2.0 ** -24 * s + u * b.abs() + 1e-30)


def test_sums_of_many_sequences_are_not_one_chain(dev):
    """fp32 sums of 20000 equal values: one after the other they are off by 1.7e-4 of the sum, all roundings going one
    way; runs of at most 79 of them joined in pairs by at most (79 + 8) half steps, and the result's."""
    B, d = 20000, 64
    w, p = torch.zeros(5, d, device=dev), torch.zeros(1, d, device=dev, requires_grad=True)
    y = tc.token_embedding(torch.zeros(B, 1, dtype=torch.long, device=dev), w, p)
    g, = torch.autograd.grad(y, p, torch.full_like(y, 0.1))
    want = B * torch.tensor(0.1).double().item()
    assert (g.double() - want).abs().max().item() <= (79 + 8 + 1) * 2.0 ** -24 * want


def rows64(z, t):
    """(lp, H, p, ln p) in 64 bits, ignored targets as 0."""
    logp = torch.log_softmax(z.double(), -1)
    lp = logp.gather(-1, t.clamp(min=0)[:, None])[:, 0].masked_fill(t == -100, 0.0)
    some = torch.where(logp == -math.inf, 0.0, logp)
    return lp, -(logp.exp() * some).sum(-1), logp.exp(), some


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,V", [((1 << 20) + 3, 33), (8191, 253), (8193, 254), (9001, 505), (1025, 506), (7, 1), (9 * 1024, 2)])
def test_many_short_rows(dev, rows, V, dtype):
    """The loss, log probabilities and entropies of rows that one wave takes, and of the first that it does not, behind
    an odd row (none of them aligned alike), with their gradients."""
    g = torch.Generator().manual_seed(rows)
    z0 = (torch.randn(rows + 1, V, generator=g) * 2).to(dev, dtype)
    t = torch.randint(0, V, (rows,), generator=g).to(dev)
    t[torch.rand(rows, generator=g).to(dev) < 0.1] = -100
    t[0] = 0
    z = z0[1:].requires_grad_()
    loss = tc.token_cross_entropy(z, t)
    dz, = torch.autograd.grad(loss, z)
    r = tc.token_logprobs(z, t, entropy=True)
    gl, ge = torch.randn(rows, generator=g).to(dev), torch.randn(rows, generator=g).to(dev)
    dz2, = torch.autograd.grad([r.logprobs, r.entropy], z, [gl, ge])
    n, u = int((t != -100).sum()), torch.finfo(dtype).eps / 2
    total = 0.0
    for a in range(0, rows, 1 << 18):
        at = slice(a, a + (1 << 18))
        lp, H, p, logp = rows64(z.detach()[at], t[at])
        total += lp.sum().item()
        # exponentials, their sum of V terms and a logarithm, each off by roundings of values up to 2 · 2 · 6
        tol = (V + 64) * 2.0 ** -24
        assert torch.allclose(r.logprobs[at].double(), lp, rtol=0, atol=tol)
        assert torch.allclose(r.entropy[at].double(), H, rtol=0, atol=24 * tol)
        keep = (t[at] != -100).double()
        hot = torch.zeros_like(p).scatter_(-1, t[at].clamp(min=0)[:, None], 1.0)
        want = (-keep / n)[:, None] * (hot - p)
        # |p| is off by tol of itself, the product rounded to the type
        assert torch.all((dz[at].double() - want).abs() <= u * want.abs() + 2 * tol / n)
        gk = (gl[at].double() * keep)[:, None]
        want = gk * (hot - p) - ge[at].double()[:, None] * p * (logp + H[:, None])
        size = gk.abs() + 48 * ge[at].double().abs()[:, None]
        assert torch.all((dz2[at].double() - want).abs() <= u * want.abs() + 2 * tol * size)
    want = -total / n
    # a thread adds rows / 1024 values, then 16 waves of 64
    assert abs(loss.double().item() - want) <= u * want + ((rows / 1024 + 22) * 2.0 ** -24 + 2 * (V + 64) * 2.0 ** -24) * max(want, 1)


def embedding64(ids, pos, tables, up, scale):
    """y and the gradients of the three tables in 64 bits, with the sums of their terms' magnitudes and numbers."""
    w, p, f = tables
    Np, d = f.shape
    y = torch.cat([f.double().expand(len(ids), -1, -1), w.double()[ids] * scale + p.double()[pos]], 1)
    g, out = up.double()[:, Np:].reshape(-1, d), []
    for index, n, c in ((ids, len(w), scale), (pos, len(p), 1.0)):
        zero, index = torch.zeros(n, d, dtype=torch.float64, device=g.device), index.reshape(-1)
        out.append((zero.index_add(0, index, g * c), zero.index_add(0, index, (g * c).abs()), index.bincount(minlength=n)))
    h = up.double()[:, :Np]
    return y, [*out, (h.sum(0), h.abs().sum(0), torch.full((Np,), len(ids), device=g.device))]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,T,V,d,given", [
    (5, 3333, 700, 16, False), (5, 3333, 20001, 16, True),   # more tokens than a wave reads in one turn (8192 in all)
    (9, 8192, 8193, 8, False),                               # nine turns of them
    (2, 40, 60, 4096, False), (3, 50, 30, 1500, True),       # rows of more pieces than a workgroup has threads
    (1, 70, 3, 9001, False),
])
@pytest.mark.parametrize("hot", [0, 1])
def test_turns_of_the_embedding(dev, B, T, V, d, given, hot, dtype):
    """Nine of ten tokens are three neighbouring ids: the first, or (hot) ones in the last, wide range."""
    g = torch.Generator().manual_seed(T + V)
    ids = torch.randint(0, V, (B, T), generator=g)
    ids = torch.where(torch.rand(B, T, generator=g) < 0.9, (V - 3) * hot + ids % 3, ids).to(dev)
    pos = torch.randint(0, 50, (B, T), generator=g).to(dev) if given else torch.arange(T, device=dev).expand(B, T)
    n_pos = 64 if given else T + 5
    tables = [torch.randn(n, d, generator=g).to(dev, dtype).requires_grad_() for n in (V, n_pos, 3)]
    up = torch.randn(B, 3 + T, d, generator=g).to(dev, dtype)
    y = tc.token_embedding(ids, *tables[:2], positions=pos if given else None, prefix=tables[2], scale=0.75)
    grads = torch.autograd.grad(y, tables, up)
    want, sums = embedding64(ids, pos, [t.detach() for t in tables], up, 0.75)
    u = torch.finfo(dtype).eps / 2
    assert torch.all((y.double() - want).abs() <= u * want.abs() + 2.0 ** -22 * (want.abs() + 5))
    for got, (a, size, n) in zip(grads, sums):
        # n fp32 additions in some order and the factor, then one rounding
        assert torch.all((got.double() - a).abs() <= u * 1.01 * a.abs() + (n[:, None] + 2) * 2.0 ** -24 * size)
        assert torch.all(got[n == 0] == 0)


@pytest.mark.parametrize("top", [0, 3])
def test_more_rows_than_workgroups(dev, top):
    """2^21 rows and some: the forward's workgroups take turns, their shared memory used again."""
    rows, V = (1 << 21) + 5003, 9
    g = torch.Generator().manual_seed(top)
    z = (torch.randn(rows, V, generator=g) * 2).to(dev, torch.bfloat16)
    t = torch.randint(0, V, (rows,), generator=g).to(dev)
    t[::7] = -100
    r = tc.token_logprobs(z, t, entropy=True, top_k=top)
    tol = (V + 64) * 2.0 ** -24
    for a in range(0, rows, 1 << 19):
        at = slice(a, a + (1 << 19))
        lp, H, _, logp = rows64(z[at], t[at])
        assert torch.allclose(r.logprobs[at].double(), lp, rtol=0, atol=tol)
        assert torch.allclose(r.entropy[at].double(), H, rtol=0, atol=24 * tol)
        if top:
            ids = torch.sort(z[at].double(), dim=-1, descending=True, stable=True).indices[:, :top]
            assert torch.equal(r.top_ids[at], ids)
            assert torch.allclose(r.top_logprobs[at].double(), logp.gather(-1, ids), rtol=0, atol=tol)


@pytest.mark.parametrize("rows", [1, 3, 700])
def test_the_loss_of_ignored_rows_alone(dev, rows):
    """No row asked for: a loss of NaN, a gradient of zeros, whatever the rows hold."""
    z = torch.full((rows, 4001), float("nan"), device=dev, dtype=torch.bfloat16)
    z[-1] = float("inf")
    z.requires_grad_()
    loss = tc.token_cross_entropy(z, torch.full((rows,), -100, device=dev))
    assert torch.isnan(loss)
    dz, = torch.autograd.grad(loss, z)
    assert torch.all(dz == 0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("given", [False, True])
def test_each_table_takes_the_tokens_within_it(dev, given, dtype):
    """A token whose id (position) is outside its table adds to the other table's gradient: that is decided per table."""
    g = torch.Generator().manual_seed(1)
    V, n_pos, B, T, d = 11, 9, 3, 40, 24
    ids = torch.randint(-2, V + 2, (B, T), generator=g).to(dev)
    pos = torch.randint(-2, n_pos + 2, (B, T), generator=g).to(dev) if given else None
    n_pos = n_pos if given else T
    w, p = (torch.randn(n, d, generator=g).to(dev, dtype).requires_grad_() for n in (V, n_pos))
    up = torch.randint(-2, 3, (B, T, d), generator=g).to(dev, dtype)  # small whole numbers: exact sums
    y = tc.token_embedding(ids, w, p, positions=pos)
    at = torch.arange(T, device=dev).expand(B, T) if pos is None else pos
    outside = (ids < 0) | (ids >= V) | (at < 0) | (at >= n_pos)
    assert torch.equal(torch.isnan(y).all(-1), outside) and torch.equal(torch.isnan(y).any(-1), outside)
    grads = torch.autograd.grad(y, (w, p), up, retain_graph=True)
    up2 = up.clone().requires_grad_()  # recorded: the gradients in torch's operations
    recorded = torch.autograd.grad(y, (w, p), up2, create_graph=True)
    for got, rec, index, n in zip(grads, recorded, (ids, at), (V, n_pos)):
        ok = (index >= 0) & (index < n)
        want = torch.zeros(n, d, device=dev).index_add(0, index[ok], up[ok].float())
        assert torch.equal(got.float(), want) and torch.equal(rec.float(), want)
