"""token_embedding against its formula in 64 bits: forward, the three gradients, refusals that need a GPU,
streams, graphs and second derivatives."""
import pytest
import torch

import titans_core as tc
from titans_core.kernels import embedding as ke

pytestmark = pytest.mark.gpu

U = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
F = 2.0 ** -24


def make(B, T, V, d, Np, dtype, dev, seed=0, hot=False, given=False, n_pos=None):
    g = torch.Generator().manual_seed(seed)
    n_pos = n_pos or T + 3
    ids = torch.randint(0, V, (B, T), generator=g)
    if hot:  # a few ids take nearly all tokens
        ids = torch.where(torch.rand(B, T, generator=g) < 0.9, ids % 3, ids)
    s = dict(ids=ids, w=torch.randn(V, d, generator=g).to(dtype), p=torch.randn(n_pos, d, generator=g).to(dtype),
             f=torch.randn(Np, d, generator=g).to(dtype) if Np else None,
             pos=torch.randint(0, n_pos, (B, T), generator=g) if given else None,
             gy=torch.randn(B, Np + T, d, generator=g).to(dtype))
    return {k: None if t is None else t.to(dev) for k, t in s.items()}


def want_fwd(s, scale):
    ids, B, T = s["ids"], *s["ids"].shape
    pos = torch.arange(T, device=ids.device).expand(B, T) if s["pos"] is None else s["pos"]
    a, b = s["w"].double()[ids] * scale, s["p"].double()[pos]
    y, mag = a + b, a.abs() + b.abs()
    if s["f"] is not None:
        f = s["f"].double().expand(B, -1, -1)
        y, mag = torch.cat([f, y], 1), torch.cat([f.abs() * 0, mag], 1)
    return y, mag


def want_grads(s, scale):
    """The gradients in 64 bits, the sums of their terms' magnitudes, and how many terms each row has."""
    ids, (B, T) = s["ids"], s["ids"].shape
    Np = 0 if s["f"] is None else s["f"].shape[0]
    pos = torch.arange(T, device=ids.device).expand(B, T) if s["pos"] is None else s["pos"]
    g = s["gy"].double()[:, Np:].reshape(B * T, -1)
    out = []
    for index, n, c in ((ids, s["w"].shape[0], scale), (pos, s["p"].shape[0], 1.0)):
        z = torch.zeros(n, g.shape[1], dtype=torch.float64, device=g.device)
        out.append((z.index_add(0, index.reshape(-1), g * c), z.index_add(0, index.reshape(-1), (g * c).abs())))
    if Np:
        h = s["gy"].double()[:, :Np]
        out.append((h.sum(0), h.abs().sum(0)))
    return out


def check(s, scale, dtype, y, grads):
    want, mag = want_fwd(s, scale)
    # one rounding to the type; before it the product and the sum in fp32
    assert torch.all((y.double() - want).abs() <= U[dtype] * 1.01 * want.abs() + 2 * F * mag)
    n = s["ids"].numel() + s["ids"].shape[0]
    for got, (wg, mg) in zip(grads, want_grads(s, scale)):
        assert got.dtype == dtype and got.shape == wg.shape
        # fp32 sums of at most n terms, one rounding; fp16's results below 2^-14 are rounded to steps of 2^-24
        tol = U[dtype] * 1.01 * wg.abs() + (min(n, 4096) + 2) * F * mg + (2.0 ** -25 if dtype == torch.float16 else 0)
        assert torch.all((got.double() - wg).abs() <= tol)
        assert torch.all(got[mg == 0] == 0)


CASES = [  # B, T, V, d, Np, hot, given
    (1, 1, 1, 8, 0, False, False), (16, 1, 50, 640, 0, False, True), (2, 5, 7, 24, 3, False, False),
    (1, 64, 3, 8, 1, False, False), (1, 65, 1, 8, 0, False, False), (3, 100, 1000, 640, 16, True, False),
    (2, 700, 11, 20, 4, False, True), (1, 4097, 600, 72, 0, True, False), (5, 1300, 513, 33, 2, True, True),
    (2, 33, 70000, 16, 5, False, False),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,T,V,d,Np,hot,given", CASES)
def test_forward_and_gradients(dev, B, T, V, d, Np, hot, given, dtype):
    s = make(B, T, V, d, Np, dtype, dev, seed=B + T + V, hot=hot, given=given)
    scale = 1.0 if V % 2 else 2.5
    tables = [s[k].requires_grad_() for k in ("w", "p", "f") if s[k] is not None]
    y = tc.token_embedding(s["ids"], s["w"], s["p"], positions=s["pos"], prefix=s["f"], scale=scale)
    grads = torch.autograd.grad(y, tables, s["gy"], retain_graph=True)
    check(s, scale, dtype, y.detach(), grads)
    again = torch.autograd.grad(y, tables, s["gy"])
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    with torch.no_grad():
        assert torch.equal(y, tc.token_embedding(s["ids"].int(), s["w"], s["p"], positions=s["pos"], prefix=s["f"],
                                                 scale=scale))


@pytest.mark.parametrize("part", ["w", "p", "f"])
def test_one_table_at_a_time(dev, part):
    s = make(2, 40, 30, 48, 4, torch.float32, dev)
    s[part].requires_grad_()
    y = tc.token_embedding(s["ids"], s["w"], s["p"], prefix=s["f"])
    y.backward(s["gy"])
    want = dict(zip("wpf", want_grads(s, 1.0)))[part]
    assert torch.all((s[part].grad.double() - want[0]).abs() <= 90 * F * want[1])
    assert all(s[k].grad is None for k in "wpf" if k != part)


def test_without_positions_or_prefix(dev):
    s = make(2, 9, 30, 48, 0, torch.bfloat16, dev)
    assert torch.equal(tc.token_embedding(s["ids"], s["w"]), s["w"][s["ids"]])
    e = tc.token_embedding(s["ids"][:, :0], s["w"], s["p"], prefix=s["p"][:2])
    assert e.shape == (2, 2, 48) and torch.equal(e, s["p"][:2].expand(2, -1, -1))
    assert tc.token_embedding(s["ids"][:0], s["w"]).shape == (0, 9, 48)
    w = s["w"].clone().requires_grad_()
    tc.token_embedding(s["ids"][:, :0], w, prefix=s["p"][:2]).sum().backward()
    assert torch.equal(w.grad, torch.zeros_like(w))


def test_strides_and_offsets(dev):
    """Tables that are column slices of wider ones, odd offsets, a gradient that is a broadcast or a slice."""
    s = make(3, 21, 40, 64, 2, torch.bfloat16, dev)
    wide = torch.randn(40, 131, device=dev).bfloat16()
    for a in (0, 1, 8):
        w = wide[:, a:a + 64].detach().requires_grad_()
        y = tc.token_embedding(s["ids"], w, s["p"], prefix=s["f"])
        want, mag = want_fwd(dict(s, w=w.detach()), 1.0)
        assert torch.all((y.double() - want).abs() <= U[torch.bfloat16] * 1.01 * want.abs() + 2 * F * mag)
        gy = torch.randn(3, 23, 70, device=dev).bfloat16()[..., 3:67]
        got, = torch.autograd.grad(y, w, gy, retain_graph=True)
        assert torch.equal(got, torch.autograd.grad(y, w, gy.contiguous(), retain_graph=True)[0])
        got, = torch.autograd.grad(y, w, gy[:1, :1].expand(3, 23, 64))
        ref, = torch.autograd.grad(tc.token_embedding(s["ids"], w, s["p"], prefix=s["f"]), w,
                                   gy[:1, :1].expand(3, 23, 64).contiguous())
        assert torch.equal(got, ref)


def test_ids_outside_the_table(dev):
    s = make(2, 200, 30, 40, 3, torch.float32, dev)
    bad = s["ids"].clone()
    bad[0, 3], bad[1, 7], bad[1, 8] = -1, 30, 2 ** 40
    s["w"].requires_grad_()
    y = tc.token_embedding(bad, s["w"], s["p"], prefix=s["f"])
    rows = torch.zeros(2, 203, dtype=torch.bool, device=dev)
    rows[0, 6] = rows[1, 10] = rows[1, 11] = True
    assert torch.isnan(y[rows]).all() and torch.isfinite(y[~rows]).all()
    got, = torch.autograd.grad(y, s["w"], s["gy"])
    gy = s["gy"].masked_fill(rows[..., None], 0.0)
    ok = tc.token_embedding(s["ids"], s["w"], s["p"], prefix=s["f"])
    ref, = torch.autograd.grad(ok, s["w"], gy)
    assert torch.all((got - ref).abs() <= 16 * F * (1 + ref.abs()) * 16)
    pos = torch.arange(200, device=dev).expand(2, -1).clone()
    pos[0, 0], pos[1, 1] = -5, 203
    y = tc.token_embedding(s["ids"], s["w"], s["p"], positions=pos)
    assert torch.isnan(y[0, 0]).all() and torch.isnan(y[1, 1]).all() and int(torch.isnan(y).any(-1).sum()) == 2


def test_gradient_against_differences(dev):
    s = make(2, 90, 5, 8, 2, torch.float32, dev, hot=True)
    w = s["w"].requires_grad_()
    f = lambda t: (tc.token_embedding(s["ids"], t, s["p"], prefix=s["f"], scale=0.5).double() * s["gy"]).sum()  # noqa: E731
    got, = torch.autograd.grad(f(w), w)
    u = torch.randn_like(w)
    h = 0.25  # linear: no truncation; each value is rounded to fp32 at |y| < 16
    with torch.no_grad():
        diff = (f(w + h * u) - f(w - h * u)) / (2 * h)
    assert abs(diff - (got.double() * u).sum()) <= 16 * F * 2 * s["gy"].abs().sum().double() / (2 * h)


def test_second_derivative(dev):
    s = make(2, 12, 5, 8, 2, torch.float32, dev)
    tables = [s[k].requires_grad_() for k in "wpf"]
    gy = s["gy"].requires_grad_()
    y = tc.token_embedding(s["ids"], s["w"], s["p"], prefix=s["f"], scale=0.5)
    first = torch.autograd.grad(y, tables, gy, create_graph=True)
    v = [torch.randn_like(t) for t in first]
    got, = torch.autograd.grad(first, gy, v)
    want = tc.token_embedding(s["ids"], v[0], v[1], prefix=v[2], scale=0.5)  # linear: its own transpose's transpose
    assert torch.allclose(got, want.detach(), rtol=0, atol=4 * F * 8)


def test_dispatched_op_agrees(dev):
    s = make(2, 77, 30, 40, 3, torch.bfloat16, dev, given=True)
    args = (s["ids"], s["w"].requires_grad_(), s["p"].requires_grad_(), s["pos"], s["f"].requires_grad_(), 3.0)
    for lists in (False, True):  # the backward makes the lists of tokens where the forward has not
        y, made = ke.token_embedding_fwd(*args, lists)
        assert made.numel() == (ke._lists_bytes(2 * 77, 30) if lists else 0)
        g = torch.autograd.grad(y, (s["w"], s["p"], s["f"]), s["gy"])
        z = tc.token_embedding(s["ids"], s["w"], s["p"], positions=s["pos"], prefix=s["f"], scale=3.0)
        h = torch.autograd.grad(z, (s["w"], s["p"], s["f"]), s["gy"])
        assert torch.equal(y, z) and all(torch.equal(a, b) for a, b in zip(g, h))


def test_other_stream_and_graph(dev):
    s = make(4, 300, 50, 64, 4, torch.bfloat16, dev, hot=True)
    s["w"].requires_grad_()

    def step():
        y = tc.token_embedding(s["ids"], s["w"], s["p"], prefix=s["f"])
        return y.detach(), torch.autograd.grad(y, s["w"], s["gy"])[0]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [step() for _ in range(2)][1]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    del other
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(3):
        new = make(4, 300, 50, 64, 4, torch.bfloat16, dev, seed=seed, hot=True)
        s["ids"].copy_(new["ids"])
        s["gy"].copy_(new["gy"])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, step()))
