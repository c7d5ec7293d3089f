"""token_logprobs and token_cross_entropy against their formulas in 64 bits: values, alternatives, gradients,
masked and degenerate rows, strides, streams, graphs and second derivatives."""
import math

import pytest
import torch

import titans_core as tc
from titans_core.kernels import logprobs as kl

pytestmark = pytest.mark.gpu

DT = [torch.float32, torch.bfloat16, torch.float16]
U = {t: torch.finfo(t).eps / 2 for t in DT}
F = 2.0 ** -24
INF = float("inf")


def logits(dev, shape, dtype, seed=0, scale=3.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=dev) * scale).to(dtype)


def targets(dev, shape, V, seed=0, drop=0.2):
    g = torch.Generator(device=dev).manual_seed(seed + 1)
    t = torch.randint(0, V, shape, generator=g, device=dev)
    return t.masked_fill(torch.rand(*shape, generator=g, device=dev) < drop, -100)


def reference(z, t, k=0):
    """In 64 bits: lp, H, ids, top lp, and what the tolerances take: p, ln p, the mean distance from the maximum."""
    zd = z.detach().double()
    logp = torch.log_softmax(zd, -1)
    p = logp.exp()
    some = torch.where(p > 0, logp, 0.0)
    lp = logp.gather(-1, t.clamp(min=0).unsqueeze(-1)).squeeze(-1).masked_fill(t == -100, 0.0)
    H = -(p * some).sum(-1)
    ids = torch.sort(zd, dim=-1, descending=True, stable=True).indices[..., :k]
    far = (p * (zd - zd.amax(-1, keepdim=True)).abs().clamp(max=100)).nan_to_num(0.0).sum(-1)
    return dict(lp=lp, H=H, ids=ids, top=logp.gather(-1, ids), p=p, logp=some, far=far)


def depth(V):
    """Additions behind one term of a row's sums: a thread of 256 or more has at most V / 256 + 2 groups' values
    (with eight to a group), then joins over the workgroup's lanes and waves and over the parts."""
    return V / 256 + 16 + 80


def row_error(V):
    """Relative error of s, or of h against sum e |d|: each exponential's argument (three roundings of |d| <= 100
    where it counts, two of them relative: 3 * |d| F, at the weight e^-|d| less than 3 F) and result (2 F), and the sum."""
    return (depth(V) + 16) * F


def check_values(r, w, V):
    e = row_error(V)
    assert torch.all((r.logprobs.double() - w["lp"]).abs() <= e * (1 + w["far"]) + 6 * F * w["lp"].abs())
    if r.entropy is not None:
        assert torch.all((r.entropy.double() - w["H"]).abs() <= 2 * e * (1 + w["far"]) + 8 * F * w["H"])
    if r.top_ids is not None:
        assert torch.equal(r.top_ids, w["ids"])
        fin = torch.isfinite(w["top"])
        assert torch.equal(torch.isfinite(r.top_logprobs), fin)
        d = (r.top_logprobs.double() - w["top"]).abs()
        assert torch.all((d <= (e * (1 + w["far"])).unsqueeze(-1) + 6 * F * w["top"].abs())[fin])


def check_grad(dz, w, t, g_lp, g_ent, V, dtype):
    given = (t != -100)
    gl = (g_lp.double() * given).unsqueeze(-1) if g_lp is not None else torch.zeros_like(w["p"][..., :1])
    at = torch.arange(V, device=t.device) == t.unsqueeze(-1)
    want = gl * (at.double() - w["p"])
    mag = gl.abs() * (w["p"] + at)
    if g_ent is not None:
        ge = g_ent.double().unsqueeze(-1)
        want = want - ge * w["p"] * (w["logp"] + w["H"].unsqueeze(-1))
        mag = mag + ge.abs() * w["p"] * (w["logp"].abs() + w["H"].unsqueeze(-1) + 2)
    # p is off by its row's sum and by its own argument (|d| <= |ln p| + 1); one rounding to the type, to steps of
    # 2^-24 below fp16's 2^-14, and fp32's underflow of p
    e = 2 * row_error(V) * (1 + w["far"]).unsqueeze(-1) + 6 * F * (w["logp"].abs() + 1)
    tol = U[dtype] * 1.01 * want.abs() + e * mag + (2.0 ** -25 if dtype == torch.float16 else 1e-37)
    assert torch.all((dz.double() - want).abs() <= tol)


SIZES = [(1, 1), (3, 2), (5, 7), (2, 64), (9, 65), (33, 1000), (300, 4099), (1, 50001), (700, 5003), (2, 130000), (40, 40001)]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("M,V", SIZES)
def test_values_and_gradient(dev, M, V, dtype):
    z, t = logits(dev, (M, V), dtype, seed=V + M).requires_grad_(), targets(dev, (M,), V, seed=M)
    k = min(V, 20)
    w = reference(z, t, k)
    r = tc.token_logprobs(z, t, entropy=True, top_k=k)
    check_values(r, w, V)
    assert not r.top_logprobs.requires_grad and not r.top_ids.requires_grad
    g_lp, g_ent = logits(dev, (M,), torch.float32, 5), logits(dev, (M,), torch.float32, 6)
    dz, = torch.autograd.grad([r.logprobs, r.entropy], z, [g_lp, g_ent], retain_graph=True)
    assert dz.dtype == dtype
    check_grad(dz, w, t, g_lp, g_ent, V, dtype)
    assert torch.equal(dz, torch.autograd.grad([r.logprobs, r.entropy], z, [g_lp, g_ent], retain_graph=True)[0])
    dz, = torch.autograd.grad(r.logprobs, z, g_lp, retain_graph=True)
    check_grad(dz, w, t, g_lp, None, V, dtype)
    assert torch.all(dz[t == -100] == 0)
    dz, = torch.autograd.grad(r.entropy, z, g_ent)
    check_grad(dz, w, t, None, g_ent, V, dtype)
    # each result alone
    with torch.no_grad():
        check_values(tc.token_logprobs(z, t), w, V)
        check_values(tc.token_logprobs(z, t.int(), entropy=True), w, V)
        check_values(tc.token_logprobs(z, t, top_k=k), w, V)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("M,V", [(4, 11), (513, 1111), (3, 33333)])
def test_cross_entropy(dev, M, V, dtype):
    z, t = logits(dev, (M, V), dtype, seed=V).requires_grad_(), targets(dev, (M,), V, seed=V)
    t[0] = 1
    n = int((t != -100).sum())
    w = reference(z, t)
    loss = tc.token_cross_entropy(z, t)
    want = -w["lp"].sum() / n
    assert loss.dtype == dtype and loss.dim() == 0
    tol = U[dtype] * 1.01 * want + (row_error(V) + (M / 1024 + 24) * F) * (1 + w["far"].max() + w["lp"].abs().max())
    assert abs(loss.double() - want) <= tol
    g = torch.tensor(0.75, device=dev, dtype=dtype)
    dz, = torch.autograd.grad(loss, z, g)
    check_grad(dz, w, t, torch.full((M,), -0.75 / n, device=dev, dtype=torch.float64), None, V, dtype)
    assert torch.all(dz[t == -100] == 0)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        wide = tc.token_cross_entropy(z, t)
    assert wide.dtype == torch.float32
    assert abs(wide.double() - want) <= tol - U[dtype] * 1.01 * want + F * want
    none = tc.token_cross_entropy(z, torch.full_like(t, -100))
    assert torch.isnan(none)
    assert torch.all(torch.autograd.grad(none, z)[0] == 0)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("M", [3, 600])
def test_masked_rows(dev, M, dtype):
    """-inf, the type's lowest value, one entry left, all of it masked, +inf and NaN."""
    V, k = 9001, 7
    z = logits(dev, (M, V), dtype, seed=1)
    low = torch.finfo(dtype).min
    t = targets(dev, (M,), V, drop=0.0)
    t[:3] = torch.tensor([5, 3000, 9000], device=dev)
    z[0, 10:] = -INF  # ten entries left
    z[1] = -INF
    z[1, 3000] = 2.0  # one left: certain, entropy 0
    z[2] = low        # masked by the lowest value alone: uniform
    w = reference(z, t, k)
    zr = z.clone().requires_grad_()
    r = tc.token_logprobs(zr, t, entropy=True, top_k=k)
    check_values(r, w, V)
    assert r.logprobs[1] == 0 and r.entropy[1] == 0
    g = torch.ones(M, device=dev)
    dz, = torch.autograd.grad([r.logprobs, r.entropy], zr, [g, g])
    check_grad(dz, w, t, g, g, V, dtype)
    assert torch.all(dz[0, 10:] == 0)
    t2 = t.clone()
    t2[0] = 77  # a masked target
    assert tc.token_logprobs(z, t2).logprobs[0] == -INF
    z[0] = -INF
    z[1, 4] = INF
    z[2, 8] = float("nan")
    zr = z.clone().requires_grad_()
    r = tc.token_logprobs(zr, t, entropy=True, top_k=k)
    for x in (r.logprobs, r.entropy, r.top_logprobs):
        assert torch.isnan(x[:3]).all() and torch.isfinite(x[3:]).all()
    assert torch.all(r.top_ids[:3] == -1) and torch.all(r.top_ids[3:] >= 0)
    dz, = torch.autograd.grad(r.logprobs, zr, g)
    assert torch.isnan(dz[0]).all() and torch.isfinite(dz[3:]).all()
    # rows that are ignored are not looked at by the loss
    t3 = t.clone()
    t3[:3] = -100
    loss = tc.token_cross_entropy(zr, t3)
    dz, = torch.autograd.grad(loss, zr) if M > 3 else (torch.zeros_like(zr),)
    assert torch.all(dz[:3] == 0) and torch.isfinite(dz).all()


def test_targets_outside_the_vocabulary(dev):
    z = logits(dev, (6, 100), torch.float32).requires_grad_()
    t = torch.tensor([-1, 100, 2 ** 40, 5, -100, -2 ** 40], device=dev)
    r = tc.token_logprobs(z, t, entropy=True)
    assert torch.isnan(r.logprobs).tolist() == [True, True, True, False, False, True] and r.logprobs[4] == 0
    assert torch.isfinite(r.entropy).all()
    dz, = torch.autograd.grad(r.logprobs, z, torch.ones(6, device=dev))
    assert torch.isnan(dz).all(-1).tolist() == [True, True, True, False, False, True]
    assert torch.isnan(tc.token_cross_entropy(z, t))


@pytest.mark.parametrize("M,V", [(2, 40000), (300, 40000), (300, 9000)])
@pytest.mark.parametrize("kind", ["equal", "down", "up", "two", "columns", "zeros", "few"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_alternatives_of_unusual_rows(dev, kind, M, V, dtype):
    """Ties, sorted rows, rows whose best values all fall to a few threads, -0 beside 0, rows with fewer finite
    entries than alternatives."""
    k = 64
    j = torch.arange(V, device=dev, dtype=torch.float32)
    if kind == "equal":
        z = torch.full((V,), 1.5, device=dev)
    elif kind == "down":
        z = -j / 64
    elif kind == "up":
        z = j / 64
    elif kind == "two":
        z = torch.where(j % 3 == 1, 2.0, 1.0)
    elif kind == "columns":  # all of 63 threads' groups are larger than any other's
        n = 4 if dtype == torch.float32 else 8
        group = (j / n).floor()
        thread = torch.minimum(group % 1024 % 256, group % 1024)
        z = torch.where(thread < 63, 10.0, -10.0) + (j % 13) / 16
    elif kind == "zeros":
        z = torch.where(j % 2 == 0, -0.0, 0.0)
    else:
        z = torch.full((V,), -INF, device=dev)
        z[5::1000] = 3.0
    z = z.to(dtype).expand(M, V).contiguous()
    z[1:] = z[1:].roll(1, -1)
    t = targets(dev, (M,), V, drop=0.0)
    w = reference(z, t, k)
    r = tc.token_logprobs(z, t, top_k=k)
    assert torch.equal(r.top_ids, w["ids"])
    for kk in (1, 63):
        assert torch.equal(tc.token_logprobs(z, t, top_k=kk).top_ids, w["ids"][:, :kk])


@pytest.mark.parametrize("dtype", DT)
def test_strides_and_offsets(dev, dtype):
    """Rows at odd offsets and pitches, [B, T, V] slices, transposed and broadcast logits: the same bits as a copy."""
    big = logits(dev, (3, 9, 2060), dtype)
    for z in (big[:, :-1, 1:2050], big[:, ::2, 5:], big[0, 1:, 3:1004], big[1, 2], big.transpose(0, 1)[..., :1001],
              big[..., ::2], big[:1].expand(4, 9, 2060), big.reshape(3, 3, 3, 2060)[:, :, 1:, 7:]):
        V = z.shape[-1]
        t = targets(dev, tuple(z.shape[:-1]), V) if z.dim() > 1 else torch.tensor(17, device=dev)
        w = reference(z, t, 9)
        check_values(tc.token_logprobs(z, t, entropy=True, top_k=9), w, V)
        g = logits(dev, tuple(t.shape), torch.float32, 3) if t.dim() else torch.tensor(0.5, device=dev)
        a = z.detach().requires_grad_()
        r = tc.token_logprobs(a, t, entropy=True)
        dz, = torch.autograd.grad([r.logprobs, r.entropy], a, [g, g])
        assert dz.shape == z.shape
        check_grad(dz, w, t, g, g, V, dtype)


def test_long_offsets(dev):
    """Rows that lie behind 2^31 elements: a wide pitch over one large buffer."""
    V, pitch = 1000, 700_000_001
    buf = torch.zeros(3 * pitch + V, dtype=torch.bfloat16, device=dev)
    z = buf.as_strided((4, V), (pitch, 1))
    z.copy_(logits(dev, (4, V), torch.bfloat16))
    t = targets(dev, (4,), V, drop=0.0)
    w = reference(z.contiguous(), t, 5)
    zr = z.detach().requires_grad_()
    r = tc.token_logprobs(zr, t, entropy=True, top_k=5)
    check_values(r, w, V)
    g = torch.ones(4, device=dev)
    check_grad(torch.autograd.grad(r.logprobs, zr, g)[0], w, t, g, None, V, torch.bfloat16)


def test_empty(dev):
    r = tc.token_logprobs(torch.zeros(2, 0, 5, device=dev), torch.zeros(2, 0, dtype=torch.long, device=dev),
                          entropy=True, top_k=3)
    assert r.logprobs.shape == (2, 0) and r.entropy.shape == (2, 0) and r.top_ids.shape == (2, 0, 3)
    z = torch.zeros(0, 5, device=dev, requires_grad=True)
    loss = tc.token_cross_entropy(z, torch.zeros(0, dtype=torch.long, device=dev))
    assert torch.isnan(loss)
    assert torch.autograd.grad(loss, z)[0].shape == (0, 5)


def test_gradient_against_differences(dev):
    z, t = logits(dev, (3, 50), torch.float32, scale=1.0).requires_grad_(), targets(dev, (3,), 50, drop=0.0)
    c = logits(dev, (2, 3), torch.float32, 7)
    f = lambda x: (lambda r: (r.logprobs.double() * c[0] + r.entropy.double() * c[1]).sum())(  # noqa: E731
        tc.token_logprobs(x, t, entropy=True))
    got, = torch.autograd.grad(f(z), z)
    u = torch.randn(3, 50, device=dev, generator=torch.Generator(device=dev).manual_seed(0))
    h = 2.0 ** -6
    with torch.no_grad():
        d1, d2 = (f(z + s * h * u) - f(z - s * h * u) for s in (1, 2))
        diff = (8 * d1 - d2) / (12 * h)  # truncation h^4 f^(5) / 30
    # values of about 10 with errors of 100 F each, and h^4 times a fifth derivative below 1e4
    assert abs(diff - (got.double() * u).sum()) <= 9 * 100 * F * 10 / (12 * h) * 6 + h ** 4 * 1e4 / 30


def test_second_derivative(dev):
    z, t = logits(dev, (3, 20), torch.float32, scale=1.0).requires_grad_(), targets(dev, (3,), 20, drop=0.4)
    v = logits(dev, (3, 20), torch.float32, 9)

    def plain(x):
        logp = torch.log_softmax(x, -1)
        lp = logp.gather(-1, t.clamp(min=0)[:, None])[:, 0] * (t != -100)
        return lp.sum() + 0.5 * (-(logp.exp() * logp).sum(-1)).sum()

    def own(x):
        r = tc.token_logprobs(x, t, entropy=True)
        return r.logprobs.sum() + 0.5 * r.entropy.sum()

    both = []
    for f, x in ((plain, z.detach().double().requires_grad_()), (own, z)):
        first, = torch.autograd.grad(f(x), x, create_graph=True)
        both.append(torch.autograd.grad((first * v).sum(), x)[0])
    assert torch.allclose(both[1].double(), both[0], rtol=1e-4, atol=1e-5)  # fp32 products of values below 10
    x = z.detach().requires_grad_()
    loss = tc.token_cross_entropy(x, t)
    first, = torch.autograd.grad(loss, x, create_graph=True)
    y = x.detach().double().requires_grad_()
    ref, = torch.autograd.grad(torch.nn.functional.cross_entropy(y, t), y, create_graph=True)
    a, b = torch.autograd.grad((first * v).sum(), x)[0], torch.autograd.grad((ref * v).sum(), y)[0]
    assert torch.allclose(a.double(), b, rtol=1e-4, atol=1e-5)


def test_dispatched_op_agrees(dev):
    z, t = logits(dev, (5, 700), torch.bfloat16).requires_grad_(), targets(dev, (5,), 700)
    lp, ent, ids, top, _ = kl.logprob_fwd(z, t, True, 6, -100)
    r = tc.token_logprobs(z, t, entropy=True, top_k=6)
    assert all(torch.equal(a, b) for a, b in zip((lp, ent, ids, top), r))
    g = torch.ones(5, device=dev)
    for pair in (((lp, r.logprobs), g), ((ent, r.entropy), g)):
        a, b = (torch.autograd.grad(x, z, pair[1], retain_graph=True)[0] for x in pair[0])
        assert torch.equal(a, b)
    loss = kl.cross_entropy_fwd(z, t, -100, False)[0]
    own = tc.token_cross_entropy(z, t)
    assert torch.equal(loss, own)
    assert torch.equal(torch.autograd.grad(loss, z)[0], torch.autograd.grad(own, z)[0])


def test_entropy_gradient_without_a_target(dev):
    """The entropy's gradient alone does not look at the targets: any of them, the same bits."""
    z = logits(dev, (4, 300), torch.float32).requires_grad_()
    g = torch.tensor([1.0, -2.0, 0.5, 3.0], device=dev)
    grads = []
    for t in ([-100] * 4, [5, 300, -1, 1 << 40]):
        ent = tc.token_logprobs(z, torch.tensor(t, device=dev), entropy=True).entropy
        grads.append(torch.autograd.grad(ent, z, g)[0])
    assert torch.isfinite(grads[0]).all() and torch.equal(*grads)


@pytest.mark.parametrize("M,V", [(4, 30000), (600, 2000)])
def test_other_stream_and_graph(dev, M, V):
    z, t = logits(dev, (M, V), torch.bfloat16).requires_grad_(), targets(dev, (M,), V)

    def step():
        loss = tc.token_cross_entropy(z, t)
        dz, = torch.autograd.grad(loss, z)
        with torch.no_grad():
            r = tc.token_logprobs(z, t, entropy=True, top_k=5)
        return [loss.detach(), dz, *r]

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
        with torch.no_grad():
            z.copy_(logits(dev, (M, V), torch.bfloat16, seed + 10))
        t.copy_(targets(dev, (M,), V, seed + 10))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, step()))


def test_refusals(dev):
    z, t = torch.zeros(2, 10, device=dev), torch.zeros(2, dtype=torch.long, device=dev)
    for k in (-1, 11, 65):
        with pytest.raises(ValueError, match="top_k"):
            tc.token_logprobs(z, t, top_k=k)
    with pytest.raises(ValueError, match="top_k"):
        tc.token_logprobs(torch.zeros(2, 100, device=dev), t, top_k=65)
    with pytest.raises(RuntimeError, match="GPU|devices"):
        tc.token_logprobs(z, t.cpu())
    assert math.isfinite(float(tc.token_logprobs(z, t, top_k=10).logprobs.sum()))
