"""Refusals, argument errors, shapes under tracing and the differentiable gradients of the token operators, on
the CPU."""
import ctypes

import pytest
import torch

import titans_core as tc
from titans_core.kernels import _lib
from titans_core.kernels import embedding as ke
from titans_core.kernels import logprobs as kl

FAKE = 1 << 20
SZ = ctypes.POINTER(ctypes.c_size_t)


def test_embedding_refusals():
    ids, w, p = torch.zeros(2, 3, dtype=torch.long), torch.zeros(5, 8), torch.zeros(4, 8)
    with pytest.raises(RuntimeError, match="GPU"):
        tc.token_embedding(ids, w, p)
    bad = [
        (ValueError, "ids must be", (ids[0], w), {}),
        (TypeError, "ids must be", (ids.float(), w), {}),
        (ValueError, "weight must be", (ids, w[0]), {}),
        (ValueError, "weight must be", (ids, w[:0]), {}),
        (ValueError, "pos_weight must be", (ids, w, p[:, :4]), {}),
        (TypeError, "pos_weight dtype", (ids, w, p.double()), {}),
        (ValueError, "3 positions", (ids, w, p[:2]), {}),
        (ValueError, "no rows", (ids, w, p[:0]), {"positions": ids}),
        (ValueError, "positions need", (ids, w), {"positions": ids}),
        (ValueError, "positions must be", (ids, w, p), {"positions": ids[:, :2]}),
        (TypeError, "positions must be", (ids, w, p), {"positions": ids.float()}),
        (ValueError, "prefix must be", (ids, w, p), {"prefix": p[0]}),
        (TypeError, "prefix dtype", (ids, w, p), {"prefix": p.half()}),
        (TypeError, "unsupported dtype", (ids, w.double()), {}),
    ]
    for err, text, args, kw in bad:
        with pytest.raises(err, match=text):
            tc.token_embedding(*args, **kw)


def test_logprob_refusals():
    z, t = torch.zeros(2, 10), torch.zeros(2, dtype=torch.long)
    for f in (tc.token_logprobs, tc.token_cross_entropy):
        with pytest.raises(RuntimeError, match="GPU"):
            f(z, t)
        with pytest.raises(ValueError, match="targets must be"):
            f(z, t[:1])
        with pytest.raises(ValueError, match="logits must be"):
            f(z[:, :0], t)
        with pytest.raises(TypeError, match="targets must be"):
            f(z, t.float())
        with pytest.raises(TypeError, match="unsupported dtype"):
            f(z.double(), t)
    for k in (-1, 11):
        with pytest.raises(ValueError, match="top_k"):
            tc.token_logprobs(z, t, top_k=k)
    with pytest.raises(ValueError, match="top_k"):
        tc.token_logprobs(torch.zeros(2, 100), t, top_k=65)


def test_sizes_past_the_kernels_integers_are_refused():
    """More rows than the kernels count in 32 bits: refused by shape, before anything is read."""
    one = torch.zeros(1, dtype=torch.bfloat16)
    for n in ((1 << 30) + 1, (1 << 32) + 5):
        ids, z = torch.zeros(1, dtype=torch.long).expand(n), one.expand(n, 1)
        for f in (tc.token_logprobs, tc.token_cross_entropy):
            with pytest.raises(ValueError, match="rows"):
                f(z, ids)
        with pytest.raises(ValueError, match="rows"):
            tc.head_logprobs(one.expand(n, 64), one.expand(10, 64), ids)
        w = one.expand(5, 8)
        for args, kw in (((ids.view(n, 1), w), {}), ((ids.view(1, n), w), {}), ((ids[:0].expand(n, 0), w), {}),
                         ((ids[:0].expand(n, 0), w), {"prefix": w[:1]}), ((ids[:1].view(1, 1), one.expand(n, 8)), {}),
                         ((ids[:1].view(1, 1), w, one.expand(n, 8)), {}), ((ids[:1].view(1, 1), one.expand(5, n)), {})):
            with pytest.raises(ValueError, match="rows"):
                tc.token_embedding(*args, **kw)
    for f in (tc.token_logprobs, tc.token_cross_entropy):
        with pytest.raises(ValueError, match="vocabulary"):
            f(one.expand(2, (1 << 28) + 1), torch.zeros(2, dtype=torch.long))


def test_fake_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        ids, w = torch.zeros(2, 3, dtype=torch.long), torch.zeros(5, 8, dtype=torch.bfloat16)
        y, lists = ke.token_embedding_fwd(ids, w, None, None, w[:4], 1.0, True)
        assert lists.shape == (32 + 2 * 32,) and lists.dtype == torch.uint8
        assert ke.token_embedding_fwd(ids, w, None, None, w[:4], 1.0, False)[1].shape == (0,)
        assert y.shape == (2, 7, 8) and y.dtype == torch.bfloat16
        dw, dp, df = ke.token_embedding_bwd(y, ids, None, lists, 4, 5, 0, 1.0, True, False, True)
        assert (dw.shape, dp.shape, df.shape) == ((5, 8), (0, 8), (4, 8))
        z = torch.zeros(2, 3, 100, dtype=torch.float16)
        lp, ent, top_ids, top, stats = kl.logprob_fwd(z, ids, False, 6, -100)
        assert (lp.shape, ent.shape, top_ids.shape, top.shape, stats.shape) == (
            (2, 3), (0,), (2, 3, 6), (2, 3, 6), (6, 2))
        assert lp.dtype == torch.float32 and top_ids.dtype == torch.int64
        assert kl.logprob_bwd(lp, None, z, ids, stats, ent, -100).dtype == torch.float16
        loss, inv, _ = kl.cross_entropy_fwd(z, ids, -100, False)
        assert loss.shape == () and loss.dtype == torch.float16 and inv.dtype == torch.float32


def test_embedding_argument_errors(lib):
    n = ctypes.c_size_t(0)
    for tokens, V in ((0, 1), (1, 3), (6, 100), (32768, 128000), (7, 4)):
        assert lib.tmac_embed_lists_bytes(tokens, V, ctypes.byref(n)) == 0 and n.value == ke._lists_bytes(tokens, V)
    assert lib.tmac_embed_lists_bytes(6, 0, ctypes.byref(n)) == -2 and lib.tmac_embed_lists_bytes(6, 1, None) == -1
    lib.tmac_embed_lists_bytes(6, 100, ctypes.byref(n))
    # ids, pos, W, ldw, P, ldp, prefix, ldpre, out, lists, bytes, B, T, n_prefix, d, V, n_pos, scale, dtype, stream
    ok = [FAKE, None, FAKE, 64, FAKE, 64, FAKE, 64, FAKE, FAKE, n.value, 2, 3, 4, 64, 100, 50, 1.0, 1, None]
    for at, value, want in ((0, None, -1), (2, None, -1), (8, None, -1), (6, None, -1), (3, 63, -2), (5, 63, -2),
                            (7, 63, -2), (11, -1, -2), (14, 0, -2), (14, (1 << 20) + 1, -2), (15, 0, -2),
                            (15, (1 << 30) + 1, -2), (16, 2, -2), (18, 3, -4), (12, 1 << 30, -2),
                            (10, n.value - 1, -6), (9, FAKE + 8, -5)):
        bad = list(ok)
        bad[at] = value
        assert lib.tmac_embed_fwd(*bad) == want, (at, value)
    empty = list(ok)
    empty[9], empty[11] = None, 0
    assert lib.tmac_embed_fwd(*empty) == 0
    n = ctypes.c_size_t(0)
    assert lib.tmac_embed_bwd_workspace(1000, 50, 0, 64, ctypes.byref(n)) == 0 and n.value >= 4 * (51 + 2000) + 2 * 16 * 64 * 4
    assert lib.tmac_embed_bwd_workspace(1000, -1, 0, 64, ctypes.byref(n)) == -2
    assert lib.tmac_embed_bwd_workspace(1000, 50, (1 << 30) + 1, 64, ctypes.byref(n)) == -2
    assert lib.tmac_embed_bwd_workspace(1000, 50, 0, 64, None) == -1
    lib.tmac_embed_bwd_workspace(6, 100, 50, 64, ctypes.byref(n))
    # ids, pos, lists, g, ldg, dW, dP, dprefix, ws, ws_bytes, B, T, n_prefix, d, V, n_pos, scale, dtype, stream
    ok = [FAKE, FAKE, None, FAKE, 64, FAKE, FAKE, FAKE, FAKE, n.value, 2, 3, 4, 64, 100, 50, 1.0, 1, None]
    for at, value, want in ((0, None, -1), (3, None, -1), (8, None, -6), (9, n.value - 1, -6), (8, FAKE + 4, -5),
                            (4, 63, -2), (14, 0, -2), (15, 0, -2), (17, 9, -4), (13, 0, -2), (12, 0, -2), (10, -1, -2),
                            (2, FAKE + 8, -5)):
        bad = list(ok)
        bad[at] = value
        assert lib.tmac_embed_bwd(*bad) == want, (at, value)
    bad = list(ok)
    bad[1], bad[15] = None, 2  # fewer position rows than positions
    assert lib.tmac_embed_bwd(*bad) == -2


def test_logprob_argument_errors(lib):
    n = ctypes.c_size_t(0)
    assert lib.tmac_logprob_workspace(1, 4, 128000, 5, 1, ctypes.byref(n)) == 0 and n.value > 0
    # z, stride_b, stride_t, targets, ignore, lp, ent, top_k, top_ids, top_lp, stats, ws, ws_bytes, B, T, V, dtype, stream
    ok = [FAKE, 0, 128000, FAKE, -100, FAKE, FAKE, 5, FAKE, FAKE, FAKE, FAKE, n.value, 1, 4, 128000, 1, None]
    for at, value, want in ((0, None, -1), (3, None, -1), (5, None, -1), (8, None, -1), (9, None, -1), (10, None, -1),
                            (11, None, -6), (12, n.value - 1, -6), (11, FAKE + 8, -5), (0, FAKE + 1, -5), (7, 65, -8),
                            (7, -1, -8), (2, -1, -2), (13, -1, -2), (15, 0, -2), (15, (1 << 28) + 1, -2), (16, 4, -4)):
        bad = list(ok)
        bad[at] = value
        assert lib.tmac_logprob_fwd(*bad) == want, (at, value)
    bad = list(ok)
    bad[15] = 4  # fewer entries than alternatives
    assert lib.tmac_logprob_fwd(*bad) == -8
    # z, stride_b, stride_t, targets, ignore, stats, ent, g_lp, st, g_ent, st, dz, B, T, V, dtype, stream
    ok = [FAKE, 0, 100, FAKE, -100, FAKE, FAKE, FAKE, 1, FAKE, 1, FAKE, 1, 4, 100, 0, None]
    for at, value, want in ((0, None, -1), (3, None, -1), (5, None, -1), (6, None, -1), (11, None, -1), (0, FAKE + 2, -5),
                            (11, FAKE + 1, -5), (14, 0, -2), (15, 3, -4)):
        bad = list(ok)
        bad[at] = value
        assert lib.tmac_logprob_bwd(*bad) == want, (at, value)
    # lp, targets, ignore, rows, loss, dtype, neg_inv, stream
    ok = [FAKE, FAKE, -100, 4, FAKE, 1, FAKE, None]
    for at, value, want in ((0, None, -1), (1, None, -1), (4, None, -1), (6, None, -1), (3, -1, -2), (5, 3, -4)):
        bad = list(ok)
        bad[at] = value
        assert lib.tmac_logprob_mean(*bad) == want, (at, value)


def test_differentiable_gradients_match_autograd():
    """The gradients in torch's operations (for second derivatives) against autograd of the plain formulas."""
    torch.manual_seed(0)
    z = torch.randn(4, 9).requires_grad_()
    z.data[1, 3] = float("-inf")
    t = torch.tensor([2, 5, -100, 8])
    gl, ge = torch.randn(4), torch.randn(4)
    logp = torch.log_softmax(z, -1)
    p = logp.exp()
    H = -(p * torch.where(p > 0, logp, 0.0)).sum(-1)
    lp = logp.gather(-1, t.clamp(min=0)[:, None])[:, 0] * (t != -100)
    want, = torch.autograd.grad([lp, H], z, [gl, ge])
    want[1, 3] = 0  # the masked entry
    got = kl._composed(gl, ge, z.detach(), t, -100)
    assert torch.allclose(got, want, rtol=1e-5, atol=1e-6)
    ids = torch.tensor([[0, 2, 2], [4, 7, -1]])
    g = torch.randn(2, 5, 6)
    dw, dp, df = ke._composed(g, ids, None, None, 2, 5, 4, 0.5, True, True, True)
    body = g[:, 2:]
    assert torch.allclose(dw[2], 0.5 * (body[0, 1] + body[0, 2])) and torch.allclose(dw[4], 0.5 * body[1, 0])
    assert torch.all(dw[[1, 3]] == 0) and torch.allclose(dw[0], 0.5 * body[0, 0])
    assert torch.allclose(dp[:3], body.sum(0)) and torch.all(dp[3] == 0)
    assert torch.allclose(df, g[:, :2].sum(0))


def test_differentiable_gradient_of_ignored_and_refused_rows():
    """Ignored rows are zeros and not read, a target outside the vocabulary makes its row NaN: in the differentiable
    form as in the kernel, the loss without any target (a gradient of NaN) among them."""
    z, t = torch.randn(3, 5), torch.tensor([1, -100, 7])
    z[1, 2] = float("nan")
    z.requires_grad_()
    gl = torch.tensor([1.0, float("nan"), 1.0])
    first = kl._composed(gl, None, z, t, -100)
    assert torch.all(first[1] == 0) and torch.isfinite(first[0]).all() and torch.isnan(first[2]).all()
    second, = torch.autograd.grad((first[:2] * torch.randn(2, 5)).sum(), z)
    assert torch.all(second[1] == 0) and torch.isfinite(second[0]).all()
    assert torch.all(kl._composed(torch.full((3,), float("nan")), None, z, torch.full((3,), -100), -100) == 0)
    # the entropy's gradient does not look at the target
    only = kl._composed(None, torch.ones(3), z, t, -100)
    assert torch.isfinite(only[[0, 2]]).all() and torch.isnan(only[1]).all()


def test_exported_from_the_package():
    assert _lib.SIGNATURES["tmac_embed_fwd"] and set(tc.__all__) >= {
        "token_embedding", "token_logprobs", "token_cross_entropy", "TokenLogprobs"}


def test_head_refusals_and_argument_errors(lib):
    x, w, t = torch.zeros(2, 64).bfloat16(), torch.zeros(5, 64).bfloat16(), torch.zeros(2, dtype=torch.long)
    with pytest.raises(RuntimeError, match="GPU"):
        tc.head_logprobs(x, w, t)
    with pytest.raises(RuntimeError, match="GPU"):
        tc.head_logprobs(x.float(), w.float(), t)
    for err, text, args in ((ValueError, "hidden must be", (x[:, :32], w, t)), (ValueError, "hidden must be", (x, w[:0], t)),
                            (ValueError, "hidden must be", (x, w[0], t)), (TypeError, "weight dtype", (x, w.half(), t)),
                            (ValueError, "targets must be", (x, w, t[:1])), (TypeError, "targets must be", (x, w, t.float()))):
        with pytest.raises(err, match=text):
            tc.head_logprobs(*args)
    n = ctypes.c_size_t(0)
    assert lib.tmac_head_logprob_workspace(300, 1000, 640, ctypes.byref(n)) == 0 and n.value >= 300 * 16
    assert lib.tmac_head_logprob_workspace(300, 1000, 640, None) == -1
    # X, ldx, W, ldw, targets, ignore, lp, ent, M, V, K, ws, ws_bytes, dtype, stream
    ok = [FAKE, 640, FAKE, 640, FAKE, -100, FAKE, None, 300, 1000, 640, FAKE, n.value, 1, None]
    for at, value, want in ((0, None, -1), (2, None, -1), (4, None, -1), (6, None, -1), (11, None, -6),
                            (12, n.value - 1, -6), (11, FAKE + 8, -5), (0, FAKE + 8, -5), (2, FAKE + 2, -5), (1, 632, -2),
                            (3, 644, -5), (1, (1 << 22) + 8, -2), (10, 600, -2), (10, 0, -2), (9, 0, -2),
                            (9, (1 << 28) + 1, -2), (8, -1, -2), (13, 0, -4)):
        bad = list(ok)
        bad[at] = value
        assert lib.tmac_head_logprob(*bad) == want, (at, value)
    for M in (1, 64, 65, 8192, 1 << 30):
        for V in (1, 129, 128000, 1 << 28):
            assert lib.tmac_head_logprob_workspace(M, V, 64, ctypes.byref(n)) == 0 and n.value >= 16 * M
