"""The two ends of the TitanMAC model: the embedding and loss kernels against the modules they stand for (a
no-op hook puts the modules back), and score() against forward()'s logits."""
import pytest
import torch
import torch.nn.functional as F

import titans_core as tc

pytestmark = pytest.mark.gpu


def model(dev, variant, dtype=torch.float32, **kw):
    torch.manual_seed(3)
    cfg = dict(vocab_size=211, d_model=128, n_heads=2, n_layers=2, d_ff=256, max_seq_len=256, window_size=40,
               n_persistent=4, segment_size=32, n_memory_tokens=8, use_neural_memory=variant != "plain")
    cfg.update({} if variant == "plain" else {"titans_variant": variant}, **kw)
    m = tc.TitanMAC(tc.TitanMACConfig(**cfg)).to(dev, dtype).eval()
    with torch.no_grad():  # logits that differ
        m.embed_tokens.weight.mul_(8)
        if m.lm_head.weight is not m.embed_tokens.weight:
            m.lm_head.weight.mul_(8)
    return m


def tokens(dev, B=3, T=70, V=211):
    return torch.randint(0, V, (B, T), generator=torch.Generator().manual_seed(T)).to(dev)


VARIANTS = ["plain", "MAC", "MAG", "MAL"]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("variant", VARIANTS)
def test_kernels_and_modules_agree(dev, variant, dtype, monkeypatch):
    m, ids = model(dev, variant, dtype), tokens(dev)
    labels = ids.clone()
    labels[0, :9], labels[2] = -100, -100
    calls = []
    real = tc.models.titanmac.token_embedding
    monkeypatch.setattr(tc.models.titanmac, "token_embedding", lambda *a, **k: calls.append(1) or real(*a, **k))
    out = m(ids, labels=labels)
    out["loss"].backward()
    assert calls
    got = {n: p.grad for n, p in m.named_parameters() if p.grad is not None}
    m.zero_grad(set_to_none=True)
    del calls[:]
    hook = m.embed_tokens.register_forward_hook(lambda *_: None)
    logits = m(ids)["logits"]
    assert not calls  # the hooked module itself
    assert torch.equal(logits, out["logits"])
    ce = F.cross_entropy(logits[:, :-1].float().reshape(-1, 211), labels[:, 1:].reshape(-1))
    u = torch.finfo(dtype).eps / 2
    key = "loss" if variant == "plain" else "ce_loss"
    assert out[key].dtype == dtype
    assert abs(out[key].double() - ce.double()) <= (u + 2.0 ** -20) * 1.01 * ce.double()
    if variant == "plain":  # else the memory's loss is in one of the two
        ce.backward()
        for n, p in m.named_parameters():
            # both round the logits' gradient, and everything after it, to the type
            assert (got[n].double() - p.grad.double()).norm() <= (24 * u + 1e-5) * p.grad.double().norm(), n
    hook.remove()


@pytest.mark.parametrize("variant", VARIANTS)
def test_score(dev, variant):
    m, ids = model(dev, variant), tokens(dev)
    with torch.no_grad():
        logp = torch.log_softmax(m(ids)["logits"].double(), -1)
        r = m.score(ids, entropy=True, top_k=5)
        assert set(r) - {"memory_loss"} == {"logprobs", "entropy", "top_ids", "top_logprobs"}
        assert ("memory_loss" in r) == (variant != "plain")
        want = logp[:, :-1].gather(-1, ids[:, 1:, None])[..., 0]
        assert torch.allclose(r["logprobs"][:, :-1].double(), want, rtol=0, atol=1e-5)
        assert torch.all(r["logprobs"][:, -1] == 0)
        assert torch.allclose(r["entropy"].double(), -(logp.exp() * logp).sum(-1), rtol=0, atol=1e-5)
        assert torch.equal(r["top_ids"][..., 0], logp.argmax(-1))
        labels = ids.clone()
        labels[1, 3:9] = -100
        s = m.score(ids, labels)
        assert torch.all(s["logprobs"][1, 2:8] == 0)
        assert torch.allclose(s["logprobs"][0], r["logprobs"][0], rtol=0, atol=1e-5)
        assert m.score(ids[:, :1])["logprobs"].tolist() == [[0.0]] * 3
    with pytest.raises(ValueError, match="labels must be"):
        m.score(ids, ids[:, :-1])


@pytest.mark.parametrize("variant", ["plain", "MAC"])
def test_score_without_logits(dev, variant, monkeypatch):
    """16 bit: the scores come from the hidden states; nearer to the 64-bit head than the rounded logits."""
    m, ids = model(dev, variant, torch.bfloat16, tie_weights=False), tokens(dev)
    seen = []
    real = tc.models.titanmac.head_logprobs
    monkeypatch.setattr(tc.models.titanmac, "head_logprobs", lambda *a, **k: seen.append(a) or real(*a, **k))
    with torch.no_grad():
        r = m.score(ids, entropy=True)
        (h, w, t), = seen
        logp = torch.log_softmax(h.double() @ w.double().t(), -1)
        want = logp[:, :-1].gather(-1, ids[:, 1:, None])[..., 0]
        assert torch.allclose(r["logprobs"][:, :-1].double(), want, rtol=0, atol=1e-4)
        assert torch.allclose(r["entropy"].double(), -(logp.exp() * logp).sum(-1), rtol=0, atol=1e-4)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            a = m.float().score(ids)
        assert torch.allclose(a["logprobs"], r["logprobs"], atol=0.2)
    g = m.bfloat16().score(ids)["logprobs"]
    assert g.requires_grad
    g.sum().backward()
    assert torch.isfinite(m.lm_head.weight.grad).all() and m.lm_head.weight.grad.abs().sum() > 0


def test_score_updates_the_memory_as_forward_does(dev):
    a = model(dev, "MAC", enable_test_time_memory=True)
    b = model(dev, "MAC", enable_test_time_memory=True)
    ids = tokens(dev)
    with torch.no_grad():
        out, r = a(ids), b.score(ids)
    assert torch.equal(out["memory_loss"], r["memory_loss"])
    for (n, x), y in zip(a.neural_memory.state_dict().items(), b.neural_memory.state_dict().values()):
        assert torch.equal(x, y), n


def test_training_steps_in_a_graph(dev):
    """A captured training step, replayed with new tokens: the eager step's loss and gradients."""
    m = model(dev, "plain", torch.bfloat16, dropout=0.0).train()
    ids = tokens(dev)
    params = [m.embed_tokens.weight, m.embed_positions.weight, m.persistent_tokens]

    def step():
        loss = m(ids, labels=ids)["loss"]
        return [loss.detach(), *torch.autograd.grad(loss, params)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(3):
        ids.copy_(torch.randint(0, 211, ids.shape, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        assert torch.equal(held[0], want[0])
        for a, b in zip(held[1:], want[1:]):
            assert (a.double() - b.double()).norm() <= 2.0 ** -7 * b.double().norm()


def test_long_positions_are_refused(dev):
    m = model(dev, "plain")
    assert m._embed(tokens(dev, 1, 256)).shape == (1, 256, 128)
    with pytest.raises(ValueError, match="positions"):
        tc.token_embedding(tokens(dev, 1, 257), m.embed_tokens.weight, m.embed_positions.weight)
