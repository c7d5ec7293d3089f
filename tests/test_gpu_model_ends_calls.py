"""TitanMAC's loss and embeddings under calls that programs make around them."""
import pytest
import torch

import titans_core as tc

pytestmark = pytest.mark.gpu


@pytest.fixture
def model(dev):
    torch.manual_seed(0)
    cfg = tc.TitanMACConfig(vocab_size=101, d_model=64, n_heads=1, n_layers=1, d_ff=128, max_seq_len=64, window_size=16,
                            n_persistent=3, use_neural_memory=False)
    return tc.TitanMAC(cfg).to(dev).eval()


def test_logits_changed_before_the_backward(dev, model):
    """In place is refused, never answered with a gradient of the changed logits; a changed copy is a program's own."""
    ids = torch.randint(0, 101, (2, 20), device=dev)
    out = model(ids, labels=ids)
    out["loss"].backward()
    want = model.embed_tokens.weight.grad.clone()
    model.zero_grad(set_to_none=True)
    out = model(ids, labels=ids)
    out["logits"].clone().mul_(2)
    out["loss"].backward()
    assert torch.equal(model.embed_tokens.weight.grad, want)
    model.zero_grad(set_to_none=True)
    out = model(ids, labels=ids)
    out["logits"].mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out["loss"].backward()


def test_ids_and_labels_outside_the_vocabulary(dev, model):
    ids = torch.randint(0, 101, (2, 20), device=dev)
    labels = ids.clone()
    labels[1, 7] = 101
    with torch.no_grad():
        assert torch.isfinite(model(ids, labels=ids)["loss"]) and torch.isnan(model(ids, labels=labels)["loss"])
        labels[1, 7] = -100
        assert torch.isfinite(model(ids, labels=labels)["loss"])
        ids[0, 10] = 500
        logits = model(ids)["logits"]
    assert torch.isnan(logits[0, 10]).all() and torch.isfinite(logits[1]).all()


@pytest.mark.parametrize("B,T", [(300, 3), (1, 1), (2, 64)])
def test_training_against_the_modules(dev, model, B, T):
    """Many sequences (whose positions are summed in runs), a single token, the longest: the modules' gradients."""
    ids = torch.randint(0, 101, (B, T), generator=torch.Generator().manual_seed(B)).to(dev)
    model(ids)["logits"].square().mean().backward()
    got = {n: p.grad for n, p in model.named_parameters()}
    model.zero_grad(set_to_none=True)
    hook = model.embed_tokens.register_forward_hook(lambda *_: None)  # puts the modules back
    model(ids)["logits"].square().mean().backward()
    hook.remove()
    for n, p in model.named_parameters():
        # fp32: sums of up to 300 sequences in another order, after the same blocks
        assert (got[n].double() - p.grad.double()).norm() <= 1e-5 * p.grad.double().norm() + 1e-9, n
