"""Calls of TitanMAC.decode that are refused, the same calls again, and calls that are not to be refused."""
import pytest
import torch

from test_gpu_decoding import close, model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("why", ["dropout", "autocast", "type"])
@pytest.mark.parametrize("draft", [False, True])
def test_again_after_a_refusal(dev, why, draft):
    m = model(dev, attention_dropout=0.1)
    ids = torch.randint(0, 211, (2, 40), device=dev)
    with torch.no_grad():
        want = m(ids)["logits"]
    state = m.new_decode_state(2, 64)
    m.decode(ids[:, :20], state)
    tree = torch.tensor([(1 << t + 1) - 1 for t in range(6)], device=dev) if draft else None
    args = (ids[:, 20:26], state)
    if why == "dropout":
        m.train()
        with pytest.raises(ValueError, match="dropout"):
            m.decode(*args, tree=tree)
        m.eval()
    elif why == "autocast":
        with torch.autocast("cuda", dtype=torch.bfloat16), pytest.raises(TypeError, match="does not hold"):
            m.decode(*args, tree=tree)
    else:
        m.double()
        with pytest.raises((TypeError, RuntimeError, ValueError)):
            m.decode(*args, tree=tree)
        m.float()
    assert state.lengths.tolist() == [25, 25] and state.used == 20
    got = [m.decode(*args, tree=tree)]
    if draft:
        state.keep(torch.arange(6, dtype=torch.int32, device=dev).expand(2, 6))
    got.append(m.decode(ids[:, 26:], state))
    assert close(torch.cat(got, 1), want[:, 20:], torch.float32) and state.used == 40


def test_many_drafts_in_a_small_room(dev):
    """Drafts of six tokens of which two stay, by paths as wide as the drafts: the room holds what is kept."""
    m = model(dev)
    ids = torch.randint(0, 211, (2, 40), device=dev)
    with torch.no_grad():
        want = m(ids)["logits"]
    state = m.new_decode_state(2, 40, page=16)
    got = [m.decode(ids[:, :20], state)]
    tree = torch.tensor([0b1, 0b10, 0b101, 0b1010, 0b10, 0b10001], device=dev)
    path = torch.tensor([[0, 2, -1, -1, -1, -1]], dtype=torch.int32, device=dev).expand(2, 6)
    for at in range(20, 36, 2):
        draft = torch.randint(0, 211, (2, 6), device=dev)
        draft[:, 0], draft[:, 2] = ids[:, at], ids[:, at + 1]
        got.append(m.decode(draft, state, tree=tree)[:, [0, 2]])
        state.keep(path)
    with pytest.raises(ValueError, match="42 tokens do not fit in 40"):
        m.decode(draft, state, tree=tree)
    got.append(m.decode(ids[:, 36:], state))
    assert close(torch.cat(got, 1), want, torch.float32) and state.used == 40


@pytest.mark.parametrize("narrow", [("embed_positions",), ("embed_tokens",), ("embed_tokens", "embed_positions"), ("rows",),
                                    ("embed_tokens", "embed_positions", "rows")])
def test_tables_of_several_types(dev, narrow):
    """Tables in bfloat16 beside layers in fp32, as forward takes them: what a row is embedded as is of the widest."""
    m = model(dev, tie_weights=False)
    for name in narrow:
        if name == "rows":
            m.persistent_tokens.data = m.persistent_tokens.data.bfloat16()
        else:
            getattr(m, name).bfloat16()
    ids = torch.randint(0, 211, (2, 40), device=dev)
    if len(narrow) == 3:  # then all of a text's rows are bfloat16, which the layers refuse
        with torch.no_grad(), pytest.raises((RuntimeError, TypeError, ValueError)):
            m(ids)
        with pytest.raises((RuntimeError, TypeError, ValueError)):
            m.decode(ids, m.new_decode_state(2))
        return
    with torch.no_grad():
        want = m(ids)["logits"]
    state = m.new_decode_state(2)
    got = torch.cat([m.decode(ids[:, a:b], state) for a, b in ((0, 25), (25, 26), (26, 40))], 1)
    assert close(got, want, torch.float32)


def test_inference_mode(dev):
    """A state made inside inference mode, used outside it and inside."""
    m = model(dev)
    ids = torch.randint(0, 211, (2, 40), device=dev)
    with torch.inference_mode():
        want = m(ids)["logits"]
        state = m.new_decode_state(2)
    got = [m.decode(ids[:, :20], state)]
    with torch.inference_mode():
        got.append(m.decode(ids[:, 20:21], state))
    got.append(m.decode(ids[:, 21:], state))
    assert close(torch.cat(got, 1), want, torch.float32)
