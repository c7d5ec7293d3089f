"""What a DecodeState keeps between calls, on the CPU."""
import pytest
import torch

import titans_core as tc


def config(**kw):
    return tc.TitanMACConfig(**{**dict(vocab_size=20, d_model=32, n_heads=2, n_layers=2, d_ff=32, max_seq_len=64,
                                       n_persistent=0, window_size=4, use_block_sparse=False), **kw})


class Rows(torch.nn.Module):
    """A layer's place: it hands its input on, and refuses it if told to."""

    def __init__(self, layer):
        super().__init__()
        self.attention, self.refuse = layer.attention, False

    def forward_cached(self, x, cache, table, lengths, **kw):
        if self.refuse:
            raise ValueError("refused")
        self.seen = lengths.tolist()
        return x


def model(monkeypatch, **kw):
    """A model whose layers do nothing, so that it decodes here."""
    from titans_core.models import decoding
    monkeypatch.setattr(decoding, "cache_keep", lambda *a: None)
    m = tc.TitanMAC(config(**kw)).eval()
    m.layers = torch.nn.ModuleList(Rows(layer) for layer in m.layers)
    m.norm = torch.nn.Identity()
    return m


@pytest.mark.parametrize("which", ["first", "last", "head"])
def test_a_refused_call_leaves_the_state(monkeypatch, which):
    """Whoever refuses: the first layer, one behind layers that have run, the head."""
    m = model(monkeypatch)
    state = m.new_decode_state(2, 20)
    ids = torch.zeros(2, 3, dtype=torch.long)
    m.decode(ids, state)
    head = m.lm_head
    counts, tree = torch.tensor([3, 1], dtype=torch.int32), torch.tensor([1, 3, 7])
    for kw in ({}, {"counts": counts}, {"tree": tree}, {"counts": counts, "tree": tree}):
        if which == "head":
            m.lm_head = torch.nn.Linear(31, 20)
        else:
            m.layers[0 if which == "first" else 1].refuse = True
        with pytest.raises((ValueError, RuntimeError)):
            m.decode(ids, state, **kw)
        assert state.lengths.tolist() == [3, 3] and state.used == 3 and state._draft is None
        m.lm_head = head
        for layer in m.layers:
            layer.refuse = False
    assert m.decode(ids, state, counts=counts).shape == (2, 3, 20)
    assert m.layers[1].seen == state.lengths.tolist() == [6, 4] and state.used == 6


def test_refusals_of_the_operators(monkeypatch):
    """The layers themselves, which run on the GPU only."""
    m = tc.TitanMAC(config()).eval()
    state = m.new_decode_state(2, 20)
    for kw in ({}, {"tree": torch.tensor([1, 3, 7])}):
        with pytest.raises(RuntimeError, match="GPU"):
            m.decode(torch.zeros(2, 3, dtype=torch.long), state, **kw)
        assert state.lengths.tolist() == [0, 0] and state.used == 0 and state._draft is None
