"""What a DecodeState keeps between calls, on the CPU."""
import pytest
import torch

import titans_core as tc
from titans_core.models.decoding import DecodeState


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


def test_drafts_of_which_little_is_kept(monkeypatch):
    """Paths as wide as their drafts, one row kept of each: the room holds as many as there are tokens."""
    state = (m := model(monkeypatch)).new_decode_state(2, 24)
    ids, tree = torch.zeros(2, 8, dtype=torch.long), torch.tensor([(1 << t + 1) - 1 for t in range(8)])
    path = torch.tensor([[0] + [-1] * 7, [0, 1] + [-1] * 6], dtype=torch.int32)
    for i in range(9):
        m.decode(ids, state, tree=tree)
        state.keep(path)
        assert state.lengths.tolist() == [i + 1, 2 * i + 2] and state.used >= 2 * i + 2
    with pytest.raises(ValueError, match="26 tokens do not fit in 24 .up to 18"):
        m.decode(ids, state, tree=tree)
    assert state.lengths.tolist() == [9, 18] and state.used >= 18
    m.decode(ids[:, :6], state)
    assert state.lengths.tolist() == [15, 24] and state.used == 24


def test_padding_is_not_held(monkeypatch):
    """Prompts of any lengths at the width of the longest."""
    m = model(monkeypatch, n_persistent=3)
    caches = [tc.KVCache.new(6, 2, 16, page=16, dtype=torch.float32, device="cpu") for _ in m.layers]
    state = DecodeState(caches, torch.zeros(2, 3, dtype=torch.int32), torch.full((2,), 3, dtype=torch.int32), 3, 20)
    ids = torch.zeros(2, 10, dtype=torch.long)
    for a, b in ((10, 1), (1, 10), (2, 5)):
        m.decode(ids, state, counts=torch.tensor([a, b], dtype=torch.int32))
    assert state.lengths.tolist() == [16, 19] and state.used == 16
    with pytest.raises(ValueError, match="21 tokens do not fit in 20 .up to 16"):
        m.decode(ids, state, counts=torch.tensor([8, 1], dtype=torch.int32))
    # a draft whose counts differ: what is held then is less than what was before it and the path's width
    m.decode(ids[:, :4], state, counts=torch.tensor([4, 1], dtype=torch.int32), tree=torch.tensor([1, 3, 7, 15]))
    state.keep(torch.tensor([[0], [0]], dtype=torch.int32))
    assert state.lengths.tolist() == [17, 20] and state.used >= 17


def test_a_capture_does_not_wait(monkeypatch):
    """Inside a capture the lengths cannot be looked at: the bound decides."""
    state = (m := model(monkeypatch)).new_decode_state(1, 10)
    ids = torch.zeros(1, 8, dtype=torch.long)
    m.decode(ids, state, counts=torch.ones(1, dtype=torch.int32))

    class OnGpu(torch.Tensor):
        is_cuda = True

    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    state.lengths = state.lengths.as_subclass(OnGpu)
    with pytest.raises(ValueError, match="16 tokens do not fit in 10 .up to 8"):
        m.decode(ids, state)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    m.decode(ids, state)
    assert state.used == 9


def test_inference_mode(monkeypatch):
    """A state that was made inside inference mode goes on outside it, and the other way round."""
    m = model(monkeypatch)
    ids = torch.zeros(2, 3, dtype=torch.long)
    for made, used in ((True, False), (False, True), (True, True)):
        with torch.inference_mode(made):
            state = m.new_decode_state(2, 20)
        with torch.inference_mode(used):
            m.decode(ids, state, counts=torch.tensor([3, 1], dtype=torch.int32))
        with torch.inference_mode(made):
            m.decode(ids, state, tree=torch.tensor([1, 3, 7]))
        with torch.inference_mode(used):
            state.keep(torch.tensor([[0], [1]], dtype=torch.int32))
        assert state.lengths.tolist() == [4, 2]
