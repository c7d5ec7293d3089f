"""TitanMAC.decode and generate against the model's own forward over the whole text."""
import pytest
import torch

import titans_core as tc

pytestmark = pytest.mark.gpu

E = 2.0 ** -24


def model(dev, dtype=torch.float32, seed=0, **kw):
    torch.manual_seed(seed)
    cfg = dict(vocab_size=211, d_model=128, n_heads=2, n_layers=3, d_ff=256, max_seq_len=96, window_size=20,
               n_persistent=5, use_block_sparse=False)
    m = tc.TitanMAC(tc.TitanMACConfig(**{**cfg, **kw}))
    with torch.no_grad():  # embeddings and persistent rows that the layers can tell apart
        for p in (m.embed_tokens.weight, m.embed_positions.weight, m.persistent_tokens):
            if p is not None:
                p.normal_()
        m.lm_head.weight.mul_(0.1)
    return m.to(dev, dtype).eval()


def close(a, b, dtype, layers=3):
    """Both run the same layers; attention's order of sums and the library's products by shape differ. Each of the about
    ten operations of a layer adds less than 512 E of its result in fp32, half a step of 2^-8 in bfloat16, and hands
    on what came in at no more than its own size."""
    ops = 10 * layers + 3
    tol = ops * (512 * E if dtype == torch.float32 else 2.0 ** -8)
    return (a.float() - b.float()).norm() <= tol * b.float().norm()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kw", [{}, {"n_persistent": 0}, {"n_heads": 4, "window_size": 200}, {"d_model": 80, "n_heads": 2},
                                {"mlp_block_ell": True}])
def test_decode_is_forward(dev, dtype, kw):
    m = model(dev, dtype, **kw)
    ids = torch.randint(0, 211, (3, 90), device=dev)
    with torch.no_grad():
        want = m(ids)["logits"]
    for parts in ([90], [1] * 12 + [78], [40, 1, 1, 33, 15]):
        state = m.new_decode_state(3, 90, page=16)
        got, at = [], 0
        for n in parts:
            got.append(m.decode(ids[:, at:at + n], state))
            at += n
        got = torch.cat(got, 1)
        assert got.shape == want.shape and close(got, want, dtype)
    state = m.new_decode_state(3)
    assert close(m.decode(ids, state, last=True), want[:, -1:], dtype)
    if dtype == torch.float32 and not kw:  # the bound tells a wrong window from the right one
        m.layers[0].attention.window_size += 1
        assert not close(m.decode(ids, m.new_decode_state(3)), want, dtype)


def test_padded_prompts(dev):
    m = model(dev)
    ids = torch.randint(0, 211, (3, 50), device=dev)
    counts = torch.tensor([50, 17, 1], dtype=torch.int32, device=dev)
    state = m.new_decode_state(3)
    logits = m.decode(ids, state, counts=counts)
    last = m.decode(ids, m.new_decode_state(3), counts=counts, last=True)
    nxt = torch.randint(0, 211, (3, 4), device=dev)
    more = m.decode(nxt, state)
    with torch.no_grad():
        for b, n in enumerate(counts.tolist()):
            want = m(torch.cat([ids[b:b + 1, :n], nxt[b:b + 1]], 1))["logits"]
            assert close(torch.cat([logits[b:b + 1, :n], more[b:b + 1]], 1), want, torch.float32)
            assert close(last[b:b + 1], want[:, n - 1:n], torch.float32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_drafts(dev, dtype):
    """Two branches behind a prompt; the branch that is kept goes on as if it had been decoded alone."""
    m = model(dev, dtype)
    text = torch.randint(0, 211, (2, 40), device=dev)
    wrong = torch.randint(0, 211, (2, 3), device=dev)
    draft = torch.stack([text[:, 30], wrong[:, 0], text[:, 31], wrong[:, 1], wrong[:, 2], text[:, 32]], 1)
    tree = torch.tensor([0b1, 0b10, 0b101, 0b1010, 0b10001, 0b100101], device=dev)
    path = torch.tensor([[0, 2, 5], [0, 2, -1]], dtype=torch.int32, device=dev)
    with torch.no_grad():
        want = m(text)["logits"]
    state = m.new_decode_state(2, 64)
    m.decode(text[:, :30], state)
    got = m.decode(draft, state, tree=tree)
    assert close(got[:, [0, 2, 5]], want[:, 30:33], dtype)
    with pytest.raises(RuntimeError, match="keep"):
        m.decode(text[:, :1], state)
    state.keep(path)
    assert state.lengths.tolist() == [5 + 33, 5 + 32] and state.used == 33
    rest = torch.stack([text[0, 33:39], text[1, 32:38]])
    got = m.decode(rest, state)
    assert close(got[0], want[0, 33:39], dtype) and close(got[1], want[1, 32:38], dtype)
    with pytest.raises(RuntimeError, match="draft"):
        state.keep(path)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_caches_in_8_bits(dev, fmt):
    """The same layers on keys and values that are off by half a step of their format (int8: of the row's largest)."""
    m = model(dev)
    ids = torch.randint(0, 211, (2, 60), device=dev)
    with torch.no_grad():
        want = m(ids)["logits"]
    state = m.new_decode_state(2, fmt=fmt)
    got = torch.cat([m.decode(ids[:, a:b], state) for a, b in ((0, 30), (30, 31), (31, 60))], 1)
    # half a step in each of three layers, of the keys (scores of the size of 10 move by that part) and the values
    step = 1 / 254 if fmt == "int8" else 2.0 ** -4
    assert (got - want).norm() <= 3 * (10 + 1) * step * want.norm()
    assert state.caches[0].k.dtype == (torch.int8 if fmt == "int8" else torch.float8_e4m3fn)


def test_generate(dev):
    m = model(dev)
    ids = torch.randint(0, 211, (2, 20), device=dev)
    counts = torch.tensor([20, 9], dtype=torch.int32, device=dev)
    got = m.generate(ids, 25, counts=counts)
    assert got.shape == (2, 25) and got.dtype == torch.int64
    with torch.no_grad():
        for b, n in enumerate(counts.tolist()):
            text = torch.cat([ids[b, :n], got[b]])[None]
            logits = m(text)["logits"][0, n - 1:-1]
            best = logits.max(-1).values
            taken = logits.gather(1, got[b][:, None])[:, 0]
            # the likeliest token by forward's logits, but for ties within the two paths' rounding
            assert torch.all(best - taken <= 33 * 512 * E * logits.norm(dim=-1))
    assert m.generate(ids, 0).shape == (2, 0)


def test_captured_steps(dev):
    """One token of each sequence as a graph: lengths, caches and logits move on by themselves."""
    m = model(dev, torch.bfloat16)
    ids = torch.randint(0, 211, (4, 30), device=dev)
    eager, held = m.new_decode_state(4), m.new_decode_state(4)
    for s in (eager, held):
        m.decode(ids[:, :20], s)
    token = ids[:, 20:21].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m.decode(token, held)  # what is set up in a first call
    torch.cuda.current_stream().wait_stream(side)
    held.lengths.sub_(1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m.decode(token, held)
    for t in range(20, 28):
        token.copy_(ids[:, t:t + 1])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, m.decode(ids[:, t:t + 1], eager)), t
        assert torch.equal(held.lengths, eager.lengths)


def test_a_draft_s_counts_are_the_state_s(dev):
    """The counts of a draft may be in a buffer that is used again; a path longer than a sequence's draft keeps no more."""
    m = model(dev)
    ids = torch.randint(0, 211, (2, 30), device=dev)
    tree = torch.tensor([0b1, 0b11, 0b111], device=dev)
    counts = torch.tensor([3, 2], dtype=torch.int32, device=dev)
    state = m.new_decode_state(2, 64)
    m.decode(ids[:, :20], state)
    m.decode(ids[:, 20:23], state, counts=counts, tree=tree)
    counts.fill_(1)
    state.keep(torch.tensor([[0, 1, 2], [0, 1, 2]], dtype=torch.int32, device=dev))
    assert state.lengths.tolist() == [5 + 23, 5 + 22]
    rest = torch.stack([ids[0, 23:28], ids[1, 22:27]])
    got = m.decode(rest, state)
    with torch.no_grad():
        want = m(ids)["logits"]
    assert close(got[0], want[0, 23:28], torch.float32) and close(got[1], want[1, 22:27], torch.float32)


@pytest.mark.parametrize("fmt", [None, "int8"])
def test_inside_autocast(dev, fmt):
    """As forward inside it: projections and caches in bfloat16 (or codes of it), the rest as the parameters are."""
    m = model(dev)
    ids = torch.randint(0, 211, (2, 40), device=dev)
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        want = m(ids)["logits"]
        state = m.new_decode_state(2, fmt=fmt)
        got = torch.cat([m.decode(ids[:, a:b], state) for a, b in ((0, 25), (25, 26), (26, 40))], 1)
        assert m.generate(ids, 3, fmt=fmt).shape == (2, 3)
    assert state.caches[0].k.dtype == (torch.bfloat16 if fmt is None else torch.int8) and got.dtype == want.dtype
    if fmt is None:
        assert close(got, want, torch.bfloat16)
    else:  # int8 rows are off by half of a 127th of the row's largest value, a bfloat16 step's size
        assert (got.float() - want.float()).norm() <= (33 * 2.0 ** -8 + 3 * 11 / 254) * want.float().norm()
