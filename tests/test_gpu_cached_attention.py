"""cached_attention against softmax(q·kᵀ·scale)·v in 64 bits, and against windowed_attention."""
import math
import threading

import pytest
import torch

import titans_core as tc
from cache_cases import FORMATS, E, check_attention, empty_cache, filled, gen, make_table, pool_rows, seen_by

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
NAN = math.nan


def queries(dev, B, H, T, d, dtype, seed=9, spread=1.0):
    return (torch.randn(B, T, H, d, generator=gen(dev, seed), device=dev) * spread).to(dtype).transpose(1, 2)


def run(dev, B, H, heads, d, page, lens, news, T, window, n_persistent, dtype, fmt, tree=None, spread=1.0, scale=None,
        seed=0):
    # what is not held is NaN, and so are the codes and scales there
    c, table, lengths = filled(dev, B, heads, d, page, lens, dtype, fmt, seed, spread, fill=NAN)
    q = queries(dev, B, H, T, d, dtype, seed + 7, spread)
    counts = torch.tensor(news, dtype=torch.int32, device=dev)
    o = tc.cached_attention(q, c, table, lengths, window, n_persistent, counts=counts, tree=tree, scale=scale)
    assert o.shape == (B, H, T, d) and o.dtype == dtype
    masks = seen_by(B, T, lens, news, window, n_persistent, None if tree is None else tree.cpu())
    check_attention(o, q, c, table, lens, news, masks, scale)
    return o, q, c, table, lengths, counts


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,heads,d", [(10, 10, 64), (8, 2, 128), (7, 1, 40), (3, 3, 1), (4, 2, 33), (32, 8, 96)])
def test_single_tokens(dev, H, heads, d, dtype, fmt):
    lens = [1, 2, 31, 32, 33, 64, 100, 257, 0, 300]
    news = [1, 1, 1, 1, 1, 1, 1, 1, 0, 0]
    for window, n_persistent, page in ((None, 0, 16), (50, 5, 64), (0, 0, 32), (37, 33, 16), (1, 300, 128)):
        run(dev, len(lens), H, heads, d, page, lens, news, 1, window, n_persistent, dtype, fmt)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,heads,d,T", [(2, 2, 64, 2), (4, 2, 64, 9), (3, 3, 128, 17), (5, 1, 40, 64), (2, 1, 64, 100),
                                         (1, 1, 33, 130), (64, 8, 64, 130), (64, 8, 128, 70), (40, 8, 40, 100),
                                         (32, 32, 96, 90)])
def test_chunks(dev, H, heads, d, T, dtype, fmt):
    """Chunks that begin at every place: in the persistent rows, behind them, far behind; fewer rows than T."""
    lens = [T, T + 1, T + 40, 200, 131, T]
    news = [T, T, T, T, T // 2, 0]
    for window, n_persistent, page in ((None, 0, 64), (33, 4, 16), (64, 20, 32)):
        run(dev, len(lens), H, heads, d, page, lens, news, T, window, n_persistent, dtype, fmt)


def trees(dev, B, T, seed, shape):
    g = torch.Generator().manual_seed(seed)
    rows = []
    for _ in range(B):
        bits = []
        for t in range(T):
            if shape == "tree":
                parent = int(torch.randint(-1, t, (1,), generator=g)) if t else -1
                x = (bits[parent] if parent >= 0 else 0) | 1 << t
            elif shape == "chain":
                x = (1 << (t + 1)) - 1
            else:  # any bits, some rows without any
                x = int(torch.randint(0, 1 << 62, (1,), generator=g)) * (1 if t % 5 else 0) * 3 & (1 << 64) - 1
            bits.append(x)
        rows.append([x - (1 << 64) if x >> 63 else x for x in bits])
    return torch.tensor(rows, dtype=torch.int64, device=dev)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", ["tree", "any"])
@pytest.mark.parametrize("H,heads,d,T", [(2, 2, 64, 1), (4, 2, 64, 13), (3, 1, 128, 64), (2, 2, 40, 61),
                                         (96, 8, 64, 40), (64, 8, 128, 64)])
def test_trees(dev, H, heads, d, T, shape, dtype, fmt):
    lens = [T, T + 1, T + 100, 200, 77 + T // 2]
    news = [T, T, T, T, T // 2]
    for window, n_persistent, page in ((None, 0, 64), (100, 4, 16), (3, 2, 32), (0, T + 3, 16)):
        run(dev, len(lens), H, heads, d, page, lens, news, T, window, n_persistent, dtype, fmt,
            tree=trees(dev, len(lens), T, T + (window or 0), shape))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", TYPES)
def test_chain_is_a_chunk(dev, dtype, fmt):
    """A draft without branches is a chunk: the same keys at the same places; one tree for all sequences."""
    lens, T = [70, 133], 20
    c, table, lengths = filled(dev, 2, 4, 64, 32, lens, dtype, fmt)
    q = queries(dev, 2, 4, T, 64, dtype)
    tree = trees(dev, 1, T, 0, "chain")[0]
    for window in (None, 5, 40):
        a = tc.cached_attention(q, c, table, lengths, window, 3)
        b = tc.cached_attention(q, c, table, lengths, window, 3, tree=tree)
        assert torch.equal(b, tc.cached_attention(q, c, table, lengths, window, 3, tree=tree.expand(2, T)))
        masks = seen_by(2, T, lens, [T, T], window, 3)
        check_attention(a, q, c, table, lens, [T, T], masks)
        check_attention(b, q, c, table, lens, [T, T], masks)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,heads,d,T", [(2, 2, 64, 1), (8, 1, 128, 1), (2, 1, 64, 30), (32, 16, 64, 1), (24, 24, 96, 2)])
def test_long_axis_in_parts(dev, H, heads, d, T, dtype, fmt):
    """Few rows over many keys: several workgroups share them, some without a key that is seen."""
    lens, news = [5000, 37, 3111], [T, T, max(1, T // 3)]
    for window, n_persistent in ((None, 0), (4000, 16)):
        first = run(dev, 3, H, heads, d, 64, lens, news, T, window, n_persistent, dtype, fmt, spread=2.0)
        o, q, c, table, lengths, counts = first
        assert torch.equal(o, tc.cached_attention(q, c, table, lengths, window, n_persistent, counts=counts))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_long_chunks_in_parts(dev, d, dtype, fmt):
    """Many rows over many keys, of which parts see none."""
    run(dev, 3, 64, 8, d, 32, [1500, 130, 700], [130, 130, 60], 130, 900, 16, dtype, fmt, spread=2.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_sharp_scores_and_scale(dev, dtype):
    for fmt in FORMATS:
        run(dev, 2, 4, 2, 64, 32, [300, 70], [1, 1], 1, None, 0, dtype, fmt, spread=6.0)
        run(dev, 2, 4, 2, 64, 32, [300, 70], [9, 9], 9, 100, 4, dtype, fmt, spread=3.0, scale=-0.7)
        run(dev, 2, 4, 2, 64, 32, [300, 70], [9, 9], 9, 100, 4, dtype, fmt, scale=0.0)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_values_far_from_one_in_fp16(dev, fmt):
    """Scales of the values from the least to the largest that fp16 has: the probabilities keep their bits."""
    lens = [200, 90]
    for spread in (2.0 ** -12, 2.0 ** 11):
        c, table, lengths = filled(dev, 2, 2, 64, 32, lens, torch.float16, fmt)
        v = (torch.randn(2, 2, 200, 64, device=dev) * spread).half()
        v[:, :, 60:] *= 4  # larger later
        tc.cache_write(torch.randn_like(v), v, c, table, lengths, counts=lengths)
        q = queries(dev, 2, 2, 3, 64, torch.float16)
        o = tc.cached_attention(q, c, table, lengths)
        masks = seen_by(2, 3, lens, [3, 3], None, 0)
        # a bit of fp16's least number lies on each result, as check_attention has it for values of the size of one
        check_attention(o, q, c, table, lens, [3, 3], masks)
        assert float(o.abs().max()) > spread / 64


@pytest.mark.parametrize("dtype", TYPES)
def test_what_a_row_does_not_see(dev, dtype):
    """Infinities and NaN in keys and values of later rows, of other branches, outside the window."""
    B, H, d, T, lens = 2, 2, 64, 40, [150, 40]
    for tree in (None, trees(dev, B, T, 3, "tree")):
        c, table, lengths = filled(dev, B, H, d, 16, lens, dtype, None)
        q = queries(dev, B, H, T, d, dtype)
        args = (q, c, table, lengths, 60, 4)
        want = tc.cached_attention(*args, tree=tree)
        masks = seen_by(B, T, lens, [T, T], 60, 4, None if tree is None else tree.cpu())
        for b in range(B):
            base = lens[b] - T
            for t, kv, bad in ((30, "v", math.inf), (33, "v", NAN), (31, "k", NAN), (35, "v", -math.inf), (21, "k", math.inf)):
                pos = base + t
                getattr(c, kv)[table[b, pos // 16].long(), :, pos % 16, 3] = bad
        got = tc.cached_attention(*args, tree=tree)
        for b in range(B):
            base = lens[b] - T
            m = masks[b].to(dev)
            hit = m[:, [base + t for t in (30, 33, 31, 35, 21)]]
            clean = ~hit.any(-1)
            assert clean.any() and torch.equal(got[b][:, clean], want[b][:, clean])
            only = hit[:, 0] & ~hit[:, 1:].any(-1)
            x = got[b][:, only]
            assert torch.all(x[..., 3] == math.inf) and torch.isfinite(x[..., 4:]).all()
            assert torch.isnan(got[b][:, hit[:, 1]][..., 3]).all()
            assert torch.isnan(got[b][:, hit[:, 2]]).all()
            both = hit[:, 0] & hit[:, 3]
            assert torch.isnan(got[b][:, both][..., 3]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window,d", [(None, 64), (90, 64), (None, 128), (70, 40)])
@pytest.mark.parametrize("H,heads", [(2, 2), (48, 24)])
def test_what_rows_of_a_chunk_do_not_see(dev, H, heads, window, d, dtype):
    """The same in a chunk of many rows: every row is as if what it does not see were not there, and what it sees reaches
    it, wherever that lies (before the chunk, in it, where all rows of some see it and not all of others)."""
    B, T, lens = 2, 200, [330, 200]
    c, table, lengths = filled(dev, B, heads, d, 32, lens, dtype, None, fill=NAN)
    q = queries(dev, B, H, T, d, dtype)
    want = tc.cached_attention(q, c, table, lengths, window, 4)
    masks = seen_by(B, T, lens, [T, T], window, 4)
    spots = ((-60, "v", math.inf), (0, "k", NAN), (63, "v", -math.inf), (64, "v", NAN), (127, "v", math.inf), (199, "v", NAN))
    for b in range(B):
        for t, kv, bad in spots:
            pos = lens[b] - T + t
            if pos >= 0:
                getattr(c, kv)[table[b, pos // 32].long(), :, pos % 32, 3] = bad
    got = tc.cached_attention(q, c, table, lengths, window, 4)
    for b in range(B):
        here = [(lens[b] - T + t, kv, bad) for t, kv, bad in spots if lens[b] - T + t >= 0]
        hit = masks[b].to(dev)[:, [p for p, _, _ in here]]
        key = torch.tensor([kv == "k" for _, kv, _ in here], device=dev)
        vals = torch.tensor([bad for _, _, bad in here], device=dev)
        assert torch.equal(got[b][:, ~hit.any(-1)], want[b][:, ~hit.any(-1)])
        nan_row = (hit & key).any(-1)
        assert torch.isnan(got[b][:, nan_row]).all()
        plus, minus, nan = ((hit & ~key & m).any(-1) & ~nan_row for m in (vals == math.inf, vals == -math.inf, vals.isnan()))
        col = got[b][:, :, 3]
        assert torch.isnan(col[:, nan | (plus & minus)]).all()
        assert torch.all(col[:, plus & ~minus & ~nan] == math.inf) and torch.all(col[:, minus & ~plus & ~nan] == -math.inf)
        assert torch.equal(got[b][:, ~nan_row, 4:], want[b][:, ~nan_row, 4:])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,H,heads", [(3, 2, 2), (40, 2, 2), (200, 2, 2), (200, 32, 8)])
def test_pages_that_are_none(dev, T, H, heads, dtype, fmt):
    """A page outside the pool is NaN for the rows that see it and nothing to the others; so are numbers that do not
    fit for a whole sequence."""
    lens = [T + 100, T + 100, T + 20, T]
    c, table, lengths = filled(dev, 4, heads, 64, 16, lens, dtype, fmt, fill=NAN)
    q = queries(dev, 4, H, T, 64, dtype)
    window, n_persistent = 50, 4
    want = tc.cached_attention(q, c, table, lengths, window, n_persistent)
    masks = seen_by(4, T, lens, [T] * 4, window, n_persistent)
    table[0, 1], table[0, 2] = -1, 2 ** 31 - 1          # in front of the window: not looked at, or not seen
    table[1, (lens[1] - 1) // 16] = c.k.shape[0]        # the last page
    bad = lengths.clone()
    bad[3] = table.shape[1] * 16 + 1
    got = tc.cached_attention(q, c, table, bad, window, n_persistent)
    assert torch.isnan(got[3]).all() and torch.equal(got[2], want[2])
    for b, pages in ((0, (1, 2)), (1, ((lens[1] - 1) // 16,))):
        m = masks[b].to(dev)
        hit = torch.stack([m[:, 16 * j:16 * j + 16].any(-1) for j in pages]).any(0)
        assert torch.isnan(got[b][:, hit]).all() and torch.equal(got[b][:, ~hit], want[b][:, ~hit])


def test_a_row_of_nan_in_8_bits(dev):
    """A row that was not finite when it was written: NaN for the rows that see its key or value, nothing to the others."""
    for fmt, dtype, T, H, heads in (("int8", torch.bfloat16, 150, 2, 2), ("e4m3", torch.float16, 150, 2, 2),
                                    ("int8", torch.float16, 9, 2, 2), ("e4m3", torch.float32, 70, 2, 2),
                                    ("int8", torch.bfloat16, 150, 128, 32), ("e4m3", torch.float16, 150, 128, 32),
                                    ("int8", torch.float32, 150, 128, 32)):
        B, d, lens = 1, 64, [T + 30]
        c, table, lengths = filled(dev, B, heads, d, 16, lens, dtype, fmt, fill=NAN)
        q = queries(dev, B, H, T, d, dtype)
        want = tc.cached_attention(q, c, table, lengths, 40)
        k = torch.randn(B, heads, 1, d, device=dev).to(dtype)
        pos = lens[0] - 5
        at = torch.tensor([pos + 1], dtype=torch.int32, device=dev)
        old = (c.k[table[0, pos // 16].long(), :, pos % 16].clone(), c.k_scale[table[0, pos // 16].long(), :, pos % 16].clone())
        v = k.clone()
        v[..., 7] = math.inf
        tc.cache_write(k, v, c, table, at)
        c.k[table[0, pos // 16].long(), :, pos % 16], c.k_scale[table[0, pos // 16].long(), :, pos % 16] = old
        got = tc.cached_attention(q, c, table, lengths, 40)
        m = seen_by(B, T, lens, [T], 40, 0)[0].to(dev)[:, pos]
        assert torch.isnan(got[0][:, m]).all() and torch.equal(got[0][:, ~m], want[0][:, ~m]) and m.any() and (~m).any()


def test_compiled(dev):
    c, table, lengths = filled(dev, 2, 2, 64, 32, [70, 40], torch.bfloat16, "int8")
    q = queries(dev, 2, 4, 3, 64, torch.bfloat16)

    def step(q, k, v):
        tc.cache_write(k, v, c, table, lengths)
        return tc.cached_attention(q * 2, c, table, lengths, 30, 2) + 1

    k, v = (torch.randn(2, 2, 3, 64, device=dev).bfloat16() for _ in range(2))
    want = step(q, k, v)
    with torch.no_grad():
        got = torch.compile(step, backend="aot_eager")(q, k, v)
    assert torch.equal(want, got)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,d,S,window,n_persistent", [(10, 64, 300, 128, 16), (3, 40, 77, 20, 0), (2, 128, 130, 500, 4)])
def test_as_windowed_attention(dev, H, d, S, window, n_persistent, dtype):
    """A text that arrives in chunks of any size gets what windowed_attention gives for all of it."""
    B, page = 2, 16
    per = -(-S // page)
    q, k, v = (torch.randn(B, H, S, d, generator=gen(dev, i), device=dev).to(dtype) for i in range(3))
    whole = tc.windowed_attention(q, k, v, window, n_persistent)
    c = empty_cache(dev, B * per, H, d, page, dtype, None, fill=NAN)
    table = make_table(dev, B, per, B * per)
    at, parts = 0, []
    for n in (n_persistent or 1, 1, 1, 31, 1, S):
        n = min(n, S - at)
        lengths = torch.full((B,), at + n, dtype=torch.int32, device=dev)
        tc.cache_write(k[:, :, at:at + n], v[:, :, at:at + n], c, table, lengths)
        parts.append(tc.cached_attention(q[:, :, at:at + n], c, table, lengths, window, n_persistent))
        at += n
    assert at == S
    got = torch.cat(parts, 2)
    # both within half a step of each probability and of the result
    half = {torch.float32: 300 * E, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
    assert torch.all((got.float() - whole.float()).abs() <= 2 * half * (whole.float().abs() + v.float().abs().amax()))


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_alignment(dev, dtype):
    B, H, T, d, lens = 3, 4, 5, 64, [50, 9, 70]
    c, table, lengths = filled(dev, B, H, d, 16, lens, dtype, None)
    q = queries(dev, B, H, T, d, dtype)
    want = tc.cached_attention(q, c, table, lengths, 30, 2)
    wide = torch.full((B, H, T, d + 3), NAN, dtype=dtype, device=dev)
    wide[..., 1:d + 1] = q
    across = torch.empty(d, T, H, B, dtype=dtype, device=dev)
    across.copy_(q.permute(3, 2, 1, 0))
    table2 = torch.full((B, 40), -7, dtype=torch.int32, device=dev)
    table2[:, 2:2 + table.shape[1]] = table
    lengths2 = torch.zeros(B, 2, dtype=torch.int32, device=dev)
    lengths2[:, 0] = lengths
    for x in (q.contiguous(), wide[..., 1:d + 1], across.permute(3, 2, 1, 0)):
        assert torch.equal(want, tc.cached_attention(x, c, table2[:, 2:2 + table.shape[1]], lengths2[:, 0], 30, 2))
        assert torch.equal(want, tc.cached_attention(x, c, table.t().contiguous().t(), lengths, 30, 2))
    one = tc.cached_attention(q[:1], c, table[:1], lengths[:1], 30, 2)
    assert torch.equal(want[:1], one)
    e = tc.cached_attention(q[:, :, :0], c, table, lengths, 30, 2)
    assert e.shape == (B, H, 0, d)


def test_dispatched_op_streams_graphs_threads(dev):
    """The registered op, another stream, two graphs whose workspaces are their own, two threads."""
    from titans_core.kernels import kv_cache as kc
    B, H, d, lens = 2, 4, 64, [5000, 4000]
    c, table, lengths = filled(dev, B, H, d, 64, lens, torch.bfloat16, "int8")
    q = queries(dev, B, H, 1, d, torch.bfloat16)
    want = tc.cached_attention(q, c, table, lengths, None, 4)
    got = kc.cached_attention_op(q, c.k, c.v, c.k_scale, c.v_scale, table, lengths, None, None, 1 << 30, 4, d ** -0.5, d)
    assert torch.equal(want, got)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = tc.cached_attention(q, c, table, lengths, None, 4)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(want, other)
    graphs, outs = [], []
    for w in (None, 3000):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(tc.cached_attention(q, c, table, lengths, w, 4))
        graphs.append(graph)
    for step in range(3):
        q.copy_(queries(dev, B, H, 1, d, torch.bfloat16, seed=step))
        lengths.copy_(torch.tensor([4990 - step * 1500, 100 + step], dtype=torch.int32))
        graphs[0].replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.synchronize()
        for w, o in zip((None, 3000), outs):
            assert torch.equal(o, tc.cached_attention(q, c, table, lengths, w, 4))
    want = tc.cached_attention(q, c, table, lengths, None, 4)
    results = [None] * 2

    def work(i):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.default_stream())
        with torch.cuda.stream(s):
            results[i] = [tc.cached_attention(q, c, table, lengths, None, 4) for _ in range(20)]
        s.synchronize()

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert all(torch.equal(want, o) for r in results for o in r)


def test_serving_step_by_step(dev):
    """A prompt, decoded tokens, a draft of which a branch is kept, and a token behind it: as all of it at once."""
    H, heads, d, page, B, dtype = 8, 2, 64, 16, 2, torch.bfloat16
    for fmt in FORMATS:
        g = gen(dev, 5)
        make = lambda h, t: torch.randn(B, h, t, d, generator=g, device=dev).to(dtype)  # noqa: E731
        q, k, v = make(H, 60), make(heads, 60), make(heads, 60)
        c = tc.KVCache.new(12, heads, d, page=page, dtype=dtype, fmt=fmt, device=dev)
        table = make_table(dev, B, 5, 12)
        at = lambda n: torch.full((B,), n, dtype=torch.int32, device=dev)  # noqa: E731

        def step(lo, hi, **kw):
            tc.cache_write(k[:, :, lo:hi], v[:, :, lo:hi], c, table, at(hi))
            return tc.cached_attention(q[:, :, lo:hi], c, table, at(hi), 25, 4, **kw)

        parts = [step(0, 40), step(40, 41), step(41, 42)]
        # drafted: 42, other, 43, other, 44 with 42 - 43 - 44 one branch
        order = [42, 50, 43, 51, 44]
        tree = torch.tensor([0b1, 0b10, 0b101, 0b1010, 0b10101], device=dev)
        tc.cache_write(k[:, :, order], v[:, :, order], c, table, at(47))
        o = tc.cached_attention(q[:, :, order], c, table, at(47), 25, 4, tree=tree)
        parts.append(o[:, :, [0, 2, 4]])
        tc.cache_keep(c, table, at(47), torch.tensor([[0, 2, 4, -1]], dtype=torch.int32, device=dev).expand(B, 4), 5)
        parts.append(step(45, 46))
        got = torch.cat(parts, 2)
        fresh = tc.KVCache.new(12, heads, d, page=page, dtype=dtype, fmt=fmt, device=dev)
        tc.cache_write(k[:, :, :46], v[:, :, :46], fresh, table, at(46))
        whole = tc.cached_attention(q[:, :, :46], fresh, table, at(46), 25, 4)
        masks = seen_by(B, 46, [46] * B, [46] * B, 25, 4)
        check_attention(whole, q[:, :, :46], fresh, table, [46] * B, [46] * B, masks)
        check_attention(got, q[:, :, :46], fresh, table, [46] * B, [46] * B, masks)
        for x, y in zip(tc.cache_read(c, table, at(46), 46), tc.cache_read(fresh, table, at(46), 46)):
            assert torch.equal(x, y)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,H,heads", [(2, 2, 2), (40, 2, 2), (200, 2, 2), (200, 128, 32)])
def test_a_large_value_beside_small_ones(dev, T, H, heads, dtype, fmt):
    """A value of the type's size beside values of 0.01: nothing to the rows that do not see it, nor to a row that gives it
    a probability of e^-40."""
    lens = [T + 60]
    c, table, lengths = filled(dev, 1, heads, 64, 32, lens, dtype, fmt)
    q = queries(dev, 1, H, T, 64, dtype)
    k = torch.randn(1, heads, lens[0], 64, device=dev).to(dtype)
    v = (torch.randn(1, heads, lens[0], 64, device=dev) * 0.01).to(dtype)
    tc.cache_write(k, v, c, table, lengths)
    want = tc.cached_attention(q, c, table, lengths, 50)
    v[:, :, -1] = 60000 * torch.rand(1, heads, 64, device=dev)
    tc.cache_write(k, v, c, table, lengths)
    got = tc.cached_attention(q, c, table, lengths, 50)
    assert torch.equal(got[:, :, :-1], want[:, :, :-1]) and not torch.equal(got[:, :, -1], want[:, :, -1])

    ones = torch.ones(1, H, 1, 64, dtype=dtype, device=dev)
    k[:, :, :-1], k[:, :, -1] = 1, -4   # scores of 8 and -32
    tc.cache_write(k, v, c, table, lengths)
    got = tc.cached_attention(ones, c, table, lengths, 50).double()
    w = pool_rows(c, table, 0, lens[0], "v")[:, -51:-1].mean(1).repeat_interleave(H // heads, 0)[None, :, None]
    # e^-40 60000 < 3e-13; the sum over 50 keys, two numbers of the probability (2^-16 of it) and the result's rounding
    half = {torch.float32: 2 * E, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
    assert torch.all((got - w).abs() <= half * w.abs() + 0.05 * (2.0 ** -16 + 500 * E) + 2.0 ** -25 * (dtype == torch.float16)
                     + 3e-13)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", TYPES)
def test_a_draft_of_one(dev, dtype, fmt):
    """A drafted row that does not see itself, and one whose window ends at a row that is not finite."""
    window, base = 20, 60
    for bits, pos in ((0, base), (1, base - 1 - window)):  # entry, position that it does not see
        c, table, lengths = filled(dev, 1, 2, 64, 16, [base + 1], dtype, fmt)
        q = queries(dev, 1, 4, 1, 64, dtype)
        tree = torch.tensor([[bits]])
        want = tc.cached_attention(q, c, table, lengths, window, tree=tree.to(dev))
        check_attention(want, q, c, table, [base + 1], [1], seen_by(1, 1, [base + 1], [1], window, 0, tree))
        for x in (c.k, c.v) if fmt is None else (c.k_scale, c.v_scale):
            x[table[0, pos // 16].long(), :, pos % 16] = NAN
        assert torch.equal(tc.cached_attention(q, c, table, lengths, window, tree=tree.to(dev)), want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,H,heads", [(9, 2, 2), (40, 2, 2), (200, 128, 32)])
def test_codes_that_are_none(dev, T, H, heads, dtype):
    """e4m3 codes of NaN in pools that cache_write has not filled: NaN in their column for the rows that see them, nothing to
    the others."""
    lens = [T + 100]
    c, table, lengths = filled(dev, 1, heads, 64, 32, lens, dtype, "e4m3")
    q = queries(dev, 1, H, T, 64, dtype)
    want = tc.cached_attention(q, c, table, lengths, 50, 4)
    mask = seen_by(1, T, lens, [T], 50, 4)[0].to(dev)
    spots = [lens[0] - 4, lens[0] - T + 2, lens[0] - T - 50]  # row 1 sees none of them
    for pos, code in zip(spots, (0x7f, 0xff, 0x7f)):
        c.v.view(torch.uint8)[table[0, pos // 32].long(), :, pos % 32, 3] = code
    got = tc.cached_attention(q, c, table, lengths, 50, 4)
    hit = mask[:, spots].any(-1)
    assert hit.any() and (~hit).any()
    assert torch.isnan(got[0][:, hit][..., 3]).all() and torch.equal(got[0][:, hit][..., 4:], want[0][:, hit][..., 4:])
    assert torch.equal(got[0][:, ~hit], want[0][:, ~hit])
