"""cached_attention in each of the ways in which its rows and keys are shared out."""
import pytest
import torch

import titans_core as tc
from cache_cases import FORMATS, SHAPES, check_two_numbers, filled, gen, seen_by

pytestmark = pytest.mark.gpu


def queries(dev, B, H, T, d, dtype):
    return torch.randn(B, T, H, d, generator=gen(dev, 9), device=dev).to(dtype).transpose(1, 2)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,T,H,heads,d,n", [(2, 1, 4, 4, 64, 300), (2, 40, 4, 4, 64, 300), (16, 200, 4, 4, 64, 300),
                                             (12, 200, 8, 8, 128, 260), (2, 40, 2, 2, 64, 3000), (2, 40, 2, 2, 128, 3000),
                                             (60, 40, 4, 4, 64, 300), (60, 40, 4, 4, 128, 300)])
def test_probabilities_keep_their_bits(dev, B, T, H, heads, d, n, dtype, fmt):
    """Few rows or many, beside many sequences or few: the result's rounding is the only one of its size."""
    lens = [n - 7 * (b % 16) for b in range(B)]
    c, table, lengths = filled(dev, B, heads, d, 32, lens, dtype, fmt)
    q = queries(dev, B, H, T, d, dtype)
    out = tc.cached_attention(q, c, table, lengths, None, 4)
    news = [min(T, length) for length in lens]
    check_two_numbers(out, q, c, table, lens, news, seen_by(B, T, lens, news, None, 4))


@pytest.mark.parametrize("T,H,heads,d,high", [(1, 4, 4, 64, 8), (1, 4, 4, 128, 8), (40, 4, 4, 64, 8), (100, 8, 1, 64, 1),
                                              (100, 8, 1, 128, 1)])
def test_small_probabilities_of_long_axes_in_fp16(dev, T, H, heads, d, high):
    """2^18 keys that have e^-17.5 of the likeliest ones' probability each, which is below half of fp16's least number,
    and together 0.0065 of one's. The likeliest (the first of each of the first tiles) have values of 0, the others of 1.

    Each probability may be off by half of fp16's least number times 2^-7 (they are held times 2^7) of the likeliest, the
    result by half a step."""
    n, page, B = 1 << 18, 256, 64  # all sequences read the same pages
    c = tc.KVCache.new(n // page, heads, d, page=page, dtype=torch.float16, device=dev)
    c.v.fill_(1)
    at = torch.arange(high, device=dev) * 32
    c.k[at // page, :, at % page, 0] = 17.5
    c.v[at // page, :, at % page] = 0
    table = torch.arange(n // page, dtype=torch.int32, device=dev).expand(B, -1).contiguous()
    lengths = torch.full((B,), n, dtype=torch.int32, device=dev)
    q = torch.ones(B, H, T, d, dtype=torch.float16, device=dev)
    out = tc.cached_attention(q, c, table, lengths, scale=1.0)
    seen = torch.arange(n - T, n, device=dev, dtype=torch.float64) + 1 - high  # of the small ones, by row
    small = seen * 2.718281828459045 ** -17.5
    want = (small / (small + high))[:, None]
    tol = 2.0 ** -11 * want + 2.0 ** -25 + n * 2.0 ** -32 / high + 2 * (n + 200) * 2.0 ** -24 * want
    assert torch.all((out.double() - want).abs() <= tol), (float(out.amin()), float(out.amax()), float(want[0]))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,T,H,heads,d,n,page", SHAPES)
def test_every_kernel(dev, B, T, H, heads, d, n, page, dtype, fmt):
    """Ragged sequences, some with fewer new rows than others; drafts where they are as short. That these shapes launch every
    kernel is tested on the CPU (test_cached_attention_host.py)."""
    lens = [n - 13 * (b % 16) for b in range(B)]
    news = [min(T - T // 3 if b % 3 == 2 else T, lens[b]) for b in range(B)]
    c, table, lengths = filled(dev, B, heads, d, page, lens, dtype, fmt, fill=float("nan"))
    assert table.shape[1] == -(-n // page)
    q = queries(dev, B, H, T, d, dtype)
    counts = torch.tensor(news, dtype=torch.int32, device=dev)
    trees = [None]
    if 1 < T <= 64:
        g = torch.Generator().manual_seed(T)
        bits = [1]
        for t in range(1, T):
            bits.append(bits[int(torch.randint(0, t, (1,), generator=g))] | 1 << t)
        trees.append(torch.tensor([x - (1 << 64) if x >> 63 else x for x in bits], device=dev))
    for tree in trees:
        out = tc.cached_attention(q, c, table, lengths, None, 4, counts=counts, tree=tree)
        check_two_numbers(out, q, c, table, lens, news, seen_by(B, T, lens, news, None, 4, None if tree is None else tree.cpu()))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,T,H,heads,d,n,page", SHAPES)
def test_values_that_are_not_finite(dev, B, T, H, heads, d, n, page, dtype):
    """An infinite value that every row sees and one that is NaN and only some see: they reach their columns, and nothing
    else changes."""
    lens = [n - 13 * (b % 16) for b in range(B)]
    news = [min(T, length) for length in lens]
    c, table, lengths = filled(dev, B, heads, d, page, lens, dtype, None)
    q = queries(dev, B, H, T, d, dtype)
    want = tc.cached_attention(q, c, table, lengths, None, 4)
    for b in range(B):
        for pos, col, value in ((1, 3, float("inf")), (lens[b] - news[b] // 2 - 1, 5, float("nan"))):
            c.v[table[b, pos // page].long(), :, pos % page, col] = value
    got = tc.cached_attention(q, c, table, lengths, None, 4)
    for b in range(B):
        sees = torch.arange(T, device=dev) >= news[b] - news[b] // 2 - 1
        real = torch.arange(T, device=dev) < news[b]
        assert torch.all(got[b][:, real, 3] == float("inf")) and torch.all(got[b][:, ~real] == 0)
        assert torch.equal(got[b][..., 5].isnan(), (sees & real).expand(H, T))
        want[b][:, real, 3] = float("inf")
        want[b][:, real & sees, 5] = 0
        assert torch.equal(got[b].nan_to_num(0.0, float("inf")), want[b])


@pytest.mark.parametrize("window", [61, 62, 63, 64, 65, 127])
def test_windows_of_a_draft_s_length(dev, window):
    """Places of a draft's rows are up to 64 apart: that of an entry without bits and that of one with all."""
    B, T, lens = 3, 64, [64, 100, 300]
    c, table, lengths = filled(dev, B, 2, 64, 16, lens, torch.float32, None, fill=float("nan"))
    q = queries(dev, B, 4, T, 64, torch.float32)
    chain = [(1 << t + 1) - 1 for t in range(T)]
    trees = [chain, [0] + [-1] * 63, [-1 if t % 3 else t & 1 for t in range(T)]]
    trees = torch.tensor([[x - (1 << 64) if x >> 63 == 1 else x for x in row] for row in trees])
    for n_persistent in (0, 5):
        out = tc.cached_attention(q, c, table, lengths, window, n_persistent, tree=trees.to(dev))
        check_two_numbers(out, q, c, table, lens, [T] * B, seen_by(B, T, lens, [T] * B, window, n_persistent, trees))
