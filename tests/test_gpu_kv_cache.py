"""cache_write, cache_read and cache_keep against their definitions."""
import math

import pytest
import torch

import titans_core as tc
from cache_cases import FORMATS, STORE, empty_cache, gen, make_table, pool_rows, quantised

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def same_bits(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def rows_of(dev, B, H, T, d, dtype, seed=0):
    """Rows of very different sizes, as views of one projection's output."""
    x = torch.randn(B, T, 3 * H, d, generator=gen(dev, seed), device=dev)
    x = x * torch.exp2(torch.randint(-8, 5, (B, T, 3 * H, 1), generator=gen(dev, seed + 1), device=dev).float())
    x = x.to(dtype).transpose(1, 2)
    return x[:, H:2 * H], x[:, 2 * H:]


def written(c, k, v, table, lens, news, was):
    """Every pool is what it was, with the new rows at their places."""
    fmt = {torch.int8: "int8", torch.float8_e4m3fn: "e4m3"}.get(c.k.dtype)
    page, d = c.k.shape[2], c.d_head
    for name, new in (("k", k), ("v", v)):
        want = was[name].clone()
        scale = None if fmt is None else was[name + "_scale"].clone()
        raw = want.view(torch.uint8) if fmt == "e4m3" else want
        for b in range(len(lens)):
            if not news[b]:
                continue
            pos = torch.arange(lens[b] - news[b], lens[b], device=want.device)
            p, at = table[b].long()[pos // page], pos % page
            x = new[b, :, :news[b]].transpose(0, 1)
            if fmt is not None:
                x, s = quantised(x, fmt)
                scale[p, :, at] = s
            raw[p, :, at] = 0
            raw[p, :, at, :d] = x.view(torch.uint8) if fmt == "e4m3" else x
        assert same_bits(getattr(c, name), want), name
        if fmt is not None:
            same = torch.equal(getattr(c, name + "_scale").nan_to_num(-1.0), scale.nan_to_num(-1.0))
            assert same, name


def snapshot(c):
    return {n: getattr(c, n).clone() for n in ("k", "v", "k_scale", "v_scale") if getattr(c, n) is not None}


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,d,page,T,lens,news", [
    (10, 64, 64, 1, [1, 64, 65, 700], [1, 1, 1, 1]),
    (2, 128, 16, 37, [37, 40, 300, 17, 0], [37, 0, 36, 17, 0]),
    (3, 40, 32, 5, [5, 4, 33], [5, 1, 3]),
    (1, 1, 16, 3, [3, 200], [3, 2]),
    (5, 33, 256, 130, [130, 257], [130, 129]),
    (7, 96, 128, 2, [2], [2]),
])
def test_write(dev, H, d, page, T, lens, news, dtype, fmt):
    B = len(lens)
    per = max(1, -(-max(lens) // page))
    c = empty_cache(dev, B * per + 3, H, d, page, dtype, fmt, fill=3.0)
    if c.k_scale is None:
        c.k.normal_(), c.v.normal_()
    table = make_table(dev, B, per, B * per + 3)
    k, v = rows_of(dev, B, H, T, d, dtype)
    lengths, counts = (torch.tensor(x, dtype=torch.int32, device=dev) for x in (lens, news))
    was = snapshot(c)
    tc.cache_write(k, v, c, table, lengths, counts=counts)
    written(c, k, v, table, lens, news, was)
    # the same from contiguous rows, and all rows of sequences that have them
    k2, v2 = k.contiguous(), v.contiguous()
    tc.cache_write(k2, v2, c, table, lengths, counts=counts)
    written(c, k, v, table, lens, news, was)
    tc.cache_write(k, v, c, table, lengths)
    written(c, k, v, table, lens, [min(T, n) for n in lens], was)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", TYPES)
def test_codes(dev, fmt, dtype):
    """Values at and beside the borders between codes; zeros, the least numbers, the largest, rows that are not finite."""
    H, d, page = 1, 128, 64
    rows = []
    for amax in (127.0, 1.0, 448.0, 449.0, 224.0, 3e-5, 6e4, 448 * 2.0 ** -9, 0.1):
        top = torch.tensor(amax).to(dtype).float()
        s = quantised(top[None], fmt)[1].double()
        steps = (torch.arange(126, dtype=torch.float64) + 0.5) * s if fmt == "int8" else top.double() * torch.exp2(
            -torch.linspace(0, 14, 126, dtype=torch.float64))
        x = torch.cat([top.double()[None], -steps, torch.zeros(1)]).to(dtype)
        x = torch.where(x.abs() > top.to(dtype), torch.zeros_like(x), x)
        rows.append(x)
        bits = x.view(torch.int32 if dtype == torch.float32 else torch.int16)
        for o in (-1, 1):  # the neighbours of every value
            y = (bits + o).view(dtype)
            y = torch.where(torch.isfinite(y) & (y.abs() <= x[0].abs()), y, x)
            rows.append(y)
    if fmt == "e4m3":
        code = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
        mid = torch.cat([(code[:-1] + code[1:]) / 2, torch.tensor([448.0, -448.0], dtype=torch.float64)])
        rows += [mid.to(dtype), (-mid * 2.0 ** -6).to(dtype)]
    tiny = torch.finfo(dtype)
    rows += [torch.zeros(d, dtype=dtype), torch.full((d,), tiny.smallest_normal, dtype=dtype),
             torch.full((d,), tiny.max, dtype=dtype), (torch.arange(d) * (tiny.smallest_normal * tiny.eps)).to(dtype)]
    for bad in (math.inf, -math.inf, math.nan):
        x = torch.ones(d, dtype=dtype)
        x[77] = bad
        rows.append(x)
    x = torch.stack(rows).to(dev)[None, None]
    T = x.shape[2]
    c = empty_cache(dev, 2, H, d, page, dtype, fmt)
    table = make_table(dev, 1, 1, 2)
    assert T <= page
    was = snapshot(c)
    tc.cache_write(x, x.flip(2), c, table, torch.tensor([T], dtype=torch.int32, device=dev))
    written(c, x, x.flip(2), table, [T], [T], was)
    k, _ = tc.cache_read(c, table, torch.tensor([T], dtype=torch.int32, device=dev), T, dtype=dtype)
    assert torch.isnan(k[0, 0, -3:]).all()
    # what a row is held as may lie past the type's largest: bf16's is 255 · 2^120, in e4m3 256 · 2^120 = 2^128
    held = pool_rows(c, table, 0, T, "k")[0, :-3].to(dtype)
    assert torch.equal(torch.isfinite(held), torch.isfinite(k[0, 0, :-3])) and torch.isfinite(held[:-2]).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,d,page,n,lens", [(10, 64, 64, 300, [300, 1, 64, 0]), (3, 40, 16, 33, [33, 7]),
                                             (2, 1, 32, 5, [3]), (1, 128, 256, 600, [257, 599]), (4, 33, 16, 20, [50])])
def test_read(dev, H, d, page, n, lens, dtype, fmt):
    B = len(lens)
    per = -(-max(*lens, n) // page)
    c = empty_cache(dev, B * per + 1, H, d, page, dtype, fmt, fill=math.nan)
    table = make_table(dev, B, per, B * per + 1)
    lengths = torch.tensor(lens, dtype=torch.int32, device=dev)
    k, v = rows_of(dev, B, H, max(lens), d, dtype)
    tc.cache_write(k, v, c, table, lengths, counts=lengths)
    got = tc.cache_read(c, table, lengths, n, dtype=dtype)
    half = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
    for name, new, x in (("k", k, got[0]), ("v", v, got[1])):
        assert x.shape == (B, H, n, d) and x.dtype == dtype
        for b in range(B):
            m = min(n, lens[b])
            assert torch.all(x[b, :, m:] == 0)
            if fmt is None:
                assert same_bits(x[b, :, :m], new[b, :, :m])
            else:  # code · scale in fp32, then in dtype (whose least numbers are multiples of its smallest)
                want = pool_rows(c, table, b, m, name)
                tol = (half + 2.0 ** -24) * want.abs() + torch.finfo(dtype).smallest_normal * half
                assert torch.all((x[b, :, :m].double() - want).abs() <= tol)
    default = tc.cache_read(c, table, lengths, n)[0].dtype
    assert default == (dtype if fmt is None else torch.bfloat16)


def test_numbers_that_do_not_fit(dev):
    """Lengths past the table or below 0, counts above T or the length, pages outside the pool: nothing is written,
    what is asked of them is NaN."""
    H, d, page, B, T = 2, 64, 16, 8, 3
    c = tc.KVCache.new(B * 2, H, d, page=page, device=dev)
    c.k.fill_(1.0), c.v.fill_(2.0)
    table = make_table(dev, B, 2, B * 2)
    table[5, 0], table[6, 1] = -1, 2 ** 31 - 1
    lens, news = [33, -1, 2 ** 31 - 1, 20, 2, 18, 18, 18], [3, 0, 3, 4, 3, 3, 3, -1]
    lengths, counts = (torch.tensor(x, dtype=torch.int32, device=dev) for x in (lens, news))
    was = snapshot(c)
    k = torch.full((B, H, T, d), 5.0, dtype=torch.bfloat16, device=dev)
    tc.cache_write(k, k, c, table, lengths, counts=counts)
    # sequence 5 is at 15, 16, 17 with page 0 missing, 6 with page 1 missing; of the others nothing fits
    for name in ("k", "v"):
        want = was[name].clone()
        want[table[5, 1], :, :2] = 5.0
        want[table[6, 0], :, 15] = 5.0
        assert torch.equal(getattr(c, name), want)
    x, y = tc.cache_read(c, table, lengths, 32)
    for t in (x, y):
        assert torch.isnan(t[:3]).all() and torch.isfinite(t[3:5]).all() and torch.isfinite(t[7]).all()
        assert torch.isnan(t[5, :, :16]).all() and torch.all(t[5, :, 16:18] == 5.0) and torch.all(t[5, :, 18:] == 0)
        assert torch.isfinite(t[6, :, :16]).all() and torch.isnan(t[6, :, 16:18]).all() and torch.all(t[6, :, 18:] == 0)
    q = torch.randn(B, H, T, d, device=dev).bfloat16()
    o = tc.cached_attention(q, c, table, lengths, counts=counts)
    assert torch.isnan(o[[0, 1, 2, 3, 4, 5, 7]]).all()
    assert torch.isfinite(o[6, :, :1]).all() and torch.isnan(o[6, :, 1:]).all()
    tc.cache_keep(c, table, lengths, torch.tensor([[1, 2]], dtype=torch.int32, device=dev).expand(B, 2), counts)
    want[table[6, 0], :, 15] = 5.0  # its sources' page is missing
    want[table[5, 1], :, 0] = 5.0
    assert torch.equal(c.k, want.where(want == 5.0, was["k"]))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H,d,page", [(10, 64, 64), (3, 128, 16), (2, 40, 32), (1, 16, 256)])
def test_keep(dev, H, d, page, dtype, fmt):
    lens, news = [100, 64, 40, 13, 30], [64, 64, 30, 13, 0]
    B = len(lens)
    c = empty_cache(dev, 5 * 8 + 1, H, d, page, dtype, fmt)
    table = make_table(dev, B, -(-100 // page), 5 * 8 + 1 if page == 16 else 5 * -(-100 // page))
    k, v = rows_of(dev, B, H, max(lens), d, dtype)
    lengths, counts = (torch.tensor(x, dtype=torch.int32, device=dev) for x in (lens, news))
    tc.cache_write(k, v, c, table, lengths, counts=lengths)
    paths = [sorted(torch.randperm(max(n, 1), generator=torch.Generator().manual_seed(n))[:9].tolist()) for n in news]
    paths = [p + [-1] * (9 - len(p)) for p in paths]
    paths[0][3], paths[1][0], paths[1][8] = 64, 63, 63  # outside the draft; backwards, and one row twice
    paths[2] = [8, 7, 6, 5, 4, 3, 2, 1, 0]              # all of them change places
    path = torch.tensor(paths, dtype=torch.int32, device=dev)
    was = snapshot(c)
    tc.cache_keep(c, table, lengths, path, counts)
    for name in was:
        want = was[name].clone()
        raw, old = (x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x for x in (want, was[name]))
        for b in range(B):
            for a, t in enumerate(paths[b]):
                if 0 <= t < news[b] and a < news[b]:
                    at = lambda p: (int(table[b, p // page]), slice(None), p % page)  # noqa: E731
                    raw[at(lens[b] - news[b] + a)] = old[at(lens[b] - news[b] + t)]
        assert same_bits(getattr(c, name), want), name
    # one number for all, sequences with fewer rows than that as they are
    tc.cache_keep(c, table, lengths, path[:, :0], 64)
    before = snapshot(c)
    tc.cache_keep(c, table, lengths, torch.arange(9, device=dev).int().expand(B, 9), 13)
    assert all(same_bits(getattr(c, n), t) for n, t in before.items())


def test_far_pages(dev):
    """A pool of more than 2^32 bytes and 2^31 values: rows on its last pages, written, read, moved and attended."""
    H, d, page = 8, 128, 256
    n_pages = (1 << 31) // (H * d * page) * 5 // 4
    c = tc.KVCache.new(n_pages, H, d, page=page, device=dev)
    assert c.k.numel() > 1 << 31
    table = torch.tensor([[n_pages - 1, n_pages - 3], [n_pages - 2, n_pages // 2 + 1]], dtype=torch.int32, device=dev)
    lens = [400, 300]
    lengths = torch.tensor(lens, dtype=torch.int32, device=dev)
    k, v = rows_of(dev, 2, H, 400, d, torch.bfloat16)
    tc.cache_write(k, v, c, table, lengths, counts=lengths)
    x, y = tc.cache_read(c, table, lengths, 400)
    for b in range(2):
        assert same_bits(x[b, :, :lens[b]], k[b, :, :lens[b]]) and same_bits(y[b, :, :lens[b]], v[b, :, :lens[b]])
    q = torch.randn(2, H, 1, d, device=dev).bfloat16()
    o = tc.cached_attention(q, c, table, lengths)
    small = tc.KVCache(c.k[table.reshape(-1).long()], c.v[table.reshape(-1).long()], d)
    near = torch.arange(4, device=dev).int().view(2, 2)
    assert same_bits(o, tc.cached_attention(q, small, near, lengths))
    tc.cache_keep(c, table, lengths, torch.tensor([[5], [63]], dtype=torch.int32, device=dev), 64)
    x = tc.cache_read(c, table, lengths, 400)[0]
    assert same_bits(x[0, :, 336], k[0, :, 341]) and same_bits(x[1, :, 236], k[1, :, 299])


def test_streams_graph_and_versions(dev):
    H, d, page, B, T = 4, 64, 32, 3, 2
    c = tc.KVCache.new(20, H, d, page=page, fmt="int8", device=dev)
    table = make_table(dev, B, 4, 20)
    k, v = rows_of(dev, B, H, T, d, torch.bfloat16)
    lengths = torch.tensor([2, 50, 128], dtype=torch.int32, device=dev)
    version = c.k._version
    tc.cache_write(k, v, c, table, lengths)
    assert c.k._version > version and c.v_scale._version > 0
    want = snapshot(c)
    for t in want:
        getattr(c, t).zero_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        tc.cache_write(k, v, c, table, lengths)
        x = tc.cache_read(c, table, lengths, 128)
    torch.cuda.current_stream().wait_stream(side)
    assert all(same_bits(getattr(c, n), t) for n, t in want.items())
    assert all(same_bits(a, b) for a, b in zip(x, tc.cache_read(c, table, lengths, 128)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tc.cache_write(k, v, c, table, lengths)
        held = tc.cache_read(c, table, lengths, 128)
    for step in range(3):
        k.copy_(torch.randn(k.shape, device=dev).bfloat16())
        lengths.copy_(torch.tensor([3 + step, 50, 90 - step], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        e = tc.KVCache(*(t.clone() if isinstance(t, torch.Tensor) else t for t in (c.k, c.v, d, c.k_scale, c.v_scale)))
        tc.cache_write(k, v, e, table, lengths)
        assert same_bits(e.k, c.k) and same_bits(e.k_scale, c.k_scale)
        assert all(same_bits(a, b) for a, b in zip(held, tc.cache_read(e, table, lengths, 128)))


def test_what_e4m3_rounds_up_past_fp16(dev):
    """Above 57344 = 448 · 2^7 a row's scale is 2^8, where e4m3 goes by 16 · 2^8 from 128 · 2^8 on: 63456 is nearer to 240 · 2^8
    than to 2^16, 63488 is a tie, which goes to 2^16."""
    c, table = empty_cache(dev, 1, 1, 16, 16, torch.float16, "e4m3"), torch.zeros(1, 1, dtype=torch.int32, device=dev)
    n = torch.tensor([4], dtype=torch.int32, device=dev)
    x = torch.zeros(1, 1, 4, 16, dtype=torch.float16, device=dev)
    x[0, 0, :, 0] = torch.tensor([57344.0, 63456.0, 63488.0, -65504.0])
    tc.cache_write(x, x, c, table, n)
    for y in tc.cache_read(c, table, n, 4, dtype=torch.float16):
        assert y[0, 0, :, 0].tolist() == [57344.0, 61440.0, math.inf, -math.inf] and torch.all(y[..., 1:] == 0)
    for y in tc.cache_read(c, table, n, 4):
        assert y[0, 0, :, 0].tolist() == [57344.0, 61440.0, 65536.0, -65536.0]
