"""Caches, sequences and the definitions in 64 bits for the tests of the key/value cache."""
import math

import torch

import titans_core as tc

E = 2.0 ** -24
FORMATS = [None, "int8", "e4m3"]
STORE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def empty_cache(dev, n_pages, H, d, page, dtype, fmt, fill=None):
    """A cache whose rows are `fill` everywhere (what an earlier user of the pages left)."""
    c = tc.KVCache.new(n_pages, H, d, page=page, dtype=dtype, fmt=fmt, device=dev)
    if fill is not None:
        for t in (c.k, c.v):
            if fmt == "int8":
                t.fill_(77)
            elif fmt == "e4m3":
                t.view(torch.uint8).fill_(0x7f)  # NaN codes
            else:
                t.fill_(fill)
        for t in (c.k_scale, c.v_scale):
            if t is not None:
                t.fill_(fill)
    return c


def make_table(dev, B, per, n_pages, seed=0):
    """A page for every place of the table, none twice, in no order."""
    return torch.randperm(n_pages, generator=gen(dev, seed), device=dev)[:B * per].view(B, per).int()


def pool_rows(c, table, b, n, name):
    """Rows [H, n, d] of sequence b in 64 bits."""
    pool = getattr(c, name)
    page = pool.shape[2]
    pos = torch.arange(n, device=pool.device)
    pages, at = table[b].long()[pos // page], pos % page
    x = pool.double()[pages, :, at] if pool.numel() < 1 << 24 else pool[pages, :, at].double()
    scale = getattr(c, name + "_scale")
    if scale is not None:
        x = x * scale[pages, :, at].double()[..., None]
    return x[..., :c.d_head].transpose(0, 1)


def quantised(x, fmt):
    """(codes, scales) of rows x [..., d] from the formats' definitions."""
    x = x.double()
    amax = x.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(x).all(-1, keepdim=True)
    if fmt == "int8":
        s = (amax / torch.full_like(amax, 127.0)).float().double().clamp(min=2.0 ** -126)  # by a number: by its inverse
        code = torch.round(x / s)  # ties to even; the quotient's own rounding is far below one border's distance
        code = code.masked_fill(bad, 0).to(torch.int8)
    else:
        m, e = torch.frexp(amax / 448.0)
        s = torch.exp2((e - (m == 0.5).int()).clamp(min=-126).double())
        s = torch.where(amax == 0, 2.0 ** -126, s)
        code = (x / s).masked_fill(bad, 0).float().to(torch.float8_e4m3fn)
    return code, s.float().masked_fill(bad, math.nan)[..., 0]


def seen_by(B, T, lens, news, window, n_persistent, tree=None):
    """Per sequence the mask [new, length]."""
    out = []
    w = window if window is not None else 1 << 40
    for b in range(B):
        n, new = lens[b], news[b]
        base = n - new
        j = torch.arange(n)
        if tree is None:
            p = torch.arange(base, n)[:, None]
            out.append((j < n_persistent) | ((p >= n_persistent) & (j >= p - w) & (j <= p)))
            continue
        bits = (tree[b] if tree.dim() == 2 else tree)[:new, None] >> torch.arange(64) & 1
        place = base + bits.sum(1) - 1  # of each drafted row
        near = torch.cat([j[:base], place]) >= place[:, None] - w
        allowed = torch.cat([torch.ones(new, base, dtype=torch.bool), bits[:, :new] == 1], dim=1)
        out.append(allowed & ((j < n_persistent) | near))
    return out


def check_attention(out, q, cache, table, lens, news, masks, scale=None):
    """out [B, H, T, d] against softmax(q·kᵀ·scale)·v in 64 bits over what the cache holds.

    Per result, with A = Σ p |v|: a score is an fp32 sum of d products (d E Σ |q k|), scaled and moved (4 E of its size);
    exponentials, sums over n keys, rescalings and joins stay below (n + 200) E of A; probabilities in 16 bit are off by
    half a step each (and by half of fp16's least number), and so is the result."""
    B, H, T, d = out.shape
    heads = cache.k.shape[1]
    half = {torch.float32: 2 * E, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[out.dtype]
    up = 0.0 if out.dtype == torch.float32 else half
    least = 2.0 ** -25 if out.dtype == torch.float16 else 0.0
    scale = d ** -0.5 if scale is None else scale
    for b in range(B):
        n, new = lens[b], news[b]
        assert torch.all(out[b, :, new:] == 0), b
        if new == 0:
            continue
        k, v = pool_rows(cache, table, b, n, "k"), pool_rows(cache, table, b, n, "v")
        mask = masks[b].to(out.device)
        k = torch.where(mask.any(0)[None, :, None], k, 0.0)  # what no row sees may be anything
        v = torch.where(mask.any(0)[None, :, None], v, 0.0)
        G = H // heads
        kk, vv = k.repeat_interleave(G, 0), v.repeat_interleave(G, 0)
        x = q[b, :, :new].double()
        z = (x @ kk.transpose(1, 2)) * scale
        size = (x.abs() @ kk.abs().transpose(1, 2)) * abs(scale)
        dz = ((d * E * size + 4 * E * z.abs()) * mask).amax(-1, keepdim=True)
        z = z.masked_fill(~mask, -math.inf)
        p = torch.softmax(z, -1).nan_to_num(0.0)
        want, A = p @ vv, p @ vv.abs()
        top = z.amax(-1, keepdim=True)
        weight = torch.exp(top - torch.logsumexp(z, -1, keepdim=True)).nan_to_num(0.0)  # 1 / Σ e^{z - max}
        tol = (A * (up + 2 * dz + 2 * (n + 200) * E) + least * 2 * weight * (vv.abs().amax(-2, keepdim=True) * n)
               + half * want.abs() + 1e-30)
        got = out[b, :, :new].double()
        bad = (got - want).abs() > tol
        assert not bad.any(), (b, int(bad.sum()), float(((got - want).abs() / tol).max()))
        empty = ~mask.any(-1)
        assert torch.all(got[:, empty] == 0)


def filled(dev, B, H, d, page, lens, dtype, fmt, seed=0, spread=1.0, fill=None, extra=2):
    """A cache that holds lens[b] random rows of each sequence (written by cache_write), its table and lengths."""
    per = max(1, -(-max(lens) // page))
    n_pages = B * per + extra
    c = empty_cache(dev, n_pages, H, d, page, dtype, fmt, fill)
    table = make_table(dev, B, per, n_pages, seed)
    lengths = torch.tensor(lens, dtype=torch.int32, device=dev)
    g = gen(dev, seed + 1)
    n = max(lens)
    k = (torch.randn(B, H, n, d, generator=g, device=dev) * spread).to(dtype)
    v = torch.randn(B, H, n, d, generator=g, device=dev).to(dtype)
    tc.cache_write(k, v, c, table, lengths, counts=lengths)
    return c, table, lengths


def check_two_numbers(out, q, cache, table, lens, news, masks, least=2.0 ** -25):
    """check_attention for probabilities that are held in two numbers in 16 bit: what both leave over is at most 2^-15 of a
    probability where the numbers are bfloat16 (whose step is 2^-7: the second is below 2^-6 and off by 2^-15), 2^-21 in
    fp16, and in fp16 `least` of the row's largest."""
    B, H, T, d = out.shape
    G = H // cache.k.shape[1]
    half = {torch.float32: 2 * E, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[out.dtype]
    of_fp16 = out.dtype == torch.float16 and cache.k_scale is None
    up = 0.0 if out.dtype == torch.float32 else 2.0 ** -21 if of_fp16 else 2.0 ** -15
    for b in range(B):
        n, new = lens[b], news[b]
        assert torch.all(out[b, :, new:] == 0), b
        if new == 0:
            continue
        mask = masks[b].to(out.device)
        any_sees = mask.any(0)[None, :, None]
        k, v = (torch.where(any_sees, pool_rows(cache, table, b, n, name), 0.0).repeat_interleave(G, 0) for name in "kv")
        x, scale = q[b, :, :new].double(), d ** -0.5
        z = ((x @ k.transpose(1, 2)) * scale).masked_fill(~mask, -math.inf)
        size = (x.abs() @ k.abs().transpose(1, 2)) * scale
        dz = ((d * E * size + 4 * E * z.abs().nan_to_num(0.0, 0.0)) * mask).amax(-1, keepdim=True)
        p = torch.softmax(z, -1).nan_to_num(0.0)
        want, A = p @ v, p @ v.abs()
        tol = A * (up + 2 * dz + 2 * (n + 200) * E) + half * want.abs() + 1e-30
        if out.dtype == torch.float16:  # the results' own least number, and that of the probabilities
            tol += 2.0 ** -25
            if of_fp16:
                tol += least * n * p.amax(-1, keepdim=True) * v.abs().amax(-2, keepdim=True)
        off = (out[b, :, :new].double() - want).abs()
        assert torch.all(off <= tol), (b, int((off > tol).sum()), float((off / tol).max()))


# B, T, H, heads, d, positions, page: between them, and over types and formats, every kernel of the attention is launched
SHAPES = [
    (10, 1, 20, 10, 64, 300, 16), (10, 1, 10, 10, 128, 300, 16),      # 16 rows, the keys over eight waves
    (30, 1, 10, 10, 64, 300, 64), (30, 1, 10, 10, 128, 300, 64),      # over four
    (6, 40, 10, 10, 128, 300, 32),
    (3, 1, 2, 2, 64, 5000, 64), (3, 1, 2, 2, 128, 5000, 64),          # in many parts
    (3, 1, 24, 24, 64, 5000, 64), (3, 1, 48, 24, 128, 5000, 64),      # in a few
    (18, 20, 10, 10, 64, 1700, 64), (18, 10, 20, 10, 128, 1700, 64),  # 32 rows, eight waves
    (27, 20, 10, 10, 64, 1700, 64), (27, 20, 10, 10, 128, 1700, 64),  # four waves
    (3, 30, 2, 2, 64, 5000, 64), (3, 30, 2, 2, 128, 5000, 64),        # in parts
    (4, 30, 16, 16, 64, 3000, 128), (4, 30, 16, 16, 128, 3000, 128),
    (15, 40, 8, 8, 96, 300, 16),                                      # fp32: 360 tiles of 16 rows
    (20, 200, 5, 5, 40, 300, 32), (12, 200, 8, 8, 128, 260, 32),      # rows over the waves
    (2, 320, 32, 4, 64, 1000, 32), (2, 320, 32, 4, 128, 1000, 256),   # in parts
]
