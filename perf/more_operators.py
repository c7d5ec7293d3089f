"""The key/value cache of the windowed attention with persistent tokens, and the attention that reads it.

- ``write``    cache_write in the model's type: new tokens' keys and values into the pages
- ``store``    cache_write in 8 bits with scales, then cache_read of everything that is held
- ``read``     cache_read: a prefix back as contiguous keys and values
- ``attend``   cached_attention: new tokens (one, or a chunk of a prompt) over the cache
- ``step``     cache_write, then cached_attention: what a layer does for each decoded token
- ``tree``     cached_attention of a tree of drafted tokens
- ``keep``     cache_keep: the draft's accepted rows move to their places

A cache is two pools [pages, key heads, page, pitch] with ``pitch`` the head's width rounded up to 16, in the
model's type or in 8 bits with a scale for each row; a table of pages for each sequence; and the sequences' lengths,
which count the new rows. Sizes are those of the model's configurations (10 heads of 64, a window of 512, 16 persistent
tokens, sequences of 4096), a grouped layout of 32 heads on 8, and odd ones around them.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}
STORED = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TINY = 2.0 ** -126  # the least scale


def _tc():
    pkg = os.path.join(os.getcwd(), "titanmac-standalone_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import titans_core
    return titans_core


# ------------------------------------------------------------------ the cases

def _case(kind, B, T, length, dtype, fmt="same", H=10, Hkv=None, d=64, page=64, window=0, np=0, ragged=False):
    """T new tokens in each of B sequences of `length` positions (these included); window 0: none. ragged: lengths
    down to half of it, and in each third sequence fewer new tokens."""
    return {"kind": kind, "B": B, "T": T, "len": length, "H": H, "Hkv": H if Hkv is None else Hkv, "d": d, "page": page,
            "window": window, "np": np, "ragged": ragged, "dtype": dtype, "fmt": fmt}


def listed():
    return [
        # 16 sequences decode: one token's keys and values each
        dict(_case("write", 16, 1, 1024, "bf16"), name="write_decode_16"),
        # prompts of up to 2047 tokens kept in 8 bits, and read back for a chunk behind them
        dict(_case("store", 8, 2047, 2047, "bf16", "e4m3", ragged=True), name="store_prompt_8x2047"),
        # a prefix that four sequences share is read back from 8 bits
        dict(_case("read", 4, 0, 4096, "bf16", "int8"), name="read_prefix_4x4096"),
        # what one layer does for a decoded token of 16 sequences, in the model's window
        dict(_case("step", 16, 1, 4096, "bf16", window=512, np=16, ragged=True), name="step_16"),
        # one sequence, one token: latency
        dict(_case("attend", 1, 1, 4096, "fp16", window=512, np=16), name="attend_one"),
        # 64 sequences on a cache in 8 bits
        dict(_case("attend", 64, 1, 4096, "bf16", "int8", window=512, np=16, ragged=True), name="attend_64_int8"),
        # long texts without a window, 32 heads on 8
        dict(_case("attend", 16, 1, 32768, "bf16", H=32, Hkv=8, d=128), name="attend_long_16x32768"),
        # a prompt that arrives in chunks of 1024
        dict(_case("attend", 2, 1024, 8192, "bf16", window=4096, np=16), name="chunk_2x1024"),
        # drafts of 61 tokens are checked at once
        dict(_case("tree", 16, 61, 4096, "bf16", "e4m3", window=512, np=16, ragged=True), name="tree_16x61"),
        # a small draft without mixed precision
        dict(_case("tree", 3, 13, 683, "fp32", H=8, page=16, window=256, np=4, ragged=True), name="tree_f32_3x13"),
        # the accepted rows of 64 drafts
        dict(_case("keep", 64, 32, 1024, "bf16"), name="keep_64"),
        # and of a few in fp32, heads of an odd width
        dict(_case("keep", 3, 13, 683, "fp32", H=8, d=40, page=16), name="keep_f32_3"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["write", "store", "read", "step", "attend", "attend", "attend", "chunk", "tree", "tree", "keep"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    fmt = "same" if kind in ("write", "step", "keep") else rng.choice(["same", "int8", "e4m3"])
    if kind == "store":
        fmt = rng.choice(["int8", "e4m3"])
    H, Hkv = rng.choice([(10, 10), (10, 10), (8, 8), (32, 8), (12, 4), (7, 1)])
    c = {"H": H, "Hkv": Hkv, "d": rng.choice([64, 64, 128, 32, 40, 96]), "page": rng.choice([16, 32, 64, 128, 256]),
         "ragged": rng.random() < 0.6}
    if kind in ("write", "store"):
        T = _log_int(rng, 1, 2048)
        B = _log_int(rng, 1, max(1, min(64, 32768 // T)))
        return _case(kind, B, T, T + rng.choice([0, 1, 100]), dtype, fmt, **c)
    if kind == "keep":
        return _case(kind, _log_int(rng, 1, 64), rng.randint(2, 64), rng.randint(200, 1500), dtype, fmt, **c)
    length = _log_int(rng, 64, 16384)
    B = _log_int(rng, 1, max(1, min(64, 131072 // length)))
    if kind == "read":
        return _case(kind, B, 0, length, dtype, fmt, **c)
    c["window"] = rng.choice([0, 128, 512, 512, 777, 4096])
    c["np"] = rng.choice([0, 4, 16, 33])
    T = 1
    if kind == "tree":
        T = min(rng.randint(2, 64), length // 2)
    elif kind == "chunk":
        kind, T = "attend", min(_log_int(rng, 2, 1024), length)
    B = max(1, min(B, 20_000_000_000 // (T * length * H * c["d"])))
    return _case(kind, B, T, length, dtype, fmt, **c)


def _lengths(c):
    """The positions that each sequence holds, and how many of them are new."""
    lens, news = [], []
    for b in range(c["B"]):
        n = c["T"] - (c["T"] // 3 if c["ragged"] and b % 3 == 2 else 0)
        short = b * 389 % (c["len"] // 2) if c["ragged"] and c["len"] > 3 else 0
        lens.append(max(c["len"] - short, n, 1))
        news.append(n)
    return lens, news


# ------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _pitch(c):
    return -(-c["d"] // 16) * 16


def _pool(g, c, pages):
    """A pool as a running server has it: every row of an earlier token, also where nothing is held now."""
    shape = (pages, c["Hkv"], c["page"], _pitch(c))
    dt = DTYPES[c["dtype"]] if c["fmt"] == "same" else None
    x = torch.randn(shape, generator=g, device=DEV, dtype=dt or torch.bfloat16)
    x[..., c["d"]:] = 0
    if dt is not None:
        return x, None
    scale = torch.rand(shape[:3], generator=g, device=DEV) * 0.5 + 0.75
    if c["fmt"] == "int8":
        return (x.float() * 42.0).round_().clamp_(-127, 127).to(torch.int8), scale / 42.0
    return (x.float() * 100.0).clamp_(-448, 448).to(torch.float8_e4m3fn), torch.exp2((scale * 4).floor() - 10.0)


def _tree(c, g):
    """Each drafted token's ancestors and itself, as bits: parents drawn among the tokens before it."""
    B, T = c["B"], c["T"]
    u = torch.rand(B, T, generator=g, device=DEV).cpu()
    rows = []
    for b in range(B):
        bits = [1]
        for t in range(1, T):
            bits.append(bits[int(u[b, t] * t * 0.999)] | 1 << t)
        rows.append([x - (1 << 64) if x >> 63 else x for x in bits])
    return torch.tensor(rows, dtype=torch.int64, device=DEV)


def prepare(case, seed):
    c, g = case, _gen(seed)
    lens, news = _lengths(c)
    per = -(-max(lens) // c["page"])
    pages = c["B"] * per + 3
    s = {"case": c}
    s["table"] = torch.randperm(pages, generator=g, device=DEV)[:c["B"] * per].view(c["B"], per).int()
    s["lengths"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    s["counts"] = torch.tensor(news, dtype=torch.int32, device=DEV) if c["ragged"] else None
    s["k_pool"], s["k_scale"] = _pool(g, c, pages)
    s["v_pool"], s["v_scale"] = _pool(g, c, pages)
    if c["kind"] == "keep":
        # a path from the root: its other nodes are behind those that it replaces, as in a draft with wide levels
        T = c["T"]
        A = max(1, min(8, T // 4))
        u = torch.rand(c["B"], T, generator=g, device=DEV)
        u[:, :A] = 2.0
        u[:, T - T // 3:] = 2.0
        path = u.argsort(dim=1)[:, :A].sort(dim=1).values
        path[:, 0] = 0
        s["path"] = path.int()
    elif c["kind"] != "read":
        # one projection's output holds the queries, keys and values
        H, K, d = c["H"], c["Hkv"], c["d"]
        x = torch.randn(c["B"], c["T"], H + 2 * K, d, generator=g, device=DEV).to(DTYPES[c["dtype"]]).transpose(1, 2)
        s["q"], s["k"], s["v"] = x[:, :H], x[:, H:H + K], x[:, H + K:]
    if c["kind"] == "tree":
        s["tree"] = _tree(c, g)
    return s


# ------------------------------------------------------------------ one pass, plain form

def _new_positions(s, c):
    """Positions [B, T] of the new rows, and which of them there are."""
    t = torch.arange(c["T"], device=DEV)
    n = s["counts"] if s["counts"] is not None else torch.full_like(s["lengths"], c["T"])
    return (s["lengths"] - n)[:, None] + t, t < n[:, None]


def _slots(s, c, pos):
    """(page, place in it) of positions [B, n]."""
    return s["table"].long().gather(1, (pos // c["page"]).clamp_(0, s["table"].shape[1] - 1).long()), pos % c["page"]


def _plain_quantise(x, fmt):
    """Codes and scales of rows [..., d]; in 64 bits, as a value next to a border goes by its quotient."""
    amax = x.abs().amax(-1, keepdim=True).float()
    if fmt == "int8":
        scale = (amax.double() / 127).float().clamp(min=TINY)
        return (x.double() / scale.double()).round().to(torch.int8), scale[..., 0]
    m, e = torch.frexp(amax)  # amax = m 2^e, 1/2 <= m < 1; 448 = 0.875 2^9
    scale = torch.exp2((e - 9 + (m > 0.875)).clamp(min=-126).float())
    scale = torch.where(amax == 0, TINY, scale)
    return (x.double() / scale.double()).float().to(torch.float8_e4m3fn), scale[..., 0]


def _plain_write(s, c):
    pos, there = _new_positions(s, c)
    page, at = _slots(s, c, pos)
    page, at = page[there], at[there]
    _plain_write_one(s, c, "k", page, at, there)
    _plain_write_one(s, c, "v", page, at, there)


def _plain_write_one(s, c, name, page, at, there):
    x = s[name].transpose(1, 2)[there]  # [rows, heads, d]
    if c["fmt"] != "same":
        x, scale = _plain_quantise(x, c["fmt"])
        s[name + "_scale"][page, :, at] = scale
    pool = s[name + "_pool"]
    if c["fmt"] == "e4m3":
        x, pool = x.view(torch.uint8), pool.view(torch.uint8)
    pool[page, :, at, :c["d"]] = x


def _plain_values(s, c, name):
    """Everything that the table names, in 32 bits: [B, Hkv, positions, d]."""
    t = s["table"].long()
    x = s[name + "_pool"][t][..., :c["d"]].float()
    if c["fmt"] != "same":
        x = x * s[name + "_scale"][t][..., None]
    return x.transpose(1, 2).flatten(2, 3)


def _plain_read(s, c):
    n = max(_lengths(c)[0])
    held = (torch.arange(n, device=DEV) < s["lengths"][:, None])[:, None, :, None]
    dt = DTYPES[c["dtype"]]
    return (torch.where(held, _plain_values(s, c, "k")[:, :, :n], 0.0).to(dt),
            torch.where(held, _plain_values(s, c, "v")[:, :, :n], 0.0).to(dt))


def _plain_seen(s, c, n):
    """Which of n positions each new row sees: [B, T, n]."""
    pos, there = _new_positions(s, c)
    j = torch.arange(n, device=DEV)
    w, np = c["window"] or 1 << 30, c["np"]
    if c["kind"] != "tree":
        p = pos[..., None]
        seen = (j < np) | ((p >= np) & (j >= p - w) & (j <= p))
    else:
        T, base = c["T"], pos[:, :1]
        bits = (s["tree"][..., None] >> torch.arange(T, device=DEV)) & 1  # [B, T, s]
        p = base + bits.sum(-1) - 1
        at = torch.where(j < base, j, p.gather(1, (j - base).clamp(0, T - 1)))  # the keys' positions
        draft = bits.gather(2, (j - base).clamp(0, T - 1)[:, None].expand(-1, T, -1)) == 1
        ok = torch.where((j < base)[:, None], True, draft & (j - base < T)[:, None])
        seen = ok & ((j < np) | (at[:, None] >= p[..., None] - w))
    return seen & (j < s["lengths"][:, None])[:, None] & there[..., None]


def _plain_attend(s, c):
    k, v = _plain_values(s, c, "k"), _plain_values(s, c, "v")
    B, K, n, d = k.shape
    G, T = c["H"] // c["Hkv"], c["T"]
    q = s["q"].reshape(B, K, G * T, d).float() * d ** -0.5
    seen = _plain_seen(s, c, n)[:, None, None]
    x = torch.where(seen, (q @ k.transpose(2, 3)).view(B, K, G, T, n), -math.inf)
    p = torch.where(seen, torch.exp(x - x.amax(-1, keepdim=True)), 0.0)
    total = p.sum(-1).view(B, K, G * T, 1)
    o = torch.where(total > 0, (p.view(B, K, G * T, n) @ v) / total, 0.0)
    return o.view(B, c["H"], T, d).to(DTYPES[c["dtype"]])


def _plain_keep(s, c):
    pos, _ = _new_positions(s, c)
    A = s["path"].shape[1]
    page, at = _slots(s, c, pos.gather(1, s["path"].long()))
    to, into = _slots(s, c, pos[:, :A])
    s["k_pool"][to, :, into] = s["k_pool"][page, :, at]
    s["v_pool"][to, :, into] = s["v_pool"][page, :, at]


def run(s):
    c = s["case"]
    kind = c["kind"]
    if own:
        return _run_own(s, c)
    if kind in ("write", "store", "step"):
        _plain_write(s, c)
    if kind in ("store", "read"):
        return _plain_read(s, c)
    if kind == "keep":
        _plain_keep(s, c)
    if kind in ("write", "keep"):
        return s["k_pool"], s["v_pool"]
    o = _plain_attend(s, c)
    return (o, s["k_pool"], s["v_pool"]) if kind == "step" else o


# ------------------------------------------------------------------ one pass, the framework's

def _run_own(s, c):
    tc = _tc()
    kind, table, lengths, counts = c["kind"], s["table"], s["lengths"], s["counts"]
    cache = tc.KVCache(s["k_pool"], s["v_pool"], c["d"], s["k_scale"], s["v_scale"])
    if kind in ("write", "store", "step"):
        tc.cache_write(s["k"], s["v"], cache, table, lengths, counts=counts)
    if kind in ("store", "read"):
        return tc.cache_read(cache, table, lengths, c["len"], dtype=DTYPES[c["dtype"]])
    if kind == "keep":
        tc.cache_keep(cache, table, lengths, s["path"], c["T"] if counts is None else counts)
    if kind in ("write", "keep"):
        return s["k_pool"], s["v_pool"]
    o = tc.cached_attention(s["q"], cache, table, lengths, c["window"] or None, c["np"], counts=counts,
                            tree=s.get("tree"))
    return (o, s["k_pool"], s["v_pool"]) if kind == "step" else o


# ------------------------------------------------------------------ the definition, in 64 bits

def _exact_rows(s, c, b, name, scaled=True):
    """Sequence b's rows [Hkv, length, d] in 64 bits."""
    n = int(s["lengths"][b])
    rows = []
    for j in range(0, n, c["page"]):
        page = int(s["table"][b, j // c["page"]])
        x = s[name + "_pool"][page, :, :min(c["page"], n - j), :c["d"]].double()
        if c["fmt"] != "same":
            x = x * s[name + "_scale"][page, :, :min(c["page"], n - j), None].double()
        rows.append(x)
    return torch.cat(rows, dim=1)


def _exact_round(x, fmt):
    """The values that rows x [..., d] in 64 bits are held as, from the formats' definitions."""
    amax = x.abs().amax(-1, keepdim=True)
    if fmt == "int8":
        s = torch.maximum((amax / 127).float().double(), torch.full_like(amax, TINY))
        return torch.round(x / s) * s
    s = torch.full_like(amax, TINY)
    e = torch.ceil(torch.log2(amax.clamp(min=1e-300) / 448.0))
    for shift in (-1, 0, 1):  # the least power of two that holds the row
        t = torch.exp2(e + shift)
        s = torch.where((448.0 * t >= amax) & (224.0 * t < amax), torch.maximum(t, s), s)
    y = x / s
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step * s


def exact(case, seed):
    c, s = case, prepare(case, seed)
    lens, news = _lengths(c)
    kind, B, K, d = c["kind"], c["B"], c["Hkv"], c["d"]
    if kind in ("write", "keep", "step"):
        pools = [s[n + "_pool"].double() for n in ("k", "v")]
        was = [p.clone() for p in pools]
        for b in range(B):
            base = lens[b] - news[b]
            if kind == "keep":
                todo = [(int(t), base + a) for a, t in enumerate(s["path"][b])]
            else:
                todo = [(t, base + t) for t in range(news[b])]
            pos = torch.tensor([p for _, p in todo], device=DEV)
            src = torch.tensor([t for t, _ in todo], device=DEV)
            page, at = s["table"][b].long()[pos // c["page"]], pos % c["page"]
            for i, name in enumerate(("k", "v")):
                if kind == "keep":
                    old = src + base
                    pools[i][page, :, at] = was[i][s["table"][b].long()[old // c["page"]], :, old % c["page"]]
                else:
                    pools[i][page, :, at, :d] = s[name][b, :, src].transpose(0, 1).double()
        if kind != "step":
            return tuple(pools)
        for i, name in enumerate(("k", "v")):
            s[name + "_pool"] = pools[i]
    if kind in ("store", "read"):
        out = []
        for name in ("k", "v"):
            y = torch.zeros(B, K, max(lens), d, dtype=torch.float64, device=DEV)
            for b in range(B):
                y[b, :, :lens[b]] = _exact_rows(s, c, b, name)
                if kind == "store":
                    y[b, :, lens[b] - news[b]:lens[b]] = _exact_round(s[name][b, :, :news[b]].double(), c["fmt"])
            out.append(y)
        return tuple(out)
    w, np = c["window"] or 1 << 30, c["np"]
    o = torch.zeros(B, c["H"], c["T"], d, dtype=torch.float64, device=DEV)
    for b in range(B):
        n, new = lens[b], news[b]
        base = n - new
        k, v = _exact_rows(s, c, b, "k"), _exact_rows(s, c, b, "v")
        at = torch.arange(n, device=DEV)
        mask = torch.zeros(new, n, dtype=torch.bool, device=DEV)
        if kind == "tree":
            bits = [int(x) & (1 << 64) - 1 for x in s["tree"][b, :new].tolist()]
            depth = torch.tensor([bin(x).count("1") - 1 for x in bits], device=DEV)
            at = torch.cat([at[:base], base + depth])
            mask[:, :base] = True
            mask[:, base:] = torch.tensor([[bool(x >> i & 1) for i in range(new)] for x in bits], device=DEV)
            p = base + depth
        else:
            p = torch.arange(base, n, device=DEV)
            mask |= at <= p[:, None]
        j = torch.arange(n, device=DEV)
        mask &= (at >= p[:, None] - w) | (j < np)
        if kind != "tree":
            mask[:, :min(np, n)] = True
            mask &= (p[:, None] >= np) | (j < np)
        for h in range(c["H"]):
            hk = h // (c["H"] // K)
            z = (s["q"][b, h, :new].double() @ k[hk].t()) / math.sqrt(d)
            o[b, h, :new] = torch.softmax(z.masked_fill(~mask, -math.inf), -1).nan_to_num(0.0) @ v[hk]
    return (o, *pools) if kind == "step" else o


# ------------------------------------------------------------------ what a pass cannot do without

def _spans(c, n, new):
    """(keys that the new rows see between them, and in all) of one sequence. In a tree each row is taken to see all
    committed keys of its window and half of the draft."""
    w, np = c["window"] or 1 << 30, min(c["np"], n)
    base = n - new
    if c["kind"] == "tree":
        own_ = n - max(np, base - w) if base > np else new
        return np + own_, new * (np + own_ - new // 2)
    first = max(np, base - w)
    total = sum(np + min(p - np, w) + 1 if p >= np else np for p in range(base, n))
    return np + max(0, n - first), total


def work(case):
    c = case
    lens, news = _lengths(c)
    e = SIZES[c["dtype"]]
    held = e * c["d"] if c["fmt"] == "same" else c["d"] + 4
    rows, kept = sum(news) * c["Hkv"], sum(lens) * c["Hkv"]
    kind = c["kind"]
    if kind == "write":
        return {"bytes": 4 * rows * e * c["d"], "flops": 0}
    if kind == "store":
        return {"bytes": 2 * rows * (e * c["d"] + held) + 2 * kept * (held + e * c["d"]), "flops": 4 * rows * c["d"]}
    if kind == "read":
        return {"bytes": 2 * kept * (held + e * c["d"]), "flops": 2 * kept * c["d"]}
    if kind == "keep":
        return {"bytes": 4 * c["B"] * max(1, min(8, c["T"] // 4)) * c["Hkv"] * held, "flops": 0}
    spans = [_spans(c, n, t) for n, t in zip(lens, news)]
    io = 2 * sum(news) * c["H"] * e * c["d"]
    seen = 2 * sum(k for k, _ in spans) * c["Hkv"] * held
    step = 4 * rows * e * c["d"] if kind == "step" else 0
    return {"bytes": io + seen + step, "flops": 4 * c["d"] * c["H"] * sum(t for _, t in spans)}
