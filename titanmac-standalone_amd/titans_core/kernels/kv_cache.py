"""Key/value cache of the windowed attention with persistent tokens, and attention over it (HIP kernels for gfx950).

``WindowedAttention`` is causal and its persistent rows see persistent keys only (attn/windowed_attention.py:97-152),
so the keys and values of a text need not be computed again for the tokens behind it. A ``KVCache`` holds them in
pages; ``cache_write`` puts new tokens' rows there, ``cached_attention`` is the attention of the new tokens (one, a
chunk of a prompt, or a tree of drafted ones) over everything that is held, ``cache_keep`` moves a draft's accepted
rows to their places and ``cache_read`` gives the rows back.

All four take the same description of the sequences:

- ``table`` int32 [B, pages]: the page of the pools with positions ``page·j .. page·j + page − 1``;
- ``lengths`` int32 [B]: the positions that each sequence holds, its new rows included;
- ``counts`` int32 [B], optional: how many rows are new, at most T (default: T, or the length where that is less).
  New row t is position ``length − count + t``; rows t ≥ count are none.

They stay on the GPU and nothing is copied to the host to look at them: a sequence whose numbers do not fit (a length
below 0 or past its table, a count below 0, above T or above the length) is not written and reads as NaN, and so does a
page outside the pools.
"""
from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import Optional, Union

import torch

from . import _lib

SAME, INT8, E4M3 = 0, 1, 2
_FORMATS = {torch.int8: INT8, torch.float8_e4m3fn: E4M3}
_NAMES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
PAGES = (16, 32, 64, 128, 256)
MAX_HEAD, MAX_TREE = 128, 64
_NO_WINDOW = 1 << 30


class CacheArg(ctypes.Structure):
    """tmac_cache."""
    _fields_ = [("d_k", ctypes.c_void_p), ("d_v", ctypes.c_void_p), ("d_k_scale", ctypes.c_void_p),
                ("d_v_scale", ctypes.c_void_p), ("d_table", ctypes.c_void_p), ("d_lengths", ctypes.c_void_p),
                ("d_counts", ctypes.c_void_p), ("n_pages", ctypes.c_int64), ("table_stride", ctypes.c_int64),
                ("n_heads", ctypes.c_int), ("page", ctypes.c_int), ("pitch", ctypes.c_int), ("d_head", ctypes.c_int),
                ("max_pages", ctypes.c_int), ("format", ctypes.c_int), ("dtype", ctypes.c_int)]


class KVCache:
    """Pools of keys and values: ``k``, ``v`` [n_pages, n_heads, page, pitch], contiguous, rows of d_head values behind
    which are zeros up to the pitch (d_head rounded up to 16); page 16, 32, 64, 128 or 256, d_head up to 128. Their
    type is the model's (float32, bfloat16, float16), or int8 or float8_e4m3fn with a scale for each row in ``k_scale``,
    ``v_scale`` (float32 [n_pages, n_heads, page]): a value is code · scale. ``KVCache.new`` makes them."""

    __slots__ = ("k", "v", "d_head", "k_scale", "v_scale")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, d_head: Optional[int] = None,
                 k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None):
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.d_head = k.shape[-1] if d_head is None else d_head

    @classmethod
    def new(cls, n_pages: int, n_heads: int, d_head: int, *, page: int = 64, dtype: torch.dtype = torch.bfloat16,
            fmt: Optional[str] = None, device="cuda") -> "KVCache":
        """An empty cache (zeros) of values of dtype, held as they are or as fmt "int8" or "e4m3"."""
        if fmt is not None and fmt not in _NAMES:
            raise ValueError(f"KVCache: fmt must be None, 'int8' or 'e4m3', got {fmt!r}")
        if dtype not in _lib._DTYPE_CODE:
            raise TypeError(f"KVCache: dtype must be float32, bfloat16 or float16, got {dtype}")
        if page not in PAGES or not 1 <= d_head <= MAX_HEAD or n_pages < 1 or n_heads < 1:
            raise ValueError(f"KVCache: page must be one of {PAGES} and d_head 1..{MAX_HEAD}, got {page}, {d_head} "
                             f"({n_pages} pages, {n_heads} heads)")
        shape = (n_pages, n_heads, page, -(-d_head // 16) * 16)
        store = dtype if fmt is None else _NAMES[fmt]
        scale = lambda: None if fmt is None else torch.zeros(shape[:3], dtype=torch.float32, device=device)  # noqa: E731
        return cls(torch.zeros(shape, dtype=store, device=device), torch.zeros(shape, dtype=store, device=device),
                   d_head, scale(), scale())


def _check_cache(what: str, c: KVCache, table, lengths, counts, dtype: torch.dtype, T: int, B: int) -> None:
    k, v, ks, vs = c.k, c.v, c.k_scale, c.v_scale
    if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype:
        raise ValueError(f"{what}: the pools must be [n_pages, n_heads, page, pitch], alike, got {tuple(k.shape)} {k.dtype} "
                         f"and {tuple(v.shape)} {v.dtype}")
    if k.shape[2] not in PAGES or not 1 <= c.d_head <= MAX_HEAD or k.shape[3] != -(-c.d_head // 16) * 16:
        raise ValueError(f"{what}: pages of {PAGES} rows of d_head (1..{MAX_HEAD}) rounded up to 16 values, got "
                         f"{tuple(k.shape)} for d_head {c.d_head}")
    if not (k.is_contiguous() and v.is_contiguous()):
        raise ValueError(f"{what}: the pools must be contiguous")
    if dtype not in _lib._DTYPE_CODE:
        raise TypeError(f"{what}: unsupported dtype {dtype}; expected float32, bfloat16 or float16")
    if k.dtype in _FORMATS:
        for s in (ks, vs):
            if s is None or s.dtype != torch.float32 or s.shape != k.shape[:3] or not s.is_contiguous():
                raise ValueError(f"{what}: a cache in {k.dtype} needs k_scale and v_scale, float32 {tuple(k.shape[:3])}, "
                                 "contiguous")
    elif k.dtype != dtype:
        raise TypeError(f"{what}: a cache of {k.dtype} does not hold {dtype}")
    if table.dtype != torch.int32 or lengths.dtype != torch.int32 or (counts is not None and counts.dtype != torch.int32):
        raise TypeError(f"{what}: table, lengths and counts must be int32")
    if table.dim() != 2 or table.shape[0] != B or table.shape[1] == 0:
        raise ValueError(f"{what}: table must be [{B}, pages], got {tuple(table.shape)}")
    for name, t in (("lengths", lengths), ("counts", counts)):
        if t is not None and t.shape != (B,):
            raise ValueError(f"{what}: {name} must be [{B}], got {tuple(t.shape)}")
    if B > 1 << 20 or T * k.shape[1] > 1 << 26 or table.shape[1] > (1 << 30) // k.shape[2]:
        raise ValueError(f"{what}: up to 2^20 sequences, 2^26 rows of one and 2^30 positions")


def _no_grad(what: str, *tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise NotImplementedError(f"{what} has no gradient: call it under torch.no_grad()")


def _unit(t: torch.Tensor) -> torch.Tensor:
    """t with its last dimension contiguous."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _flat(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return t if t is None or t.is_contiguous() else t.contiguous()


def _pitch(t: torch.Tensor) -> int:
    """Pitch of a table's rows (any, if there is one row)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _arg(k, v, ks, vs, table, lengths, counts, d, dtype) -> CacheArg:
    n, h, page, pitch = k.shape
    p = _lib.ptr
    return CacheArg(k.data_ptr(), v.data_ptr(), p(ks), p(vs), table.data_ptr(), lengths.data_ptr(), p(counts), n,
                    _pitch(table), h, page, pitch, d, table.shape[1], _FORMATS.get(k.dtype, SAME),
                    _lib._DTYPE_CODE[dtype])


def _strides(t: torch.Tensor):
    """(batch, head, row) strides of [B, H, T, d]."""
    return (ctypes.c_int64 * 3)(t.stride(0), t.stride(1), t.stride(2))


def _table(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(1) == 1 and (t.shape[0] == 1 or t.stride(0) >= t.shape[1]) else t.contiguous()


# ------------------------------------------------------------------ write

def _native_write(new_k, new_v, k, v, ks, vs, table, lengths, counts, d) -> None:
    dev = _lib.require_device(*(t for t in (k, v, new_k, new_v, ks, vs, table, lengths, counts) if t is not None),
                              what="cache_write")
    B, _, T, _ = new_k.shape
    if new_k.numel() == 0:
        return
    new_k, new_v, table, lengths, counts = _unit(new_k), _unit(new_v), _table(table), _flat(lengths), _flat(counts)
    arg = _arg(k, v, ks, vs, table, lengths, counts, d, new_k.dtype)
    with _lib.device_guard(dev):
        rc = _lib.lib().tmac_cache_write(ctypes.byref(arg), new_k.data_ptr(), _strides(new_k), new_v.data_ptr(),
                                         _strides(new_v), B, T, _lib.stream_ptr(dev))
    _lib.check(rc, "tmac_cache_write")


@torch.library.custom_op("titanmac::cache_write", mutates_args=("k", "v", "ks", "vs"))
def cache_write_op(new_k: torch.Tensor, new_v: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                   ks: Optional[torch.Tensor], vs: Optional[torch.Tensor], table: torch.Tensor, lengths: torch.Tensor,
                   counts: Optional[torch.Tensor], d: int) -> None:
    _native_write(new_k, new_v, k, v, ks, vs, table, lengths, counts, d)


@cache_write_op.register_fake
def _(new_k, new_v, k, v, ks, vs, table, lengths, counts, d):
    return None


def cache_write(k: torch.Tensor, v: torch.Tensor, cache: KVCache, table: torch.Tensor, lengths: torch.Tensor, *,
                counts: Optional[torch.Tensor] = None) -> None:
    """The new rows k, v [B, n_heads, T, d_head] (any strides) into the cache, in place.

    In 8 bits every row has its own scale: int8 codes are value / scale rounded to nearest (ties to even) with scale =
    max |value| / 127, e4m3 codes likewise with the least power of two that holds the row as scale (both at least
    2^-126). A row that is not finite is held as NaN. Pages that are written must not belong to two sequences."""
    what = "cache_write"
    if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype:
        raise ValueError(f"{what}: k and v must be [B, n_heads, T, d_head], alike, got {tuple(k.shape)} {k.dtype} and "
                         f"{tuple(v.shape)} {v.dtype}")
    B, H, T, d = k.shape
    _check_cache(what, cache, table, lengths, counts, k.dtype, T, B)
    if H != cache.k.shape[1] or d != cache.d_head:
        raise ValueError(f"{what}: the cache has {cache.k.shape[1]} heads of {cache.d_head}, k is {tuple(k.shape)}")
    _no_grad(what, k, v, cache.k, cache.v)
    args = (k, v, cache.k, cache.v, cache.k_scale, cache.v_scale, table, lengths, counts, cache.d_head)
    if _lib.direct_call(*args[:-1]):
        _native_write(*args)
        _changed(cache)
    else:
        cache_write_op(*args)


def _changed(cache: KVCache) -> None:
    """What autograd (or a caller's cache) keeps of the pools is out of date."""
    for t in (cache.k, cache.v, cache.k_scale, cache.v_scale):
        if t is not None and not t.is_inference():
            torch.autograd.graph.increment_version(t)


# ------------------------------------------------------------------ read

def _native_read(k, v, ks, vs, table, lengths, T, d, dtype):
    dev = _lib.require_device(*(t for t in (k, v, ks, vs, table, lengths) if t is not None), what="cache_read")
    B, H = table.shape[0], k.shape[1]
    out_k = torch.empty((B, H, T, d), dtype=dtype, device=dev)
    out_v = torch.empty((B, H, T, d), dtype=dtype, device=dev)
    if out_k.numel() == 0:
        return out_k, out_v
    table, lengths = _table(table), _flat(lengths)
    arg = _arg(k, v, ks, vs, table, lengths, None, d, dtype)
    with _lib.device_guard(dev):
        rc = _lib.lib().tmac_cache_read(ctypes.byref(arg), out_k.data_ptr(), out_v.data_ptr(), B, T, _lib.stream_ptr(dev))
    _lib.check(rc, "tmac_cache_read")
    return out_k, out_v


@torch.library.custom_op("titanmac::cache_read", mutates_args=())
def cache_read_op(k: torch.Tensor, v: torch.Tensor, ks: Optional[torch.Tensor], vs: Optional[torch.Tensor],
                  table: torch.Tensor, lengths: torch.Tensor, T: int, d: int,
                  dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
    return _native_read(k, v, ks, vs, table, lengths, T, d, dtype)


@cache_read_op.register_fake
def _(k, v, ks, vs, table, lengths, T, d, dtype):
    return tuple(k.new_empty((table.shape[0], k.shape[1], T, d), dtype=dtype) for _ in range(2))


def cache_read(cache: KVCache, table: torch.Tensor, lengths: torch.Tensor, n_positions: int, *,
               dtype: Optional[torch.dtype] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Positions 0 .. n_positions − 1 of every sequence as k, v [B, n_heads, n_positions, d_head]: zeros behind a
    sequence's length. dtype: the values' type (default: the cache's, bfloat16 for one in 8 bits)."""
    what = "cache_read"
    if dtype is None:
        dtype = torch.bfloat16 if cache.k.dtype in _FORMATS else cache.k.dtype
    T = int(n_positions)
    if T < 0:
        raise ValueError(f"{what}: n_positions must not be negative, got {T}")
    _check_cache(what, cache, table, lengths, None, dtype, T, lengths.shape[0] if lengths.dim() == 1 else -1)
    _no_grad(what, cache.k, cache.v)
    args = (cache.k, cache.v, cache.k_scale, cache.v_scale, table, lengths)
    run = _native_read if _lib.direct_call(*args) else cache_read_op
    return run(*args, T, cache.d_head, dtype)


# ------------------------------------------------------------------ keep

def _native_keep(k, v, ks, vs, table, lengths, counts, path, T, d) -> None:
    dev = _lib.require_device(*(t for t in (k, v, ks, vs, table, lengths, counts, path) if t is not None),
                              what="cache_keep")
    B, A = path.shape
    if B == 0 or A == 0:
        return
    table, lengths, counts, path = _table(table), _flat(lengths), _flat(counts), _table(path)
    arg = _arg(k, v, ks, vs, table, lengths, counts, d, torch.bfloat16 if k.dtype in _FORMATS else k.dtype)
    with _lib.device_guard(dev):
        rc = _lib.lib().tmac_cache_keep(ctypes.byref(arg), path.data_ptr(), _pitch(path), A, B, T, _lib.stream_ptr(dev))
    _lib.check(rc, "tmac_cache_keep")


@torch.library.custom_op("titanmac::cache_keep", mutates_args=("k", "v", "ks", "vs"))
def cache_keep_op(k: torch.Tensor, v: torch.Tensor, ks: Optional[torch.Tensor], vs: Optional[torch.Tensor],
                  table: torch.Tensor, lengths: torch.Tensor, counts: Optional[torch.Tensor], path: torch.Tensor, T: int,
                  d: int) -> None:
    _native_keep(k, v, ks, vs, table, lengths, counts, path, T, d)


@cache_keep_op.register_fake
def _(k, v, ks, vs, table, lengths, counts, path, T, d):
    return None


def cache_keep(cache: KVCache, table: torch.Tensor, lengths: torch.Tensor, path: torch.Tensor,
               counts: Union[int, torch.Tensor]) -> None:
    """Of each sequence's draft, its last ``counts`` rows (up to 64; one number for all, or int32 [B]): row path[b, a]
    (int32 [B, A]) moves to place a of the draft, for all a at once. An entry outside the draft (−1) leaves its place as
    it is. The caller then shortens ``lengths`` to the rows that were kept."""
    what = "cache_keep"
    T = MAX_TREE if isinstance(counts, torch.Tensor) else int(counts)
    n = counts if isinstance(counts, torch.Tensor) else None
    if path.dim() != 2 or path.dtype != torch.int32:
        raise ValueError(f"{what}: path must be int32 [B, rows], got {path.dtype} {tuple(path.shape)}")
    if not 0 <= T <= MAX_TREE or path.shape[1] > T:
        raise ValueError(f"{what}: drafts of up to {MAX_TREE} rows, no more kept than drafted, got {T} and "
                         f"{path.shape[1]}")
    dtype = torch.bfloat16 if cache.k.dtype in _FORMATS else cache.k.dtype
    _check_cache(what, cache, table, lengths, n, dtype, T, path.shape[0])
    _no_grad(what, cache.k, cache.v)
    args = (cache.k, cache.v, cache.k_scale, cache.v_scale, table, lengths, n, path)
    if _lib.direct_call(*args):
        _native_keep(*args, T, cache.d_head)
        _changed(cache)
    else:
        cache_keep_op(*args, T, cache.d_head)


# ------------------------------------------------------------------ attention

@lru_cache(maxsize=512)
def _workspace(shape, max_pages, d, fmt, dtype, B, T, Hq, window, n_persistent) -> int:
    n, h, page, pitch = shape
    fake = 256  # sizes only: nothing is read there
    arg = CacheArg(fake, fake, fake, fake, fake, fake, None, n, max_pages, h, page, pitch, d, max_pages, fmt, dtype)
    nb = ctypes.c_size_t(0)
    _lib.check(_lib.lib().tmac_cached_attn_workspace(ctypes.byref(arg), B, T, Hq, window, n_persistent, ctypes.byref(nb)),
               "tmac_cached_attn_workspace")
    return nb.value


def _native_attn(q, k, v, ks, vs, table, lengths, counts, tree, window, n_persistent, scale, d):
    """[B, T, Hq, d]."""
    dev = _lib.require_device(*(t for t in (q, k, v, ks, vs, table, lengths, counts, tree) if t is not None),
                              what="cached_attention")
    B, H, T, _ = q.shape
    out = torch.empty((B, T, H, d), dtype=q.dtype, device=dev)
    if out.numel() == 0:
        return out
    q, table, lengths, counts = _unit(q), _table(table), _flat(lengths), _flat(counts)
    arg = _arg(k, v, ks, vs, table, lengths, counts, d, q.dtype)
    if tree is None:
        tree_stride = 0
    else:
        tree = _unit(tree)
        tree_stride = 0 if tree.dim() == 1 else _pitch(tree)
        if tree.dim() == 2 and tree_stride < T and tree_stride != 0:
            tree, tree_stride = tree.contiguous(), T
    nb = _workspace(tuple(k.shape), table.shape[1], d, arg.format, arg.dtype, B, T, H, window, n_persistent)
    ws = torch.empty(nb, dtype=torch.uint8, device=dev) if nb else None
    with _lib.device_guard(dev):
        rc = _lib.lib().tmac_cached_attn(ctypes.byref(arg), q.data_ptr(), _strides(q), _lib.ptr(tree), tree_stride,
                                         out.data_ptr(), _lib.ptr(ws), nb, B, T, H, window, n_persistent, scale,
                                         _lib.stream_ptr(dev))
    _lib.check(rc, "tmac_cached_attn")
    return out


@torch.library.custom_op("titanmac::cached_attention", mutates_args=())
def cached_attention_op(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, ks: Optional[torch.Tensor],
                        vs: Optional[torch.Tensor], table: torch.Tensor, lengths: torch.Tensor,
                        counts: Optional[torch.Tensor], tree: Optional[torch.Tensor], window: int, n_persistent: int,
                        scale: float, d: int) -> torch.Tensor:
    return _native_attn(q, k, v, ks, vs, table, lengths, counts, tree, window, n_persistent, scale, d)


@cached_attention_op.register_fake
def _(q, k, v, ks, vs, table, lengths, counts, tree, window, n_persistent, scale, d):
    B, H, T, _ = q.shape
    return q.new_empty((B, T, H, d))


def cached_attention(q: torch.Tensor, cache: KVCache, table: torch.Tensor, lengths: torch.Tensor,
                     window_size: Optional[int] = None, n_persistent: int = 0, *,
                     counts: Optional[torch.Tensor] = None, tree: Optional[torch.Tensor] = None,
                     scale: Optional[float] = None) -> torch.Tensor:
    """softmax(q·kᵀ·scale)·v of the new rows q [B, H, T, d_head] (any strides) over the cache, which already holds their
    keys and values: [B, H, T, d_head]. H is a multiple of the cache's heads; query head h reads head h / (H / heads).

    The row at position p sees position j as in ``windowed_attention`` (causal): a persistent row (p < n_persistent) the
    persistent ones, any other j < n_persistent or p − window_size ≤ j ≤ p (None: no window).

    tree: int64 [B, T] or [T], T up to 64, makes the new rows a draft behind the ``base = length − count`` positions that are
    held: bit s of row t's entry says that row t sees drafted row s (itself included, its ancestors for a tree). A
    drafted row's place for the window is base + the number of its bits − 1; it sees the held positions as above and
    its drafted rows inside its window. A row that sees nothing, and rows t ≥ count, give zeros.

    What a row does not see never reaches its result, whatever is stored there. Scores, sums and the accumulation are in
    fp32; in 16 bit the probabilities are rounded to q's type before they meet the values. scale defaults to
    1/sqrt(d_head). No gradient."""
    what = "cached_attention"
    if q.dim() != 4:
        raise ValueError(f"{what}: q must be [B, H, T, d_head], got {tuple(q.shape)}")
    B, H, T, d = q.shape
    _check_cache(what, cache, table, lengths, counts, q.dtype, T, B)
    heads = cache.k.shape[1]
    if d != cache.d_head or H == 0 or H % heads:
        raise ValueError(f"{what}: the cache has {heads} heads of {cache.d_head}, q is {tuple(q.shape)}")
    if B * H * T > 1 << 26:
        raise ValueError(f"{what}: up to 2^26 query rows, got {B * H * T}")
    window = _NO_WINDOW if window_size is None else min(int(window_size), _NO_WINDOW)
    n_persistent = int(n_persistent)
    if window < 0 or n_persistent < 0:
        raise ValueError(f"{what}: window_size and n_persistent must not be negative, got {window_size}, {n_persistent}")
    if tree is not None:
        if tree.dtype != torch.int64 or tuple(tree.shape) not in ((B, T), (T,)):
            raise ValueError(f"{what}: tree must be int64 [{B}, {T}] or [{T}], got {tree.dtype} {tuple(tree.shape)}")
        if T > MAX_TREE:
            raise ValueError(f"{what}: a draft has up to {MAX_TREE} rows, got {T}")
    _no_grad(what, q, cache.k, cache.v)
    tensors = (q, cache.k, cache.v, cache.k_scale, cache.v_scale, table, lengths, counts, tree)
    run = _native_attn if _lib.direct_call(*tensors) else cached_attention_op
    out = run(*tensors, window, min(n_persistent, _NO_WINDOW), float(d ** -0.5 if scale is None else scale), d)
    return out.transpose(1, 2)
