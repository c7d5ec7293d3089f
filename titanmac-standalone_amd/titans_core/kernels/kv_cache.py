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
import struct
from functools import lru_cache
from operator import itemgetter
from typing import Optional, Union

import torch

from . import _lib

SAME, INT8, E4M3 = 0, 1, 2
_FORMATS = {torch.int8: INT8, torch.float8_e4m3fn: E4M3}
_NAMES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
PAGES = (16, 32, 64, 128, 256)
MAX_HEAD, MAX_TREE = 128, 64
_NO_WINDOW = 1 << 30

# tmac_cache as bytes (a ctypes.Structure takes 2 us more to fill, as much as such a call's launch), and strides
_CACHE_ARG = struct.Struct("7Q2q7i4x").pack
_STRIDES = struct.Struct("3q").pack
_DTYPE = _lib._DTYPE_CODE


class KVCache(tuple):
    """Pools of keys and values: ``k``, ``v`` [n_pages, n_heads, page, pitch], contiguous, rows of d_head values behind
    which are zeros up to the pitch (d_head rounded up to 16); page 16, 32, 64, 128 or 256, d_head up to 128. Their
    type is the model's (float32, bfloat16, float16), or int8 or float8_e4m3fn with a scale for each row in ``k_scale``,
    ``v_scale`` (float32 [n_pages, n_heads, page]): a value is code · scale. ``KVCache.new`` makes them.

    Immutable, and checked here once: the tensors' contents change, they themselves are not to be resized or replaced
    (a change of device makes another KVCache)."""

    __slots__ = ()
    k, v, k_scale, v_scale, d_head = (property(itemgetter(i)) for i in range(5))

    def __new__(cls, k: torch.Tensor, v: torch.Tensor, d_head: Optional[int] = None,
                k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None):
        shape, dtype = k.shape, k.dtype
        if len(shape) != 4 or v.shape != shape or v.dtype != dtype:
            raise ValueError(f"KVCache: the pools must be [n_pages, n_heads, page, pitch], alike, got {tuple(shape)} {dtype} "
                             f"and {tuple(v.shape)} {v.dtype}")
        n, heads, page, pitch = shape
        d = pitch if d_head is None else int(d_head)
        if page not in PAGES or not 1 <= d <= MAX_HEAD or pitch != (d + 15) // 16 * 16 or n < 1 or heads < 1:
            raise ValueError(f"KVCache: pages of {PAGES} rows of d_head (1..{MAX_HEAD}) rounded up to 16 values, got "
                             f"{tuple(shape)} for d_head {d}")
        if heads * page * pitch >= 1 << 29 or n >= 1 << 31 or n * heads * page >= 1 << 40:
            raise ValueError(f"KVCache: a page has fewer than 2^29 values, pools fewer than 2^31 pages and 2^40 rows, got "
                             f"{tuple(shape)}")
        if not (k.is_contiguous() and v.is_contiguous()):
            raise ValueError("KVCache: the pools must be contiguous")
        device = k.device
        if v.device != device:
            raise RuntimeError(f"KVCache: tensors on different devices ({device} and {v.device})")
        fmt = _FORMATS.get(dtype, SAME)
        if fmt != SAME:
            for s in (k_scale, v_scale):
                if s is None or s.dtype != torch.float32 or s.shape != shape[:3] or not s.is_contiguous():
                    raise ValueError(f"KVCache: pools of {dtype} need k_scale and v_scale, float32 {tuple(shape[:3])}, "
                                     "contiguous")
                if s.device != device:
                    raise RuntimeError(f"KVCache: tensors on different devices ({device} and {s.device})")
            changing = (k, v, k_scale, v_scale)
        else:
            if dtype not in _DTYPE:
                raise TypeError(f"KVCache: unsupported dtype {dtype}; expected float32, bfloat16, float16, int8 or "
                                "float8_e4m3fn")
            k_scale = v_scale = None
            changing = (k, v)
        return tuple.__new__(cls, (k, v, k_scale, v_scale, d, fmt, heads, shape, device, changing,
                                   dtype if fmt == SAME else None, (1 << 30) // page,
                                   tuple(t for t in changing if not t.is_inference())))  # those have no version

    def __getnewargs__(self):
        return self.k, self.v, self.d_head, self.k_scale, self.v_scale

    def __repr__(self):
        n, heads, page, _ = self.k.shape
        return (f"KVCache({n} pages of {page}, {heads} heads of {self.d_head}, {self.k.dtype}, {self.k.device})")

    @classmethod
    def new(cls, n_pages: int, n_heads: int, d_head: int, *, page: int = 64, dtype: torch.dtype = torch.bfloat16,
            fmt: Optional[str] = None, device="cuda") -> "KVCache":
        """An empty cache (zeros) of values of dtype, held as they are or as fmt "int8" or "e4m3"."""
        if fmt is not None and fmt not in _NAMES:
            raise ValueError(f"KVCache: fmt must be None, 'int8' or 'e4m3', got {fmt!r}")
        if dtype not in _DTYPE:
            raise TypeError(f"KVCache: dtype must be float32, bfloat16 or float16, got {dtype}")
        if page not in PAGES or not 1 <= d_head <= MAX_HEAD or n_pages < 1 or n_heads < 1:
            raise ValueError(f"KVCache: page must be one of {PAGES} and d_head 1..{MAX_HEAD}, got {page}, {d_head} "
                             f"({n_pages} pages, {n_heads} heads)")
        shape = (n_pages, n_heads, page, -(-d_head // 16) * 16)
        store = dtype if fmt is None else _NAMES[fmt]
        scale = lambda: None if fmt is None else torch.zeros(shape[:3], dtype=torch.float32, device=device)  # noqa: E731
        return cls(torch.zeros(shape, dtype=store, device=device), torch.zeros(shape, dtype=store, device=device),
                   d_head, scale(), scale())


def _sequences(what: str, cache: KVCache, table, lengths, counts, dtype: torch.dtype, T: int, B: int):
    """(table, its pitch, lengths, counts) as the kernels read them, of sequences whose description is in order and whose
    values the cache holds."""
    held, i32 = cache[10], torch.int32
    if held is not dtype and (held is not None or dtype not in _DTYPE):
        if dtype not in _DTYPE:
            raise TypeError(f"{what}: unsupported dtype {dtype}; expected float32, bfloat16 or float16")
        raise TypeError(f"{what}: a cache of {held} does not hold {dtype}")
    if not (table.dtype is i32 and lengths.dtype is i32 and (counts is None or counts.dtype is i32)):
        raise TypeError(f"{what}: table, lengths and counts must be int32")
    at, n = table.shape, lengths.shape
    if len(at) != 2 or at[0] != B or at[1] == 0:
        raise ValueError(f"{what}: table must be [{B}, pages], got {tuple(at)}")
    if len(n) != 1 or n[0] != B:
        raise ValueError(f"{what}: lengths must be [{B}], got {tuple(n)}")
    if counts is not None:
        if counts.shape != n:
            raise ValueError(f"{what}: counts must be [{B}], got {tuple(counts.shape)}")
        if not counts.is_contiguous():
            counts = counts.contiguous()
    if B > 1 << 20 or T * cache[6] > 1 << 26 or at[1] > cache[11]:
        raise ValueError(f"{what}: up to 2^20 sequences, 2^26 rows of one and 2^30 positions")
    if not lengths.is_contiguous():
        lengths = lengths.contiguous()
    pitch, step = table.stride()
    if step != 1 or pitch < at[1]:
        table, pitch = _rows(table)
    return table, pitch, lengths, counts


def _refuse_grad(what: str, *tensors) -> None:
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise NotImplementedError(f"{what} has no gradient: call it under torch.no_grad()")


def _rows(t: torch.Tensor):
    """(a table [B, n] that the kernels can read, its pitch; any where there is one row)."""
    n = t.shape[1]
    pitch, step = t.stride()
    if (step != 1 and n != 1) or (pitch < n and t.shape[0] > 1):
        return t.contiguous(), n
    return t, pitch if t.shape[0] > 1 else n


def _run(what: str, device: torch.device, tensors, name: str, *args) -> None:
    """The library's function on the current stream of the device of all of the tensors."""
    if device.type != "cuda":
        _lib.require_device(*(t for t in tensors if t is not None), what=what)
        index, now = None, None  # on the CPU the library's calls are replaced
    else:
        for t in tensors:
            if t is not None and t.device != device:
                raise RuntimeError(f"{what}: tensors on different devices ({device} and {t.device})")
        index, now = device.index, torch._C._cuda_getDevice()
    fn = getattr(_lib.lib(), name)
    if index == now:
        rc = fn(*args, _lib.stream_ptr(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _lib.stream_ptr(device))
    if rc != 0:
        _lib.check(rc, name)


def _arg(cache: KVCache, table, pitch: int, lengths, counts, dtype: torch.dtype) -> bytes:
    """tmac_cache."""
    k, v, ks, vs, d, fmt, heads, shape = cache[:8]
    return _CACHE_ARG(k.data_ptr(), v.data_ptr(), 0 if ks is None else ks.data_ptr(), 0 if vs is None else vs.data_ptr(),
                      table.data_ptr(), lengths.data_ptr(), 0 if counts is None else counts.data_ptr(), shape[0], pitch,
                      heads, shape[2], shape[3], d, table.shape[1], fmt, _DTYPE[dtype])


def _changed(cache: KVCache) -> None:
    """What autograd (or a caller's own cache) keeps of the pools is out of date."""
    torch.autograd.graph.increment_version(cache[12])


# ------------------------------------------------------------------ write

def _native_write(k, v, cache, table, pitch, lengths, counts) -> None:
    B, _, T, d = k.shape
    if B * T == 0:
        return
    at_k, at_v = k.stride(), v.stride()
    if (at_k[3] != 1 or at_v[3] != 1) and d > 1:
        k, v = k.contiguous(), v.contiguous()
        at_k, at_v = k.stride(), v.stride()
    _run("cache_write", cache[8], (k, v, table, lengths, counts), "tmac_cache_write",
         _arg(cache, table, pitch, lengths, counts, k.dtype), k.data_ptr(), _STRIDES(*at_k[:3]), v.data_ptr(),
         _STRIDES(*at_v[:3]), B, T)


@torch.library.custom_op("titanmac::cache_write", mutates_args=("k", "v", "ks", "vs"))
def cache_write_op(new_k: torch.Tensor, new_v: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                   ks: Optional[torch.Tensor], vs: Optional[torch.Tensor], table: torch.Tensor, lengths: torch.Tensor,
                   counts: Optional[torch.Tensor], d: int) -> None:
    cache = KVCache(k, v, d, ks, vs)
    _native_write(new_k, new_v, cache, *_sequences("cache_write", cache, table, lengths, counts, new_k.dtype,
                                                   new_k.shape[2], new_k.shape[0]))


@cache_write_op.register_fake
def _(new_k, new_v, k, v, ks, vs, table, lengths, counts, d):
    return None


def cache_write(k: torch.Tensor, v: torch.Tensor, cache: KVCache, table: torch.Tensor, lengths: torch.Tensor, *,
                counts: Optional[torch.Tensor] = None) -> None:
    """The new rows k, v [B, n_heads, T, d_head] (any strides) into the cache, in place.

    In 8 bits every row has its own scale: int8 codes are value / scale rounded to nearest (ties to even) with scale =
    max |value| / 127, e4m3 codes likewise with the least power of two that holds the row as scale (both at least
    2^-126). A row that is not finite is held as NaN. Pages that are written must not belong to two sequences, and k and v
    must not share memory with the pools."""
    shape, dtype = k.shape, k.dtype
    if len(shape) != 4 or v.shape != shape or v.dtype is not dtype:
        raise ValueError(f"cache_write: k and v must be [B, n_heads, T, d_head], alike, got {tuple(shape)} {dtype} and "
                         f"{tuple(v.shape)} {v.dtype}")
    B, H, T, d = shape
    table, pitch, lengths, counts = _sequences("cache_write", cache, table, lengths, counts, dtype, T, B)
    if H != cache[6] or d != cache[4]:
        raise ValueError(f"cache_write: the cache has {cache[6]} heads of {cache[4]}, k is {tuple(shape)}")
    if _lib.direct_call(k, v, table, lengths, counts, *cache[9]):
        _native_write(k, v, cache, table, pitch, lengths, counts)
        _changed(cache)
    else:
        _refuse_grad("cache_write", k, v, cache[0], cache[1])
        cache_write_op(k, v, *cache[:4], table, lengths, counts, cache[4])


# ------------------------------------------------------------------ read

def _native_read(cache, table, pitch, lengths, T, dtype):
    B, H, d, device = lengths.shape[0], cache[6], cache[4], cache[8]
    k = torch.empty((B, H, T, d), dtype=dtype, device=device)
    v = torch.empty((B, H, T, d), dtype=dtype, device=device)
    if B * T:
        _run("cache_read", device, (table, lengths), "tmac_cache_read", _arg(cache, table, pitch, lengths, None, dtype),
             k.data_ptr(), v.data_ptr(), B, T)
    return k, v


@torch.library.custom_op("titanmac::cache_read", mutates_args=())
def cache_read_op(k: torch.Tensor, v: torch.Tensor, ks: Optional[torch.Tensor], vs: Optional[torch.Tensor],
                  table: torch.Tensor, lengths: torch.Tensor, T: int, d: int,
                  dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
    cache = KVCache(k, v, d, ks, vs)
    table, pitch, lengths, _ = _sequences("cache_read", cache, table, lengths, None, dtype, T, lengths.shape[0])
    return _native_read(cache, table, pitch, lengths, T, dtype)


@cache_read_op.register_fake
def _(k, v, ks, vs, table, lengths, T, d, dtype):
    return tuple(k.new_empty((table.shape[0], k.shape[1], T, d), dtype=dtype) for _ in range(2))


def cache_read(cache: KVCache, table: torch.Tensor, lengths: torch.Tensor, n_positions: int, *,
               dtype: Optional[torch.dtype] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Positions 0 .. n_positions − 1 of every sequence as k, v [B, n_heads, n_positions, d_head]: zeros behind a
    sequence's length. dtype: the values' type (default: the cache's, bfloat16 for one in 8 bits). A value that e4m3 rounded
    up to more than dtype holds (one of 63488 or more in float16) is infinite."""
    if dtype is None:
        dtype = cache[10] or torch.bfloat16
    T = int(n_positions)
    if T < 0:
        raise ValueError(f"cache_read: n_positions must not be negative, got {T}")
    table, pitch, lengths, _ = _sequences("cache_read", cache, table, lengths, None, dtype, T,
                                          lengths.shape[0] if lengths.dim() == 1 else -1)
    if _lib.direct_call(table, lengths, *cache[9]):
        return _native_read(cache, table, pitch, lengths, T, dtype)
    _refuse_grad("cache_read", cache[0], cache[1])
    return cache_read_op(*cache[:4], table, lengths, T, cache[4], dtype)


# ------------------------------------------------------------------ keep

def _native_keep(cache, table, pitch, lengths, counts, path, T) -> None:
    B, A = path.shape
    if B == 0 or A == 0:
        return
    path_pitch, step = path.stride()
    if step != 1 or path_pitch < A:
        path, path_pitch = _rows(path)
    # 8-bit rows are moved as they are, whatever the type of the values
    _run("cache_keep", cache[8], (table, lengths, counts, path), "tmac_cache_keep",
         _arg(cache, table, pitch, lengths, counts, cache[10] or torch.bfloat16), path.data_ptr(), path_pitch, A, B, T)


@torch.library.custom_op("titanmac::cache_keep", mutates_args=("k", "v", "ks", "vs"))
def cache_keep_op(k: torch.Tensor, v: torch.Tensor, ks: Optional[torch.Tensor], vs: Optional[torch.Tensor],
                  table: torch.Tensor, lengths: torch.Tensor, counts: Optional[torch.Tensor], path: torch.Tensor, T: int,
                  d: int) -> None:
    cache = KVCache(k, v, d, ks, vs)
    _native_keep(cache, *_sequences("cache_keep", cache, table, lengths, counts, cache[10] or torch.bfloat16, T,
                                    path.shape[0]), path, T)


@cache_keep_op.register_fake
def _(k, v, ks, vs, table, lengths, counts, path, T, d):
    return None


def cache_keep(cache: KVCache, table: torch.Tensor, lengths: torch.Tensor, path: torch.Tensor,
               counts: Union[int, torch.Tensor]) -> None:
    """Of each sequence's draft, its last ``counts`` rows (up to 64; one number for all, or int32 [B]): row path[b, a]
    (int32 [B, A]) moves to place a of the draft, for all a at once. An entry outside the draft (−1) leaves its place as
    it is. The caller then shortens ``lengths`` to the rows that were kept."""
    n = counts if isinstance(counts, torch.Tensor) else None
    T = MAX_TREE if n is not None else int(counts)
    at = path.shape
    if len(at) != 2 or path.dtype is not torch.int32:
        raise ValueError(f"cache_keep: path must be int32 [B, rows], got {path.dtype} {tuple(path.shape)}")
    if not 0 <= T <= MAX_TREE or at[1] > T:
        raise ValueError(f"cache_keep: drafts of up to {MAX_TREE} rows, no more kept than drafted, got {T} and "
                         f"{path.shape[1]}")
    if at[0] > 32767:
        raise ValueError(f"cache_keep: up to 32767 sequences, got {at[0]}")
    table, pitch, lengths, n = _sequences("cache_keep", cache, table, lengths, n, cache[10] or torch.bfloat16, T, at[0])
    if _lib.direct_call(table, lengths, n, path, *cache[9]):
        _native_keep(cache, table, pitch, lengths, n, path, T)
        _changed(cache)
    else:
        _refuse_grad("cache_keep", cache[0], cache[1])
        cache_keep_op(*cache[:4], table, lengths, n, path, T, cache[4])


# ------------------------------------------------------------------ attention

@lru_cache(maxsize=512)
def _workspace(heads, page, d, max_pages, fmt, dtype, B, T, Hq, window, n_persistent) -> int:
    at = 256  # sizes only: nothing is read there
    arg = _CACHE_ARG(at, at, at, at, at, at, 0, 1, max_pages, heads, page, (d + 15) // 16 * 16, d, max_pages, fmt, dtype)
    nb = ctypes.c_size_t(0)
    _lib.check(_lib.lib().tmac_cached_attn_workspace(arg, B, T, Hq, window, n_persistent, ctypes.byref(nb)),
               "tmac_cached_attn_workspace")
    return nb.value


def _native_attn(q, cache, table, pitch, lengths, counts, tree, window, n_persistent, scale):
    """[B, H, T, d], a view of [B, T, H, d]."""
    B, H, T, d = q.shape
    dtype, device = q.dtype, cache[8]
    out = torch.empty_strided((B, H, T, d), (T * H * d, d, H * d, 1), dtype=dtype, device=device)
    if B * T == 0:
        return out
    at_q = q.stride()
    if at_q[3] != 1 and d > 1:
        q = q.contiguous()
        at_q = q.stride()
    tree_stride = tree_ptr = 0
    if tree is not None:
        if tree.dim() == 1:
            tree = tree.contiguous()
        else:
            tree_stride, step = tree.stride()
            if step != 1 or tree_stride < T:
                tree, tree_stride = _rows(tree)
        tree_ptr = tree.data_ptr()
    nb = _workspace(cache[6], cache[7][2], d, table.shape[1], cache[5], _DTYPE[dtype], B, T, H, window, n_persistent)
    ws = torch.empty(nb, dtype=torch.uint8, device=device) if nb else None
    _run("cached_attention", device, (q, table, lengths, counts, tree), "tmac_cached_attn",
         _arg(cache, table, pitch, lengths, counts, dtype), q.data_ptr(), _STRIDES(*at_q[:3]), tree_ptr, tree_stride,
         out.data_ptr(), 0 if ws is None else ws.data_ptr(), nb, B, T, H, window, n_persistent, scale)
    return out


@torch.library.custom_op("titanmac::cached_attention", mutates_args=())
def cached_attention_op(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, ks: Optional[torch.Tensor],
                        vs: Optional[torch.Tensor], table: torch.Tensor, lengths: torch.Tensor,
                        counts: Optional[torch.Tensor], tree: Optional[torch.Tensor], window: int, n_persistent: int,
                        scale: float, d: int) -> torch.Tensor:
    cache = KVCache(k, v, d, ks, vs)
    return _native_attn(q, cache, *_sequences("cached_attention", cache, table, lengths, counts, q.dtype, q.shape[2],
                                              q.shape[0]), tree, window, n_persistent, scale)


@cached_attention_op.register_fake
def _(q, k, v, ks, vs, table, lengths, counts, tree, window, n_persistent, scale, d):
    B, H, T, _ = q.shape
    return q.new_empty((B, T, H, d)).transpose(1, 2)


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
    fp32; in 16 bit the probabilities meet the values as two numbers of q's type (of bfloat16 for float16 on a cache in
    8 bits), which together keep 16 bits of them and more. scale defaults to 1/sqrt(d_head). No gradient."""
    shape = q.shape
    if len(shape) != 4:
        raise ValueError(f"cached_attention: q must be [B, H, T, d_head], got {tuple(shape)}")
    B, H, T, d = shape
    table, pitch, lengths, counts = _sequences("cached_attention", cache, table, lengths, counts, q.dtype, T, B)
    if d != cache[4] or H == 0 or H % cache[6]:
        raise ValueError(f"cached_attention: the cache has {cache[6]} heads of {cache[4]}, q is {tuple(q.shape)}")
    if B * H * T > 1 << 26:
        raise ValueError(f"cached_attention: up to 2^26 query rows, got {B * H * T}")
    window = _NO_WINDOW if window_size is None else min(int(window_size), _NO_WINDOW)
    n_persistent = min(int(n_persistent), _NO_WINDOW)
    if window < 0 or n_persistent < 0:
        raise ValueError(f"cached_attention: window_size and n_persistent must not be negative, got {window_size}, "
                         f"{n_persistent}")
    if tree is not None:
        if tree.dtype != torch.int64 or tuple(tree.shape) not in ((B, T), (T,)):
            raise ValueError(f"cached_attention: tree must be int64 [{B}, {T}] or [{T}], got {tree.dtype} "
                             f"{tuple(tree.shape)}")
        if T > MAX_TREE:
            raise ValueError(f"cached_attention: a draft has up to {MAX_TREE} rows, got {T}")
    scale = d ** -0.5 if scale is None else float(scale)
    if _lib.direct_call(q, table, lengths, counts, tree, *cache[9]):
        return _native_attn(q, cache, table, pitch, lengths, counts, tree, window, n_persistent, scale)
    _refuse_grad("cached_attention", q, cache[0], cache[1])
    return cached_attention_op(q, *cache[:4], table, lengths, counts, tree, window, n_persistent, scale, d)
