"""Token embedding in front of the blocks (HIP kernels for gfx950).

The model looks its tokens up, adds the rows of their positions and puts the persistent tokens in front
(models/titanmac.py:183-190):

    out[b, p]      = prefix[p]                                     p < Np
    out[b, Np + t] = scale * weight[ids[b, t]] + pos_weight[position(b, t)]

``token_embedding`` does that in one launch. Its gradients are dense, as ``nn.Embedding``'s: the tokens are
sorted by id (where the table needs a gradient, in the lookup's launch) and each row's sum is formed in a fixed
order (deterministic, fp32) and written once.
"""
from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import Optional

import torch

from . import _lib
from .norm import _rows

_INDEX = (torch.int64, torch.int32)
_MAX_ROWS, _MAX_D = 1 << 30, 1 << 20  # of the result and of a table; of a row


def _table(t: Optional[torch.Tensor]):
    """(a table whose rows the kernels can read, copied only if they cannot be; its row pitch)."""
    if t is None:
        return t, 0
    n, d = t.shape
    pitch, step = t.stride()
    if (step != 1 and d > 1) or (pitch < d and n > 1):
        return t.contiguous(), d
    return t, max(pitch, d)


def _check(ids, weight, pos_weight, positions, prefix) -> None:
    if ids.dim() != 2:
        raise ValueError(f"token_embedding: ids must be [B, T], got {tuple(ids.shape)}")
    if weight.dim() != 2 or weight.shape[0] == 0 or weight.shape[1] == 0:
        raise ValueError(f"token_embedding: weight must be [V, d], got {tuple(weight.shape)}")
    for name, t in (("ids", ids), ("positions", positions)):
        if t is not None and t.dtype not in _INDEX:
            raise TypeError(f"token_embedding: {name} must be int64 or int32, got {t.dtype}")
    for name, t in (("pos_weight", pos_weight), ("prefix", prefix)):
        if t is None:
            continue
        if t.dim() != 2 or t.shape[1] != weight.shape[1]:
            raise ValueError(f"token_embedding: {name} must be [n, {weight.shape[1]}], got {tuple(t.shape)}")
        if t.dtype != weight.dtype:
            raise TypeError(f"token_embedding: {name} dtype {t.dtype} != weight dtype {weight.dtype}")
    if positions is not None:
        if pos_weight is None:
            raise ValueError("token_embedding: positions need pos_weight")
        if tuple(positions.shape) not in (tuple(ids.shape), (ids.shape[1],)):
            raise ValueError(f"token_embedding: positions must be {tuple(ids.shape)} or ({ids.shape[1]},), got "
                             f"{tuple(positions.shape)}")
    if pos_weight is not None:
        if pos_weight.shape[0] == 0:
            raise ValueError("token_embedding: pos_weight has no rows")
        if positions is None and ids.shape[1] > pos_weight.shape[0]:
            raise ValueError(f"token_embedding: {ids.shape[1]} positions, but pos_weight has "
                             f"{pos_weight.shape[0]} rows")
    n_prefix = 0 if prefix is None else prefix.shape[0]
    rows = ids.shape[0] * (ids.shape[1] + n_prefix)
    if (max(rows, weight.shape[0], 0 if pos_weight is None else pos_weight.shape[0], n_prefix) > _MAX_ROWS
            or max(ids.shape) > _MAX_ROWS or weight.shape[1] > _MAX_D):
        raise ValueError(f"token_embedding: up to {_MAX_ROWS} rows of up to {_MAX_D} values")


def _index(t: Optional[torch.Tensor], like: torch.Tensor) -> Optional[torch.Tensor]:
    if t is None or t.dtype == torch.int64 and t.shape == like.shape and t.is_contiguous():
        return t
    return t.expand(like.shape).to(torch.int64).contiguous()


def _lists_bytes(n_tokens: int, V: int) -> int:
    """tmac_embed_lists_bytes (in Python, for sizes that are symbols)."""
    return (4 * V + 19) // 16 * 16 + 2 * ((4 * n_tokens + 15) // 16 * 16)


def _native_fwd(ids, weight, pos_weight, positions, prefix, scale, make_lists):
    """([B, Np + T, d] in weight's dtype, the tokens of each row of weight as the backward reads them or None)."""
    _check(ids, weight, pos_weight, positions, prefix)
    code = _lib.dtype_code(weight.dtype)
    dev = _lib.require_device(*(t for t in (weight, ids, pos_weight, positions, prefix) if t is not None),
                              what="token_embedding")
    (B, T), (V, d) = ids.shape, weight.shape
    n_prefix = 0 if prefix is None else prefix.shape[0]
    out = torch.empty((B, n_prefix + T, d), dtype=weight.dtype, device=dev)
    nb = _lists_bytes(B * T, V) if make_lists else 0
    lists = torch.empty(nb, dtype=torch.uint8, device=dev) if make_lists else None
    if out.numel() == 0 and not make_lists:
        return out, lists
    i, q = _index(ids, ids), _index(positions, ids)
    (w, ldw), (p, ldp), (f, ldf) = _table(weight), _table(pos_weight), _table(prefix)
    with _lib.device_guard(dev):
        rc = _lib.lib().tmac_embed_fwd(i.data_ptr(), _lib.ptr(q), w.data_ptr(), ldw, _lib.ptr(p), ldp, _lib.ptr(f), ldf,
                                       out.data_ptr(), _lib.ptr(lists), nb, B, T, n_prefix, d, V,
                                       0 if p is None else p.shape[0], scale, code, _lib.stream_ptr(dev))
    _lib.check(rc, "tmac_embed_fwd")
    return out, lists


def _token_embedding(ids: torch.Tensor, weight: torch.Tensor, pos_weight: Optional[torch.Tensor],
                     positions: Optional[torch.Tensor], prefix: Optional[torch.Tensor], scale: float,
                     make_lists: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """_native_fwd; an operator's results are tensors: empty lists for None."""
    out, lists = _native_fwd(ids, weight, pos_weight, positions, prefix, scale, make_lists)
    return out, out.new_empty(0, dtype=torch.uint8) if lists is None else lists


token_embedding_fwd = torch.library.custom_op("titanmac::token_embedding", mutates_args=())(_token_embedding)


@token_embedding_fwd.register_fake
def _(ids, weight, pos_weight, positions, prefix, scale, make_lists):
    n_prefix, (B, T) = 0 if prefix is None else prefix.shape[0], ids.shape
    nb = _lists_bytes(B * T, weight.shape[0]) if make_lists else 0
    return weight.new_empty((B, n_prefix + T, weight.shape[1])), weight.new_empty((nb,), dtype=torch.uint8)


@lru_cache(maxsize=256)
def _workspace(n_tokens: int, V: int, n_pos: int, d: int, need_w: bool) -> int:
    if not need_w and n_pos == 0:
        return 0
    nb = ctypes.c_size_t(0)
    _lib.check(_lib.lib().tmac_embed_bwd_workspace(n_tokens, V, n_pos, d, ctypes.byref(nb)), "tmac_embed_bwd_workspace")
    return nb.value


def _native_bwd(grad, ids, positions, lists, n_prefix, V, n_pos, scale, need_w, need_p, need_f):
    """Gradients of weight [V, d], pos_weight [n_pos, d] and prefix [n_prefix, d] in grad's dtype, None where not
    needed."""
    (B, T), d, dtype, dev = ids.shape, grad.shape[-1], grad.dtype, grad.device
    if grad.is_contiguous():
        g, ldg = grad, d
    else:
        g = _rows(grad)
        ldg = max(g.stride(0), d)
    dw = torch.empty((V, d), dtype=dtype, device=dev) if need_w else None
    dp = torch.empty((n_pos, d), dtype=dtype, device=dev) if need_p else None
    df = torch.empty((n_prefix, d), dtype=dtype, device=dev) if need_f else None
    i = _index(ids, ids) if need_w and lists is None else None
    q = _index(positions, ids) if need_p else None
    nb = _workspace(B * T, V if i is not None else 0, n_pos if q is not None else 0, d, need_w)
    ws = torch.empty(nb, dtype=torch.uint8, device=dev) if nb else None
    ptr = _lib.ptr
    with _lib.device_guard(dev):
        rc = _lib.lib().tmac_embed_bwd(ptr(i), ptr(q), ptr(lists), g.data_ptr(), ldg, ptr(dw), ptr(dp),
                                       ptr(df) if n_prefix else 0, ptr(ws), nb, B, T, n_prefix, d, V, n_pos, scale,
                                       _lib.dtype_code(dtype), _lib.stream_ptr(dev))
    _lib.check(rc, "tmac_embed_bwd")
    return dw, dp, df


def _token_embedding_bwd(grad: torch.Tensor, ids: torch.Tensor, positions: Optional[torch.Tensor],
                         lists: Optional[torch.Tensor], n_prefix: int, V: int, n_pos: int, scale: float,
                         need_w: bool, need_p: bool, need_f: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """_native_bwd; an operator's results are tensors: empty ones for None."""
    _lib.require_device(*(t for t in (grad, ids, positions, lists) if t is not None), what="token_embedding backward")
    out = _native_bwd(grad, ids, positions, lists, n_prefix, V, n_pos, scale, need_w, need_p, need_f)
    return tuple(grad.new_empty((0, grad.shape[-1])) if t is None else t for t in out)


token_embedding_bwd = torch.library.custom_op("titanmac::token_embedding_bwd",
                                              mutates_args=())(_token_embedding_bwd)


@token_embedding_bwd.register_fake
def _(grad, ids, positions, lists, n_prefix, V, n_pos, scale, need_w, need_p, need_f):
    d = grad.shape[-1]
    return tuple(grad.new_empty((n if need else 0, d))
                 for n, need in ((V, need_w), (n_pos, need_p), (n_prefix, need_f)))


def _setup(ctx, inputs, output):
    ids, weight, pos_weight, positions, prefix, scale, make_lists = inputs
    ctx.save_for_backward(ids, positions, output[1] if make_lists else None)
    ctx.sizes = (0 if prefix is None else prefix.shape[0], weight.shape[0],
                 0 if pos_weight is None else pos_weight.shape[0], scale)


def _composed(grad, ids, positions, lists, n_prefix, V, n_pos, scale, need_w, need_p, need_f):
    """The gradients in torch's operations, for a backward that is itself differentiated."""
    g = grad[:, n_prefix:].float()

    def scatter(index, n, factor):
        ok = (index >= 0) & (index < n)
        rows = torch.where(ok.unsqueeze(-1), g, 0.0).reshape(-1, g.shape[-1]) * factor
        out = torch.zeros((n, g.shape[-1]), dtype=torch.float32, device=g.device)
        return out.index_add(0, torch.where(ok, index, 0).reshape(-1).long(), rows).to(grad.dtype)

    if positions is None:
        positions = torch.arange(ids.shape[1], device=ids.device)
    return (scatter(ids, V, scale) if need_w else None,
            scatter(positions.expand(ids.shape), n_pos, 1.0) if need_p else None,
            grad[:, :n_prefix].float().sum(0).to(grad.dtype) if need_f else None)


def _backward(ctx, grad, *_):
    ids, positions, lists = ctx.saved_tensors
    _, need_w, need_p, _, need_f, _, _ = ctx.needs_input_grad
    if torch.is_grad_enabled() and grad.requires_grad:
        run = _composed
    elif _lib.direct_backward(grad, ids):
        run = _native_bwd
    else:
        run = token_embedding_bwd
    dw, dp, df = run(grad, ids, positions, lists, *ctx.sizes, need_w, need_p, need_f)
    return None, dw if need_w else None, dp if need_p else None, None, df if need_f else None, None, None


token_embedding_fwd.register_autograd(_backward, setup_context=_setup)
_native = _lib.native_function(_native_fwd, _setup, _backward)


def token_embedding(ids: torch.Tensor, weight: torch.Tensor, pos_weight: Optional[torch.Tensor] = None, *,
                    positions: Optional[torch.Tensor] = None, prefix: Optional[torch.Tensor] = None,
                    scale: float = 1.0) -> torch.Tensor:
    """scale * weight[ids] + pos_weight[positions], behind the rows of prefix: [B, Np + T, d].

    ids: int64 or int32 [B, T]; weight [V, d], pos_weight [n_pos, d] and prefix [Np, d] of one dtype
    (float32, bfloat16, float16), d up to 2^20, up to 2^30 rows. positions: [B, T] or [T], by default
    0 .. T - 1. The sum is formed in fp32 and rounded once. Nothing is copied to the host to look at the ids:
    one outside [0, V), or a position outside its table, gives a row of NaN and adds nothing to the gradient of the
    table that it is outside of (the other table's takes the row's gradient as any).

    Differentiable in the three tables (a second time too)."""
    tables = (ids, weight, pos_weight, positions, prefix)
    # a training step's lists of tokens are made beside the lookup
    args = (*tables, float(scale), torch.is_grad_enabled() and weight.requires_grad)
    if _lib.direct_call(*tables):
        return _native_fwd(*args)[0]
    if _lib.eager_native(*tables):
        return _native(*args)
    return token_embedding_fwd(*args)[0]
