"""Log probabilities of given tokens (HIP kernels for gfx950).

The model's loss is the mean of -log softmax(logits)[target] over the tokens (models/titanmac.py:666-680),
a server wants the same number for each token, with the entropy of its distribution and the most probable
alternatives, and a policy update the gradients of both:

    lp = z[target] - lse(z),   H = -sum p ln p,   dz = g_lp (delta - p) - g_H p (ln p + H)

``token_logprobs`` reads the logits once, whatever is asked, and once more for their gradient;
``token_cross_entropy`` is the loss; ``head_logprobs`` scores hidden states without storing their logits.
All sums and results are fp32; gradients have their input's dtype.
"""
from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import NamedTuple, Optional

import torch
import torch.nn.functional as F

from . import _lib
from .linear import _HALF, _MAX_PITCH, _rows

MAX_TOP = 64
_MAX_ROWS, _MAX_V = 1 << 30, 1 << 28
_INDEX = (torch.int64, torch.int32)


class TokenLogprobs(NamedTuple):
    """What token_logprobs returns; None for what was not asked."""
    logprobs: torch.Tensor
    entropy: Optional[torch.Tensor] = None
    top_ids: Optional[torch.Tensor] = None
    top_logprobs: Optional[torch.Tensor] = None


def _check(logits: torch.Tensor, targets: torch.Tensor, what: str) -> None:
    if logits.dim() < 1 or logits.shape[-1] == 0:
        raise ValueError(f"{what}: logits must be [..., V], got {tuple(logits.shape)}")
    if targets.shape != logits.shape[:-1]:
        raise ValueError(f"{what}: targets must be {tuple(logits.shape[:-1])} for logits {tuple(logits.shape)}, got "
                         f"{tuple(targets.shape)}")
    if targets.dtype not in _INDEX:
        raise TypeError(f"{what}: targets must be int64 or int32, got {targets.dtype}")
    _check_sizes(targets, logits.shape[-1], what)


def _check_sizes(targets: torch.Tensor, V: int, what: str) -> None:
    if targets.numel() > _MAX_ROWS or max(targets.shape, default=0) > _MAX_ROWS or V > _MAX_V:
        raise ValueError(f"{what}: up to {_MAX_ROWS} rows of a vocabulary of up to {_MAX_V}, got {tuple(targets.shape)} "
                         f"of {V}")


def _rows3(z: torch.Tensor):
    """(z whose rows the kernels can read, stride of B, stride of T, B, T, V), rows seen as [B, T, V]: in place,
    copied only if their values are not neighbours or more than two strides lead to them."""
    V = z.shape[-1]
    if z.is_contiguous():
        return z, 0, V, 1, z.numel() // V, V
    z = z.unsqueeze(0).unsqueeze(0) if z.dim() == 1 else z.unsqueeze(0) if z.dim() == 2 else z
    if z.dim() > 3:
        z = z.reshape(1, -1, V)
    if V > 1 and z.stride(2) != 1:
        z = z.contiguous()
    return z, z.stride(0), z.stride(1), z.shape[0], z.shape[1], V


def _flat(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype == torch.int64 and t.is_contiguous() else t.to(torch.int64).contiguous()


@lru_cache(maxsize=256)
def _workspace(B: int, T: int, V: int, top_k: int, code: int) -> int:
    nb = ctypes.c_size_t(0)
    _lib.check(_lib.lib().tmac_logprob_workspace(B, T, V, top_k, code, ctypes.byref(nb)), "tmac_logprob_workspace")
    return nb.value


def _fwd(logits, targets, entropy, top_k, ignore_index, dev):
    """(logprobs, entropy, top_ids, top_logprobs, stats), None for what is not asked."""
    code = _lib.dtype_code(logits.dtype)
    z, sb, st, B, T, V = _rows3(logits)
    lead, n, f32 = targets.shape, B * T, torch.float32
    lp, stats = torch.empty(lead, dtype=f32, device=dev), torch.empty((n, 2), dtype=f32, device=dev)
    ent = torch.empty(lead, dtype=f32, device=dev) if entropy else None
    ids = torch.empty((*lead, top_k), dtype=torch.int64, device=dev) if top_k else None
    top = torch.empty((*lead, top_k), dtype=f32, device=dev) if top_k else None
    if n:
        nb, tg = _workspace(B, T, V, top_k, code), _flat(targets)
        ws = torch.empty(nb, dtype=torch.uint8, device=dev) if nb else None
        with _lib.device_guard(dev):
            rc = _lib.lib().tmac_logprob_fwd(z.data_ptr(), sb, st, tg.data_ptr(), ignore_index, lp.data_ptr(),
                                             _lib.ptr(ent), top_k, _lib.ptr(ids), _lib.ptr(top), stats.data_ptr(),
                                             _lib.ptr(ws), nb, B, T, V, code, _lib.stream_ptr(dev))
        _lib.check(rc, "tmac_logprob_fwd")
    return lp, ent, ids, top, stats


def _check_call(logits, targets, top_k):
    _check(logits, targets, "token_logprobs")
    _lib.dtype_code(logits.dtype)
    if not 0 <= top_k <= min(MAX_TOP, logits.shape[-1]):
        raise ValueError(f"token_logprobs: top_k must be in [0, {min(MAX_TOP, logits.shape[-1])}], got {top_k}")
    return _lib.require_device(logits, targets, what="token_logprobs")


def _logprob_fwd(logits: torch.Tensor, targets: torch.Tensor, entropy: bool, top_k: int, ignore_index: int
                 ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(logprobs, entropy, top_ids, top_logprobs, stats fp32 [rows, 2]); empty tensors for what is not asked."""
    dev = _check_call(logits, targets, top_k)
    out = _fwd(logits, targets, entropy, top_k, ignore_index, dev)
    # an operator's results are tensors
    return tuple(torch.empty((0,), dtype=torch.int64 if i == 2 else torch.float32, device=dev) if t is None else t
                 for i, t in enumerate(out))


logprob_fwd = torch.library.custom_op("titanmac::token_logprobs", mutates_args=())(_logprob_fwd)


@logprob_fwd.register_fake
def _(logits, targets, entropy, top_k, ignore_index):
    lead = logits.shape[:-1]
    n = 1
    for s in lead:
        n *= s
    f = lambda shape, dt=torch.float32: logits.new_empty(shape, dtype=dt)  # noqa: E731
    return (f(lead), f(lead if entropy else (0,)), f((*lead, top_k) if top_k else (0,), torch.int64),
            f((*lead, top_k) if top_k else (0,)), f((n, 2)))


def _row_grad(g: Optional[torch.Tensor]):
    """(fp32 values of a per-row gradient, stride): stride 0 for one value for all rows."""
    if g is None:
        return None, 0
    if g.dtype != torch.float32:
        g = g.to(torch.float32)
    if g.is_contiguous():
        return g, 1
    if all(s == 0 for s, n in zip(g.stride(), g.shape) if n > 1):
        return g, 0
    return g.contiguous(), 1


def _native_bwd(g_lp, g_ent, logits, targets, stats, entropy, ignore_index):
    """The gradient of the logits; g_lp, g_ent: per row, or one value for all."""
    z, sb, st, B, T, V = _rows3(logits)
    dz = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    if B * T == 0:
        return dz
    (gl, sl), (ge, se) = _row_grad(g_lp), _row_grad(g_ent)
    tg, ptr, dev = _flat(targets), _lib.ptr, logits.device
    with _lib.device_guard(dev):
        rc = _lib.lib().tmac_logprob_bwd(z.data_ptr(), sb, st, tg.data_ptr(), ignore_index, stats.data_ptr(),
                                         ptr(entropy), ptr(gl), sl, ptr(ge), se, dz.data_ptr(), B, T, V,
                                         _lib.dtype_code(z.dtype), _lib.stream_ptr(dev))
    _lib.check(rc, "tmac_logprob_bwd")
    return dz


def _logprob_bwd(g_lp: Optional[torch.Tensor], g_ent: Optional[torch.Tensor], logits: torch.Tensor,
                 targets: torch.Tensor, stats: torch.Tensor, entropy: Optional[torch.Tensor], ignore_index: int
                 ) -> torch.Tensor:
    _lib.require_device(*(t for t in (logits, targets, stats, entropy, g_lp, g_ent) if t is not None),
                        what="token_logprobs backward")
    return _native_bwd(g_lp, g_ent, logits, targets, stats, entropy, ignore_index)


logprob_bwd = torch.library.custom_op("titanmac::token_logprobs_bwd", mutates_args=())(_logprob_bwd)


@logprob_bwd.register_fake
def _(g_lp, g_ent, logits, targets, stats, entropy, ignore_index):
    return logits.new_empty(logits.shape)


def _composed(g_lp, g_ent, logits, targets, ignore_index):
    """The gradient in torch's operations, for a backward that is itself differentiated."""
    given = targets != ignore_index
    if g_ent is None:  # ignored rows are not read
        logits = torch.where(given.unsqueeze(-1), logits, 0.0)
    logp = torch.log_softmax(logits.float(), dim=-1)
    p = logp.exp()
    dz = torch.zeros_like(p)
    if g_lp is not None:
        outside = given & ((targets < 0) | (targets >= p.shape[-1]))  # lp is NaN
        g = torch.where(given, g_lp.float(), 0.0).masked_fill(outside, float("nan")).unsqueeze(-1)
        at = torch.arange(p.shape[-1], device=p.device) == targets.unsqueeze(-1)
        dz = dz + g * (at.to(p.dtype) - p)
    if g_ent is not None:
        some = torch.where(p > 0, logp, 0.0)
        H = -(p * some).sum(-1, keepdim=True)
        dz = dz - g_ent.float().unsqueeze(-1) * p * (some + H)
    return dz.to(logits.dtype)


def _gradient(g_lp, g_ent, logits, targets, stats, entropy, ignore_index):
    if g_lp is None and g_ent is None:
        return None
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (g_lp, g_ent, logits)):
        return _composed(g_lp, g_ent, logits, targets, ignore_index)
    direct = all(_lib.direct_backward(g, logits) for g in (g_lp, g_ent) if g is not None)
    run = _native_bwd if direct else logprob_bwd
    return run(g_lp, g_ent, logits, targets, stats, entropy, ignore_index)


def _setup(ctx, inputs, output):
    logits, targets, entropy, _top_k, ignore_index = inputs
    ctx.save_for_backward(logits, targets, output[4], output[1])
    ctx.with_entropy, ctx.ignore_index = entropy, ignore_index
    ctx.set_materialize_grads(False)


def _backward(ctx, g_lp, g_ent, _g_ids, _g_top, _g_stats):
    dz = _gradient(g_lp, g_ent if ctx.with_entropy else None, *ctx.saved_tensors, ctx.ignore_index)
    return dz, None, None, None, None


logprob_fwd.register_autograd(_backward, setup_context=_setup)


def _native_fwd(logits, targets, entropy, top_k, ignore_index):
    return _fwd(logits, targets, entropy, top_k, ignore_index, _check_call(logits, targets, top_k))


_native = _lib.native_function(_native_fwd, _setup, _backward, all_outputs=True)


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, *, entropy: bool = False, top_k: int = 0,
                   ignore_index: int = -100) -> TokenLogprobs:
    """Log probabilities of `targets` under softmax(logits), with what else is asked of each row.

    logits [..., V] (float32, bfloat16, float16; any strides, read in place where a row's values are
    neighbours), V up to 2^28 and up to 2^30 rows, targets int64 or int32 [...]. Results, fp32:

    - logprobs [...]: log softmax(logits)[target]; 0 where target == ignore_index, and NaN for any other
      target outside [0, V) (nothing is copied to the host to look at them);
    - entropy [...]: -sum p ln p in nats, of every row;
    - top_ids, top_logprobs [..., top_k] (top_k <= 64): the most probable tokens in order, equal logits by
      the lower index, of every row.

    -inf is probability 0. A row with a NaN or +inf, or nothing but -inf, has no distribution: its values are
    NaN and its top_ids -1. logprobs and entropy are differentiable (a second time too), top_logprobs is not."""
    args = (logits, targets, bool(entropy), int(top_k), int(ignore_index))
    if _lib.direct_call(logits, targets):
        return TokenLogprobs(*_fwd(*args, _check_call(logits, targets, args[3]))[:4])
    if _lib.eager_native(logits, targets):
        lp, ent, ids, top, _ = _native(*args)
    else:
        lp, ent, ids, top, _ = logprob_fwd(*args)
    return TokenLogprobs(lp, ent if entropy else None, ids if top_k else None, top.detach() if top_k else None)


# ------------------------------------------------------------------ the loss

def _loss_fwd(logits, targets, ignore_index, wide, memory):
    """(the mean of -lp over the given targets, in logits' dtype or (wide) fp32; what memory(rows, device) gave). That
    begins with the addresses of lp [rows], stats [rows, 2] and -1 / the targets' number, fp32, which are written."""
    _check(logits, targets, "token_cross_entropy")
    code = _lib.dtype_code(logits.dtype)
    dev = _lib.require_device(logits, targets, what="token_cross_entropy")
    z, sb, st, B, T, V = _rows3(logits)
    n, tg, L = B * T, _flat(targets), _lib.lib()
    loss = torch.empty((), dtype=torch.float32 if wide else logits.dtype, device=dev)
    lp, stats, inv, *kept = memory(n, dev)
    nb = _workspace(B, T, V, 0, code) if n else 0
    ws = torch.empty(nb, dtype=torch.uint8, device=dev) if nb else None
    with _lib.device_guard(dev):
        stream, at = _lib.stream_ptr(dev), tg.data_ptr()
        if n:
            rc = L.tmac_logprob_fwd(z.data_ptr(), sb, st, at, ignore_index, lp, 0, 0, 0, 0, stats, _lib.ptr(ws), nb, B, T,
                                    V, code, stream)
            _lib.check(rc, "tmac_logprob_fwd")
        rc = L.tmac_logprob_mean(lp, at, ignore_index, n, loss.data_ptr(), _lib.F32 if wide else code, inv, stream)
    _lib.check(rc, "tmac_logprob_mean")
    return loss, kept


def _apart(n, dev):
    lp, stats, inv = (torch.empty(s, dtype=torch.float32, device=dev) for s in (n, (n, 2), ()))
    return lp.data_ptr(), stats.data_ptr(), inv.data_ptr(), inv, stats, lp


def _in_one(n, dev):
    """stats, lp, inv in one tensor: fewer allocations, and one to keep for the backward."""
    m = torch.empty(3 * n + 1, dtype=torch.float32, device=dev)
    at = m.data_ptr()
    return at + 8 * n, at, at + 12 * n, m


def _cross_entropy_fwd(logits: torch.Tensor, targets: torch.Tensor, ignore_index: int, wide: bool
                       ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(the loss, fp32 -1 / the targets' number, stats)."""
    loss, (inv, stats, _) = _loss_fwd(logits, targets, ignore_index, wide, _apart)
    return loss, inv, stats


cross_entropy_fwd = torch.library.custom_op("titanmac::token_cross_entropy", mutates_args=())(_cross_entropy_fwd)


@cross_entropy_fwd.register_fake
def _(logits, targets, ignore_index, wide):
    n = 1
    for s in logits.shape[:-1]:
        n *= s
    f = lambda shape, dt=torch.float32: logits.new_empty(shape, dtype=dt)  # noqa: E731
    return f((), torch.float32 if wide else logits.dtype), f(()), f((n, 2))


def _ce_setup(ctx, inputs, output):
    logits, targets, ignore_index, _wide = inputs
    ctx.save_for_backward(logits, targets, output[1], output[2])
    ctx.ignore_index = ignore_index


def _ce_backward(ctx, g_loss, *_):
    logits, targets, inv, stats = ctx.saved_tensors
    g_lp = (g_loss.to(inv.dtype) * inv).expand(targets.shape)
    return _gradient(g_lp, None, logits, targets, stats, None, ctx.ignore_index), None, None, None


cross_entropy_fwd.register_autograd(_ce_backward, setup_context=_ce_setup)


def _ce_native_fwd(logits, targets, ignore_index, wide):
    loss, (kept,) = _loss_fwd(logits, targets, ignore_index, wide, _in_one)
    return loss, kept


def _ce_native_setup(ctx, inputs, output):
    logits, targets, ctx.ignore_index, _wide = inputs
    ctx.save_for_backward(logits, targets, output[1])


def _ce_native_backward(ctx, g_loss):
    """One launch for g_loss and all: this runs in autograd's thread, where a torch operation costs the host as much as
    the launch (and the product of a 16-bit g_loss and the fp32 -1 / n 35 us)."""
    logits, targets, kept = ctx.saved_tensors
    n, ignore = targets.numel(), ctx.ignore_index
    if not _lib.direct_backward(g_loss, logits):
        g_lp = (g_loss.to(kept.dtype) * kept[3 * n]).expand(targets.shape)
        return _gradient(g_lp, None, logits, targets, kept[:2 * n].view(n, 2), None, ignore), None, None, None
    z, sb, st, B, T, V = _rows3(logits)
    dev, at = logits.device, kept.data_ptr()
    dz = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
    if n:
        tg = _flat(targets)
        with _lib.device_guard(dev):
            rc = _lib.lib().tmac_logprob_mean_bwd(z.data_ptr(), sb, st, tg.data_ptr(), ignore, at, at + 12 * n,
                                                  g_loss.data_ptr(), _lib.dtype_code(g_loss.dtype), dz.data_ptr(), B, T, V,
                                                  _lib.dtype_code(z.dtype), _lib.stream_ptr(dev))
        _lib.check(rc, "tmac_logprob_mean_bwd")
    return dz, None, None, None


_ce_native = _lib.native_function(_ce_native_fwd, _ce_native_setup, _ce_native_backward)


def token_cross_entropy(logits: torch.Tensor, targets: torch.Tensor, *, ignore_index: int = -100) -> torch.Tensor:
    """The mean of -log softmax(logits)[target] over the targets other than ignore_index (NaN where there are
    none), as F.cross_entropy of [..., V] logits: in their dtype, or fp32 inside torch.autocast. Ignored
    rows are not read and get zeros as gradient. Other targets outside [0, V) make it NaN. The gradient reads the
    logits again: autograd refuses it if they were changed in place since."""
    args = (logits, targets, int(ignore_index), torch.is_autocast_enabled("cuda"))
    if _lib.direct_call(logits, targets):
        return _loss_fwd(*args, _in_one)[0]
    if _lib.eager_native(logits, targets):
        return _ce_native(*args)
    return cross_entropy_fwd(*args)[0]


# ------------------------------------------------------------------ scores from the hidden states

@lru_cache(maxsize=256)
def _head_workspace(M: int, V: int, K: int) -> int:
    nb = ctypes.c_size_t(0)
    _lib.check(_lib.lib().tmac_head_logprob_workspace(M, V, K, ctypes.byref(nb)), "tmac_head_logprob_workspace")
    return nb.value


def _head_logprobs(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, entropy: bool,
                   ignore_index: int) -> tuple[torch.Tensor, torch.Tensor]:
    """(logprobs, entropy or an empty tensor) of 16-bit hidden [..., K] and weight [V, K], K a multiple of 64."""
    _check_head(hidden, weight, targets)
    dev = _lib.require_device(hidden, weight, targets, what="head_logprobs")
    (V, K), lead, M = weight.shape, targets.shape, targets.numel()
    lp = torch.empty(lead, dtype=torch.float32, device=dev)
    ent = lp.new_empty(lead if entropy else (0,))
    if M:
        x, w, tg, nb = _rows(hidden), _rows(weight), _flat(targets), _head_workspace(M, V, K)
        ws = torch.empty(nb, dtype=torch.uint8, device=dev)
        with _lib.device_guard(dev):
            rc = _lib.lib().tmac_head_logprob(x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), tg.data_ptr(),
                                              ignore_index, lp.data_ptr(), ent.data_ptr() if entropy else 0, M, V, K,
                                              ws.data_ptr(), nb, _lib.dtype_code(x.dtype), _lib.stream_ptr(dev))
        _lib.check(rc, "tmac_head_logprob")
    return lp, ent


head_logprobs_fwd = torch.library.custom_op("titanmac::head_logprobs", mutates_args=())(_head_logprobs)


@head_logprobs_fwd.register_fake
def _(hidden, weight, targets, entropy, ignore_index):
    f = lambda shape: hidden.new_empty(shape, dtype=torch.float32)  # noqa: E731
    return f(targets.shape), f(targets.shape if entropy else (0,))


def _check_head(hidden, weight, targets) -> None:
    if weight.dim() != 2 or weight.shape[0] == 0 or hidden.dim() < 1 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"head_logprobs: hidden must be [..., K] and weight [V, K], got {tuple(hidden.shape)} and "
                         f"{tuple(weight.shape)}")
    if weight.dtype != hidden.dtype:
        raise TypeError(f"head_logprobs: weight dtype {weight.dtype} != hidden dtype {hidden.dtype}")
    if targets.shape != hidden.shape[:-1]:
        raise ValueError(f"head_logprobs: targets must be {tuple(hidden.shape[:-1])} for hidden "
                         f"{tuple(hidden.shape)}, got {tuple(targets.shape)}")
    if targets.dtype not in _INDEX:
        raise TypeError(f"head_logprobs: targets must be int64 or int32, got {targets.dtype}")
    _check_sizes(targets, weight.shape[0], "head_logprobs")


def head_logprobs(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *, entropy: bool = False,
                  ignore_index: int = -100) -> TokenLogprobs:
    """token_logprobs(F.linear(hidden, weight), targets) with logprobs and (if asked) entropy, the logits [..., V]
    never stored: one kernel multiplies and keeps the running softmax statistics. The logits' fp32 sums are not
    rounded on the way, so the scores are nearer to exact than those of 16-bit logits.

    hidden [..., K] and weight [V, K] of one dtype, targets int64 or int32 [...]. Where the kernel does not
    apply (fp32, K not a multiple of 64, a gradient is needed) the logits are formed by F.linear and scored by
    token_logprobs, which has the gradient."""
    _check_head(hidden, weight, targets)
    K = weight.shape[1]
    grad = torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad)
    if grad or hidden.dtype not in _HALF or K == 0 or K % 64 or K > _MAX_PITCH or weight.stride(0) > _MAX_PITCH:
        _lib.require_device(hidden, weight, targets, what="head_logprobs")
        return token_logprobs(F.linear(hidden, weight), targets, entropy=entropy, ignore_index=ignore_index)
    args = (hidden, weight, targets, bool(entropy), int(ignore_index))
    lp, ent = _head_logprobs(*args) if _lib.direct_call(hidden, weight, targets) else head_logprobs_fwd(*args)
    return TokenLogprobs(lp, ent if entropy else None)
