"""Token-by-token decoding with ``TitanMAC``: what a run of it keeps between calls.

The reference has no such path (every token costs a forward over the whole text). It exists for the model whose layers
allow it: causal ``WindowedAttention`` without a neural memory. There the persistent rows see each other only
(attn/windowed_attention.py:97-152), so all keys and values stay as they are when tokens follow;
``BlockSparseAttention``'s persistent rows see every key (attn/block_sparse_attention.py:277-286), and theirs change with
every token.
"""
from __future__ import annotations

from typing import List, Optional, Tuple, Union

import torch

from ..kernels.kv_cache import MAX_TREE, KVCache, cache_keep


class DecodeState:
    """The caches of a model's layers for ``batch`` sequences, which share one table of pages and their lengths.

    ``lengths`` (int32 [batch], persistent rows included) is on the GPU; so is everything that a call changes, and a call
    can be captured into a graph and replayed (the host's bound of the tokens that are held, ``used``, then stands still:
    tokens past the room are not written and give NaN). The bound counts a call's padding and a path's −1 as tokens; a call
    that does not fit by it, outside a capture, waits for the GPU and goes by the lengths.
    ``TitanMAC.new_decode_state`` makes it."""

    def __init__(self, caches: List[KVCache], table: torch.Tensor, lengths: torch.Tensor, n_persistent: int, room: int):
        self.caches, self.table, self.lengths = caches, table, lengths
        self.n_persistent = n_persistent
        self.room = room          # tokens that each sequence has room for
        self.used = 0             # no sequence holds more
        self._held = 0            # nor did before the last call
        self._draft: Optional[Union[int, torch.Tensor]] = None

    def _ahead(self, T: int, counts: Optional[torch.Tensor]) -> Tuple[torch.Tensor, int, int]:
        """The lengths with T new rows for each sequence (counts of them, if given), and bounds of the tokens held before
        and then. Nothing here changes before the logits are made (``_advance``): a call that is refused on the way
        leaves the state as it was."""
        if self._draft is not None:
            raise RuntimeError("DecodeState: the last call's draft was not settled: call keep()")
        ahead, held, then = self.lengths + (T if counts is None else counts), self.used, self.used + T
        if then > self.room and not (ahead.is_cuda and torch.cuda.is_current_stream_capturing()):
            # the bounds count padding, and places of a draft that its path left free: the lengths themselves
            held, then = (n - self.n_persistent for n in torch.stack([self.lengths.amax(), ahead.amax()]).tolist())
        if then > self.room:
            raise ValueError(f"DecodeState: {then} tokens do not fit in {self.room} (up to {held} are held)")
        return ahead, held, then

    def _advance(self, T: int, counts: Optional[torch.Tensor], draft: bool, held: int, then: int) -> None:
        """The caches hold the rows of ``_ahead``."""
        self.lengths.add_(T if counts is None else counts)
        self.used, self._held = then, held
        if draft:
            self._draft = T if counts is None else counts.clone()  # the caller's may be a buffer that changes
            self._draft_rows = T

    def keep(self, path: torch.Tensor) -> None:
        """Settles a draft: of its rows those that path (int32 [batch, rows]; −1 behind a sequence's last) names stay, in
        this order, and the others are dropped. Every entry of 0 or more counts as a row of the draft."""
        if self._draft is None:
            raise RuntimeError("DecodeState: there is no draft to keep rows of")
        if path.dim() != 2 or path.shape[0] != self.lengths.shape[0] or path.shape[1] > self._draft_rows:
            raise ValueError(f"DecodeState: path must be [{self.lengths.shape[0]}, up to {self._draft_rows}], got "
                             f"{tuple(path.shape)}")
        with torch.no_grad():
            for cache in self.caches:
                cache_keep(cache, self.table, self.lengths, path, self._draft)
            kept = (path >= 0).sum(1, dtype=torch.int32)
            if isinstance(self._draft, torch.Tensor):
                kept = torch.minimum(kept, self._draft)  # places behind a shorter draft are none
            self.lengths.add_(kept - self._draft)
        self.used = min(self.used, self._held + path.shape[1])
        self._draft = None


def draft_depths(tree: torch.Tensor) -> torch.Tensor:
    """Places of a draft's rows behind its base: the number of their bits − 1."""
    return (tree.unsqueeze(-1) >> torch.arange(MAX_TREE, device=tree.device) & 1).sum(-1) - 1
