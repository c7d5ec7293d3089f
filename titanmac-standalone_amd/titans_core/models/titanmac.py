"""TitanMAC language model (drop-in for models/titanmac.py).

Same constructor, submodules, parameters, buffers and state_dict keys as the reference
(models/titanmac.py:36-158), and the same forwards with the same outputs:

- ``forward`` dispatches to ``forward_mac`` / ``forward_mag`` / ``forward_mal`` when the neural
  memory is on (:554-600), and otherwise runs embeddings → [persistent | sequence] → blocks →
  norm → head (:601-686);
- ``forward_mac`` (:160-313) splits the sequence into segments. For each one it retrieves
  ``n_memory_tokens`` memory tokens from the segment mean, runs the blocks over
  [persistent | memory | segment], updates the memory (training or test-time memory) or only
  measures its loss, and gates the segment output by sigmoid(gate_proj(M*(y)));
- ``forward_mag`` (:315-432) and ``forward_mal`` (:434-547).

Every block op runs on the HIP kernels (RMSNorm, depthwise conv, tile-sparse attention,
Block-ELL MLP when configured), the neural memory's update on its HIP step, the embeddings and the
loss on theirs (``token_embedding``, ``token_cross_entropy``), and the dense projections and the LM
head on hipBLASLt. ``score``, which the reference lacks, gives each token's log probability without
storing the logits; ``decode`` and ``generate``, which it lacks too, answer token by token from a cache of
keys and values (``models/decoding.py``).

One change of schedule, not of result: when the memory is read-only (eval mode without
``enable_test_time_memory``), ``forward_mac``'s segments do not depend on each other. The
reference still runs them one after another, each as B sequences of S = Np + N_l + segment
tokens. Here all full segments run through the blocks as one batch of (n_segments·B)
sequences, and a shorter last segment as a second batch. That is the same arithmetic per
sequence, in a few large launches instead of many small ones. With updates on, segment i+1
reads the memory that segment i wrote, so they run in order as in the reference.
"""
from __future__ import annotations

from typing import Dict, Optional

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.utils.checkpoint import checkpoint

from ..blocks.norms import RMSNorm
from ..blocks.titan_block import TitanBlock
from ..config import TitanMACConfig
from ..kernels import _lib
from ..kernels.embedding import token_embedding
from ..kernels.kv_cache import MAX_TREE, KVCache
from ..kernels.logprobs import head_logprobs, token_cross_entropy, token_logprobs
from ..attn.windowed_attention import WindowedAttention
from ..memory.neural_memory import NeuralMemory
from .decoding import DecodeState, draft_depths


_IGNORE = -100  # F.cross_entropy's ignore_index


def _untouched(m: nn.Module, kind: type) -> bool:
    """Whether calling m does just what `kind`'s own forward does: no subclass, replaced forward or hook."""
    return (type(m) is kind and "forward" not in m.__dict__ and not m._forward_hooks and not m._forward_pre_hooks
            and not m._backward_hooks and not m._backward_pre_hooks
            and not torch.nn.modules.module._has_any_global_hook())


def _plain_lookup(m: nn.Module) -> bool:
    return (_untouched(m, nn.Embedding) and m.padding_idx is None and m.max_norm is None
            and not m.scale_grad_by_freq and not m.sparse)


class TitanMAC(nn.Module):
    """Titan Memory-Augmented Context model: input_ids [B, T] → {"logits": [B, T, vocab], ...}."""

    def __init__(self, config: TitanMACConfig):
        super().__init__()
        self.config = config
        config.validate()
        if config.use_memory_bank:
            raise NotImplementedError(
                "use_memory_bank: the legacy MemoryBank is not part of this build (no forward of "
                "the reference reads it)")
        d = config.d_model
        self.embed_tokens = nn.Embedding(config.vocab_size, d)
        self.embed_positions = nn.Embedding(config.max_seq_len, d)
        if config.n_persistent > 0:
            self.persistent_tokens = nn.Parameter(torch.zeros(config.n_persistent, d))
        else:
            self.register_parameter("persistent_tokens", None)
        self.layers = nn.ModuleList([TitanBlock(config) for _ in range(config.n_layers)])
        self.norm = RMSNorm(d, eps=config.norm_eps)
        self.lm_head = nn.Linear(d, config.vocab_size, bias=False)
        if config.tie_weights:
            self.lm_head.weight = self.embed_tokens.weight
        self.memory_bank = None
        if config.use_neural_memory:
            d_mem = config.d_memory if config.d_memory is not None else d
            self.neural_memory = NeuralMemory(
                d_model=d, d_memory=d_mem, n_memory_layers=config.n_memory_layers,
                theta_lr=config.memory_theta_lr, forget_hidden=config.memory_forget_hidden,
                decay_hidden=config.memory_decay_hidden)
            self.memory_proj = nn.Linear(d_mem, d)
            self.gate_proj = nn.Linear(d_mem, d)
        else:
            self.neural_memory = None
            self.memory_proj = None
            self.gate_proj = None
        self.gradient_checkpointing = False
        self._block_graph = None
        self._init_weights()

    def _init_weights(self) -> None:
        """N(0, 0.02) embeddings, persistent tokens, untied head, memory projections (:140-158)."""
        nn.init.normal_(self.embed_tokens.weight, mean=0.0, std=0.02)
        nn.init.normal_(self.embed_positions.weight, mean=0.0, std=0.02)
        if self.persistent_tokens is not None:
            nn.init.normal_(self.persistent_tokens, mean=0.0, std=0.02)
        if not self.config.tie_weights:
            nn.init.normal_(self.lm_head.weight, mean=0.0, std=0.02)
        if self.memory_proj is not None:
            nn.init.normal_(self.memory_proj.weight, mean=0.0, std=0.02)
        if self.gate_proj is not None:
            nn.init.normal_(self.gate_proj.weight, mean=0.0, std=0.02)

    # ------------------------------------------------------------------ helpers

    def _embed(self, input_ids: torch.Tensor, persistent: bool = False) -> torch.Tensor:
        """Token plus position rows [B, T, d], behind the persistent tokens if asked (and there are any):
        one kernel for plain embedding modules on the GPU, the modules themselves otherwise."""
        B, T = input_ids.shape
        tok, pos = self.embed_tokens, self.embed_positions
        prefix = self.persistent_tokens if persistent and self.config.n_persistent > 0 else None
        if _plain_lookup(tok) and _plain_lookup(pos) and T <= pos.num_embeddings:
            tables = [t for t in (tok.weight, pos.weight, prefix) if t is not None]
            if (input_ids.dtype in (torch.int64, torch.int32) and _lib.eager_native(input_ids, *tables)
                    and all(t.is_cuda and t.device == input_ids.device and t.dtype == tok.weight.dtype
                            and t.dtype in _lib._DTYPE_CODE for t in tables)):
                return token_embedding(input_ids, tok.weight, pos.weight, prefix=prefix)
        x = tok(input_ids) + pos(torch.arange(T, device=input_ids.device)).unsqueeze(0)
        return x if prefix is None else torch.cat([prefix.unsqueeze(0).expand(B, -1, -1), x], dim=1)

    def _persistent(self, B: int) -> Optional[torch.Tensor]:
        if self.persistent_tokens is not None and self.config.n_persistent > 0:
            return self.persistent_tokens.unsqueeze(0).expand(B, -1, -1)
        return None

    def _n_persistent(self) -> int:
        return 0 if self.persistent_tokens is None else self.config.n_persistent

    def _blocks(self, y: torch.Tensor, layers=None) -> torch.Tensor:
        for layer in (self.layers if layers is None else layers):
            if self.gradient_checkpointing and self.training:
                y = checkpoint(lambda h, m=layer: m(h, attn_mask=None), y, use_reentrant=False)
            else:
                y = layer(y, attn_mask=None)
        return y

    # ------------------------------------------------------------------ block-stack graph

    def _tensor_ptrs(self):
        return tuple(t.data_ptr() for t in list(self.parameters()) + list(self.buffers()))

    def capture_block_graph(self, batch: int, seq_len: Optional[int] = None) -> None:
        """Capture the layer stack for one input shape [batch, seq_len, d_model] in a HIP graph.

        For eval forwards with test-time memory, whose segments run the layers one after
        another with small batches: there the host's launch rate, not the GPU, sets the pace,
        and one graph replay replaces a few hundred launches. seq_len defaults to the MAC
        segment shape, n_persistent + n_memory_tokens + segment_size. Without gradients and
        outside training, ``forward_mac`` then replays the graph for every input of that
        shape, dtype and device; other inputs, and any call after a parameter or buffer was
        replaced (not updated in place, e.g. by ``.to()``), run the layers eagerly again.
        Results are bit-identical to the eager layers (the same kernels on the same data).
        Capture again after such changes; ``release_block_graph`` frees the graph.
        """
        if seq_len is None:
            seq_len = self.config.n_persistent + self.config.n_memory_tokens + self.config.segment_size
        p = next(self.parameters())
        if not p.is_cuda:
            raise RuntimeError("capture_block_graph needs the model on a GPU")
        self.release_block_graph()
        static_in = torch.zeros(batch, seq_len, self.config.d_model, dtype=p.dtype, device=p.device)
        was_training = self.training
        self.eval()
        try:
            side = torch.cuda.Stream(device=p.device)
            side.wait_stream(torch.cuda.current_stream(p.device))
            with torch.cuda.stream(side), torch.no_grad():
                for _ in range(2):  # warm-up outside the capture (lazy caches, libraries)
                    self._blocks(static_in)
            torch.cuda.current_stream(p.device).wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph), torch.no_grad():
                static_out = self._blocks(static_in)
        finally:
            self.train(was_training)
        self._block_graph = {"graph": graph, "in": static_in, "out": static_out,
                             "ptrs": self._tensor_ptrs(), "replays": 0}

    def release_block_graph(self) -> None:
        self._block_graph = None

    def _graph_blocks(self, parts) -> torch.Tensor:
        """blocks(cat(parts, dim=1)) through the captured graph when it applies; the result
        stays valid until the next call (the graph's output buffer)."""
        gr = self._block_graph
        if gr is not None and not self.training and not torch.is_grad_enabled():
            st = gr["in"]
            if (all(t.dtype == st.dtype and t.device == st.device for t in parts)
                    and sum(t.shape[1] for t in parts) == st.shape[1]
                    and all(t.shape[0] == st.shape[0] and t.shape[2] == st.shape[2] for t in parts)
                    and self._tensor_ptrs() == gr["ptrs"]):
                torch.cat(parts, dim=1, out=st)
                gr["graph"].replay()
                gr["replays"] += 1
                return gr["out"]
        return self._blocks(torch.cat(parts, dim=1))

    def _memory_step(self, y: torch.Tensor) -> torch.Tensor:
        if self.training or self.config.enable_test_time_memory:
            return self.neural_memory.update(y)
        return self.neural_memory.compute_loss(y)

    @staticmethod
    def _next_tokens(labels: torch.Tensor) -> torch.Tensor:
        """The token that each position is to predict; the last one's is ignored."""
        return F.pad(labels[..., 1:], (0, 1), value=_IGNORE)

    def _cross_entropy(self, logits: torch.Tensor, labels: torch.Tensor) -> torch.Tensor:
        """F.cross_entropy of the logits [B, T, V] against the next token: on its kernel (the logits read in
        place, once) for plain GPU tensors."""
        V = self.config.vocab_size
        if (logits.is_cuda and labels.is_cuda and logits.device == labels.device and logits.dtype in _lib._DTYPE_CODE
                and labels.dtype == torch.int64 and logits.shape == (*labels.shape, V) and labels.shape[-1] > 0
                and _lib.eager_native(logits, labels)):
            return token_cross_entropy(logits, self._next_tokens(labels), ignore_index=_IGNORE)
        return F.cross_entropy(logits[..., :-1, :].contiguous().reshape(-1, V),
                               labels[..., 1:].contiguous().reshape(-1), reduction="mean", ignore_index=_IGNORE)

    def _output(self, logits: torch.Tensor, labels: Optional[torch.Tensor],
                memory_loss: Optional[torch.Tensor]) -> Dict[str, torch.Tensor]:
        out = {"logits": logits}
        if memory_loss is not None:
            out["memory_loss"] = memory_loss
        if labels is not None:
            ce = self._cross_entropy(logits, labels)
            if memory_loss is None:
                out["loss"] = ce
            else:
                out["ce_loss"] = ce
                out["loss"] = ce + memory_loss
        return out

    # ------------------------------------------------------------------ MAC

    def _mac_segments(self, xs: torch.Tensor, persistent_row: Optional[torch.Tensor],
                      n_seq: int, acc: torch.Tensor) -> torch.Tensor:
        """Blocks and gated output for a batch of independent segments xs [n·B, L, d]
        (segment-major) against a read-only memory; adds each segment's memory loss
        F.mse_loss(M(W_K y), W_V y) over its B sequences to ``acc`` in order, as the reference's
        per-segment loop does. Returns o [n·B, L, d]."""
        nl = self.config.n_memory_tokens
        NB, L, d = xs.shape
        h = self.memory_proj(self.neural_memory.retrieve(xs.mean(dim=1, keepdim=True)))
        parts = [h.expand(NB, nl, d), xs]
        if persistent_row is not None:
            parts.insert(0, persistent_row.unsqueeze(0).expand(NB, -1, -1))
        y = self._blocks(torch.cat(parts, dim=1))
        ys = y[:, y.shape[1] - L:]
        nm = self.neural_memory
        pred, target = nm.memory_mlp(nm.W_K(ys)), nm.W_V(ys)
        B = NB // n_seq
        for s in range(n_seq):
            acc.add_(F.mse_loss(pred[s * B:(s + 1) * B], target[s * B:(s + 1) * B]))
        gate = torch.sigmoid(self.gate_proj(nm.retrieve(ys)))
        return ys * gate

    def forward_mac(self, input_ids: torch.Tensor, labels: Optional[torch.Tensor] = None,
                    attention_mask: Optional[torch.Tensor] = None) -> Dict[str, torch.Tensor]:
        """Memory as Context (models/titanmac.py:160-313)."""
        h, memory_loss = self._hidden_mac(input_ids)
        return self._output(self.lm_head(h), labels, memory_loss)

    def _hidden_mac(self, input_ids: torch.Tensor):
        """(the head's input [B, T, d], memory loss) of forward_mac."""
        if self.neural_memory is None:
            raise ValueError("forward_mac requires use_neural_memory=True")
        B, T = input_ids.shape
        x = self._embed(input_ids)
        seg = self.config.segment_size
        nl = self.config.n_memory_tokens
        n_segments = (T + seg - 1) // seg
        persistent = self._persistent(B)
        Np = 0 if persistent is None else self.config.n_persistent

        if not (self.training or self.config.enable_test_time_memory):
            # Read-only memory: all full segments in one batch, the remainder in another.
            n_full, tail = divmod(T, seg)
            prow = None if persistent is None else self.persistent_tokens
            outs, acc = [], torch.zeros(1, device=x.device, dtype=x.dtype)
            if n_full:
                xs = x[:, :n_full * seg].reshape(B, n_full, seg, -1).transpose(0, 1)
                o = self._mac_segments(xs.reshape(n_full * B, seg, -1), prow, n_full, acc)
                outs.append(o.reshape(n_full, B, seg, -1).transpose(0, 1).reshape(B, n_full * seg, -1))
            if tail:
                outs.append(self._mac_segments(x[:, n_full * seg:], prow, 1, acc))
            o = x if not outs else (outs[0] if len(outs) == 1 else torch.cat(outs, dim=1))
            memory_loss = (acc / n_segments).squeeze()  # nan for T = 0, as in the reference
        else:
            o = torch.empty_like(x)
            acc = torch.zeros(1, device=x.device, dtype=x.dtype)
            for s in range(n_segments):
                a, b = s * seg, min(s * seg + seg, T)
                xs = x[:, a:b]
                q = xs.mean(dim=1, keepdim=True).expand(B, nl, -1)
                h = self.memory_proj(self.neural_memory.retrieve(q))
                parts = [h, xs] if persistent is None else [persistent, h, xs]
                y = self._graph_blocks(parts)
                ys = y[:, Np + nl:]
                acc = acc + self._memory_step(ys)
                gate = torch.sigmoid(self.gate_proj(self.neural_memory.retrieve(ys)))
                o[:, a:b] = ys * gate
            memory_loss = (acc / n_segments).squeeze()
        return self.norm(o), memory_loss

    # ------------------------------------------------------------------ MAG / MAL

    def forward_mag(self, input_ids: torch.Tensor, labels: Optional[torch.Tensor] = None,
                    attention_mask: Optional[torch.Tensor] = None) -> Dict[str, torch.Tensor]:
        """Memory as Gate (models/titanmac.py:315-432): o = blocks(x̃) ⊙ sigmoid(gate_proj(M*(x̃)))."""
        h, memory_loss = self._hidden_mag(input_ids)
        return self._output(self.lm_head(h), labels, memory_loss)

    def _hidden_mag(self, input_ids: torch.Tensor):
        """(the head's input [B, T, d], memory loss) of forward_mag."""
        if self.neural_memory is None:
            raise ValueError("forward_mag requires use_neural_memory=True")
        xc = self._embed(input_ids, persistent=True)
        gate = torch.sigmoid(self.gate_proj(self.neural_memory.retrieve(xc)))
        y = self._blocks(xc)
        o = y * gate
        Np = self._n_persistent()
        memory_loss = self._memory_step(y[:, Np:])
        return self.norm(o)[:, Np:], memory_loss

    def forward_mal(self, input_ids: torch.Tensor, labels: Optional[torch.Tensor] = None,
                    attention_mask: Optional[torch.Tensor] = None) -> Dict[str, torch.Tensor]:
        """Memory as Layer (models/titanmac.py:434-547): even layers are blocks, odd layers add
        memory_proj(M*(y))."""
        h, memory_loss = self._hidden_mal(input_ids)
        return self._output(self.lm_head(h), labels, memory_loss)

    def _hidden_mal(self, input_ids: torch.Tensor):
        """(the head's input [B, T, d], memory loss) of forward_mal."""
        if self.neural_memory is None:
            raise ValueError("forward_mal requires use_neural_memory=True")
        y = self._embed(input_ids, persistent=True)
        for i, layer in enumerate(self.layers):
            if i % 2 == 0:
                y = self._blocks(y, [layer])
            else:
                y = y + self.memory_proj(self.neural_memory.retrieve(y))
        Np = self._n_persistent()
        memory_loss = self._memory_step(y[:, Np:])
        return self.norm(y)[:, Np:], memory_loss

    def forward_with_memory(self, *args, **kwargs):
        """Alias of forward_mac (models/titanmac.py:550-552)."""
        return self.forward_mac(*args, **kwargs)

    # ------------------------------------------------------------------ dispatch

    def forward(self, input_ids: torch.Tensor, labels: Optional[torch.Tensor] = None,
                attention_mask: Optional[torch.Tensor] = None) -> Dict[str, torch.Tensor]:
        """The variant's forward: ``logits``, with a neural memory ``memory_loss``, with labels ``loss``.

        On the kernels nothing is copied to the host to look at ids and labels: an id outside the vocabulary gives
        its positions NaN, a label outside it (other than -100) a loss of NaN. The loss keeps the logits for its
        gradient, so autograd refuses the backward if they were changed in place before it: change a copy."""
        if self.neural_memory is not None and self.config.use_neural_memory:
            variant = self.config.titans_variant
            if variant == "MAC":
                return self.forward_mac(input_ids, labels, attention_mask)
            if variant == "MAG":
                return self.forward_mag(input_ids, labels, attention_mask)
            if variant == "MAL":
                return self.forward_mal(input_ids, labels, attention_mask)
            raise ValueError(f"Unknown titans_variant: {variant}")
        logits = self.lm_head(self.norm(self._blocks(self._embed(input_ids, persistent=True))))
        if self._n_persistent():
            logits = logits[:, self.config.n_persistent:, :]
        return self._output(logits, labels, None)

    # ------------------------------------------------------------------ scores

    def score(self, input_ids: torch.Tensor, labels: Optional[torch.Tensor] = None, *, entropy: bool = False,
              top_k: int = 0) -> Dict[str, torch.Tensor]:
        """Per-token scores of a text: ``logprobs`` [B, T] fp32, at position t the log probability of
        labels[:, t + 1] (labels defaults to input_ids) given the tokens up to t, 0 at the last position and
        where that label is -100; on request ``entropy`` [B, T] and ``top_ids``, ``top_logprobs``
        [B, T, top_k] of each position's distribution; with a neural memory its ``memory_loss``, and the
        memory is updated exactly as by ``forward``.

        Under ``torch.no_grad()`` in 16 bit and without top_k the logits are never stored (``head_logprobs``);
        otherwise they are formed as in ``forward`` and read once (``token_logprobs``)."""
        labels = input_ids if labels is None else labels
        if labels.shape != input_ids.shape:
            raise ValueError(f"score: labels must be {tuple(input_ids.shape)}, got {tuple(labels.shape)}")
        memory_loss = None
        if self.neural_memory is not None and self.config.use_neural_memory:
            hidden = {"MAC": self._hidden_mac, "MAG": self._hidden_mag,
                      "MAL": self._hidden_mal}.get(self.config.titans_variant)
            if hidden is None:
                raise ValueError(f"Unknown titans_variant: {self.config.titans_variant}")
            h, memory_loss = hidden(input_ids)
        else:
            h = self.norm(self._blocks(self._embed(input_ids, persistent=True)))[:, self._n_persistent():]
        targets = self._next_tokens(labels)[..., :labels.shape[-1]]
        head = self.lm_head
        if (top_k == 0 and _untouched(head, nn.Linear) and head.bias is None and head.weight.dtype == h.dtype
                and not torch.is_autocast_enabled("cuda")):
            r = head_logprobs(h, head.weight, targets, entropy=entropy, ignore_index=_IGNORE)
        else:
            r = token_logprobs(head(h), targets, entropy=entropy, top_k=top_k, ignore_index=_IGNORE)
        out = {n: t for n, t in r._asdict().items() if t is not None}
        if memory_loss is not None:
            out["memory_loss"] = memory_loss
        return out

    # ------------------------------------------------------------------ decoding

    def new_decode_state(self, batch: int, max_tokens: Optional[int] = None, *, fmt: Optional[str] = None,
                         page: int = 64) -> DecodeState:
        """Empty caches for ``batch`` sequences of up to max_tokens (default: max_seq_len) tokens, with the persistent rows
        already in them. fmt: None holds keys and values in the model's type (made inside ``torch.autocast``: in
        autocast's; decode inside it then too), "int8" and "e4m3" in 8 bits with a scale per row (``KVCache``). For models
        of causal WindowedAttention (use_block_sparse=False) without a neural memory."""
        cfg = self.config
        if self.neural_memory is not None:
            raise ValueError("new_decode_state: a neural memory's tokens depend on whole segments; there is no cache of it")
        for layer in self.layers:
            if not isinstance(layer.attention, WindowedAttention) or not layer.attention.causal:
                raise ValueError("new_decode_state: the layers must be causal WindowedAttention (use_block_sparse=False)")
        room = cfg.max_seq_len if max_tokens is None else int(max_tokens)
        if batch < 1 or not 1 <= room <= cfg.max_seq_len:
            raise ValueError(f"new_decode_state: batch must be positive and max_tokens 1..{cfg.max_seq_len}, got {batch}, "
                             f"{room}")
        w, Np = self.embed_tokens.weight, self._n_persistent()
        per = -(-(Np + room) // page)
        dev = w.device.type
        if torch.is_autocast_enabled(dev):  # the projections' outputs
            dtype = torch.get_autocast_dtype(dev)
        else:
            dtype = self.layers[0].attention.qkv_proj.weight.dtype if self.layers else w.dtype
        # what changes from call to call is not an inference tensor, which could be written inside inference mode only
        with torch.inference_mode(False), torch.no_grad():
            caches = [KVCache.new(batch * per, cfg.n_heads, cfg.d_head, page=page, dtype=dtype, fmt=fmt, device=w.device)
                      for _ in self.layers]
            table = torch.arange(batch * per, dtype=torch.int32, device=w.device).view(batch, per)
            state = DecodeState(caches, table, torch.full((batch,), Np, dtype=torch.int32, device=w.device), Np, room)
            if Np:
                x = self.persistent_tokens.unsqueeze(0).expand(batch, -1, -1)
                for table_of in (self.embed_tokens, self.embed_positions):  # as behind the tokens' rows
                    x = x.to(torch.promote_types(x.dtype, table_of.weight.dtype))
                for layer, cache in zip(self.layers, caches):
                    x = layer.forward_cached(x, cache, table, state.lengths)
        return state

    @torch.no_grad()
    def decode(self, input_ids: torch.Tensor, state: DecodeState, *, counts: Optional[torch.Tensor] = None,
               tree: Optional[torch.Tensor] = None, last: bool = False) -> torch.Tensor:
        """Logits [B, T, vocab] of tokens that follow those which ``state`` holds, and which it then holds too: forward's
        rows for them, to rounding. Any T: a prompt, a part of one, single tokens. last: only of each sequence's last new
        token, [B, 1, vocab].

        counts (int32 [B]): how many of the T are tokens; the rest is padding, whose logits say nothing. tree (int64
        [B, T] or [T], T up to 64): the tokens are a draft, as in ``cached_attention``; ``state.keep`` then says
        which of them stay. Hooks of the blocks and their attention are not run. A call that raises an error leaves
        ``state`` as it was."""
        B, T = input_ids.shape
        if B != state.lengths.shape[0]:
            raise ValueError(f"decode: the state has {state.lengths.shape[0]} sequences, input_ids is "
                             f"{tuple(input_ids.shape)}")
        if T == 0:
            return self.lm_head.weight.new_empty((B, 0, self.config.vocab_size))
        if counts is not None and (counts.shape != (B,) or counts.dtype != torch.int32):
            raise ValueError(f"decode: counts must be int32 [{B}], got {counts.dtype} {tuple(counts.shape)}")
        if tree is not None and (T > MAX_TREE or tree.dtype != torch.int64 or tuple(tree.shape) not in ((B, T), (T,))):
            raise ValueError(f"decode: tree must be int64 [{B}, {T}] or [{T}], T up to {MAX_TREE}, got {tree.dtype} "
                             f"{tuple(tree.shape)}")
        place = torch.arange(T, device=input_ids.device) if tree is None else draft_depths(tree)
        positions = (state.lengths - state.n_persistent).unsqueeze(1) + place
        lengths, *bounds = state._ahead(T, counts)
        x = self._embed_at(input_ids, positions)
        for layer, cache in zip(self.layers, state.caches):
            x = layer.forward_cached(x, cache, state.table, lengths, counts=counts, tree=tree)
        if last:
            if counts is None:
                x = x[:, -1:]
            else:
                at = (counts.long() - 1).clamp(min=0)
                x = x.gather(1, at.view(B, 1, 1).expand(B, 1, x.shape[-1]))
        logits = self.lm_head(self.norm(x))
        state._advance(T, counts, tree is not None, *bounds)
        return logits

    def _embed_at(self, input_ids: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
        """Token plus position rows [B, T, d] at given positions; padding may be past the table's last."""
        tok, pos = self.embed_tokens, self.embed_positions
        if (_plain_lookup(tok) and _plain_lookup(pos) and input_ids.dtype in (torch.int64, torch.int32)
                and tok.weight.is_cuda and tok.weight.dtype == pos.weight.dtype and tok.weight.dtype in _lib._DTYPE_CODE
                and _lib.eager_native(input_ids, tok.weight, pos.weight)):
            x = token_embedding(input_ids, tok.weight, pos.weight, positions=positions)
        else:
            x = tok(input_ids) + pos(positions.clamp(0, pos.num_embeddings - 1))
        rows = self.persistent_tokens  # forward's rows have a type for both
        return x if rows is None else x.to(torch.promote_types(x.dtype, rows.dtype))

    @torch.no_grad()
    def generate(self, input_ids: torch.Tensor, n_tokens: int, *, counts: Optional[torch.Tensor] = None,
                 fmt: Optional[str] = None) -> torch.Tensor:
        """The n_tokens [B, n_tokens] that follow the prompts input_ids [B, T] if each is the likeliest (ties: the lower
        id). counts (int32 [B]): the prompts' lengths, at least 1; fmt: how keys and values are held (``new_decode_state``)."""
        B, T = input_ids.shape
        if T < 1 or n_tokens < 0:
            raise ValueError(f"generate: needs prompts and n_tokens >= 0, got {tuple(input_ids.shape)}, {n_tokens}")
        out = torch.empty((B, n_tokens), dtype=torch.int64, device=input_ids.device)
        if n_tokens == 0:
            return out
        state = self.new_decode_state(B, T + n_tokens - 1, fmt=fmt)
        logits = self.decode(input_ids, state, counts=counts, last=True)
        for i in range(n_tokens):
            out[:, i] = logits[:, 0].argmax(-1)
            if i + 1 < n_tokens:
                logits = self.decode(out[:, i:i + 1], state, last=True)
        return out

    # ------------------------------------------------------------------ utilities

    def _should_update_memory(self) -> bool:
        return True if self.training else self.config.enable_test_time_memory

    def get_num_params(self, non_embedding: bool = True) -> int:
        """Parameter count, optionally without the embeddings (and an untied head) (:701-730)."""
        total = sum(p.numel() for p in self.parameters())
        if not non_embedding:
            return total
        emb = self.embed_tokens.weight.numel() + self.embed_positions.weight.numel()
        if not self.config.tie_weights:
            emb += self.lm_head.weight.numel()
        return total - emb

    def reset_memory(self) -> None:
        """Resets the MemoryBank in the reference; there is none here (see __init__)."""

    def get_memory_stats(self) -> Optional[Dict[str, float]]:
        return None

    def enable_gradient_checkpointing(self) -> None:
        self.gradient_checkpointing = True

    def disable_gradient_checkpointing(self) -> None:
        self.gradient_checkpointing = False
