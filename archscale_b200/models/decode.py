"""Key-value cache of a model during generation: one paged cache per attention call of a forward pass, and the tokens they hold.

The reference generates by re-running the whole prefix for every token (`eval.py:36-111`), which stays the default of
:meth:`archscale_b200.eval.ModelWrapper.generate`; with this a step computes its own tokens only.  Attention models are
covered: grouped, windowed, sink, gated, with QK-norm, differential, and the cross-attention of YOCO layers, which read the
cache of the layer that made their keys.
"""
from __future__ import annotations

from typing import Callable, Dict, Hashable, List, Optional, Tuple

import torch

from archscale_b200 import ops


def unsupported(model) -> Optional[str]:
    """What in a model a cache does not cover, or None."""
    cfg = model.config
    for block in model.transformer.h:
        if block.use_rnn:
            return f"{cfg.rnn_type} layers (their states are not kept)"
        if block.use_gmu:
            return "gated memory units (their memories are not kept)"
    for on, what in ((cfg.lc, "token-skipping layers"), (cfg.sc_attn, "short convolutions on queries, keys and values"), (cfg.use_sigmoid, "sigmoid attention"),
                     (not cfg.fa2, "attention by the root of the softmax"), (cfg.use_cu_seqlen, "packed rows of several documents"),
                     (getattr(model, "tp_size", 1) > 1, "tensor parallelism"), (cfg.use_da and cfg.sink_attn, "sinks of differential attention")):
        if on:
            return what
    return None


class DecodeCache:
    """``model(idx, cache=cache)`` appends the tokens ``idx`` (B, T) to it and computes them over everything it holds.

    ``dtype``: bfloat16 or float32 (default: the model's compute type), or float8_e4m3fn with a power of two per token and head.  All sequences
    have the same number of tokens.

    Once a cache holds tokens, calls can be captured by ``torch.cuda.graph``.  A capture appends nothing; each replay takes its positions from
    ``lengths`` on the device and advances them.  A replay that the capacity has no room for gives NaN.  Replays and other calls may follow one another
    on a stream in any order: after a capture ``tokens`` (and so the next call that is not captured) reads ``lengths``, which waits for the device."""

    def __init__(self, model, batch: int, capacity: int, page_size: int = 64, dtype: Optional[torch.dtype] = None, device=None) -> None:
        why = unsupported(model)
        if why is not None:
            raise ValueError(f"a key-value cache does not cover {why}: generate without it")
        if batch < 1 or capacity < 1 or page_size < 1:
            raise ValueError(f"a cache of {batch} sequences of {capacity} tokens in pages of {page_size}: all must be positive")
        cfg, bc = model.config, model.block_cfg
        device = model.transformer.wte.weight.device if device is None else device
        reps = bc.n_layer // bc.share_group // bc.share_per_layer if bc.share_per_layer > 0 else 1
        layers = reps * sum(not block.yoco_cross for block in model.transformer.h)
        pages = -(-capacity // page_size)
        self.batch, self.capacity = batch, capacity
        self.table = torch.arange(batch * pages, dtype=torch.int32, device=device).view(batch, pages)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self.layers: List[ops.PagedCache] = [ops.new_paged_cache(batch * pages, cfg.n_query_groups, page_size, cfg.head_size, dtype or model.compute_dtype, device)
                                             for _ in range(layers)]
        self._at, self._open, self._tokens = -1, 0, 0
        self._capturing, self._captured = False, False
        self._rows: Optional[torch.Tensor] = None                 # positions of a captured call's tokens
        self._tables: Dict[Hashable, Tuple[torch.Tensor, torch.Tensor]] = {}       # captured calls read them: they live as long as the cache

    def _in_capture(self) -> bool:
        if not self.lengths.is_cuda:
            return False
        with torch.cuda.device(self.lengths.device):
            return torch.cuda.is_current_stream_capturing()

    @property
    def tokens(self) -> int:
        """Tokens of each sequence."""
        if self._captured and not self._in_capture():             # replays have moved lengths
            self._tokens = int(self.lengths[0]) - self._open
        return self._tokens

    def begin(self, idx: torch.Tensor) -> None:
        """Before the first layer: room for the tokens."""
        B, T = idx.shape
        self._capturing = self._in_capture()
        if B != self.batch:
            raise ValueError(f"the cache holds {self.batch} sequences, got {B}")
        if self.tokens + T > self.capacity:
            raise ValueError(f"the cache holds {self.capacity} tokens: {self._tokens} are there, {T} more were given")
        if torch.is_grad_enabled():
            raise RuntimeError("a key-value cache has no gradients: call the model under torch.no_grad()")
        self._at = -1
        if self._capturing:
            if self._tokens == 0:
                raise RuntimeError("the first tokens of a cache cannot be captured: its replays would be further ones")
            if self._open:
                raise RuntimeError("the last call with this cache failed: call the model once before a capture")
            self._captured = True
            self.lengths += T
            self._rows = (self.lengths[:1] - T + torch.arange(T, dtype=torch.int32, device=self.lengths.device)).clamp(0, self.capacity - 1)
            return
        if self._open:                                             # the call before did not come to its end
            self.lengths -= self._open
        self.lengths += T
        self._open = T

    def end(self, T: int) -> None:
        """After the last operation of a call."""
        self._rows = None
        if not self._capturing:
            self._tokens += T
            self._open = 0

    @property
    def filling(self) -> bool:
        """Whether the tokens of this call are the first ones: attention over them alone."""
        return self._tokens == 0

    def positions(self, name: Hashable, table: Callable[[], Tuple[torch.Tensor, torch.Tensor]], T: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """Rows of a rotary table, which covers the capacity, at the positions of the T new tokens.  ``name`` tells the tables of a model apart.  One is kept
        as the first call had it, since graphs read it; a captured call gathers the rows on the device."""
        if name not in self._tables and not self._capturing:
            self._tables[name] = table()
        if self._capturing:
            return tuple(t.index_select(0, self._rows) for t in self._tables[name])
        return tuple(t[self._tokens:self._tokens + T] for t in self._tables[name])

    def bounded(self, x: torch.Tensor) -> torch.Tensor:
        """The model's output, NaN in replays past the capacity."""
        return x.masked_fill(self.lengths[0] > self.capacity, float("nan")) if self._capturing else x

    def write(self, k: torch.Tensor, v: torch.Tensor) -> None:
        """Keys and values (B, T, G, D) of the next attention layer; layers that only read use the last ones written."""
        self._at += 1
        ops.paged_cache_write(self.layers[self._at], k, v, self.table, self.lengths)

    def attend(self, q: torch.Tensor, scale: float, window, sink: Optional[torch.Tensor]) -> torch.Tensor:
        return ops.paged_attention(q, self.layers[self._at], self.table, self.lengths, scale=scale, window=window, sink=sink)

    def attend_diff(self, q: torch.Tensor, scale: float, window, lam: torch.Tensor, weight: torch.Tensor, c: float, eps: float) -> torch.Tensor:
        return ops.paged_diff_attention(q, self.layers[self._at], self.table, self.lengths, lam, weight, c, eps, scale=scale, window=window)
