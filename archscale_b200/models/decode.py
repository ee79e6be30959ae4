"""Key-value cache of a model during generation: one paged cache per attention call of a forward pass, and the tokens they hold.

The reference generates by re-running the whole prefix for every token (`eval.py:36-111`), which stays the default of
:meth:`archscale_b200.eval.ModelWrapper.generate`; with this a step computes its own tokens only.  Attention models are
covered: grouped, windowed, sink, gated, with QK-norm, differential, and the cross-attention of YOCO layers, which read the
cache of the layer that made their keys.
"""
from __future__ import annotations

from typing import List, Optional

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
    have the same number of tokens.  A call under ``torch.cuda.graph`` must not be the one that fills an empty cache, and its replays
    add to ``lengths`` on the device, not to ``tokens``."""

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
        self.batch, self.capacity, self.tokens = batch, capacity, 0
        self.table = torch.arange(batch * pages, dtype=torch.int32, device=device).view(batch, pages)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self.layers: List[ops.PagedCache] = [ops.new_paged_cache(batch * pages, cfg.n_query_groups, page_size, cfg.head_size, dtype or model.compute_dtype, device)
                                             for _ in range(layers)]
        self._at, self._open = -1, 0

    def begin(self, idx: torch.Tensor) -> int:
        """Before the first layer: room for the tokens; returns the position of the first one."""
        B, T = idx.shape
        if B != self.batch:
            raise ValueError(f"the cache holds {self.batch} sequences, got {B}")
        if self.tokens + T > self.capacity:
            raise ValueError(f"the cache holds {self.capacity} tokens: {self.tokens} are there, {T} more were given")
        if torch.is_grad_enabled():
            raise RuntimeError("a key-value cache has no gradients: call the model under torch.no_grad()")
        if self._open:                                             # the call before did not come to its end
            self.lengths -= self._open
        self.lengths += T
        self._at, self._open = -1, T
        return self.tokens

    def end(self, T: int) -> None:
        self.tokens += T
        self._open = 0

    @property
    def filling(self) -> bool:
        """Whether the tokens of this call are the first ones: attention over them alone."""
        return self.tokens == 0

    def write(self, k: torch.Tensor, v: torch.Tensor) -> None:
        """Keys and values (B, T, G, D) of the next attention layer; layers that only read use the last ones written."""
        self._at += 1
        ops.paged_cache_write(self.layers[self._at], k, v, self.table, self.lengths)

    def attend(self, q: torch.Tensor, scale: float, window, sink: Optional[torch.Tensor]) -> torch.Tensor:
        return ops.paged_attention(q, self.layers[self._at], self.table, self.lengths, scale=scale, window=window, sink=sink)

    def attend_diff(self, q: torch.Tensor, scale: float, window, lam: torch.Tensor, weight: torch.Tensor, c: float, eps: float) -> torch.Tensor:
        return ops.paged_diff_attention(q, self.layers[self._at], self.table, self.lengths, lam, weight, c, eps, scale=scale, window=window)
