"""``Linear``: an ``nn.Linear`` whose matmuls run the tcgen05 GEMM (or its MXFP8 variant)."""
from __future__ import annotations

import torch
import torch.nn as nn

from archscale_b200 import ops
from archscale_b200.ops import gemm


class Linear(nn.Linear):
    """Drop-in ``nn.Linear`` (same parameter names / state-dict keys).

    * bf16 CUDA inputs → ``ops.linear`` (hand-written GEMM for fwd, dgrad, wgrad);
    * ``mxfp8=True`` → block-scaled E4M3 GEMM with bf16 master weights
      (replaces the ``te.Linear`` swap of the reference, `precision.py:192-251`);
    * ``nvfp4=True`` → NVFP4 GEMM (e2m1 elements, E4M3 block scales; the ``--fp4`` recipe, `precision.py:92-96`),
      emulated in PyTorch off the GPU;
    * ``fp8_block=True`` → E4M3 GEMM with one fp32 scale per 128 elements (``ops.linear_fp8_block``), for weights of any size; after
      :func:`freeze_fp8_block` calls without gradients read the stored 8-bit weight (``ops.linear_fp8_weight``);
    * anything else (CPU, fp32) → ``F.linear``.
    The weight is cast to the activation dtype when they differ (fp32 masters, bf16 compute).
    """

    mxfp8: bool = False
    nvfp4: bool = False
    fp8_block: bool = False
    steering: bool = False      # the outputs are routing scores, decays, step sizes or a gate per head: never in 8-bit blocks
    fp8_stored = None           # StoredFP8 of a frozen layer
    widen: bool = False         # odd feature counts on operands widened to a multiple of 8 (``ops.gemm.linear_widened``)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        w, b = self.weight, self.bias
        g = getattr(w, "_fsdp_group", None)
        if g is not None and getattr(g, "ag_pending", False) and (self.mxfp8 or self.nvfp4 or self.fp8_block or not (
                w._fsdp_first and x.is_cuda and x.dtype == torch.bfloat16 and w.dtype == torch.bfloat16)):
            w._fsdp_engine.finish_pending_gather(g)
        if self.fp8_block:
            stored = self.stored_fp8()
            return ops.linear_fp8_block(x, w, b) if stored is None else ops.linear_fp8_weight(x, *stored, b)
        if w.dtype != x.dtype:
            w = w.to(x.dtype)
            b = b.to(x.dtype) if b is not None else None
        if self.nvfp4:
            from archscale_b200.ops import nvfp4
            return nvfp4.linear_nvfp4(x, w, b)
        if self.mxfp8 and x.is_cuda:
            from archscale_b200.ops import mxfp8
            return mxfp8.linear_mxfp8(x, w, b)
        if self.widen and b is None and gemm.widened_ok(x, w):
            return gemm.linear_widened(x, w)
        return ops.linear(x, w, b)

    def stored_fp8(self):
        """(elements, scales) of a frozen layer in a call without gradients, else None.  Raises when the weight was written since."""
        s = self.fp8_stored
        if s is None:
            return None
        if torch.is_grad_enabled():
            if self.weight.requires_grad:
                s.operands = None
            return None
        if not s.current(self.weight):
            raise RuntimeError("the weight of a frozen 8-bit layer has changed: call freeze_fp8_block(model) again")
        return s.operands

    plain_forward = forward     # what ``ops.gemm.plain_linear`` compares with: a replaced ``forward`` is never passed by


def apply_mxfp8(model: nn.Module, skip=("lm_head", "lc_proj")) -> int:
    """Switch every :class:`Linear` of ``model`` to the MXFP8 path, except modules whose name contains one of
    ``skip`` and layers whose dimensions are not multiples of 128 (the rule of `precision.py:192-251`, with
    the block-scaled kernel's granularity instead of 16).  Returns the number of layers switched."""
    n = 0
    for name, mod in model.named_modules():
        if isinstance(mod, Linear) and not any(s in name for s in skip) \
                and mod.in_features % 128 == 0 and mod.out_features % 128 == 0:
            mod.mxfp8 = True
            n += 1
    return n


def apply_nvfp4(model: nn.Module, skip=("lm_head", "lc_proj")) -> int:
    """Switch every :class:`Linear` of ``model`` to the NVFP4 path, with the same exclusions as :func:`apply_mxfp8` and
    the NVFP4 kernels' granularity (multiples of 256).  Returns the number of layers switched."""
    n = 0
    for name, mod in model.named_modules():
        if isinstance(mod, Linear) and not any(s in name for s in skip) \
                and mod.in_features % 256 == 0 and mod.out_features % 256 == 0:
            mod.nvfp4 = True
            n += 1
    return n


def apply_fp8_block(model: nn.Module, skip=("lm_head", "lc_proj")) -> int:
    """Switch every :class:`Linear` of ``model`` to 8-bit operands with an fp32 scale per 128 elements, except modules whose name
    contains one of ``skip`` and those that are ``steering``: few outputs that go into a softmax over experts, an exponential or a sigmoid
    per head, where an operand's error of 2⁻⁴ is one of the whole token (sizes alone keep them out of the MXFP8 path).  Returns the number
    of layers switched."""
    n = 0
    for name, mod in model.named_modules():
        if isinstance(mod, Linear) and not mod.steering and not any(s in name for s in skip):
            mod.fp8_block = True
            n += 1
    return n


class StoredFP8:
    """8-bit form of the weight of a frozen layer, and what shows that the weight is still the one it was made from: the parameter itself, its
    version counter and the memory it lies in, or, where an engine owns that memory (it gathers and frees it, and its optimizers write the
    shards), the engine's count of changes.  The memory is kept alive, so that no later weight can lie at the same address."""

    def __init__(self, weight: torch.Tensor, operands) -> None:
        from archscale_b200.parallel.fsdp import engine_of
        self.weight, self.operands, self.engine = weight, operands, engine_of(weight)
        self.memory = None if self.engine is not None else weight.detach()
        self.stamp = self._stamp()

    def _stamp(self):
        w = self.weight
        return (w._version, self.engine.params_version) if self.engine is not None else (w._version, w.data_ptr(), w.shape, w.stride(), w.dtype, w.device)

    def current(self, weight: torch.Tensor) -> bool:
        return weight is self.weight and self.stamp == self._stamp()

    def __reduce__(self):                               # copies and pickles of a frozen layer are frozen, unless its weight has changed
        return StoredFP8, (self.weight, self.operands if self.current(self.weight) else None)


@torch.no_grad()
def freeze_fp8_block(model: nn.Module, frozen: bool = True) -> int:
    """Store the 8-bit form of the weights of all ``fp8_block`` layers for calls without gradients (evaluation, generation), which otherwise
    quantise them every time; ``frozen=False`` drops it.  Returns the number of layers; a model without any (see :func:`apply_fp8_block`) is
    refused.

    Weights that change afterwards make such a call raise: by an operation on the parameter, a state dict, a move, new memory, or a step
    or load of the engine that shards the model.  What goes past PyTorch's version counters (in-place operations on ``weight.data``, NumPy views,
    kernels that are given the address) cannot be seen; freeze again after it.  A layer that is called with gradients, as it is in training,
    drops its stored form, so that the calls after it take the weights as they are then.

    Of a sharded model every rank has to make this call, since the weights are gathered."""
    from archscale_b200.parallel.fsdp import gathered
    n = 0
    for mod in model.modules():
        if isinstance(mod, Linear) and mod.fp8_block:
            mod.fp8_stored = None
            if frozen:
                if mod.weight.is_inference():
                    raise RuntimeError("freeze_fp8_block: weights made under torch.inference_mode() keep no version that shows whether they "
                                       "change; make them outside of it")
                with gathered(mod.weight):
                    q, _, scale = ops.quantize_fp8_weight(mod.weight)
                    mod.fp8_stored = StoredFP8(mod.weight, (q, scale))
            n += 1
    if frozen and not n:
        raise ValueError("freeze_fp8_block: no layer of the model is in 8-bit blocks; call apply_fp8_block(model) first")
    return n
