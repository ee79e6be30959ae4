"""Linear layers in 8-bit floating point with one fp32 scale per block of 128 (e4m3 elements).

A block is 128 neighbouring values of a row (activations, gradients) or a 128 × 128 tile (weights); the last one may be shorter.
With ``a = max(max|block|, 1e-30)``, every operation in fp32 and rounded once,

    ``scale = a / 448``,   ``q = e4m3(x · (448 / a))``,   ``x ≈ q · scale``

(:func:`quantize_fp8_block`, :func:`quantize_fp8_block_both`, :func:`quantize_fp8_weight`), and the product of two such operands is

    ``out[m, n] = Σ_b sa[m, b] · sb[n, b] · Σ_{k in b} a[m, k] · b[n, k]``                        (:func:`matmul_fp8_block`)

with the inner sums on the tensor cores and the outer ones in fp32.  One scale of a block may be as large as the other is small.  Where their
product is below 2⁻¹²⁶, or one of them below 2⁻¹⁰⁹ (the quantisers make none), the block may count as zero, and where the product is past the range of fp32 as infinite.  Any size is taken: no dimension has to be a multiple of 128.

* :func:`linear_fp8_block` trains: ``y = Q(x) Q(W)ᵀ``, ``dx = Q(dy) Q(W)``, ``dW = Qᵗ(dy)ᵀ Qᵗ(x)``, where ``Qᵗ`` takes its blocks along the
  tokens; the rounding itself has gradient one.  Weights stay bf16 / fp32 and are quantised in every call.
* :func:`linear_fp8_weight` serves weights that were quantised beforehand (``quantize_fp8_weight``, or a checkpoint's elements and
  scales), from one token on.
* :func:`add_rms_norm_fp8` is the block entry ``x = res + h_scale · h``, ``n = rmsnorm(x) · w`` with ``n`` delivered in this format (it is never
  rounded to 16 bits; an element is what ``n · 448 / a`` rounds to as a real number, which the formula in fp32 misses for about one value in ten
  thousand, those half way between two elements); :func:`add_rms_norm_linear_fp8` trains it with the layer behind it.  Its backward makes the transposed operand of
  the weight gradient from the residual stream, which is kept anyway, so that ``n`` itself is kept in no form.

Quantisers, product, stored layer and :func:`add_rms_norm_fp8` have no gradients, on any device: with gradients enabled they refuse operands that ask
for one (store weights under ``torch.no_grad()``), and operands with a forward-mode tangent.  Under ``vmap`` and ``torch.jit.trace`` they run as
PyTorch operators.  The layers that train are traced in the same way; forward-mode and functorch transforms raise.

Scales are returned as ``(rows, blocks)``; in memory the rows are the fast dimension, which is what the GEMM reads.  Elements
have rows of a multiple of 16 bytes (TMA); others are copied into such rows within the call.

The functions ending in ``_ref`` are plain PyTorch restatements used as the CPU path and as test oracles.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import backend

BLOCK, E4M3_MAX, BLOCK_FLOOR = 128, 448.0, 1e-30
FP8 = torch.float8_e4m3fn
_FLOATS = (torch.bfloat16, torch.float32)


# ------------------------------------------------------------------------------------------------ references
def _flat(x: torch.Tensor) -> torch.Tensor:
    """x:(..., C) → (rows, C), of no rows or no columns too."""
    return x if x.dim() == 2 else x.reshape(math.prod(x.shape[:-1]), x.shape[-1])


def _to(x: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """``x.to(dtype)``; in a trace as a copy, since the fuser of ``torch.jit`` writes code for it that names an e4m3 type CUDA does not have."""
    return x.to(dtype) if torch._C._get_tracing_state() is None else torch.empty_like(x, dtype=dtype).copy_(x)


def _padded(x: torch.Tensor, rows: int, cols: int) -> torch.Tensor:
    return torch.nn.functional.pad(x, (0, -x.shape[1] % cols, 0, -x.shape[0] % rows))


def _factors(amax: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(scale, 448 / a).  Both are divisions of tensors: with a Python number torch multiplies by a rounded reciprocal."""
    a = amax.clamp_min(BLOCK_FLOOR)
    top = torch.full_like(a, E4M3_MAX)
    return a / top, top / a


def quantize_ref(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    R, C = x.shape
    blocks = (C + BLOCK - 1) // BLOCK
    xb = _padded(x.float(), 1, BLOCK).reshape(R, blocks, BLOCK)
    scale, u = _factors(xb.abs().amax(-1))
    return _to(xb * u.unsqueeze(-1), FP8).reshape(R, blocks * BLOCK)[:, :C].contiguous(), scale


def quantize_weight_ref(w: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    N, K = w.shape
    wb = _padded(w.float(), BLOCK, BLOCK)
    nb, kb = wb.shape[0] // BLOCK, wb.shape[1] // BLOCK
    wb = wb.view(nb, BLOCK, kb, BLOCK)
    scale, u = _factors(wb.abs().amax((1, 3)))
    return _to(wb * u.view(nb, 1, kb, 1), FP8).view(nb * BLOCK, kb * BLOCK)[:N, :K].contiguous(), scale


def dequantize_ref(q: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Values of elements with one scale per row and block, or per 128 × 128 tile."""
    R, C = q.shape
    s = scale.to(dtype)
    if s.shape[0] != R:
        s = s.repeat_interleave(BLOCK, 0)[:R]
    return _to(q, dtype) * s.repeat_interleave(BLOCK, 1)[:, :C]


def matmul_fp8_block_ref(a, a_scale, b, b_scale, bias=None, out_dtype=torch.bfloat16, acc=None):
    y = dequantize_ref(a, a_scale) @ dequantize_ref(b, b_scale).t()
    if bias is not None:
        y = y + bias.float()
    return acc.add_(y) if acc is not None else y.to(out_dtype)


def _norm_ref(res, h, weight, eps, h_scale, stream_dtype):
    x = res.float()
    if h is not None:
        x = (x + h_scale * h.float()).to(stream_dtype)
    xf = x.float()
    rstd = torch.rsqrt(xf.square().mean(-1, keepdim=True) + eps)
    return (x if h is not None else res), rstd, xf * rstd * weight.float()


def add_rms_norm_fp8_ref(res, h, weight, eps: float = 1e-5, h_scale: float = 1.0, stream_dtype: Optional[torch.dtype] = None):
    x, _, n = _norm_ref(res, h, weight, eps, h_scale, _stream(res, stream_dtype))
    q, scale = quantize_ref(_flat(n))
    return x, q, scale


# ------------------------------------------------------------------------------------------------ checks
# The bindings check the operands of the kernels (and raise the same exceptions); these are for the restatements.
def _stream(res: torch.Tensor, stream_dtype: Optional[torch.dtype]) -> torch.dtype:
    return res.dtype if stream_dtype is None else stream_dtype


def _stream_code(stream_dtype: Optional[torch.dtype]) -> int:
    if stream_dtype is not None and stream_dtype not in _FLOATS:
        raise TypeError(f"a residual stream is kept in bfloat16 or float32, not in {stream_dtype}")
    return -1 if stream_dtype is None else int(stream_dtype is torch.bfloat16)


def _need_float(name: str, **tensors) -> None:
    for what, t in tensors.items():
        if t is not None and t.dtype not in _FLOATS:
            raise TypeError(f"{name}: {what} must be bfloat16 or float32, got {t.dtype}")


def _need_matrix(name: str, x: torch.Tensor) -> None:
    if x.dim() != 2:
        raise ValueError(f"{name}: a matrix is needed, got shape {tuple(x.shape)}")
    _need_float(name, x=x)


def _kernel(x: torch.Tensor) -> bool:
    """Transforms and traces see the restatements, whose operators they know."""
    return x.is_cuda and not backend.transformed() and backend.use_cuda_kernel("fp8_block", x)


def _no_grad(name: str, *tensors) -> None:
    """A call that has no gradients must not cut a graph silently (the bindings check the operands of the kernels)."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{name} has no gradients: call it under torch.no_grad(), or use the training form")
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{name} has no gradients, nor forward-mode tangents")


def _ext():
    backend.count_launch()
    return backend.require_extension()


# ------------------------------------------------------------------------------------------------ quantisers
def quantize_fp8_block(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """x:(R,C) → (elements (R,C), scales (R, ⌈C/128⌉)), blocks along the rows."""
    if _kernel(x):
        return tuple(_ext().fp8_quantize(x, 1))
    _no_grad("quantize_fp8_block", x)
    _need_matrix("quantize_fp8_block", x)
    return quantize_ref(x)


def quantize_fp8_block_t(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """x:(R,C) → (elements (C,R), scales (C, ⌈R/128⌉)) of the transposed matrix, blocks along the original columns."""
    if _kernel(x):
        return tuple(_ext().fp8_quantize(x, 2))
    _no_grad("quantize_fp8_block_t", x)
    _need_matrix("quantize_fp8_block_t", x)
    return quantize_ref(x.t())


def quantize_fp8_block_both(x: torch.Tensor):
    """:func:`quantize_fp8_block` and :func:`quantize_fp8_block_t` from one read of x: (q, scale, q_t, scale_t)."""
    if _kernel(x):
        return tuple(_ext().fp8_quantize(x, 3))
    _no_grad("quantize_fp8_block_both", x)
    _need_matrix("quantize_fp8_block_both", x)
    return (*quantize_ref(x), *quantize_ref(x.t()))


def quantize_fp8_weight(w: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """w:(N,K) → (elements (N,K), the same transposed (K,N), scales (⌈N/128⌉, ⌈K/128⌉) of 128 × 128 tiles)."""
    if _kernel(w):
        return tuple(_ext().fp8_quantize(w, 4))
    _no_grad("quantize_fp8_weight", w)
    _need_matrix("quantize_fp8_weight", w)
    q, scale = quantize_weight_ref(w)
    return q, q.t().contiguous(), scale


# ------------------------------------------------------------------------------------------------ product
def matmul_fp8_block(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor, bias: Optional[torch.Tensor] = None,
                     out_dtype: torch.dtype = torch.bfloat16, acc: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``a:(M,K) · b:(N,K)ᵀ (+ bias)``, each operand with scales per row and block of 128, ``(rows, ⌈K/128⌉)``, or per 128 × 128 tile,
    ``(⌈rows/128⌉, ⌈K/128⌉)`` → (M,N) in ``out_dtype``; with ``acc`` (fp32) the product is added to it in place.  ``a`` may have more leading
    dimensions than one (M: their product), which the result then has too."""
    if out_dtype not in _FLOATS:
        raise TypeError(f"matmul_fp8_block: out_dtype must be bfloat16 or float32, got {out_dtype}")
    if _kernel(a):
        return _ext().gemm_fp8_block(a, a_scale, b, b_scale, bias, out_dtype is torch.float32, acc)
    _no_grad("matmul_fp8_block", a, a_scale, b, b_scale, bias, acc)
    if a.dtype != FP8 or b.dtype != FP8:
        raise TypeError(f"matmul_fp8_block: operands must be float8_e4m3fn, got {a.dtype} and {b.dtype}")
    if a.dim() < 2 or b.dim() != 2 or a.shape[-1] != b.shape[1]:
        raise ValueError(f"matmul_fp8_block: contraction lengths differ: {tuple(a.shape)} and {tuple(b.shape)}")
    lead, a = a.shape[:-1], _flat(a)
    blocks = (a.shape[1] + BLOCK - 1) // BLOCK
    for what, q, s in (("a_scale", a, a_scale), ("b_scale", b, b_scale)):
        if s.dtype != torch.float32 or s.dim() != 2 or s.shape[1] != blocks or s.shape[0] not in (q.shape[0], (q.shape[0] + BLOCK - 1) // BLOCK):
            raise ValueError(f"matmul_fp8_block: {what} must be float32 ({q.shape[0]} or {(q.shape[0] + BLOCK - 1) // BLOCK}, {blocks}), "
                             f"got {s.dtype} {tuple(s.shape)}")
    if bias is not None and (bias.shape != (b.shape[0],) or bias.dtype not in _FLOATS):
        raise ValueError(f"matmul_fp8_block: bias must be ({b.shape[0]},) in bfloat16 or float32, got {bias.dtype} {tuple(bias.shape)}")
    if acc is not None and (acc.dtype != torch.float32 or acc.shape != (a.shape[0], b.shape[0])):
        raise ValueError(f"matmul_fp8_block: acc must be float32 ({a.shape[0]}, {b.shape[0]}), got {acc.dtype} {tuple(acc.shape)}")
    y = matmul_fp8_block_ref(a, a_scale, b, b_scale, bias, out_dtype, acc)
    return y if len(lead) == 1 or acc is not None else y.view(*lead, b.shape[0])


Quantised = Tuple[torch.Tensor, torch.Tensor]


def linear_fp8_weight(x: Union[torch.Tensor, Quantised], weight: torch.Tensor, scale: torch.Tensor, bias: Optional[torch.Tensor] = None,
                      out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``x · Wᵀ (+ bias)`` with stored elements ``weight:(N,K)`` and scales of 128 × 128 tiles.  ``x:(..., K)`` is quantised here, or is the
    pair (elements, scales) of :func:`add_rms_norm_fp8` / :func:`quantize_fp8_block` with any leading dimensions of the elements.  It has
    no gradients and refuses operands that ask for one."""
    if not isinstance(x, torch.Tensor):
        return matmul_fp8_block(x[0], x[1], weight, scale, bias, out_dtype or torch.bfloat16)
    dtype = out_dtype or x.dtype
    if dtype not in _FLOATS:
        raise TypeError(f"linear_fp8_weight: results are bfloat16 or float32, not {dtype}")
    if _kernel(x):
        backend.count_launch(2)
        return backend.require_extension().linear_fp8_stored(x, weight, scale, bias, dtype is torch.float32)
    _no_grad("linear_fp8_weight", x, scale, bias)
    q, s = quantize_fp8_block(_flat(x))
    y = matmul_fp8_block(q, s, weight, scale, bias, dtype)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], weight.shape[0])


# ------------------------------------------------------------------------------------------------ training
# CUDA operands go through the autograd nodes of the bindings (``csrc/bindings_fp8.inc``); these are the same on the restatements.
def _layer_backward(gy2, w_t, w_scale, x_t, weight, want_x, x_dtype, want_w):
    """(dx | None, dW | None); dW goes into ``main_grad`` where the weight carries one.  ``x_t``: (elements, scales) of xᵀ."""
    main_grad = getattr(weight, "main_grad", None)
    dx = matmul_fp8_block(*quantize_fp8_block(gy2), w_t, w_scale.t(), out_dtype=x_dtype) if want_x else None
    dw = matmul_fp8_block(*quantize_fp8_block_t(gy2), *x_t, out_dtype=weight.dtype, acc=main_grad) if want_w else None
    return dx, (None if main_grad is not None else dw)


class _LinearFP8Fn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
        x2 = _flat(x)
        wq, w_t, w_scale = quantize_fp8_weight(weight)
        q, scale = quantize_fp8_block(x2)
        need_w = bool(ctx.needs_input_grad) and ctx.needs_input_grad[1]
        ctx.save_for_backward(w_t, w_scale, *(quantize_fp8_block_t(x2) if need_w else ()))
        ctx.weight, ctx.x_shape, ctx.x_dtype = weight, x.shape, x.dtype
        ctx.bias_dtype = None if bias is None else bias.dtype
        return matmul_fp8_block(q, scale, wq, w_scale, bias, x.dtype).view(*x.shape[:-1], weight.shape[0])

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        w_t, w_scale, *x_t = ctx.saved_tensors
        gy2 = _flat(gy)
        need_x, need_w, need_b = ctx.needs_input_grad
        dx, dw = _layer_backward(gy2, w_t, w_scale, x_t, ctx.weight, need_x, ctx.x_dtype, need_w)
        return (None if dx is None else dx.view(ctx.x_shape)), dw, (gy2.sum(0, dtype=torch.float32).to(ctx.bias_dtype) if need_b else None)


def _check_layer(name, cols, weight, bias=None):
    if weight.dim() != 2 or weight.shape[1] != cols:
        raise ValueError(f"{name}: weight must be (out, {cols}), got {tuple(weight.shape)}")
    _need_float(name, weight=weight, bias=bias)
    if bias is not None and bias.shape != (weight.shape[0],):
        raise ValueError(f"{name}: bias must be ({weight.shape[0]},), got {tuple(bias.shape)}")


def linear_fp8_block(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x · weightᵀ (+ bias)`` with x:(..., K) and weight:(N, K) quantised in the call; trains (see the head of this file)."""
    if _kernel(x):
        backend.count_launch(3)
        return backend.require_extension().linear_fp8(x, weight, bias)
    _need_float("linear_fp8_block", x=x)
    _check_layer("linear_fp8_block", x.shape[-1], weight, bias)
    return backend.apply(_LinearFP8Fn, x, weight, bias)


# ------------------------------------------------------------------------------------------------ residual addition + RMSNorm
def _check_norm(name, res, h, weight, stream_dtype):
    _need_float(name, res=res, weight=weight)
    if weight.shape != (res.shape[-1],):
        raise ValueError(f"{name}: the norm's weight must be ({res.shape[-1]},), got {tuple(weight.shape)}")
    if h is not None and (h.shape != res.shape or h.dtype != torch.bfloat16):
        raise ValueError(f"{name}: the branch must be bfloat16 {tuple(res.shape)}, got {h.dtype} {tuple(h.shape)}")
    if stream_dtype not in _FLOATS or (stream_dtype == torch.bfloat16 and res.dtype != torch.bfloat16):
        raise TypeError(f"{name}: a {res.dtype} residual stream cannot be kept in {stream_dtype}")


def _norm_kernel(res, h, weight, eps, h_scale, stream_dtype, want_rstd):
    """(x of the shape of res, elements (rows, C), scales, 1 / rms (rows,))."""
    C = res.shape[-1]
    if not _kernel(res) or not 1 <= C <= 32768:
        _check_norm("add_rms_norm_fp8", res, h, weight, _stream(res, stream_dtype))
        x, rstd, n = _norm_ref(res, h, weight, eps, h_scale, _stream(res, stream_dtype))
        return (x, *quantize_ref(_flat(n)), rstd.reshape(-1))
    return _ext().add_rmsnorm_fp8(res, h, weight, eps, h_scale, _stream_code(stream_dtype), want_rstd)


def add_rms_norm_fp8(res: torch.Tensor, h: Optional[torch.Tensor], weight: torch.Tensor, eps: float = 1e-5, h_scale: float = 1.0,
                     stream_dtype: Optional[torch.dtype] = None):
    """``x = res + h_scale · h`` (fp32, kept in ``stream_dtype``, by default the type of ``res``; without ``h`` x is ``res``) and ``rmsnorm(x) · weight`` as
    elements and scales: (x of the shape of res, elements (rows, C), scales (rows, ⌈C/128⌉)).  It has no gradients and refuses operands that
    ask for one: training goes through :func:`add_rms_norm_linear_fp8`."""
    _no_grad("add_rms_norm_fp8", res, h, weight)
    x, q, scale, _ = _norm_kernel(res, h, weight, eps, h_scale, stream_dtype, False)
    return x, q, scale


def _norm_backward_ref(gx, dn, x, weight, rstd, h_scale, want_h):
    """Formula of the norm's gradients in fp32: (d_res fp32, d_h | None, d_weight fp32)."""
    xhat = x.float() * rstd.view(-1, 1)
    t = dn.float() * weight.float()
    d = rstd.view(-1, 1) * (t - xhat * (t * xhat).mean(-1, keepdim=True))
    if gx is not None:
        d = d + gx.float()
    return d, ((h_scale * d).to(torch.bfloat16) if want_h else None), (dn.float() * xhat).sum(0)


class _AddNormLinearFP8Fn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, res, h, norm_weight, weight, bias, eps, h_scale, stream_dtype):
        x, q, s, rstd = _norm_kernel(res, h, norm_weight, eps, h_scale, stream_dtype, True)
        wq, w_t, w_scale = quantize_fp8_weight(weight)
        ctx.save_for_backward(x, rstd, norm_weight, w_t, w_scale)
        ctx.weight, ctx.shape, ctx.res_dtype, ctx.h_scale, ctx.has_h = weight, res.shape, res.dtype, h_scale, h is not None
        ctx.bias_dtype = None if bias is None else bias.dtype
        ctx.set_materialize_grads(False)
        y = matmul_fp8_block(q, s, wq, w_scale, bias, torch.bfloat16)
        return (x if h is not None else res.view_as(res)), (y if res.dim() == 2 else y.view(*res.shape[:-1], weight.shape[0]))

    @staticmethod
    @once_differentiable
    def backward(ctx, gx, gy):
        x, rstd, norm_weight, w_t, w_scale = ctx.saved_tensors
        C = ctx.shape[-1]
        x = _flat(x)
        need_res, need_h, need_nw, need_w, need_b = ctx.needs_input_grad[:5]
        need_n = need_res or need_h or need_nw
        gx2 = None if gx is None else _flat(gx)
        dn = dw = db = dres = dh = dnw = None
        if gy is not None:
            gy2 = _flat(gy)
            if need_n or need_w:
                x_t = quantize_ref((x.float() * rstd.view(-1, 1) * norm_weight.float()).t()) if need_w else None
                dn, dw = _layer_backward(gy2, w_t, w_scale, x_t, ctx.weight, need_n, torch.float32, need_w)
            if need_b:
                db = gy2.sum(0, dtype=torch.float32).to(ctx.bias_dtype)
        if dn is None:                                           # the layer behind the norm was not used
            dres = gx2
            dh = (ctx.h_scale * gx2.float()).to(torch.bfloat16) if need_h and gx2 is not None else None
        else:
            dres, dh, dnw = _norm_backward_ref(gx2, dn, x, norm_weight, rstd, ctx.h_scale, need_h)
        return (dres.to(ctx.res_dtype).view(ctx.shape) if need_res and dres is not None else None,
                dh.view(ctx.shape) if need_h and dh is not None else None,
                dnw.to(norm_weight.dtype) if need_nw and dnw is not None else None, dw, db, None, None, None)


def add_rms_norm_linear_fp8(res: torch.Tensor, h: Optional[torch.Tensor], norm_weight: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5,
                            h_scale: float = 1.0, stream_dtype: Optional[torch.dtype] = None, bias: Optional[torch.Tensor] = None):
    """``x = res + h_scale · h``, ``y = Q(rmsnorm(x) · norm_weight) · Q(weight)ᵀ (+ bias)`` → (x, y in bf16), with gradients of all inputs."""
    if _kernel(res) and 1 <= res.shape[-1] <= 32768:
        backend.count_launch(3)
        return tuple(backend.require_extension().add_norm_linear_fp8(res, h, norm_weight, weight, eps, h_scale, _stream_code(stream_dtype), bias))
    stream_dtype = _stream(res, stream_dtype)
    _check_norm("add_rms_norm_linear_fp8", res, h, norm_weight, stream_dtype)
    _check_layer("add_rms_norm_linear_fp8", res.shape[-1], weight, bias)
    return backend.apply(_AddNormLinearFP8Fn, res, h, norm_weight, weight, bias, eps, h_scale, stream_dtype)
