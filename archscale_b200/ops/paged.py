"""Paged key-value cache and the attention of new tokens over it, for generation.

A cache holds the keys and values of G heads in pages of S tokens, elements ``(pages, G, S, D)`` (:func:`new_paged_cache`); pages of a sequence lie
anywhere in it: ``table[b, i]`` (int32) is the page of tokens ``i·S … i·S + S − 1`` of sequence b.  ``lengths[b]`` (int32) counts the tokens of a
sequence, *the new ones included*; of T rows of new tokens the first ``new_lengths[b]`` are real (all T without it), and row i sits at
position ``lengths[b] − new_lengths[b] + i``.  Tables and lengths stay on the device: no call waits for them, and a captured call follows their values.

    cache = ops.new_paged_cache(pages, G, 64, D)                     # or dtype=torch.float8_e4m3fn
    lengths += 1                                                     # one step of decoding; q, k, v: (B, 1, H | G, D)
    ops.paged_cache_write(cache, k, v, table, lengths)
    o = ops.paged_attention(q, cache, table, lengths)

* :func:`paged_cache_write` puts new keys and values into their slots, :func:`paged_cache_read` returns the tokens of each sequence as dense
  tensors, which :func:`~archscale_b200.ops.attention` takes.
* :func:`paged_attention` is ``o_i = Σ_j softmax_j(scale · q_i·k_j) v_j`` over the positions ``j`` up to the row's own, at most ``window[0]`` back,
  with the options of :func:`~archscale_b200.ops.attention` (grouped heads, window, sink, log-sum-exp).  Any number of new tokens is right; it is made
  for a few: keys and values are read once for every 16 rows (tokens times heads) of a group, or 8 of a pair of heads.  Queries in float32, and caches in
  float32 or of odd layouts, take a kernel that reads them once for each row.  Weights are good to 2⁻¹⁷, sums are in 32 bits.
* :func:`paged_diff_attention` is the same for pairs of heads ``(1, 2)``: ``a_i = softmax(q_i k_iᵀ) [v_1 | v_2]`` and
  ``y = RMSNorm(a_1 − λ a_2) · weight · c`` over the 2 D values of a pair, in fp32 up to the one rounding of y (the training layer rounds ``a_1`` and ``a_2``).

In e4m3 a head of one token has one power of two: with ``a = max |x|`` and ``e`` the smallest integer ≥ −127 with ``448 · 2^e ≥ a``,

    ``q = e4m3(x · 2^−e)``,  scale byte ``e + 127`` (float8_e8m0fnu),  ``x ≈ q · 2^e``

so that what is read back is a bf16 number; a head with an infinity or NaN reads back as NaN.

What is not there: a row past ``new_lengths[b]``, or whose position or window leaves it no key, gives zeros and a log-sum-exp of −∞ (with a
sink: the sink).  Positions before the first token or past the table are neither written nor seen, nor are pages outside the cache (they also
raise the status word of ``device_status()``); table entries behind the last token are not looked at.  Stale contents of a slot, infinities and NaN
among them, reach no row that does not see the slot.  Two tokens that are written to one slot in one call leave it undefined: a page that
several sequences share may be read by all and written by none (copy it first).  ``lengths`` below ``new_lengths`` drop the tokens before position 0.

None of these has gradients, on any device: with gradients enabled they refuse operands that ask for one, and operands with a forward-mode
tangent.  Under ``vmap`` and traces the PyTorch restatements (``*_ref``, also the CPU path and the test oracles) run.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional, Tuple

import torch

from . import backend
from .fp8_block import FP8, _FLOATS, _ext, _no_grad

E8M0 = torch.float8_e8m0fnu
MAX_HEAD = 256


class PagedCache(NamedTuple):
    """Keys and values ``(pages, heads, page size, head size)`` in bfloat16, float32 or float8_e4m3fn, any strides but a dense head; with
    float8_e4m3fn the scales ``(pages, heads, page size)`` in float8_e8m0fnu."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: Optional[torch.Tensor] = None
    v_scale: Optional[torch.Tensor] = None


def new_paged_cache(pages: int, heads: int, page_size: int, head_size: int, dtype: torch.dtype = torch.bfloat16, device=None) -> PagedCache:
    """A cache of zeros."""
    if dtype not in (*_FLOATS, FP8):
        raise TypeError(f"new_paged_cache: a cache holds bfloat16, float32 or float8_e4m3fn, got {dtype}")
    shape = (pages, heads, page_size, head_size)
    k, v = (torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
    if dtype != FP8:
        return PagedCache(k, v)
    return PagedCache(k, v, *(torch.zeros(shape[:3], dtype=torch.uint8, device=device).view(E8M0) for _ in range(2)))


# ------------------------------------------------------------------------------------------------ references
def _pow2(e: torch.Tensor) -> torch.Tensor:
    """2^e in fp32, e an int32 tensor from −127 on."""
    return torch.where(e > -127, (e + 127) << 23, torch.full_like(e, 1 << 22)).view(torch.float32)


def quantize_head_ref(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """x:(..., D) → (elements, scale bytes (...))."""
    x = x.float()
    top = x.abs().amax(-1)
    code = (((top.contiguous().view(torch.int32) + 0x1FFFFF) >> 23) - 8).clamp_min(0)
    finite = torch.isfinite(top)
    code = torch.where(finite, code, torch.zeros_like(code))
    x = torch.where(finite.unsqueeze(-1), x, torch.zeros_like(x))
    q = (x * ((254 - code) << 23).view(torch.float32).unsqueeze(-1)).to(FP8)
    return q, torch.where(finite, code, torch.full_like(code, 255)).to(torch.uint8)


def _head_values(q: torch.Tensor, scale: Optional[torch.Tensor]) -> torch.Tensor:
    if scale is None:
        return q.float()
    code = scale.to(torch.int32)
    s = torch.where(code == 255, torch.full(code.shape, math.nan, device=code.device), _pow2(code.clamp_max(254) - 127))
    return q.float() * s.unsqueeze(-1)


def _counts(lengths, new_lengths, T):
    n = torch.full_like(lengths, T) if new_lengths is None else new_lengths.clamp(0, T)
    return lengths.long(), n.long()


def _pages_of(cache: PagedCache, table: torch.Tensor, b: torch.Tensor, pos: torch.Tensor):
    """(page, slot, whether there is one) of positions of sequences."""
    S, cols = cache.k.shape[2], table.shape[1]
    inside = (pos >= 0) & (pos < cols * S)
    if cols == 0:
        return torch.zeros_like(pos), torch.zeros_like(pos), inside
    page = table.long()[b, (pos // S).clamp(0, cols - 1)]
    ok = inside & (page >= 0) & (page < cache.k.shape[0])
    return torch.where(ok, page, torch.zeros_like(page)), torch.where(ok, pos % S, torch.zeros_like(pos)), ok


def paged_cache_write_ref(cache, k, v, table, lengths, new_lengths=None) -> None:
    B, T = k.shape[:2]
    lengths, n = _counts(lengths, new_lengths, T)
    i = torch.arange(T, device=k.device).expand(B, T)
    b = torch.arange(B, device=k.device).unsqueeze(1).expand(B, T)
    page, slot, ok = _pages_of(cache, table, b, lengths.unsqueeze(1) - n.unsqueeze(1) + i)
    ok &= i < n.unsqueeze(1)
    page, slot = page[ok], slot[ok]
    for x, old, scale in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
        x = x[ok]
        if scale is None:
            old[page, :, slot] = x.to(old.dtype)
        else:
            q, code = quantize_head_ref(x)
            old.view(torch.uint8)[page, :, slot] = q.view(torch.uint8)
            scale.view(torch.uint8)[page, :, slot] = code


def _gather(cache: PagedCache, table: torch.Tensor, tokens: int):
    """fp32 (B, tokens, G, D) keys and values, and whether a token's slot exists (B, tokens)."""
    B = table.shape[0]
    pos = torch.arange(tokens, device=table.device).expand(B, tokens)
    b = torch.arange(B, device=table.device).unsqueeze(1).expand(B, tokens)
    page, slot, ok = _pages_of(cache, table, b, pos)
    out = []
    for x, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        if cache.k.shape[0] == 0:
            out.append(torch.zeros(B, tokens, x.shape[1], x.shape[3], device=x.device))
        elif scale is None:
            out.append(x[page, :, slot].float())
        else:
            out.append(_head_values(x.view(torch.uint8)[page, :, slot].view(FP8), scale.view(torch.uint8)[page, :, slot]))
    return (*out, ok)


def paged_cache_read_ref(cache, table, lengths, tokens: int, dtype=torch.bfloat16):
    k, v, ok = _gather(cache, table, tokens)
    live = (ok & (torch.arange(tokens, device=table.device) < lengths.unsqueeze(1)))[..., None, None]
    return tuple(torch.where(live, x, torch.zeros((), device=x.device)).to(dtype) for x in (k, v))


def _softmax_sum(q, k, v, seen, scale, sink):
    """q:(B,T,G,r,D) k:(B,L,G,D) v:(B,L,G,E) seen:(B,T,L), all fp32 → (out (B,T,G,r,E), log-sum-exp (B,T,G,r)).  A value that a row does not
    see adds nothing to it, whatever it is; one that it sees and that is not finite makes it NaN."""
    s = torch.einsum("btgrd,blgd->btgrl", q, k) * scale
    m = seen[:, :, None, None, :]
    s = s.masked_fill(~m, -math.inf)
    top = s.amax(-1, keepdim=True) if s.shape[-1] else torch.full((*s.shape[:-1], 1), -math.inf, device=s.device)
    if sink is not None:
        top = torch.maximum(top, sink.float().view(q.shape[2], q.shape[3], 1))
    ref = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(s - ref).masked_fill(~m, 0.0)
    total = p.sum(-1, keepdim=True)
    if sink is not None:
        total = total + torch.exp(sink.float().view(q.shape[2], q.shape[3], 1) - ref)
    good = torch.isfinite(v)
    o = torch.einsum("btgrl,blge->btgre", p, torch.where(good, v, torch.zeros_like(v)))
    bad = torch.einsum("btl,blge->btge", seen.to(p.dtype), (~good).to(p.dtype)) > 0
    o = torch.where(total == 0, torch.zeros_like(o), o / total).masked_fill(bad[:, :, :, None], math.nan)
    return o, (ref + torch.log(total)).squeeze(-1)


def _seen(lengths, new_lengths, T: int, L: int, window: int, ok) -> torch.Tensor:
    lengths, n = _counts(lengths, new_lengths, T)
    i, j = torch.arange(T, device=ok.device), torch.arange(L, device=ok.device)
    pos = (lengths - n).unsqueeze(1) + i                                  # (B, T)
    seen = (j <= pos.unsqueeze(2)) & ok.unsqueeze(1)
    if window >= 0:
        seen = seen & (j >= pos.unsqueeze(2) - window)
    return seen & (i < n.unsqueeze(1)).unsqueeze(2)


def _span(cache, table, lengths) -> int:
    """Tokens that any row can see."""
    room = table.shape[1] * cache.k.shape[2]
    return room if backend.transformed() or not lengths.numel() else max(0, min(int(lengths.max()), room))


def paged_attention_ref(q, cache, table, lengths, new_lengths=None, scale: Optional[float] = None, window: Tuple[int, int] = (-1, -1), sink=None,
                        return_lse: bool = False):
    B, T, H, D = q.shape
    G = cache.k.shape[1]
    k, v, ok = _gather(cache, table, _span(cache, table, lengths))
    seen = _seen(lengths, new_lengths, T, k.shape[1], window[0], ok)
    o, lse = _softmax_sum(q.float().reshape(B, T, G, H // G, D), k, v, seen, 1.0 / math.sqrt(D) if scale is None else scale, sink)
    if sink is not None:                                                  # rows that are not there have no sink either
        _, n = _counts(lengths, new_lengths, T)
        lse = lse.masked_fill((torch.arange(T, device=q.device) >= n.unsqueeze(1))[:, :, None, None], -math.inf)
    o = o.reshape(B, T, H, D).to(q.dtype)
    return (o, lse.reshape(B, T, H).transpose(1, 2).contiguous()) if return_lse else o


def paged_diff_attention_ref(q, cache, table, lengths, lam, weight, c: float, eps: float = 1e-5, new_lengths=None, scale: Optional[float] = None,
                             window: Tuple[int, int] = (-1, -1)):
    B, T, H, D = q.shape
    G = cache.k.shape[1]
    k, v, ok = _gather(cache, table, _span(cache, table, lengths))
    seen = _seen(lengths, new_lengths, T, k.shape[1], window[0], ok)
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    q = q.reshape(B, T, G // 2, H // G, 2, D)
    v = v.reshape(B, v.shape[1], G // 2, 2 * D)
    a1, a2 = (_softmax_sum(q[..., i, :].float(), k[:, :, i::2], v, seen, scale, None)[0] for i in range(2))
    a = a1 - lam.float() * a2
    y = a * torch.rsqrt(a.square().mean(-1, keepdim=True) + eps) * weight.float() * c
    _, n = _counts(lengths, new_lengths, T)
    y = y.masked_fill((torch.arange(T, device=q.device) >= n.unsqueeze(1))[:, :, None, None, None], 0.0)
    return y.reshape(B, T, H, D).to(q.dtype)


# ------------------------------------------------------------------------------------------------ checks
# The bindings check the operands of the kernels (and raise the same exceptions); these are for the restatements.
def _check(name: str, cache: PagedCache, table, lengths, new_lengths, batch: int) -> None:
    k, v = cache.k, cache.v
    if k.dim() != 4 or v.shape != k.shape:
        raise ValueError(f"{name}: keys and values of the cache must be (pages, heads, page size, head size) alike, got {tuple(k.shape)} and {tuple(v.shape)}")
    if v.dtype != k.dtype or k.dtype not in (*_FLOATS, FP8):
        raise TypeError(f"{name}: a cache holds bfloat16, float32 or float8_e4m3fn, got {k.dtype} and {v.dtype}")
    if any(t.shape[3] > 1 and t.stride(3) != 1 for t in (k, v)):
        raise ValueError(f"{name}: values of a head must be neighbours in the cache")
    scales = [s for s in (cache.k_scale, cache.v_scale) if s is not None]
    if len(scales) != (2 if k.dtype == FP8 else 0):
        raise ValueError(f"{name}: a float8_e4m3fn cache has scales for keys and values, others have none")
    if min(k.shape[1:]) < 1 or k.shape[3] > MAX_HEAD:
        raise ValueError(f"{name}: heads, page size and head size (at most {MAX_HEAD}) must be positive, got {tuple(k.shape)}")
    for s in scales:
        if s.dtype != E8M0:
            raise TypeError(f"{name}: scales must be float8_e8m0fnu, got {s.dtype}")
        if s.shape != k.shape[:3]:
            raise ValueError(f"{name}: scales must be {tuple(k.shape[:3])}, got {tuple(s.shape)}")
    for what, t in (("the page table", table), ("lengths", lengths), ("new_lengths", new_lengths)):
        if t is not None and t.dtype != torch.int32:
            raise TypeError(f"{name}: {what} must be int32, got {t.dtype}")
    if table.dim() != 2 or table.shape[0] != batch or (table.shape[1] > 1 and table.stride(1) != 1):
        raise ValueError(f"{name}: the page table must be ({batch}, pages of a sequence) with dense rows, got {tuple(table.shape)}")
    for what, t in (("lengths", lengths), ("new_lengths", new_lengths)):
        if t is not None and (t.shape != (batch,) or (batch > 1 and t.stride(0) != 1)):
            raise ValueError(f"{name}: {what} must be ({batch},) and dense, got {tuple(t.shape)}")
    _devices(name, k, v, *scales, table, lengths, new_lengths)


def _devices(name: str, like, *tensors) -> None:
    for t in tensors:
        if t is not None and t.device != like.device:
            raise ValueError(f"{name}: operands on {like.device} and {t.device}")


def _check_rows(name: str, what: str, x, cache: PagedCache) -> None:
    if x.dtype not in _FLOATS:
        raise TypeError(f"{name}: {what} must be bfloat16 or float32, got {x.dtype}")
    if x.dim() != 4:
        raise ValueError(f"{name}: {what} must be (batch, new tokens, heads, head size), got {tuple(x.shape)}")
    _devices(name, cache.k, x)


def _check_query(name: str, q, cache: PagedCache) -> None:
    _check_rows(name, "queries", q, cache)
    G, D = cache.k.shape[1], cache.k.shape[3]
    if q.shape[3] != D or q.shape[2] < 1 or q.shape[2] % G:
        raise ValueError(f"{name}: queries must be (batch, new tokens, a multiple of {G} heads, {D}), got {tuple(q.shape)}")


def _check_small(name: str, what: str, t, n: int, cache: PagedCache) -> None:
    if t.dtype not in _FLOATS:
        raise TypeError(f"{name}: {what} must be bfloat16 or float32, got {t.dtype}")
    if t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{name}: {what} must have {n} values, dense, got {tuple(t.shape)}")
    _devices(name, cache.k, t)


def _left(name: str, window) -> int:
    if len(window) != 2 or window[1] not in (0, -1):
        raise ValueError(f"{name}: a window is (keys back, 0): rows see no keys after their own position, got {tuple(window)}")
    return int(window[0])


def _kernel(cache: PagedCache) -> bool:
    return cache.k.is_cuda and not backend.transformed() and backend.use_cuda_kernel("paged", cache.k)


# ------------------------------------------------------------------------------------------------ operators
def paged_cache_write(cache: PagedCache, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor,
                      new_lengths: Optional[torch.Tensor] = None) -> PagedCache:
    """Puts the new tokens ``k``, ``v`` ``(B, T, G, D)`` (bfloat16 or float32, any strides) into their slots, converted to the cache's type, and
    returns the cache, which is changed in place."""
    name = "paged_cache_write"
    if _kernel(cache):
        _ext().paged_write(*cache, k, v, table, lengths, new_lengths)
        return cache
    _no_grad(name, cache.k, cache.v, k, v)
    _check(name, cache, table, lengths, new_lengths, k.shape[0] if k.dim() else 0)
    for what, x in (("keys", k), ("values", v)):
        _check_rows(name, what, x, cache)
    if k.shape != v.shape or k.shape[2] != cache.k.shape[1] or k.shape[3] != cache.k.shape[3]:
        raise ValueError(f"{name}: new keys and values must be (batch, new tokens, {cache.k.shape[1]}, {cache.k.shape[3]}), got {tuple(k.shape)} and {tuple(v.shape)}")
    if k.dtype != v.dtype:
        raise TypeError(f"{name}: new keys and values must be of one type, got {k.dtype} and {v.dtype}")
    if any(t is not None and t.shape[d] > 1 and t.stride(d) == 0 for t in cache for d in range(3)):
        raise ValueError(f"{name}: an expanded cache cannot be written")
    paged_cache_write_ref(cache, k, v, table, lengths, new_lengths)
    return cache


def paged_cache_read(cache: PagedCache, table: torch.Tensor, lengths: torch.Tensor, tokens: int,
                     dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    """The first ``tokens`` tokens of each sequence as dense keys and values ``(B, tokens, G, D)`` in ``dtype`` (bfloat16 or float32); zeros where a
    sequence has none."""
    name = "paged_cache_read"
    if dtype not in _FLOATS:
        raise TypeError(f"{name}: tokens are read as bfloat16 or float32, not as {dtype}")
    if _kernel(cache):
        return _ext().paged_read(*cache, table, lengths, tokens, dtype)
    _no_grad(name, cache.k, cache.v)
    _check(name, cache, table, lengths, None, table.shape[0] if table.dim() else 0)
    if tokens < 0:
        raise ValueError(f"{name}: the number of tokens cannot be negative")
    return paged_cache_read_ref(cache, table, lengths, tokens, dtype)


def paged_attention(q: torch.Tensor, cache: PagedCache, table: torch.Tensor, lengths: torch.Tensor, new_lengths: Optional[torch.Tensor] = None,
                    scale: Optional[float] = None, window: Tuple[int, int] = (-1, -1), sink: Optional[torch.Tensor] = None, return_lse: bool = False):
    """Attention of the new tokens ``q`` ``(B, T, H, D)`` (bfloat16 or float32) over the cache → ``(B, T, H, D)`` in q's type, and with
    ``return_lse`` the natural log-sum-exp ``(B, H, T)`` (fp32).  Query heads ``g·H/G …`` read head g of the cache.  ``scale``: 1/√D by default;
    ``window = (w, 0)``: at most w positions back; ``sink`` ``(H,)``: a logit of each head that adds to the denominator."""
    name = "paged_attention"
    left = _left(name, window)
    scale = 1.0 / math.sqrt(max(q.shape[-1], 1)) if scale is None else scale
    if _kernel(cache):
        out, lse = _ext().paged_attention(q, *cache, table, lengths, new_lengths, scale, left, sink, return_lse, None, None, 0.0, 0.0)
        return (out, lse) if return_lse else out
    _no_grad(name, q, cache.k, cache.v, sink)
    _check(name, cache, table, lengths, new_lengths, q.shape[0] if q.dim() else 0)
    _check_query(name, q, cache)
    if sink is not None:
        _check_small(name, "sink", sink, q.shape[2], cache)
    return paged_attention_ref(q, cache, table, lengths, new_lengths, scale, (left, 0), sink, return_lse)


def paged_diff_attention(q: torch.Tensor, cache: PagedCache, table: torch.Tensor, lengths: torch.Tensor, lam: torch.Tensor, weight: torch.Tensor,
                         c: float, eps: float = 1e-5, new_lengths: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                         window: Tuple[int, int] = (-1, -1)) -> torch.Tensor:
    """Differential attention of the new tokens over the cache.  Heads ``2p``, ``2p + 1`` of ``q`` ``(B, T, H, D)`` and of the cache are pairs; ``lam`` is
    a tensor of one value, ``weight`` the ``(2·D,)`` gain of the norm, ``c`` a constant gain → ``(B, T, H, D)``, pairs side by side."""
    name = "paged_diff_attention"
    left = _left(name, window)
    scale = 1.0 / math.sqrt(max(q.shape[-1], 1)) if scale is None else scale
    if _kernel(cache):
        return _ext().paged_attention(q, *cache, table, lengths, new_lengths, scale, left, None, False, lam, weight, c, eps)[0]
    _no_grad(name, q, cache.k, cache.v, lam, weight)
    _check(name, cache, table, lengths, new_lengths, q.shape[0] if q.dim() else 0)
    _check_query(name, q, cache)
    if cache.k.shape[1] % 2:
        raise ValueError(f"{name}: heads come in pairs, got {cache.k.shape[1]} of the cache")
    _check_small(name, "lam", lam, 1, cache)
    _check_small(name, "weight", weight, 2 * q.shape[3], cache)
    return paged_diff_attention_ref(q, cache, table, lengths, lam, weight, c, eps, new_lengths, scale, (left, 0))
