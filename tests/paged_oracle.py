"""The paged cache and its attentions from their definitions, in 64 bits, token by token, for the tests."""
import math

import torch

FP8 = torch.float8_e4m3fn


def exponent(a: float) -> int:
    """The smallest integer e ≥ −127 with 448 · 2^e ≥ a."""
    e = -127
    while 448.0 * 2.0 ** e < a:
        e += 1
    return e


def e4m3(v: torch.Tensor) -> torch.Tensor:
    """Nearest e4m3 value of |v| ≤ 448 (64 bits), ties to even: 3 bits after the leading one, spacing 2⁻⁹ below 2⁻⁶."""
    _, e = torch.frexp(v)
    step = torch.exp2((e - 1).clamp_min(-6).double() - 3)
    return torch.round(v / step) * step


def head(x: torch.Tensor):
    """(elements, scale byte, value) of one head (64 bits)."""
    a = float(x.abs().max())
    if not math.isfinite(a):
        return torch.zeros_like(x), 255, torch.full_like(x, math.nan)
    e = exponent(a)
    q = e4m3(x * 2.0 ** -e)
    return q, e + 127, q * 2.0 ** e


def value(cache, page: int, g: int, slot: int):
    """Key and value (64 bits) of one head of one slot."""
    out = []
    for x, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        y = x[page, g, slot].to(torch.float32).double().cpu()
        if s is not None:
            code = int(s.view(torch.uint8)[page, g, slot])
            y = y * (math.nan if code == 255 else 2.0 ** (code - 127))
        out.append(y)
    return out


def sequence(cache, table, b: int, length: int):
    """The tokens of a sequence that have a slot: (positions, keys (n, G, D), values)."""
    pages, G, S, D = cache.k.shape
    rows = table[b].tolist()
    pos = [j for j in range(max(0, min(length, len(rows) * S))) if 0 <= rows[j // S] < pages]
    where = torch.tensor([(rows[j // S], j % S) for j in pos], dtype=torch.long).reshape(-1, 2)
    out = []
    for x, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        y = x.cpu().view(torch.uint8 if s is not None else x.dtype)[where[:, 0], :, where[:, 1]]
        y = (y.view(FP8).float() if s is not None else y).double()
        if s is not None:
            code = s.cpu().view(torch.uint8)[where[:, 0], :, where[:, 1]].double()
            y = y * torch.where(code == 255, math.nan, torch.exp2(code - 127))[..., None]
        out.append(y)
    return torch.tensor(pos, dtype=torch.long), *out


def _rows(q, cache, table, lengths, new_lengths, window):
    """Of every row that is there: (b, t, visible keys, values (n, G, D))."""
    B, T = q.shape[:2]
    for b in range(B):
        n = T if new_lengths is None else max(0, min(T, int(new_lengths[b])))
        pos, k, v = sequence(cache, table, b, int(lengths[b]))
        for t in range(n):
            at = int(lengths[b]) - n + t
            see = pos <= at
            if window >= 0:
                see &= pos >= at - window
            yield b, t, k[see], v[see]


def attention(q, cache, table, lengths, new_lengths=None, scale=None, window=-1, sink=None):
    """(out, lse, spread): ``spread`` bounds Σ_d |q_d k_d| · scale, what the rounding of a score is relative to."""
    B, T, H, D = q.shape
    G = cache.k.shape[1]
    scale = 1 / math.sqrt(D) if scale is None else scale
    x = q.double().cpu()
    out, lse, spread = torch.zeros_like(x), torch.full((B, H, T), -math.inf, dtype=torch.float64), 0.0
    for b, t, k, v in _rows(q, cache, table, lengths, new_lengths, window):
        for h in range(H):
            g = h // (H // G)
            s = k[:, g] @ x[b, t, h] * scale
            if len(s):
                spread = max(spread, float((k[:, g].abs() @ x[b, t, h].abs()).max() * abs(scale)))
            every = s if sink is None else torch.cat((s, sink[h:h + 1].double().cpu()))
            lse[b, h, t] = torch.logsumexp(every, 0) if len(every) else -math.inf
            if len(s):
                out[b, t, h] = torch.softmax(every, 0)[:len(s)] @ v[:, g]
    return out, lse, spread


def diff_attention(q, cache, table, lengths, lam, weight, c, eps, new_lengths=None, scale=None, window=-1):
    """(y, spread, smallest rms of a1 − λ a2 over the rows that see a key)."""
    B, T, H, D = q.shape
    G = cache.k.shape[1]
    scale = 1 / math.sqrt(D) if scale is None else scale
    x, w, lam = q.double().cpu(), weight.double().cpu(), float(lam.double())
    out, spread, low = torch.zeros_like(x), 0.0, math.inf
    for b, t, k, v in _rows(q, cache, table, lengths, new_lengths, window):
        if not len(k):
            continue
        for p in range(H // 2):
            g = 2 * (p // (H // G))
            both = torch.cat((v[:, g], v[:, g + 1]), 1)
            a = []
            for i in range(2):
                spread = max(spread, float((k[:, g + i].abs() @ x[b, t, 2 * p + i].abs()).max() * abs(scale)))
                a.append(torch.softmax(k[:, g + i] @ x[b, t, 2 * p + i] * scale, 0) @ both)
            a = a[0] - lam * a[1]
            rms = math.sqrt(float(a.square().mean()) + eps)
            low = min(low, rms)
            out[b, t, 2 * p:2 * p + 2] = (a / rms * w * c).view(2, D)
    return out, spread, low
