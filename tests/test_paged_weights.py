"""Weights of the attention over caches in e4m3 keep what 32 bits hold: outputs are those of the definition up to their own rounding."""
import math

import pytest
import torch

import paged_oracle as oracle
from archscale_b200 import ops
from test_paged import BF16, FP8, filled, half_step, table_of

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]

CASES = {
    # T, H, G, D, S, lengths, window
    "heads_of_128": (1, 16, 4, 128, 16, [40, 3, 7, 21], -1),
    "heads_of_64": (1, 4, 2, 64, 16, [9, 33], -1),
    "drafts": (4, 16, 2, 128, 16, [12, 31], 9),
    "odd_head": (3, 8, 4, 124, 7, [20, 5], -1),
    "heads_of_256": (1, 4, 2, 256, 16, [30, 4], -1),
}


def inputs(case, device):
    T, H, G, D, S, lengths, window = CASES[case]
    g = torch.Generator().manual_seed(7)
    B, n = len(lengths), -(-max(lengths) // S)
    cache = filled(B * n + 1, G, S, D, FP8, g, device)
    q = torch.randn(B, T, H, D, generator=g).to(BF16).to(device)
    return q, cache, table_of(B, n, B * n + 1, g).to(device), torch.tensor(lengths, dtype=torch.int32, device=device), window, 0.02 / math.sqrt(D), g


def bound(q, cache, spread, lengths):
    """Scores are near zero, so that their own roundings ((D + 4) of 2⁻²⁴ each, of at most Σ|q k|) are small beside those of weights.  An exponential is off by
    2⁻²⁰ with its rescaling.  A weight is two halves in fp16: the second, at most 2⁻¹¹ of it, is off by 2⁻¹¹ of itself, and by 2⁻²⁵ of a largest weight of 2¹⁴ where
    it is subnormal.  Sums of L terms are rounded L times.  Numerator and denominator both count."""
    L = max(lengths.tolist())
    return 2 * ((q.shape[-1] + 4) * 2.0 ** -24 * spread + 2.0 ** -20) + 2 * L * 2.0 ** -24 + 2.0 ** -22 + L * 2.0 ** -39


def largest(cache, table, lengths):
    return max(float(oracle.sequence(cache, table.cpu(), b, int(n))[2].abs().max()) for b, n in enumerate(lengths))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("case", list(CASES))
def test_attention(case, device):
    q, cache, table, lengths, window, scale, _ = inputs(case, device)
    got = ops.paged_attention(q, cache, table, lengths, scale=scale, window=(window, 0))
    want, _, spread = oracle.attention(q, cache, table.cpu(), lengths, None, scale, window)
    tol = half_step(BF16) * want.abs() + bound(q, cache, spread, lengths) * largest(cache, table, lengths) * (1 + half_step(BF16))
    assert bool(((got.double().cpu() - want).abs() <= tol).all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("case", ["heads_of_128", "heads_of_64", "drafts"])
def test_diff_attention(case, device):
    q, cache, table, lengths, window, scale, g = inputs(case, device)
    D = q.shape[-1]
    lam, w = torch.full((1,), 0.25, device=device), (1 + 0.2 * torch.randn(2 * D, generator=g)).to(device)
    got = ops.paged_diff_attention(q, cache, table, lengths, lam, w, 0.5, 1e-5, scale=scale, window=(window, 0))
    want, spread, low = oracle.diff_attention(q, cache, table.cpu(), lengths, lam, w, 0.5, 1e-5, None, scale, window)
    # a1 − λ a2 is off by a, its root mean square by no more: y by (a / rms) (w c + |y|); the norm's own roundings are 2⁻²⁰ of y
    a = bound(q, cache, spread, lengths) * 1.25 * largest(cache, table, lengths)
    tol = half_step(BF16) * want.abs() + 1.01 * a / low * (0.5 * float(w.abs().max()) + want.abs()) + 2.0 ** -20 * want.abs()
    assert bool(((got.double().cpu() - want).abs() <= tol).all())
