"""Sequences whose keys are divided over CTAs: every form of the kernel that joins their parts, several launches of one call, against the definitions in 64 bits."""
import math

import pytest
import torch

import paged_oracle as oracle
from archscale_b200 import ops
from paged_plan import workspace
from test_paged import BF16, FP8, check_attn, check_diff, filled, table_of

pytestmark = pytest.mark.gpu


def ragged(B, top):
    """Lengths from 0 to top, the ends and what lies around a chunk of keys among them."""
    g = torch.Generator().manual_seed(B + top)
    some = [top, 0, 1, 63, 64, 65, 127, 128, 129, top - 1][:B]
    return some + torch.randint(0, top + 1, (B - len(some),), generator=g).tolist()


# name: (diff, lengths, T, H, G, D, S, window, sink, warps of the second kernel that share a row)
CASES = {
    "few_long": (False, [9000, 33, 5000], 1, 8, 2, 128, 64, -1, True, 16),
    "few_long_64": (False, [9000, 0, 5000], 1, 4, 2, 64, 64, -1, False, 16),
    "few_long_256": (False, [9000, 1, 6300], 1, 4, 2, 256, 64, -1, False, 16),
    "few_long_124": (False, [9000, 33, 5000], 1, 8, 2, 124, 48, -1, False, 16),
    "few_long_drafts": (False, [9000, 3, 5000], 4, 12, 2, 128, 64, -1, True, 16),
    "few_long_drafts_window": (False, [9900, 3, 8800], 4, 12, 2, 128, 64, 8700, True, 16),
    "few_long_drafts_256": (False, [9000, 3], 3, 8, 2, 256, 64, -1, False, 16),
    "some": (False, ragged(17, 1500), 1, 8, 4, 128, 64, -1, True, 4),
    "some_64": (False, ragged(25, 1500), 1, 12, 4, 64, 16, -1, False, 4),
    "some_124": (False, ragged(17, 1500), 1, 8, 4, 124, 48, -1, False, 4),
    "some_256": (False, ragged(31, 900), 1, 4, 2, 256, 64, -1, False, 4),
    "some_drafts": (False, ragged(15, 1500), 5, 8, 4, 128, 16, 1000, True, 4),
    "many": (False, ragged(64, 800), 1, 16, 4, 128, 64, -1, False, 1),
    "many_40": (False, ragged(64, 800), 1, 8, 4, 40, 16, -1, True, 1),
    "many_256": (False, ragged(50, 800), 1, 4, 4, 256, 64, -1, False, 1),
    "many_drafts": (False, ragged(40, 700), 4, 12, 4, 64, 64, 300, True, 1),
    "pairs_few_long": (True, [9000, 33, 5000], 1, 8, 4, 64, 64, -1, False, 16),
    "pairs_few_long_128": (True, [9000, 33, 5000], 1, 8, 2, 128, 64, -1, False, 16),
    "pairs_few_long_drafts": (True, [9000, 33], 4, 8, 2, 128, 64, -1, False, 16),
    "pairs_some": (True, ragged(40, 1000), 1, 8, 4, 64, 64, -1, False, 4),
    "pairs_some_60": (True, ragged(40, 1000), 1, 8, 4, 60, 48, -1, False, 4),
    "pairs_some_128": (True, ragged(41, 900), 1, 8, 4, 128, 64, -1, False, 4),
    "pairs_some_drafts": (True, ragged(24, 900), 3, 12, 4, 64, 16, 600, False, 4),
    "pairs_many": (True, ragged(80, 500), 1, 16, 8, 64, 64, -1, False, 1),
    "pairs_many_drafts_128": (True, ragged(80, 500), 3, 8, 8, 128, 64, 200, False, 1),
}


def second_kernel(diff, B, T, H, G):
    """Warps that share a row there: 16 or 4 where the device's 32 warps of an SM hold that many for every row of every item."""
    per = H // G * T
    tile = (4 if diff else 8) * (1 if per <= (4 if diff else 8) else 2)
    rows = B * -(-per // tile) * (G // 2 if diff else G) * tile
    return next(w for w in (16, 4, 1) if w == 1 or rows * w <= 32 * torch.cuda.get_device_properties(0).multi_processor_count)


@pytest.mark.parametrize("dtype", [BF16, FP8])
@pytest.mark.parametrize("case", list(CASES))
def test_parts_of_sequences(case, dtype):
    diff, lengths, T, H, G, D, S, window, sink, warps = CASES[case]
    g = torch.Generator().manual_seed(sum(map(ord, case)))
    B, n = len(lengths), -(-max(lengths) // S)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert second_kernel(diff, B, T, H, G) == warps and workspace(B, T, H, G, D, S, n, window, diff, dtype == FP8, sms) > 0
    pages = B * n + 2 if B < 30 else 300                                # the larger batches share pages
    cache = filled(pages, G, S, D, dtype, g, "cuda")
    table = (table_of(B, n, pages, g) if B < 30 else torch.randint(0, pages, (B, n), generator=g).to(torch.int32)).cuda()
    q = (1.5 * torch.randn(B, T, H, D, generator=g)).to(BF16).cuda()
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    new = torch.randint(0, T + 1, (B,), generator=g).to(torch.int32).cuda() if T > 1 else None
    if diff:
        lam, w = torch.full((1,), 0.3, device="cuda"), (1 + 0.2 * torch.randn(2 * D, generator=g)).cuda()
        check_diff(q, cache, table, lens, new, window, lam, w)
    else:
        check_attn(q, cache, table, lens, new, window, torch.randn(H, generator=g).cuda() if sink else None)


def near_rows(out, rows, cache):
    # a rounding to bf16 and what both sums leave (weights of two halves, 2⁻²¹, L · 2⁻²³ of at most 3000 terms)
    return float((out.float() - rows).abs().max()) <= (2.0 ** -8 + 2.0 ** -11) * float(cache_top(cache))


def cache_top(cache):
    v = cache.v.float()
    return (v if cache.v_scale is None else v * cache.v_scale.float().unsqueeze(-1)).abs().max()


@pytest.mark.parametrize("diff", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP8])
def test_more_sequences_than_a_launch_takes(dtype, diff):
    """2500 sequences of several chunks: three launches, which use one workspace in turn."""
    B, H, G, D, S, n = 2500, 4, 2, 64, 16, 40
    g = torch.Generator().manual_seed(0)
    cache = filled(64, G, S, D, dtype, g, "cuda")
    table = torch.randint(0, 64, (B, n), generator=g).to(torch.int32).cuda()
    lengths = (torch.randint(0, n * S + 1, (B,), generator=g) * (torch.rand(B, generator=g) < 0.7)).to(torch.int32).cuda()
    q = torch.randn(B, 1, H, D, generator=g).to(BF16).cuda()
    assert workspace(B, 1, H, G, D, S, n, -1, diff, dtype == FP8) > 0
    pick = [0, 1023, 1024, 2047, 2048, 2499]
    if diff:
        lam, w = torch.full((1,), 0.3, device="cuda"), torch.ones(2 * D, device="cuda")
        call = lambda at: ops.paged_diff_attention(q[at], cache, table[at], lengths[at], lam, w, 0.4)  # noqa: E731
        check_diff(q[pick], cache, table[pick], lengths[pick], None, -1, lam, w)
    else:
        call = lambda at: ops.paged_attention(q[at], cache, table[at], lengths[at])  # noqa: E731
        check_attn(q[pick], cache, table[pick], lengths[pick], None, -1, None)
        assert near_rows(call(slice(None)), ops.paged_attention(q.float(), cache, table, lengths), cache)
    out = call(slice(None))
    assert torch.equal(out, call(slice(None))) and not out[lengths == 0].any()
    top = 1.0 if diff else float(cache_top(cache))
    for at in (slice(0, 700), slice(900, 1500), slice(2000, 2500)):         # other shares, other orders of the sums: a step of bf16 at most
        size = out[at].float().abs().clamp_min(2.0 ** -6 * top)
        assert bool(((call(at).float() - out[at].float()).abs() <= 2.0 ** -6 * size).all())


@pytest.mark.parametrize("dtype", [BF16, FP8])
def test_more_tiles_of_rows_than_a_launch_takes(dtype):
    """A prompt part of 2100 tokens with 8 query heads on one key head: 1050 tiles of 16 rows, over up to 3000 keys each."""
    T, H, G, D, S, L = 2100, 8, 1, 64, 64, 3000
    g = torch.Generator().manual_seed(1)
    n = -(-L // S)
    cache = filled(2 * n, G, S, D, dtype, g, "cuda")
    table = table_of(2, n, 2 * n, g).cuda()
    lengths, new = torch.tensor([L, 2500], dtype=torch.int32).cuda(), torch.tensor([T, 1300], dtype=torch.int32).cuda()
    q = torch.randn(2, T, H, D, generator=g).to(BF16).cuda()
    assert workspace(2, T, H, G, D, S, n, -1, False, dtype == FP8) > 0
    out, lse = ops.paged_attention(q, cache, table, lengths, new, return_lse=True)
    rows, row_lse = ops.paged_attention(q.float(), cache, table, lengths, new, return_lse=True)
    assert near_rows(out, rows, cache)
    there = torch.isfinite(row_lse)
    assert torch.equal(there, torch.isfinite(lse)) and float((lse - row_lse)[there].abs().max()) <= 2.0 ** -9
    assert not out[1, 1300:].any() and bool((lse[1, :, 1300:] == -math.inf).all())
    pick = [0, 1, 2047, 2048, 2099]                                            # around the border of the launches
    for t in pick:
        want, _, _ = oracle.attention(q[:1, t:t + 1], cache, table[:1].cpu(), torch.tensor([L - T + t + 1]))
        assert float((out[:1, t:t + 1].double().cpu() - want).abs().max()) <= (2.0 ** -8 + 2.0 ** -11) * float(cache_top(cache))
