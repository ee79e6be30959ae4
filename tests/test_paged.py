"""Paged cache: writer, reader, attention and differential attention against the definitions in 64 bits, on the CPU and on the GPU."""
import math

import pytest
import torch

import paged_oracle as oracle
from archscale_b200 import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
FP8, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
BF16, F32 = torch.bfloat16, torch.float32


def half_step(t):
    return torch.finfo(t).eps / 2


def table_of(B, n, pages, g):
    return torch.randperm(pages, generator=g)[:B * n].to(torch.int32).view(B, n)


def filled(pages, G, S, D, dtype, g, device, order="groups"):
    """A cache with contents: keys with strong channels, values that differ in size.  ``order``: how it lies in memory."""
    k = torch.randn(pages, G, S, D, generator=g) * torch.exp(0.5 * torch.randn(G, 1, D, generator=g))
    v = torch.randn(pages, G, S, D, generator=g) * torch.exp(0.7 * torch.randn(pages, G, S, 1, generator=g))
    if dtype == FP8:
        (k, ks), (v, vs) = (ops.paged.quantize_head_ref(x) for x in (k, v))
        parts = [k, v, ks.view(E8M0), vs.view(E8M0)]
    else:
        parts = [k.to(dtype), v.to(dtype), None, None]
    parts = [t if t is None else t.to(device) for t in parts]
    if order == "tokens":                                  # [pages, S, G, D] in memory
        parts = [t if t is None else t.transpose(1, 2).contiguous().transpose(1, 2) for t in parts]
    elif order == "both":                                  # [pages, 2, S, G, D] in memory, keys and values side by side
        for i in (0, 2):
            if parts[i] is not None:
                u = lambda t: t.view(torch.uint8) if t.element_size() == 1 else t  # noqa: E731
                both = torch.stack([u(parts[i]).transpose(1, 2), u(parts[i + 1]).transpose(1, 2)], 1)
                parts[i], parts[i + 1] = (both[:, j].transpose(1, 2).view(parts[i].dtype) for j in range(2))
    elif order == "odd":                                   # rows that start anywhere
        for i in (0, 1):
            wide = torch.zeros(pages, G, S, D + 1, dtype=parts[i].dtype, device=device)
            wide[..., :D] = parts[i]
            parts[i] = wide[..., :D]
    return ops.PagedCache(*parts)


# ------------------------------------------------------------------------------------------------ writer and reader
WRITES = [
    # B, T, G, D, S, lengths, new_lengths
    (1, 1, 4, 128, 64, [1], None),
    (1, 1, 4, 128, 64, [700], None),
    (3, 5, 2, 64, 16, [5, 37, 64], None),
    (4, 7, 3, 124, 48, [7, 100, 3, 0], [7, 0, 3, 5]),      # nothing new, everything new, more new than tokens
    (2, 33, 1, 256, 16, [33, 70], [-4, 99]),               # counts outside 0 … T are held to it
    (2, 3, 2, 40, 5, [3, 11], None),
    (2, 2, 2, 1, 1, [2, 4], None),
    (1, 300, 20, 64, 128, [513], None),
    (2, 0, 4, 64, 16, [3, 4], None),
    (0, 3, 4, 64, 16, [], None),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, F32, FP8])
@pytest.mark.parametrize("src", [BF16, F32])
@pytest.mark.parametrize("case", range(len(WRITES)))
def test_write_and_read(case, src, dtype, device):
    B, T, G, D, S, lengths, new = WRITES[case]
    g = torch.Generator().manual_seed(case)
    n = max([-(-x // S) for x in lengths], default=0)
    cache = filled(B * n + 2, G, S, D, dtype, g, device, order=["groups", "tokens", "both", "odd"][case % 4])
    table = table_of(B, n, B * n + 2, g)
    k, v = ((torch.randn(B, T, G, D, generator=g) * torch.exp(3 * torch.randn(B, T, G, 1, generator=g))).to(src) for _ in range(2))
    want = [t if t is None else (t.view(torch.uint8) if t.element_size() == 1 else t).clone().cpu() for t in cache]
    for b in range(B):
        m = T if new is None else max(0, min(T, new[b]))
        for i in range(m):
            pos = lengths[b] - m + i
            if pos < 0:
                continue
            page, slot = int(table[b, pos // S]), pos % S
            for j, x in enumerate((k, v)):
                for h in range(G):
                    if dtype == FP8:
                        q, code, _ = oracle.head(x[b, i, h].double())
                        want[j][page, h, slot] = q.to(FP8).view(torch.uint8)
                        want[j + 2][page, h, slot] = code
                    else:
                        want[j][page, h, slot] = x[b, i, h].to(dtype)
    dev = lambda t: None if t is None else t.to(device)  # noqa: E731
    lens, news = torch.tensor(lengths, dtype=torch.int32), None if new is None else torch.tensor(new, dtype=torch.int32)
    got = ops.paged_cache_write(cache, dev(k), dev(v), dev(table), dev(lens), dev(news))
    assert got is cache
    for x, y in zip(cache, want):
        assert (x is None) == (y is None)
        if x is not None:
            x = x.cpu()
            x, y = (t.view(torch.uint8).view(FP8).float() if t.dtype in (FP8, torch.uint8) and y.dim() == 4 and dtype == FP8 else t for t in (x, y))
            if x.dtype == E8M0:
                x = x.view(torch.uint8)
            assert torch.equal(x, y)                       # every slot that was not written is as it was; −0 and 0 are one value
    tokens = n * S + 3
    for out in (BF16, F32):
        rk, rv = ops.paged_cache_read(cache, dev(table), dev(lens), tokens, out)
        assert rk.shape == rv.shape == (B, tokens, G, D) and rk.dtype == rv.dtype == out
        for b in range(B):
            pos, wk, wv = oracle.sequence(cache, table, b, lengths[b])
            assert len(pos) == max(0, lengths[b])
            for x, y in ((rk, wk), (rv, wv)):
                assert torch.equal(x[b, :len(pos)].cpu(), y.float().to(out)) and not x[b, len(pos):].any()


@pytest.mark.parametrize("device", DEVICES)
def test_scales_at_their_borders(device):
    """Maxima just at, below and above 448 · 2^e, zero heads, the smallest and largest numbers, infinities and NaN."""
    tops = [0.0, 448.0, 449.0, 447.0, 448.0 * 2 ** -20, 450.0 * 2 ** -20, 1.0, 1.75, 1.7578125, 2.0, 3e38, 1e-38, 2.0 ** -126, 2.0 ** -133, 2.0 ** -149, 1e-42]
    x = torch.zeros(1, len(tops), 1, 16)
    for i, a in enumerate(tops):
        x[0, i, 0] = torch.linspace(-1, 1, 16) * a
        x[0, i, 0, 5] = a
    x = torch.cat((x, x[:, 1:2].repeat(1, 3, 1, 1)), 1)
    x[0, -3, 0, 2], x[0, -2, 0, 3], x[0, -1, 0, 4] = math.inf, -math.inf, math.nan
    n = x.shape[1]
    cache = ops.new_paged_cache(2, 1, 32, 16, FP8, device)
    table, lengths = torch.tensor([[1]], dtype=torch.int32, device=device), torch.tensor([n], dtype=torch.int32, device=device)
    ops.paged_cache_write(cache, x.to(device), x.to(device), table, lengths)
    k, v = ops.paged_cache_read(cache, table, lengths, n, F32)
    for i in range(n):
        q, code, val = oracle.head(x[0, i, 0].double())
        for e, s, r in ((cache.k, cache.k_scale, k), (cache.v, cache.v_scale, v)):
            assert int(s.view(torch.uint8)[1, 0, i]) == code
            assert torch.equal(e[1, 0, i].float().cpu().double(), q)
            assert torch.equal(r[0, i, 0].cpu(), val.float()) if code != 255 else bool(r[0, i, 0].isnan().all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, FP8])
def test_tables_that_point_nowhere(device, dtype):
    """Pages outside the cache, positions past the table and before 0: nothing is written, nothing is read, the rest is right."""
    g = torch.Generator().manual_seed(3)
    cache = filled(4, 2, 4, 64, dtype, g, device)
    before = [t if t is None else t.clone() for t in cache]
    table = torch.tensor([[1, -1, 7], [4, 2, 1 << 30]], dtype=torch.int32, device=device)
    lengths = torch.tensor([14, 11], dtype=torch.int32, device=device)      # 12 positions have a place in the table
    k, v = (torch.randn(2, 14, 2, 64, generator=g).to(device) for _ in range(2))
    ops.paged_cache_write(cache, k, v, table, lengths)
    one = ops.PagedCache(*(t if t is None else t.clone() for t in before))
    for b, page, at in ((0, 1, 0), (1, 2, 4)):
        for j in range(4):
            i = at + j if b == 0 else at + j + 3                             # 14 rows for 11 tokens: the first three lie before position 0
            part = torch.tensor([[page]], dtype=torch.int32, device=device)
            ops.paged_cache_write(one, k[b:b + 1, i:i + 1], v[b:b + 1, i:i + 1], part, torch.tensor([j + 1], dtype=torch.int32, device=device))
    for x, y in zip(cache, one):
        assert x is None or torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    rk, rv = ops.paged_cache_read(cache, table, lengths, 16, F32)
    for b in range(2):
        pos, wk, wv = oracle.sequence(cache, table.cpu(), b, int(lengths[b]))
        assert pos.tolist() == ([0, 1, 2, 3] if b == 0 else [4, 5, 6, 7])
        for x, y in ((rk, wk), (rv, wv)):
            assert torch.equal(x[b, pos].cpu(), y.float())
            x[b, pos] = 0
            assert not x[b].any()
    if device == "cuda":
        ext = ops.backend.require_extension()
        assert ext.device_status() == 8
        ext.reset_device_status()


# ------------------------------------------------------------------------------------------------ attention
ATTN = {
    # B, T, H, G, D, S, lengths, new_lengths, window, sink
    "one_token": (1, 1, 4, 1, 64, 16, [1], None, -1, False),
    "two_heads": (2, 1, 8, 2, 128, 64, [65, 1], None, -1, False),
    "empty_sequence": (3, 1, 16, 4, 128, 64, [0, 300, 5], None, -1, False),
    "group_of_8": (2, 1, 16, 2, 128, 16, [130, 77], None, -1, True),
    "group_of_12": (2, 1, 24, 2, 64, 64, [257, 31], None, -1, False),
    "group_of_20": (1, 1, 20, 1, 128, 32, [100], None, -1, False),
    "drafts": (3, 4, 8, 2, 128, 16, [4, 61, 200], None, -1, False),
    "ragged_drafts": (4, 5, 6, 3, 64, 16, [9, 2, 0, 150], [5, 0, 3, 2], -1, True),
    "drafts_of_17_heads": (2, 9, 4, 2, 128, 16, [33, 90], [9, 7], 20, True),
    "window": (2, 1, 8, 2, 128, 64, [500, 40], None, 63, False),
    "window_drafts": (2, 6, 4, 4, 64, 48, [301, 6], None, 10, False),
    "window_zero": (2, 3, 4, 2, 64, 16, [50, 3], None, 0, True),
    "more_new_than_tokens": (2, 8, 4, 2, 64, 16, [3, 20], None, -1, True),
    "odd_head": (2, 3, 8, 2, 124, 48, [150, 49], None, -1, False),
    "head_of_40": (2, 2, 4, 2, 40, 7, [60, 8], None, -1, False),
    "head_of_66": (2, 1, 4, 2, 66, 16, [60, 8], None, -1, False),
    "head_of_1": (2, 1, 4, 2, 1, 3, [10, 3], None, -1, False),
    "head_of_256": (2, 2, 4, 2, 256, 32, [70, 129], None, -1, True),
    "pages_of_1": (2, 1, 4, 2, 64, 1, [70, 29], None, -1, False),
    "past_the_table": (2, 2, 4, 2, 64, 16, [70, 33], None, -1, False),
    "long": (2, 1, 4, 1, 128, 128, [3001, 1500], None, -1, False),
    "long_drafts": (2, 3, 8, 2, 64, 64, [2500, 700], None, 1500, True),
    "no_rows": (2, 0, 4, 2, 64, 16, [5, 6], None, -1, False),
    "no_sequences": (0, 1, 4, 2, 64, 16, [], None, -1, False),
}


def attn_inputs(case, cache_type, q_type, device, order="groups", seed=0):
    B, T, H, G, D, S, lengths, new, window, sink = ATTN[case]
    g = torch.Generator().manual_seed(seed + sum(map(ord, case)))
    n = max([-(-x // S) for x in lengths], default=0)
    pages = B * n + 2
    cache = filled(pages, G, S, D, cache_type, g, device, order)
    table = table_of(B, n, pages, g)
    if case == "past_the_table":
        table = table[:, :3].contiguous()
    q = (1.5 * torch.randn(B, T, H, D, generator=g)).to(q_type).to(device)
    s = torch.randn(H, generator=g).to(device) if sink else None
    ints = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    return q, cache, table.to(device), ints(lengths), ints(new), window, s


def attn_bound(q, cache, spread, L):
    """What an output may be off before its rounding, relative to the largest value.  A score of D products and a scale is rounded D + 2 times
    (2⁻²⁴ each, of at most Σ|q k|), and once more where log₂ e is folded in (of |s| ≤ Σ|q k|); its exponential is off by that and by 2⁻²¹ (exp2 in
    hardware: 2⁻²²; the rescaling by the maximum once more).  Numerator and denominator both count.  Sums of L terms are rounded L times.
    Weights enter the product rounded: over e4m3 to fp16, by half a step of 2⁻¹¹ at most; else as two halves in bf16, where the second, at most 2⁻⁸ of a
    weight, is off by 2⁻⁸ of itself.  Σ p |v| / Σ p is at most the largest value."""
    D = q.shape[-1]
    score = (D + 4) * 2.0 ** -24 * spread
    return 2 * (score + 2.0 ** -20) + 2 * L * 2.0 ** -24 + (2.0 ** -11 if cache.k.dtype == FP8 else 2.0 ** -16)


def visible_top(cache, table, lengths):
    top = 0.0
    for b in range(len(lengths)):
        _, _, v = oracle.sequence(cache, table.cpu(), b, int(lengths[b]))
        top = max(top, float(v.abs().max()) if v.numel() else 0.0)
    return top


def check_attn(q, cache, table, lengths, new, window, sink, scale=None):
    with torch.no_grad():
        out, lse = ops.paged_attention(q, cache, table, lengths, new, scale=scale, window=(window, 0), sink=sink, return_lse=True)
        alone = ops.paged_attention(q, cache, table, lengths, new, scale=scale, window=(window, 0), sink=sink)
    assert out.shape == q.shape and out.dtype == q.dtype and lse.shape == (q.shape[0], q.shape[2], q.shape[1]) and lse.dtype == F32
    assert torch.equal(out, alone)
    want, want_lse, spread = oracle.attention(q, cache, table.cpu(), lengths, new, scale, window, sink)
    L = max([0, *lengths.tolist()])
    rel = attn_bound(q, cache, spread, L)
    tol = half_step(q.dtype) * want.abs() + rel * visible_top(cache, table, lengths) * (1 + half_step(q.dtype))
    err = (out.double().cpu() - want).abs()
    assert bool((err <= tol).all()), float((err - tol).max())
    gone = want_lse == -math.inf
    assert bool((lse.cpu()[gone] == -math.inf).all()) and bool(torch.isfinite(lse.cpu()[~gone]).all())
    # the logarithm: as the sum, which is off by rel, and its own rounding of up to |lse| and of the maximum
    off = (lse.double().cpu() - want_lse)[~gone].abs()
    assert off.numel() == 0 or bool((off <= rel + 2.0 ** -21 + 2.0 ** -22 * want_lse[~gone].abs() + 2.0 ** -22 * spread).all())
    gone = gone.transpose(1, 2).to(out.device)
    assert not out[gone].any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("cache_type,q_type", [(BF16, BF16), (FP8, BF16), (F32, F32), (FP8, F32), (BF16, F32), (F32, BF16)])
@pytest.mark.parametrize("case", list(ATTN))
def test_attention(case, cache_type, q_type, device):
    check_attn(*attn_inputs(case, cache_type, q_type, device))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("cache_type", [BF16, FP8])
@pytest.mark.parametrize("order", ["tokens", "both", "odd"])
@pytest.mark.parametrize("case", ["group_of_8", "ragged_drafts", "odd_head"])
def test_attention_of_caches_in_any_order(case, order, cache_type, device):
    check_attn(*attn_inputs(case, cache_type, BF16, device, order))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("cache_type", [BF16, FP8])
def test_attention_of_sharp_and_flat_scores(cache_type, device):
    """Scores of hundreds, where one key takes all, a scale of zero, a negative one, and values whose scales lie 2^40 apart."""
    q, cache, table, lengths, new, window, sink = attn_inputs("drafts", cache_type, BF16, device)
    for scale in (8.0, 0.0, -0.3):
        check_attn(q, cache, table, lengths, new, window, sink, scale)
    for page in range(0, cache.v.shape[0], 2):
        if cache_type == FP8:
            codes = cache.v_scale.view(torch.uint8)
            codes[page] -= 40
        else:
            cache.v[page] *= 2.0 ** -40
    check_attn(q, cache, table, lengths, new, window, sink)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("case", ["group_of_8", "ragged_drafts"])
def test_queries_as_slices_of_a_projection(case, device):
    """Rows of heads that lie in a wider tensor, as the output of a fused projection does, and at odd offsets."""
    q, *rest = attn_inputs(case, BF16, BF16, device)
    B, T, H, D = q.shape
    want = ops.paged_attention(q, rest[0], rest[1], rest[2], rest[3])
    for off in (0, 8, 3):
        wide = torch.full((B, T, H * D + 64), math.nan, dtype=BF16, device=device)
        wide[..., off:off + H * D] = q.reshape(B, T, H * D)
        assert torch.equal(ops.paged_attention(wide[..., off:off + H * D].view(B, T, H, D), rest[0], rest[1], rest[2], rest[3]), want)
    moved = q.permute(3, 2, 0, 1).contiguous().permute(2, 3, 1, 0)          # values of a head far apart
    assert torch.equal(ops.paged_attention(moved, rest[0], rest[1], rest[2], rest[3]), want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("cache_type", [BF16, F32, FP8])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("case", ["drafts", "window_drafts", "drafts_of_17_heads", "odd_head", "empty_sequence"])
def test_stale_slots_reach_no_row(case, bad, cache_type, device):
    """Slots behind the last token, before every window, and of other pages hold infinities and NaN: bit for bit the same outputs.  What a later new
    token holds reaches no earlier one."""
    q, cache, table, lengths, new, window, sink = attn_inputs(case, cache_type, BF16 if cache_type != F32 else F32, device)
    S, T = cache.k.shape[2], q.shape[1]
    call = lambda c: ops.paged_attention(q, c, table, lengths, new, window=(window, 0), sink=sink, return_lse=True)  # noqa: E731
    want = call(cache)
    keep = torch.zeros(cache.k.shape[0], S, dtype=torch.bool)
    for b in range(len(lengths)):
        n = T if new is None else int(new[b])
        for j in range(0 if window < 0 else max(0, int(lengths[b]) - n - window), int(lengths[b])):
            keep[int(table[b, j // S]), j % S] = True
    stale = (~keep).to(device)

    def spoil(where):
        parts = [t if t is None else t.clone() for t in cache]
        for i in (0, 1):
            if cache_type == FP8:
                parts[i].view(torch.uint8).transpose(1, 2)[where] = 0x7F if bad != -math.inf else 0x00
                parts[i + 2].view(torch.uint8).transpose(1, 2)[where] = 255
            else:
                parts[i].transpose(1, 2)[where] = bad
        return ops.PagedCache(*parts)

    for x, y in zip(call(spoil(stale)), want):
        assert torch.equal(x, y)
    if T > 1:                                                # the last token of every sequence as well: only the rows that see it change
        for b in range(len(lengths)):
            if int(lengths[b]):
                stale[int(table[b, (int(lengths[b]) - 1) // S]), (int(lengths[b]) - 1) % S] = True
        out, lse = call(spoil(stale))
        for b in range(len(lengths)):
            n = T if new is None else int(new[b])
            if not int(lengths[b]) or not n:
                continue
            assert torch.equal(out[b, :n - 1], want[0][b, :n - 1]) and torch.equal(lse[b, :, :n - 1], want[1][b, :, :n - 1])
            assert not torch.isfinite(out[b, n - 1]).any()


# ------------------------------------------------------------------------------------------------ differential attention
DIFF = {
    # B, T, H, G, D, S, lengths, new_lengths, window
    "one_pair": (1, 1, 2, 2, 64, 16, [1], None, -1),
    "pairs_over_20": (2, 1, 40, 20, 64, 64, [70, 1], None, -1),
    "heads_of_128": (2, 1, 16, 4, 128, 64, [130, 300], None, -1),
    "empty_sequence": (3, 1, 8, 4, 64, 64, [0, 300, 5], None, -1),
    "drafts": (3, 4, 8, 2, 64, 16, [4, 61, 200], None, -1),
    "ragged_drafts": (4, 5, 12, 4, 64, 16, [9, 2, 0, 150], [5, 0, 3, 2], -1),
    "many_rows": (2, 9, 8, 2, 128, 16, [33, 90], [9, 7], 20),
    "window": (2, 1, 8, 4, 64, 64, [500, 40], None, 63),
    "more_new_than_tokens": (2, 8, 4, 2, 64, 16, [3, 20], None, -1),
    "odd_head": (2, 2, 4, 2, 62, 7, [60, 8], None, -1),
    "head_of_124": (2, 1, 4, 4, 124, 16, [60, 80], None, -1),
    "head_of_33": (2, 1, 4, 2, 33, 16, [60, 8], None, -1),
    "head_of_200": (1, 2, 4, 2, 200, 16, [60], None, -1),
    "long": (2, 1, 8, 2, 64, 128, [3001, 1500], None, -1),
    "no_rows": (2, 0, 4, 2, 64, 16, [5, 6], None, -1),
}


def diff_inputs(case, cache_type, q_type, device, order="groups"):
    B, T, H, G, D, S, lengths, new, window = DIFF[case]
    g = torch.Generator().manual_seed(sum(map(ord, case)))
    n = max([-(-x // S) for x in lengths], default=0)
    pages = B * n + 2
    cache = filled(pages, G, S, D, cache_type, g, device, order)
    table = table_of(B, n, pages, g).to(device)
    q = (1.5 * torch.randn(B, T, H, D, generator=g)).to(q_type).to(device)
    ints = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    lam, w = (0.3 + 0.1 * torch.randn(1, generator=g)).to(device), (1 + 0.2 * torch.randn(2 * D, generator=g)).to(device)
    return q, cache, table, ints(lengths), ints(new), window, lam, w


def check_diff(q, cache, table, lengths, new, window, lam, w, scale=None, c=0.4, eps=1e-5):
    with torch.no_grad():
        out = ops.paged_diff_attention(q, cache, table, lengths, lam, w, c, eps, new, scale=scale, window=(window, 0))
    assert out.shape == q.shape and out.dtype == q.dtype
    want, spread, low = oracle.diff_attention(q, cache, table.cpu(), lengths, lam, w, c, eps, new, scale, window)
    L = max([0, *lengths.tolist()])
    # a1 − λ a2 is off by a; its root mean square by no more, so that y is off by (a / rms) (1 + |y| / (w c)), and |y| ≤ w c √(2 D)
    a = attn_bound(q, cache, spread, L) * (1 + abs(float(lam))) * visible_top(cache, table, lengths)
    gain = float(w.float().abs().max()) * abs(c)
    size = want.abs()
    tol = half_step(q.dtype) * size + (a / low if math.isfinite(low) else 0) * (gain + size) * 1.1 + 2.0 ** -20 * size
    err = (out.double().cpu() - want).abs()
    assert bool((err <= tol).all()), float((err - tol).max())
    assert not out[(want == 0).all(-1).to(out.device)].any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("cache_type,q_type", [(BF16, BF16), (FP8, BF16), (F32, F32), (FP8, F32), (F32, BF16)])
@pytest.mark.parametrize("case", list(DIFF))
def test_diff_attention(case, cache_type, q_type, device):
    check_diff(*diff_inputs(case, cache_type, q_type, device))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("cache_type", [BF16, FP8])
@pytest.mark.parametrize("order", ["tokens", "both", "odd"])
def test_diff_attention_of_caches_in_any_order(order, cache_type, device):
    q, cache, table, lengths, new, window, lam, w = diff_inputs("ragged_drafts", cache_type, BF16, device, order)
    check_diff(q, cache, table, lengths, new, window, lam.bfloat16(), w.bfloat16())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("cache_type", [BF16, FP8])
@pytest.mark.parametrize("case", ["drafts", "many_rows", "empty_sequence"])
def test_diff_attention_stale_slots_reach_no_row(case, cache_type, device):
    q, cache, table, lengths, new, window, lam, w = diff_inputs(case, cache_type, BF16, device)
    S = cache.k.shape[2]
    call = lambda c: ops.paged_diff_attention(q, c, table, lengths, lam, w, 0.4, 1e-5, new, window=(window, 0))  # noqa: E731
    want = call(cache)
    keep = torch.zeros(cache.k.shape[0], S, dtype=torch.bool)
    last = torch.zeros_like(keep)
    for b in range(len(lengths)):
        n = q.shape[1] if new is None else int(new[b])
        for j in range(0 if window < 0 else max(0, int(lengths[b]) - n - window), int(lengths[b])):
            keep[int(table[b, j // S]), j % S] = True
            last[int(table[b, j // S]), j % S] = j == int(lengths[b]) - 1

    def spoil(where):
        parts = [t if t is None else t.clone() for t in cache]
        for i in (0, 1):
            if cache_type == FP8:
                parts[i + 2].view(torch.uint8).transpose(1, 2)[where.to(device)] = 255
                parts[i].view(torch.uint8).transpose(1, 2)[where.to(device)] = 0xFF
            else:
                parts[i].transpose(1, 2)[where.to(device)] = math.nan
        return ops.PagedCache(*parts)

    assert torch.equal(call(spoil(~keep)), want)
    if q.shape[1] > 1:
        out = call(spoil(~keep | last))
        for b in range(len(lengths)):
            n = q.shape[1] if new is None else int(new[b])
            if int(lengths[b]) and n:
                assert torch.equal(out[b, :n - 1], want[b, :n - 1]) and bool(out[b, n - 1].isnan().all())


@pytest.mark.parametrize("device", DEVICES)
def test_diff_attention_is_the_training_layer(device):
    """The last token of a sequence through the layer that trains: its a1 and a2 are rounded to bf16, the cached form's are not."""
    from archscale_b200.models.attention import DiffAttention
    g = torch.Generator().manual_seed(5)
    B, T, H, G, D = 2, 70, 8, 4, 64
    q, k, v = (torch.randn(B, T, h, D, generator=g).to(device).to(BF16) for h in (H, G, G))
    da = DiffAttention(D, 3, 0.125, (30, 0)).to(device)
    torch.manual_seed(0)
    da.reset_parameters()
    lam = torch.exp((da.lambda_q1 * da.lambda_k1).sum()) - torch.exp((da.lambda_q2 * da.lambda_k2).sum()) + da.lambda_init
    with torch.no_grad():
        want = da(q, k, v)[:, -3:].float()
        cache = ops.new_paged_cache(2 * B * 5, G, 16, D, BF16, device)
        table = torch.randperm(2 * B * 5, generator=g)[:B * 5].view(B, 5).to(torch.int32).to(device)
        lengths = torch.full((B,), T, dtype=torch.int32, device=device)
        ops.paged_cache_write(cache, k, v, table, lengths)
        got = ops.paged_diff_attention(q[:, -3:], cache, table, lengths, lam, da.subln.weight, 1 - da.lambda_init, 1e-5, scale=0.125, window=(30, 0))
    # a_i ≤ max|v|, each rounded twice at most (product in bf16 weights, result), λ rounded: 4 half steps of (1 + λ) max|v|, through a norm whose rms
    # is what 30 random values leave
    a = want / ((1 - da.lambda_init) * da.subln.weight.repeat(H // 2).view(H, D))
    rms = 1 / math.sqrt(31)
    tol = 4 * 2.0 ** -8 * (1 + float(lam)) * float(v.float().abs().max()) / rms * (1 + float(a.abs().max())) * (1 - da.lambda_init)
    assert float((got.float() - want).abs().max()) <= tol
    # and by far less on average: roundings of 2⁻⁹ relative at random against whole steps in one direction
    assert float((got.float() - want).norm() / want.norm()) <= 2.0 ** -6
