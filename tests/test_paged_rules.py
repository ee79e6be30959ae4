"""What the paged cache's operators refuse, on every device alike, and how they go with streams, graphs, traces and large caches."""
import math

import pytest
import torch

import paged_oracle as oracle
from archscale_b200 import ops
from test_paged import attn_inputs, check_attn, check_diff, diff_inputs, filled

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
FP8, E8M0, BF16, F32 = torch.float8_e4m3fn, torch.float8_e8m0fnu, torch.bfloat16, torch.float32


def operands(device, dtype=BF16):
    g = torch.Generator().manual_seed(0)
    cache = filled(6, 4, 16, 64, dtype, g, device)
    table = torch.tensor([[0, 2], [5, 1]], dtype=torch.int32, device=device)
    lengths = torch.tensor([20, 7], dtype=torch.int32, device=device)
    k, v = (torch.randn(2, 3, 4, 64, generator=g).to(device) for _ in range(2))
    q = torch.randn(2, 3, 8, 64, generator=g).to(device).to(BF16)
    lam, w = torch.full((1,), 0.3, device=device), torch.ones(128, device=device)
    return cache, table, lengths, k, v, q, lam, w


@pytest.mark.parametrize("device", DEVICES)
def test_operands_that_ask_for_gradients(device):
    cache, table, lengths, k, v, q, lam, w = operands(device)
    sink = torch.zeros(8, device=device)
    ask = lambda t: t.detach().clone().requires_grad_()  # noqa: E731
    calls = {
        "write": (lambda a, b: ops.paged_cache_write(cache, a, b, table, lengths), (k, v)),
        "write to": (lambda a: ops.paged_cache_write(cache._replace(k=a), k, v, table, lengths), (cache.k,)),
        "read": (lambda a: ops.paged_cache_read(cache._replace(v=a), table, lengths, 5), (cache.v,)),
        "attention": (lambda a, b, c, d: ops.paged_attention(a, ops.PagedCache(b, c), table, lengths, sink=d), (q, cache.k, cache.v, sink)),
        "diff": (lambda a, b, c: ops.paged_diff_attention(a, cache, table, lengths, b, c, 0.4), (q, lam, w)),
    }
    for name, (call, args) in calls.items():
        call(*args)
        for i in range(len(args)):
            some = [ask(t) if j == i else t for j, t in enumerate(args)]
            with pytest.raises(RuntimeError, match="has no gradients"):
                call(*some)
            with torch.no_grad():
                call(*some)


@pytest.mark.parametrize("device", DEVICES)
def test_forward_mode_tangents(device):
    from torch.autograd import forward_ad
    cache, table, lengths, k, v, q, lam, w = operands(device)
    with torch.no_grad(), forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: ops.paged_cache_write(cache, dual(k), v, table, lengths), lambda: ops.paged_attention(dual(q), cache, table, lengths),
                     lambda: ops.paged_diff_attention(q, cache, table, lengths, dual(lam), w, 0.4)):
            with pytest.raises(RuntimeError, match="has no gradients"):
                call()


@pytest.mark.parametrize("device", DEVICES)
def test_wrong_operands(device):
    cache, table, lengths, k, v, q, lam, w = operands(device)
    eight = operands(device, FP8)[0]
    wide = torch.zeros(6, 4, 16, 257, dtype=BF16, device=device)
    T, V = TypeError, ValueError
    half = lambda t: t.half()  # noqa: E731
    write = lambda c=cache, a=k, b=v, t=table, n=lengths, m=None: ops.paged_cache_write(c, a, b, t, n, m)  # noqa: E731
    read = lambda c=cache, t=table, n=lengths, x=5, d=BF16: ops.paged_cache_read(c, t, n, x, d)  # noqa: E731
    attn = lambda a=q, c=cache, t=table, n=lengths, **kw: ops.paged_attention(a, c, t, n, **kw)  # noqa: E731
    diff = lambda a=q, c=cache, l=lam, x=w, **kw: ops.paged_diff_attention(a, c, table, lengths, l, x, 0.4, **kw)  # noqa: E731
    odd = filled(6, 3, 16, 64, BF16, torch.Generator().manual_seed(0), device)
    wrong = [
        # types
        (T, lambda: write(a=half(k), b=half(v))), (T, lambda: write(a=k.bfloat16())), (T, lambda: read(d=torch.float16)), (T, lambda: attn(a=half(q))),
        (T, lambda: attn(t=table.long())), (T, lambda: attn(n=lengths.long())), (T, lambda: attn(new_lengths=lengths.long())), (T, lambda: read(n=lengths.float())),
        (T, lambda: attn(c=ops.PagedCache(half(cache.k), half(cache.v)))), (T, lambda: attn(c=cache._replace(v=cache.v.float()))),
        (T, lambda: read(c=eight._replace(k_scale=eight.k_scale.view(torch.uint8)))), (T, lambda: attn(sink=torch.zeros(8, device=device, dtype=torch.float16))),
        (T, lambda: diff(l=half(lam))), (T, lambda: ops.new_paged_cache(2, 2, 2, 2, torch.int8, device)),
        # shapes
        (V, lambda: write(a=k[0])), (V, lambda: write(a=k[:, :2])), (V, lambda: write(a=k[..., :32], b=v[..., :32])), (V, lambda: write(a=k[:, :, :2], b=v[:, :, :2])),
        (V, lambda: write(a=k[:1], b=v[:1])), (V, lambda: write(n=lengths[:1])), (V, lambda: write(m=lengths[:1])), (V, lambda: write(t=table[0])),
        (V, lambda: read(x=-1)), (V, lambda: read(c=cache._replace(v=cache.v[:5]))), (V, lambda: read(c=ops.PagedCache(cache.k[0], cache.v[0]))),
        (V, lambda: read(c=eight._replace(k_scale=None))), (V, lambda: read(c=cache._replace(k_scale=eight.k_scale))),
        (V, lambda: read(c=eight._replace(v_scale=eight.v_scale[:3]))), (V, lambda: read(c=ops.PagedCache(wide, wide))),
        (V, lambda: read(c=ops.PagedCache(cache.k.transpose(2, 3), cache.v.transpose(2, 3)))), (V, lambda: read(c=ops.PagedCache(cache.k[:, :0], cache.v[:, :0]))),
        (V, lambda: attn(a=q[:, :, :6])), (V, lambda: attn(a=q[..., :32])), (V, lambda: attn(a=q[0])), (V, lambda: attn(a=q[:1])), (V, lambda: attn(a=q[:, :, :0])),
        (V, lambda: attn(window=(3, 1))), (V, lambda: attn(window=(3,))), (V, lambda: attn(sink=torch.zeros(4, device=device))),
        (V, lambda: attn(t=torch.zeros(2, 4, dtype=torch.int32, device=device)[:, ::2])), (V, lambda: attn(n=torch.zeros(4, dtype=torch.int32, device=device)[::2])),
        (V, lambda: diff(c=odd, a=q[:, :, :6])), (V, lambda: diff(l=torch.zeros(2, device=device))), (V, lambda: diff(x=w[:64])), (V, lambda: diff(window=(-1, 5))),
        # a cache whose slots are one memory
        (V, lambda: write(c=ops.PagedCache(cache.k[:1].expand(6, -1, -1, -1), cache.v))),
    ]
    for i, (kind, call) in enumerate(wrong):
        with pytest.raises(kind):
            call()
            print("not refused:", i)
    expanded = ops.PagedCache(cache.k[:, :1].expand(-1, 4, -1, -1), cache.v[:, :1].expand(-1, 4, -1, -1))          # one head for all may be read
    dense = ops.PagedCache(expanded.k.contiguous(), expanded.v.contiguous())
    assert torch.equal(attn(c=expanded), attn(c=dense))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("field", ["k", "v", "k_scale", "v_scale"])
def test_expanded_parts_are_not_written(device, field):
    _, table, lengths, k, v, *_ = operands(device)
    cache = ops.new_paged_cache(6, 4, 8, 64, torch.float8_e4m3fn, device)
    whole = getattr(cache, field)
    wrong = cache._replace(**{field: whole[:, :, :1].expand(whole.shape)})
    with pytest.raises(ValueError, match="an expanded cache"):
        ops.paged_cache_write(wrong, k, v, table, lengths)
    ops.paged_cache_read(wrong, table, lengths, 4)


@pytest.mark.gpu
def test_operands_on_two_devices():
    cache, table, lengths, k, v, q, lam, w = operands("cuda")
    host = lambda t: t.cpu()  # noqa: E731
    for call in (lambda: ops.paged_cache_write(cache, host(k), host(v), table, lengths), lambda: ops.paged_cache_write(cache, k, v, host(table), lengths),
                 lambda: ops.paged_cache_read(cache, table, host(lengths), 4), lambda: ops.paged_attention(host(q), cache, table, lengths),
                 lambda: ops.paged_attention(q, cache._replace(v=host(cache.v)), table, lengths), lambda: ops.paged_attention(q, cache, table, lengths, host(lengths)),
                 lambda: ops.paged_diff_attention(q, cache, table, lengths, host(lam), w, 0.4), lambda: ops.paged_diff_attention(q, cache, table, lengths, lam, host(w), 0.4)):
        with pytest.raises(ValueError, match="operands on"):
            call()


@pytest.mark.parametrize("device", DEVICES)
def test_vmap_and_traces(device):
    cache, table, lengths, k, v, q, lam, w = operands(device)
    many = torch.stack((q, 2 * q, -q))
    with torch.no_grad():
        got = torch.vmap(lambda a: ops.paged_attention(a, cache, table, lengths))(many)
        for a, b in zip(got, many):
            want, _, spread = oracle.attention(b, cache, table.cpu(), lengths)
            assert float((a.double().cpu() - want).abs().max()) <= 2.0 ** -7 * float(cache.v.abs().max())
        traced = torch.jit.trace(lambda a, t, n: ops.paged_attention(a, cache, t, n), (q, table, lengths), check_trace=False)
        other = torch.tensor([3, 30], dtype=torch.int32, device=device)
        near = lambda x, y: float((x.float() - y.float()).abs().max()) <= 2.0 ** -7 * float(cache.v.abs().max())  # noqa: E731
        assert near(traced(many[1], table, other), ops.paged_attention(many[1], cache, table, other))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP8, F32])
def test_graphs_follow_lengths_and_tables(dtype):
    """Two captured steps that share nothing but the cache, replayed on two streams with other lengths, pages and tokens than at capture."""
    g = torch.Generator().manual_seed(0)
    cache = filled(64, 4, 16, 128, dtype, g, "cuda")
    qt = F32 if dtype == F32 else BF16
    graphs = []
    for i in range(2):
        st = dict(table=torch.randperm(64, generator=g)[:60].view(3, 20).to(torch.int32).cuda(), lengths=torch.tensor([1, 1, 1], dtype=torch.int32).cuda(),
                  q=torch.randn(3, 2, 16, 128, generator=g).to(qt).cuda())
        call = lambda st=st: ops.paged_attention(st["q"], cache, st["table"], st["lengths"], return_lse=True)  # noqa: E731
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        graphs.append((graph, st, out, torch.cuda.Stream(), call))
    for turn in range(6):
        for graph, st, *_ in graphs:
            st["table"].copy_(torch.randperm(64, generator=g)[:60].view(3, 20).to(torch.int32))
            st["lengths"].copy_(torch.randint(0, 321, (3,), generator=g).to(torch.int32))
            st["q"].copy_(torch.randn(3, 2, 16, 128, generator=g))
        torch.cuda.synchronize()
        for graph, _, _, stream, _ in graphs:
            with torch.cuda.stream(stream):
                for _ in range(3):
                    graph.replay()
        torch.cuda.synchronize()
        for graph, st, out, _, call in graphs:
            for x, y in zip(out, call()):
                assert torch.equal(x, y)
            check_attn(st["q"], cache, st["table"], st["lengths"], None, -1, None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP8])
def test_two_streams_at_once_and_repeats(dtype):
    """Calls on two streams give bit for bit what each gives alone; the split over CTAs is joined in a fixed order."""
    sets = []
    for i in range(2):
        g = torch.Generator().manual_seed(i)
        cache = filled(700, 4, 64, 128, dtype, g, "cuda")
        table = torch.randperm(700, generator=g)[:640].view(5, 128).to(torch.int32).cuda()
        lengths = torch.tensor([8192, 1, 5000, 0, 77], dtype=torch.int32).cuda()
        q = torch.randn(5, 1, 16, 128, generator=g).to(BF16).cuda()
        sets.append((q, cache, table, lengths))
    want = [ops.paged_attention(*s, return_lse=True) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for s, stream, out in zip(sets, streams, got):
            with torch.cuda.stream(stream):
                out.append(ops.paged_attention(*s, return_lse=True))
    torch.cuda.synchronize()
    for out, w in zip(got, want):
        for pair in out:
            assert torch.equal(pair[0], w[0]) and torch.equal(pair[1], w[1])
    check_attn(*sets[0], None, -1, None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP8])
def test_offsets_past_32_bits(dtype):
    """Pages whose elements lie more than 2^31 (and, in bytes, 2^32) behind the first."""
    size = 1 if dtype == FP8 else 2
    G, S, D = 2, 64, 128
    pages = (1 << 32) // (G * S * D * size) + 300 if dtype == BF16 else (1 << 31) // (G * S * D) + 300
    k, v = (torch.empty(pages, G, S, D, dtype=torch.uint8 if dtype == FP8 else dtype, device="cuda") for _ in range(2))
    cache = ops.PagedCache(k, v) if dtype == BF16 else ops.PagedCache(k.view(FP8), v.view(FP8), *(torch.zeros(pages, G, S, dtype=torch.uint8, device="cuda").view(E8M0)
                                                                                                 for _ in range(2)))
    g = torch.Generator().manual_seed(0)
    table = torch.stack((torch.arange(pages - 4, pages), torch.arange(4))).to(torch.int32).cuda()
    lengths = torch.tensor([200, 200], dtype=torch.int32, device="cuda")
    new = torch.randn(2, 200, G, D, generator=g).cuda()
    ops.paged_cache_write(cache, new, 2 * new, table, lengths)
    rk, rv = ops.paged_cache_read(cache, table, lengths, 200, F32)
    small = ops.new_paged_cache(8, G, S, D, dtype, "cuda")
    near = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    ops.paged_cache_write(small, new, 2 * new, near, lengths)
    sk, sv = ops.paged_cache_read(small, near, lengths, 200, F32)
    assert torch.equal(rk, sk) and torch.equal(rv, sv) and rk.abs().max() > 1
    q = torch.randn(2, 1, 8, D, generator=g).cuda().to(BF16)
    assert torch.equal(ops.paged_attention(q, cache, table, lengths), ops.paged_attention(q, small, near, lengths))
    lam, w = torch.full((1,), 0.3, device="cuda"), torch.ones(2 * D, device="cuda")
    assert torch.equal(ops.paged_diff_attention(q, cache, table, lengths, lam, w, 0.4), ops.paged_diff_attention(q, small, near, lengths, lam, w, 0.4))
    qf = q.float()                                          # the kernel that takes any type
    assert torch.equal(ops.paged_attention(qf, cache, table, lengths), ops.paged_attention(qf, small, near, lengths))


@pytest.mark.gpu
def test_nothing_is_written_beside_the_slots():
    """A cache, queries and outputs in the middle of larger memory: the bands around them stay as they were."""
    g = torch.Generator().manual_seed(0)
    room = torch.full((8, 6, 20, 96), 7.0, dtype=BF16, device="cuda")
    k, v = room[2:6, 1:3, 2:18, 16:80], room[2:6, 3:5, 2:18, 16:80]
    cache = ops.PagedCache(k, v)
    table = torch.tensor([[3, 0]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([21], dtype=torch.int32, device="cuda")
    x = torch.randn(1, 40, 2, 64, generator=g).cuda()
    new = torch.tensor([5], dtype=torch.int32, device="cuda")
    ops.paged_cache_write(cache, x, x + 1, table, lengths, new)
    want = torch.full_like(room, 7.0)
    for i in range(5):
        page, slot = int(table[0, (16 + i) // 16]), (16 + i) % 16
        want[2 + page, 1:3, 2 + slot, 16:80] = x[0, i].bfloat16()
        want[2 + page, 3:5, 2 + slot, 16:80] = (x[0, i] + 1).bfloat16()
    assert torch.equal(room, want)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [40, 700])
def test_many_new_tokens(T):
    """Whole chunks of a prompt at once: many tiles of rows, more than one launch takes."""
    B, H, G, D, S = 3, 8, 1, 64, 32
    g = torch.Generator().manual_seed(0)
    n = -(-900 // S)
    cache = filled(B * n, G, S, D, BF16, g, "cuda")
    table = torch.randperm(B * n, generator=g).view(B, n).to(torch.int32).cuda()
    lengths = torch.tensor([900, T, 333], dtype=torch.int32).cuda()
    new = torch.tensor([T, T, min(T, 300)], dtype=torch.int32).cuda()
    q = torch.randn(B, T, H, D, generator=g).to(BF16).cuda()
    out, lse = ops.paged_attention(q, cache, table, lengths, new, window=(100, 0), return_lse=True)
    rows = ops.paged_attention(q.float(), cache, table, lengths, new, window=(100, 0))          # a kernel of one row per CTA, without tiles
    top = float(cache.v.abs().max())
    assert float((out.float() - rows).abs().max()) <= (2.0 ** -8 + 2.0 ** -12) * top
    assert not out[2, int(new[2]):].any() and bool((lse[2, :, int(new[2]):] == -math.inf).all())
    pick = [0, 1, T // 2, T - 1]
    want, _, _ = oracle.attention(q[:1, pick[-1:]], cache, table[:1].cpu(), lengths[:1], window=100)
    assert float((out[:1, -1:].double().cpu() - want).abs().max()) <= (2.0 ** -8 + 2.0 ** -12) * top


@pytest.mark.gpu
def test_many_sequences():
    """More sequences than one launch takes, most of them empty."""
    B = 2500
    g = torch.Generator().manual_seed(0)
    cache = filled(64, 2, 16, 64, BF16, g, "cuda")
    table = torch.randint(0, 64, (B, 4), generator=g).to(torch.int32).cuda()
    lengths = (torch.randint(0, 65, (B,), generator=g) * (torch.rand(B, generator=g) < 0.3)).to(torch.int32).cuda()
    q = torch.randn(B, 1, 4, 64, generator=g).to(BF16).cuda()
    out = ops.paged_attention(q, cache, table, lengths)
    rows = ops.paged_attention(q.float(), cache, table, lengths)
    assert float((out.float() - rows).abs().max()) <= (2.0 ** -8 + 2.0 ** -12) * float(cache.v.abs().max())
    assert not out[lengths == 0].any()


@pytest.mark.gpu
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", [BF16, FP8])
def test_queries_that_are_not_finite(dtype, value):
    """A query with an infinity or NaN makes its own row not finite and no other."""
    q, cache, table, lengths, new, window, sink = attn_inputs("group_of_8", dtype, BF16, "cuda")
    want = ops.paged_attention(q, cache, table, lengths)
    bad = q.clone()
    bad[1, 0, 5, 9] = value
    out = ops.paged_attention(bad, cache, table, lengths)
    assert not torch.isfinite(out[1, 0, 5]).any()
    out[1, 0, 5] = want[1, 0, 5]
    assert torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("shift", [1e-30, 1e30])
@pytest.mark.parametrize("dtype", [BF16, FP8])
def test_queries_and_keys_of_any_size(dtype, shift):
    """Queries of 1e-30 against keys of 1e30 and the reverse: products of the order of one."""
    q, cache, table, lengths, new, window, sink = attn_inputs("two_heads", BF16, BF16, "cuda")
    q = (q.float() * shift).to(BF16)
    k = (cache.k.float() / shift).to(BF16)
    if dtype == FP8:
        (ke, ks), (ve, vs) = ops.paged.quantize_head_ref(k), ops.paged.quantize_head_ref(cache.v)
        cache = ops.PagedCache(ke, ve, ks.view(E8M0), vs.view(E8M0))
    else:
        cache = ops.PagedCache(k, cache.v)
    check_attn(q, cache, table, lengths, new, window, sink)


@pytest.mark.gpu
def test_parameters_of_differential_attention_in_bf16():
    q, cache, table, lengths, new, window, lam, w = diff_inputs("pairs_over_20", BF16, BF16, "cuda")
    check_diff(q, cache, table, lengths, new, window, lam.bfloat16(), w.bfloat16(), c=-1.5, eps=1e-2, scale=-0.2)
    check_diff(q, cache, table, lengths, new, window, lam.view(()), w, c=1.0)
