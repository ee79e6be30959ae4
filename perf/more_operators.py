"""Decoding from a paged key-value cache, as cases that a timing tool can run.

The cache holds keys and values of G heads in pages of S tokens, elements ``[pages, G, S, D]``; ``table[b, i]`` is the page of tokens ``i·S … i·S + S − 1``
of sequence b and ``lengths[b]`` counts its tokens, the newest ones included.  The i-th of ``n`` new tokens sits at position ``lengths[b] − n + i``.
Elements are bf16, or e4m3 with one power of two per token and head, held as its biased exponent in a byte (e8m0):

    e = smallest integer with 448 · 2^e ≥ max |x| (never below −127),    q = e4m3(x · 2^−e),    x ≈ q · 2^e

A case is a plain dict; its ``op`` says which operator a pass goes through:

* ``write``   new keys and values into the cache; a pass returns the cache
* ``read``    the tokens of each sequence as dense bf16 tensors, zeros behind the last one
* ``attn``    attention of the new tokens over the cache: query i sees the keys up to its own position, at most ``window`` back, and with
              ``sink`` the denominator of its softmax has one more term per head
* ``diff``    differential attention of the new tokens: heads in pairs (1, 2), ``a_i = softmax(q_i k_iᵀ)[v_1 | v_2]``,
              ``y = rmsnorm(a_1 − λ a_2) · w · c`` over the 2 D values of a pair

Sizes are those of the models of depth 16 and 24 (heads of 128 in groups of 4 and 8 and, gated, of 124), of the Phi-4-mini-flash shape
(40 heads of 64 in pairs over 20, window 512), and odd ones.
"""
import math

import torch

own = False             # False: elementary torch operations; True: the framework's operators

E4M3_MAX, EPS = 448.0, 1e-5


def listed():
    return [
        # one decoding step of one request: the write alone, latency
        dict(name="write_1x1_e4m3", op="write", batch=1, new=1, length=700, groups=4, dim=128, page=64, cache="e4m3"),
        # four prompts of a long chunk each
        dict(name="write_4x4096_e4m3", op="write", batch=4, new=4096, length=8192, groups=4, dim=128, page=64, cache="e4m3"),
        # a ragged batch of drafts at a head size that no 16 bytes divide, pages that are no power of two
        dict(name="write_33x37_d124_ragged", op="write", batch=33, new=37, length=1000, groups=4, dim=124, page=48, cache="bf16", ragged=True),
        # a short prefix of a request for the dense attention kernels
        dict(name="read_3x100", op="read", batch=3, length=100, groups=4, dim=128, page=64, cache="bf16", ragged=True),
        # long prefixes, stored in 8 bits
        dict(name="read_8x8192_e4m3", op="read", batch=8, length=8192, groups=4, dim=128, page=64, cache="e4m3", ragged=False),
        # one request, early in its answer: latency
        dict(name="attn_1x1000", op="attn", batch=1, new=1, length=1000, heads=16, groups=4, dim=128, page=64, cache="bf16"),
        # samples of one problem, some long, some short
        dict(name="attn_64x8192_ragged", op="attn", batch=64, new=1, length=8192, heads=16, groups=4, dim=128, page=64, cache="bf16", ragged=True),
        # one request over a very long document, 8 query heads to a key head, stored in 8 bits
        dict(name="attn_1x131072_e4m3", op="attn", batch=1, new=1, length=131072, heads=32, groups=4, dim=128, page=128, cache="e4m3"),
        # drafts of four tokens with a window and sinks, pages of 16, odd lengths
        dict(name="attn_7x3001_draft4_window_sink", op="attn", batch=7, new=4, length=3001, heads=24, groups=6, dim=128, page=16, cache="bf16",
             ragged=True, window=2047, sink=True),
        # differential attention of one token in a window
        dict(name="diff_1x2000_window", op="diff", batch=1, new=1, length=2000, heads=40, groups=20, dim=64, page=64, cache="bf16", window=511),
        # the same without one (the layer whose cache the cross-attention layers share), a ragged batch
        dict(name="diff_32x8192_ragged", op="diff", batch=32, new=1, length=8192, heads=40, groups=20, dim=64, page=64, cache="bf16", ragged=True),
        # pairs of heads of 128, stored in 8 bits
        dict(name="diff_4x32768_e4m3", op="diff", batch=4, new=1, length=32768, heads=16, groups=4, dim=128, page=128, cache="e4m3"),
    ]


def draw(rng):
    """Another case of these ranges: operator, sizes (spread over their logarithm, odd ones among them), types."""
    def log(lo, hi):
        n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        n = rng.choice([n, n, (n + 15) // 16 * 16])
        return min(max(n, lo), hi)

    op = rng.choice(["write", "read", "attn", "attn", "attn", "diff", "diff"])
    case = dict(op=op, batch=log(1, 64), page=rng.choice([16, 48, 64, 64, 128]), cache=rng.choice(["bf16", "e4m3"]), ragged=rng.random() < 0.6)
    dim = rng.choice([64, 64, 128]) if op == "diff" else rng.choice([64, 124, 128, 128])
    groups = rng.choice([2, 4, 20] if op == "diff" else [1, 4, 4, 6])
    token = groups * dim
    if op in ("write", "read"):
        tokens = log(1, 8192 * 2048 // token)
        case["batch"] = min(case["batch"], tokens)
        length = max(1, tokens // case["batch"])
        case.update(groups=groups, dim=dim, length=length)
        if op == "write":
            case.update(new=length, length=length + rng.randrange(0, 2000))
        return case
    case["new"] = 1 if rng.random() < 0.6 else rng.randrange(2, 9)
    length = log(1, 131072)
    case["batch"] = max(1, min(case["batch"], 64 * 8192 * 512 // (length * token)))
    per = rng.choice([1, 2, 4, 5, 8]) if op == "attn" else rng.choice([1, 2, 4])
    while case["batch"] * length * token > 64 * 8192 * 512:
        length //= 2
    case.update(length=max(length, case["new"]), groups=groups, heads=groups * per, dim=dim)
    if rng.random() < 0.4:
        case["window"] = rng.choice([127, 511, 2047])
    if op == "attn" and rng.random() < 0.3:
        case["sink"] = True
    return case


# ------------------------------------------------------------------------------------------------ what a program has in hand
def _inputs(case, seed):
    """Keys with a few strong channels, values that differ in size from token to token, pages in no order, as in a cache that is in use."""
    g = torch.Generator(device="cuda").manual_seed(1_000_003 * seed + 31)
    rnd = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    rand = lambda lo, hi, *shape: torch.randint(lo, hi + 1, shape, generator=g, device="cuda", dtype=torch.int32)  # noqa: E731
    B, G, D, S, L, new = case["batch"], case["groups"], case["dim"], case["page"], case["length"], case.get("new", 1)
    s, op = {"case": case}, case["op"]
    if case.get("ragged"):
        s["lengths"] = rand(min(max(new, L // 8), L), L, B)
        s["lengths"][0] = L
    else:
        s["lengths"] = torch.full((B,), L, dtype=torch.int32, device="cuda")
    s["new_lengths"] = rand(0, new, B) if case.get("ragged") and new > 1 else None
    n = -(-L // S)
    pages = B * n + 3
    s["table"] = torch.randperm(pages, generator=g, device="cuda")[:B * n].to(torch.int32).view(B, n)
    strong = torch.exp(0.5 * rnd(G, 1, D))
    if op == "write":
        s["k"] = (rnd(B, new, G, D) * strong.view(G, D)).bfloat16()
        s["v"] = (rnd(B, new, G, D) * torch.exp(0.5 * rnd(B, new, G, 1))).bfloat16()
    s["old_k"] = (rnd(pages, G, S, D) * strong).bfloat16()
    s["old_v"] = (rnd(pages, G, S, D) * torch.exp(0.5 * rnd(pages, G, S, 1))).bfloat16()
    if op in ("attn", "diff"):
        s["q"] = (1.5 * rnd(B, new, case["heads"], D)).bfloat16()
        s["scale"] = 1 / math.sqrt(D)
        s["sink"] = rnd(case["heads"]) if case.get("sink") else None
    if op == "diff":
        s["lam"] = 0.3 + 0.1 * rnd(1)
        s["w"] = 1 + 0.1 * rnd(2 * D)
        s["c"] = 0.4
    return s


def _pow2(e):
    """2^e as 32-bit numbers, e an integer tensor from −127 on."""
    bits = torch.where(e > -127, (e + 127) << 23, torch.full_like(e, 1 << 22))
    return bits.to(torch.int32).view(torch.float32)


def _quant(x):
    """(elements, biased exponents) of heads in the last dimension."""
    a = x.float().abs().amax(-1)
    m, e = torch.frexp(a)                                            # a = m · 2^e, m in [0.5, 1)
    e = torch.where(m > 0.875, e - 8, e - 9).clamp_min(-127).to(torch.int32)
    e = torch.where(a > 0, e, torch.full_like(e, -127))
    up = torch.where(e > -127, 127 - e, torch.full_like(e, 254)) << 23
    q = (x.float() * up.to(torch.int32).view(torch.float32).unsqueeze(-1)).to(torch.float8_e4m3fn)
    return q, (e + 127).to(torch.uint8)


def prepare(case, seed):
    s = _inputs(case, seed)
    k, v = s.pop("old_k"), s.pop("old_v")
    if case["cache"] == "e4m3":
        (k, ks), (v, vs) = _quant(k), _quant(v)
        s["cache"] = (k, v, ks.view(torch.float8_e8m0fnu), vs.view(torch.float8_e8m0fnu))
    else:
        s["cache"] = (k, v, None, None)
    return s


# ------------------------------------------------------------------------------------------------ the plain form, in 32 bits
def _counts(s):
    case = s["case"]
    new = case.get("new", 1)
    n = s["new_lengths"] if s["new_lengths"] is not None else torch.full_like(s["lengths"], new)
    return s["lengths"].long(), n.long()


def _plain_write(s):
    case = s["case"]
    lengths, n = _counts(s)
    i = torch.arange(case["new"], device="cuda")
    b, i = (i[None] < n[:, None]).nonzero(as_tuple=True)
    pos = lengths[b] - n[b] + i
    page, slot = s["table"][b, pos // case["page"]].long(), pos % case["page"]
    out = []
    for x, old, scale in ((s["k"], s["cache"][0], s["cache"][2]), (s["v"], s["cache"][1], s["cache"][3])):
        x = x[b, i]
        if scale is None:
            old[page, :, slot] = x
        else:
            q, e = _quant(x)
            old.view(torch.uint8)[page, :, slot] = q.view(torch.uint8)
            scale.view(torch.uint8)[page, :, slot] = e
        out.append((old, scale))
    return out


def _dense(s, tokens):
    """Keys and values of all sequences in 32 bits, (B, G, tokens, D)."""
    case = s["case"]
    pos = torch.arange(tokens, device="cuda")
    page, slot = s["table"][:, pos // case["page"]].long(), (pos % case["page"]).expand(case["batch"], -1)
    out = []
    for x, scale in ((s["cache"][0], s["cache"][2]), (s["cache"][1], s["cache"][3])):
        if scale is None:
            y = x[page, :, slot].float()
        else:
            y = x.view(torch.uint8)[page, :, slot].view(torch.float8_e4m3fn).float()
            e = scale.view(torch.uint8)[page, :, slot].to(torch.int32) - 127
            y = y * _pow2(e).unsqueeze(-1)
        out.append(y.transpose(1, 2))
    return out


def _weights(s, q, k):
    """Numerators and denominators of the softmax: q (B, T, G, r, D), k (B, G, L, D) -> (B, G, r, T, L), (B, G, r, T, 1)."""
    case = s["case"]
    lengths, n = _counts(s)
    T, L = q.shape[1], k.shape[2]
    x = torch.einsum("btgrd,bgld->bgrtl", q.float(), k) * s["scale"]
    pos = (lengths - n)[:, None] + torch.arange(T, device="cuda")
    key = torch.arange(L, device="cuda")
    seen = (key <= pos[..., None]) & (torch.arange(T, device="cuda") < n[:, None])[..., None]
    if case.get("window") is not None:
        seen &= key >= pos[..., None] - case["window"]
    x = x.masked_fill(~seen[:, None, None], float("-inf"))
    top = x.amax(-1, keepdim=True)
    sink = None
    if s.get("sink") is not None:
        sink = s["sink"].view(1, q.shape[2], q.shape[3], 1, 1)
        top = torch.maximum(top, sink)
    top = top.masked_fill(top == float("-inf"), 0.0)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    if sink is not None:
        total = total + torch.exp(sink - top)
    return p, total


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "write":
        (k, ks), (v, vs) = _plain_write(s)
        return {"k": k, "v": v} if ks is None else {"k": k, "v": v, "k_scale": ks, "v_scale": vs}
    if op == "read":
        live = torch.arange(case["length"], device="cuda")[None] < s["lengths"][:, None]
        k, v = (torch.where(live[:, :, None, None], x.transpose(1, 2), torch.zeros((), device="cuda")).bfloat16() for x in _dense(s, case["length"]))
        return {"k": k, "v": v}
    B, T, H, D = s["q"].shape
    G = case["groups"]
    k, v = _dense(s, case["length"])
    if op == "attn":
        p, total = _weights(s, s["q"].view(B, T, G, H // G, D), k)
        o = torch.einsum("bgrtl,bgld->bgrtd", p, v) / total.clamp_min(1e-30)
        return {"out": o.permute(0, 3, 1, 2, 4).reshape(B, T, H, D).bfloat16()}
    # heads h = 2 p + i of queries and 2 g + i of keys; pair p reads keys of pair g = p // (H / G)
    q = s["q"].view(B, T, G // 2, H // G, 2, D)
    v = torch.cat((v[:, 0::2], v[:, 1::2]), -1)
    a = []
    for i in range(2):
        p, total = _weights(s, q[:, :, :, :, i], k[:, i::2])
        a.append(torch.einsum("bgrtl,bgld->bgrtd", p, v) / total.clamp_min(1e-30))
    a = a[0] - s["lam"] * a[1]
    a = a * torch.rsqrt(a.square().mean(-1, keepdim=True) + EPS) * s["w"] * s["c"]
    return {"out": a.permute(0, 3, 1, 2, 4).reshape(B, T, H, D).bfloat16()}


# ------------------------------------------------------------------------------------------------ the framework's operators
def _own(s):
    from archscale_b200 import ops
    case = s["case"]
    op = case["op"]
    cache = ops.PagedCache(*s["cache"])
    if op == "write":
        ops.paged_cache_write(cache, s["k"], s["v"], s["table"], s["lengths"], s["new_lengths"])
        return {"k": cache.k, "v": cache.v} if cache.k_scale is None else {"k": cache.k, "v": cache.v, "k_scale": cache.k_scale, "v_scale": cache.v_scale}
    if op == "read":
        k, v = ops.paged_cache_read(cache, s["table"], s["lengths"], case["length"])
        return {"k": k, "v": v}
    window = (case.get("window", -1), 0)
    if op == "attn":
        return {"out": ops.paged_attention(s["q"], cache, s["table"], s["lengths"], s["new_lengths"], scale=s["scale"], window=window, sink=s["sink"])}
    return {"out": ops.paged_diff_attention(s["q"], cache, s["table"], s["lengths"], s["lam"], s["w"], s["c"], EPS, s["new_lengths"],
                                            scale=s["scale"], window=window)}


def run(state):
    with torch.no_grad():
        return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    B, G, D, L, new = case["batch"], case["groups"], case["dim"], case["length"], case.get("new", 1)
    head = D + 1 if case["cache"] == "e4m3" else 2 * D               # one head of one token in the cache
    op = case["op"]
    # ragged lengths are even between L / 8 and L, ragged counts between 0 and new
    mean = (L + L / 8) / 2 if case.get("ragged") else L
    live = new / 2 if case.get("ragged") and new > 1 else new
    if op == "write":
        n = B * live * G
        return {"bytes": int(2 * n * (2 * D + head)), "flops": int(4 * n * D)}
    if op == "read":
        return {"bytes": int(2 * G * B * (mean * head + L * 2 * D)), "flops": int(2 * G * B * mean * D)}
    seen = min(mean, case["window"] + new) if case.get("window") is not None else mean
    H = case["heads"]
    products = 4 if op == "attn" else 6                              # operations per query head, key and D
    return {"bytes": int(2 * G * B * seen * head + 4 * B * new * H * D), "flops": int(products * B * live * H * seen * D)}


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def _e4m3(v):
    """Nearest e4m3 value, ties to even: 3 bits after the leading one, spacing 2⁻⁹ below 2⁻⁶."""
    _, e = torch.frexp(v)
    step = torch.exp2((e - 1).clamp_min(-6).double() - 3)
    return torch.round(v / step) * step


def _exact_quant(x):
    """(elements, powers of two) of x (64 bits), heads in the last dimension."""
    a = torch.maximum(x.amax(-1), -x.amin(-1))
    e = torch.where(a > 0, torch.floor(torch.log2(a.clamp(min=1e-45))) - 10, -127.0)
    for _ in range(3):                                               # raised until 448 · 2^e reaches a
        e = e + (E4M3_MAX * torch.exp2(e) < a).double()
    s = torch.exp2(e.clamp(min=-127.0))
    return _e4m3(x / s[..., None]), s


def exact(case, seed):
    s = _inputs(case, seed)
    op, S = case["op"], case["page"]
    lengths, table = s["lengths"].tolist(), s["table"].tolist()
    counts = s["new_lengths"].tolist() if s["new_lengths"] is not None else [case.get("new", 1)] * case["batch"]
    eight = case["cache"] == "e4m3"

    if op == "write":
        out = {}
        for name, new, old in (("k", s["k"], s["old_k"]), ("v", s["v"], s["old_v"])):
            whole = old.double()
            at, what = [], []
            for b, (L, n) in enumerate(zip(lengths, counts)):
                at += [table[b][p // S] * S + p % S for p in range(L - n, L)]
                what += [b * new.shape[1] + i for i in range(n)]
            at, what = (torch.tensor(t, dtype=torch.long, device="cuda") for t in (at, what))
            by_slot = whole.transpose(1, 2).reshape(-1, *whole.shape[1::2])
            by_slot[at] = new.double().flatten(0, 1)[what]
            whole = by_slot.view(whole.shape[0], S, *whole.shape[1::2]).transpose(1, 2)
            out[name], scale = _exact_quant(whole) if eight else (whole, None)
            if eight:
                out[name + "_scale"] = scale
        return {n: out[n] for n in (("k", "v", "k_scale", "v_scale") if eight else ("k", "v"))}

    def sequence(b, old):
        """Tokens of a sequence, (length, G, D)."""
        pages = torch.tensor(table[b][:-(-lengths[b] // S)], dtype=torch.long, device="cuda")
        x = old[pages].double().transpose(1, 2).flatten(0, 1)[:lengths[b]]
        if eight:
            q, e = _exact_quant(x)
            x = q * e[..., None]
        return x

    if op == "read":
        out = {}
        for name in ("k", "v"):
            out[name] = torch.zeros(case["batch"], case["length"], case["groups"], case["dim"], dtype=torch.float64, device="cuda")
            for b in range(case["batch"]):
                out[name][b, :lengths[b]] = sequence(b, s["old_" + name])
        return out
    q = s["q"].double()
    B, T, H, D = q.shape
    per = H // case["groups"]
    out = torch.zeros_like(q)
    for b in range(B):
        k, v = sequence(b, s["old_k"]), sequence(b, s["old_v"])
        for t in range(counts[b]):
            pos = lengths[b] - counts[b] + t
            lo = max(0, pos - case["window"]) if case.get("window") is not None else 0
            if op == "attn":
                kk, vv = k[lo:pos + 1].transpose(0, 1), v[lo:pos + 1].transpose(0, 1)
                x = torch.matmul(q[b, t].view(-1, per, D), kk.transpose(1, 2)).flatten(0, 1) / math.sqrt(D)    # H, keys
                if s["sink"] is not None:
                    x = torch.cat((x, s["sink"].double()[:, None]), 1)
                w = torch.softmax(x, 1)[:, :kk.shape[1]].view(-1, per, kk.shape[1])
                out[b, t] = torch.matmul(w, vv).flatten(0, 1)
            else:
                P = case["groups"] // 2
                vv = v[lo:pos + 1].reshape(-1, P, 2 * D).transpose(0, 1)
                a = []
                for i in range(2):
                    kk = k[lo:pos + 1, i::2].transpose(0, 1)
                    x = torch.matmul(q[b, t, i::2].reshape(P, per, D), kk.transpose(1, 2)) / math.sqrt(D)
                    a.append(torch.matmul(torch.softmax(x, 2), vv))
                y = a[0] - s["lam"].double() * a[1]
                y = y / (y.square().mean(2, keepdim=True) + EPS).sqrt() * s["w"].double() * s["c"]
                out[b, t] = y.reshape(H, D)
    return {"out": out}
