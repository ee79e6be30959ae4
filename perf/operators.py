"""Linear layers in 8-bit floating point with one fp32 scale for each block of 128, as cases that a timing tool can run.

Elements are e4m3 (largest value 448).  With ``BLOCK = 128`` and ``a`` the largest magnitude of a block, never taken below ``TINY``,

    scale = a / 448,    u = 448 / a,    q = e4m3(x · u),    x ≈ q · scale

where scale, u and x · u are 32-bit numbers and e4m3() rounds to nearest, ties to even.  A block is 128 neighbouring values of a
row (activations, gradients) or a 128 × 128 tile (weights); the last block of a row, column or matrix may be shorter.  A case is
a plain dict; its ``op`` says which operators a pass goes through:

* ``quant``   quantisation: ``both`` = rows and, transposed, columns of a token matrix; ``weight`` = 128 × 128 tiles, with the transpose
* ``norm``    residual addition + RMSNorm whose output is quantised: the new residual stream, elements and scales
* ``serve``   a layer with weights that were quantised beforehand: ``y = x̂ ŵᵀ (+ bias)``, x quantised within the call, or (``norm``) by
              the addition and norm that precede the layer
* ``train``   forward and backward of a layer with high-precision weights: ``y = x̂ ŵᵀ``, ``dx = ĝ ŵ``, ``dw = g̃ᵀ x̃`` (tilde: blocks along
              the tokens); with ``norm``, the addition and norm in front of it and their gradients too

Sizes are those of the dense depth-16 model (2048 wide, 5632 in the MLP), of the Phi-4-mini-flash shape (2560 wide), and odd ones.
"""
import math

import torch

own = False             # False: elementary torch operations; True: the framework's operators

BLOCK, E4M3_MAX, TINY = 128, 448.0, 1e-30
EPS = 1e-5


def listed():
    return [
        # what the backward pass of a layer does first to its incoming gradient: both orientations from one read
        dict(name="quant_both_16384x2048", op="quant", what="both", rows=16384, cols=2048, dtype="bf16"),
        # after an optimizer step: the fp32 master weights of the gate and up projections
        dict(name="quant_weight_11264x2048", op="quant", what="weight", rows=11264, cols=2048, dtype="fp32"),
        # one decoding step of one request: latency alone
        dict(name="norm_1x2048", op="norm", rows=1, cols=2048, stream="bf16", branch=True),
        # a training batch with the fp32 residual stream
        dict(name="norm_32768x2048_fp32", op="norm", rows=32768, cols=2048, stream="fp32", branch=True),
        # a ragged batch at a width that no vector load divides
        dict(name="norm_777x1001", op="norm", rows=777, cols=1001, stream="bf16", branch=True),
        # one decoding step: norm + gate and up projections of the MLP
        dict(name="serve_1_2048x11264_norm", op="serve", tokens=1, inner=2048, outer=11264, norm=True, bias=False),
        # a batch of 48 requests in decoding: down projection
        dict(name="serve_48_5632x2048", op="serve", tokens=48, inner=5632, outer=2048, norm=False, bias=False),
        # a short prompt with an odd number of outputs and a bias
        dict(name="serve_700_2560x7679_bias", op="serve", tokens=700, inner=2560, outer=7679, norm=False, bias=True),
        # a long prompt
        dict(name="serve_8192_2048x11264_norm", op="serve", tokens=8192, inner=2048, outer=11264, norm=True, bias=False),
        # training: down projection, fp32 weights
        dict(name="train_16384_5632x2048", op="train", tokens=16384, inner=5632, outer=2048, norm=False, weight="fp32"),
        # training: norm + gate and up projections, the batch of the headline run
        dict(name="train_32768_2048x11264_norm", op="train", tokens=32768, inner=2048, outer=11264, norm=True, weight="bf16"),
        # training on a ragged batch at odd widths
        dict(name="train_1003_1000x1501", op="train", tokens=1003, inner=1000, outer=1501, norm=False, weight="bf16"),
    ]


def draw(rng):
    """Another case of these ranges: operator, sizes (spread over their logarithm, odd ones among them), types."""
    def log(lo, hi):
        n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        n = rng.choice([n, n, (n + 7) // 8 * 8, (n + 127) // 128 * 128])
        return min(max(n, lo), hi)

    op = rng.choice(["quant", "norm", "serve", "serve", "train", "train"])
    if op == "quant":
        return dict(op=op, what=rng.choice(["both", "weight"]), rows=log(1, 32768), cols=log(64, 8192), dtype=rng.choice(["bf16", "fp32"]))
    if op == "norm":
        return dict(op=op, rows=log(1, 32768), cols=log(64, 8192), stream=rng.choice(["bf16", "fp32"]), branch=rng.random() < 0.8)
    tokens, norm = log(1 if op == "serve" else 64, 32768), rng.random() < 0.5
    # stored weights have rows of whole 16-byte pieces; at training every width may come
    inner, outer = log(256, 8192), log(64, 11264)
    inner = (inner + 15) // 16 * 16 if op == "serve" else inner
    tokens = max(1, min(tokens, 32768 * 2048 * 11264 // (inner * outer)))
    if op == "serve":
        return dict(op=op, tokens=tokens, inner=inner, outer=outer, norm=norm, bias=rng.random() < 0.3)
    return dict(op=op, tokens=tokens, inner=inner, outer=outer, norm=norm, weight="bf16" if norm else rng.choice(["bf16", "fp32"]))


# ------------------------------------------------------------------------------------------------ what a program has in hand
_DTYPE = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _inputs(case, seed):
    """Activations with a few strong channels, gradients that differ in size from token to token, weights as after training."""
    g = torch.Generator(device="cuda").manual_seed(1_000_003 * seed + 29)
    rnd = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    act = lambda rows, cols: rnd(rows, cols) * torch.exp(0.7 * rnd(cols))  # noqa: E731
    grad = lambda rows, cols: rnd(rows, cols) * torch.exp(rnd(rows, 1)) * 1e-5  # noqa: E731
    s, op = {"case": case}, case["op"]
    if op == "quant":
        make = grad if case["what"] == "both" else (lambda r, c: rnd(r, c) * 0.02)
        s["x"] = make(case["rows"], case["cols"]).to(_DTYPE[case["dtype"]])
        return s
    rows, cols = (case["rows"], case["cols"]) if op == "norm" else (case["tokens"], case["inner"])
    if op == "norm" or case["norm"]:
        stream = _DTYPE[case["stream"]] if op == "norm" else torch.bfloat16
        s["res"] = act(rows, cols).to(stream)
        s["h"] = act(rows, cols).bfloat16() if case.get("branch", True) else None
        s["norm_w"] = (1 + 0.1 * rnd(cols)).bfloat16()
        s["h_scale"] = 1 / math.sqrt(32)                             # the branch scale of a depth-16 model
    else:
        s["x"] = act(rows, cols).bfloat16()
    if op == "norm":
        return s
    w = rnd(case["outer"], cols) * 0.02
    if op == "serve":
        s["bias"] = rnd(case["outer"]).bfloat16() if case["bias"] else None
        s["w"] = w.bfloat16()                                        # what the stored elements and scales are made from
        return s
    s["w"] = w.to(_DTYPE[case["weight"]])
    s["gy"] = grad(rows, case["outer"]).bfloat16()
    if case["norm"]:
        s["gx"] = grad(rows, cols).bfloat16()                        # gradient that reaches the residual stream from behind
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "serve":                                        # the stored form of the weights, as a checkpoint has it
        s["wq"], s["ws"] = _quant_tiles(s.pop("w"))
    return s


# ------------------------------------------------------------------------------------------------ the plain form, in 32 bits
def _pad(x, row_block, col_block):
    r, c = x.shape
    return torch.nn.functional.pad(x, (0, -c % col_block, 0, -r % row_block))


def _factors(a):
    """(scale, u) of blocks with the largest magnitudes a.  A Python number as dividend or divisor would make these two roundings."""
    a = a.clamp_min(TINY)
    top = torch.full_like(a, E4M3_MAX)
    return a / top, top / a


def _quant_rows(x):
    r, c = x.shape
    xb = _pad(x.float(), 1, BLOCK).view(r, -1, BLOCK)
    scale, u = _factors(xb.abs().amax(-1))
    q = (xb * u.unsqueeze(-1)).to(torch.float8_e4m3fn)
    return q.view(r, -1)[:, :c].contiguous(), scale


def _quant_tiles(w):
    n, k = w.shape
    wb = _pad(w.float(), BLOCK, BLOCK)
    nb, kb = wb.shape[0] // BLOCK, wb.shape[1] // BLOCK
    wb = wb.view(nb, BLOCK, kb, BLOCK)
    scale, u = _factors(wb.abs().amax((1, 3)))
    q = (wb * u.view(nb, 1, kb, 1)).to(torch.float8_e4m3fn)
    return q.view(nb * BLOCK, -1)[:n, :k].contiguous(), scale


def _value_rows(q, s):
    return q.float() * s.repeat_interleave(BLOCK, 1)[:, :q.shape[1]]


def _value_tiles(q, s):
    n, k = q.shape
    return q.float() * s.repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]


def _norm(s):
    """(new stream, its 32-bit values, 1 / rms, normalised values)."""
    x = s["res"].float()
    if s["h"] is not None:
        x = x + s["h_scale"] * s["h"].float()
    x = x.to(s["res"].dtype)
    xf = x.float()
    rstd = torch.rsqrt(xf.square().mean(-1, keepdim=True) + EPS)
    return x, xf, rstd, xf * rstd * s["norm_w"].float()


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "quant":
        if case["what"] == "weight":
            q, scale = _quant_tiles(s["x"])
            return {"q": q, "scale": scale, "q_t": q.t().contiguous()}
        q, scale = _quant_rows(s["x"])
        q_t, scale_t = _quant_rows(s["x"].t())
        return {"q": q, "scale": scale, "q_t": q_t, "scale_t": scale_t}
    if op == "norm":
        x, _, _, n = _norm(s)
        q, scale = _quant_rows(n)
        return {"stream": x, "q": q, "scale": scale}
    out = {}
    if case["norm"]:
        x, xf, rstd, n = _norm(s)
        out["stream"] = x
    else:
        n = s["x"].float()
    xv = _value_rows(*_quant_rows(n))
    if op == "serve":
        y = xv @ _value_tiles(s["wq"], s["ws"]).t()
        if s["bias"] is not None:
            y = y + s["bias"].float()
        out["y"] = y.bfloat16()
        return out
    wv = _value_tiles(*_quant_tiles(s["w"]))
    out["y"] = (xv @ wv.t()).bfloat16()
    dn = _value_rows(*_quant_rows(s["gy"])) @ wv
    out["dw"] = (_value_rows(*_quant_rows(s["gy"].t())) @ _value_rows(*_quant_rows(n.t())).t()).to(s["w"].dtype)
    if not case["norm"]:
        out["dx"] = dn.bfloat16()
        return out
    nw = s["norm_w"].float()
    xhat = xf * rstd
    out["dnorm_w"] = (dn * xhat).sum(0).bfloat16()
    t = dn * nw
    dres = s["gx"].float() + rstd * (t - xhat * (t * xhat).mean(-1, keepdim=True))
    out["dres"], out["dh"] = dres.bfloat16(), (s["h_scale"] * dres).bfloat16()
    return out


# ------------------------------------------------------------------------------------------------ the framework's operators
def _own(s):
    from archscale_b200 import ops
    case = s["case"]
    op = case["op"]
    if op == "quant":
        if case["what"] == "weight":
            q, q_t, scale = ops.quantize_fp8_weight(s["x"])
            return {"q": q, "scale": scale, "q_t": q_t}
        q, scale, q_t, scale_t = ops.quantize_fp8_block_both(s["x"])
        return {"q": q, "scale": scale, "q_t": q_t, "scale_t": scale_t}
    if op == "norm":
        x, q, scale = ops.add_rms_norm_fp8(s["res"], s["h"], s["norm_w"], EPS, s["h_scale"])
        return {"stream": x, "q": q, "scale": scale}
    if op == "serve":
        if case["norm"]:
            x, q, scale = ops.add_rms_norm_fp8(s["res"], s["h"], s["norm_w"], EPS, s["h_scale"])
            return {"stream": x, "y": ops.linear_fp8_weight((q, scale), s["wq"], s["ws"], s["bias"])}
        return {"y": ops.linear_fp8_weight(s["x"], s["wq"], s["ws"], s["bias"])}
    leaf = lambda t: t.detach().requires_grad_()  # noqa: E731
    w = leaf(s["w"])
    if not case["norm"]:
        x = leaf(s["x"])
        y = ops.linear_fp8_block(x, w)
        dx, dw = torch.autograd.grad(y, (x, w), s["gy"])
        return {"y": y.detach(), "dx": dx, "dw": dw}
    res, h, nw = leaf(s["res"]), leaf(s["h"]), leaf(s["norm_w"])
    x, y = ops.add_rms_norm_linear_fp8(res, h, nw, w, EPS, s["h_scale"])
    dres, dh, dnw, dw = torch.autograd.grad((x, y), (res, h, nw, w), (s["gx"], s["gy"]))
    return {"stream": x.detach(), "y": y.detach(), "dres": dres, "dh": dh, "dnorm_w": dnw, "dw": dw}


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op, size = case["op"], {"bf16": 2, "fp32": 4}
    up = lambda n: -(-n // BLOCK)  # noqa: E731
    if op == "quant":
        r, c = case["rows"], case["cols"]
        scales = up(r) * up(c) if case["what"] == "weight" else r * up(c) + c * up(r)
        return {"bytes": r * c * (size[case["dtype"]] + 2) + 4 * scales, "flops": 2 * r * c}
    if op == "norm":
        r, c = case["rows"], case["cols"]
        b = size[case["stream"]]
        moved = r * c * ((2 * b + 2 if case["branch"] else 2 * b) + 1) + 4 * r * up(c) + 2 * c
        return {"bytes": moved, "flops": 6 * r * c}
    t, k, n = case["tokens"], case["inner"], case["outer"]
    front = 6 * t * k if case["norm"] else 2 * t * k                   # stream, branch, new stream; or x alone
    if op == "serve":
        return {"bytes": front + n * k + 4 * up(n) * up(k) + 2 * t * n, "flops": 2 * t * k * n}
    weight = size[case["weight"]]
    back = 6 * t * k if case["norm"] else 2 * t * k                    # stream gradient, dres, dh; or dx alone
    return {"bytes": front + back + 4 * t * n + 2 * weight * n * k, "flops": 6 * t * k * n}


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def _e4m3(v):
    """Nearest e4m3 value, ties to even: 3 bits after the leading one, spacing 2⁻⁹ below 2⁻⁶."""
    _, e = torch.frexp(v)
    step = torch.exp2((e - 1).clamp_min(-6).double() - 3)
    return torch.round(v / step) * step


def _exact_quant(x, rb, cb):
    """Elements and scales of x (64 bits) in blocks of rb × cb."""
    r, c = x.shape
    nr, nc = -(-r // rb), -(-c // cb)
    full = x.new_zeros(nr * rb, nc * cb)
    full[:r, :c] = x
    t = full.view(nr, rb, nc, cb)
    top = torch.maximum(t.amax((1, 3)), -t.amin((1, 3))).clamp(min=TINY)
    u = (E4M3_MAX / top).float().double()                             # a 32-bit number by definition
    q = _e4m3((t * u[:, None, :, None]).float().double())             # so is the product: many bf16 values lie on ties
    value = (q * (top / E4M3_MAX)[:, None, :, None]).reshape(nr * rb, nc * cb)[:r, :c]
    return q.reshape(nr * rb, nc * cb)[:r, :c], top / E4M3_MAX, value


def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    if op == "quant":
        x = s["x"].double()
        if case["what"] == "weight":
            q, scale, _ = _exact_quant(x, BLOCK, BLOCK)
            return {"q": q, "scale": scale, "q_t": q.t()}
        q, scale, _ = _exact_quant(x, 1, BLOCK)
        q_t, scale_t, _ = _exact_quant(x, BLOCK, 1)
        return {"q": q, "scale": scale, "q_t": q_t.t(), "scale_t": scale_t.t()}
    out = {}
    if op == "norm" or case["norm"]:
        x = s["res"].double()
        if s["h"] is not None:
            x = x + s["h_scale"] * s["h"].double()
        x = x.to(s["res"].dtype).double()                             # the stream as it is kept
        out["stream"] = x
        inv = 1 / (x.square().mean(1) + EPS).sqrt()
        nw = s["norm_w"].double()
        xhat = x * inv[:, None]
        n = xhat * nw
    else:
        n = s["x"].double()
    q, scale, value = _exact_quant(n, 1, BLOCK)
    if op == "norm":
        out["q"], out["scale"] = q, scale
        return out
    _, _, w = _exact_quant(s["w"].double(), BLOCK, BLOCK)
    y = torch.einsum("tk,nk->tn", value, w)
    if op == "serve":
        out["y"] = y if s["bias"] is None else y + s["bias"].double()
        return out
    out["y"] = y
    gy = s["gy"].double()
    dn = torch.einsum("tn,nk->tk", _exact_quant(gy, 1, BLOCK)[2], w)
    out["dw"] = torch.einsum("tn,tk->nk", _exact_quant(gy, BLOCK, 1)[2], _exact_quant(n, BLOCK, 1)[2])
    if not case["norm"]:
        out["dx"] = dn
        return out
    # dL/dx_j = inv · nw_j dn_j − x_j inv³ / C · Σ_i nw_i dn_i x_i
    along = (dn * nw * x).sum(1)
    out["dnorm_w"] = (dn * xhat).sum(0)
    out["dres"] = s["gx"].double() + inv[:, None] * nw * dn - x * (inv ** 3 * along / x.shape[1])[:, None]
    out["dh"] = s["h_scale"] * out["dres"]
    return out
