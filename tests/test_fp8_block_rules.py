"""What the 8-bit operators refuse, and that they do so on every device alike."""
import pytest
import torch

from archscale_b200 import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _operands(device):
    g = torch.Generator().manual_seed(0)
    x, w, bias, nw = (torch.randn(*s, generator=g).to(device) for s in ((5, 160), (40, 160), (40,), (160,)))
    return x, w, bias, nw, ops.quantize_fp8_block(x), ops.quantize_fp8_weight(w)


@pytest.mark.parametrize("device", DEVICES)
def test_calls_without_gradients_refuse_operands_that_ask_for_one(device):
    x, w, bias, nw, (q, s), (wq, _, ws) = _operands(device)
    ask = lambda t: t.detach().clone().requires_grad_()  # noqa: E731
    calls = {
        "rows": (ops.quantize_fp8_block, (x,)),
        "columns": (ops.quantize_fp8_block_t, (x,)),
        "both": (ops.quantize_fp8_block_both, (x,)),
        "weight": (ops.quantize_fp8_weight, (w,)),
        "product": (lambda a, b, c: ops.matmul_fp8_block(q, a, wq, b, c), (s, ws, bias)),
        "accumulated": (lambda a: ops.matmul_fp8_block(q, s, wq, ws, acc=a), (torch.zeros(5, 40, device=device),)),
        "stored": (lambda a, b, c: ops.linear_fp8_weight(a, wq, b, c), (x, ws, bias)),
        "stored, of elements": (lambda a, b, c: ops.linear_fp8_weight((q, a), wq, b, c), (s, ws, bias)),
        "norm": (lambda a, b, c: ops.add_rms_norm_fp8(a, b, c), (x, x.bfloat16(), nw)),
    }
    for name, (call, args) in calls.items():
        plain = call(*args)
        for t in plain if isinstance(plain, tuple) else (plain,):
            assert not t.requires_grad, name
        for i in range(len(args)):
            some = [ask(t) if j == i else t for j, t in enumerate(args)]
            with pytest.raises(RuntimeError, match="has no gradients"):
                call(*some)
            with torch.no_grad():
                call(*some)


@pytest.mark.parametrize("device", DEVICES)
def test_forward_mode_tangents_are_refused(device):
    from torch.autograd import forward_ad
    x, w, bias, nw, _, (wq, _, ws) = _operands(device)
    calls = [ops.quantize_fp8_block, ops.quantize_fp8_weight, lambda t: ops.linear_fp8_weight(t, wq, ws),
             lambda t: ops.add_rms_norm_fp8(t, None, nw), lambda t: ops.linear_fp8_block(t, w),
             lambda t: ops.add_rms_norm_linear_fp8(t, None, nw, w)]
    for call in calls:
        for ctx in (torch.no_grad, torch.enable_grad):
            with ctx(), forward_ad.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
                call(forward_ad.make_dual(x, torch.ones_like(x)))
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.func.jvp(call, (x,), (x,))
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda t: call(t)[0].float().sum())(x)
    with forward_ad.dual_level():                                  # operands without one
        assert torch.equal(ops.linear_fp8_weight(x, wq, ws), ops.linear_fp8_weight(x, wq, ws))


def _near(got, want, top):
    """The same elements and scales through another order of sums: 160 products of fp32 and two blocks, every step rounded or cut; ``top`` bounds a product
    of two values.  Results in bf16 may round to neighbours."""
    tol = 160 * top * 170 * 2.0 ** -23 + (2.0 ** -7 * want.float().abs() if want.dtype == torch.bfloat16 else 0)
    return bool(((got.float() - want.float()).abs() <= tol).all())


@pytest.mark.parametrize("device", DEVICES)
def test_vmap_and_traces(device):
    x, w, bias, nw, _, (wq, _, ws) = _operands(device)
    batch = torch.randn(3, 5, 160, generator=torch.Generator().manual_seed(1)).to(device)
    top = float(batch.abs().max() * w.abs().max())
    top_n = 160 ** 0.5 * float(nw.abs().max() * w.abs().max())          # a normalised value is at most the root of the width
    stored = lambda t: ops.linear_fp8_weight(t, wq, ws, bias)  # noqa: E731
    assert _near(torch.vmap(stored)(batch), stored(batch), top)
    assert torch.equal(torch.vmap(lambda t: ops.quantize_fp8_block(t)[1])(batch)[1], ops.quantize_fp8_block(batch[1])[1])
    _, q, s = torch.vmap(lambda t: ops.add_rms_norm_fp8(t, None, nw))(batch)
    assert q.shape == (3, 5, 160) and s.shape == (3, 5, 2)
    layers = ((stored, top), (lambda t: ops.linear_fp8_block(t, w), top), (lambda t: ops.add_rms_norm_linear_fp8(t, None, nw, w)[1], top_n))
    for call, bound in layers:
        for ctx in (torch.no_grad, torch.enable_grad):
            with ctx():
                traced = torch.jit.trace(call, (x,), check_trace=False)
                assert _near(traced(batch[2]), call(batch[2]), bound) and not torch.allclose(traced(batch[2]), traced(x))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("lead", [(0,), (4,), (2, 3), (0, 3), (2, 0)])
@pytest.mark.parametrize("K,N", [(160, 40), (0, 40), (160, 0), (0, 0)])
def test_sizes_of_zero(device, lead, K, N):
    """No tokens, an empty sum, no outputs: the shapes and zeros that F.linear gives, gradients too."""
    g = torch.Generator().manual_seed(0)
    x, w, gy = (torch.randn(*s, generator=g).to(device) for s in ((*lead, K), (N, K), (*lead, N)))
    x.requires_grad_(), w.requires_grad_()
    bias = torch.ones(N, device=device)
    y, z = ops.linear_fp8_block(x, w, bias), torch.nn.functional.linear(x, w, bias)
    assert y.shape == z.shape and (K > 0 or (y == 1).all())
    for got, want in zip(torch.autograd.grad(y, (x, w), gy), torch.autograd.grad(z, (x, w), gy)):
        assert got.shape == want.shape and (want.numel() == 0 or want.abs().max() > 0 or (got == 0).all())
    with torch.no_grad():
        wq, wt, ws = ops.quantize_fp8_weight(w)
        assert wq.shape == (N, K) and wt.shape == (K, N) and ws.shape == (-(-N // 128), -(-K // 128))
        y = ops.linear_fp8_weight(x, wq, ws, bias)
        assert y.shape == z.shape and (K > 0 or (y == 1).all())
        if K:
            n = torch.ones(K, device=device)
            s, q, scale = ops.add_rms_norm_fp8(x, x.bfloat16(), n)
            rows = z.numel() // N if N else x.numel() // K
            assert s.shape == x.shape and q.shape == (rows, K) and scale.shape == (rows, -(-K // 128))
            assert ops.linear_fp8_weight((q.view(x.shape), scale), wq, ws).shape == z.shape
    if K:
        s, y = ops.add_rms_norm_linear_fp8(x, None, n.requires_grad_(), w)
        dx, dn, dw = torch.autograd.grad(y, (x, n, w), gy.bfloat16())
        assert y.shape == z.shape and dx.shape == x.shape and dn.shape == n.shape and dw.shape == w.shape


@pytest.mark.gpu
@pytest.mark.parametrize("K", [160, 200])
def test_operands_on_two_devices(K):
    """Refused as such, whether or not the rows of the elements would have to be copied first."""
    x, w = torch.randn(5, K, device="cuda"), torch.randn(40, K, device="cuda")
    (q, s), (wq, _, ws) = ops.quantize_fp8_block(x), ops.quantize_fp8_weight(w)
    host = lambda t: t.cpu().contiguous()  # noqa: E731
    for args in ((q, s, host(wq), ws), (q, s, wq, host(ws)), (q, host(s), wq, ws), (q, s, wq, ws, torch.zeros(40))):
        with pytest.raises(ValueError):
            ops.matmul_fp8_block(*args)
    for call in (lambda: ops.linear_fp8_block(x, host(w)), lambda: ops.linear_fp8_weight(x, host(wq), ws),
                 lambda: ops.add_rms_norm_fp8(x, None, torch.ones(K)), lambda: ops.add_rms_norm_linear_fp8(x, None, torch.ones(K, device="cuda"), host(w))):
        with pytest.raises(ValueError):
            call()
