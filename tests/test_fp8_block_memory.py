"""What a call of an 8-bit layer allocates and keeps: nothing that no gradient will ask for."""
import pytest
import torch

from archscale_b200 import ops

pytestmark = pytest.mark.gpu
C = 4096


def _measure(call):
    """(peak while it runs, what it keeps), in bytes per element of the weight."""
    call()
    torch.cuda.synchronize()
    base = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    kept = call()
    torch.cuda.synchronize()
    return (torch.cuda.max_memory_allocated() - base) / C ** 2, (torch.cuda.memory_allocated() - base) / C ** 2, kept


@pytest.mark.parametrize("norm", [False, True])
def test_the_transposed_weight_is_made_for_the_gradient_of_the_input_alone(norm):
    x, w, n = torch.randn(2, C, device="cuda").bfloat16(), torch.randn(C, C, device="cuda").bfloat16(), torch.ones(C, device="cuda")

    def call():
        return ops.add_rms_norm_linear_fp8(x, None, n, w)[1] if norm else ops.linear_fp8_block(x, w)
    with torch.no_grad():
        peak, kept, _ = _measure(call)
        assert peak < 1.2 and kept < 0.1                     # one set of elements, one byte each
    w.requires_grad_()
    peak, kept, _ = _measure(call)
    assert peak < 1.2                                        # dW alone
    x.requires_grad_()
    peak, kept, y = _measure(call)
    assert 1.9 < peak < 2.2 and 0.9 < kept < 1.2             # and dx, for which the transpose is kept
    dx, dw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
    assert torch.isfinite(dx).all() and torch.isfinite(dw).all()


@pytest.mark.parametrize("want", [(0,), (1,), (2,), (0, 1), (0, 2), (1, 2), (0, 1, 2)])
def test_any_set_of_gradients(want):
    """The gradients that are asked for are the ones of a call that asks for all."""
    g = torch.Generator(device="cuda").manual_seed(0)
    given = [torch.randn(*s, generator=g, device="cuda") for s in ((30, 160), (200, 160), (200,))]
    gy = torch.randn(30, 200, generator=g, device="cuda")
    full = [t.clone().requires_grad_() for t in given]
    all_ = torch.autograd.grad(ops.linear_fp8_block(*full), full, gy)
    some = [t.clone().requires_grad_(i in want) for i, t in enumerate(given)]
    got = torch.autograd.grad(ops.linear_fp8_block(*some), [some[i] for i in want], gy)
    assert all(torch.equal(a, all_[i]) for a, i in zip(got, want))


@pytest.mark.parametrize("branch", [False, True])
@pytest.mark.parametrize("with_bias", [False, True])
def test_any_set_of_gradients_behind_a_norm(branch, with_bias):
    g = torch.Generator(device="cuda").manual_seed(0)
    shapes = {"res": (30, 160), "h": (30, 160), "norm": (160,), "weight": (200, 160), "bias": (200,)}
    names = [n for n in shapes if (n != "h" or branch) and (n != "bias" or with_bias)]
    given = {n: torch.randn(*shapes[n], generator=g, device="cuda").bfloat16() for n in names}
    gx, gy = (torch.randn(30, k, generator=g, device="cuda").bfloat16() for k in (160, 200))

    def grads(want):
        t = {n: v.clone().requires_grad_(n in want) for n, v in given.items()}
        x, y = ops.add_rms_norm_linear_fp8(t["res"], t.get("h"), t["norm"], t["weight"], bias=t.get("bias"))
        outs, ins = [(o, d) for o, d in ((x, gx), (y, gy)) if o.requires_grad], [t[n] for n in names if n in want]
        return dict(zip([n for n in names if n in want], torch.autograd.grad([o for o, _ in outs], ins, [d for _, d in outs])))

    full = grads(names)
    for bits in range(1, 2 ** len(names)):
        want = [n for i, n in enumerate(names) if bits >> i & 1]
        for n, got in grads(want).items():
            assert torch.equal(got, full[n]), (want, n)
