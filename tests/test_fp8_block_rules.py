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
