"""Products of operands whose magnitudes lie far apart, or that are small both: what has to fit fp32 is the result."""
import pytest
import torch

from archscale_b200 import ops
from archscale_b200.ops import fp8_block as fb

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("M,N", [(1, 200), (3, 64), (20, 130), (60, 300), (130, 260), (300, 640), (700, 1100)])
@pytest.mark.parametrize("kinds", ["row,tile", "row,row", "tile,row"])
@pytest.mark.parametrize("large", ["a", "b"])
def test_large_times_small(device, M, N, kinds, large):
    """Elements of 10³⁵ against 10⁻²⁰.  The bound is that of any product: 128 steps rounded or cut in a block, its scaling, the sum of the blocks."""
    K = 400
    g = torch.Generator(device=device).manual_seed(M)
    sizes = (1e35, 1e-20) if large == "a" else (1e-20, 1e35)
    quant = {"row": ops.quantize_fp8_block, "tile": lambda t: ops.quantize_fp8_weight(t)[::2]}
    (a, sa), (b, sb) = (quant[k]((torch.rand(r, K, generator=g, device=device) + 0.5) * s) for k, r, s in zip(kinds.split(","), (M, N), sizes))
    want = fb.dequantize_ref(a, sa, torch.float64) @ fb.dequantize_ref(b, sb, torch.float64).t()
    out = ops.matmul_fp8_block(a, sa, b, sb, out_dtype=torch.float32)
    assert torch.isfinite(out).all()
    assert ((out.double() - want).abs() <= want * (K * 2.0 ** -23 + 8 * 2.0 ** -24)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("M", [3, 40, 300])
@pytest.mark.parametrize("kinds", ["row,tile", "row,row"])
def test_results_below_the_range(M, kinds):
    """10⁻²³ against 10⁻²³."""
    quant = {"row": ops.quantize_fp8_block, "tile": lambda t: ops.quantize_fp8_weight(t)[::2]}
    g = torch.Generator(device="cuda").manual_seed(M)
    (a, sa), (b, sb) = (quant[k](torch.randn(r, 256, generator=g, device="cuda") * 1e-23) for k, r in zip(kinds.split(","), (M, 300)))
    assert (ops.matmul_fp8_block(a, sa, b, sb, out_dtype=torch.float32) == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("M", [3, 40, 300])
@pytest.mark.parametrize("kinds", ["row,tile", "row,row"])
def test_empty_blocks_against_large_ones(M, kinds):
    """Blocks of zeros have the smallest scale, 10⁻³⁰ / 448; the others' magnitudes go up to the end of the range."""
    quant = {"row": ops.quantize_fp8_block, "tile": lambda t: ops.quantize_fp8_weight(t)[::2]}
    x = torch.zeros(M, 384, device="cuda")
    x[:, 128:256] = 1e-30
    w = torch.full((300, 384), 1e30, device="cuda")
    w[:, 128:256] = 3e38
    (a, sa), (b, sb) = (quant[k](t) for k, t in zip(kinds.split(","), (x, w)))
    out = ops.matmul_fp8_block(a, sa, b, sb, out_dtype=torch.float32)
    want = 128 * 1e-30 * 3e38
    assert ((out - want).abs() <= want * 200 * 2.0 ** -23).all()


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(1, 128, 40000), (5, 300, 70000), (30, 2000, 20000), (64, 1000, 36100), (64, 20000, 9000)])
@pytest.mark.parametrize("kinds", ["row,tile", "row,row", "tile,row"])
def test_few_rows_of_long_contractions(M, N, K, kinds):
    """More than 32 blocks of K per CTA, so that the table of scales is filled more than once.  The bound is that of any product; a few hundred blocks are
    added in an order that is the same from call to call."""
    g = torch.Generator(device="cuda").manual_seed(K)
    quant = {"row": ops.quantize_fp8_block, "tile": lambda t: ops.quantize_fp8_weight(t)[::2]}
    (a, sa), (b, sb) = (quant[k](torch.randn(r, K, generator=g, device="cuda").bfloat16()) for k, r in zip(kinds.split(","), (M, N)))
    A, B = (fb.dequantize_ref(*t, torch.float64) for t in ((a, sa), (b, sb)))
    want, mag = A @ B.t(), A.abs() @ B.abs().t()
    out = ops.matmul_fp8_block(a, sa, b, sb, out_dtype=torch.float32)
    assert ((out.double() - want).abs() <= mag * (128 * 2.0 ** -23 + (-(-K // 128) + 3) * 2.0 ** -24)).all()
    assert torch.equal(out, ops.matmul_fp8_block(a, sa, b, sb, out_dtype=torch.float32))
