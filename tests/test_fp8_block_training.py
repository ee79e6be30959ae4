"""8-bit layers as a training run uses them: fp32 gradient buffers, captured steps, the engine; and the operand that the backward pass makes again."""
import pytest
import torch

from archscale_b200 import ops
from archscale_b200.config import Config
from archscale_b200.models.gpt import GPT, Block
from archscale_b200.models.layers import Linear, apply_fp8_block
from archscale_b200.ops import backend, fp8_block as fb
from archscale_b200.optim.sharded import ShardedOptimizer
from archscale_b200.parallel.fsdp import FSDPEngine
from archscale_b200.parallel.mesh import build_mesh

pytestmark = pytest.mark.gpu


def _rand(shape, dtype, seed, size=1.0):
    return (torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda") * size).to(dtype)


@pytest.mark.parametrize("rows,cols", [(1, 128), (130, 200), (300, 1001), (257, 4096)])
@pytest.mark.parametrize("xt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("wt", [torch.bfloat16, torch.float32])
def test_the_normalised_operand_bit_for_bit(rows, cols, xt, wt):
    """(x · rstd) · w, each product rounded to fp32, quantised along the rows of x."""
    x, w = _rand((rows, cols), xt, 1), _rand((cols,), wt, 2)
    rstd = torch.rand(rows, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda") + 0.1
    q, s = backend.require_extension().fp8_quantize(x, 2, rstd, w)
    want_q, want_s = fb.quantize_ref((x.float() * rstd[:, None] * w.float()).t())
    assert torch.equal(q.float(), want_q.float()) and torch.equal(s, want_s)


@pytest.mark.parametrize("wt", [torch.bfloat16, torch.float32])
def test_norm_and_layer_add_to_main_grad(wt):
    """dW goes into the fp32 buffer: what was there, plus dW to fp32 rounding of the sum (the same kernel, one addition more)."""
    res, h, n = _rand((200, 256), torch.bfloat16, 1), _rand((200, 256), torch.bfloat16, 2), _rand((256,), torch.float32, 3)
    w = _rand((130, 256), wt, 4).requires_grad_()
    wf = w.detach().float().requires_grad_()
    gy = _rand((200, 130), torch.bfloat16, 5)
    dw, = torch.autograd.grad(ops.add_rms_norm_linear_fp8(res, h, n, wf)[1], wf, gy)
    w.main_grad = _rand((130, 256), torch.float32, 6)
    before = w.main_grad.clone()
    for k in (1, 2):                                                   # two micro-steps
        ops.add_rms_norm_linear_fp8(res, h, n, w)[1].backward(gy)
        assert w.grad is None
        want = before.double() + k * dw.double()
        assert ((w.main_grad.double() - want).abs() <= 2.0 ** -22 * (before.abs() + k * dw.abs()).double()).all()


def test_a_captured_training_step():
    """Forward and backward in a CUDA graph, replayed on other inputs."""
    T, C, N = 300, 520, 700
    res, h, gy = (_rand((T, k), torch.bfloat16, i) for i, k in enumerate((C, C, N)))
    leaves = [t.requires_grad_() for t in (res, h, torch.ones(C, device="cuda"), _rand((N, C), torch.bfloat16, 7, 0.05), torch.zeros(N, device="cuda"))]
    res, h, n, w, b = leaves
    w2 = _rand((N, N), torch.float32, 8, 0.05).requires_grad_()

    def step():
        _, y = ops.add_rms_norm_linear_fp8(res, h, n, w, bias=b)
        z = ops.linear_fp8_block(y, w2)
        return (z.detach(), *torch.autograd.grad(z, [*leaves, w2], gy))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (20, 30):
        with torch.no_grad():
            res.copy_(_rand((T, C), torch.bfloat16, seed))
            gy.copy_(_rand((T, N), torch.bfloat16, seed + 1))
        graph.replay()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, e) for a, e in zip(got, step()))


@pytest.mark.parametrize("stream32", [False, True])
def test_steps_of_the_engine(stream32):
    """Three steps on one batch: the loss falls as with bf16 layers, whose first loss it starts from within the operands' 2⁻⁴."""
    losses = {}
    idx = torch.randint(0, 512, (2, 129), generator=torch.Generator().manual_seed(0)).cuda()
    for fp8 in (False, True):
        torch.manual_seed(3)
        m = GPT(Config.from_name("transformer_gqa4_d8", n_layer=2, n_embd=256, ar=None, n_head=2, n_query_groups=1, head_dim=128, intermediate_size=512,
                                 block_size=128, padded_vocab_size=512, vocab_size=512, residual_in_fp32=stream32)).cuda()
        m.reset_parameters()
        if fp8:
            apply_fp8_block(m)
        eng = FSDPEngine(m, build_mesh(), unit_classes=(Block,), param_dtype=torch.bfloat16)
        opt = ShardedOptimizer(eng, lr=1e-3, betas=(0.9, 0.95), algorithm="adamw", weight_decay=0.0)
        mats = {s.name: g for g in eng.groups() for s in g.specs}
        losses[fp8] = []
        for _ in range(3):
            logits = m(idx[:, :-1]).logits.float()
            loss = torch.nn.functional.cross_entropy(logits.reshape(-1, 512), idx[:, 1:].reshape(-1))
            eng.backward(loss)
            for n, l in m.named_modules():
                if isinstance(l, Linear):
                    g = mats[n + ".weight"]
                    sp = next(s for s in g.specs if s.name == n + ".weight")
                    part = g.grad[sp.offset:sp.offset + sp.numel]
                    assert torch.isfinite(part).all() and part.abs().max() > 0, n
            opt.step()
            opt.zero_grad()
            losses[fp8].append(loss.item())
        assert losses[fp8][2] < losses[fp8][1] < losses[fp8][0]
    assert abs(losses[True][0] - losses[False][0]) <= 2.0 ** -4 * losses[False][0]
