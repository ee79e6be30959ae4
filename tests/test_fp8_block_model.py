"""Models whose linear layers take 8-bit operands with an fp32 scale per 128 elements: training, and stored weights for evaluation."""
import pytest
import torch

from archscale_b200 import ops
from archscale_b200.config import Config
from archscale_b200.models.gpt import GPT
from archscale_b200.models.layers import Linear, apply_fp8_block, freeze_fp8_block
from archscale_b200.train.pretrain import setup

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _model(device, width=512, **kw):
    torch.manual_seed(3)
    cfg = Config.from_name("transformer_gqa4_d8", n_layer=2, n_embd=width, ar=None, n_head=4, n_query_groups=2, intermediate_size=width * 5 // 2,
                           block_size=256, padded_vocab_size=512, vocab_size=512, **kw)
    with torch.device(device):
        m = GPT(cfg)
    m.reset_parameters()
    with torch.no_grad():
        for p in m.parameters():
            p.copy_(torch.randn(p.shape, generator=torch.Generator().manual_seed(p.numel())) * (0.05 if p.dim() > 1 else 0.1) + (p.dim() == 1))
    return m


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("shape", [(4, 96), (2, 3, 96)])
def test_linear_layer(device, shape):
    torch.manual_seed(0)
    lin = Linear(96, 200, bias=True).to(device)
    lin.fp8_block = True
    x = torch.randn(*shape, device=device, dtype=torch.bfloat16)
    y = lin(x)
    y2 = ops.linear_fp8_block(x, lin.weight, lin.bias)
    assert y.shape == (*shape[:-1], 200) and torch.equal(y, y2)
    with torch.no_grad():
        assert torch.equal(lin(x), y)
        assert freeze_fp8_block(lin) == 1 and torch.equal(lin(x), y)
        lin.weight.mul_(2.0)
        with pytest.raises(RuntimeError, match="frozen"):
            lin(x)
        freeze_fp8_block(lin, False)
        assert not torch.equal(lin(x), y)
    freeze_fp8_block(lin)
    lin.weight.data.add_(1.0)
    lin(x).sum().backward()                       # with gradients the live weight is used
    assert lin.weight.grad is not None


@pytest.mark.gpu
@pytest.mark.parametrize("width,fp32_stream", [(512, False), (512, True), (520, False)])
def test_model_trains_near_bf16(width, fp32_stream):
    """Logits and gradients of the 8-bit model against the bf16 one.  An operand is off by at most 2⁻⁴ of its value, 2⁻⁴ / √3 in the mean square for an even
    spread of its digits; two layers with seven products each and their operands' errors independent: below a quarter of the norm."""
    m = _model("cuda", width, residual_in_fp32=fp32_stream).to(torch.bfloat16)
    idx = torch.randint(0, 512, (2, 200), device="cuda")
    gy = torch.randn(2, 200, 512, device="cuda") / 512

    def run():
        m.zero_grad()
        out = m(idx).logits
        (out * gy).sum().backward()
        return out.detach(), {n: p.grad.clone() for n, p in m.named_parameters() if p.grad is not None}

    ref, gref = run()
    assert apply_fp8_block(m) > 0
    got, ggot = run()
    rel = lambda a, b: ((a.float() - b.float()).norm() / b.float().norm()).item()  # noqa: E731
    assert 0 < rel(got, ref) < 0.25
    assert gref.keys() == ggot.keys()
    for n in gref:
        assert torch.isfinite(ggot[n]).all() and rel(ggot[n], gref[n]) < 0.5, n
    with torch.no_grad():
        live = m(idx).logits
        freeze_fp8_block(m)
        assert torch.equal(m(idx).logits, live)
        one = m(idx[:, :1]).logits
        assert one.shape == (2, 1, 512) and torch.isfinite(one).all()


@pytest.mark.gpu
def test_the_norm_of_the_mlp_writes_its_operand(monkeypatch):
    m = _model("cuda").to(torch.bfloat16)
    apply_fp8_block(m)
    calls = []
    real = ops.add_rms_norm_linear_fp8
    monkeypatch.setattr(ops, "add_rms_norm_linear_fp8", lambda *a, **k: calls.append(1) or real(*a, **k))
    idx = torch.randint(0, 512, (1, 64), device="cuda")
    m(idx)
    assert len(calls) == 2
    m.transformer.h[0].mlp.w1.register_forward_hook(lambda *a: None)      # a layer with a hook is called
    m(idx)
    assert len(calls) == 3


def test_trainer_takes_the_field_and_refuses_mixtures(tmp_path):
    kw = dict(train_data_dir="synthetic", train_model="transformer_gqa4", train_name="scaling_mup_muonh", depth=8, ctx_len=64, micro_bsz=1,
              max_tokens=1e6, return_trainer=True, quiet=True)
    small = {"n_layer": 1, "intermediate_size": 128, "padded_vocab_size": 256}
    tr = setup(**kw, config_overrides={**small, "fp8_block": True})
    mods = [(n, l) for n, l in tr.model.named_modules() if isinstance(l, Linear)]
    assert mods and all(l.fp8_block == ("lm_head" not in n) for n, l in mods)
    with pytest.raises(ValueError):
        setup(**kw, fp8=True, config_overrides={**small, "fp8_block": True})
