"""8-bit layers next to other modules: layers that were replaced, families of models, the evaluation loader."""
import pytest
import torch
import torch.nn as nn

from archscale_b200.config import Config
from archscale_b200.eval import load_model
from archscale_b200.models.gpt import GPT
from archscale_b200.models.layers import Linear, apply_fp8_block, freeze_fp8_block

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


class _Wrapped(nn.Module):
    """A layer around another one, as adapters are."""

    def __init__(self, inner):
        super().__init__()
        self.inner = inner

    def forward(self, x):
        return self.inner(x)


def _dense(device):
    torch.manual_seed(3)
    m = GPT(Config.from_name("transformer_gqa4_d8", n_layer=2, n_embd=128, ar=None, n_head=2, n_query_groups=1, head_dim=64, intermediate_size=256,
                             block_size=64, padded_vocab_size=128, vocab_size=128)).to(device)
    m.reset_parameters()
    return m.to(torch.bfloat16)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fp8", [False, True])
def test_models_with_replaced_layers(device, fp8):
    m = _dense(device)
    if fp8:
        apply_fp8_block(m)
    idx = torch.randint(0, 128, (1, 16), device=device)
    with torch.no_grad():
        want = m(idx).logits
        mlp = m.transformer.h[0].mlp
        mlp.w1 = _Wrapped(mlp.w1)
        plain = nn.Linear(128, 512, bias=False, device=device, dtype=mlp.w3.weight.dtype)
        plain.weight.copy_(m.transformer.h[1].mlp.w1.weight)
        assert not m.transformer.h[0]._fp8_mlp(torch.zeros(1, dtype=torch.bfloat16), torch.bfloat16)
        got = m(idx).logits
        # the norm's own 8-bit output is not rounded to 16 bits first, which moves elements to their neighbours
        assert (got - want).abs().max() <= (0.1 if device == "cuda" else 0) * want.abs().max()
        m.transformer.h[1].mlp.w1 = plain
        assert torch.isfinite(m(idx).logits).all()
        assert not m.transformer.h[1]._fp8_mlp(torch.zeros(1, dtype=torch.bfloat16), torch.bfloat16)


SMALL = dict(n_layer=2, ar=None, n_embd=256, n_head=2, n_query_groups=1, intermediate_size=256, block_size=64, padded_vocab_size=128, vocab_size=128)
FAMILIES = {
    "experts": ("transformer_gqa4_h2_moe_s2_k2_d8", dict(head_dim=128), ("router",)),
    "experts, one by one": ("transformer_gqa4_h2_moe_s2_k2_d8", dict(head_dim=128, use_sonicmoe=False), ("router.lc_proj",)),
    "gates per head": ("transformer_gqa4_d8", dict(head_dim=128, gated_attn=True), ("attn.g_proj",)),
    "selective scan": ("samba_d8", {}, ("x_proj", "dt_proj")),
    "state space duality": ("mambay2_d16", dict(n_layer=4), ()),
    "delta rule": ("gdny_d16", dict(n_layer=4), ("a_proj", "b_proj")),
}


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("family", FAMILIES)
def test_families(device, family):
    """One step of every family: which layers are switched, that gradients arrive everywhere, and that stored weights give what live ones give."""
    name, more, kept = FAMILIES[family]
    torch.manual_seed(3)
    m = GPT(Config.from_name(name, **{**SMALL, **more})).to(device)
    m.reset_parameters()
    m = m.to(torch.bfloat16)
    n = apply_fp8_block(m)
    layers = {n: l for n, l in m.named_modules() if isinstance(l, Linear)}
    steering = [n for n in layers if n.endswith(kept)] if kept else []
    assert bool(steering) == bool(kept)
    assert {n for n, l in layers.items() if not l.fp8_block} == {"lm_head", *steering} and n == len(layers) - 1 - len(steering)
    idx = torch.randint(0, 128, (2, 32), device=device)
    out = m(idx).logits
    out.float().square().mean().backward()
    assert torch.isfinite(out).all()
    for n, l in layers.items():
        assert l.weight.grad is not None and torch.isfinite(l.weight.grad).all(), n
    with torch.no_grad():
        live = m(idx).logits
        assert freeze_fp8_block(m) == len(layers) - 1 - len(steering)
        assert torch.equal(m(idx).logits, live)


@pytest.mark.parametrize("device", DEVICES)
def test_evaluation_loads_what_was_trained(device, tmp_path):
    """A checkpoint of a model that was trained in this format is evaluated in it, on stored weights; the caller may say otherwise."""
    name = "transformer_gqa4_d8"
    torch.manual_seed(0)
    cfg = Config.from_name(name)
    cfg.rope_base = 10000
    small = dict(n_layer=1, n_embd=128, n_head=1, n_query_groups=1, head_dim=128, intermediate_size=256, vocab_size=128, padded_vocab_size=128)
    real = Config.from_name.__func__
    with pytest.MonkeyPatch.context() as mp:
        mp.setattr(Config, "from_name", classmethod(lambda cls, n, **kw: real(cls, n, **{**small, "ar": None, **kw})))
        trained = GPT(Config.from_name(name))
        trained.reset_parameters()
        paths = {}
        for fp8 in (False, True):
            config = {**trained.config.to_dict(), "fp8_block": fp8}
            paths[fp8] = str(tmp_path / f"{fp8}.pth")
            torch.save({"model": trained.state_dict(), "config": config}, paths[fp8])
        paths["bare"] = str(tmp_path / "bare.pth")
        torch.save(trained.state_dict(), paths["bare"])
        idx = torch.randint(0, 128, (1, 8), device=device)

        def logits(path, **kw):
            m = load_model(path, name, device=device, **kw).model
            on = {l.fp8_block for n, l in m.named_modules() if isinstance(l, Linear) and n != "lm_head"}
            with torch.no_grad():
                stored = {l.stored_fp8() is not None for n, l in m.named_modules() if isinstance(l, Linear) and n != "lm_head"}
                assert len(on) == 1 and on == stored == {m.config.fp8_block}
                return m.config.fp8_block, m(idx).logits

        assert [logits(paths[p])[0] for p in (False, True, "bare")] == [False, True, False]
        assert logits(paths[True], fp8_block=False)[0] is False and logits(paths["bare"], fp8_block=True)[0] is True
        plain, eight = logits(paths[False])[1], logits(paths[True])[1]
        assert not torch.equal(plain, eight) and (plain - eight).norm() <= 0.25 * plain.norm()


def test_freezing_needs_layers():
    m = _dense("cpu")
    with pytest.raises(ValueError, match="apply_fp8_block"):
        freeze_fp8_block(m)
    assert freeze_fp8_block(m, False) == 0
