"""Generation over a key-value cache: the writer, both attentions and the models that call them, step by step against the whole prefix."""
import pytest
import torch

from archscale_b200.config import Config
from archscale_b200.eval import ModelWrapper
from archscale_b200.models.decode import DecodeCache, unsupported
from archscale_b200.models.gpt import GPT

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
SMALL = dict(vocab_size=96, padding_multiple=32, block_size=64, n_layer=4, ar=None, n_embd=64, intermediate_size=96)
MODELS = {
    "grouped": ("transformer_gqa4_d8", dict(n_head=4, n_query_groups=2, head_dim=32, qk_norm=True)),
    "one_head_each": ("transformer_mha_d8", dict(n_head=2, n_query_groups=2, head_dim=64)),
    "sinks": ("transformersa_d8", dict(n_head=4, n_query_groups=1, head_dim=32)),
    "gated": ("transformerga_gqa4_d8", dict(n_head=4, n_query_groups=4, head_dim=30)),
    "windows": ("transformerls_d8", dict(n_head=4, n_query_groups=2, head_dim=32, local_window=7)),
    "extended_window": ("transformer_gqa4_d8", dict(n_head=4, n_query_groups=2, head_dim=32, full_swa_extend=True, block_size=12)),
    "fused_projection": ("transformer_gqa4_d8", dict(n_head=4, n_query_groups=2, head_dim=32, separate_qkv=False, attn_norm=True)),
    "differential": ("transformer_gqa4_d8", dict(n_head=8, n_query_groups=4, head_dim=16, use_da=True)),
    "differential_window": ("transformerls_d8", dict(n_head=4, n_query_groups=2, head_dim=32, use_da=True, local_window=9)),
    "cross": ("swayoco_d8", dict(n_head=4, n_query_groups=2, head_dim=32, local_window=8)),
    "cross_differential": ("swayoco_d8", dict(n_head=4, n_query_groups=2, head_dim=32, local_window=8, use_da=True)),
    "windowed_rotary": ("swayoco_d8", dict(n_head=4, n_query_groups=2, head_dim=32, local_window=8, ada_rope=True, yoco_window=True)),
    "experts": ("transformer_gqa4_h2_moe_s4_k2_d8", dict(n_head=4, n_query_groups=2, head_dim=32)),
    "shared_layers": ("transformer_gqa4_d8", dict(n_head=4, n_query_groups=2, head_dim=32, share_per_layer=2, share_group=1)),
    "post_norm": ("transformer_gqa4_d8", dict(n_head=4, n_query_groups=2, head_dim=32, post_norm=True)),
}


def make(name, device="cpu", dtype=torch.float32, **more):
    base, over = MODELS[name]
    torch.manual_seed(3)
    m = GPT(Config.from_name(base, **{**SMALL, **over, **more}))
    m.reset_parameters()
    with torch.no_grad():
        for p in m.parameters():
            if p.dim() > 1:
                p.normal_(0, 0.08)
        for n, p in m.named_parameters():
            if n.endswith("softmax_offset"):
                p.normal_()
    m.compute_dtype = dtype
    return m.to(device=device, dtype=dtype).eval()


def run(m, ids, cuts, **kw):
    """Logits of ids, its columns given in pieces."""
    cache = DecodeCache(m, ids.shape[0], ids.shape[1], **kw)
    with torch.no_grad():
        out = [m(ids[:, a:b], cache=cache).logits for a, b in zip([0, *cuts], [*cuts, ids.shape[1]])]
    assert cache.tokens == ids.shape[1] and cache.lengths.tolist() == [ids.shape[1]] * ids.shape[0]
    return torch.cat(out, 1)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("cuts", [[13, 14, 15, 16, 17, 18, 19, 20], [1, 2, 3], [9, 14, 15, 20]])
@pytest.mark.parametrize("name", list(MODELS))
def test_steps_give_the_logits_of_the_whole_prefix(name, cuts, device):
    m = make(name, device)
    ids = torch.randint(0, 96, (3, 21), generator=torch.Generator().manual_seed(1)).to(device)
    with torch.no_grad():
        want = m(ids).logits
    got = run(m, ids, cuts, page_size=5)
    # the same sums of fp32 in another order: four layers whose values are of the order of one, widths below 100; on a GPU products of fp32
    # may be in TF32 on neither side (torch's default)
    assert float((got - want).abs().max()) <= 2e-4 * max(1.0, float(want.abs().max()))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("name", ["grouped", "windows", "differential", "cross", "experts"])
def test_generation(name, device):
    m = make(name, device)
    w = ModelWrapper(m)
    ids = torch.randint(0, 96, (2, 6), generator=torch.Generator().manual_seed(2)).to(device)
    plain = w.generate(ids, max_gen_toks=12, return_dict_in_generate=False)
    cached = w.generate(ids, max_gen_toks=12, return_dict_in_generate=False, kv_cache=True)
    assert cached.shape == plain.shape == (2, 18) and torch.equal(cached[:, :6], ids)
    # greedy choices agree up to ties of what the orders of sums leave
    with torch.no_grad():
        logits = m(cached[:, :-1]).logits[:, 5:]
    chosen = logits.gather(-1, cached[:, 6:, None]).squeeze(-1)
    assert bool((chosen >= logits.amax(-1) - 4e-4 * max(1.0, float(logits.abs().max()))).all())
    stop = int(cached[0, 8])
    short = w.generate(ids, max_gen_toks=12, eos_token_id=stop, kv_cache=True)
    assert short.sequences.shape[1] <= 18
    eight = w.generate(ids, max_gen_toks=12, return_dict_in_generate=False, kv_cache=True, kv_cache_dtype=torch.float8_e4m3fn)
    assert eight.shape == (2, 18)
    assert w.generate(ids, max_gen_toks=0, return_dict_in_generate=False, kv_cache=True).shape == ids.shape


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("name", ["grouped", "differential"])
def test_cache_in_8_bits(name, device):
    """What a cache in e4m3 leaves of the logits: elements are off by half a step of 2⁻³ at most, 0.036 of their size if even, in every layer after the prompt's."""
    m = make(name, device)
    ids = torch.randint(0, 96, (2, 30), generator=torch.Generator().manual_seed(1)).to(device)
    with torch.no_grad():
        want = m(ids).logits
    got = run(m, ids, list(range(10, 30)), dtype=torch.float8_e4m3fn)
    assert torch.allclose(got[:, :10], want[:, :10], atol=2e-4 * max(1.0, float(want.abs().max())), rtol=0)
    assert float((got - want).norm() / want.norm()) < 0.1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("name,over", [("grouped", dict(n_head=8, n_query_groups=2, head_dim=128)), ("differential", dict(n_head=8, n_query_groups=4, head_dim=64)),
                                       ("cross", dict(n_head=4, n_query_groups=2, head_dim=128, local_window=64)),
                                       ("cross_differential", dict(n_head=4, n_query_groups=2, head_dim=128, local_window=64))])
def test_models_in_bf16(name, over, dtype):
    """Steps over the cache are as near to the model in fp32 as the pass over the whole prefix."""
    over = dict(over, n_embd=256, intermediate_size=512, block_size=256)
    ids = torch.randint(0, 96, (3, 150), generator=torch.Generator().manual_seed(1)).cuda()
    with torch.no_grad():
        exact = make(name, "cuda", torch.float32, **over)(ids).logits
        m = make(name, "cuda", torch.bfloat16, **over)
        whole = m(ids).logits
    got = run(m, ids, [130, *range(131, 140), 143, *range(144, 150)], dtype=dtype)
    off = lambda t: float((t[:, 130:].float() - exact[:, 130:]).norm() / exact[:, 130:].norm())  # noqa: E731
    # the same roundings to bf16 in every layer, at other places: half as much again; with e4m3, a random 0.026 of each key and value through four layers
    assert off(got) <= 1.5 * off(whole) + (0.1 if dtype != torch.bfloat16 else 1e-3)


@pytest.mark.gpu
def test_captured_steps():
    """One captured step, replayed: lengths move on the device, and a second graph on the same cache goes on where the first one stopped."""
    m = make("grouped", "cuda", torch.bfloat16, n_head=8, n_query_groups=2, head_dim=128, n_embd=256, nope=True)
    ids = torch.randint(0, 96, (2, 40), generator=torch.Generator().manual_seed(1)).cuda()
    want = run(m, ids, list(range(10, 40)))
    cache = DecodeCache(m, 2, 40)
    token = ids[:, 10:11].clone()
    with torch.no_grad():
        m(ids[:, :10], cache=cache)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            m(token, cache=cache)                                       # warm-up: token 10
        torch.cuda.current_stream().wait_stream(stream)
        graphs = []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                out = m(token, cache=cache).logits
            graphs.append((g, out))
        for t in range(11, 40):
            token.copy_(ids[:, t:t + 1])
            g, out = graphs[t % 2]
            g.replay()
            assert torch.equal(out[:, 0], want[:, t])
    assert cache.lengths.tolist() == [40, 40]


def test_what_a_cache_refuses():
    m = make("grouped")
    ids = torch.zeros(2, 4, dtype=torch.long)
    with torch.no_grad():
        cache = DecodeCache(m, 2, 6)
        with pytest.raises(ValueError, match="sequences"):
            m(ids[:1], cache=cache)
        m(ids, cache=cache)
        with pytest.raises(ValueError, match="6 tokens"):
            m(ids[:, :3], cache=cache)
        m(ids[:, :2], cache=cache)
    with pytest.raises(RuntimeError, match="no gradients"):
        m(ids, cache=DecodeCache(m, 2, 6))
    for args in ((0, 4), (2, 0)):
        with pytest.raises(ValueError, match="positive"):
            DecodeCache(m, *args)
    with pytest.raises(TypeError):
        DecodeCache(m, 2, 4, dtype=torch.float16)
    for name, over, what in (("samba_d8", dict(head_dim=32), "mamba"), ("sambay_d8", dict(head_dim=32), "mamba"), ("transformer_d8", dict(sc_attn=True), "convolutions"),
                             ("transformer_d8", dict(use_sigmoid=True), "sigmoid"), ("transformer_d8", dict(fa2=False), "root"),
                             ("transformer_d8", dict(use_cu_seqlen=True), "packed"), ("transformer_d8", dict(lc=True), "skipping")):
        other = GPT(Config.from_name(name, **{**SMALL, "n_head": 2, "n_query_groups": 2, "n_layer": 4, **over}))
        assert what in unsupported(other)
        with pytest.raises(ValueError, match="does not cover"):
            DecodeCache(other, 1, 8)
        with pytest.raises(ValueError, match="does not cover"):
            ModelWrapper(other.eval()).generate(ids, max_gen_toks=2, kv_cache=True)


def test_a_call_that_failed_leaves_the_cache_as_it_was():
    m = make("grouped")
    ids = torch.randint(0, 96, (2, 9), generator=torch.Generator().manual_seed(1))
    with torch.no_grad():
        want = m(ids).logits
        cache = DecodeCache(m, 2, 9)
        m(ids[:, :6], cache=cache)
        last = m.transformer.h[-1]
        hook = last.mlp.register_forward_pre_hook(lambda *a: (_ for _ in ()).throw(KeyError("stop")))
        with pytest.raises(KeyError):
            m(ids[:, 6:], cache=cache)
        hook.remove()
        got = m(ids[:, 6:], cache=cache).logits
    assert torch.allclose(got, want[:, 6:], atol=2e-4, rtol=0) and cache.lengths.tolist() == [9, 9]
