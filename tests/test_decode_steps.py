"""Steps over a key-value cache that are captured, replayed, mixed with others, or fail."""
import copy

import pytest
import torch

from archscale_b200.eval import ModelWrapper
from archscale_b200.models.decode import DecodeCache
from test_decode_cache import MODELS, make, run

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
IDS = torch.randint(0, 96, (3, 40), generator=torch.Generator().manual_seed(1))


def near(got, want):
    # the same sums of fp32 in another order: four layers whose values are of the order of one, widths below 100
    return float((got - want).abs().max()) <= 2e-4 * max(1.0, float(want.abs().max()))


@pytest.mark.parametrize("name", list(MODELS))
def test_what_a_captured_call_does(name, monkeypatch):
    """Calls as a capture and its replays make them, on the CPU, where a recorded call also runs: positions come from ``lengths``, the count of the host stays,
    and the next call that is not captured goes on where they stopped."""
    m = make(name)
    cache = DecodeCache(m, 3, 21, page_size=5)
    with torch.no_grad():
        want = m(IDS[:, :21]).logits
        m(IDS[:, :9], cache=cache)
        with monkeypatch.context() as patch:
            patch.setattr(DecodeCache, "_in_capture", lambda self: True, raising=False)
            for a, b in ((9, 10), (10, 11), (11, 14), (14, 15)):
                assert near(m(IDS[:, a:b], cache=cache).logits, want[:, a:b])
                assert cache.tokens == 9
        assert near(m(IDS[:, 15:17], cache=cache).logits, want[:, 15:17]) and cache.tokens == 17
        with monkeypatch.context() as patch:
            patch.setattr(DecodeCache, "_in_capture", lambda self: True, raising=False)
            for t in range(17, 21):
                assert near(m(IDS[:, t:t + 1], cache=cache).logits, want[:, t:t + 1])
            assert bool(m(IDS[:, :1], cache=cache).logits.isnan().all())          # a replay that there is no room for
        assert cache.lengths.tolist() == [22] * 3 and cache.tokens == 22
        with pytest.raises(ValueError, match="22 are there"):
            m(IDS[:, :1], cache=cache)


def test_captures_that_are_refused(monkeypatch):
    m = make("grouped")
    cache = DecodeCache(m, 3, 12)
    with torch.no_grad():
        patch = monkeypatch.setattr
        patch(DecodeCache, "_in_capture", lambda self: True, raising=False)
        with pytest.raises(RuntimeError, match="first tokens"):
            m(IDS[:, :4], cache=cache)
        monkeypatch.undo()
        m(IDS[:, :4], cache=cache)
        hook = m.transformer.h[1].mlp.register_forward_pre_hook(lambda *a: (_ for _ in ()).throw(KeyError("stop")))
        with pytest.raises(KeyError):
            m(IDS[:, 4:6], cache=cache)
        hook.remove()
        patch(DecodeCache, "_in_capture", lambda self: True, raising=False)
        with pytest.raises(RuntimeError, match="failed"):
            m(IDS[:, 4:6], cache=cache)
        monkeypatch.undo()
        assert near(m(IDS[:, 4:6], cache=cache).logits, m(IDS[:, :6]).logits[:, 4:]) and cache.lengths.tolist() == [6] * 3


@pytest.mark.parametrize("part", ["ln_f", "lm_head"])
def test_a_call_that_fails_behind_the_last_layer(part):
    m = make("grouped")
    cache = DecodeCache(m, 3, 9)
    with torch.no_grad():
        want = m(IDS[:, :9]).logits
        for a, b in ((0, 6), (6, 9)):
            module = m.lm_head if part == "lm_head" else m.transformer.ln_f
            hook = module.register_forward_pre_hook(lambda *a: (_ for _ in ()).throw(MemoryError("stop")))
            with pytest.raises(MemoryError):
                m(IDS[:, a:b], cache=cache)
            hook.remove()
            assert cache.tokens == a
            assert near(m(IDS[:, a:b], cache=cache).logits, want[:, a:b])
    assert cache.tokens == 9 and cache.lengths.tolist() == [9] * 3


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [None, torch.float8_e4m3fn])
@pytest.mark.parametrize("name", ["grouped", "differential"])
def test_generation_ends_with_its_token(name, dtype, device):
    """The choices are those of the steps' logits; with one of them as the end of a text, that is where it ends."""
    m = make(name, device)
    w = ModelWrapper(m)
    ids = IDS[:1, :6].repeat(2, 1).to(device)
    kw = dict(max_gen_toks=12, return_dict_in_generate=False, kv_cache=True, kv_cache_dtype=dtype)
    out = w.generate(ids, **kw)
    logits = run(m, out, list(range(6, 18)), dtype=dtype)[:, 5:-1]
    chosen = logits.gather(-1, out[:, 6:, None]).squeeze(-1)
    assert bool((chosen >= logits.amax(-1) - 4e-4 * max(1.0, float(logits.abs().max()))).all())
    with torch.no_grad():
        exact = m(out).logits[:, 5:-1]
    # fp32: other orders of sums; e4m3: elements off by half a step of 2⁻³ at most, 0.036 of their size if even, in every layer
    assert near(logits, exact) if dtype is None else float((logits - exact).norm() / exact.norm()) < 0.1
    for step in (0, 7, 11):
        eos = int(out[0, 6 + step])
        first = out[0, 6:].tolist().index(eos)
        short = w.generate(ids, **kw, eos_token_id=eos)
        assert torch.equal(short, out[:, :6 + first + 1])


def captured(m, cache, token):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m(token, cache=cache).logits
    return graph, out


# experts at widths that their kernels take: the others are sorted with the host's help, which no capture allows
WIDE = dict(n_embd=512, intermediate_size=1024, head_dim=128)


@pytest.mark.gpu
@pytest.mark.parametrize("name,dtype", [(n, t) for n in MODELS for t in (torch.float32, torch.bfloat16) if n != "experts" or t == torch.bfloat16])
def test_replays(name, dtype):
    """Two graphs on one cache and calls that are not captured, in turn: bit for bit the steps that are not captured."""
    m = make(name, "cuda", dtype, **(WIDE if name == "experts" else {}))
    ids = IDS.cuda()
    want = run(m, ids, list(range(10, 40)))
    cache = DecodeCache(m, 3, 40)
    token = ids[:, 10:11].clone()
    with torch.no_grad():
        m(ids[:, :10], cache=cache)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            m(token, cache=cache)
        torch.cuda.current_stream().wait_stream(side)
        graphs = [captured(m, cache, token) for _ in range(2)]
        assert cache.tokens == 11
        other = ids[:, :7].repeat(1, 40)                             # the model's own rotary table grows meanwhile
        m(other)
        for t in range(11, 40):
            if t % 5 == 0:
                assert torch.equal(m(ids[:, t:t + 1], cache=cache).logits[:, 0], want[:, t]), t
                continue
            token.copy_(ids[:, t:t + 1])
            graph, out = graphs[t % 2]
            graph.replay()
            assert torch.equal(out[:, 0], want[:, t]), t
        assert cache.tokens == 40
        graphs[0][0].replay()
        assert bool(graphs[0][1].isnan().all())
        with pytest.raises(ValueError, match="41 are there"):
            m(token, cache=cache)


@pytest.mark.parametrize("name", ["grouped", "windowed_rotary"])
def test_copies_of_a_cache(name, monkeypatch):
    """A copy goes on by itself, captured or not, and holds no copy of the model."""
    m = make(name)

    def refuse(self, memo):
        raise AssertionError("a copy of a module")

    cache = DecodeCache(m, 3, 12, page_size=5)
    with torch.no_grad():
        want = m(IDS[:, :12]).logits
        m(IDS[:, :7], cache=cache)
        with monkeypatch.context() as patch:
            patch.setattr(torch.nn.Module, "__deepcopy__", refuse, raising=False)
            other = copy.deepcopy(cache)
        for c in (other, cache):
            assert near(m(IDS[:, 7:9], cache=c).logits, want[:, 7:9])
            with monkeypatch.context() as patch:
                patch.setattr(DecodeCache, "_in_capture", lambda self: True)
                for t in (9, 10, 11):
                    assert near(m(IDS[:, t:t + 1], cache=c).logits, want[:, t:t + 1])
