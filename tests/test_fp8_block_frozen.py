"""Frozen 8-bit layers: a stored weight is never used once the weight has changed, whatever changed it."""
import copy
import io
import os

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from archscale_b200.config import Config
from archscale_b200.models.gpt import GPT, Block
from archscale_b200.models.layers import Linear, apply_fp8_block, freeze_fp8_block
from archscale_b200.optim.sharded import ShardedOptimizer
from archscale_b200.parallel.fsdp import FSDPEngine
from archscale_b200.parallel.mesh import build_mesh


def _layer(seed=0):
    torch.manual_seed(seed)
    lin = Linear(160, 200, bias=True)
    lin.fp8_block = True
    return lin, torch.randn(5, 160)


def _model():
    torch.manual_seed(3)
    m = GPT(Config.from_name("transformer_gqa4_d8", n_layer=2, n_embd=64, ar=None, n_head=2, n_query_groups=1, head_dim=32, intermediate_size=96,
                             block_size=32, padded_vocab_size=128, vocab_size=128))
    m.reset_parameters()
    m.compute_dtype = torch.float32
    apply_fp8_block(m)
    return m


def _engine(m):
    return FSDPEngine(m, build_mesh(), unit_classes=(Block,), param_dtype=torch.float32)


def _train(m, eng, opt, idx):
    eng.backward(m(idx).logits.float().square().mean())
    opt.step()
    opt.zero_grad()


def _fresh(m, idx):
    """Logits with weights that are frozen now."""
    freeze_fp8_block(m)
    with torch.no_grad():
        return m(idx).logits


def test_a_training_step_of_the_engine_is_noticed():
    m = _model()
    eng = _engine(m)
    opt = ShardedOptimizer(eng, lr=1e-2, betas=(0.9, 0.95), algorithm="adamw")
    idx = torch.randint(0, 128, (2, 16))
    before = _fresh(m, idx)                       # before the first forward pass: the weights are gathered for it
    with torch.no_grad():
        assert torch.equal(m(idx).logits, before)
    _train(m, eng, opt, idx)
    with torch.no_grad(), pytest.raises(RuntimeError, match="frozen"):
        m(idx)
    after = _fresh(m, idx)
    assert not torch.equal(after, before)
    freeze_fp8_block(m, False)
    with torch.no_grad():
        assert torch.equal(m(idx).logits, after)


def test_a_load_through_the_engine_is_noticed():
    m = _model()
    eng = _engine(m)
    idx = torch.randint(0, 128, (2, 16))
    before = _fresh(m, idx)
    eng.load_full_state_dict({n: t * 1.5 if t.dim() == 2 else t for n, t in eng.full_state_dict().items()})
    with torch.no_grad(), pytest.raises(RuntimeError, match="frozen"):
        m(idx)
    assert not torch.equal(_fresh(m, idx), before)


def test_other_engines_steps_do_not_disturb():
    teacher, student = _model(), _model()
    idx = torch.randint(0, 128, (2, 16))
    want = _fresh(teacher, idx)
    eng = _engine(student)
    _train(student, eng, ShardedOptimizer(eng, lr=1e-2, betas=(0.9, 0.95), algorithm="adamw"), idx)
    with torch.no_grad():
        assert torch.equal(teacher(idx).logits, want)


CHANGES = {
    "operation": lambda l: l.weight.mul_(2.0),
    "detached": lambda l: l.weight.detach().mul_(2.0),
    "state dict": lambda l: l.load_state_dict({k: 2 * v for k, v in l.state_dict().items()}),
    "state dict, assigned": lambda l: l.load_state_dict({k: 2 * v for k, v in l.state_dict().items()}, assign=True),
    "new memory": lambda l: setattr(l.weight, "data", l.weight.data * 2),
    "new parameter": lambda l: setattr(l, "weight", torch.nn.Parameter(l.weight * 2)),
    "flat vector": lambda l: torch.nn.utils.vector_to_parameters(2 * torch.nn.utils.parameters_to_vector(l.parameters()), l.parameters()),
    "type": lambda l: l.to(torch.bfloat16),
}


@pytest.mark.parametrize("what", CHANGES)
def test_changes_are_noticed(what):
    lin, x = _layer()
    freeze_fp8_block(lin)
    with torch.no_grad():
        lin(x)
        CHANGES[what](lin)
        with pytest.raises(RuntimeError, match="frozen"):
            lin(x)
        freeze_fp8_block(lin)
        stored = lin(x)
        freeze_fp8_block(lin, False)
        assert torch.equal(lin(x), stored)


def test_an_optimizer_that_writes_data():
    """Updates through ``.data`` move no version; the gradients that they follow come from a call that drops the stored weight."""
    lin, x = _layer()
    freeze_fp8_block(lin)
    for _ in range(2):
        lin(x).square().sum().backward()
        lin.weight.data.sub_(lin.weight.grad, alpha=1e-2)
        with torch.no_grad():
            got = lin(x)
            fresh = Linear(160, 200, bias=True)
            fresh.load_state_dict(lin.state_dict())
            fresh.fp8_block = True
            assert torch.equal(got, fresh(x))


def test_gradients_of_inputs_alone_keep_it():
    lin, x = _layer()
    lin.weight.requires_grad_(False)
    freeze_fp8_block(lin)
    lin(x.requires_grad_()).sum().backward()
    assert x.grad is not None
    with torch.no_grad():
        assert lin.stored_fp8() is not None


def test_copies_and_pickles_are_frozen_or_live():
    lin, x = _layer()
    with torch.no_grad():
        lin.weight.mul_(0.5)                                           # a version that a copy does not have
        freeze_fp8_block(lin)
        want = lin(x)
        buf = io.BytesIO()
        torch.save(lin, buf)
        buf.seek(0)
        for other in (copy.deepcopy(lin), torch.load(buf, weights_only=False)):
            assert other.stored_fp8() is not None and torch.equal(other(x), want)
            other.weight.mul_(2.0)
            with pytest.raises(RuntimeError, match="frozen"):
                other(x)
            assert torch.equal(lin(x), want)
        lin.weight.mul_(2.0)                                           # a copy of a changed layer takes its weight as it is
        other = copy.deepcopy(lin)
        freeze_fp8_block(lin)
        assert other.stored_fp8() is None and torch.equal(other(x), lin(x))


def test_weights_without_a_version_are_refused():
    with torch.inference_mode():
        lin = Linear(160, 200)
    lin.fp8_block = True
    with pytest.raises(RuntimeError, match="inference_mode"):
        freeze_fp8_block(lin)
    with torch.no_grad():
        assert lin(torch.randn(2, 160)).shape == (2, 200)


def _worker(rank, world, port, q):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE=str(world))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        idx = torch.randint(0, 128, (2, 16), generator=torch.Generator().manual_seed(0))
        whole = _model()
        with torch.no_grad():
            want = whole(idx).logits
        m = _model()
        eng = _engine(m)
        opt = ShardedOptimizer(eng, lr=1e-2, betas=(0.9, 0.95), algorithm="adamw")
        got = _fresh(m, idx)
        with torch.no_grad():
            again = m(idx).logits                                       # units were sharded and gathered in between
        _train(m, eng, opt, idx)
        with torch.no_grad():
            try:
                m(idx)
                raised = False
            except RuntimeError as e:
                raised = "frozen" in str(e)
        after = _fresh(m, idx)
        q.put((rank, torch.equal(got, want), torch.equal(again, want), raised, torch.equal(after, want)))
        dist.barrier()
    finally:
        dist.destroy_process_group()


def test_two_ranks():
    ctx = mp.get_context("spawn")
    q = ctx.SimpleQueue()
    mp.spawn(_worker, args=(2, 29641, q), nprocs=2, join=True)
    for _ in range(2):
        rank, got, again, raised, same = q.get()
        assert got and again and raised and not same, rank


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_inference_mode(device):
    """Frozen and live layers in it, a store that was made in it, and a change that is made in it."""
    lin, x = _layer()
    lin, x = lin.to(device), x.to(device)
    with torch.no_grad():
        want = lin(x)
    with torch.inference_mode():
        assert torch.equal(lin(x), want)
        freeze_fp8_block(lin)
        assert lin.stored_fp8() is not None and torch.equal(lin(x), want)
    with torch.no_grad():
        assert torch.equal(lin(x), want)
    with torch.inference_mode():
        lin.weight.mul_(2.0)
        with pytest.raises(RuntimeError, match="frozen"):
            lin(x)
    freeze_fp8_block(lin)
    lin(x).sum().backward()
    assert lin.weight.grad is not None
