"""Autograd knows that a write changes a cache."""
import pytest
import torch

from archscale_b200 import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float8_e4m3fn])
def test_a_write_counts_as_one(dtype, device):
    cache = ops.new_paged_cache(3, 2, 4, 16, dtype, device)
    table, lengths = torch.tensor([[2, 0]], dtype=torch.int32, device=device), torch.tensor([6], dtype=torch.int32, device=device)
    x = torch.randn(1, 6, 2, 16, device=device)
    parts = [t for t in cache if t is not None]
    before = [t._version for t in parts]
    ops.paged_cache_write(cache, x, x, table, lengths)
    assert all(t._version > n for t, n in zip(parts, before))
    before = [t._version for t in parts]
    ops.paged_cache_read(cache, table, lengths, 6)
    with torch.no_grad():
        ops.paged_attention(x.bfloat16(), cache, table, lengths)
    assert [t._version for t in parts] == before
    with torch.inference_mode():                                            # tensors made there have no version, and others may be written there
        ops.paged_cache_write(cache, x, x, table, lengths)
        ops.paged_cache_write(ops.new_paged_cache(3, 2, 4, 16, dtype, device), x, x, table, lengths)


@pytest.mark.parametrize("device", DEVICES)
def test_a_gradient_through_old_keys_is_refused(device):
    """A product that saved cached keys for its gradient must not get the new ones instead."""
    cache = ops.new_paged_cache(3, 2, 4, 16, torch.float32, device)
    table, lengths = torch.tensor([[2, 0]], dtype=torch.int32, device=device), torch.tensor([6], dtype=torch.int32, device=device)
    x = torch.randn(1, 6, 2, 16, device=device)
    w = torch.ones(16, device=device, requires_grad=True)
    y = (cache.k[2] * w).sum()
    ops.paged_cache_write(cache, x, x, table, lengths)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
