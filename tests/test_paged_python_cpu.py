"""The Python entries of the paged cache on tensors that are not on a GPU: refused, on any host."""
import pytest
import torch

from picolm_qwen_b200 import abi, runtime


def test_tensors_on_the_cpu_are_refused():
    cfg = abi.Config.make(1, 4, 2, 64, 64, 1e4)
    cache = runtime.PagedCache(cfg, 16, 4, device="cpu")
    i32 = dict(dtype=torch.int32)
    batch = cache.batch(torch.zeros((1, 4), **i32), torch.tensor([0, 1], **i32), torch.tensor([5], **i32), 1, 1, 64)
    q, k = torch.zeros((1, 4, 64)).half(), torch.zeros((1, 2, 64)).half()
    tab = torch.zeros((64, 32)), torch.zeros((64, 32))
    with pytest.raises(ValueError):
        cache.attend(0, batch, q, torch.empty_like(q))
    with pytest.raises(ValueError):
        cache.append(0, batch, q, k, k, *tab, torch.empty_like(q))
    with pytest.raises(ValueError):
        batch.status()
    with pytest.raises(ValueError):
        runtime.rope(q, None, torch.zeros(1, **i32), *tab, torch.empty_like(q), None, torch.zeros(256, dtype=torch.uint8))
