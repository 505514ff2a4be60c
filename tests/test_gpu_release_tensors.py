"""``PagedCache.release`` of numbers that lie in tensors, on the host or the device."""

import pytest
import torch

from adasplash_amd.paged import PagedCache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("request_", [torch.tensor(1), torch.tensor([1]), torch.tensor(1, dtype=torch.int32), torch.tensor([[1, 9], [-1, 1]]), torch.zeros(0, dtype=torch.int64)])
def test_host_and_device(request_):
    states = []
    for where in ("cpu", "cuda"):
        cache = PagedCache(20, 4, 3, 1, 32, 30)
        rows = torch.ones(17, 1, 32, dtype=torch.bfloat16, device="cuda")
        cache.append(rows, rows, torch.tensor([5, 9, 3], device="cuda"))
        cache.release(request_.to(where))
        states.append([t.tolist() for t in (cache.lengths, cache.block_tables, cache.free_pages, cache.free_range, cache.shares)])
    assert states[0] == states[1]
    assert states[0][0] == ([5, 0, 3] if request_.numel() else [5, 9, 3])
