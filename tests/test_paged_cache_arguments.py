"""What ``PagedCache`` refuses, on the CPU: every check stands in front of the look at the device, and of any change."""

import pytest
import torch

import adasplash_amd as A
from adasplash_amd.paged import PagedCache


def cache_of():
    return PagedCache(8, 16, 2, 2, 64, 100, dtype=torch.float32, device="cpu")


@pytest.mark.parametrize("k, v, new", [
    (torch.zeros(5, 2, 64, dtype=torch.float16), torch.zeros(5, 2, 64, dtype=torch.float16), torch.tensor([3, 2])),
    (torch.zeros(5, 3, 64), torch.zeros(5, 3, 64), torch.tensor([3, 2])),
    (torch.zeros(5, 2, 32), torch.zeros(5, 2, 32), torch.tensor([3, 2])),
    (torch.zeros(5, 2, 64), torch.zeros(4, 2, 64), torch.tensor([3, 2])),
    (torch.zeros(5, 2, 64), torch.zeros(5, 2, 64, dtype=torch.float16), torch.tensor([3, 2])),
    (torch.zeros(5, 64), torch.zeros(5, 64), torch.tensor([3, 2])),
    (torch.zeros(5, 2, 64), torch.zeros(5, 2, 64), torch.tensor([3, 2, 0])),
    (torch.zeros(5, 2, 64), torch.zeros(5, 2, 64), torch.tensor([3.0, 2.0])),
    (torch.zeros(2, 2, 64), torch.zeros(3, 2, 64), None),
])
def test_append_refuses(k, v, new):
    with pytest.raises(AssertionError):
        cache_of().append(k, v, new)


def test_append_has_no_gradient():
    with pytest.raises(RuntimeError, match="no gradient"):
        cache_of().append(torch.zeros(2, 2, 64, requires_grad=True), torch.zeros(2, 2, 64))


def test_a_cpu_tensor_is_refused_behind_the_other_checks():
    for new in (None, torch.tensor([1, 1])):
        with pytest.raises(RuntimeError, match="ROCm device only"):
            cache_of().append(torch.zeros(2, 2, 64), torch.zeros(2, 2, 64), new)
    with pytest.raises(RuntimeError, match="ROCm device only"):
        cache_of().append(torch.zeros(2, 2, 1, 64), torch.zeros(2, 2, 1, 64))


def test_inference_tensors_are_not_written_to_outside_of_the_mode():
    with torch.inference_mode():
        cache = cache_of()
        pages = torch.zeros(5, 2, 16, 64)
    for call in (
        lambda: cache.append(torch.zeros(2, 2, 64), torch.zeros(2, 2, 64)),
        lambda: A.write_pages(torch.zeros(2, 2, 64), torch.zeros(2, 2, 64), torch.arange(2), pages, torch.zeros(5, 2, 16, 64)),
        lambda: A.write_pages(torch.zeros(2, 2, 64), torch.zeros(2, 2, 64), torch.arange(2), torch.zeros(5, 2, 16, 64), pages),
        lambda: A.build_block_tables(torch.zeros(2, dtype=torch.int32), torch.ones(2, dtype=torch.int32), cache.block_tables, torch.arange(8, dtype=torch.int32),
                                     torch.tensor([0, 8]), 16, 2),
    ):
        with pytest.raises(RuntimeError, match="inference"):
            call()
        with torch.inference_mode(), pytest.raises(RuntimeError, match="ROCm device only"):
            call()
