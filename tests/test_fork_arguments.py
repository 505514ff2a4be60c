"""What ``fork_requests``, ``compact_pages`` and a prefix table refuse, on the CPU: every check stands in front of the look at the device, and of any change."""

import pytest
import torch

import adasplash_amd as A
from adasplash_amd.paged import PagedCache


def _fork(**change):
    a = {"parents": torch.tensor([0, 0]), "lengths": torch.tensor([3, 0], dtype=torch.int32), "block_tables": torch.full((2, 4), -1, dtype=torch.int32),
         "free_pages": torch.arange(8, dtype=torch.int32), "free_range": torch.tensor([1, 8]), "shares": torch.zeros(8, dtype=torch.int32),
         "k_pages": torch.zeros(8, 2, 16, 64), "v_pages": torch.zeros(8, 2, 16, 64)}
    a.update(change)
    return A.fork_requests(**a)


def _compact(**change):
    a = {"lengths": torch.tensor([3, 0], dtype=torch.int32), "block_tables": torch.full((2, 4), -1, dtype=torch.int32), "k_pages": torch.zeros(8, 2, 16, 64),
         "v_pages": torch.zeros(8, 2, 16, 64), "k_to": torch.zeros(5, 2, 16, 64), "v_to": torch.zeros(5, 2, 16, 64)}
    a.update(change)
    return A.compact_pages(**a)


@pytest.mark.parametrize("change, text", [
    ({"parents": torch.tensor([0])}, "parents"),
    ({"parents": torch.tensor([0.0, 0.0])}, "int32/int64"),
    ({"lengths": torch.zeros(3, dtype=torch.int32)}, "lengths"),
    ({"lengths": torch.zeros(4, dtype=torch.int32)[::2]}, "contiguous"),
    ({"block_tables": torch.zeros(2, 4, dtype=torch.int64)}, "int32"),
    ({"block_tables": torch.zeros(2, 8, dtype=torch.int32)[:, ::2]}, "unit stride"),
    ({"block_tables": torch.zeros(1, 4, dtype=torch.int32).expand(2, 4)}, "overlap"),
    ({"block_tables": torch.zeros(2, 0, dtype=torch.int32)}, "int32"),
    ({"free_pages": torch.arange(8)}, "free_pages"),
    ({"free_pages": torch.zeros(0, dtype=torch.int32)}, "free_pages"),
    ({"free_pages": torch.arange(16, dtype=torch.int32)[::2]}, "free_pages"),
    ({"free_range": torch.tensor([0, 8], dtype=torch.int32)}, "free_range"),
    ({"free_range": torch.tensor([0, 8, 8])}, "free_range"),
    ({"shares": torch.zeros(7, dtype=torch.int32)}, "shares"),
    ({"shares": torch.zeros(8, dtype=torch.int64)}, "shares"),
    ({"shares": torch.zeros(16, dtype=torch.int32)[::2]}, "shares"),
    ({"v_pages": torch.zeros(8, 2, 16, 32)}, "share one shape"),
    ({"v_pages": torch.zeros(8, 2, 16, 64, dtype=torch.float16)}, "dtype"),
    ({"k_pages": torch.zeros(8, 2, 16, 6), "v_pages": torch.zeros(8, 2, 16, 6)}, "16"),
    ({"k_pages": torch.zeros(1, 2, 16, 64).expand(8, 2, 16, 64)}, "16-byte aligned rows"),
])
def test_fork_refuses(change, text):
    with pytest.raises(AssertionError, match=text):
        _fork(**change)


@pytest.mark.parametrize("change, text", [
    ({"lengths": torch.zeros(3, dtype=torch.int32)}, "lengths"),
    ({"block_tables": torch.zeros(2, 4, dtype=torch.int64)}, "int32"),
    ({"k_to": torch.zeros(5, 2, 16, 32), "v_to": torch.zeros(5, 2, 16, 32)}, "both pools"),
    ({"k_to": torch.zeros(5, 2, 8, 64), "v_to": torch.zeros(5, 2, 8, 64)}, "both pools"),
    ({"k_to": torch.zeros(5, 1, 16, 64), "v_to": torch.zeros(5, 1, 16, 64)}, "both pools"),
    ({"k_to": torch.zeros(5, 2, 16, 64, dtype=torch.float16), "v_to": torch.zeros(5, 2, 16, 64, dtype=torch.float16)}, "both pools"),
    ({"v_to": torch.zeros(6, 2, 16, 64)}, "share one shape"),
    ({"k_to": torch.zeros(0, 2, 16, 64), "v_to": torch.zeros(0, 2, 16, 64)}, "hold pages"),
    ({"k_to": torch.zeros(1, 2, 16, 64).expand(5, 2, 16, 64)}, "16-byte aligned rows"),
])
def test_compact_refuses(change, text):
    with pytest.raises(AssertionError, match=text):
        _compact(**change)


def test_a_pool_of_its_own():
    k, v, to = torch.zeros(8, 2, 16, 64), torch.zeros(8, 2, 16, 64), torch.zeros(5, 2, 16, 64)
    for change in ({"k_to": k, "v_to": v}, {"k_to": k[:5], "v_to": to}, {"k_to": v[:5], "v_to": to}, {"k_to": to, "v_to": k[3:]}, {"k_to": to, "v_to": to}):
        with pytest.raises(AssertionError, match="tensors"):
            _compact(**{"k_pages": k, "v_pages": v, **change})


def test_a_cpu_tensor_is_refused_behind_the_other_checks():
    for call in (_fork, _compact):
        with pytest.raises(RuntimeError, match="ROCm device only"):
            call()
        with pytest.raises(RuntimeError, match="no gradient"):
            call(k_pages=torch.zeros(8, 2, 16, 64, requires_grad=True))
    cache = PagedCache(8, 16, 2, 2, 64, 100, dtype=torch.float32, device="cpu")
    for call in (lambda: cache.fork(torch.tensor([0, 0])), lambda: cache.release(1), lambda: cache.release([0, 1]), lambda: cache.resize(4)):
        with pytest.raises(RuntimeError, match="ROCm device only"):
            call()
    for request in (2, -3, [0, 2]):
        with pytest.raises(IndexError):
            cache.release(request)
    for request in (torch.tensor([True, False]), torch.tensor(1.0), 1.0, [0.5], None):
        with pytest.raises(TypeError):
            cache.release(request)
    with pytest.raises(ValueError):
        cache.resize(0)
    with torch.inference_mode():
        pages = torch.zeros(8, 2, 16, 64)
    with pytest.raises(RuntimeError, match="inference"):
        _fork(k_pages=pages)
    with pytest.raises(RuntimeError, match="inference"):
        _compact(k_to=pages, v_to=torch.zeros(8, 2, 16, 64))


@pytest.mark.parametrize("prefix", [torch.zeros(2, dtype=torch.int64), torch.zeros(1, 2, dtype=torch.int32)])
def test_a_prefix_table_is_int32(prefix):
    with pytest.raises(AssertionError, match="prefix_table"):
        A.paged_attention(torch.zeros(2, 8, 1, 64), torch.zeros(5, 2, 16, 64), torch.zeros(5, 2, 16, 64), torch.zeros(2, 3, dtype=torch.int32),
                          torch.ones(2, dtype=torch.int32), prefix_table=prefix)
