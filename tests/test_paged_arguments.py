"""What the paged cache's entry points refuse, on the CPU: every check stands in front of the look at the device."""

import pytest
import torch

import adasplash_amd as A
from adasplash_amd.paged import PagedCache


def _call(**change):
    a = {
        "q": torch.zeros(2, 8, 1, 64),
        "k_pages": torch.zeros(5, 2, 16, 64),
        "v_pages": torch.zeros(5, 2, 16, 64),
        "block_tables": torch.zeros(2, 3, dtype=torch.int32),
        "lengths": torch.ones(2, dtype=torch.int32),
    }
    a.update(change)
    return A.paged_attention(**a)


def test_a_cpu_tensor_is_refused_behind_the_other_checks():
    with pytest.raises(RuntimeError, match="ROCm device only"):
        _call()


@pytest.mark.parametrize("change, text", [
    ({"q": torch.zeros(2, 8, 2, 64)}, "one new token"),
    ({"q": torch.zeros(2, 8, 64)}, "one new token"),
    ({"q": torch.zeros(2, 7, 1, 64)}, "multiple"),
    ({"q": torch.zeros(2, 130, 1, 64)}, "at most 64"),
    ({"q": torch.zeros(2, 8, 1, 32)}, "head_dim"),
    ({"q": torch.zeros(2, 8, 1, 48), "k_pages": torch.zeros(5, 2, 16, 48), "v_pages": torch.zeros(5, 2, 16, 48)}, "head_dim must be"),
    ({"q": torch.zeros(2, 8, 1, 64, dtype=torch.bfloat16)}, "share a dtype"),
    ({"v_pages": torch.zeros(5, 2, 16, 64, dtype=torch.bfloat16)}, "share a dtype"),
    ({"v_pages": torch.zeros(4, 2, 16, 64)}, "share one shape"),
    ({"k_pages": torch.zeros(5, 2, 16, 128)[..., ::2], "v_pages": torch.zeros(5, 2, 16, 64)}, "unit stride"),
    ({"k_pages": torch.zeros(5, 2, 16, 66)[..., 1:65], "v_pages": torch.zeros(5, 2, 16, 64)}, "unit stride"),
    ({"k_pages": torch.zeros(0, 2, 16, 64), "v_pages": torch.zeros(0, 2, 16, 64)}, "hold pages"),
    ({"block_tables": torch.zeros(3, 3, dtype=torch.int32)}, "block_tables"),
    ({"block_tables": torch.zeros(2, 3, dtype=torch.int64)}, "int32"),
    ({"block_tables": torch.zeros(2, 6, dtype=torch.int32)[:, ::2]}, "unit stride"),
    ({"block_tables": torch.zeros(1, 3, dtype=torch.int32).expand(2, 3)}, "overlap"),
    ({"lengths": torch.ones(3, dtype=torch.int32)}, "lengths"),
    ({"lengths": torch.ones(2)}, "int32/int64"),
    ({"alpha": 1.0}, "alpha"),
    ({"alpha": 2.5}, "alpha"),
    ({"alpha": float("nan")}, "alpha"),
    ({"max_length": 49}, "max_length"),
    ({"max_length": -1}, "max_length"),
])
def test_paged_attention_refuses(change, text):
    with pytest.raises(AssertionError, match=text):
        _call(**change)


def test_paged_attention_has_no_gradient():
    with pytest.raises(RuntimeError, match="no gradient"):
        _call(q=torch.zeros(2, 8, 1, 64, requires_grad=True))
    with torch.no_grad(), pytest.raises(RuntimeError, match="ROCm device only"):
        _call(q=torch.zeros(2, 8, 1, 64, requires_grad=True))


def test_unknown_types():
    with pytest.raises(TypeError):
        _call(q=torch.zeros(2, 8, 1, 64, dtype=torch.float64), k_pages=torch.zeros(5, 2, 16, 64, dtype=torch.float64),
              v_pages=torch.zeros(5, 2, 16, 64, dtype=torch.float64))


def _tables(**change):
    a = {
        "lengths": torch.zeros(2, dtype=torch.int32),
        "new_tokens": torch.ones(2, dtype=torch.int32),
        "block_tables": torch.zeros(2, 3, dtype=torch.int32),
        "free_pages": torch.arange(5, dtype=torch.int32),
        "free_range": torch.tensor([0, 5]),
        "page_size": 16,
        "total_tokens": 2,
    }
    a.update(change)
    return A.build_block_tables(**a)


@pytest.mark.parametrize("change, text", [
    ({"lengths": torch.zeros(3, dtype=torch.int32)}, "lengths"),
    ({"new_tokens": torch.ones(2)}, "new_tokens"),
    ({"block_tables": torch.zeros(2, 3, dtype=torch.int64)}, "int32"),
    ({"block_tables": torch.zeros(1, 3, dtype=torch.int32).expand(2, 3)}, "overlap"),
    ({"block_tables": torch.zeros(2, 0, dtype=torch.int32)}, "int32"),
    ({"block_tables": torch.zeros(8193, 1, dtype=torch.int32)}, "8192"),
    ({"free_pages": torch.zeros(0, dtype=torch.int32)}, "free_pages"),
    ({"free_pages": torch.zeros(5)}, "free_pages"),
    ({"free_range": torch.zeros(2, dtype=torch.int32)}, "free_range"),
    ({"free_range": torch.zeros(3, dtype=torch.int64)}, "free_range"),
    ({"page_size": 0}, "page_size"),
    ({"total_tokens": -1}, "total_tokens"),
    ({"block_tables": torch.zeros(2, 1 << 12, dtype=torch.int32), "page_size": 1 << 20}, "2\\^31"),
])
def test_build_block_tables_refuses(change, text):
    with pytest.raises(AssertionError, match=text):
        _tables(**change)
    with pytest.raises(RuntimeError, match="ROCm device only"):
        _tables()


def _write(**change):
    a = {
        "k": torch.zeros(4, 2, 64),
        "v": torch.zeros(4, 2, 64),
        "slots": torch.arange(4),
        "k_pages": torch.zeros(5, 2, 16, 64),
        "v_pages": torch.zeros(5, 2, 16, 64),
    }
    a.update(change)
    return A.write_pages(**a)


@pytest.mark.parametrize("change, text", [
    ({"k": torch.zeros(4, 3, 64), "v": torch.zeros(4, 3, 64)}, "shape"),
    ({"k": torch.zeros(4, 2, 32), "v": torch.zeros(4, 2, 32)}, "shape"),
    ({"v": torch.zeros(3, 2, 64)}, "shape"),
    ({"k": torch.zeros(4, 2, 64, dtype=torch.float16)}, "dtype"),
    ({"slots": torch.arange(3)}, "slots"),
    ({"slots": torch.arange(4, dtype=torch.int32)}, "slots"),
    ({"k_pages": torch.zeros(1, 2, 16, 64).expand(5, 2, 16, 64)}, "unit stride"),
    ({"k": torch.zeros(4, 2, 6), "v": torch.zeros(4, 2, 6), "k_pages": torch.zeros(5, 2, 2, 6), "v_pages": torch.zeros(5, 2, 2, 6)}, "16-byte|16 bytes"),
])
def test_write_pages_refuses(change, text):
    with pytest.raises(AssertionError, match=text):
        _write(**change)
    with pytest.raises(RuntimeError, match="ROCm device only"):
        _write()


def test_paged_cache_refuses():
    with pytest.raises(ValueError):
        PagedCache(0, 16, 2, 2, 64, 100, device="cpu")
    cache = PagedCache(8, 16, 2, 2, 64, 100, dtype=torch.float32, device="cpu")
    assert cache.block_tables.shape == (2, 7)
    with pytest.raises(ValueError, match="one token of each"):
        cache.append(torch.zeros(3, 2, 64), torch.zeros(3, 2, 64))
