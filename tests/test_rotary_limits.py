"""How many rows ``rotary`` takes, on the CPU: a launch has fewer than 2^32 threads along an axis, eight elements of a head to each.  (Tensors of one row, seen many times.)"""

import ctypes

import pytest
import torch

import adasplash_amd as A
from adasplash_amd import _lib
from adasplash_amd.paged import PagedCache

MOST = (1 << 24) - 1  # workgroups of 256


def rows(tokens, D, heads=1):
    return torch.zeros(1, 1, 1, D).expand(1, heads, tokens, D)


def positions(tokens):
    return torch.zeros(1, dtype=torch.int64).expand(tokens)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_rows_of_a_head(D):
    f, most = torch.zeros(D // 2, dtype=torch.float64), MOST * 2048 // D
    with pytest.raises(RuntimeError, match="ROCm device only"):
        A.rotary(rows(most - 8, D), None, positions(most - 8), f)
    for tokens in (most + 8, 1 << 31):
        with pytest.raises(AssertionError, match="elements of a head"):
            A.rotary(rows(tokens, D), None, positions(tokens), f)
        with pytest.raises(AssertionError, match="elements of a head"):
            A.rotary(rows(tokens, D), rows(tokens, D), positions(tokens), f)
        k, slots = rows(tokens, D)[0].transpose(0, 1), positions(tokens)
        pages = torch.zeros(2, 1, 16, D)
        with pytest.raises(AssertionError, match="elements of a head"):
            A.write_pages(k, k, slots, pages, pages.clone(), positions=slots, rotary=A.Rotary(f))
        cache = PagedCache(2, 16, 1, 1, D, 30, dtype=torch.float32, device="cpu", rotary=A.Rotary(f))
        with pytest.raises(AssertionError, match="elements of a head"):
            cache.append(k, k, torch.ones(1, dtype=torch.int32))
        assert cache.lengths.tolist() == [0]


@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
def test_the_c_calls_refuse_the_same(D):
    """Sizes are looked at before anything is launched: a call with too many rows returns the status of a shape."""
    lib = _lib.load()
    some = ctypes.create_string_buffer(4096)
    at = (ctypes.addressof(some) + 255) // 256 * 256
    strides = (ctypes.c_int64 * 18)()
    shape = 1 << 31 if D == 16 else MOST * 2048 // D + 1
    tokens = min(shape, 0x7fff0001)
    refused = lib.adsp_rotary_fwd(at, None, at, None, at, 64, 0, 0, at, None, 0, None, 0, 1, 1, 0, tokens, D, 8, 0, ctypes.addressof(strides), 1e-6, 1.0, 0, None)
    empty = lib.adsp_rotary_fwd(at, None, at, None, at, 64, 0, 0, at, None, 0, None, 0, 1, 1, 0, 0, D, 8, 0, ctypes.addressof(strides), 1e-6, 1.0, 0, None)
    assert refused == empty != 0
    assert lib.adsp_paged_write_rotary(at, at, at, at, at, at, 64, 0, at, None, 0, tokens, 1, D, 8, 0, 1, 16, ctypes.addressof(strides), 1e-6, 1.0, 0, None) == empty
