"""Keys and values with one token, or one head, whose stride along that dimension is any number: they are written as contiguous ones are, and an ``append`` of them is not refused half way."""

import pytest
import torch

import adasplash_amd as A
from adasplash_amd.paged import PagedCache
from tests import positions_reference as pos

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rows_of(T, H, D, dtype, seed):
    """The same rows twice: contiguous, and with odd strides along the dimensions of one entry."""
    x = torch.randn(T, H, D, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)
    odd = x.as_strided(x.shape, (D * H + 1 if T == 1 else D * H, D + 3 if H == 1 else D, 1))
    assert torch.equal(odd, x) and odd.stride() != x.stride()
    return x, odd


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T, H", [(1, 2), (5, 1), (1, 1)])
@pytest.mark.parametrize("turned", [False, True])
def test_write_pages(dtype, T, H, turned):
    D, page = 64, 4
    more = {"positions": torch.arange(T, device=DEV) + 7, "rotary": A.Rotary(pos.frequencies_of(D).to(DEV))} if turned else {}
    slots = torch.arange(T, device=DEV) * 3 + 1
    pools = []
    for k, v in zip(rows_of(T, H, D, dtype, 1), rows_of(T, H, D, dtype, 2)):
        kp, vp = (torch.zeros(6, H, page, D, dtype=dtype, device=DEV) for _ in range(2))
        A.write_pages(k, v, slots, kp, vp, **more)
        pools.append((kp, vp))
    assert torch.equal(pools[0][0], pools[1][0]) and torch.equal(pools[0][1], pools[1][1]) and pools[0][1].any()


@pytest.mark.parametrize("batch, H", [(1, 2), (3, 1), (1, 1)])
@pytest.mark.parametrize("turned", [False, True])
def test_append(batch, H, turned):
    D = 64
    turn = A.Rotary(pos.frequencies_of(D).to(DEV)) if turned else None
    caches = [PagedCache(8, 4, batch, H, D, 12, rotary=turn) for _ in range(2)]
    for step in range(6):
        for cache, k, v in zip(caches, rows_of(batch, H, D, torch.bfloat16, step), rows_of(batch, H, D, torch.bfloat16, 50 + step)):
            cache.append(k, v)
    for name in ("lengths", "block_tables", "free_pages", "free_range", "shares", "k_pages", "v_pages"):
        assert torch.equal(getattr(caches[0], name), getattr(caches[1], name)), name
    assert caches[0].lengths.tolist() == [6] * batch
