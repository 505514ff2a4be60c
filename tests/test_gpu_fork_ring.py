"""Free lists of fewer entries than the cache has pages: what is free already is never written over, and a page that finds no place says so."""

import pytest
import torch

import adasplash_amd as A

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("width", [4, 2000])  # tables for one workgroup, and for several
@pytest.mark.parametrize("free, went", [(4, 0), (6, 3), (0, 5), (2, 6 * 7 + 5)])
def test_more_pages_than_entries(width, free, went):
    """Four requests of three pages end in a cache of 20, whose list has 6 entries, some of them free; a fifth goes on and copies its last page."""
    entries, pages, page, B = 6, 20, 2, 6
    tables = torch.full((B, width), -1, dtype=torch.int32)
    for b in range(4):
        tables[b, :3] = torch.tensor([2 * b + 7, 2 * b + 8, 15 + b])
    tables[4, :1] = 19
    lengths = torch.tensor([6, 6, 5, 6, 1, 0], dtype=torch.int32)
    ring = torch.full((entries,), -5, dtype=torch.int32)
    for i in range(free):
        ring[(went + i) % entries] = i
    limit, shares = torch.tensor([went, went + free]), torch.zeros(pages, dtype=torch.int32)
    k = torch.randn(pages, 1, page, 8, generator=torch.Generator().manual_seed(1))
    state = [t.to(DEV) for t in (lengths, tables, ring, limit, shares, k, k + 1)]
    A.fork_requests(torch.tensor([-1, -1, -1, -1, 4, 4], device=DEV), *state)
    lengths, tables, ring, limit, shares, kp, _ = (t.cpu() for t in state)
    freed = [p for b in range(4) for p in (2 * b + 7, 2 * b + 8, 15 + b)]
    listed = [*range(free), *freed][:entries]
    lost = freed[entries - free:]
    # (freed pages are placed before the copy's page is taken from the front)
    assert limit.tolist() == [went + 1, went + entries]
    assert [ring[i % entries].item() for i in range(went, went + entries)] == listed
    assert shares.tolist() == [-1 if p in lost else 0 for p in range(pages)]
    assert lengths.tolist() == [0, 0, 0, 0, 1, 1] and tables[4, 0] == 19 and tables[5, 0] == listed[0]
    assert torch.equal(kp[listed[0], :, :1], k[19, :, :1])
    assert (tables[:4] == -1).all()


@pytest.mark.parametrize("width", [4, 2000])
def test_one_page_after_another(width):
    """A full list stays full and in its order, step after step."""
    entries, pages, B = 3, 9, 3
    ring, limit = torch.arange(entries, dtype=torch.int32, device=DEV), torch.tensor([7, 10], device=DEV)
    shares = torch.zeros(pages, dtype=torch.int32, device=DEV)
    kp, vp = (torch.zeros(pages, 1, 4, 8, device=DEV) for _ in range(2))
    tables = torch.full((B, width), -1, dtype=torch.int32, device=DEV)
    tables[:, 0] = torch.tensor([3, 4, 5])
    lengths = torch.tensor([4, 4, 4], device=DEV)
    for b in range(B):
        parents = torch.arange(B, device=DEV)
        parents[b] = -1
        A.fork_requests(parents, lengths, tables, ring, limit, shares, kp, vp)
        assert ring.tolist() == [0, 1, 2] and limit.tolist() == [7, 10] and lengths[b] == 0
        assert shares.tolist() == [-1 if 3 <= p <= 3 + b else 0 for p in range(pages)]
