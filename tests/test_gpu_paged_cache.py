"""``PagedCache`` as an object: a captured step, tokens that were not handed over, refused calls."""

import pytest
import torch

from adasplash_amd.paged import PagedCache
from tests.test_gpu_paged import check_rows

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16
B, HQ, HKV, D, PAGE = 3, 4, 2, 64, 4


def tokens(n, g, dtype=BF16):
    return [torch.randn(n, HKV, D, generator=g).to(dtype) for _ in range(2)]


def state_of(cache):
    return [x.clone() for x in (cache.lengths, cache.free_range, cache.free_pages, cache.block_tables, cache.k_pages, cache.v_pages)]


def test_a_captured_step_goes_on():
    """``append`` and ``attend`` in a graph: every replay adds a token behind the last, as the same calls without a graph do."""
    g = torch.Generator().manual_seed(1)
    caches = [PagedCache(64, PAGE, B, HKV, D, 80, dtype=BF16) for _ in range(2)]
    held = [7, 0, 4]
    k, v = tokens(sum(held), g)
    for cache in caches:
        cache.append(k.to(DEV), v.to(DEV), torch.tensor(held, device=DEV))
    ks, vs = ([list(t.split(held))[b].transpose(0, 1) for b in range(B)] for t in (k, v))
    kn, vn = (torch.zeros(B, HKV, D, dtype=BF16, device=DEV) for _ in range(2))
    q = torch.zeros(B, HQ, 1, D, dtype=BF16, device=DEV)

    def step(cache):
        cache.append(kn, vn)
        return cache.attend(q)

    other = PagedCache(64, PAGE, B, HKV, D, 80, dtype=BF16)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(other)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(caches[0])
    for i in range(20):
        k, v = tokens(B, g)
        kn.copy_(k), vn.copy_(v), q.copy_(torch.randn(q.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        ks, vs = ([torch.cat([x[b], t[b][:, None]], 1) for b in range(B)] for x, t in ((ks, k), (vs, v)))
        check_rows(out, q, ks, vs, 1.5, f"replay {i}")
        assert torch.equal(out, step(caches[1])), f"replay {i}"
        for a, b in zip(state_of(caches[0]), state_of(caches[1])):
            assert torch.equal(a, b), f"replay {i}"
    # calls without the graph go on where it stopped, and it where they did
    caches[0].release(1)
    caches[1].release(1)
    for _ in range(2):
        step(caches[0]), step(caches[1])
        graph.replay()
        assert torch.equal(out, step(caches[1]))
    assert caches[0].lengths.tolist() == [7 + 24, 4, 4 + 24] == caches[1].lengths.tolist()


def test_tokens_that_were_not_handed_over_are_not_counted():
    """25 rows where ``new_tokens`` says 20 and 20: the second request gets the 5 that are there, and pages for no more."""
    g = torch.Generator().manual_seed(2)
    cache = PagedCache(40, PAGE, B, HKV, D, 60, dtype=BF16)
    k, v = tokens(25, g)
    # (a slot that is not written holds what an earlier request left in it)
    cache.k_pages.fill_(3.0)
    cache.v_pages.fill_(100.0)
    slots = cache.append(k.to(DEV), v.to(DEV), torch.tensor([20, 20, 9], dtype=torch.int32, device=DEV))
    assert cache.lengths.tolist() == [20, 5, 0] and (slots >= 0).all()
    assert cache.free_range.tolist() == [5 + 2, 40]
    q = torch.randn(B, HQ, 1, D, generator=g).to(BF16).to(DEV)
    ks, vs = ([t[:20].transpose(0, 1), t[20:].transpose(0, 1), t[:0].transpose(0, 1)] for t in (k, v))
    check_rows(cache.attend(q), q, ks, vs, 1.5, "25 of 40")
    # none at all, negative counts, and more rows than tokens
    cache.append(k[:0].to(DEV), v[:0].to(DEV), torch.tensor([3, 3, 3], device=DEV))
    assert cache.lengths.tolist() == [20, 5, 0] and cache.free_range.tolist() == [7, 40]
    slots = cache.append(k[:8].to(DEV), v[:8].to(DEV), torch.tensor([-5, 2, 3], device=DEV))
    assert cache.lengths.tolist() == [20, 7, 3] and slots.tolist()[5:] == [-1] * 3


def test_many_requests_with_fewer_rows_than_tokens():
    g = torch.Generator().manual_seed(3)
    for n in (1, 256, 257, 1025):
        new = torch.randint(0, 9, (n,), generator=g)
        rows = int(new.sum()) * 2 // 3
        cache = PagedCache(n * 3, PAGE, n, 1, 32, 12, dtype=BF16)
        k = torch.randn(rows, 1, 32, generator=g).to(BF16).to(DEV)
        slots = cache.append(k, k, new.to(DEV))
        ends = new.cumsum(0).clamp(max=rows)
        want = ends - torch.cat([ends.new_zeros(1), ends[:-1]])
        assert cache.lengths.tolist() == want.tolist()
        assert int(cache.free_range[0]) == int(((want + PAGE - 1) // PAGE).sum())
        assert (slots >= 0).all() and slots.unique().numel() == rows
        got = cache.k_pages.transpose(1, 2).reshape(-1, 1, 32)[slots]
        assert torch.equal(got, k)


@pytest.mark.parametrize("what", ["type", "heads", "head_dim", "v longer", "v of another type", "a gradient", "new_tokens of another batch", "new_tokens of another type", "on the CPU", "one dimension less"])
def test_a_refused_append_changes_nothing(what):
    g = torch.Generator().manual_seed(4)
    cache = PagedCache(40, PAGE, B, HKV, D, 60, dtype=BF16)
    k, v = (t.to(DEV) for t in tokens(9, g))
    cache.append(k, v, torch.tensor([4, 0, 5], device=DEV))
    before, mine = state_of(cache), (cache.lengths, cache.free_range)
    new = torch.tensor([3, 3, 3], device=DEV)
    if what == "type":
        k, v = k.float(), v.float()
    elif what == "heads":
        k, v = torch.cat([k, k], 1), torch.cat([v, v], 1)
    elif what == "head_dim":
        k, v = k[..., :32].contiguous(), v[..., :32].contiguous()
    elif what == "v longer":
        v = torch.cat([v, v])
    elif what == "v of another type":
        v = v.half()
    elif what == "a gradient":
        v = v.clone().requires_grad_(True)
    elif what == "new_tokens of another batch":
        new = new[:2]
    elif what == "new_tokens of another type":
        new = new.float()
    elif what == "on the CPU":
        v = v.cpu()
    else:
        k, v = k[:, 0], v[:, 0]
    with pytest.raises((AssertionError, RuntimeError, TypeError)):
        cache.append(k, v, new)
    assert cache.lengths is mine[0] and cache.free_range is mine[1]
    for a, b in zip(state_of(cache), before):
        assert torch.equal(a, b)


def test_a_cache_of_inference_tensors():
    """Made under ``inference_mode`` it is used there; outside of it, where tensors made in it may not be written to, a call is refused before anything has changed."""
    g = torch.Generator().manual_seed(5)
    k, v = (t.to(DEV) for t in tokens(B, g))
    first = [t.to(DEV) for t in tokens(B * PAGE, g)]
    with torch.inference_mode():
        cache = PagedCache(40, PAGE, B, HKV, D, 60, dtype=BF16)
        cache.append(*first, torch.full((B,), PAGE, device=DEV))  # (the next token of each needs a page)
        before = state_of(cache)
    with pytest.raises(RuntimeError, match="inference"):
        cache.append(k, v)
    with torch.inference_mode():
        for a, b in zip(state_of(cache), before):
            assert torch.equal(a, b)
        cache.append(k, v)
        assert cache.lengths.tolist() == [PAGE + 1] * B
    cache = PagedCache(40, PAGE, B, HKV, D, 60, dtype=BF16)
    with torch.inference_mode():
        cache.append(k, v)
    cache.append(k, v)
    assert cache.lengths.tolist() == [2] * B
