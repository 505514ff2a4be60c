"""Requests that go on from others, end, and move, on the GPU, against the books kept on the host."""

import random

import pytest
import torch

import adasplash_amd as A
from adasplash_amd.paged import PagedCache
from tests import op_reference as op
from tests import positions_reference as pos
from tests.cache_reference import Books

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


class Pair:
    """A cache on the GPU and its books: the value that the books hold for a token is its row of K (V's is that and a quarter)."""

    def __init__(self, pages, page, batch, H, D, most, dtype, seed):
        self.cache = PagedCache(pages, page, batch, H, D, most, dtype=dtype)
        self.books = Books(pages, page, batch, -(-most // page))
        self.H, self.D, self.dtype, self.count = H, D, dtype, 0
        self.g = torch.Generator().manual_seed(seed)
        self.rows = torch.zeros(0, H, D, dtype=dtype)

    def append(self, new):
        n = sum(new)
        k = torch.randn(n, self.H, self.D, generator=self.g).to(self.dtype)
        names = list(range(len(self.rows), len(self.rows) + n))
        self.rows = torch.cat([self.rows, k])
        self.cache.append(k.to(DEV), (k + 0.25).to(DEV), torch.tensor(new, device=DEV))
        split, at = [], 0
        for m in new:
            split.append(names[at:at + m])
            at += m
        self.books.append(split)

    def fork(self, parents, dtype=torch.int64):
        self.cache.fork(torch.tensor(parents, dtype=dtype, device=DEV))
        self.books.fork(parents)

    def resize(self, pages):
        self.cache.resize(pages)
        self.books.compact(pages)

    def check(self, what):
        c, b = self.cache, self.books
        assert c.lengths.tolist() == b.lengths, what
        tables = c.block_tables.tolist()
        for i, t in enumerate(b.tables):
            assert tables[i][: len(t)] == t, f"{what}: table {i}"
        first, end = c.free_range.tolist()
        ring = c.free_pages.tolist()
        assert [ring[i % len(ring)] for i in range(first, end)] == b.free, what
        assert c.shares.tolist() == b.shares(), what
        k, v = c.k_pages.cpu(), c.v_pages.cpu()
        for i in range(len(b.tables)):
            names = b.values(i)
            for j, name in enumerate(names):
                p, s = b.tables[i][j // b.page], j % b.page
                assert torch.equal(k[p, :, s], self.rows[name]) and torch.equal(v[p, :, s], self.rows[name] + 0.25), f"{what}: request {i} token {j}"


@pytest.mark.parametrize("page, batch, H, D, dtype", [(4, 5, 2, 32, BF16), (1, 3, 1, 16, F32), (16, 9, 3, 64, F16), (7, 2, 2, 8, BF16), (3, 17, 1, 32, F32)])
def test_steps_in_any_order(page, batch, H, D, dtype):
    rng = random.Random(page * 100 + batch)
    pair = Pair(batch * 12, page, batch, H, D, 12 * page, dtype, page)
    for step in range(30):
        pair.append([rng.choice((0, 1, 1, 2, page, page + 1)) for _ in range(batch)])
        pair.check(f"step {step} append")
        if step % 2:
            parents = [rng.choice((b, b, rng.randrange(batch), rng.randrange(batch), -1, batch, 1 << 30)) for b in range(batch)]
            pair.fork(parents, rng.choice((torch.int32, torch.int64)))
            pair.check(f"step {step} fork {parents}")
        if step % 7 == 6:
            pair.resize(batch * rng.choice((10, 12, 14)))
            pair.check(f"step {step} resize")


def test_a_cache_that_runs_out():
    for pages in (3, 4, 5, 7):
        pair = Pair(pages, 4, 4, 1, 32, 40, BF16, pages)
        pair.append([10, 0, 0, 0])
        pair.fork([0, 0, 0, 0])
        pair.check(f"{pages} pages, samples")
        pair.append([1, 1, 1, 1])
        pair.check(f"{pages} pages, a token more")
        pair.fork([3, 2, 1, 0])
        pair.check(f"{pages} pages, places changed")
        pair.fork([-1, -1, -1, 0])
        pair.check(f"{pages} pages, ended")
        pair.fork([3, 3, 3, 3])
        pair.check(f"{pages} pages, samples again")
        pair.resize(2)
        pair.check(f"{pages} pages, two left")
        pair.fork([-1, -1, -1, -1])
        pair.check("all ended")


def test_many_requests():
    rng = random.Random(5)
    pair = Pair(3000, 2, 700, 1, 8, 8, F32, 9)
    pair.append([rng.randint(0, 8) for _ in range(700)])
    pair.fork([rng.choice((b, rng.randrange(700), rng.randrange(20), -1)) for b in range(700)])
    pair.check("700 requests")
    pair.append([1] * 700)
    pair.fork([rng.randrange(700) for b in range(700)])
    pair.check("700 requests again")
    pair.resize(2500)
    pair.check("700 requests moved")
    pair.fork([-1] * 700)
    pair.check("700 ended")


def test_tables_of_every_size():
    """Around the borders between one workgroup and several: entries of all tables, requests, runs of 64."""
    for batch, width in ((1, 1), (2, 63), (3, 64), (5, 65), (16, 512), (17, 482), (64, 128), (128, 64), (129, 64), (1024, 8), (1025, 7), (1100, 9)):
        rng = random.Random(batch * width)
        pair = Pair(batch * 3 + width * 4 + 10, 2, batch, 1, 8, 2 * width, F32, batch)
        long = {rng.randrange(batch) for _ in range(3)}
        pair.append([rng.randint(0, 2 * width) if b in long else rng.randint(0, min(6, 2 * width)) for b in range(batch)])
        for _ in range(2):
            pair.fork([rng.choice((b, b, rng.randrange(batch), -1)) for b in range(batch)])
            pair.append([1] * batch)
        pair.check(f"{batch} tables of {width}")
        pair.resize(pair.books.pages - 3)
        pair.check(f"{batch} tables of {width}, moved")


@pytest.mark.parametrize("batch, width", [(64, 80), (64, 81), (512, 10), (1024, 5), (64, 64), (17, 241), (1024, 4), (31, 133)])
def test_tables_around_one_workgroups(batch, width):
    """4096 entries and 5120, and one more."""
    rng = random.Random(batch * width)
    pair = Pair(batch * width // 2 + 40, 1, batch, 1, 8, width, F32, width)
    long = [b for b in range(batch) if rng.random() < 0.3]
    pair.append([width - 1 if b in long else rng.randint(0, min(3, width - 1)) for b in range(batch)])
    for step in range(2):
        pair.fork([rng.choice((b, b, rng.randrange(batch), -1)) for b in range(batch)])
        pair.check(f"{batch} tables of {width}, step {step}")
    pair.resize(pair.books.pages - 3)
    pair.check(f"{batch} tables of {width}, moved")


@pytest.mark.parametrize("room", [65536, 65537])
def test_a_small_cache_in_a_large_pool(room):
    pair = Pair(40, 2, 3, 1, 8, 20, F32, 5)
    pair.append([17, 0, 5])
    pair.fork([0, 0, 2])
    for pages in (room, 12, room, 40):
        pair.resize(pages)
        pair.check(f"{pages} pages")
        pair.fork([1, 0, 2])
        pair.append([1, 0, 2])
        pair.check(f"goes on in {pages}")


def test_one_request_of_many_pages():
    pair = Pair(2000, 1, 3, 1, 8, 900, F32, 9)
    pair.append([0, 801, 0])
    pair.fork([1, 1, -1])
    pair.check("a copy")
    pair.append([30, 20, 40])
    pair.fork([-1, 2, 2])
    pair.check("one ends")


def test_release():
    pair = Pair(40, 4, 4, 1, 32, 60, BF16, 1)
    pair.append([10, 5, 0, 9])
    pair.cache.release(1)
    pair.books.fork([0, -1, 2, 3])
    pair.check("one")
    pair.cache.release(1)
    pair.books.fork([0, -1, 2, 3])
    pair.check("an empty one")
    pair.fork([0, 0, 3, 3])
    pair.cache.release(-1)
    pair.books.fork([0, 1, 2, -1])
    pair.check("the last, some of whose pages another holds")
    pair.cache.release([0, 2])
    pair.books.fork([-1, 1, -1, 3])
    pair.check("two")
    pair.cache.release(torch.tensor([1, 7, -1], device=DEV))
    pair.books.fork([-1] * 4)
    pair.check("the last")
    assert sorted(pair.books.free) == list(range(40))


def test_what_is_not_held_stays():
    """Entries behind a request's pages, free pages and slots behind its tokens stay as they are where the request does; what changes ends in -1."""
    cache = PagedCache(20, 4, 3, 1, 32, 30, dtype=BF16)
    k = torch.randn(11, 1, 32, generator=torch.Generator().manual_seed(1)).to(BF16).to(DEV)
    cache.append(k, k, torch.tensor([6, 5, 0], device=DEV))
    cache.block_tables[0, 5] = 77
    cache.k_pages[:, :, 3] = 5.0
    before = cache.k_pages.clone()
    cache.fork(torch.tensor([0, 0, -1], device=DEV))
    assert cache.block_tables[0].tolist()[:6] == [0, 1, -1, -1, -1, 77] and cache.block_tables[1].tolist() == [0, 4, -1, -1, -1, -1, -1, -1]
    before[4, :, :2] = before[1, :, :2]
    assert torch.equal(cache.k_pages, before)


def test_tables_of_other_kinds():
    """Numbers that name no page, lengths outside the table, a free list whose numbers have gone round it, views, parents that are the lengths' own tensor."""
    pages, page = 12, 4
    k = torch.randn(pages, page, 2, 16, generator=torch.Generator().manual_seed(3)).to(DEV).transpose(1, 2)
    v = (k + 1).clone(memory_format=torch.preserve_format)
    wide = torch.full((3, 9), -3, dtype=torch.int32, device=DEV)
    tables = wide[:, 1:6]
    tables.copy_(torch.tensor([[3, -1, 99, 4, -5], [7, 1 << 30, 8, 0, 0], [5, 6, 0, 0, 0]], dtype=torch.int32))
    lengths = torch.tensor([14, 10, -9], device=DEV)
    free = torch.tensor([0, 1, 2, 9, 10, 11] + [0] * 6, dtype=torch.int32, device=DEV).roll(4)
    free_range, shares = torch.tensor([12 * 5 + 4, 12 * 5 + 10], device=DEV), torch.zeros(pages, dtype=torch.int32, device=DEV)
    k0 = k.clone()
    A.fork_requests(torch.tensor([0, 0, 0], device=DEV), lengths, tables, free, free_range, shares, k, v)
    assert lengths.tolist() == [14, 14, 14]
    assert tables.tolist() == [[3, -1, 99, 4, -5], [3, -1, 99, 0, -1], [3, -1, 99, 1, -1]]
    assert (wide[:, 0] == -3).all() and (wide[:, 6:] == -3).all()
    assert shares.tolist() == [0, 0, 0, 2] + [0] * 8 and free_range.tolist() == [66, 72]
    assert [free[i % 12].item() for i in range(66, 72)] == [2, 9, 10, 11, 7, 8]
    k0[0, :, :2] = k0[1, :, :2] = k0[4, :, :2]
    assert torch.equal(k, k0) and torch.equal(v, k0 + 1)
    lengths = torch.tensor([2, 1, 0], device=DEV)
    A.fork_requests(lengths, lengths, tables, free, free_range, shares, k, v)  # the first becomes the last's, the last the first's
    assert lengths.tolist() == [0, 1, 2]
    lengths.copy_(torch.tensor([1 << 40, 7, 3]))
    out = A.compact_pages(lengths, tables, k, v, torch.zeros_like(k[:5]), torch.zeros_like(v[:5]))
    assert out[0].tolist() == [20, 7, 3] and out[1].shape == (3, 5)
    for limit in (torch.tensor([5, 5], device=DEV), torch.tensor([9, 4], device=DEV), torch.tensor([-3, 0], device=DEV)):  # nothing is free
        lengths = torch.tensor([6, 0, 0], device=DEV)
        tables.copy_(torch.tensor([[3, 4, -1, -1, -1]] + [[-1] * 5] * 2, dtype=torch.int32))
        A.fork_requests(torch.tensor([0, 0, -1], device=DEV), lengths, tables, free, limit, torch.zeros_like(shares), k, v)
        assert lengths.tolist() == [6, 4, 0] and tables[1].tolist() == [3, -1, -1, -1, -1]


def test_other_pools():
    """Pools of other sizes and strides; what is not taken stays."""
    pair = Pair(30, 4, 5, 2, 32, 40, F16, 3)
    pair.append([9, 4, 0, 15, 1])
    pair.fork([0, 0, 3, 3, -1])
    c = pair.cache
    for room in (1, 3, 6, 7, 8, 30, 100):
        k_to, v_to = (torch.full((room, 4, 2, 32), 3.0, dtype=F16, device=DEV).transpose(1, 2) for _ in range(2))
        old = [t.clone() for t in (c.lengths, c.block_tables, c.k_pages, c.v_pages)]
        lengths, tables, shares, free, limit = A.compact_pages(c.lengths, c.block_tables, c.k_pages, c.v_pages, k_to, v_to)
        assert all(torch.equal(a, b) for a, b in zip(old, (c.lengths, c.block_tables, c.k_pages, c.v_pages)))
        moved = PagedCache(room, 4, 5, 2, 32, 40, dtype=F16)
        moved.k_pages, moved.v_pages, moved.lengths, moved.block_tables, moved.shares, moved.free_pages, moved.free_range = k_to, v_to, lengths, tables, shares, free, limit
        other = Pair(30, 4, 5, 2, 32, 40, F16, 3)
        other.append([9, 4, 0, 15, 1])
        other.fork([0, 0, 3, 3, -1])
        other.cache = moved
        other.books.compact(room)
        other.check(f"room {room}")
        taken = {p for t in other.books.tables for p in t}
        for p in range(room):
            if p not in taken:
                assert (k_to[p] == 3.0).all() and (v_to[p] == 3.0).all()
        assert sorted(free.tolist()) == list(range(room))


def test_a_cache_beyond_32_bits():
    """Pages whose numbers in elements pass 2^31, and 2^32 bytes: written, copied and moved; and a table large enough for the launches of large tables."""
    pages, H, page, D, B = 1100000, 1, 16, 128, 40
    kp, vp = (torch.empty(pages, H, page, D, dtype=BF16, device=DEV) for _ in range(2))
    g = torch.Generator().manual_seed(12)
    tokens = 3 * page + 5
    k, v = (torch.randn(tokens, H, D, generator=g).to(BF16).to(DEV) for _ in range(2))
    own = torch.arange(pages - 4, pages).flip(0)
    at = torch.arange(tokens)
    f = pos.frequencies_of(D).to(DEV)
    A.write_pages(k, v, (own[at // page] * page + at % page).to(DEV), kp, vp, positions=at.to(DEV), rotary=A.Rotary(f))
    turned, _ = A.rotary(k, None, at.to(DEV), f)
    for width in (8, 400):
        tables = torch.full((B, width), -1, dtype=torch.int32, device=DEV)
        tables[0, :4] = own.int().to(DEV)
        lengths = torch.zeros(B, dtype=torch.int32, device=DEV)
        lengths[0] = tokens
        shares, free = torch.zeros(pages, dtype=torch.int32, device=DEV), torch.arange(pages - 400, pages - 4, dtype=torch.int32, device=DEV)
        limit = torch.tensor([0, 396], device=DEV)
        A.fork_requests(torch.zeros(B, dtype=torch.int64, device=DEV), lengths, tables, free, limit, shares, kp, vp)
        assert lengths.tolist() == [tokens] * B and limit.tolist() == [B - 1, 396] and int(shares[pages - 1]) == B - 1
        to = [torch.zeros(3 + B, H, page, D, dtype=BF16, device=DEV) for _ in range(2)]
        moved = A.compact_pages(lengths, tables, kp, vp, *to)
        for b in (0, 1, B - 1):
            assert moved[1][b, :4].tolist() == [0, 1, 2, 3 + b]
            for pool, table, want in ((kp, tables, turned), (vp, tables, v), (to[0], moved[1], turned), (to[1], moved[1], v)):
                assert torch.equal(pool[table[b, :4].long()].transpose(1, 2).reshape(-1, H, D)[:tokens], want)


def test_captured_steps():
    """A beam step, an ending and new tokens in a graph: each replay goes on from the last, as the same calls without a graph do."""
    B, H, D, page = 6, 2, 32, 4
    g = torch.Generator().manual_seed(4)
    caches = [PagedCache(80, page, B, H, D, 60, dtype=BF16) for _ in range(2)]
    k = torch.randn(30, H, D, generator=g).to(BF16).to(DEV)
    for c in caches:
        c.append(k, k + 1, torch.tensor([5, 5, 5, 5, 5, 5], device=DEV))
    parents, kn = torch.zeros(B, dtype=torch.int64, device=DEV), torch.zeros(B, H, D, dtype=BF16, device=DEV)

    def step(c):
        c.fork(parents)
        c.append(kn, kn)
        c.release(5)

    warm = PagedCache(80, page, B, H, D, 60, dtype=BF16)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(warm)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(caches[0])
    for i in range(8):
        parents.copy_(torch.randint(-1, B, (B,), generator=g))
        kn.copy_(torch.randn(kn.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        step(caches[1])
        for name in ("lengths", "block_tables", "free_pages", "free_range", "shares", "k_pages", "v_pages"):
            assert torch.equal(getattr(caches[0], name), getattr(caches[1], name)), f"replay {i}: {name}"


def test_a_prompt_and_its_samples():
    """All together: a prompt with turned keys goes on in samples and beams, which attend to it once for all; against 64 bits."""
    page, B, Hq, Hkv, D, n = 16, 8, 8, 2, 64, 1033
    g = torch.Generator().manual_seed(10)
    f = pos.frequencies_of(48)
    wq, wk = ((1 + 0.2 * torch.randn(D, generator=g)).to(F32) for _ in range(2))
    turn = A.Rotary(f.to(DEV), "interleaved", q_weight=wq.to(DEV), k_weight=wk.to(DEV), factor=1.1)
    cache = PagedCache(160, page, B, Hkv, D, 1200, dtype=F32, rotary=turn)
    k, v = (torch.randn(n, Hkv, D, generator=g) for _ in range(2))
    cache.append(k.to(DEV), v.to(DEV), torch.tensor([n] + [0] * (B - 1), device=DEV))
    cache.fork(torch.zeros(B, dtype=torch.int64, device=DEV))
    assert cache.lengths.tolist() == [n] * B and int(cache.free_range[0]) == -(-n // page) + B - 1
    prefix = cache.block_tables[0, : n // page].clone()
    ks, vs = [k.clone() for _ in range(B)], [v.clone() for _ in range(B)]
    beams = torch.Generator().manual_seed(11)
    for step in range(20):
        if step % 4 == 3:
            parents = torch.randint(0, B, (B,), generator=beams)
            if step == 11:
                parents[2] = -1
            cache.fork(parents.to(DEV))
            ks, vs = ([x[int(p)].clone() if p >= 0 else x[0][:0] for p in parents] for x in (ks, vs))
        kn, vn = (torch.randn(B, Hkv, 1, D, generator=g) for _ in range(2))
        cache.append(kn.to(DEV), vn.to(DEV))
        ks, vs = ([torch.cat([x[b], t[b].transpose(0, 1)]) for b in range(B)] for x, t in ((ks, kn), (vs, vn)))
        q = torch.randn(B, Hq, 1, D, generator=g)
        if step % 3 == 0:
            got = cache.attend(q.to(DEV), prefix_table=prefix)
            assert torch.allclose(got, cache.attend(q.to(DEV)), atol=2e-5)
            at = [torch.arange(len(x)) for x in ks]
            # (the reference takes the turned heads in fp32, as the cache holds them)
            keys = [pos.forward(x, a[:, None], f, "interleaved", wk, 1e-6, 1.1).float().transpose(0, 1) for x, a in zip(ks, at)]
            turned = torch.stack([pos.forward(q[b], at[b][-1:], f, "interleaved", wq, 1e-6, 1.1) for b in range(B)]).float()
            for b in range(B):
                for h in range(Hkv):
                    G = Hq // Hkv
                    want, tol = op.attend(turned[b, h * G:(h + 1) * G, 0], keys[b][h], vs[b][:, h], 1.5)
                    # (turned heads of kernel and reference differ by 20 half steps of fp32 each: a score by 40 of sum |q k|, which the bound of a score, 4 sqrt(64) = 32 of it, does not have)
                    op.check(got[b, h * G:(h + 1) * G, 0], want, 3 * tol, f"step {step} request {b}")
    cache.resize(130)
    assert torch.equal(cache.attend(q.to(DEV)), cache.attend(q.to(DEV)))
    again = cache.attend(q.to(DEV), prefix_table=cache.block_tables[0, : n // page])
    assert torch.allclose(again, cache.attend(q.to(DEV)), atol=2e-5)
