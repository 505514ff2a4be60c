"""The paged cache on the GPU: attention of one new token a request, block tables and slots, writes, and a run of them together."""

import math

import pytest
import torch

import adasplash_amd as A
from adasplash_amd.paged import PagedCache
from tests import op_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def make_cache(lens, Hkv, D, page, dtype, seed, spare=3, slots_first=False, fill=float("nan"), width=None):
    """Keys and values of requests of the given lengths in shuffled pages; every slot that no token has holds `fill`."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    width = max(max(need), 1) if width is None else width
    order = torch.randperm(pages, generator=g)
    shape = (pages, page, Hkv, D) if slots_first else (pages, Hkv, page, D)
    kp, vp = (torch.full(shape, fill, dtype=dtype) for _ in range(2))
    tables = torch.full((len(lens), width), -7, dtype=torch.int32)
    ks, vs, at = [], [], 0
    for b, n in enumerate(lens):
        k, v = (torch.randn(Hkv, n, D, generator=g).to(dtype) for _ in range(2))
        ks.append(k)
        vs.append(v)
        for i in range(need[b]):
            pg = int(order[at])
            at += 1
            tables[b, i] = pg
            part = slice(i * page, min(n, (i + 1) * page))
            for to, x in ((kp, k), (vp, v)):
                if slots_first:
                    to[pg, : part.stop - part.start] = x[:, part].transpose(0, 1)
                else:
                    to[pg, :, : part.stop - part.start] = x[:, part]
    kp, vp = kp.to(DEV), vp.to(DEV)
    if slots_first:
        kp, vp = kp.transpose(1, 2), vp.transpose(1, 2)
    return kp, vp, tables.to(DEV), ks, vs


def check_rows(got, q, ks, vs, alpha, what):
    B, Hq = q.shape[:2]
    for b in range(B):
        Hkv = ks[b].shape[0]
        G = Hq // Hkv
        for h in range(Hkv):
            want, tol = ref.attend(q[b, h * G:(h + 1) * G, 0].cpu(), ks[b][h], vs[b][h], alpha)
            ref.check(got[b, h * G:(h + 1) * G, 0], want, tol, f"{what} request {b} head {h}")


def run_case(lens, Hq, Hkv, D, page, dtype, alpha, q_scale=1.0, bits=torch.int32, **more):
    what = f"lens={lens} Hq={Hq} Hkv={Hkv} D={D} page={page} {dtype} alpha={alpha} q*{q_scale}"
    print(what, flush=True)
    kp, vp, tables, ks, vs = make_cache(lens, Hkv, D, page, dtype, seed=len(lens) + D + page, **more)
    q = (torch.randn(len(lens), Hq, 1, D, generator=torch.Generator().manual_seed(5)) * q_scale).to(dtype).to(DEV)
    lengths = torch.tensor(lens, dtype=bits, device=DEV)
    out = A.paged_attention(q, kp, vp, tables, lengths, alpha=alpha)
    assert out.shape == q.shape and out.dtype == dtype
    check_rows(out, q, ks, vs, alpha, what)
    assert torch.equal(out, A.paged_attention(q, kp, vp, tables, lengths, alpha=alpha))
    return out


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_types_and_head_dims(dtype, D):
    run_case([1, 17, 300, 2049], 8, 2, D, 16, dtype, 1.5)


@pytest.mark.parametrize("alpha", [1.05, 1.25, 1.333, 1.5, 1.75, 2.0])
@pytest.mark.parametrize("q_scale", [0.125, 1.0, 4.0])
def test_alphas_and_spreads(alpha, q_scale):
    run_case([700, 65, 2500], 4, 2, 64, 32, F32, alpha, q_scale)
    run_case([700, 65, 2500], 4, 2, 64, 32, BF16, alpha, q_scale)


@pytest.mark.parametrize("page", [1, 7, 8, 16, 100, 257])
def test_lengths_around_the_borders(page):
    lens = [0, 1, page - 1, page, page + 1, 2 * page, 63, 64, 65, 127, 128, 129, 255, 256, 257]
    run_case(lens, 4, 2, 64, page, BF16, 1.5, bits=torch.int64)


def test_lengths_around_the_parts():
    run_case([2047, 2048, 2049, 4095, 4096, 4097, 6145], 2, 1, 128, 16, BF16, 1.5)


@pytest.mark.parametrize("group", [1, 2, 3, 5, 8, 15, 16, 17, 33, 64])
def test_groups(group):
    run_case([200, 1100], group * 2, 2, 64, 16, BF16, 1.5)
    run_case([130, 513], group, 1, 128, 16, F32, 1.5)


def test_one_request_over_many_parts():
    run_case([40000], 8, 2, 64, 16, F16, 1.5)
    run_case([40000], 1, 1, 64, 16, BF16, 2.0, q_scale=0.125)


def test_many_requests():
    run_case([(37 * i) % 400 for i in range(300)], 4, 4, 64, 16, BF16, 1.5)


def test_slots_first_layout_and_a_view_of_a_larger_cache():
    run_case([50, 333], 8, 4, 128, 16, BF16, 1.5, slots_first=True)
    run_case([50, 333], 8, 4, 64, 10, F32, 1.5, slots_first=True)
    # two layers in one tensor: pages with a stride of their own
    kp, vp, tables, ks, vs = make_cache([90, 10], 2, 64, 16, BF16, 3)
    both = torch.stack([kp, vp, kp, vp], dim=1)
    q = torch.randn(2, 4, 1, 64, device=DEV).to(BF16)
    lengths = torch.tensor([90, 10], device=DEV)
    out = A.paged_attention(q, both[:, 0], both[:, 1], tables, lengths)
    assert torch.equal(out, A.paged_attention(q, kp, vp, tables, lengths))


@pytest.mark.parametrize("n", [1500, 4097, 9000])
def test_rows_of_equal_scores(n):
    """Every key is a member: more than the second kernel's list holds from 4097 on."""
    kp, vp, tables, ks, vs = make_cache([n], 1, 64, 16, F32, 4)
    q = torch.zeros(1, 2, 1, 64, device=DEV)
    for alpha in (1.5, 2.0, 1.25):
        out = A.paged_attention(q, kp, vp, tables, torch.tensor([n], device=DEV), alpha=alpha)
        want = vs[0][0].double().mean(0)
        # the mean of n values below 5: fp32 sums of them, sqrt(n) half steps, and the weights' sum to 2e-6
        tol = 5 * (4 * math.sqrt(n) * 2.0 ** -24 + 2e-6) * torch.ones(64, dtype=torch.float64)
        for h in range(2):
            ref.check(out[0, h, 0], want, tol, f"n={n} alpha={alpha}")


def test_one_key_far_above_the_others():
    kp, vp, tables, ks, vs = make_cache([5000], 1, 64, 16, BF16, 6)
    q = (ks[0][0, 3210].float() * 8).to(BF16).view(1, 1, 1, 64).to(DEV)
    out = A.paged_attention(q, kp, vp, tables, torch.tensor([5000], device=DEV))
    assert torch.equal(out[0, 0, 0].cpu(), vs[0][0, 3210])


def test_entries_outside_the_cache_are_pages_without_keys():
    lens = [100, 64, 40]
    kp, vp, tables, ks, vs = make_cache(lens, 2, 64, 16, BF16, 8)
    pages = kp.shape[0]
    tables[0, 2], tables[0, 4], tables[1] = -1, pages, 2 ** 31 - 1
    for b, gone in ((0, [2, 4]), (1, [0, 1, 2, 3])):
        keep = [i for i in range(lens[b]) if i // 16 not in gone]
        ks[b], vs[b] = ks[b][:, keep], vs[b][:, keep]
    q = torch.randn(3, 4, 1, 64, device=DEV).to(BF16)
    out = A.paged_attention(q, kp, vp, tables, torch.tensor(lens, device=DEV))
    check_rows(out, q, ks, vs, 1.5, "holes")
    assert (out[1] == 0).all()


def test_lengths_are_cut_off_and_max_length():
    kp, vp, tables, ks, vs = make_cache([300, 48], 2, 64, 16, BF16, 9)
    q = torch.randn(2, 4, 1, 64, device=DEV).to(BF16)
    full = A.paged_attention(q, kp, vp, tables, torch.tensor([300, 48], device=DEV))
    assert torch.equal(full, A.paged_attention(q, kp, vp, tables, torch.tensor([300, 48], device=DEV), max_length=300))
    out = A.paged_attention(q, kp, vp, tables, torch.tensor([300, 48], device=DEV), max_length=100)
    check_rows(out, q, [k[:, :100] for k in ks], [v[:, :100] for v in vs], 1.5, "max_length 100")
    # beyond the table, and negative
    out = A.paged_attention(q, kp.nan_to_num(), vp.nan_to_num(), tables, torch.tensor([10 ** 6, -3], device=DEV))
    assert (out[1] == 0).all() and torch.isfinite(out).all()
    assert (A.paged_attention(q, kp, vp, tables, torch.tensor([300, 48], device=DEV), max_length=0) == 0).all()
    assert A.paged_attention(q[:0], kp, vp, tables[:0], torch.zeros(0, dtype=torch.int32, device=DEV)).shape == (0, 4, 1, 64)


def test_infinities_and_nan_behind_the_length():
    for fill in (float("inf"), float("-inf"), float("nan")):
        run_case([5, 33, 1000], 4, 2, 64, 16, BF16, 1.5, fill=fill)


def test_offsets_beyond_32_bits():
    """Pages of 2 MiB, more than 2^31 elements apart."""
    page, D = 8192, 128
    n_pages = (1 << 31) // (page * D) + 3
    kp = torch.empty(n_pages, 1, page, D, dtype=F16, device=DEV)
    last, n = n_pages - 1, 1000
    kp[last, 0, :n] = torch.randn(n, D, device=DEV).to(F16)
    kp[0].zero_()
    tables = torch.tensor([[last]], dtype=torch.int32, device=DEV)
    q = torch.randn(1, 4, 1, D, device=DEV).to(F16)
    out = A.paged_attention(q, kp, kp, tables, torch.tensor([n], device=DEV))
    k = [kp[last, :, :n].cpu()]
    check_rows(out, q, k, k, 1.5, "far page")
    # and a write behind them
    new = torch.randn(2, 1, D, device=DEV).to(F16)
    A.write_pages(new, new, torch.tensor([last * page + n, last * page + 5], device=DEV), kp, kp)
    assert torch.equal(kp[last, 0, n], new[0, 0]) and torch.equal(kp[last, 0, 5], new[1, 0])


def test_a_query_that_is_a_view():
    kp, vp, tables, ks, vs = make_cache([90, 10], 2, 64, 16, BF16, 3)
    wide = torch.randn(2, 4, 3, 66, device=DEV).to(BF16)
    q = wide[:, :, 1:2, 1:65]
    out = A.paged_attention(q, kp, vp, tables, torch.tensor([90, 10], device=DEV))
    assert torch.equal(out, A.paged_attention(q.contiguous(), kp, vp, tables, torch.tensor([90, 10], device=DEV)))


def test_two_streams_at_once():
    kp, vp, tables, ks, vs = make_cache([3000, 700], 2, 64, 16, BF16, 11)
    lengths = torch.tensor([3000, 700], device=DEV)
    qs = [torch.randn(2, 4, 1, 64, device=DEV).to(BF16) for _ in range(8)]
    want = [A.paged_attention(q, kp, vp, tables, lengths) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i, q in enumerate(qs):
        with torch.cuda.stream(streams[i % 2]):
            got.append(A.paged_attention(q, kp, vp, tables, lengths))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


# ---- block tables -----------------------------------------------------------------------------------------------------
def tables_reference(held, new, tables, free, first, end, page, total):
    """The rules of the documentation, request by request and token by token."""
    tables = [list(r) for r in tables]
    width, avail, off = len(tables[0]), max(0, min(end - first, len(free))), 0
    slots, after = [], []
    for b, (h, n) in enumerate(zip(held, new)):
        h, n = max(0, min(h, width * page)), max(0, n)
        have = -(-h // page)
        need = min(-(-(h + n) // page), width) - have
        got = min(max(avail - off, 0), need)
        for i in range(got):
            tables[b][have + i] = free[(first + off + i) % len(free)]
        off += need
        last = min(h + n, (have + got) * page)
        after.append(last)
        for x in range(h, h + n):
            slots.append(tables[b][x // page] * page + x % page if x < last else -1)
    slots = (slots + [-1] * total)[:total]
    return tables, slots, after, [first + min(off, avail), end]


def run_tables(held, new, width, page, free, first, end, extra=0, dtypes=(torch.int32, torch.int32), padded=0):
    B = len(held)
    rows = [[1000 + 100 * b + i if i * page < held[b] else -5 for i in range(width)] for b in range(B)]
    wide = torch.full((B, width + padded), 77, dtype=torch.int32)
    wide[:, :width] = torch.tensor(rows, dtype=torch.int32)
    wide = wide.to(DEV)
    tables = wide[:, :width]
    total = sum(max(0, n) for n in new) + extra
    lengths = torch.tensor(held, dtype=dtypes[0], device=DEV)
    rng = torch.tensor([first, end], device=DEV)
    fresh = torch.tensor(new, dtype=dtypes[1], device=DEV)
    want = tables_reference(held, new, rows, free, first, end, page, total)
    for _ in range(2):  # (the same call again gives the same: what it reads it does not change)
        slots, after, left = A.build_block_tables(lengths, fresh, tables, torch.tensor(free, dtype=torch.int32, device=DEV), rng,
                                                  page_size=page, total_tokens=total)
        assert tables.tolist() == want[0]
        assert slots.tolist() == want[1] and slots.dtype == torch.int64
        assert after.tolist() == want[2] and after.dtype == dtypes[0]
        assert left.tolist() == want[3]
    assert lengths.tolist() == held and rng.tolist() == [first, end]
    assert padded == 0 or (wide[:, width:] == 77).all()


def test_tables_of_a_decoding_step():
    run_tables([0, 1, 15, 16, 17, 31, 32, 100], [1] * 8, 10, 16, list(range(200, 260)), 0, 60)


def test_tables_of_prompts_and_of_nothing():
    run_tables([0, 0, 5, 40], [100, 1, 0, 33], 10, 16, list(range(50, 90)), 3, 40, dtypes=(torch.int64, torch.int32))
    run_tables([0, 0], [0, 0], 2, 16, [1, 2, 3], 0, 3)
    run_tables([0], [0], 1, 1, [9], 0, 1, extra=5)


def test_tables_the_free_list_is_a_ring():
    run_tables([0, 7, 8], [20, 9, 1], 6, 8, list(range(300, 310)), 7, 17)
    run_tables([0, 7, 8], [20, 9, 1], 6, 8, list(range(300, 310)), 10 ** 12 + 7, 10 ** 12 + 14, dtypes=(torch.int32, torch.int64))


def test_tables_too_few_pages():
    run_tables([0, 0, 16, 0], [40, 40, 5, 3], 8, 16, list(range(10)), 0, 4)
    run_tables([0, 0, 16, 0], [40, 40, 5, 3], 8, 16, list(range(10)), 5, 5)
    run_tables([0, 0, 16, 0], [40, 40, 5, 3], 8, 16, list(range(10)), 6, 5)


def test_tables_too_narrow():
    run_tables([0, 30, 48], [100, 10, 7], 3, 16, list(range(40)), 0, 40)
    run_tables([10 ** 6], [4], 3, 16, list(range(40)), 0, 40)


def test_tables_negative_counts_and_padding():
    run_tables([-3, 5], [4, -2], 3, 4, list(range(20)), 0, 20, extra=7, padded=3)


def test_tables_of_many_requests():
    g = torch.Generator().manual_seed(1)
    for B, most in ((1, 5000), (255, 60), (256, 60), (257, 60), (1025, 9), (8192, 5)):
        held = torch.randint(0, 200, (B,), generator=g).tolist()
        new = torch.randint(0, most, (B,), generator=g).tolist()
        run_tables(held, new, 400 if B == 1 else 40, 16, list(range(5000, 5000 + 3 * B + 400)), 11, 11 + 2 * B + 300)


def test_more_tokens_than_slots_asked_for():
    tables = torch.full((2, 4), -1, dtype=torch.int32, device=DEV)
    zero = torch.zeros(2, dtype=torch.int32, device=DEV)
    slots, after, left = A.build_block_tables(zero, torch.tensor([20, 20], dtype=torch.int32, device=DEV), tables,
                                              torch.arange(9, dtype=torch.int32, device=DEV), torch.tensor([0, 9], device=DEV), 16, 25)
    assert slots.tolist() == list(range(20)) + list(range(32, 37)) and after.tolist() == [20, 20] and left.tolist() == [4, 9]


# ---- writes -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("D", [32, 40, 128, 256])
def test_writes(dtype, D):
    g = torch.Generator().manual_seed(2)
    for T, Hkv, page, slots_first in ((1, 1, 1, False), (77, 3, 10, False), (500, 8, 16, True)):
        pages = T // page + 3
        shape = (pages, page, Hkv, D) if slots_first else (pages, Hkv, page, D)
        kp, vp = (torch.randn(shape, generator=g).to(dtype).to(DEV) for _ in range(2))
        if slots_first:
            kp, vp = kp.transpose(1, 2), vp.transpose(1, 2)
        k, v = (torch.randn(T, Hkv, D, generator=g).to(dtype).to(DEV) for _ in range(2))
        slots = torch.randperm(pages * page, generator=g)[:T]
        slots[::7] = -1
        if T > 4:
            slots[3], slots[4] = pages * page, 10 ** 15
        want = [kp.clone(), vp.clone()]
        for t, s in enumerate(slots.tolist()):
            if 0 <= s < pages * page:
                want[0][s // page, :, s % page] = k[t]
                want[1][s // page, :, s % page] = v[t]
        A.write_pages(k, v, slots.to(DEV), kp, vp)
        assert torch.equal(kp, want[0]) and torch.equal(vp, want[1])


def test_writes_from_views():
    qkv = torch.randn(20, 3, 4, 64, device=DEV).to(BF16)
    kp, vp = (torch.zeros(4, 4, 8, 64, device=DEV, dtype=BF16) for _ in range(2))
    version = kp._version
    A.write_pages(qkv[:, 1], qkv[:, 2], torch.arange(20, device=DEV), kp, vp)
    assert torch.equal(kp.transpose(1, 2).reshape(32, 4, 64)[:20], qkv[:, 1]) and (vp[3] == 0).all() and kp._version > version
    odd = torch.randn(20, 4, 65, device=DEV).to(BF16)
    A.write_pages(odd[..., 1:], odd[..., :64], torch.arange(20, device=DEV), kp, vp)
    assert torch.equal(kp.transpose(1, 2).reshape(32, 4, 64)[:20], odd[..., 1:])
    assert torch.equal(vp.transpose(1, 2).reshape(32, 4, 64)[:20], odd[..., :64])
    A.write_pages(odd[:0, :, :64], odd[:0, :, :64], torch.zeros(0, dtype=torch.int64, device=DEV), kp, vp)


# ---- together ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_decoding_run(dtype):
    """Prompts of different lengths enter, requests grow token by token, one leaves and another takes its pages: every step's attention is that of all
    tokens so far."""
    g = torch.Generator().manual_seed(3)
    B, Hq, Hkv, D, page = 3, 8, 2, 64, 4
    cache = PagedCache(40, page, B, Hkv, D, 60, dtype=dtype)
    ks, vs = [torch.zeros(Hkv, 0, D, dtype=dtype) for _ in range(B)], [torch.zeros(Hkv, 0, D, dtype=dtype) for _ in range(B)]

    def add(counts):
        new = [[torch.randn(Hkv, n, D, generator=g).to(dtype) for n in counts] for _ in range(2)]
        for b in range(B):
            ks[b] = torch.cat([ks[b], new[0][b]], 1)
            vs[b] = torch.cat([vs[b], new[1][b]], 1)
        k, v = (torch.cat([x.transpose(0, 1) for x in part]).to(DEV) for part in new)
        if counts == [1, 1, 1]:
            cache.append(k[:, :, None], v[:, :, None])
        else:
            cache.append(k, v, torch.tensor(counts, dtype=torch.int32, device=DEV))

    def look(what):
        q = torch.randn(B, Hq, 1, D, generator=g).to(dtype).to(DEV)
        check_rows(cache.attend(q), q, ks, vs, 1.5, what)

    add([13, 0, 5])
    look("prompts")
    for i in range(9):
        add([1, 1, 1])
        look(f"step {i}")
    cache.release(0)
    ks[0], vs[0] = ks[0][:, :0], vs[0][:, :0]
    look("released")
    add([30, 4, 20])
    look("the next prompt")
    for i in range(20):
        add([1, 1, 1])
        look(f"later step {i}")
    assert cache.lengths.tolist() == [k.shape[1] for k in ks]


def test_a_captured_step():
    """A step of tables, write and attention in a graph, replayed with eager work and new inputs between: each replay is the eager result."""
    g = torch.Generator().manual_seed(4)
    B, Hkv, D, page = 4, 2, 64, 16
    kp, vp = (torch.zeros(64, Hkv, page, D, device=DEV, dtype=BF16) for _ in range(2))
    tables = torch.full((B, 12), -1, dtype=torch.int32, device=DEV)
    free, rng = torch.randperm(64, generator=g).to(torch.int32).to(DEV), torch.tensor([0, 64], device=DEV)
    lengths = torch.zeros(B, dtype=torch.int32, device=DEV)
    one = torch.ones(B, dtype=torch.int32, device=DEV)
    k, v = (torch.zeros(B, Hkv, D, device=DEV, dtype=BF16) for _ in range(2))
    q = torch.zeros(B, 4, 1, D, device=DEV, dtype=BF16)

    def step():
        slots, after, left = A.build_block_tables(lengths, one, tables, free, rng, page, B)
        A.write_pages(k, v, slots, kp, vp)
        out = A.paged_attention(q, kp, vp, tables, after)
        lengths.copy_(after)
        rng.copy_(left)
        return out

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    state = [x.clone() for x in (kp, vp, tables, rng, lengths)]
    for i in range(40):
        for x in (k, v, q):
            x.copy_(torch.randn(x.shape, generator=g).to(BF16))
        graph.replay()
        torch.cuda.synchronize()
        got, behind = out.clone(), [x.clone() for x in (kp, vp, tables, rng, lengths)]
        for x, s in zip((kp, vp, tables, rng, lengths), state):
            x.copy_(s)
        assert torch.equal(step(), got), f"replay {i}"
        for x, s in zip((kp, vp, tables, rng, lengths), behind):
            assert torch.equal(x, s)
        state = behind
    assert lengths.tolist() == [41] * B


def test_a_batch_in_more_than_one_launch():
    """Tables with room for 131072 tokens and 64 query heads: 64 MiB of workspace a request."""
    run_case([1000 + 37 * b for b in range(20)], 64, 1, 32, 64, BF16, 1.5, width=2048)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_alpha_close_to_one(dtype):
    for alpha in (1.01, 1.001):
        run_case([700, 65, 2500], 4, 2, 64, 32, dtype, alpha)


def test_scratch_may_hold_anything():
    lens = [1, 600, 2500, 0, 9000]
    kp, vp, tables, ks, vs = make_cache(lens, 2, 64, 16, BF16, seed=1)
    q = torch.randn(len(lens), 8, 1, 64, generator=torch.Generator().manual_seed(5)).to(BF16).to(DEV)
    lengths = torch.tensor(lens, device=DEV)
    results = []
    for fill in (0, 255, 1, 127):
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        soil = torch.full((1 << 30,), fill, dtype=torch.uint8, device=DEV)  # (what the allocator hands out next)
        soil_small = [torch.full((1 << 19,), fill, dtype=torch.uint8, device=DEV) for _ in range(64)]
        del soil, soil_small
        results.append(A.paged_attention(q, kp, vp, tables, lengths))
    for other in results[1:]:
        assert torch.equal(results[0], other)
