"""Paged attention behind a prefix that requests have in common, on the GPU: the same as without it, whatever the tables hold."""

import pytest
import torch

import adasplash_amd as A
from adasplash_amd import _lib
from tests import op_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def family(lens, front, Hkv, D, page, dtype, seed, fill=float("nan"), extra=0):
    """Requests of the given lengths whose first `front` pages are the same (where they reach so far), in shuffled pages; unused slots hold `fill`."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    pages = front + sum(need) + 3
    order = torch.randperm(pages, generator=g)
    kp, vp = (torch.full((pages, Hkv, page, D), fill, dtype=dtype) for _ in range(2))
    shared = [torch.randn(Hkv, front * page, D, generator=g).to(dtype) for _ in range(2)]
    for i in range(front):
        for to, x in ((kp, shared[0]), (vp, shared[1])):
            to[order[i]] = x[:, i * page:(i + 1) * page]
    tables = torch.full((len(lens), max(max(need), front, 1) + extra), -7, dtype=torch.int32)
    ks, vs, at = [], [], front
    for b, n in enumerate(lens):
        k, v = (torch.cat([s[:, :n], torch.randn(Hkv, max(n - front * page, 0), D, generator=g).to(dtype)], 1) for s in shared)
        ks.append(k)
        vs.append(v)
        for i in range(need[b]):
            if i < front:
                tables[b, i] = order[i]
                continue
            part = slice(i * page, min(n, (i + 1) * page))
            kp[order[at], :, : part.stop - part.start], vp[order[at], :, : part.stop - part.start] = k[:, part], v[:, part]
            tables[b, i] = order[at]
            at += 1
    return kp.to(DEV), vp.to(DEV), tables.to(DEV), order[:front].to(torch.int32).to(DEV), ks, vs


def check_rows(got, q, ks, vs, alpha, what):
    for b in range(q.shape[0]):
        Hkv, G = ks[b].shape[0], q.shape[1] // ks[b].shape[0]
        for h in range(Hkv):
            want, tol = ref.attend(q[b, h * G:(h + 1) * G, 0].cpu(), ks[b][h], vs[b][h], alpha)
            ref.check(got[b, h * G:(h + 1) * G, 0], want, tol, f"{what} request {b} head {h}")


def is_shared(B, Hq, Hkv, D, dtype, most, page, front):
    """Whether the call computes a prefix of `front` pages for all requests together (else they take the kernels of a call without one)."""
    keys = _lib.load().adsp_attn_paged_shared_keys(B, Hq, Hkv, D, {F32: 0, BF16: 1, F16: 2}[dtype], most, page, front)
    assert keys in (0, min(front * page, most))
    return keys > 0


def run(lens, front, Hq, Hkv, D, page, dtype, alpha=1.5, q_scale=1.0, bits=torch.int32, max_length=None, shared=True, **more):
    what = f"lens={lens[:6]}.. of {len(lens)} front={front} Hq={Hq} Hkv={Hkv} D={D} page={page} {dtype} alpha={alpha} q*{q_scale}"
    print(what, flush=True)
    kp, vp, tables, prefix, ks, vs = family(lens, front, Hkv, D, page, dtype, seed=len(lens) + D + page, **more)
    q = (torch.randn(len(lens), Hq, 1, D, generator=torch.Generator().manual_seed(5)) * q_scale).to(dtype).to(DEV)
    lengths = torch.tensor(lens, dtype=bits, device=DEV)
    assert is_shared(len(lens), Hq, Hkv, D, dtype, tables.shape[1] * page if max_length is None else max_length, page, front) == shared

    def call():
        return A.paged_attention(q, kp, vp, tables, lengths, alpha=alpha, max_length=max_length, prefix_table=prefix)

    out = call()
    assert out.shape == q.shape and out.dtype == dtype
    check_rows(out, q, ks, vs, alpha, what)
    assert torch.equal(out, call())


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_types_and_head_dims(dtype, D):
    run([900, 1020, 857, 990, 856], 53, 8, 2, D, 16, dtype)  # twenty rows of a head
    run([1100 + 7 * i for i in range(9)], 68, 4, 1, D, 16, dtype)
    run([900, 1020, 857], 53, 4, 2, D, 16, dtype)  # six
    run([2100, 1500], 90, 32, 2, D, 16, dtype)  # 32 rows of two requests


@pytest.mark.parametrize("alpha", [1.05, 1.25, 1.333, 1.5, 1.75, 2.0])
@pytest.mark.parametrize("q_scale", [0.125, 1.0, 4.0])
def test_alphas_and_spreads(alpha, q_scale):
    for dtype in (F32, BF16):
        run([900, 1000, 841], 26, 4, 2, 64, 32, dtype, alpha, q_scale)
        run([900 + 40 * i for i in range(11)], 27, 4, 2, 64, 32, dtype, alpha, q_scale)


@pytest.mark.parametrize("page", [1, 7, 8, 16, 100, 257])
def test_lengths_around_the_prefix(page):
    """Requests that end inside the prefix, at its end and behind it, and empty ones."""
    front = 800 // page + 1
    n = front * page
    lens = [0, 1, n - 1, n, n + 1, n // 2, n + page, n + 300, 2, 63, 64, 65, 128]
    run(lens, front, 4, 2, 64, page, BF16, bits=torch.int64)
    run([0, n - 1, n, n + 1, n // 2, n + page], front, 2, 2, 64, page, BF16, bits=torch.int64)


@pytest.mark.parametrize("group", [1, 2, 3, 5, 8, 15, 16, 17, 33, 64])
def test_groups(group):
    run([900, 1100, 820, 850], 50, group * 2, 2, 64, 16, BF16)
    run([870, 1013], 50, group, 1, 128, 16, F32)


def test_parts():
    run([5000 + 100 * i for i in range(6)], 300, 8, 2, 128, 16, BF16)
    run([5000 + 100 * i for i in range(3)], 300, 8, 2, 128, 16, BF16)
    run([20000, 20001], 1250, 4, 1, 64, 16, F16, 2.0, 0.125)
    run([20000 + i for i in range(20)], 1250, 1, 1, 32, 16, F16, 2.0, 0.125)
    run([3000] * 40, 187, 8, 8, 64, 16, BF16, max_length=3000, extra=50)
    run([1030 + i for i in range(4)], 64, 2, 2, 128, 16, BF16)


def test_short_prefixes_take_the_other_kernels():
    run([300, 420, 257, 390, 256], 16, 8, 2, 64, 16, BF16, shared=False)
    run([1000] * 200, 60, 4, 2, 32, 16, BF16, shared=False)
    run([1000], 60, 4, 2, 64, 16, BF16, shared=False)


def test_many_requests():
    run([1300 + (37 * i) % 200 for i in range(200)], 80, 2, 1, 64, 16, BF16)


def test_a_prefix_that_does_not_fit():
    """Tables that differ from the prefix table somewhere, a prefix longer than the tables or than ``max_length``, of pages outside the cache: every request's own table counts."""
    g = torch.Generator().manual_seed(2)
    page, front, lens = 16, 60, [1400, 1350, 1000, 961, 900, 300]
    kp, vp, tables, prefix, ks, vs = family(lens, front, 2, 64, page, BF16, 3)
    q = torch.randn(len(lens), 8, 1, 64, generator=g).to(BF16).to(DEV)
    lengths = torch.tensor(lens, device=DEV)

    def call(prefix, tables=tables, max_length=None):
        return A.paged_attention(q, kp, vp, tables, lengths, max_length=max_length, prefix_table=prefix)

    for what, p in (("none", None), ("empty", prefix[:0]), ("one page", prefix[:1]), ("shorter", prefix[:11]), ("longer", torch.cat([prefix, prefix, prefix, prefix])),
                    ("another order", prefix.flip(0)), ("another page", torch.cat([prefix[:13], prefix[:1], prefix[14:]])), ("another last page", torch.cat([prefix[:-1], prefix[:1]])), ("outside", torch.full_like(prefix, -1)),
                    ("far outside", torch.full_like(prefix, 1 << 30)), ("strides", torch.stack([prefix, prefix], 1)[:, 0])):
        check_rows(call(p), q, ks, vs, 1.5, what)
    # one request has other pages in the middle
    kp2, vp2 = torch.cat([kp, kp.roll(5, 0)]), torch.cat([vp, vp.roll(5, 0)])
    for at in (0, 5, 29, 59):
        other = tables.clone()
        other[1, at] = kp.shape[0] + (other[1, at] + 5) % kp.shape[0]
        check_rows(A.paged_attention(q, kp2, vp2, other, lengths, prefix_table=prefix), q, ks, vs, 1.5, f"other page at {at}")
    # cut off inside the prefix, and behind it
    for most in (1, 100, 800, 950, 960, 961, 1100):
        cut = [[x[:, :most] for x in t] for t in (ks, vs)]
        check_rows(call(prefix, max_length=most), q, *cut, 1.5, f"max_length {most}")
    # entries outside the cache are pages without keys, in the prefix too
    holes = tables.clone()
    holes[:, 4] = -1
    holes[:, 20] = 1 << 29
    keep = torch.ones(1400, dtype=torch.bool)
    keep[4 * page:5 * page] = keep[20 * page:21 * page] = False
    cut = [[x[:, keep[: x.shape[1]]] for x in t] for t in (ks, vs)]
    for p in (prefix, torch.where((torch.arange(front, device=DEV) == 4) | (torch.arange(front, device=DEV) == 20), holes[0, :front], prefix)):
        check_rows(call(p, tables=holes), q, *cut, 1.5, "holes")


def test_scores_that_are_not_finite():
    """In the prefix: a key with a score of -inf or NaN has no weight, a row with one of +inf is zeros, for every request."""
    for lens, front, page in (([900, 910, 890], 55, 16), ([900 + i for i in range(9)], 55, 16)):
        scores_that_are_not_finite(lens, front, page)


def scores_that_are_not_finite(lens, front, page):
    kp, vp, tables, prefix, ks, vs = family(lens, front, 1, 64, page, F32, 4, fill=0.0)
    q = torch.ones(len(lens), 4, 1, 64)
    assert is_shared(len(lens), 4, 1, 64, F32, tables.shape[1] * page, page, front)
    at = int(prefix[3])
    plain = A.paged_attention(q.to(DEV), kp, vp, tables, torch.tensor(lens, device=DEV))
    for bad in (-float("inf"), float("nan"), float("inf")):
        kp[at, 0, 5, 0] = bad
        got, want = (A.paged_attention(q.to(DEV), kp, vp, tables, torch.tensor(lens, device=DEV), prefix_table=p) for p in (prefix, None))
        assert torch.isfinite(got).all() and torch.allclose(got, want, atol=1e-6)
        assert (got == 0).all() if bad == float("inf") else not torch.equal(got, torch.zeros_like(got))
    assert torch.isfinite(plain).all()


def test_a_batch_in_several_launches():
    """A workspace beyond 1 GiB: 60 requests of a table of 40000 tokens are several launches, and so are 300 behind a prefix that is too short for so many."""
    run([1700 + i % 50 for i in range(60)], 100, 64, 8, 64, 16, BF16, extra=2400)
    run([200 + i % 50 for i in range(300)], 12, 64, 8, 64, 16, BF16, extra=500, shared=False)


def test_streams_and_graphs():
    g = torch.Generator().manual_seed(6)
    lens = [1300 + 13 * i for i in range(8)]
    kp, vp, tables, prefix, ks, vs = family(lens, 75, 2, 64, 16, BF16, 7, extra=4)
    q = torch.zeros(8, 8, 1, 64, dtype=BF16, device=DEV)
    assert is_shared(8, 8, 2, 64, BF16, tables.shape[1] * 16, 16, 75)
    lengths = torch.tensor(lens, device=DEV)

    def call(p=prefix):
        return A.paged_attention(q, kp, vp, tables, lengths, prefix_table=p)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(4):
        q.copy_(torch.randn(q.shape, generator=g))
        lengths.copy_(torch.tensor([n - 100 * i for n in lens]))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call())
        cut = [[x[:, : n - 100 * i] for x, n in zip(t, lens)] for t in (ks, vs)]
        check_rows(out, q, *cut, 1.5, f"replay {i}")
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = call()
        torch.cuda.synchronize()
        assert torch.equal(out, other)


def test_a_cache_beyond_32_bits():
    """Pages whose numbers in elements pass 2^31, and 2^32 bytes."""
    pages, Hkv, page, D = 1100000, 1, 16, 128
    kp, vp = (torch.empty(pages, Hkv, page, D, dtype=BF16, device=DEV) for _ in range(2))
    g = torch.Generator().manual_seed(8)
    lens, front = [1000, 1020, 990, 1040, 1005], 61
    far = torch.arange(pages - 400, pages).flip(0)
    kp[pages - 400:], vp[pages - 400:] = (torch.randn(400, Hkv, page, D, generator=g).to(BF16).to(DEV) for _ in range(2))
    tables = torch.full((5, 66), -1, dtype=torch.int32)
    for b in range(5):
        tables[b, :front], tables[b, front:] = far[:front].int(), far[front + 5 * b:front + 5 * b + 5].int()
    q = torch.randn(5, 4, 1, D, generator=g).to(BF16).to(DEV)
    got = A.paged_attention(q, kp, vp, tables.to(DEV), torch.tensor(lens, device=DEV), prefix_table=far[:front].int().to(DEV))
    assert is_shared(5, 4, 1, D, BF16, 66 * page, page, front)
    rows = [[t[tables[b].long().to(DEV)].transpose(1, 2).reshape(-1, Hkv, D)[:n].transpose(0, 1).cpu() for b, n in enumerate(lens)] for t in (kp, vp)]
    check_rows(got, q, *rows, 1.5, "far pages")
