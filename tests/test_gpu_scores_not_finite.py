"""Infinite and NaN scores inside the valid lengths, for attention to keys of another length and over pages: a row with a score of +inf is 0, as are
its gradients; keys of score -inf or NaN have no weight and no gradients.  Whatever kernels serve a call, and whatever else is in its batch."""

import math

import pytest
import torch

import adasplash_amd as A
from tests import op_reference as ref
from tests.test_gpu_cross import inputs
from tests.test_gpu_paged import make_cache

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
INF, NAN = math.inf, math.nan

ROUTES = {
    "parts of 64 keys": (2, 4, 2, 3, 700, 64, F32),
    "one kernel or parts": (2, 4, 2, 3, 700, 64, BF16),
    "parts of 2048 keys, the last short": (64, 16, 16, 1, 2100, 32, F16),
    "parts of 256 keys": (16, 8, 8, 4, 700, 128, BF16),
    "32 rows, single precision": (2, 4, 2, 100, 700, 64, F32),
    "32 rows, single precision, D = 128": (1, 4, 2, 70, 300, 128, F32),
    "few keys, single precision": (1, 4, 2, 90, 20, 64, F32),
    "resident": (2, 4, 2, 100, 700, 64, BF16),
    "resident, f16": (2, 4, 2, 100, 300, 128, F16),
    "32 rows, 16 bits": (2, 4, 2, 100, 2500, 128, F16),
    "all pairs beyond 16-bit keys": (1, 2, 1, 100, 66000, 64, BF16),
    "tiles": (2, 4, 2, 70, 150, 32, F32),
    "tiles, 16 bits": (2, 4, 2, 70, 150, 256, BF16),
}


def one_bad_key(shape, key, row, value, by):
    """Key `key` has `value` in its column 5, query `row` has `by` there, every other key and query 0."""
    q, k, v, do = inputs(*shape)
    q[..., 5], k[..., 5] = 0.0, 0.0
    q[:, :, row, 5] = by
    k[:, :, key, 5] = value
    return q, k, v, do


def expected(q, k, v, do, b, h, rows, keys, train, alpha):
    """(want, tolerance) of the output of `rows`, and of the gradients that they alone give, over `keys` alone; column 5 is 0 in both."""
    G = q.shape[1] // k.shape[1]
    D = q.shape[-1]
    hs = slice(h * G, (h + 1) * G)
    qq, dd = (t[b, hs][:, rows].reshape(-1, D) for t in (q, do))
    kk, vv = k[b, h, keys], v[b, h, keys]
    return ref.attend(qq, kk, vv, alpha, roundings=2), ref.gradients(qq, kk, vv, dd, alpha) if train else None


def run(shape, key, row, value, by, alpha=1.5, train=True):
    B, Hq, Hkv, Nq, Nk, D, dtype = shape
    G = Hq // Hkv
    print(shape, key, row, value, by, alpha, flush=True)
    q, k, v, do = one_bad_key(shape, key, row, value, by)
    ts = [t.to(DEV).requires_grad_(train) for t in (q, k, v)]
    out = A.cross_attention(*ts, alpha=alpha)
    if train:
        with torch.no_grad():
            ref.check(out, out.detach().double().cpu(), torch.zeros(()), "a training step's output")  # (finite)
        dq, dk, dv = torch.autograd.grad(out, ts, do.to(DEV))
    top = value * by == INF
    rows = [r for r in range(Nq) if not (top and r == row)]
    # with an infinite or NaN operand every other row's score is 0 * it, NaN; where only the product overflows it is an ordinary one
    ordinary = math.isfinite(value)
    keys = [j for j in range(Nk) if j != key]
    if top:
        assert (out[:, :, row] == 0).all(), "a row with a score of +inf is 0"
    if ordinary:
        return
    columns = [c for c in range(D) if c != 5]
    for b in {0, B - 1}:
        for h in {0, Hkv - 1}:
            if not rows:
                continue
            want, grads = expected(q, k, v, do, b, h, rows, keys, train, alpha)
            hs = slice(h * G, (h + 1) * G)
            ref.check(out[b, hs][:, rows].reshape(-1, D), *want, f"item {b} head {h}")
            if train:
                for name, got, (w, tol) in (("dq", dq[b, hs][:, rows].reshape(-1, D), grads[0]), ("dk", dk[b, h, keys], grads[1]), ("dv", dv[b, h, keys], grads[2])):
                    # (dq's column 5 is 0 times an infinite key; dk's is 0 times the row's, or the row's where it is infinite)
                    ref.check(got[:, columns], w[:, columns], tol[:, columns], f"{name}, item {b} head {h}")
    if train:
        assert (dk[:, :, key][..., columns] == 0).all() and (dv[:, :, key] == 0).all()
        if top:
            assert (dq[:, :, row][..., columns] == 0).all()
            if Nq == 1:
                assert (dv == 0).all()


@pytest.mark.parametrize("value", [INF, -INF, NAN])
@pytest.mark.parametrize("route", list(ROUTES))
def test_an_infinite_or_nan_key(route, value):
    shape = ROUTES[route]
    Nq, Nk = shape[3], shape[4]
    run(shape, Nk - 1, Nq // 2, value, 1.0)
    run(shape, min(5, Nk - 1), Nq - 1, value, 1.0, train=False)


@pytest.mark.parametrize("alpha", [1.333, 2.0])
@pytest.mark.parametrize("route", ["parts of 64 keys", "one kernel or parts", "parts of 2048 keys, the last short", "parts of 256 keys", "32 rows, single precision", "resident"])
def test_an_infinite_key_and_alphas(route, alpha):
    shape = ROUTES[route]
    run(shape, shape[4] - 1, shape[3] // 2, INF, 1.0, alpha)
    run(shape, 3, 0, INF, 1.0, alpha, train=False)


@pytest.mark.parametrize("route", [r for r in ROUTES if ROUTES[r][6] != F16])
def test_products_beyond_the_type(route):
    shape = ROUTES[route]
    run(shape, shape[4] - 1, 0, 3e38, 100.0, train=False)


@pytest.mark.parametrize("keep", ["never", "always"])
@pytest.mark.parametrize("value", [INF, -INF, NAN])
@pytest.mark.parametrize("alpha", [1.333, 1.5, 2.0])
def test_supports(value, alpha, keep):
    """Large enough for the kernels on the supports, forward and gradients."""
    shape = (10, 4, 2, 1030, 2600, 128, BF16)
    B, Hq, Hkv, Nq, Nk, D, _ = shape
    q, k, v, do = one_bad_key(shape, Nk - 1, 130, value, 1.0)
    ts = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
    before = A.set_keep_supports(keep)
    try:
        out = A.cross_attention(*ts, alpha=alpha)
        grads = torch.autograd.grad(out, ts, do.to(DEV))
        with torch.no_grad():
            alone = A.cross_attention(*ts, alpha=alpha)
    finally:
        A.set_keep_supports(before)
    if value == INF:
        assert (out[:, :, 130] == 0).all() and (alone[:, :, 130] == 0).all()
    assert torch.isfinite(out).all() and torch.isfinite(alone).all()
    rows, keys = [0, 129, 131, 1029], list(range(Nk - 1))
    want, _ = expected(q, k, v, do, 9, 1, rows, keys, False, alpha)
    ref.check(out[9, 2:4][:, rows].reshape(-1, D), *want, "rows beside it")
    columns = [c for c in range(D) if c != 5]
    assert (grads[1][:, :, -1][..., columns] == 0).all() and (grads[2][:, :, -1] == 0).all()
    for g in grads:
        assert torch.isfinite(g[..., columns]).all()
    if value == INF:
        assert (grads[0][:, :, 130][..., columns] == 0).all()


@pytest.mark.parametrize("value", [INF, -INF, NAN])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("lens, width", [([700, 65, 2500], None), ([40, 30], None), ([2049] * 128, None), ([2100, 300] * 40, 600)])
def test_pages(lens, width, dtype, value):
    """Short parts, one kernel for all keys, long parts with a short last one, tables with room to spare: the last key of every request."""
    print(len(lens), width, dtype, value, flush=True)
    kp, vp, tables, ks, vs = make_cache(lens, 8, 32, 16, dtype, seed=3, width=width)
    B, Hq, D = len(lens), 16, 32
    q = torch.randn(B, Hq, 1, D, generator=torch.Generator().manual_seed(5)).to(dtype)
    q[..., 5] = 0.0
    q[:, 1::2, :, 5] = 1.0
    for b, n in enumerate(lens):
        ks[b][..., 5] = 0.0
        page, at = int(tables[b, (n - 1) // 16]), (n - 1) % 16
        for i in range(-(-n // 16)):
            kp[int(tables[b, i]), :, :, 5] = 0.0
        kp[page, :, at, 5] = value
    out = A.paged_attention(q.to(DEV), kp, vp, tables, torch.tensor(lens, device=DEV))
    if value == INF:
        assert (out[:, 1::2] == 0).all(), "a row with a score of +inf is 0"
    for b in {0, 1, B - 1}:
        for h in range(0, 8, 7):
            sees = [h * 2] if value == INF else [h * 2, h * 2 + 1]
            want, tol = ref.attend(q[b, sees, 0], ks[b][h, :-1], vs[b][h, :-1], 1.5)
            ref.check(out[b, sees, 0], want, tol, f"request {b} head {h}")
