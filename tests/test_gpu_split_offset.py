"""Entmax does not change when a row's scores all move by the same amount: the weights of the kernels that split the keys sum to 1 wherever the scores lie.

A column of V that is 1 for every key makes that column of the output the sum of the weights over what they are divided by, and dO of ones makes the sum of dv
over the keys the same.  Both are sums of n non-negative terms in single precision: off by some sqrt(n) half steps, of which four times are allowed here for each
of the two sums.
"""

import math

import pytest
import torch

import adasplash_amd as A
from tests import op_reference as ref
from tests.test_gpu_paged import make_cache

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
# where (alpha - 1) q k / sqrt(D) lies: the powers of two keep the offset itself exact in 16 bits, too
OFFSETS = [0.0, 16.0, 64.0, 2.0 ** 14, 5 * 2.0 ** 20, 2.0 ** 26, -64.0, -2.0 ** 26]


def allowed(n, dtype):
    return 8 * math.sqrt(n) * ref.half_step(F32) + (ref.half_step(dtype) if dtype != F32 else 0.0)


def moved(q, k, offset, alpha):
    """Column 0 of q and k: a common score of `offset`, exact in every type here."""
    D = q.shape[-1]
    total = offset * math.sqrt(D) / (alpha - 1.0)
    a = 2.0 ** math.floor(math.log2(abs(total)) / 2) if total else 0.0
    q[..., 0], k[..., 0] = a, (total / a if total else 0.0)


@pytest.mark.parametrize("offset", OFFSETS)
@pytest.mark.parametrize("alpha", [1.25, 1.5, 2.0])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_paged_weights_sum_to_one(dtype, alpha, offset):
    """Parts of 64 keys and a request in one kernel; spreads that leave a few, some hundred and thousands of members (more than a list holds)."""
    D = 64
    for lens, spread in (([3000, 700], 1.0), ([3000, 700], 1 / 32), ([20000], 1 / 512), ([300] * 200, 1 / 32)):
        print(len(lens), lens[0], spread, dtype, alpha, offset, flush=True)
        kp, vp, tables, ks, vs = make_cache(lens, 1, D, 16, dtype, seed=7)
        q = torch.randn(len(lens), 4, 1, D, generator=torch.Generator().manual_seed(1)) * spread
        q = q.to(dtype)
        moved(q, kp, offset, alpha)
        vp[..., 1] = 1.0
        out = A.paged_attention(q.to(DEV), kp, vp, tables, torch.tensor(lens, device=DEV), alpha=alpha)
        assert torch.isfinite(out).all()
        off = (out[..., 1].double() - 1).abs().max().item()
        assert off <= allowed(max(lens), dtype), f"weights sum to 1 but for {off:.2e}"


@pytest.mark.parametrize("offset", OFFSETS)
@pytest.mark.parametrize("alpha", [1.25, 1.5, 2.0])
def test_few_queries_and_their_gradients(alpha, offset):
    D = 64
    for n, spread in ((700, 1.0), (5000, 1 / 32), (20000, 1 / 512)):
        print(n, spread, alpha, offset, flush=True)
        g = torch.Generator().manual_seed(3)
        q, k, v = (torch.randn(1, 2, m, D, generator=g) for m in (1, n, n))
        q *= spread
        moved(q, k, offset, alpha)
        v[..., 1] = 1.0
        ts = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
        out = A.cross_attention(*ts, alpha=alpha)
        dv, = torch.autograd.grad(out, (ts[2],), torch.ones_like(out))
        for what, x in (("output", out[..., 1]), ("dv", dv.double().sum(2))):
            off = (x.double() - 1).abs().max().item()
            assert off <= allowed(n, F32), f"{what}: weights sum to 1 but for {off:.2e}"


@pytest.mark.parametrize("alpha", [1.5, 2.0])
def test_an_offset_changes_nothing_else(alpha):
    """Scores that single precision holds exactly with and without the offset (multiples of 2^-4 below 2^10): the same weights, and so the same output, to the
    roundings of the threshold and the sums (2e-6 of the weights' sum is the solver's own limit)."""
    D, n = 64, 3000
    g = torch.Generator().manual_seed(4)
    q, k = torch.zeros(1, 2, 1, D), torch.zeros(1, 2, n, D)
    q[..., 1] = 8.0 / (alpha - 1.0)
    k[..., 1] = torch.randint(-8, 9, (1, 2, n), generator=g) / 16.0
    v = torch.randn(1, 2, n, D, generator=g)
    do = torch.randn(1, 2, 1, D, generator=g)
    results = []
    for offset in (0.0, 512.0):
        moved(q, k, offset, alpha)
        ts = [t.clone().to(DEV).requires_grad_(True) for t in (q, k, v)]
        out = A.cross_attention(*ts, alpha=alpha)
        results.append([out, *torch.autograd.grad(out, ts, do.to(DEV))])
    # dq's one column is a sum of dX k / sqrt(D) in which a row's dX cancel: its size is that of the terms, |dk| / q of dX / sqrt(D) times k
    terms = (results[0][2][..., 1].double().abs() * k[..., 1].to(DEV).abs()).sum(-1) / q[0, 0, 0, 1].item()
    for name, a, b in zip(("out", "dq", "dk", "dv"), *results):
        a, b = a[..., 1:].double(), b[..., 1:].double()
        size = terms.norm() if name == "dq" else a.norm()
        assert (a - b).norm() <= 1e-5 * size, (name, ((a - b).norm() / size).item())
