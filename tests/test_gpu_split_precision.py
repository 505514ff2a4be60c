"""Scores in single precision where the keys are split: four sums of every fourth product each.

A sum of n products in turn has n roundings of the running sum's size, sqrt(k) behind k products, so its error goes with sqrt(1 + 2 + ... + n) = n / sqrt(2).  Four sums of n / 4 have
2 (n / 4) / sqrt(2) together, half of that.  The outputs' error follows the scores'; three quarters of what one sum gives (formed here, and everything behind it in 64 bits) leave room for the kernels'
other roundings.
"""

import math

import pytest
import torch

import adasplash_amd as A
from oracle import exact
from tests.test_gpu_paged import make_cache

pytestmark = pytest.mark.gpu
DEV = "cuda"


def one_sum(q, k):
    """q (m, D), k (n, D) in single precision: products as a fused multiply-add forms them, one after another."""
    s = torch.zeros(q.shape[0], k.shape[0])
    for d in range(q.shape[1]):
        s = (s.double() + q[:, d:d + 1].double() * k[:, d].double()).float()
    return s.double()


@pytest.mark.parametrize("n, D, alpha, spread", [(2386, 128, 2.0, 1.0), (2316, 128, 1.5, 1.0), (1500, 256, 1.5, 1.0), (464, 64, 1.5, 3.0), (3000, 64, 2.0, 3.0)])
def test_scores_are_four_sums(n, D, alpha, spread):
    heads = 8
    kp, vp, tables, ks, vs = make_cache([n], heads, D, 16, torch.float32, seed=11)
    q = torch.randn(1, heads, 1, D, generator=torch.Generator().manual_seed(2)) * spread
    out = A.paged_attention(q.to(DEV), kp, vp, tables, torch.tensor([n], device=DEV), alpha=alpha)[0, :, 0].double().cpu()
    cross = A.cross_attention(q.to(DEV), ks[0][None].to(DEV), vs[0][None].to(DEV), alpha=alpha)[0, :, 0].double().cpu()
    want, model = torch.zeros(heads, D, dtype=torch.float64), torch.zeros(heads, D, dtype=torch.float64)
    for h in range(heads):
        k, v = ks[0][h], vs[0][h].double()
        want[h] = (exact.entmax_rows(q[0, h].double() @ k.double().T / math.sqrt(D), alpha) @ v)[0]
        model[h] = (exact.entmax_rows(one_sum(q[0, h], k) / math.sqrt(D), alpha) @ v)[0]
    bound = 0.75 * (model - want).norm()
    for name, got in (("paged", out), ("cross", cross)):
        assert (got - want).norm() <= bound, (name, ((got - want).norm() / want.norm()).item(), (bound / want.norm()).item())
