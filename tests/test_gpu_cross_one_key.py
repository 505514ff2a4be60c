"""An item of one key: its weight is 1 whatever the scores are, so dq and dk are zeros, and dv is the sum of dO."""

import pytest
import torch

import adasplash_amd as A
from tests import op_reference as ref
from tests.test_gpu_cross import inputs

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("B, Hq, Hkv, Nq, Nk", [(2, 4, 2, 76, 1), (20, 12, 12, 22, 1), (5, 8, 2, 3, 1), (3, 8, 2, 700, 1), (2, 4, 4, 100, 40), (2, 4, 2, 100, 700), (2, 4, 2, 60, 2500)])
def test_one_key(B, Hq, Hkv, Nq, Nk, D, dtype):
    for alpha in (1.333, 1.5, 2.0):
        q, k, v, do = inputs(B, Hq, Hkv, Nq, Nk, D, dtype, seed=1, q_scale=3.0)
        ts = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
        lens = torch.ones(B, dtype=torch.int32, device=DEV)
        out = A.cross_attention(*ts, alpha=alpha, varlen_k=lens if Nk > 1 else None)
        dq, dk, dv = torch.autograd.grad(out, ts, do.to(DEV))
        assert (dq == 0).all() and (dk == 0).all() and (dv[:, :, 1:] == 0).all()
        terms = do.double().view(B, Hkv, -1, D)
        want, size = terms.sum(2), terms.abs().sum(2)
        # a sum of n terms in single precision: four times sqrt(n) half steps of their size; rounded to the type; f16's steps end at 2^-24
        n = terms.shape[2]
        tol = 4 * n ** 0.5 * ref.half_step(F32) * size + ref.half_step(dtype) * (want.abs() + size * 2.0 ** -12) * (1 if dtype != F32 else 2) + ref.least_half_step(dtype)
        ref.check(dv[:, :, 0], want, tol, f"dv alpha={alpha}")
