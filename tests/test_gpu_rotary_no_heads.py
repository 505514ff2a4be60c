"""``rotary`` of queries, or keys, without heads beside others that have some: their weight's gradient is zero."""

import pytest
import torch

import adasplash_amd as A
from tests import positions_reference as pos

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("heads", [(0, 2), (3, 0), (0, 0)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_no_rows_no_gradient(heads, dtype):
    f, at = pos.frequencies_of(256).to(DEV), torch.arange(6, device=DEV)
    q, k = (torch.ones(2, h, 6, 256, dtype=dtype, device=DEV, requires_grad=True) for h in heads)
    weights = [torch.ones(256, dtype=dtype, device=DEV, requires_grad=True) for _ in range(2)]
    a, b = A.rotary(q, k, at, f, q_weight=weights[0], k_weight=weights[1])
    ones = torch.ones_like(a), torch.ones_like(b)
    torch.cuda.synchronize()
    left = [torch.full((256,), float("nan"), dtype=dtype, device=DEV) for _ in range(64)]  # what the allocator hands out next
    del left
    grads = torch.autograd.grad((a, b), (q, k, *weights), ones)
    for i in range(2):
        assert grads[i].shape[1] == heads[i] and torch.isfinite(grads[2 + i]).all()
        if heads[i] == 0:
            assert (grads[2 + i] == 0).all()
        else:
            assert (grads[2 + i] != 0).any()
