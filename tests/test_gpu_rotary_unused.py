"""Outputs of ``rotary`` that nothing is computed from: no gradient comes back for their rows and weights, and the others' are what they are without them."""

import pytest
import torch

import adasplash_amd as A
from tests import positions_reference as pos

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("norms", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_no_gradient_for_what_is_not_used(dtype, norms):
    g = torch.Generator().manual_seed(1)
    f, at = pos.frequencies_of(64).to(DEV), torch.arange(50, device=DEV)
    q, k = (torch.randn(2, h, 50, 64, generator=g).to(dtype).to(DEV).requires_grad_(True) for h in (4, 2))
    wq, wk = (torch.rand(64, generator=g).to(DEV).requires_grad_(True) if norms else None for _ in range(2))
    leaves = [t for t in (q, k, wq, wk) if t is not None]
    dq, dk = (torch.randn(t.shape, generator=g).to(dtype).to(DEV) for t in (q, k))

    def outs():
        return A.rotary(q, k, at, f, q_weight=wq, k_weight=wk)

    both = torch.autograd.grad(outs(), leaves, (dq, dk))
    for i, dy in enumerate((dq, dk)):
        grads = torch.autograd.grad(outs()[i], leaves, dy, allow_unused=True)
        for j, grad in enumerate(grads):
            if j % 2 == i and j < 2:
                assert torch.equal(grad, both[j])
            elif j % 2 == i:
                # (a weight's sum over n rows may be taken in another order: each is off by n half steps of the terms' size; a turned gradient is at most sqrt(2) as large, a normed element 8)
                rows = dy.numel() // 64
                assert (grad - both[j]).abs().max() <= 2 * rows * 2.0 ** -24 * 8 * 2 ** 0.5 * dy.float().abs().sum((0, 1, 2)).max()
            else:
                assert grad is None
    a, b = outs()
    assert torch.autograd.grad(a.detach().sum() + q.sum(), leaves, allow_unused=True)[1] is None
    (a.sum() + 0 * b.detach().sum()).backward()
    assert q.grad is not None and k.grad is None


def test_half_of_two_calls():
    """The queries of one call and the keys of another: each leaf has the gradient of its own use."""
    g = torch.Generator().manual_seed(2)
    f, at = pos.frequencies_of(32).to(DEV), torch.arange(9, device=DEV)
    x = torch.randn(1, 3, 9, 32, generator=g).to(DEV).requires_grad_(True)
    a, b = A.rotary(x, x, at, f)[0], A.rotary(x, x, at + 3, f)[1]
    got = torch.autograd.grad(a.sum() + 2 * b.sum(), x)[0]
    one = [torch.autograd.grad(A.rotary(x, None, at + s, f)[0].sum(), x)[0] for s in (0, 3)]
    assert torch.allclose(got, one[0] + 2 * one[1], atol=1e-5)
