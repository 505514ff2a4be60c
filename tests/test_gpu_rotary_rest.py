"""The part of a head that is not turned stays as it is, whatever its elements are: infinities, NaN and zeros of either sign, forward, on the way into pages, and in gradients."""

import pytest
import torch

import adasplash_amd as A
from tests import positions_reference as pos

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
ODD = [float("inf"), -float("inf"), float("nan"), 0.0, -0.0, 1.0, -2.5]


def same_bits(a, b):
    kind = torch.int32 if a.dtype == F32 else torch.int16
    return torch.equal(a.contiguous().view(kind), b.contiguous().view(kind))


def rows(shape, D, rot, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, D, generator=g)
    x[..., rot:] = torch.tensor(ODD)[torch.randint(0, len(ODD), (*shape, D - rot), generator=g)]
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("D, rot", [(16, 8), (64, 0), (64, 32), (128, 96), (256, 8)])
def test_the_rest_of_a_head(dtype, layout, D, rot):
    f, at = pos.frequencies_of(rot), torch.arange(21) * 3
    q, dy = rows((2, 3, 21), D, rot, dtype, 1), rows((2, 3, 21), D, rot, dtype, 2)
    qd = q.to(DEV).requires_grad_(True)
    out, _ = A.rotary(qd, None, at.to(DEV), f.to(DEV), layout=layout, factor=1.5)
    dq = torch.autograd.grad(out, qd, dy.to(DEV))[0]
    for got, x in ((out.detach(), q), (dq, dy)):
        assert same_bits(got[..., rot:].cpu(), x[..., rot:])
        assert torch.isfinite(got[..., :rot]).all()
    k, v = rows((21, 3), D, rot, dtype, 3), rows((21, 3), D, rot, dtype, 4)
    kp, vp = (torch.zeros(6, 3, 4, D, dtype=dtype, device=DEV) for _ in range(2))
    A.write_pages(k.to(DEV), v.to(DEV), torch.arange(21, device=DEV), kp, vp, positions=at.to(DEV), rotary=A.Rotary(f.to(DEV), layout))
    got = [x.transpose(1, 2).reshape(-1, 3, D)[:21].cpu() for x in (kp, vp)]
    assert same_bits(got[0][..., rot:], k[..., rot:]) and torch.isfinite(got[0][..., :rot]).all()
    assert same_bits(got[1], v)
