"""The 64-bit gradients that the kernels are held to, against differences of the 64-bit output."""

import pytest
import torch

from tests import op_reference as ref


@pytest.mark.parametrize("alpha", [1.25, 1.333, 1.5, 1.75, 2.0])
def test_gradients_are_the_differences(alpha):
    g = torch.Generator().manual_seed(1)
    q, k, v, do = (torch.randn(n, 16, generator=g, dtype=torch.float64) for n in (5, 9, 9, 5))
    grads = ref.gradients(q, k, v, do, alpha)
    for i, name in enumerate("qkv"):
        at = [q, k, v]
        way = torch.randn(at[i].shape, generator=g, dtype=torch.float64)
        step = 1e-6

        def loss(sign):
            moved = list(at)
            moved[i] = at[i] + sign * step * way
            return (ref.attend(*moved, alpha)[0] * do).sum()

        slope = (loss(1) - loss(-1)) / (2 * step)
        assert abs(slope - (grads[i][0] * way).sum()) < 1e-6 * (1 + abs(slope)), name


def test_nothing_to_attend_to():
    q, do = torch.randn(3, 16), torch.randn(3, 16)
    none = torch.zeros(0, 16)
    assert (ref.attend(q, none, none, 1.5)[0] == 0).all()
    assert all((want == 0).all() for want, _ in ref.gradients(q, none, none, do, 1.5))
