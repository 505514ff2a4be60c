"""The 64-bit reference of turned heads: against complex numbers, differences, and what turning is for."""

import math

import pytest
import torch

import adasplash_amd as A
from tests import positions_reference as ref


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_scores_go_by_the_distance(layout):
    g = torch.Generator().manual_seed(0)
    q, k = (torch.randn(32, generator=g, dtype=torch.float64) for _ in range(2))
    f = ref.frequencies_of(24)
    at = torch.tensor([5, 1000, 12345])
    scores = (ref.forward(q.expand(3, 32), at, f, layout) * ref.forward(k.expand(3, 32), at - 3, f, layout)).sum(-1)
    assert torch.allclose(scores, scores[0].expand(3), atol=1e-9)
    assert torch.allclose(ref.forward(q.expand(1, 32), torch.tensor([0]), f, layout)[0], q, atol=0)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("norm", [False, True])
def test_gradients_against_differences(layout, norm):
    g = torch.Generator().manual_seed(1)
    x, dy = (torch.randn(2, 3, 5, 16, generator=g, dtype=torch.float64) for _ in range(2))
    w = 1 + 0.3 * torch.randn(16, generator=g, dtype=torch.float64) if norm else None
    f, at = ref.frequencies_of(8, 100.0), torch.arange(5) * 3
    (dx, _), more = ref.backward(x, dy, at, f, layout, w, 1e-3, 1.3)

    def loss(x, w):
        return (ref.forward(x, at, f, layout, w, 1e-3, 1.3) * dy).sum()

    for _ in range(4):
        v, h = torch.randn(x.shape, generator=g, dtype=torch.float64), 1e-5
        assert math.isclose((loss(x + h * v, w) - loss(x - h * v, w)).item() / (2 * h), (dx * v).sum().item(), rel_tol=1e-6, abs_tol=1e-7)
        if norm:
            u = torch.randn(16, generator=g, dtype=torch.float64)
            assert math.isclose((loss(x, w + h * u) - loss(x, w - h * u)).item() / (2 * h), (more[0] * u).sum().item(), rel_tol=1e-6, abs_tol=1e-7)


def test_frequencies():
    f, factor = A.rotary_frequencies(64, device="cpu")
    assert f.dtype == torch.float64 and factor == 1.0 and torch.allclose(f, ref.frequencies_of(64), rtol=1e-14, atol=0)
    f, factor = A.rotary_frequencies(64, base=500000.0, stretch=4.0, device="cpu")
    assert factor == 1.0 and torch.allclose(f, ref.frequencies_of(64, 500000.0) / 4, rtol=1e-14, atol=0)
    f, factor = A.rotary_frequencies(64, stretch=8.0, trained_length=4096, device="cpu")
    plain = ref.frequencies_of(64)
    turns = 4096 * plain / (2 * math.pi)
    assert math.isclose(factor, 0.1 * math.log(8.0) + 1.0)
    assert torch.allclose(f[turns >= 32], plain[turns >= 32], rtol=1e-14, atol=0) and torch.allclose(f[turns <= 1], plain[turns <= 1] / 8, rtol=1e-14, atol=0)
    assert (f <= plain * (1 + 1e-14)).all() and (f >= plain / 8 * (1 - 1e-14)).all() and (f[:-1] > f[1:]).all()
    assert A.rotary_frequencies(64, stretch=1.0, trained_length=4096, device="cpu")[1] == 1.0
    for bad in ({"rotary_dim": 12}, {"rotary_dim": 0}, {"rotary_dim": 64, "base": 0.0}, {"rotary_dim": 64, "stretch": 0.5}, {"rotary_dim": 64, "stretch": float("nan")},
                {"rotary_dim": 64, "stretch": 2.0, "trained_length": 0}, {"rotary_dim": 64, "stretch": 2.0, "trained_length": 10, "slow": 5.0, "fast": 5.0}):
        with pytest.raises(ValueError):
            A.rotary_frequencies(device="cpu", **bad)
