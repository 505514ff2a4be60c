"""Which pools ``compact_pages`` takes pages into, on the CPU: those that share no memory with the cache or with each other, whatever tensors they are views of."""

import random

import pytest
import torch

import adasplash_amd as A

H, P, D = 2, 4, 8


def taken(k, v, k_to, v_to, lengths=None, tables=None):
    """Whether the pools pass the checks (all of which stand in front of the look at the device)."""
    lengths = torch.tensor([3, 0], dtype=torch.int32) if lengths is None else lengths
    tables = torch.full((2, 4), -1, dtype=torch.int32) if tables is None else tables
    try:
        A.compact_pages(lengths, tables, k, v, k_to, v_to)
    except AssertionError as e:
        assert "tensors" in str(e)
        return False
    except RuntimeError as e:
        assert "ROCm device only" in str(e)
        return True
    raise AssertionError("a CPU tensor was taken")


def common(a, b):
    """Whether two tensors have an element in common, element by element."""
    def of(t):
        offsets = torch.zeros(1, dtype=torch.int64)
        for n, s in zip(t.shape, t.stride()):
            offsets = (offsets[:, None] + torch.arange(n) * s).reshape(-1)
        return set((t.data_ptr() + offsets * t.element_size()).tolist())

    return bool(of(a) & of(b))


def test_pools_of_one_tensor():
    arena = torch.zeros(4, 10, H, P, D)
    k, v, k_to, v_to = arena
    assert taken(k, v, k_to, v_to) and taken(k, v, k_to[3:], v_to[:7])
    assert taken(k[:5], v[:5], k[5:], v[5:])
    assert not taken(k[:6], v[:6], k[5:], v[5:])
    side = torch.zeros(10, 2, H, P, D)  # k and v of a page side by side
    assert taken(k, v, side[:, 0], side[:, 1]) and taken(side[:, 0], side[:, 1], k_to, v_to)
    assert taken(side[:5, 0], side[:5, 1], side[5:, 0], side[5:, 1])
    heads = torch.zeros(10, P, 2 * H, D)  # and of a slot
    assert taken(k, v, heads[:, :, :H].transpose(1, 2), heads[:, :, H:].transpose(1, 2))
    assert not taken(k, v, heads[:, :, :H].transpose(1, 2), heads[:, :, 1:H + 1].transpose(1, 2))
    rows = torch.zeros(10, H, P, 2 * D)
    assert taken(k, v, rows[..., :D], rows[..., D:])
    assert taken(k, v, arena.flatten()[2 * k.numel():][: k.numel()].view_as(k), v_to)


@pytest.mark.parametrize("shift", [4, D, P * D, H * P * D, 3 * H * P * D])
def test_two_pools_at_different_addresses(shift):
    flat = torch.zeros(14 * H * P * D)
    k_to, v_to = flat[:10 * H * P * D].view(10, H, P, D), flat[shift:][:10 * H * P * D].view(10, H, P, D)
    assert not taken(torch.zeros(10, H, P, D), torch.zeros(10, H, P, D), k_to, v_to)
    assert not taken(v_to, torch.zeros(10, H, P, D), k_to, torch.zeros(10, H, P, D))
    assert not taken(torch.zeros(10, H, P, D), v_to, torch.zeros(10, H, P, D), k_to)


def test_tables_and_lengths_in_a_pool():
    pool, other = (torch.zeros(10, H, P, D) for _ in range(2))
    words = pool.view(torch.int32).flatten()
    k = torch.zeros(10, H, P, D)
    assert not taken(k, k + 1, pool, other, lengths=words[5:7]) and not taken(k, k + 1, other, pool, tables=words[-8:].view(2, 4))
    assert taken(k, k + 1, pool[2:], other[2:], lengths=words[5:7])
    half = torch.zeros(10, H, P, D, dtype=torch.bfloat16)
    assert not taken(half.clone(), half.clone(), half, half.clone(), lengths=half.flatten().view(torch.int64)[-4::2])
    assert taken(half.clone(), half.clone(), half, half.clone(), lengths=half.new_zeros(8).view(torch.int64))


def test_against_elements():
    """Views of any strides and places, against the elements that they have."""
    rng = random.Random(3)
    seen = [0, 0]
    for _ in range(400):
        flat = torch.zeros(6000)
        views = []
        for _ in range(2):
            sizes, order, strides, step = (rng.choice((1, 2, 3)), H, P), rng.sample(range(3), 3), [0, 0, 0], D
            for d in order:
                strides[d] = step
                step *= sizes[d] + rng.choice((0, 0, 1))
            views.append(flat.as_strided((*sizes, D), (*strides, 1), 4 * rng.randrange(60)))
        k_to, v_to = views
        if k_to.shape != v_to.shape:
            v_to = v_to[: min(len(k_to), len(v_to))]
            k_to = k_to[: len(v_to)]
        free = not common(k_to, v_to)
        seen[free] += 1
        assert taken(torch.zeros(3, H, P, D), torch.zeros(3, H, P, D), k_to, v_to) == free
    assert min(seen) > 50


def test_large_pools():
    """At sizes of a server: found without a look at every page.  (The memory is only named, never touched.)"""
    side = torch.empty(60000, 2, 8, 16, 128, dtype=torch.bfloat16)
    parts = [side[30000:, 0], side[30000:, 1]]
    assert taken(side[:30000, 0], side[:30000, 1], *parts) and taken(*parts, side[:30000, 0], side[:30000, 1])
    assert not taken(side[:30001, 0], side[:30001, 1], *parts) and not taken(*parts, side[:30001, 1], side[:30001, 0])
    slots = side.view(30000, 8, 16, 4, 128)  # all four side by side in a slot
    assert taken(*(slots[..., i, :] for i in range(4))) and not taken(*(slots[..., i, :] for i in (0, 1, 2, 1)))
