"""Rows and weights of ``rotary`` that want no gradient beside others that do: their output wants none either, and what reads it does not refuse it."""

import pytest
import torch

import adasplash_amd as A
from adasplash_amd.paged import PagedCache
from tests import positions_reference as pos

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("q_grad, k_grad, wq_grad, wk_grad", [(0, 1, 0, 0), (1, 0, 0, 0), (0, 0, 1, 0), (0, 0, 0, 1), (1, 0, 0, 1), (0, 1, 0, 1), (1, 1, 1, 1)])
def test_outputs_ask_as_their_inputs_do(q_grad, k_grad, wq_grad, wk_grad):
    g = torch.Generator().manual_seed(1)
    f, at = pos.frequencies_of(64).to(DEV), torch.arange(20, device=DEV)
    values = [torch.randn(2, h, 20, 64, generator=g).to(DEV) for h in (4, 2)] + [torch.rand(64, generator=g).to(DEV) for _ in range(2)]
    want = [bool(x) for x in (q_grad, k_grad, wq_grad, wk_grad)]
    q, k, wq, wk = leaves = [t.clone().requires_grad_(w) for t, w in zip(values, want)]
    outs = A.rotary(q, k, at, f, q_weight=wq, k_weight=wk)
    assert [o.requires_grad for o in outs] == [want[0] or want[2], want[1] or want[3]]
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(outs, A.rotary(q, k, at, f, q_weight=wq, k_weight=wk)))
    every = [t.clone().requires_grad_(True) for t in values]
    dy = [torch.randn(o.shape, generator=g).to(DEV) for o in outs]
    all_outs = A.rotary(*every[:2], at, f, q_weight=every[2], k_weight=every[3])
    used = [i for i in range(2) if outs[i].requires_grad]
    got = torch.autograd.grad([outs[i] for i in used], [t for t, w in zip(leaves, want) if w], [dy[i] for i in used])
    expected = torch.autograd.grad([all_outs[i] for i in used], [t for t, w in zip(every, want) if w], [dy[i] for i in used])
    assert all(torch.equal(a, b) for a, b in zip(got, expected))


def test_a_fixed_query_attends():
    """Keys that train beside queries that do not: the turned queries go into a call that takes no gradient."""
    f, B, D = pos.frequencies_of(64).to(DEV), 2, 64
    cache = PagedCache(8, 4, B, 2, D, 12, dtype=torch.float32)
    rows = torch.randn(B, 2, D, generator=torch.Generator().manual_seed(3)).to(DEV)
    cache.append(rows, rows)
    q, k = torch.ones(B, 4, 1, D, device=DEV), torch.ones(B, 2, 1, D, device=DEV, requires_grad=True)
    turned, keys = A.rotary(q, k, torch.zeros(1, dtype=torch.int64, device=DEV), f)
    assert torch.equal(cache.attend(turned), cache.attend(q)) and keys.requires_grad
    turned.mul_(2)  # (and can be written to, as any tensor without a gradient)
    keys.sum().backward()
    assert k.grad is not None
