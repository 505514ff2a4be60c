"""Attention behind a common prefix: a row's result hangs on its own numbers and not on what lies beside it in its workgroup, bit for bit."""

import pytest
import torch

import adasplash_amd as A
from tests.test_gpu_prefix import BF16, DEV, F16, F32, family, is_shared

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype, D", [(BF16, 128), (F16, 64), (F32, 64), (BF16, 256), (F32, 256)])
@pytest.mark.parametrize("scale", [0.02, 0.4, 1.0])
def test_rows_do_not_hang_on_their_neighbours(dtype, D, scale):
    """24 requests that are the same but for their place, beside others that are not: the same bits in every place, in every order."""
    page, front, Hq, Hkv, n = 16, 70, 8, 2, 1170
    g = torch.Generator().manual_seed(D)
    lens = [n] * 24
    kp, vp, tables, prefix, _, _ = family(lens, front, Hkv, D, page, dtype, seed=3)
    tables[:] = tables[:1]  # (one request, 24 times: its own part too)
    lengths = torch.tensor(lens, device=DEV)
    assert is_shared(24, Hq, Hkv, D, dtype, tables.shape[1] * page, page, front)
    one = torch.randn(Hq, 1, D, generator=g) * scale
    others = torch.randn(24, Hq, 1, D, generator=g) * scale * 3
    want = None
    for turn in range(4):
        same = torch.randperm(24, generator=g)[: 24 - 5 * turn]
        q = others.clone()
        q[same] = one
        got = A.paged_attention(q.to(dtype).to(DEV), kp, vp, tables, lengths, prefix_table=prefix)
        want = got[same[0]].clone() if want is None else want
        for b in same.tolist():
            assert torch.equal(got[b], want), f"turn {turn}, request {b}"
