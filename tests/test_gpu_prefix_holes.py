"""Paged attention behind a common prefix whose parts start in pages that are none, with so many keys of weight that the second kernel solves on the parts' entries in memory."""

import pytest
import torch

import adasplash_amd as A
from tests.test_gpu_prefix import BF16, DEV, F16, F32, check_rows, family, is_shared

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype, D, alpha", [(BF16, 64, 1.5), (F32, 32, 2.0), (F16, 128, 1.25)])
@pytest.mark.parametrize("requests", [20, 3])
def test_flat_scores_behind_holes(dtype, D, alpha, requests):
    """Lists of a part are filled up with entries without weight, which name the part's first key: of a page that is none here, the first page of every 128 keys."""
    page, front, Hq, Hkv = 16, 250, 4, 2
    lens = [4000 + 7 * i for i in range(requests)]
    kp, vp, tables, prefix, ks, vs = family(lens, front, Hkv, D, page, dtype, seed=D, extra=1)
    for hole in (-1, -(1 << 31), kp.shape[0], (1 << 31) - 1):
        print(dtype, D, alpha, requests, "hole", hole, flush=True)
        holes, common = tables.clone(), prefix.clone()
        holes[:, :front:8] = hole
        common[::8] = hole
        keep = torch.ones(max(lens), dtype=torch.bool)
        for i in range(0, front, 8):
            keep[i * page:(i + 1) * page] = False
        cut = [[x[:, keep[: x.shape[1]]] for x in t] for t in (ks, vs)]
        lengths = torch.tensor(lens, device=DEV)
        assert is_shared(requests, Hq, Hkv, D, dtype, holes.shape[1] * page, page, front)
        for scale in (0.0, 0.003):
            q = (torch.randn(requests, Hq, 1, D, generator=torch.Generator().manual_seed(5)) * scale).to(dtype).to(DEV)
            got = A.paged_attention(q, kp, vp, holes, lengths, alpha=alpha, prefix_table=common)
            check_rows(got, q, *cut, alpha, f"scores * {scale}")
