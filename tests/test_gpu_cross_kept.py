"""ADSP_SPARSE changed between a forward and its backward: what the forward kept is of no use to the other kernels, and the gradients are right without it."""

import os

import pytest
import torch

import adasplash_amd as A
from tests import op_reference as ref
from tests.test_gpu_cross import SUPPORTS, SUPPORTS_LENGTHS, inputs, reference

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("forward, backward", [(None, "0"), ("0", None)])
def test_gradients_of_other_kernels_than_the_forward(forward, backward, monkeypatch):
    def sparse(value):
        monkeypatch.delenv("ADSP_SPARSE", raising=False)
        if value is not None:
            monkeypatch.setenv("ADSP_SPARSE", value)

    q, k, v, do = inputs(*SUPPORTS, torch.bfloat16, q_scale=2.0)
    lq, lk = SUPPORTS_LENGTHS["lq"], SUPPORTS_LENGTHS["lk"]
    want = reference(q, k, v, do, 1.5, lq, lk, True)
    lens = {"varlen_q": torch.tensor(lq, device=DEV), "varlen_k": torch.tensor(lk, device=DEV)}
    ts = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
    before = A.set_keep_supports("always")
    try:
        sparse(forward)
        out = A.cross_attention(*ts, **lens)
        sparse(backward)
        grads = torch.autograd.grad(out, ts, do.to(DEV))
    finally:
        A.set_keep_supports(before)
    assert os.environ.get("ADSP_SPARSE") == backward
    for name, got, pair in zip(("out", "dq", "dk", "dv"), (out, *grads), want):
        ref.check(got, *pair, f"{name}, forward {forward}, backward {backward}")
