"""How exact dQ of short 16-bit training steps is: its weights are multiplied as two 16-bit values each, so the result's own rounding is all that is left, as in the attention
of a sequence to itself.

A rounding's error is spread evenly over a step, so its size over many values is the step over sqrt(12): eps 2^e / sqrt(12) for a value of [2^e, 2^(e + 1)), at most
eps / sqrt(12) of the value (2.26e-3 in bf16, 2.8e-4 in f16).  One more rounding, of the weights, makes sqrt(2) times that of the mean value's (2.4e-3 and 3.0e-4 where 1.7e-3 and 2.1e-4 are left without).
"""

import math

import pytest
import torch

import adasplash_amd as A
from oracle import exact
from tests.test_gpu_cross import inputs

pytestmark = pytest.mark.gpu
DEV = "cuda"


def relative(got, want):
    return ((got.double().cpu() - want).norm() / want.norm()).item()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("alpha", [1.333, 1.5, 2.0])
@pytest.mark.parametrize("shape", [(2, 4, 4, 130, 500, 64), (2, 4, 4, 130, 500, 128), (16, 16, 16, 140, 300, 64), (8, 32, 32, 160, 200, 64), (2, 4, 4, 200, 1900, 64), (2, 4, 4, 150, 60, 128), (2, 4, 4, 100, 600, 128)])
def test_dq_is_as_exact_as_its_type(shape, alpha, dtype):
    print(shape, alpha, dtype, flush=True)
    for spread, size in ((1.0, 1.0), (0.05, 1.0), (1.0, 1e-3)):
        q, k, v, do = inputs(*shape, dtype, q_scale=spread)
        do = (do.float() * size).to(dtype)
        ts = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
        out = A.cross_attention(*ts, alpha=alpha)
        dq, = torch.autograd.grad(out, ts[:1], do.to(DEV))
        items = [0, shape[0] - 1]
        parts = []
        for b in items:
            qd, kd, vd, dd = (t[b].double() for t in (q, k, v, do))
            x = qd @ kd.transpose(-1, -2) / math.sqrt(shape[5])
            p, tau = exact.entmax_rows(x, alpha, return_tau=True)
            w = (x * (alpha - 1.0) - tau[..., None]).clamp(min=0.0)
            u = torch.where(w > 0, w.pow((2.0 - alpha) / (alpha - 1.0)), torch.zeros_like(w))
            dp = dd @ vd.transpose(-1, -2)
            dx = u * (dp - (u * dp).sum(-1, keepdim=True) / u.sum(-1, keepdim=True))
            parts.append(dx @ kd / math.sqrt(shape[5]))
        got = relative(dq[items], torch.stack(parts))
        # (f16 of 1e-3: its numbers below 2^-14 lie 2^-24 apart, a step whatever the value)
        least = 2.0 ** -24 / math.sqrt(12.0) * math.sqrt(sum(t.numel() for t in parts)) / torch.stack(parts).norm().item() if dtype == torch.float16 else 0.0
        assert got <= torch.finfo(dtype).eps / math.sqrt(12.0) * 0.95 + least, (spread, size, got)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_dv_and_dk_on_the_supports(dtype):
    """Large enough for the kernels on the supports.  p and dX are rounded once on their way into the products, the results once: two errors of sums over many rows, which add as their
    squares do.  Each is formed here from the exact values; a fiftieth is left for the scores and for what the lists hold."""
    shape = (2, 16, 4, 1030, 4000, 64)
    B, Hq, Hkv, Nq, Nk, D = shape
    q, k, v, do = inputs(*shape, dtype)
    ts = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
    out = A.cross_attention(*ts)
    _, dk, dv = torch.autograd.grad(out, ts, do.to(DEV))
    G, b, h = Hq // Hkv, 1, 2
    qd, dd = (t[b, h * G:(h + 1) * G].double().reshape(G * Nq, D) for t in (q, do))
    kd, vd = k[b, h].double(), v[b, h].double()
    p, tau = exact.entmax_rows(qd @ kd.T / math.sqrt(D), 1.5, return_tau=True)
    u = p.sqrt()
    dp = dd @ vd.T
    dx = u * (dp - (u * dp).sum(-1, keepdim=True) / u.sum(-1, keepdim=True))
    rounding = lambda t: relative(t.to(dtype).double(), t)  # noqa: E731
    for name, got, weights, with_, scale in (("dk", dk, dx, qd, 1 / math.sqrt(D)), ("dv", dv, p, dd, 1.0)):
        want = weights.T @ with_ * scale
        bound = 1.02 * math.hypot(rounding(want), rounding(weights))
        assert relative(got[b, h], want) <= bound, (name, relative(got[b, h], want), bound)
