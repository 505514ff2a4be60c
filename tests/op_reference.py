"""Entmax attention of any queries against any keys in 64 bits, and how far a kernel may be from it."""

import math

import torch

from oracle import exact


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def attend(q, k, v, alpha):
    """q (m, D), k and v (n, D) on the CPU, any type: the exact output and the tolerance of every element of it.

    Rounded to its type the output is off by at most half a step of its size.  Before that the kernels work in fp32: a score of D products and
    sums has roundings of either sign, about sqrt(D) half steps of its terms' size in all; four times that is allowed.  Threshold and score each
    move u by that much and the threshold is solved to 2e-6 in the weights' sum, a weight u^c0 moves c0 u^(c0 - 1) times as far, and the output by
    at most the sum of that times the largest value.  In 16 bits a weight is moreover rounded once (half a step of it) where the products run on matrix tiles,
    so that the weights' roundings add up to half a step of the sum of |p v|.
    """
    m, D = q.shape
    if k.shape[0] == 0:
        return torch.zeros(m, v.shape[1], dtype=torch.float64), torch.zeros(m, v.shape[1], dtype=torch.float64)
    qd, kd, vd = q.double(), k.double(), v.double()
    x = qd @ kd.T / math.sqrt(D)
    p, tau = exact.entmax_rows(x, alpha, return_tau=True)
    out = p @ vd
    size = (qd.abs() @ kd.abs().T).amax(-1, keepdim=True) * (alpha - 1.0) / math.sqrt(D)
    dz = 4 * math.sqrt(D) * half_step(torch.float32) * size + 2e-6
    c0 = 1.0 / (alpha - 1.0)
    u = torch.clamp(x * (alpha - 1.0) - tau[..., None], min=0.0)
    moved = torch.where(u > 0, u.pow(c0 - 1.0), torch.zeros_like(u)).sum(-1, keepdim=True) + 1.0
    tol = 2 * c0 * dz * moved * vd.abs().max()
    if q.dtype != torch.float32:
        tol = tol + half_step(q.dtype) * (out.abs() + p @ vd.abs())
    else:
        tol = tol + 4 * math.sqrt(k.shape[0]) * half_step(torch.float32) * (p @ vd.abs())
    return out, tol


def check(got, want, tol, what):
    err = (got.detach().double().cpu() - want).abs()
    assert torch.isfinite(got.double()).all(), f"{what}: not finite"
    worst = (err - tol).max().item() if err.numel() else -1.0
    assert worst <= 0, f"{what}: off by {err.max().item():.3e}, {worst:.3e} more than allowed"
