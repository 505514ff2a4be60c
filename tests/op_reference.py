"""Entmax attention of any queries against any keys in 64 bits, and how far a kernel may be from it."""

import math

import torch

from oracle import exact


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def least_half_step(dtype):
    """f16's numbers below 2^-14 lie 2^-24 apart; the other types' are as fine as theirs are anywhere near here."""
    return 2.0 ** -25 if dtype == torch.float16 else 0.0


def _row_errors(q, k, alpha):
    """How far score and threshold may each be off in z = (alpha - 1) q k / sqrt(D), per row.

    The kernels work in fp32: a score of D products and sums has roundings of either sign, about sqrt(D) half steps of its terms' size in all; four times
    that is allowed.  The threshold is solved to 2e-6 in the weights' sum."""
    D = q.shape[-1]
    size = (q.abs() @ k.abs().T).amax(-1, keepdim=True) * (alpha - 1.0) / math.sqrt(D)
    return 4 * math.sqrt(D) * half_step(torch.float32) * size + 2e-6


def attend(q, k, v, alpha, roundings=1):
    """q (m, D), k and v (n, D) on the CPU, any type: the exact output and the tolerance of every element of it.

    Rounded to its type the output is off by at most half a step of its size.  Threshold and score each move u by what ``_row_errors`` says, a weight u^c0
    moves c0 u^(c0 - 1) times as far, and the output by at most the sum of that times the largest value.  In 16 bits the weights' own roundings add up to
    half a step of the sum of |p v| each: ``roundings`` is 1 for a product on rounded weights, 2 where the threshold is moreover only solved to below the weights'
    rounding (the kernels that walk all pairs).
    """
    m, n = q.shape[0], k.shape[0]
    if n == 0:
        return torch.zeros(m, v.shape[1], dtype=torch.float64), torch.zeros(m, v.shape[1], dtype=torch.float64)
    qd, kd, vd = q.double(), k.double(), v.double()
    x = qd @ kd.T / math.sqrt(q.shape[1])
    p, tau = exact.entmax_rows(x, alpha, return_tau=True)
    out = p @ vd
    dz = _row_errors(qd, kd, alpha)
    c0 = 1.0 / (alpha - 1.0)
    u = torch.clamp(x * (alpha - 1.0) - tau[..., None], min=0.0)
    moved = torch.where(u > 0, u.pow(c0 - 1.0), torch.zeros_like(u)).sum(-1, keepdim=True) + 1.0
    tol = 2 * c0 * dz * moved * vd.abs().max()
    if q.dtype != torch.float32:
        least = least_half_step(q.dtype)
        tol = tol + half_step(q.dtype) * (out.abs() + roundings * (p @ vd.abs())) + least * (1 + ((p > 0).double() @ vd.abs()))
    else:
        tol = tol + 4 * math.sqrt(n) * half_step(torch.float32) * (p @ vd.abs())
    return out, tol


def gradients(q, k, v, do, alpha):
    """Exact dq, dk, dv of ``attend`` for the upstream gradient `do`, and their tolerances.

    dX = u (dP - delta) with u = p^(2 - alpha), dq = dX k / sqrt(D), dk = dX^T q / sqrt(D), dv = p^T do.  Score and threshold move z - tau by up to
    2 dz, u = (z - tau)^e with e = (2 - alpha) / (alpha - 1) by e (z - tau + 2 dz)^(e - 1) times that, or for e <= 1 by at most (2 dz)^e (|a^e - b^e| <= |a - b|^e;
    with alpha = 2 a key at the border comes or goes: 1 there, 0 elsewhere); delta, a mean weighted with u, by the means of the changes; dP by fp32's roundings.  In 16 bits
    p and dX are rounded once each, the threshold's error (below a weight's rounding) makes another half step of p and of u's change with it, and the results are
    rounded (that rounding is of the value with its errors).  A sum of n terms in fp32 adds four times sqrt(n) half steps of their size.
    """
    D, n, m = q.shape[1], k.shape[0], q.shape[0]
    qd, kd, vd, dod = (t.double() for t in (q, k, v, do))
    if n == 0 or m == 0:
        return [(torch.zeros_like(t), torch.zeros_like(t)) for t in (qd, kd, vd)]
    scale = 1.0 / math.sqrt(D)
    x = qd @ kd.T * scale
    p, tau = exact.entmax_rows(x, alpha, return_tau=True)
    w = torch.clamp(x * (alpha - 1.0) - tau[..., None], min=0.0)
    near = x * (alpha - 1.0) - tau[..., None]
    e, c0 = (2.0 - alpha) / (alpha - 1.0), 1.0 / (alpha - 1.0)
    u = torch.where(w > 0, w.pow(e), torch.zeros_like(w))
    dp = dod @ vd.T
    usum = u.sum(-1, keepdim=True).clamp(min=1e-300)
    delta = (u * dp).sum(-1, keepdim=True) / usum
    dx = u * (dp - delta)
    dz = 2 * _row_errors(qd, kd, alpha)
    low = q.dtype != torch.float32
    hs, f32 = half_step(q.dtype), half_step(torch.float32)
    touched = near > -dz
    least = least_half_step(q.dtype)
    if e == 0.0:
        du = (near.abs() <= dz).double()
    elif e < 1.0:
        du = torch.where(touched, torch.minimum(dz.pow(e), e * torch.clamp(w - dz, min=1e-12).pow(e - 1.0) * dz), torch.zeros_like(w))
    else:
        du = torch.where(touched, e * (w + dz).pow(e - 1.0) * dz, torch.zeros_like(w))
    dp_err = 4 * math.sqrt(D) * f32 * (dod.abs() @ vd.abs().T)
    if low:
        du = du + hs * u
    delta_err = ((du * (dp - delta).abs()).sum(-1, keepdim=True) + (u * dp_err).sum(-1, keepdim=True)) / usum
    dx_err = du * (dp - delta).abs() + (u + du) * (dp_err + delta_err) + (hs * dx.abs() if low else 4 * f32 * dx.abs())
    p_err = torch.where(touched, c0 * (w + dz).pow(c0 - 1.0) * dz, torch.zeros_like(w)) + (2 * hs * p if low else 8 * f32 * p) + 4e-6 * p
    dx_err, p_err = (x + least * touched for x in (dx_err, p_err))
    out = []
    for want, err, size, terms in (
        (dx @ kd * scale, dx_err @ kd.abs() * scale, dx.abs() @ kd.abs() * scale, n),
        (dx.T @ qd * scale, dx_err.T @ qd.abs() * scale, dx.abs().T @ qd.abs() * scale, m),
        (p.T @ dod, p_err.T @ dod.abs(), p.T @ dod.abs(), m),
    ):
        err = err + 4 * math.sqrt(terms) * f32 * size
        out.append((want, err + (hs if low else 2 * f32) * (want.abs() + err) + least + 1e-12))
    return out


def check(got, want, tol, what):
    assert torch.isfinite(got.double()).all(), f"{what}: not finite"
    err = (got.detach().double().cpu() - want).abs()
    worst = (err - tol).max().item() if err.numel() else -1.0
    assert worst <= 0, f"{what}: off by {err.max().item():.3e}, {worst:.3e} more than allowed"
