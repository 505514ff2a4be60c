"""Heads normed and turned by positions in 64 bits, their gradients, and how far a kernel that works in fp32 may be from them."""

import math

import torch

from tests.op_reference import half_step, least_half_step

F32 = half_step(torch.float32)


def frequencies_of(rot, base=10000.0):
    return torch.tensor([base ** (-2.0 * i / rot) for i in range(rot // 2)], dtype=torch.float64) if rot else torch.zeros(0, dtype=torch.float64)


def pair_index(rot, layout):
    i = torch.arange(rot // 2)
    return (i, i + rot // 2) if layout == "half" else (2 * i, 2 * i + 1)


def normed(x, weight, eps):
    """x / sqrt(mean x^2 + eps), the size of the root, and the product with the weight."""
    x = x.double()
    if weight is None:
        return x, torch.ones_like(x[..., :1]), x
    size = (x.square().mean(-1, keepdim=True) + eps).sqrt()
    return x / size, size, x / size * weight.double()


def turned(n, positions, frequencies, layout, factor, back=False):
    """n (..., D) turned by positions that broadcast against its leading dimensions."""
    a, b = pair_index(2 * frequencies.numel(), layout)
    angle = positions.double()[..., None] * frequencies
    c, s = angle.cos() * factor, angle.sin() * factor * (-1.0 if back else 1.0)
    y = n.clone()
    y[..., a], y[..., b] = n[..., a] * c - n[..., b] * s, n[..., b] * c + n[..., a] * s
    return y


def forward(x, positions, frequencies, layout="half", weight=None, eps=1e-6, factor=1.0):
    return turned(normed(x, weight, eps)[2], positions, frequencies, layout, factor)


def _sizes(n, positions, frequencies, layout, factor, steps):
    """Bound of fp32's errors in a turned element: `steps` roundings of the pair's elements, and that of the angle in 64 bits."""
    a, b = pair_index(2 * frequencies.numel(), layout)
    size = n.abs()
    err = steps * F32 * size
    angle = (positions.double()[..., None] * frequencies).abs()
    both = (size[..., a] + size[..., b]) * abs(factor)
    pair = both * (steps * F32 + 4 * 2.0 ** -53 * angle)
    err[..., a], err[..., b] = pair, pair
    size[..., a], size[..., b] = both, both
    return err, size


def forward_tolerance(x, positions, frequencies, layout="half", weight=None, eps=1e-6, factor=1.0):
    """The sum of D squares, eight of a lane and five joins, has 13 half steps, of which the root takes half; the root itself 2, two products 2; an angle's cosine 5 (the rest of the
    angle, its series, the factor); products and sum 2: fewer than 20 of the pair's size.  And the rounding to the element type."""
    want = forward(x, positions, frequencies, layout, weight, eps, factor)
    err, _ = _sizes(normed(x, weight, eps)[2], positions, frequencies, layout, factor, 20)
    return want, err + half_step(x.dtype) * (want.abs() + err) + least_half_step(x.dtype)


def backward(x, dy, positions, frequencies, layout="half", weight=None, eps=1e-6, factor=1.0):
    """(dx, tolerance), (dw, tolerance) or None.

    dn = dy turned back; dw = sum over rows of dn xn; dx = (w dn - xn mean(w dn xn)) / size.  Fewer than 24 half steps in each term; the sum over rows four times the root of their number."""
    xn, size, _ = normed(x, weight, eps)
    dn = turned(dy.double(), positions, frequencies, layout, factor, back=True)
    err, _ = _sizes(dy.double(), positions, frequencies, layout, factor, 24)
    least = least_half_step(x.dtype)
    if weight is None:
        return (dn, err + half_step(x.dtype) * (dn.abs() + err) + least), None
    w = weight.double()
    rows = tuple(range(x.dim() - 1))
    n = math.prod(x.shape[:-1])
    dw = (dn * xn).sum(rows)
    dw_err = ((err + 24 * F32 * dn.abs()) * xn.abs()).sum(rows) + 4 * math.sqrt(max(n, 1)) * F32 * (dn * xn).abs().sum(rows)
    g = dn * w
    dx = (g - xn * (g * xn).mean(-1, keepdim=True)) / size
    g_err = (err + 24 * F32 * dn.abs()) * w.abs()
    dx_err = (g_err + xn.abs() * ((g_err + 24 * F32 * g.abs()) * xn.abs()).mean(-1, keepdim=True)) / size
    return ((dx, dx_err + half_step(x.dtype) * (dx.abs() + dx_err) + least),
            (dw, dw_err + half_step(weight.dtype) * (dw.abs() + dw_err) + least_half_step(weight.dtype)))
