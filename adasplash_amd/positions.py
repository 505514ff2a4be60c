"""Positions for queries and keys, on gfx950: each head's pairs of elements are turned by its token's position, and normed before that where asked for.

The attention of this package has no positions of its own but the dense path's slopes; a model whose scores go by the distance of two tokens turns its heads.  One
pass reads the heads as a projection left them (any strides with unit stride along the head) and writes them as the attention takes them.  No counterpart in the reference.
"""

import math

import torch

from . import _lib

_LAYOUTS = {"half": True, "interleaved": False}


def _half(layout):
    if layout not in _LAYOUTS:
        raise ValueError(f'layout must be "half" or "interleaved"; got {layout!r}.')
    return _LAYOUTS[layout]


def rotary_frequencies(rotary_dim, base=10000.0, stretch=1.0, trained_length=None, slow=1.0, fast=32.0, device="cuda"):
    """Frequencies ``base ** (-2 i / rotary_dim)``, in radians a position, as a float64 tensor of ``rotary_dim / 2``, and the factor that goes with them.

    ``stretch`` > 1 takes the positions of a context that many times as long as the model was trained on: without ``trained_length`` all frequencies are divided by it (factor 1).  With the
    length of the training's contexts, pairs that make ``fast`` turns or more in it keep their frequencies, those with ``slow`` turns or fewer have theirs divided, and those between are
    blended; the factor is then ``0.1 log(stretch) + 1`` (Peng et al., "YaRN", 2023).
    """
    if rotary_dim <= 0 or rotary_dim % 8:
        raise ValueError(f"rotary_dim must be a positive multiple of 8; got {rotary_dim}.")
    if not base > 0.0 or not stretch >= 1.0 or not math.isfinite(base) or not math.isfinite(stretch):
        raise ValueError(f"base must be positive and stretch at least 1; got {base} and {stretch}.")
    frequencies = torch.tensor([base ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)], dtype=torch.float64)
    if trained_length is None or stretch == 1.0:
        return (frequencies / stretch).to(device), 1.0
    if not trained_length > 0 or not 0.0 < slow < fast:
        raise ValueError(f"trained_length must be positive and slow below fast; got {trained_length}, {slow} and {fast}.")
    turns = trained_length * frequencies / (2.0 * math.pi)
    keep = ((turns - slow) / (fast - slow)).clamp(0.0, 1.0)
    return (frequencies * keep + frequencies / stretch * (1.0 - keep)).to(device), 0.1 * math.log(stretch) + 1.0


def rotary(q, k, positions, frequencies, layout="half", q_weight=None, k_weight=None, eps=1e-6, factor=1.0):
    """Queries and keys turned by their positions: returns ``(q, k)``, contiguous tensors of the inputs' shapes and type.

    q: ``(batch, n_heads, length, head_dim)`` or ``(tokens, n_heads, head_dim)`` with head_dim 16, 32, 64, 128 or 256; k: the same with its own number of heads, or None (then None
    comes back); views are read in place where their rows lie on 16 bytes.  positions: int32/int64, ``(length,)`` or ``(batch, length)``, ``(tokens,)`` of three dimensions.
    frequencies: float64, half as many as elements are turned (a multiple of 8 elements, the first of the head; the others stay as they are); angles are formed in 64 bits.
    layout: "half" turns elements i and i + rotary_dim / 2 against each other, "interleaved" 2 i and 2 i + 1.  With ``q_weight`` (``k_weight``), ``(head_dim,)`` of
    the heads' type or float32, the heads are divided by their root mean square (``eps`` is added to the mean) and multiplied with it first.  ``factor`` multiplies what is turned.
    Differentiable in q, k and the weights, once; an output whose rows and weight want no gradient wants none.
    """
    return _lib.native().rotary(q, k, positions, frequencies, _half(layout), eps, factor, q_weight, k_weight)


class Rotary:
    """``rotary`` with its frequencies, layout and weights: ``q, k = turn(q, k, positions)``.  A ``PagedCache`` that is given one turns the keys on their way into its pages."""

    def __init__(self, frequencies, layout="half", q_weight=None, k_weight=None, eps=1e-6, factor=1.0):
        _half(layout)
        self.frequencies, self.layout, self.q_weight, self.k_weight, self.eps, self.factor = frequencies, layout, q_weight, k_weight, eps, factor

    def __call__(self, q, k, positions):
        return rotary(q, k, positions, self.frequencies, self.layout, self.q_weight, self.k_weight if k is not None else None, self.eps, self.factor)

    def _keys(self):
        return self.frequencies, _half(self.layout), self.eps, self.factor, self.k_weight
