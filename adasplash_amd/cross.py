"""Entmax attention of a decoder to an encoder's states, on gfx950: queries of one length, keys of another.

The reference serves ``q_len != k_len`` with its dense example path (``examples/attention.py:34-91``); ``adasplash_amd.dense`` is that path.
``cross_attention`` computes the same (without a causal mask and slopes, right padding) without a score matrix, with grouped K/V heads and lengths of
its own on either side, and has a gradient.
"""

from . import _attention, _lib


def cross_attention(q, k, v, alpha=1.5, varlen_q=None, varlen_k=None):
    """alpha-entmax attention of q ``(batch, n_heads, q_len, head_dim)`` to k, v ``(batch, n_kv_heads, k_len, head_dim)``.

    Contiguous tensors of one type (float32, bfloat16, float16), head_dim 16, 32, 64, 128 or 256, ``n_heads`` a multiple of ``n_kv_heads``; ``alpha``
    in (1, 2]; ``varlen_q``, ``varlen_k``: optional ``(batch,)`` int32/int64 valid lengths (right padding).  Output rows past ``varlen_q``, and
    those of an item without keys, are zeros, and so are their gradients; the padding may hold anything.  Returns a tensor like q.  A few queries
    (one new token of each sequence) take kernels that split the keys.  Where a gradient is wanted the forward keeps the rows' supports for it, as
    ``set_keep_supports`` says (some 0.8 KB a row of q in single precision and, in 16 bits, over many keys; "auto" keeps none beyond 256 MiB or twice the bytes of q, and the
    gradients then take up to three times as long); the lengths must not change before the backward.  A row with a score of +inf is zeros, and so are
    its gradients; a key whose score is -inf or NaN has no weight.
    """
    return _lib.native().cross_attention(q, k, v, alpha, varlen_q, varlen_k, _attention.keep_code())
