"""Entmax attention over a cache that lies in pages: what a decoding server keeps for its requests.

The cache is two tensors ``(pages, n_kv_heads, page_size, head_dim)``; the tokens of request ``b`` are, in order, the slots of the pages
``block_tables[b]``.  ``build_block_tables`` gives the new tokens of a step their pages and slots, ``write_pages`` puts their keys and values
there, ``paged_attention`` attends to them with one new query a request; ``PagedCache`` keeps the tensors and makes the three calls.
Everything stays on the GPU and in the order of the current stream; nothing waits for the host.  No counterpart in the reference.
"""

import torch

from . import _lib


def paged_attention(q, k_pages, v_pages, block_tables, lengths, alpha=1.5, max_length=None):
    """alpha-entmax attention of one new token of every request against its tokens in the cache.

    q: ``(batch, n_heads, 1, head_dim)``, head_dim 32, 64, 128 or 256, ``n_heads`` a multiple of ``n_kv_heads`` (up to 64 times);
    k_pages, v_pages: ``(pages, n_kv_heads, page_size, head_dim)``, strides of any order along the first three dimensions (rows 16-byte
    aligned), of q's type; block_tables: ``(batch, max_blocks)`` int32, an entry outside the cache is a page without keys; lengths:
    ``(batch,)`` int32/int64 tokens of a request, the new one among them.  ``alpha`` in (1, 2].  ``max_length``: no request is longer (what
    lies behind it is not looked at); the scratch memory of a call is 8 bytes for each head, request and token up to it (default: what the tables
    can hold).  Returns a tensor like q; a request without keys gets zeros, and so does a row with a score of +inf; a key whose score is -inf or NaN
    has no weight.  No gradient.
    """
    return _lib.native().paged_attention(q, k_pages, v_pages, block_tables, lengths, alpha, max_length)


def build_block_tables(lengths, new_tokens, block_tables, free_pages, free_range, page_size, total_tokens):
    """The pages and slots that the new tokens of a step take.

    lengths, new_tokens: ``(batch,)`` int32/int64 tokens that a request has and gets (batch up to 8192); block_tables: ``(batch, max_blocks)`` int32,
    written in place where a request gets a page; free_pages: 1-D int32 ring of page numbers, of which the entries ``free_range[0]`` to
    ``free_range[1] - 1`` (modulo its length; two int64 on the GPU) are free; ``total_tokens``: the sum of ``new_tokens``, or more.

    Returns ``(slots, lengths, free_range)``: ``(total_tokens,)`` int64 slots (page times page_size plus place), the new tokens request behind
    request, -1 for a token that got no page and behind the last one; the tokens of a request that its pages hold; and what is free then.  Pages are
    handed out in the order of the requests; where they run out, the returned lengths fall short of ``lengths + new_tokens``.  (With a smaller
    ``total_tokens`` all of ``new_tokens`` have pages and count all the same; only the slots behind it are not told.)
    """
    return _lib.native().build_block_tables(lengths, new_tokens, block_tables, free_pages, free_range, page_size, total_tokens)


def write_pages(k, v, slots, k_pages, v_pages):
    """Write keys and values ``(tokens, n_kv_heads, head_dim)`` to their slots of a cache, in place.  A slot outside the cache (-1) is skipped; the
    others must differ from each other."""
    _lib.native().write_pages(k, v, slots, k_pages, v_pages)


class PagedCache:
    """Keys and values of ``batch`` requests in ``pages`` pages of ``page_size`` slots, and where each request's tokens are; a request's table has
    room for ``max_length`` tokens, in whole pages.

    ``append`` adds tokens to the requests, ``attend`` attends to them with one query a request, ``release`` gives a request's pages back.
    ``k_pages``, ``v_pages``, ``block_tables``, ``lengths``, ``free_pages`` and ``free_range`` are tensors on the device, which the calls change in place: ``append`` and
    ``attend`` can be captured into a graph, and each replay goes on from what the last one, or a call without the graph, left.
    """

    def __init__(self, pages, page_size, batch, n_kv_heads, head_dim, max_length, dtype=torch.bfloat16, device="cuda"):
        if min(pages, page_size, batch, n_kv_heads, max_length) < 1:
            raise ValueError("pages, page_size, batch, n_kv_heads and max_length must be positive.")
        self.page_size = page_size
        shape = (pages, n_kv_heads, page_size, head_dim)
        self.k_pages = torch.zeros(shape, dtype=dtype, device=device)
        self.v_pages = torch.zeros(shape, dtype=dtype, device=device)
        self.block_tables = torch.full((batch, -(-max_length // page_size)), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self.free_pages = torch.arange(pages, dtype=torch.int32, device=device)
        self.free_range = torch.tensor([0, pages], dtype=torch.int64, device=device)

    def append(self, k, v, new_tokens=None):
        """Add tokens: k, v ``(tokens, n_kv_heads, head_dim)``, request behind request, ``new_tokens`` ``(batch,)`` of each; without it one of each
        request, then ``(batch, n_kv_heads, 1, head_dim)`` is taken too.  Tokens for which no page is free are left out, and so are those of ``new_tokens``
        that k and v do not hold (``lengths`` says so).  A call that is refused changes nothing.  Returns the tokens' slots."""
        batch = self.lengths.shape[0]
        if new_tokens is None:
            if k.dim() == 4 and k.shape[2] == 1 and v.dim() == 4 and v.shape[2] == 1:
                k, v = k[:, :, 0], v[:, :, 0]
            if k.shape[0] != batch:
                raise ValueError(f"without new_tokens k and v hold one token of each of the {batch} requests; got {k.shape[0]}.")
            new_tokens = torch.ones_like(self.lengths)
        return _lib.native().append(
            k, v, self.lengths, new_tokens, self.block_tables, self.free_pages, self.free_range, self.page_size, self.k_pages, self.v_pages)

    def attend(self, q, alpha=1.5, max_length=None):
        """Entmax attention of q ``(batch, n_heads, 1, head_dim)`` to the requests' tokens."""
        return paged_attention(q, self.k_pages, self.v_pages, self.block_tables, self.lengths, alpha=alpha, max_length=max_length)

    def release(self, request):
        """Give the pages of request number ``request`` back and empty it (waits for the GPU: their number is read)."""
        used = -(-int(self.lengths[request]) // self.page_size)
        end = int(self.free_range[1])
        at = (torch.arange(used, device=self.free_pages.device) + end) % self.free_pages.numel()
        self.free_pages[at] = self.block_tables[request, :used]
        self.free_range[1] += used
        self.block_tables[request] = -1
        self.lengths[request] = 0
