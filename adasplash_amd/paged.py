"""Entmax attention over a cache that lies in pages: what a decoding server keeps for its requests.

The cache is two tensors ``(pages, n_kv_heads, page_size, head_dim)``; the tokens of request ``b`` are, in order, the slots of the pages
``block_tables[b]``.  ``build_block_tables`` gives the new tokens of a step their pages and slots, ``write_pages`` puts their keys and values
there, ``paged_attention`` attends to them with one new query a request; ``fork_requests`` lets requests go on from others, or end, and ``compact_pages`` moves a cache's
pages into another pool.  ``PagedCache`` keeps the tensors and makes these calls.
Everything stays on the GPU and in the order of the current stream; nothing waits for the host.  No counterpart in the reference.
"""

import operator

import torch

from . import _lib


def paged_attention(q, k_pages, v_pages, block_tables, lengths, alpha=1.5, max_length=None, prefix_table=None):
    """alpha-entmax attention of one new token of every request against its tokens in the cache.

    q: ``(batch, n_heads, 1, head_dim)``, head_dim 32, 64, 128 or 256, ``n_heads`` a multiple of ``n_kv_heads`` (up to 64 times);
    k_pages, v_pages: ``(pages, n_kv_heads, page_size, head_dim)``, strides of any order along the first three dimensions (rows 16-byte
    aligned), of q's type; block_tables: ``(batch, max_blocks)`` int32, an entry outside the cache is a page without keys; lengths:
    ``(batch,)`` int32/int64 tokens of a request, the new one among them.  ``alpha`` in (1, 2].  ``max_length``: no request is longer (what
    lies behind it is not looked at); the scratch memory of a call is 8 bytes for each head, request and token up to it (default: what the tables
    can hold).  Returns a tensor like q; a request without keys gets zeros, and so does a row with a score of +inf; a key whose score is -inf or NaN
    has no weight.  No gradient.

    ``prefix_table``: 1-D int32, the pages that many of the requests have in front (a prompt that they all go on from).  Their keys are computed once for all requests whose tables start
    with them.  It says what is worth sharing and no more: where a request's table differs from it, or the request ends before, its own pages are attended to as without it.
    It pays where supports are small beside the prefix; where scores are so flat that thousands of keys have weight it gains little, and can take longer than a call without it.
    Give ``max_length`` with it where the tables have room far behind the requests: what lies behind the prefix is laid out for all of it (64 requests behind 8192 tokens, 51 us with tables or a ``max_length`` of
    8500, 168 with 32768 and 693 with 131072; without the prefix table 139, 139 and 184).
    """
    return _lib.native().paged_attention(q, k_pages, v_pages, block_tables, lengths, alpha, max_length, prefix_table)


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


def write_pages(k, v, slots, k_pages, v_pages, positions=None, rotary=None):
    """Write keys and values ``(tokens, n_kv_heads, head_dim)`` to their slots of a cache, in place.  A slot outside the cache (-1) is skipped; the
    others must differ from each other.  With ``rotary`` (an ``adasplash_amd.Rotary``; head_dim 16, 32, 64, 128 or 256) and ``positions``, ``(tokens,)`` int32/int64, the keys are
    normed and turned on the way."""
    if (rotary is None) != (positions is None):
        raise ValueError("positions and rotary go together.")
    if rotary is None:
        _lib.native().write_pages(k, v, slots, k_pages, v_pages)
    else:
        _lib.native().write_pages_rotary(k, v, slots, k_pages, v_pages, positions, *rotary._keys())


def fork_requests(parents, lengths, block_tables, free_pages, free_range, shares, k_pages, v_pages):
    """Requests go on from others, or end, in place: request ``b`` is behind the call what request ``parents[b]`` was before it.

    parents: ``(batch,)`` int32/int64; ``parents[b] = b`` leaves a request alone, a number outside the batch (-1) ends it: it has no tokens then and entries of -1.  Any number of requests may go on from one.
    lengths, block_tables, free_pages, free_range: as ``build_block_tables`` takes them; shares: ``(pages,)`` int32, the requests that hold a page, less one (0 for a free one).
    Whole pages are shared.  A last page that is filled in part stays with the request itself, or with the first that goes on from it, and the others copy its tokens into free pages, in the order of their
    numbers; where none is left a request has its whole pages only (``lengths`` says so).  Pages that no request holds any more are free again, behind the others, before pages are taken.
    (A free list with fewer entries than the cache has pages may have no room for one: such a page is in no list, and its ``shares`` are -1 until the caller makes it 0 and a page of a list or a table again.)
    (A page that is filled in part must be one request's alone, as it is where tables come from ``build_block_tables`` and from here, and no page may stand twice in one table.)
    """
    _lib.native().fork_requests(parents, lengths, block_tables, free_pages, free_range, shares, k_pages, v_pages)


def compact_pages(lengths, block_tables, k_pages, v_pages, k_to, v_to):
    """Copy the pages that requests hold into another pool, side by side in the order of the requests and their tables (a page of several where the first of them has it).

    k_to, v_to: ``(other_pages, n_kv_heads, page_size, head_dim)`` that share no memory with the cache; of them the pages that are taken are written.  Returns what goes with them in new tensors,
    ``(lengths, block_tables, shares, free_pages, free_range)``.  Entries outside the cache become -1.  Where the pool has too few pages, requests end in front of the first that found none.
    """
    return _lib.native().compact_pages(lengths, block_tables, k_pages, v_pages, k_to, v_to)


class PagedCache:
    """Keys and values of ``batch`` requests in ``pages`` pages of ``page_size`` slots, and where each request's tokens are; a request's table has
    room for ``max_length`` tokens, in whole pages.

    ``append`` adds tokens to the requests, ``attend`` attends to them with one query a request, ``fork`` lets requests go on from others, ``release`` gives a request's pages back,
    ``resize`` moves the cache into another number of pages.  With ``rotary`` (an ``adasplash_amd.Rotary``) keys are normed and turned by their places in their requests on the way into the
    pages, and queries by those of the requests' last tokens.
    ``k_pages``, ``v_pages``, ``block_tables``, ``lengths``, ``free_pages``, ``free_range`` and ``shares`` are tensors on the device, which the calls but ``resize`` change in place: they
    can be captured into a graph, and each replay goes on from what the last one, or a call without the graph, left.
    """

    def __init__(self, pages, page_size, batch, n_kv_heads, head_dim, max_length, dtype=torch.bfloat16, device="cuda", rotary=None):
        if min(pages, page_size, batch, n_kv_heads, max_length) < 1:
            raise ValueError("pages, page_size, batch, n_kv_heads and max_length must be positive.")
        self.page_size = page_size
        self.rotary = rotary
        shape = (pages, n_kv_heads, page_size, head_dim)
        self.k_pages = torch.zeros(shape, dtype=dtype, device=device)
        self.v_pages = torch.zeros(shape, dtype=dtype, device=device)
        self.block_tables = torch.full((batch, -(-max_length // page_size)), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self.free_pages = torch.arange(pages, dtype=torch.int32, device=device)
        self.free_range = torch.tensor([0, pages], dtype=torch.int64, device=device)
        self.shares = torch.zeros(pages, dtype=torch.int32, device=device)

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
        call = (k, v, self.lengths, new_tokens, self.block_tables, self.free_pages, self.free_range, self.page_size, self.k_pages, self.v_pages)
        if self.rotary is not None:
            return _lib.native().append_rotary(*call, *self.rotary._keys())
        return _lib.native().append(*call)

    def attend(self, q, alpha=1.5, max_length=None, prefix_table=None):
        """Entmax attention of q ``(batch, n_heads, 1, head_dim)`` to the requests' tokens; ``prefix_table`` as in ``paged_attention``: pages that many requests have in front,
        ``block_tables[b, :n]`` of one of them (with a ``max_length`` where the cache's own is far behind the requests' lengths)."""
        if self.rotary is not None:
            q, _ = self.rotary(q, None, (self.lengths - 1)[:, None])
        return paged_attention(q, self.k_pages, self.v_pages, self.block_tables, self.lengths, alpha=alpha, max_length=max_length, prefix_table=prefix_table)

    def fork(self, parents):
        """Requests go on from others, or end (``fork_requests``): parents ``(batch,)`` on the device.  ``[0, 0, 0]`` makes three samples of the first request; the step of a
        beam search takes the beams that its hypotheses come from."""
        fork_requests(parents, self.lengths, self.block_tables, self.free_pages, self.free_range, self.shares, self.k_pages, self.v_pages)

    def release(self, request):
        """Give the pages of request number ``request`` back and empty it; of those of a list of numbers, or of an int32/int64 tensor of them (numbers outside the batch are no requests;
        a call that is captured takes one on the device)."""
        parents = torch.arange(self.lengths.shape[0], device=self.lengths.device)
        if isinstance(request, torch.Tensor):
            if request.dtype not in (torch.int32, torch.int64):
                raise TypeError(f"requests must be int32/int64 numbers; got {request.dtype}.")
            parents = parents.masked_fill((parents[:, None] == request.reshape(1, -1).to(parents.device)).any(1), -1)
        else:
            for r in request if isinstance(request, (list, tuple)) else [request]:
                parents[operator.index(r)].fill_(-1)
        self.fork(parents)

    def resize(self, pages):
        """Move the requests into a cache of ``pages`` pages, side by side: the cache's tensors are new ones then, and graphs that hold the old ones are of no use to it.  Both exist for the
        time of the copy.  Where ``pages`` is too few for what the requests hold they are cut off (``lengths`` says so)."""
        if pages < 1:
            raise ValueError("pages must be positive.")
        shape = (pages, *self.k_pages.shape[1:])
        k_to, v_to = (torch.zeros(shape, dtype=t.dtype, device=t.device) for t in (self.k_pages, self.v_pages))
        self.lengths, self.block_tables, self.shares, self.free_pages, self.free_range = compact_pages(
            self.lengths, self.block_tables, self.k_pages, self.v_pages, k_to, v_to)
        self.k_pages, self.v_pages = k_to, v_to
