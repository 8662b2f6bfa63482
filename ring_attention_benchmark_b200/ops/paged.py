"""A paged key/value cache and the attention over it (sm_100a).

A pool holds pages of tokens: ``k_pages`` and ``v_pages`` are
``[pages, heads_kv, page_size, dim]`` (bf16, fp16 or fp32); ``copy_pages`` and
``compact_path`` also take a leading layer dimension and then move every layer in
one launch.  ``block_table[b, i]`` (int32) names the page that holds tokens
``i * page_size ...`` of request b, ``context_lens[b]`` (int32) the tokens cached
before the call.  The call's own tokens are packed, ``[tokens, heads, dim]``, with
the requests' borders in ``cu_q`` (int32, one more entry than requests); without
``cu_q`` every request has the same number.  Token i of request b lies at place
``context_lens[b] + i`` of its request.  Rows behind the last border are neither
read nor written.

What device tensors hold cannot be refused without waiting for the GPU.  A page
id outside the pool, a place outside the table or a path that is not increasing
is not written to, and reported in ``status`` (int32[8], see `new_status` and
`check_status` in `ops.attention`) when one is given; attention reads a page outside
the pool as zeros, whose keys score 0 and take weight.  Other requests of the call
are unaffected.  The word keeps its first report; later calls may be given it.

All calls run on the current stream of the tensors' GPU, keep nothing from one
call to the next, and can be captured into CUDA graphs.  None has a gradient.  What
they write counts as changed in place, and must not overlap what they read; ``q_out``
may be ``q``, and ``out`` the queries.  New tokens must not be slices of the pages
that a call writes.
"""
from __future__ import annotations

from typing import Optional, Sequence, Tuple, Union

import torch

from .._ext import load


def append_kv(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
              block_table: torch.Tensor, context_lens: torch.Tensor,
              cu_q: Optional[torch.Tensor] = None, *, positions: Optional[torch.Tensor] = None,
              inv_freq: Optional[torch.Tensor] = None, interleaved: bool = False,
              scale: float = 1.0, q: Optional[torch.Tensor] = None,
              q_out: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None):
    """Write new tokens' ``k`` and ``v`` (``[tokens, heads_kv, dim]``) into the pages.

    With ``inv_freq`` K is rotated on the way (see `ops.rotary`), at ``positions``
    or, without them, at the token's place in the cache; a drafted tree passes
    ``context + depth``.  ``q`` is rotated in the same launch and returned
    (``q_out`` takes the result; else a new tensor).
    """
    return load().append_kv(k, v, k_pages, v_pages, block_table, context_lens, cu_q, positions,
                            inv_freq, interleaved, scale, q, q_out, status)


def _indices(x) -> torch.Tensor:
    return x if isinstance(x, torch.Tensor) else torch.as_tensor(list(x), dtype=torch.int64)


def copy_pages(k_pages: torch.Tensor, v_pages: torch.Tensor,
               src: Union[Sequence[int], torch.Tensor],
               dst: Union[Sequence[int], torch.Tensor]) -> None:
    """Copy page ``src[i]`` to page ``dst[i]`` for every i, K and V of every layer.

    The lists are the scheduler's and live on the host; they are checked before
    anything is copied: a page may be read many times, but is written at most
    once and never both read and written.
    """
    load().copy_pages(k_pages, v_pages, _indices(src), _indices(dst))


def compact_path(k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                 context_lens: torch.Tensor, path: torch.Tensor, path_lens: torch.Tensor,
                 status: Optional[torch.Tensor] = None) -> None:
    """Keep the accepted path of drafted trees, in place: the new token at
    ``path[b, i]`` moves to place ``context_lens[b] + i`` for ``i < path_lens[b]``.

    ``path`` (int32 ``[requests, width]``) increases along each row; what lies
    behind the path is left as it was.  Requests must not share the pages that
    hold their new tokens.
    """
    load().compact_path(k_pages, v_pages, block_table, context_lens, path, path_lens, status)


def tree_mask(parents: torch.Tensor, cu_q: Optional[torch.Tensor] = None, *, max_q: int,
              batch: int = 1, status: Optional[torch.Tensor] = None
              ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Masks and depths of drafted trees from ``parents`` (int32, one per packed
    token: the parent's index within its own tree, before the token itself; -1 for
    a root).  A token sees its ancestors and itself.

    Returns ``(mask, depth)``: int32 words of 32 bits ``[tokens, ceil(max_q / 32)]``
    for `tree_attention` (ancestors behind the last column are left out), and int32 depths (0 for a root), so that a token's
    position is ``context + depth``.  One call serves every layer of a step.
    """
    return load().tree_mask(parents, cu_q, batch, max_q, status)


def pack_mask(mask: torch.Tensor) -> torch.Tensor:
    """A bool mask ``[tokens, columns]`` as the words `tree_attention` reads."""
    return load().pack_mask(mask)


def tree_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                   block_table: torch.Tensor, context_lens: torch.Tensor,
                   cu_q: Optional[torch.Tensor] = None, *, max_q: Optional[int] = None,
                   mask: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                   return_lse: bool = False, out: Optional[torch.Tensor] = None,
                   status: Optional[torch.Tensor] = None, timeout_s: float = 10.0):
    """Attention of new tokens over a paged cache that already holds their K and V.

    A token sees every cached token of its request, and among the new ones those
    whose bit is set in its row of ``mask`` (bool ``[tokens, columns]`` or the int32
    words of `tree_mask` / `pack_mask`; columns beyond the mask are not seen).
    Without a mask the new tokens are causal: one token is a decoding step, many
    are a chunk of a prompt.  A row that sees nothing gives zeros and ``lse = -inf``.

    ``q`` is ``[tokens, heads, dim]`` with dim 64 or 128 and heads a multiple of
    the cache's; page sizes 16 to 256, powers of two.  ``max_q`` is the most new
    tokens of any request where the caller knows it.  Any value is right; it chooses the
    kernel: with ``cu_q`` alone a request could hold all the tokens, and a batch of
    decoding steps would run on tiles of 256 rows.  A bool mask is packed in every call;
    layers share one packed by `pack_mask`.

    ``timeout_s`` bounds the kernel's waits for its own loads and products; one that runs out
    is reported in ``status``, and calls given the word end early until it is cleared.
    Returns ``out``, or ``(out, lse)`` with the natural-log sums ``[tokens, heads]`` in
    fp32.
    """
    o, lse = load().tree_attention(q, k_pages, v_pages, block_table, context_lens, cu_q, max_q,
                                   mask, scale, return_lse, out, status, timeout_s)
    return (o, lse) if return_lse else o
