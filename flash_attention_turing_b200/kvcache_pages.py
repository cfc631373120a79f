"""The pages of a paged KV cache: reserving, forking, freeing, compacting and copying them, on the device.

The cache is the one that ``flash_attn_with_kvcache`` and ``flash_diff_attn_with_kvcache`` read: per layer a K and a V tensor
(num_pages, page_size, nheads_k, d), one block table (batch, columns) and one cache_seqlens (batch,) for all of them.  Besides, these
functions keep ``page_refs`` (num_pages,) int32: by how many rows a page is held, 0 = free.  A row's pages come first in the block
table, and -1 stands behind them; an unused row has length 0 and no page.  A fresh cache::

    block_table = torch.full((batch, columns), -1, dtype=torch.int32, device="cuda")
    cache_seqlens = torch.zeros(batch, dtype=torch.int32, device="cuda")
    page_refs = torch.zeros(num_pages, dtype=torch.int32, device="cuda")

and a step of a serving loop: ``kvcache_reserve`` for the tokens to come, the attention of every layer (which appends them),
``cache_seqlens += 1``, ``kvcache_fork`` and ``kvcache_free`` as sequences split and end.  The tensors are changed in place; free pages
are taken in ascending order, so that the outcome does not depend on scheduling.  Nothing synchronises: what could not be done is told
by a bool tensor on the device.  Calls on the same tables have to be ordered, by one stream for instance, and may be captured in a CUDA
graph (after a first call outside a capture).

Pages that rows share are full, and attention only appends, so they are never written.  A row that is cut back into a shared
page (``cache_seqlens`` lowered by hand) must not be appended to: fork it instead, which copies the page, and free the original.
No counterpart in Cy-47/flash-attention-turing.
"""
from __future__ import annotations

from typing import Sequence, Union

import torch

from . import _ext


def _caches(caches) -> list:
    if isinstance(caches, torch.Tensor):
        raise TypeError("caches must be a sequence of tensors: k and v of every layer")
    return caches if type(caches) is list else list(caches)


def _blame(caches, **tensors) -> None:
    """The binding did not take the types that it was given: names the argument that is not a tensor, if there is one."""
    for x in caches:
        if not isinstance(x, torch.Tensor):
            raise TypeError("every cache must be a torch.Tensor") from None
    for key, x in tensors.items():
        if not isinstance(x, torch.Tensor):
            raise TypeError(f"{key} must be a torch.Tensor") from None


def kvcache_reserve(block_table: torch.Tensor, cache_seqlens: torch.Tensor, page_refs: torch.Tensor,
                    new_tokens: Union[int, torch.Tensor], page_size: int) -> torch.Tensor:
    """Gives every row the pages that ``cache_seqlens + new_tokens`` tokens need (an int for all rows, or int32 (batch,); negative
    entries count as 0).  An int gives pages to rows that are not in use as well, and a row that holds pages cannot become the child of
    a fork: 0 in a tensor for those.  Returns bool (batch,): whether the row has them.  Rows are served in order while the free pages last, each
    with all it needs or nothing, and what a refused row needs is kept from the rows behind it.  A row whose columns do not suffice is
    refused and keeps nothing from others.  Calling it again for the same tokens changes nothing."""
    each = isinstance(new_tokens, torch.Tensor)
    if not each and (isinstance(new_tokens, bool) or not isinstance(new_tokens, int)):
        raise TypeError("new_tokens must be an int or a torch.Tensor")
    try:
        return _ext.load().pages_reserve(block_table, cache_seqlens, page_refs, new_tokens if each else None, 0 if each else new_tokens,
                                         page_size)
    except TypeError:
        _blame((), block_table=block_table, cache_seqlens=cache_seqlens, page_refs=page_refs)
        raise


def kvcache_fork(caches: Sequence[torch.Tensor], block_table: torch.Tensor, cache_seqlens: torch.Tensor, page_refs: torch.Tensor,
                 parents: torch.Tensor, children: torch.Tensor) -> torch.Tensor:
    """Row ``children[i]`` (which holds no page) becomes a copy of row ``parents[i]``, int32 (n,) both: it shares the full pages of the
    parent's tokens, and the tokens of a last page that is not full are copied to a free page, in every cache.  Pages that the parent has
    reserved ahead are not shared.  A parent may have several children.  Returns bool (n,): whether it was done.  Not done, and
    nothing changed: a row out of range (-1 pads), a child that holds pages or that an earlier entry names, a parent that holds no page
    or fewer than its length says or has -1 among them, or no page left for the copy (entries are served in order)."""
    caches = _caches(caches)
    try:
        return _ext.load().pages_fork(caches, block_table, cache_seqlens, page_refs, parents, children)
    except TypeError:
        _blame(caches, block_table=block_table, cache_seqlens=cache_seqlens, page_refs=page_refs, parents=parents, children=children)
        raise


def kvcache_free(block_table: torch.Tensor, cache_seqlens: torch.Tensor, page_refs: torch.Tensor, rows: torch.Tensor) -> None:
    """Rows ``rows`` (int32 (n,)) give their pages back and become empty.  Rows out of range (-1 pads) are skipped, empty ones
    stay as they are, and a row that is named twice is freed once."""
    try:
        _ext.load().pages_free(block_table, cache_seqlens, page_refs, rows)
    except TypeError:
        _blame((), block_table=block_table, cache_seqlens=cache_seqlens, page_refs=page_refs, rows=rows)
        raise


def kvcache_compact(caches: Sequence[torch.Tensor], block_table: torch.Tensor, page_refs: torch.Tensor) -> torch.Tensor:
    """Moves pages so that those in use are the first ones of every cache, and rewrites ``block_table`` and ``page_refs``: the i-th page
    in use that lies behind the first ``live`` pages goes to the i-th free one among them.  Returns ``live``, the number of pages in
    use, int32 (1,).  Pages that do not have to move keep their place."""
    caches = _caches(caches)
    try:
        return _ext.load().pages_compact(caches, block_table, page_refs)
    except TypeError:
        _blame(caches, block_table=block_table, page_refs=page_refs)
        raise


def kvcache_copy_pages(caches: Sequence[torch.Tensor], src: torch.Tensor, dst: torch.Tensor) -> torch.Tensor:
    """Page ``dst[i]`` of every cache becomes a copy of page ``src[i]``, int32 (n,) both.  A page may be the source of several entries.
    Returns bool (n,): whether it holds.  Not done: a page out of range (-1 pads), a destination that a later entry has too (the last one
    wins), and a source that another entry overwrites.  Neither block tables nor ``page_refs`` are looked at."""
    caches = _caches(caches)
    try:
        return _ext.load().pages_copy(caches, src, dst)
    except TypeError:
        _blame(caches, src=src, dst=dst)
        raise
