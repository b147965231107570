"""Pages of a cache that several requests hold, on CUDA: requests that go on from another's tokens, requests that end, and a pool
that is put together again.  No counterpart in the reference.

`shares` (int32, one number for every page) says how many requests hold a page beyond the first one.  Pages that
paged_resize hands out have one holder, so it needs no shares; it must not give back tokens in pages that are shared."""

from __future__ import annotations

import torch

from ._common import native, native_result, require_on_device
from .cuda_paged import PAGE_SIZES, _bare, _refuse_gradient, _require_ints, _require_pages, _require_table


def _require_caches(what, caches, like):
    caches = tuple(tuple(pair) for pair in caches)
    if not caches or any(len(pair) != 2 for pair in caches):
        raise ValueError(f"{what} expects the (key_pages, value_pages) of one layer or more")
    sample = caches[0][0]
    for keys, values in caches:
        _require_pages(keys, values, sample)
        _refuse_gradient(what, keys, values)
        if keys.shape != sample.shape or keys.device != like.device or keys.stride() != sample.stride() \
                or values.stride() != caches[0][1].stride():
            raise ValueError(f"{what} expects caches of one shape and layout on the block tables' device")
    if sample.shape[3] % 8:
        raise ValueError(f"{what}: the head dimension must be a multiple of 8")
    return tuple((_bare(keys), _bare(values)) for keys, values in caches)


def paged_fork(block_tables, lengths, sources, counts, free_pages, free_state, shares, caches, *, advance=False):
    """Let empty requests go on from the first tokens of others.

    block_tables int32 [requests, width], lengths int32 [requests]; a request r with sources[r] >= 0 (int32) and no tokens becomes
    the first counts[r] > 0 (int32) tokens of request sources[r].  Full pages are shared: their ids go to its row and their
    shares (int32 [pages]) grow.  The page begun, into which both would write, is copied, in all caches (the (key_pages,
    value_pages) of every layer), into one from the head of the ring of free ids (free_pages int32, free_state int32 [2], as for
    paged_resize).  block_tables and caches are written in place; returns the new (lengths, free_state, shares), with `advance` in
    place too.  Without it a call with the same arguments does the same again.

    A request stays as it is when its source, count or length makes no sense, or when the free pages do not reach for it and all
    before it that need one.  A request of the same call is no source: it had no tokens."""
    arguments = (block_tables, lengths, sources, counts, free_pages, free_state, shares)
    out = native().paged_fork(*arguments, caches, bool(advance))
    if out is None:
        _require_table(block_tables)
        requests = block_tables.shape[0]
        for tensor, what in ((lengths, "lengths"), (sources, "sources"), (counts, "counts")):
            _require_ints(tensor, block_tables, what, requests)
        require_on_device(free_pages, block_tables, "free_pages", dtype=torch.int32, min_numel=1)
        _require_ints(free_state, block_tables, "free_state", 2)
        caches = _require_caches("paged_fork", caches, block_tables)
        _require_ints(shares, block_tables, "shares", caches[0][0].shape[0])
        out = native().paged_fork(*map(_bare, arguments), caches, bool(advance))
        if out is None:
            raise ValueError("paged_fork: sizes beyond what the kernel takes")
    return native_result(out, "paged_fork")


def paged_free(block_tables, lengths, ended, free_pages, free_state, shares, *, page_size, advance=False):
    """Let the requests with ended[r] (bool [requests]) give back all their pages.

    A page goes to the tail of the ring of free ids when all who hold it (shares + 1 requests) have dropped it, in the order of
    requests and blocks, one that several drop at the first of them.  The ring's tail is written in place; returns the new
    (lengths, free_state, shares), with `advance` in place.  Without it a call with the same arguments does the same again."""
    arguments = (block_tables, lengths, ended, free_pages, free_state, shares)
    out = native().paged_free(*arguments, page_size, bool(advance))
    if out is None:
        _require_table(block_tables)
        requests = block_tables.shape[0]
        if not isinstance(page_size, int) or page_size not in PAGE_SIZES:
            raise ValueError(f"the page size must be one of {PAGE_SIZES}, got {page_size}")
        _require_ints(lengths, block_tables, "lengths", requests)
        _require_ints(ended, block_tables, "ended", requests, torch.bool)
        require_on_device(free_pages, block_tables, "free_pages", dtype=torch.int32, min_numel=1)
        _require_ints(free_state, block_tables, "free_state", 2)
        require_on_device(shares, block_tables, "shares", dtype=torch.int32, min_numel=1)
        out = native().paged_free(*map(_bare, arguments), page_size, bool(advance))
        if out is None:
            raise ValueError("paged_free: sizes beyond what the kernel takes")
    return native_result(out, "paged_free")


def paged_compact(block_tables, lengths, caches):
    """Move the pages that the block tables hold to the lowest ids, 0 up to their number.

    Of the pages above, in ascending order, the n-th goes to the n-th free id below, in all caches ((key_pages, value_pages) of
    every layer), in place.  What is held, shared and free is taken from the tables alone: pages that nobody holds any more, as
    beams leave them that were dropped, are free afterwards.  Returns (block_tables, free_pages, free_state, shares): the tables
    with the new ids, the ring of the others in ascending order (int32 [pages]), its state, and shares int32 [pages]."""
    out = native().paged_compact(block_tables, lengths, caches)
    if out is None:
        _require_table(block_tables)
        _require_ints(lengths, block_tables, "lengths", block_tables.shape[0])
        caches = _require_caches("paged_compact", caches, block_tables)
        out = native().paged_compact(_bare(block_tables), _bare(lengths), caches)
        if out is None:
            raise ValueError("paged_compact: sizes beyond what the kernel takes")
    return native_result(out, "paged_compact")
