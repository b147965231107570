"""Beam search on CUDA: the selection over beams and vocabulary, and the reordering of the paged cache behind it.

The reference decodes greedily and has no counterpart."""

from __future__ import annotations

import torch

from ._common import native, native_result, require_on_device
from .cuda_paged import _bare, _refuse_gradient, _require_cuda, _require_ints, _require_pages, _require_table

MAX_BEAMS, MAX_KEEP = 32, 64
MAX_ROWS, MAX_VOCABULARY = 0x000FFFFF, 0x00080000
LOGIT_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def beam_select(logits, scores, *, keep=None, finished=None, end_token=None):
    """The `keep` best continuations (default: as many as beams) of every group of beams.

    logits [groups * beams, vocabulary] bfloat16, float16 or float32; scores float32 [groups, beams], the sums of
    log-probabilities so far.  A candidate is worth scores + log_softmax(logits), in 64 bits; the largest come first, among
    equals the lower beam, then the larger logit, then the lower token.  A beam that has `finished` (bool [groups, beams]) offers `end_token`
    alone, at the score it has.  A score up to -1e9 is a mask: that beam's candidates count as -inf, and so do those of
    logits with a NaN, with +inf or with nothing above -inf.

    Returns (scores float32, parents int32 -- the beam within its group --, tokens int64, finished bool), all
    [groups, keep].  finished: the parent had finished or the token is end_token.  A score is rounded to 32 bits, and may be off
    by 2^-18 before that; where two beams are closer than that allows, their order is the one of sums in 64 bits."""
    kept = scores.shape[1] if keep is None and isinstance(scores, torch.Tensor) and scores.ndim == 2 else keep
    end = -1 if end_token is None else -2 if end_token == -1 else end_token
    out = None
    if finished is None or end_token is not None:
        out = native().beam_select(logits, scores, kept, finished, end)
    if out is None:
        _require_cuda(logits, "logits", LOGIT_DTYPES, 2)
        _require_cuda(scores, "scores", (torch.float32,), 2)
        _refuse_gradient("beam_select", logits, scores)
        groups, beams = scores.shape
        rows, vocabulary = logits.shape
        if rows != groups * beams:
            raise ValueError("beam_select expects a row of logits for every score")
        if not 1 <= beams <= MAX_BEAMS or rows > MAX_ROWS or not 1 <= vocabulary <= MAX_VOCABULARY:
            raise ValueError(f"beam_select serves 1 to {MAX_BEAMS} beams, {MAX_ROWS} rows and vocabularies up to {MAX_VOCABULARY}")
        if not isinstance(kept, int) or not 1 <= kept <= min(MAX_KEEP, beams * vocabulary):
            raise ValueError(f"beam_select: keep must be from 1 to {MAX_KEEP} and at most beams * vocabulary")
        if not isinstance(end, int) or not -1 <= end < vocabulary or (end_token is not None and end < 0):
            raise ValueError("beam_select: the end token is not in the vocabulary")
        require_on_device(scores, logits, "scores", contiguous=False)
        if finished is not None:
            if end_token is None:
                raise ValueError("beam_select: finished beams need an end token")
            require_on_device(finished, logits, "finished", dtype=torch.bool, contiguous=False)
            if finished.shape != scores.shape:
                raise ValueError("finished must be shaped like scores")
            finished = _bare(finished).contiguous()
        logits = _bare(logits)
        if logits.stride(1) != 1:
            logits = logits.contiguous()
        if groups == 0:
            shape, device = (0, kept), logits.device
            return (torch.empty(shape, device=device), torch.empty(shape, dtype=torch.int32, device=device),
                    torch.empty(shape, dtype=torch.int64, device=device), torch.empty(shape, dtype=torch.bool, device=device))
        out = native().beam_select(logits, _bare(scores).contiguous(), kept, finished, end)
        if out is None:
            raise ValueError("beam_select: arguments beyond what the kernel takes")
    return native_result(out, "beam_select")


def beam_reorder(block_tables, lengths, parents, caches):
    """Let the block tables of a paged cache, and its pages in work, follow the surviving beams.

    block_tables int32 [groups * beams, width], lengths int32 [groups * beams] (equal within a group; the first counts),
    parents int32 [groups, beams]: which beam of its group each row continues; caches: the (key_pages, value_pages) of every
    layer.  Returns the new block tables.  Full pages are shared with the parent.  The page in work is written on, so
    it stays one beam's own: a parent's first child goes on in it, any other child takes that of a beam without children,
    and what the parent's holds is copied there, in place, in every cache.  Entries behind it stay each row's own.  The pages in
    work of a group must be distinct before the call, and are after it."""
    out = native().beam_reorder(block_tables, lengths, parents, caches)
    if out is None:
        _require_table(block_tables)
        _require_cuda(parents, "parents", (torch.int32,), 2)
        rows = block_tables.shape[0]
        if parents.device != block_tables.device or parents.numel() != rows or not 1 <= parents.shape[1] <= MAX_BEAMS:
            raise ValueError(f"beam_reorder expects a parent for every row of block_tables and 1 to {MAX_BEAMS} beams")
        _require_ints(lengths, block_tables, "lengths", rows)
        caches = tuple(tuple(pair) for pair in caches)
        if not caches or any(len(pair) != 2 for pair in caches):
            raise ValueError("beam_reorder expects the (key_pages, value_pages) of one layer or more")
        sample = caches[0][0]
        for keys, values in caches:
            _require_pages(keys, values, sample)
            _refuse_gradient("beam_reorder", keys, values)
            if keys.shape != sample.shape or keys.device != block_tables.device or keys.stride() != sample.stride() \
                    or values.stride() != caches[0][1].stride():
                raise ValueError("beam_reorder expects caches of one shape and layout on the block tables' device")
        if sample.shape[3] % 8:
            raise ValueError("beam_reorder: the head dimension must be a multiple of 8")
        if rows == 0:
            return torch.empty_like(block_tables)
        caches = tuple((_bare(keys), _bare(values)) for keys, values in caches)
        out = native().beam_reorder(_bare(block_tables), _bare(lengths), _bare(parents).contiguous(), caches)
        if out is None:
            raise ValueError("beam_reorder: sizes beyond what the kernel takes")
    return native_result(out, "beam_reorder")
