"""A key-value cache in pages on CUDA: block tables and slot maps, rotary embedding + append, attention of one new token per
request and of several.

The reference keeps one contiguous cache per sequence (metile/integrations/mlx_lm.py takes MLX-LM's) and has no
counterpart.  Pages are [pages, kv_heads, page_size, head_dim] tensors of bfloat16 or float16, any strides with a dense
last dimension (a view of [pages, page_size, kv_heads, head_dim] as well as of a pool of several layers), page_size 8,
16, 32, 64, 128 or 256.  Row r of a block table (int32 [requests, width]) names the pages of request r in order: its
token t is in slot table[r, t // page_size] * page_size + t % page_size.

An index outside its table is left out by the kernel that meets it and recorded: `_lib.device_status()` tells.
"""

from __future__ import annotations

import numbers

import torch

from ._common import native, native_result, require_on_device
from .cuda_quantized import _flags

PAGE_SIZES = (8, 16, 32, 64, 128, 256)
PAGE_DTYPES = (torch.bfloat16, torch.float16)


def _require_cuda(tensor, what, dtypes, ndim):
    if not isinstance(tensor, torch.Tensor):
        raise TypeError(f"{what} must be a torch tensor")
    if tensor.dtype not in dtypes:
        raise TypeError(f"{what} must be {' or '.join(str(d) for d in dtypes)}, got {tensor.dtype}")
    if not tensor.is_cuda:
        raise ValueError(f"{what} must be a CUDA tensor; there is no CPU path")
    if tensor.ndim != ndim:
        raise ValueError(f"{what} must have {ndim} dimensions, got {tensor.ndim}")


def _require_ints(tensor, like, what, count, dtype=torch.int32):
    require_on_device(tensor, like, what, dtype=dtype)
    if tensor is None or tensor.numel() != count:
        raise ValueError(f"{what} must hold {count} elements")


def _require_table(table, what="block_tables"):
    _require_cuda(table, what, (torch.int32,), 2)
    if table.shape[1] < 1 or (table.numel() and table.shape[1] > 1 and table.stride(1) != 1) or (
            table.shape[0] > 1 and table.stride(0) < table.shape[1]):
        raise ValueError(f"{what} must be rows of one block or more, dense and apart")


def _require_pages(key_pages, value_pages, like=None):
    for tensor, what in ((key_pages, "key_pages"), (value_pages, "value_pages")):
        _require_cuda(tensor, what, PAGE_DTYPES, 4)
        if like is not None and (tensor.device != like.device or tensor.dtype != like.dtype):
            raise ValueError(f"{what} must match the rows' device and type ({like.device}, {like.dtype})")
        if tensor.numel() == 0:
            raise ValueError(f"{what} holds no page")
        if tensor.stride(3) != 1 or any(n > 1 and s % 8 for n, s in zip(tensor.shape[:3], tensor.stride())) \
                or tensor.data_ptr() % 16:
            raise ValueError(f"{what} must have a dense last dimension and rows that start on 16 bytes")
        extent = tensor.shape[3]
        for stride, size in sorted((s, n) for n, s in zip(tensor.shape[:3], tensor.stride()) if n > 1):
            if stride < extent:
                raise ValueError(f"{what} must not overlap itself")
            extent += stride * (size - 1)
    if key_pages.shape != value_pages.shape:
        raise ValueError("key_pages and value_pages must have one shape")
    if key_pages.shape[2] not in PAGE_SIZES:
        raise ValueError(f"the page size must be one of {PAGE_SIZES}, got {key_pages.shape[2]}")


def _refuse_gradient(what, *tensors):
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise ValueError(f"{what} has no gradient: call it under torch.no_grad() or on detached tensors")


def _bare(tensor):
    """The tensor itself where a subclass wraps it."""
    return tensor.detach().as_subclass(torch.Tensor)


def paged_resize(block_tables, lengths, counts, free_pages, free_state, *, page_size, tokens, advance=False):
    """Let every request grow by counts[r] > 0 tokens, or lose its last -counts[r], on the GPU.

    block_tables int32 [requests, width], lengths and counts int32 [requests]; free_pages int32 [pool] is a ring of the ids no
    request uses, free_state int32 [2] the index of the first of them and how many there are.  Pages are taken from the
    head of the ring, in the order of the requests, and given back at its tail (for the next call).  Returns
    (slots, positions, starts, lengths, free_state): of the new tokens, request after request, slots int64 [tokens] and
    positions int32 [tokens] (-1 and 0 behind the last one); starts int32 [requests + 1], each request's first token;
    the new lengths and state, with `advance` in place.  block_tables and the ring's tail are written in place; a call with the
    same lengths and state does the same again.

    A request stays as it is, its tokens with -1 and 0, when its length or count makes no sense, when `width` blocks or
    the `tokens` of the map have no room for it, or when the free pages do not reach for it and all requests before it.
    No page may belong to two requests that give it back."""
    arguments = (block_tables, lengths, counts, free_pages, free_state)
    out = native().paged_resize(*arguments, page_size, tokens, bool(advance))
    if out is None:
        _require_table(block_tables)
        requests = block_tables.shape[0]
        if not isinstance(page_size, int) or page_size not in PAGE_SIZES:
            raise ValueError(f"the page size must be one of {PAGE_SIZES}, got {page_size}")
        if not isinstance(tokens, int) or not 0 <= tokens <= 0x7FFFFFFF:
            raise ValueError("paged_resize: tokens must be a whole number from 0 to 2^31 - 1")
        _require_ints(lengths, block_tables, "lengths", requests)
        _require_ints(counts, block_tables, "counts", requests)
        require_on_device(free_pages, block_tables, "free_pages", dtype=torch.int32, min_numel=1)
        _require_ints(free_state, block_tables, "free_state", 2)
        out = native().paged_resize(*map(_bare, arguments), page_size, tokens, bool(advance))
        if out is None:
            raise ValueError("paged_resize: sizes beyond what the kernel takes")
    return native_result(out, "paged_resize")


def rope_kv_append_paged(query, key, value, inverse, positions, slots, key_pages, value_pages):
    """Rotate the query and key rows of a ragged batch and write key and value to their slots of the pages, in place.

    query [rows, Hq, D], key / value [rows, Hkv, D] -- dense, or views into the rows of one fused q|k|v projection;
    inverse fp32 [D/2]: pair (i, i + D/2) of a row is turned by positions[r] * inverse[i], taken in 64 bits; positions int32
    [rows], slots int64 [rows] (as paged_resize gives them): a row whose slot is negative is rotated and not written.
    No two rows name one slot.  Returns the rotated query as a dense [rows, Hq, D] tensor."""
    arguments = (query, key, value, inverse, positions, slots, key_pages, value_pages)
    out = native().rope_kv_append_paged(*arguments)
    if out is None:
        for tensor, what in ((query, "query"), (key, "key"), (value, "value")):
            _require_cuda(tensor, what, PAGE_DTYPES, 3)
        _require_pages(key_pages, value_pages, query)
        _refuse_gradient("rope_kv_append_paged", query, key, value, key_pages, value_pages)
        rows, _, dim = query.shape
        kv_heads = key_pages.shape[1]
        if key.shape != (rows, kv_heads, dim) or value.shape != key.shape or key_pages.shape[3] != dim:
            raise ValueError("rope_kv_append_paged expects key and value rows [rows, kv_heads, head_dim] as the pages have them")
        for tensor, what in ((key, "key"), (value, "value")):
            require_on_device(tensor, query, what, dtype=query.dtype, contiguous=False)
        if dim < 16 or dim % 16 or dim > 4096:
            raise ValueError("rope_kv_append_paged: the head dimension must be a multiple of 16 up to 4096")
        _require_ints(inverse, query, "inverse", dim // 2, torch.float32)
        _require_ints(positions, query, "positions", rows)
        _require_ints(slots, query, "slots", rows, torch.int64)
        if query.shape[1] < 1:
            raise ValueError("rope_kv_append_paged expects a query head or more")
        if rows == 0:
            return torch.empty_like(query)
        # What remains is the layout of the rows: a fresh dense copy is aligned.
        query, key, value = (_bare(t).clone(memory_format=torch.contiguous_format) for t in (query, key, value))
        out = native().rope_kv_append_paged(query, key, value, *map(_bare, arguments[3:]))
        if out is None:
            raise ValueError("rope_kv_append_paged: sizes beyond what the kernel takes")
    return native_result(out, "rope_kv_append_paged")


def paged_attention_decode(query, key_pages, value_pages, block_tables, lengths, *, scale):
    """softmax(scale * q k^T) v for one query row per request and head over a cache in pages.

    query [requests, Hq, D], D 64, 128 or 256, Hq a multiple of the pages' heads; lengths int32 [requests]: how many tokens of
    its row of block_tables a request has, the new one among them.  No tokens: a row of zeros.  A NaN in what is used comes
    out as NaN.  Returns [requests, Hq, D].
    A request's bits depend on its own tokens only, not on the others of the call.  The scratch of a call follows the
    width of block_tables, not the lengths: requests * Hq * min(width * page_size / 128, 128) * (D + 2) numbers of 32 bits, up to
    four times as many splits with fewer than four KV heads."""
    arguments = (query, key_pages, value_pages, block_tables, lengths)
    out = native().paged_attention_decode(*arguments, scale)
    if out is None:
        _require_cuda(query, "query", PAGE_DTYPES, 3)
        _require_pages(key_pages, value_pages, query)
        _refuse_gradient("paged_attention_decode", query, key_pages, value_pages)
        _require_table(block_tables)
        requests, heads, dim = query.shape
        if block_tables.device != query.device or block_tables.shape[0] != requests:
            raise ValueError("paged_attention_decode expects a row of block_tables for every query, on its device")
        if key_pages.shape[3] != dim or dim not in (64, 128, 256):
            raise ValueError("paged_attention_decode: the head dimension must be 64, 128 or 256 and match")
        if heads < 1 or heads % key_pages.shape[1]:
            raise ValueError("key/value heads must divide query heads")
        _require_ints(lengths, query, "lengths", requests)
        if requests == 0:
            return torch.empty_like(query)
        query = _bare(query).clone(memory_format=torch.contiguous_format)
        out = native().paged_attention_decode(query, *map(_bare, arguments[1:]), float(scale))
        if out is None:
            raise ValueError("paged_attention_decode: sizes beyond what the kernel takes")
    return native_result(out, "paged_attention_decode")


def paged_attention_chunk(query, key_pages, value_pages, block_tables, lengths, starts, *, scale):
    """softmax(scale * q k^T) v for several new tokens per request over a cache in pages, each seeing the tokens up to its own.

    query [rows, Hq, D], D 64, 128 or 256, Hq a multiple of the pages' heads; lengths int32 [requests]: how many tokens of its row
    of block_tables a request has, the new ones among them; starts int32 [requests + 1], ascending: rows starts[r] up to
    starts[r + 1] are the last tokens of request r (as paged_resize returns it).  A piece of a prompt, a draft and a single token
    may stand beside each other.  Rows that see nothing (more rows than tokens) and rows of no request are zeros.  What a row
    does not see weighs nothing, whatever lies there; a NaN that it sees comes out as NaN.  Returns [rows, Hq, D].
    Within batch_invariant() or fixed_order() a row's bits depend on the tokens it sees only, not on the others of the call nor on
    how its prompt was cut into pieces; elsewhere long requests with few rows are cut as the sizes of the call ask."""
    arguments = (query, key_pages, value_pages, block_tables, lengths, starts)
    out = native().paged_attention_chunk(*arguments, scale, _flags())
    if out is None:
        _require_cuda(query, "query", PAGE_DTYPES, 3)
        _require_pages(key_pages, value_pages, query)
        _refuse_gradient("paged_attention_chunk", query, key_pages, value_pages)
        _require_table(block_tables)
        rows, heads, dim = query.shape
        requests = block_tables.shape[0]
        if block_tables.device != query.device:
            raise ValueError("paged_attention_chunk expects block_tables on the queries' device")
        if key_pages.shape[3] != dim or dim not in (64, 128, 256):
            raise ValueError("paged_attention_chunk: the head dimension must be 64, 128 or 256 and match")
        if heads < 1 or heads % key_pages.shape[1]:
            raise ValueError("key/value heads must divide query heads")
        _require_ints(lengths, query, "lengths", requests)
        _require_ints(starts, query, "starts", requests + 1)
        if not isinstance(scale, numbers.Real):
            raise TypeError("paged_attention_chunk: scale must be a number")
        if rows == 0:
            return torch.empty_like(query)
        query = _bare(query).clone(memory_format=torch.contiguous_format)
        out = native().paged_attention_chunk(query, *map(_bare, arguments[1:]), float(scale), _flags())
        if out is None:
            raise ValueError("paged_attention_chunk: sizes beyond what the kernel takes")
    return native_result(out, "paged_attention_chunk")
