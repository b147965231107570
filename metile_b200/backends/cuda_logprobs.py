"""Log-probabilities of given tokens on CUDA.  No counterpart in the reference, which decodes greedily."""

from __future__ import annotations

import torch

from ._common import native, native_result, require_on_device
from .cuda_beam import LOGIT_DTYPES
from .cuda_paged import _bare, _refuse_gradient, _require_cuda

MAX_TOP = 64
MAX_ROWS, MAX_VOCABULARY = 0x000FFFFF, 0x00080000


def token_logprobs(logits, tokens, *, top=0):
    """log_softmax(logits) at the given tokens, the entropy of every row and its `top` best alternatives.

    logits [rows, vocabulary] bfloat16, float16 or float32; tokens int64 [rows].  A token below 0 asks for nothing and gives 0; one
    outside the vocabulary gives NaN and is recorded.  Returns (logprobs, entropy, top_logprobs, top_tokens): float32 [rows], float32
    [rows], float32 [rows, top] and int64 [rows, top], the largest logits first, among equals the lower token.  A row with a NaN,
    with +inf or with nothing above -inf has no distribution: NaN, and -1 for its top tokens.
    Exponentials and their sums are of 32 bits, joined in 64; a row's bits do not depend on the others of the call."""
    out = native().token_logprobs(logits, tokens, top)
    if out is None:
        _require_cuda(logits, "logits", LOGIT_DTYPES, 2)
        _refuse_gradient("token_logprobs", logits)
        rows, vocabulary = logits.shape
        if rows > MAX_ROWS or not 1 <= vocabulary <= MAX_VOCABULARY:
            raise ValueError(f"token_logprobs serves up to {MAX_ROWS} rows and vocabularies up to {MAX_VOCABULARY}")
        if not isinstance(top, int) or not 0 <= top <= min(MAX_TOP, vocabulary):
            raise ValueError(f"token_logprobs: top must be from 0 to {MAX_TOP} and at most the vocabulary")
        if not isinstance(tokens, torch.Tensor):
            raise TypeError("tokens must be a torch tensor")
        if tokens.ndim != 1 or tokens.shape[0] != rows:
            raise ValueError("token_logprobs expects a token for every row of logits")
        require_on_device(tokens, logits, "tokens", dtype=torch.int64, contiguous=False)
        logits = _bare(logits)
        if rows == 0:
            device = logits.device
            return (torch.empty((0,), device=device), torch.empty((0,), device=device), torch.empty((0, top), device=device),
                    torch.empty((0, top), dtype=torch.int64, device=device))
        if logits.stride(1) != 1:
            logits = logits.contiguous()
        out = native().token_logprobs(logits, _bare(tokens).contiguous(), top)
        if out is None:
            raise ValueError("token_logprobs: arguments beyond what the kernel takes")
    return native_result(out, "token_logprobs")
