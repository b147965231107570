"""Log-probabilities of given texts under a model, over a paged cache.

Prompts are read in pieces, all of them together.  Continuations of one prompt share its pages: it is read once, a branch of it
made for each of them, and its continuation read there.  The reference has no counterpart."""

from __future__ import annotations

from dataclasses import dataclass

import torch

from .. import backends


@dataclass
class TokenScores:
    """Of every token of a text: its log-probability, the entropy of the distribution it was drawn from, and the best
    alternatives (float32 [tokens], float32 [tokens], float32 [tokens, top], int64 [tokens, top])."""

    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_logprobs: torch.Tensor
    top_tokens: torch.Tensor


def _pages_for(lengths, page_size):
    return sum(-(-n // page_size) for n in lengths)


def _flat(texts, what):
    texts = [torch.as_tensor(text).reshape(-1).to(torch.int64) for text in texts]
    if not texts or not all(text.numel() for text in texts):
        raise ValueError(f"{what}: every text needs a token")
    return texts


def _read(model, cache, texts, rows, piece, wanted):
    """Read texts[i] as the next tokens of request rows[i], in passes of up to `piece` tokens, and yield (text, first position,
    logits) of the positions that wanted(text, first, count) names, relative to `first`."""
    if piece < 1:
        raise ValueError("a pass reads a token or more")
    tables = cache[0].tables
    device = tables.lengths.device
    done = [0] * len(texts)
    while True:
        counts, parts, at, asked, left = [0] * tables.requests, [], 0, [], piece
        # The requests of a pass come in their order, whatever that of the texts is.
        for i in sorted(range(len(texts)), key=lambda i: rows[i]):
            count = min(texts[i].numel() - done[i], left)
            if count == 0:
                continue
            counts[rows[i]] = count
            parts.append(texts[i][done[i]:done[i] + count])
            positions = wanted(i, done[i], count)
            if positions:
                asked.append((i, done[i], len(positions)))
                parts[-1] = (parts[-1], [at + position for position in positions])
            else:
                parts[-1] = (parts[-1], [])
            at, left = at + count, left - count
            done[i] += count
        if not parts:
            return
        tables.extend(counts)
        tokens = torch.cat([tokens for tokens, _ in parts]).to(device)[None]
        positions = torch.tensor([p for _, ps in parts for p in ps] or [at - 1], device=device)
        logits = model(tokens, cache=cache, logits_at=positions)[0]
        first = 0
        for i, start, count in asked:
            yield i, start, logits[first:first + count]
            first += count


def _scores(logits, tokens, top):
    return backends.token_logprobs(logits, tokens.to(logits.device), top=top)


def _joined(parts):
    return TokenScores(*(torch.cat([part[k] for part in parts]) for k in range(4)))


@torch.no_grad()
def score_prompts(model, prompts, *, top=0, piece=2048, page_size=16):
    """TokenScores of every prompt (a row of token ids each) but for its first token, which nothing predicts.

    The model must offer `make_paged_cache` and take `logits_at` (blocks.TinyCausalLM does)."""
    prompts = _flat(prompts, "score_prompts")
    cache = model.make_paged_cache(len(prompts), _pages_for([p.numel() for p in prompts], page_size), page_size,
                                   max(p.numel() for p in prompts))
    parts = [[] for _ in prompts]

    def wanted(i, first, count):  # the last position predicts nothing that is there
        return list(range(min(count, prompts[i].numel() - 1 - first)))

    for i, first, logits in _read(model, cache, prompts, list(range(len(prompts))), piece, wanted):
        parts[i].append(_scores(logits, prompts[i][first + 1:first + 1 + logits.shape[0]], top))
    empty = torch.empty((0,), device=cache[0].tables.lengths.device)
    nothing = (empty, empty, empty.new_empty((0, top)), torch.empty((0, top), dtype=torch.int64, device=empty.device))
    return [_joined(part or [nothing]) for part in parts]


@torch.no_grad()
def score_continuations(model, prompts, continuations, *, top=0, piece=2048, page_size=16):
    """For every prompt a list with the TokenScores of each of its continuations (rows of token ids).

    A prompt is read once, and its pages shared by its continuations.  The model must offer `make_paged_cache` and take
    `logits_at` (blocks.TinyCausalLM does)."""
    prompts = _flat(prompts, "score_continuations")
    if len(continuations) != len(prompts):
        raise ValueError("score_continuations expects a list of continuations for every prompt")
    texts, owner = [], []
    for i, several in enumerate(continuations):
        several = _flat(several, "score_continuations") if len(several) else []
        texts += several
        owner += [i] * len(several)
    if not texts:
        return [[] for _ in prompts]
    # The pages of a prompt, then of each continuation what is behind the prompt's full pages.
    pages = _pages_for([p.numel() for p in prompts], page_size)
    pages += sum(_pages_for([prompts[i].numel() % page_size + text.numel()], page_size) for text, i in zip(texts, owner))
    cache = model.make_paged_cache(len(prompts) + len(texts), pages, page_size,
                                   max(prompts[i].numel() + text.numel() for text, i in zip(texts, owner)))
    tables = cache[0].tables
    last = [None] * len(prompts)  # logits behind each prompt

    def end(i, first, count):
        return [count - 1] if first + count == prompts[i].numel() else []

    for i, _, logits in _read(model, cache, prompts, list(range(len(prompts))), piece, end):
        last[i] = logits
    parts = [[_scores(last[i], text[:1], top)] for text, i in zip(texts, owner)]
    rows = [len(prompts) + k for k in range(len(texts))]
    tables.branch([None] * len(prompts) + owner, [0] * len(prompts) + [prompts[i].numel() for i in owner], cache)
    tables.release(range(len(prompts)))  # what they hold alone goes back; the branches hold the rest
    longer = [k for k, text in enumerate(texts) if text.numel() > 1]
    for j, first, logits in _read(model, cache, [texts[k][:-1] for k in longer], [rows[k] for k in longer], piece,
                                  lambda j, first, count: list(range(count))):
        text = texts[longer[j]]
        parts[longer[j]].append(_scores(logits, text[first + 1:first + 1 + logits.shape[0]], top))
    tables.release(rows)
    scores = [[] for _ in prompts]
    for i, part in zip(owner, parts):
        scores[i].append(_joined(part))
    return scores
