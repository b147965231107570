"""Prompts read in pieces, shared by branches, scored and given back: the operators together, in a model."""

import numpy as np
import pytest
import torch

from metile_b200 import _lib, backends as B
from metile_b200.integrations import blocks, scoring
from metile_b200.integrations.torch_lm import apply_metile_to_torch_lm

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def nothing_was_recorded(cuda_device):
    yield
    ok, words = _lib.device_status()
    assert ok, [hex(w) for w in words]


@pytest.fixture(scope="module")
def model(cuda_device):
    return blocks.random_model(seed=6, device=cuda_device)


def texts_of(lengths, seed):
    generator = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 512, (n,), generator=generator) for n in lengths]


def read(model, cache, pieces):
    """Logits of every new token; pieces: a row of tokens or None for every request."""
    tables = cache[0].tables
    tables.extend([0 if p is None else p.numel() for p in pieces])
    return model(torch.cat([p for p in pieces if p is not None]).to(tables.lengths.device)[None], cache=cache)[0]


def test_a_prompt_in_pieces_has_the_bits_of_one_read_at_once(cuda_device, model):
    texts = texts_of([100, 37, 1], 1)
    with torch.no_grad(), B.batch_invariant():
        cache = model.make_paged_cache(3, 40, 16, 256)
        whole = read(model, cache, texts).split([100, 37, 1])
        for cuts in ((0, 1, 50, 99, 100), (0, 64, 100)):
            cache = model.make_paged_cache(3, 40, 16, 256)
            out = [read(model, cache, [texts[0][a:b], texts[1] if a == 0 else None, texts[2] if a == 0 else None]) for a, b in zip(cuts, cuts[1:])]
            got = torch.cat([out[0][:cuts[1]]] + out[1:])
            assert torch.equal(got, whole[0]) and torch.equal(out[0][cuts[1]:cuts[1] + 37], whole[1])
        alone = model.make_paged_cache(1, 40, 16, 256)
        assert torch.equal(read(model, alone, texts[1:2]), whole[1])


def test_pieces_against_the_prompt_path_and_decoding(cuda_device, model):
    """Attention by torch over a prompt and by the decode kernel for a token: other sums of the same numbers."""
    text = texts_of([90], 2)[0]
    with torch.no_grad(), B.batch_invariant():
        cache = model.make_paged_cache(1, 20, 16, 256)
        cache[0].tables.grow([80])
        plain = [model(text[None, :80].to(cuda_device), cache=cache)[0]]
        for i in range(80, 90):
            cache[0].tables.grow()
            plain.append(model(text[None, i:i + 1].to(cuda_device), cache=cache)[0])
        plain = torch.cat(plain)
        cache = model.make_paged_cache(1, 20, 16, 256)
        got = torch.cat([read(model, cache, [text[:33]]), read(model, cache, [text[33:]])])
    # The bound the patched model is held to against the module by module form.
    assert (got - plain).float().abs().max() <= 2e-2 * plain.float().abs().max()


def test_a_patched_model_reads_pieces(cuda_device, model):
    text = texts_of([70], 3)[0]
    with torch.no_grad(), B.batch_invariant():
        plain_cache = model.make_paged_cache(1, 20, 16, 128)
        plain = torch.cat([read(model, plain_cache, [text[:64]]), read(model, plain_cache, [text[64:69]]), read(model, plain_cache, [text[69:]])])
        with apply_metile_to_torch_lm(model, attention=True):
            cache = model.make_paged_cache(1, 20, 16, 128)
            patched = torch.cat([read(model, cache, [text[:64]]), read(model, cache, [text[64:69]]), read(model, cache, [text[69:]])])
            cache[0].tables.grow()  # and decodes behind them
            assert model(text[None, :1].to(cuda_device), cache=cache).shape == (1, 1, 512)
    assert (plain - patched).float().abs().max() <= 2e-2 * plain.float().abs().max()


def test_branches_release_and_compact_keep_what_is_held(cuda_device, model):
    texts = texts_of([53, 20, 9, 30], 4)
    with torch.no_grad(), B.batch_invariant():
        alone = model.make_paged_cache(1, 40, 16, 256)
        read(model, alone, [texts[0][:40]])
        expected = read(model, alone, [texts[1]])
        cache = model.make_paged_cache(5, 30, 16, 256)
        tables = cache[0].tables

        def agrees():
            assert tables.lengths.tolist() == tables.held and int(tables.free_state[1]) == tables.free
            held = {}
            for r, n in enumerate(tables.held):
                for page in tables.block_tables[r, :-(-n // 16)].tolist():
                    held[page] = held.get(page, 0) + 1
            shares = tables.shares.tolist()
            assert all(shares[page] == held.get(page, 1) - 1 for page in range(30)) and len(held) + tables.free == 30

        read(model, cache, [texts[0], None, texts[3], None, None])
        tables.branch([None, 0, None, 0, 2], [0, 40, 0, 48, 30], cache)
        agrees()
        got = read(model, cache, [None, texts[1], None, texts[2], texts[2]])
        assert torch.equal(got[:20], expected)
        agrees()
        tables.release([0, 2])
        agrees()
        tables.compact(cache)
        agrees()
        assert int(tables.block_tables[1, 0]) < 30 - tables.free
        more = read(model, cache, [None, texts[2], None, texts[1], None])
        assert torch.equal(more[:9], read(model, alone, [texts[2]]))
        agrees()
        tables.branch([1, None, 1, None, None], [60, 0, 1, 0, 0], cache)
        tables.release([1, 3])
        agrees()
        tables.release([0, 2, 4])
        agrees()
        assert tables.free == 30


def test_compact_collects_the_pages_of_dropped_beams(cuda_device, model):
    cache = model.make_paged_cache(4, 40, 16, 128)
    tables = cache[0].tables
    with torch.no_grad():
        read(model, cache, [texts_of([50], 5)[0], None, None, None])
        tables.fork(4, cache)
        for step in range(20):
            tables.grow()
            model(torch.full((4, 1), step, dtype=torch.long, device=cuda_device), cache=cache)
            tables.reorder(torch.tensor([[0, 0, 2, 2]], dtype=torch.int32, device=cuda_device), cache)
        for refused in (lambda: tables.release([0]), lambda: tables.branch([None] * 4, [0] * 4, cache)):
            with pytest.raises(ValueError, match="not counted"):
                refused()
        before = tables.free
        kept = [cache[0].keys[tables.block_tables[r, :4].long()].clone() for r in range(4)]
        tables.compact(cache)
        assert tables.free > before and int(tables.free_state[1]) == tables.free
        for r in range(4):
            assert torch.equal(cache[0].keys[tables.block_tables[r, :4].long()], kept[r])
        tables.release(range(4))
        assert tables.free == 40 and not tables.shares.any()


def expected_scores(model, text, first, top):
    """Of tokens `first` on of a text that is read on its own."""
    cache = model.make_paged_cache(1, 40, 16, 512)
    logits = read(model, cache, [text])[first - 1:-1]
    return B.token_logprobs(logits, text[first:].to(logits.device), top=top)


def same(scores, expected):
    for a, b in zip((scores.logprobs, scores.entropy, scores.top_logprobs, scores.top_tokens), expected):
        assert torch.equal(a, b)


@pytest.mark.parametrize("piece", [7, 64, 2048])
def test_scores_of_prompts(cuda_device, model, piece):
    prompts = texts_of([1, 50, 131, 2], 6)
    with B.batch_invariant():
        scores = scoring.score_prompts(model, prompts, top=3, piece=piece)
        assert [s.logprobs.numel() for s in scores] == [0, 49, 130, 1] and scores[0].top_tokens.shape == (0, 3)
        with torch.no_grad():
            for s, text in zip(scores[1:], prompts[1:]):
                same(s, expected_scores(model, text, 1, 3))


@pytest.mark.parametrize("piece", [5, 2048])
def test_scores_of_continuations(cuda_device, model, piece):
    prompts, several = texts_of([40, 33, 1, 16], 7), [texts_of([6, 1, 30], 8), [], texts_of([17], 9), texts_of([2, 20], 10)]
    with B.batch_invariant():
        scores = scoring.score_continuations(model, prompts, several, top=2, piece=piece)
        assert [len(s) for s in scores] == [3, 0, 1, 2]
        with torch.no_grad():
            for prompt, own, texts in zip(prompts, scores, several):
                for s, text in zip(own, texts):
                    same(s, expected_scores(model, torch.cat([prompt, text]), prompt.numel(), 2))
    assert scoring.score_continuations(model, prompts[:1], [[]]) == [[]]
    for wrong in (lambda: scoring.score_continuations(model, prompts, several[:2]), lambda: scoring.score_prompts(model, []),
                  lambda: scoring.score_prompts(model, [torch.empty(0, dtype=torch.long)]),
                  lambda: scoring.score_continuations(model, prompts[:1], [[torch.empty(0, dtype=torch.long)]])):
        with pytest.raises(ValueError):
            wrong()


def test_log_probabilities_against_torch(cuda_device, model):
    text = texts_of([60], 11)[0]
    scores = scoring.score_prompts(model, [text])[0]
    cache = model.make_cache(1, 64)
    with torch.no_grad():
        logs = torch.log_softmax(model(text[None].to(cuda_device), cache=cache)[0].double(), -1)
    expected = logs[torch.arange(59), text[1:].to(cuda_device)]
    # Logits within the patched model's bound of 2e-2 of their largest: twice that between two of them.
    assert (scores.logprobs.double() - expected).abs().max() <= 4e-2 * float(model(text[None].to(cuda_device))[0].abs().max())
    assert np.isfinite(scores.entropy.cpu().numpy()).all()


def test_passes_of_nothing_are_refused(cuda_device, model):
    prompt = torch.tensor([3, 4, 5])
    for piece in (0, -3):
        with pytest.raises(ValueError, match="a token or more"):
            scoring.score_prompts(model, [prompt], piece=piece)
        with pytest.raises(ValueError, match="a token or more"):
            scoring.score_continuations(model, [prompt], [[prompt]], piece=piece)
