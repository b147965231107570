"""GraphedBeamDecoder beyond short searches: what fails on the way to the captured step, sequences of several splits, the first
use in a process, and all tokens of a search with one beam."""

import os
import subprocess
import sys

import pytest
import torch

from metile_b200 import _lib, backends as B
from metile_b200.integrations import blocks
from metile_b200.integrations.graphed import GraphedBeamDecoder

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(autouse=True)
def nothing_was_recorded(cuda_device):
    yield
    ok, words = _lib.device_status()
    assert ok, [hex(w) for w in words]


@pytest.fixture(scope="module")
def model(cuda_device):
    return blocks.random_model(seed=5, device=cuda_device)


def prompts_of(lengths, device, seed=1):
    generator = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 512, (n,), generator=generator).to(device) for n in lengths]


def test_a_first_step_that_fails_leaves_the_decoder_as_it_was(cuda_device, model, monkeypatch):
    prompts = prompts_of([30, 9], cuda_device)
    with B.batch_invariant():
        expected = GraphedBeamDecoder(model, batch=2, beams=3, capacity=64).search(prompts, 12)
        decoder = GraphedBeamDecoder(model, batch=2, beams=3, capacity=64)
        decoder.prefill(prompts)
        tables, cache = decoder.tables, decoder.cache
        before = [t.clone() for t in (decoder.token, decoder.scores, decoder.parents, decoder.finished, tables.lengths, tables.free_state)]
        counts = (tables.held[:], tables.free, tables.shared[:])
        forward = type(model).forward
        for calls in (1, 2):  # in the step on the scratch cache, and inside the capture
            left = [calls]

            def failing(self, *args, **kwargs):
                left[0] -= 1
                if left[0] == 0:
                    raise RuntimeError("no step")
                return forward(self, *args, **kwargs)

            with monkeypatch.context() as patch:
                patch.setattr(type(model), "forward", failing)
                with pytest.raises(RuntimeError, match="no step"):
                    decoder.step()
            assert decoder.tables is tables and decoder.cache is cache and decoder.graph is None
            after = (decoder.token, decoder.scores, decoder.parents, decoder.finished, tables.lengths, tables.free_state)
            assert all(torch.equal(a, b) for a, b in zip(after, before))
            assert counts == (tables.held, tables.free, tables.shared)
        for _ in range(11):
            decoder.step()
        assert torch.equal(decoder.scores, expected[1]) and torch.equal(decoder.token.view(2, 3), expected[0][:, :, -1])
        again = decoder.search(prompts, 12)
    assert all(torch.equal(a, b) for a, b in zip(again, expected))


def test_a_first_step_without_room_is_refused_before_the_capture(cuda_device, model):
    decoder = GraphedBeamDecoder(model, batch=1, beams=2, capacity=32)
    decoder.prefill(prompts_of([32], cuda_device))
    held, free, token = decoder.tables.held[:], decoder.tables.free, decoder.token.clone()
    with pytest.raises(ValueError, match="no room"):
        decoder.step()
    assert decoder.graph is None and decoder.tables.held == held and decoder.tables.free == free and torch.equal(decoder.token, token)
    assert decoder.tables.lengths.tolist() == held
    for beams in (0, 33):
        with pytest.raises(ValueError):
            GraphedBeamDecoder(model, batch=1, beams=beams, capacity=32)


def eager_search(model, prompts, beams, steps, capacity, page_size=16):
    """The decoder's steps one by one without a graph, through the same tables."""
    rows, width = len(prompts) * beams, -(-capacity // page_size)
    cache = model.make_paged_cache(rows, rows * width, page_size, capacity)
    tables = cache[0].tables
    chosen, came_from = [], []
    with torch.no_grad():
        logits = []
        for g, prompt in enumerate(prompts):
            tables.grow([prompt.numel() if r == g * beams else 0 for r in range(rows)])
            logits.append(model(prompt[None], cache=cache)[:, -1])
        tables.fork(beams, cache)
        scores = torch.full((len(prompts), beams), -torch.inf, device=prompts[0].device)
        scores[:, 0] = 0.0
        logits = torch.cat(logits).repeat_interleave(beams, dim=0)
        for step in range(steps):
            scores, parents, tokens, _ = B.beam_select(logits, scores, keep=beams)
            if step:
                tables.reorder(parents, cache)
            chosen.append(tokens)
            came_from.append(parents.long())
            if step < steps - 1:
                tables.grow()
                logits = model(tokens.reshape(-1, 1), cache=cache)[:, -1]
    at = torch.arange(beams, device=scores.device).expand(len(prompts), -1)
    out = []
    for tokens, parents in zip(chosen[::-1], came_from[::-1]):
        out.append(torch.gather(tokens, 1, at))
        at = torch.gather(parents, 1, at)
    return torch.stack(out[::-1], dim=2), scores


@pytest.mark.parametrize("lengths,beams,steps", [([120], 4, 20), ([301, 7, 127], 3, 16), ([700], 2, 40), ([5, 130], 1, 30)])
def test_a_search_over_several_splits(cuda_device, model, lengths, beams, steps):
    """The default capacity, where the attention of a replayed step splits its sequences; with some that grow past a split's
    end on the way."""
    prompts = prompts_of(lengths, cuda_device, seed=sum(lengths))
    decoder = GraphedBeamDecoder(model, batch=len(lengths), beams=beams)
    assert decoder.tables.capacity == 4096
    with B.batch_invariant():
        tokens, scores = decoder.search(prompts, steps)
        expected, best = eager_search(model, prompts, beams, steps, 4096)
    assert torch.equal(tokens, expected) and torch.equal(scores, best)
    assert decoder.tables.lengths.tolist() == decoder.tables.held == [n + steps - 1 for n in lengths for _ in range(beams)]


def test_one_beam_is_greedy_decoding_token_by_token(cuda_device, model):
    prompts = prompts_of([12, 140], cuda_device, seed=8)
    decoder = GraphedBeamDecoder(model, batch=2, beams=1)
    with B.batch_invariant():
        tokens, _ = decoder.search(prompts, 25)
        cache = model.make_paged_cache(2, 64, 16, 4096)
        with torch.no_grad():
            cache[0].tables.grow([12, 140])
            logits = model(torch.cat(prompts)[None], cache=cache)[0, [11, 151]]
            greedy = [logits.argmax(-1)]
            for _ in range(24):
                cache[0].tables.grow()
                greedy.append(model(greedy[-1][:, None], cache=cache)[:, -1].argmax(-1))
    assert torch.equal(tokens[:, 0], torch.stack(greedy, 1))


FIRST_USE = """
import torch
from metile_b200 import _lib
from metile_b200.integrations import blocks
from metile_b200.integrations.graphed import GraphedBeamDecoder
model = blocks.random_model(seed=5, layers=1, device="cuda")
generator = torch.Generator().manual_seed(3)
prompts = [torch.randint(0, 512, (n,), generator=generator).cuda() for n in (300, 126)]
decoder = GraphedBeamDecoder(model, batch=2, beams=3)
launches = []
step = decoder._step
def watched():
    launches.append((decoder.tables.width, torch.cuda.is_current_stream_capturing()))
    step()
decoder._step = watched
tokens, scores = decoder.search(prompts, 8)
again = decoder.search(prompts, 8)
assert torch.equal(tokens, again[0]) and torch.equal(scores, again[1]) and bool(torch.isfinite(scores).all())
# The step before the capture goes through tables as wide as the captured one's, and so through the same launches.
assert launches == [(256, False), (256, True)], launches
assert _lib.device_status()[0]
print("searched")
"""


def test_the_first_use_of_a_process_over_several_splits(cuda_device):
    run = subprocess.run([sys.executable, "-c", FIRST_USE], capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert run.returncode == 0 and "searched" in run.stdout, run.stdout[-2000:] + run.stderr[-2000:]
