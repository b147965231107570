"""GraphedBeamDecoder beyond short searches: what fails on the way to the captured step, sequences of several splits, the first
use in a process, and all tokens of a search with one beam."""

import pytest
import torch

from metile_b200 import _lib, backends as B
from metile_b200.integrations import blocks
from metile_b200.integrations.graphed import GraphedBeamDecoder

pytestmark = pytest.mark.gpu


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
