"""The paged cache and beam search as a model uses them: prompts of different lengths, decode steps eager, patched and as
a captured graph, requests that come and go, beams that share pages."""

import numpy as np
import pytest
import torch

from metile_b200 import _lib, backends as B
from metile_b200.integrations import blocks
from metile_b200.integrations.graphed import GraphedBeamDecoder, GraphedDecoder
from metile_b200.integrations.torch_lm import apply_metile_to_torch_lm
from oracle import paged as O

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


def paged_steps(model, prompts, steps, page_size=16, pages=64, order=None):
    """Logits of every prompt's last position and of `steps` greedy tokens, [steps + 1, requests, vocabulary]."""
    cache = model.make_paged_cache(len(prompts), pages, page_size, 256)
    tables = cache[0].tables
    if order is not None:
        tables.free_pages.copy_(order)
    out = []
    with torch.no_grad(), B.batch_invariant():
        tables.grow([p.numel() for p in prompts])
        logits = model(torch.cat(prompts)[None], cache=cache)
        ends = torch.tensor([p.numel() for p in prompts]).cumsum(0) - 1
        out.append(logits[0, ends.to(logits.device)])
        for _ in range(steps):
            tables.grow()
            out.append(model(out[-1].argmax(-1)[:, None], cache=cache)[:, -1])
    assert tables.lengths.tolist() == tables.held == [p.numel() + steps for p in prompts]
    assert int(tables.free_state[1]) == tables.free
    return torch.stack(out)


def test_requests_together_alone_and_in_other_pages_have_the_same_bits(cuda_device, model):
    prompts = prompts_of([1, 40, 16, 130], cuda_device)
    together = paged_steps(model, prompts, 20)
    for index, prompt in enumerate(prompts):
        assert torch.equal(paged_steps(model, [prompt], 20)[:, 0], together[:, index]), index
    shuffled = torch.randperm(64, generator=torch.Generator().manual_seed(2)).to(torch.int32).to(cuda_device)
    assert torch.equal(paged_steps(model, prompts, 20, order=shuffled), together)
    assert torch.equal(paged_steps(model, prompts, 20, page_size=64, pages=20), together)


def test_the_paged_cache_against_the_contiguous_one(cuda_device, model):
    prompt = prompts_of([33], cuda_device, seed=3)[0]
    paged = paged_steps(model, [prompt], 1)
    cache = model.make_cache(1, 64)
    with torch.no_grad(), B.batch_invariant():
        plain = model(prompt[None], cache=cache)[:, -1]
        after = model(plain.argmax(-1)[:, None], cache=cache)[:, -1]
    # The angles differ (64 bits here, products of 32 bits there) and with them roundings to bf16: the bound the patched
    # model is held to against the module by module form.
    for a, b in ((paged[0], plain), (paged[1], after)):
        assert (a - b).float().abs().max() <= 2e-2 * b.float().abs().max()


def test_a_patched_step_is_the_eager_one(cuda_device, model):
    prompts = prompts_of([20, 7], cuda_device, seed=4)

    def run():
        cache = model.make_paged_cache(2, 32, 16, 128)
        with torch.no_grad(), B.batch_invariant():
            cache[0].tables.grow([20, 7])
            model(torch.cat(prompts)[None], cache=cache)
            before = [(c.keys.clone(), c.values.clone()) for c in cache]
            cache[0].tables.grow()
            logits = model(torch.tensor([[3], [4]], device=cuda_device), cache=cache)[:, -1]
        return logits, before, cache

    plain, _, _ = run()
    with apply_metile_to_torch_lm(model, attention=True) as patch:
        patched, _, _ = run()
        assert not patch.refusals, patch.refusals
    assert (plain - patched).float().abs().max() <= 2e-2 * plain.float().abs().max()


def test_requests_come_and_go_in_a_pool_that_is_just_large_enough(cuda_device, model):
    prompts = prompts_of([30, 50, 17, 64, 5], cuda_device, seed=5)
    alone = [paged_steps(model, [p], 6)[:, 0] for p in prompts]
    cache = model.make_paged_cache(2, 9, 16, 128)
    tables = cache[0].tables
    with torch.no_grad(), B.batch_invariant():
        for first, second in ((0, 1), (2, 3), (4, 0)):
            counts = [prompts[first].numel(), prompts[second].numel()]
            tables.grow(counts)
            logits = model(torch.cat([prompts[first], prompts[second]])[None], cache=cache)
            last = torch.stack([logits[0, counts[0] - 1], logits[0, -1]])
            for step in range(6):
                assert torch.equal(last[0], alone[first][step]) and torch.equal(last[1], alone[second][step])
                tables.grow()
                last = model(last.argmax(-1)[:, None], cache=cache)[:, -1]
            tables.grow([-held for held in tables.held])
            assert tables.free == 9 and tables.free_state.tolist()[1] == 9 and tables.lengths.tolist() == [0, 0]
        with pytest.raises(ValueError, match="out of pages"):
            tables.grow([128, 17])
        with pytest.raises(ValueError, match="no room"):
            tables.grow([129, 0])
        tables.grow([3, 2])
        with pytest.raises(ValueError, match="tokens that its tables grew by"):
            model(torch.zeros((1, 4), dtype=torch.long, device=cuda_device), cache=cache)
        model(torch.zeros((1, 5), dtype=torch.long, device=cuda_device), cache=cache)
        tables.grow([2, 0])
        with pytest.raises(ValueError, match="continuation"):
            model(torch.zeros((1, 2), dtype=torch.long, device=cuda_device), cache=cache)


def search_with_pages_of_their_own(model, prompts, beams, steps, end, capacity, page_size):
    """Beam search with the oracle's selection, every beam's pages its own and copied whole, step by step."""
    width = -(-capacity // page_size)
    rows = len(prompts) * beams
    cache = model.make_paged_cache(rows, rows * width, page_size, capacity)
    tables = cache[0].tables
    with torch.no_grad():
        repeated = [p for p in prompts for _ in range(beams)]
        tables.grow([p.numel() for p in repeated])
        packed = torch.cat(repeated)[None]
        ends = torch.tensor([p.numel() for p in repeated]).cumsum(0) - 1
        logits = model(packed, cache=cache)[0, ends.to(packed.device)]
        scores = np.full((len(prompts), beams), -np.inf)
        scores[:, 0] = 0.0
        finished = np.zeros((len(prompts), beams), bool)
        chosen = [[[] for _ in range(beams)] for _ in prompts]
        for step in range(steps):
            scores, parents, tokens, finished = O.beam_select(logits.detach().cpu().double().numpy(), scores, beams, finished if end >= 0 else None, end)
            scores = scores.astype(np.float32).astype(np.float64)
            chosen = [[chosen[g][parents[g, k]] + [int(tokens[g, k])] for k in range(beams)] for g in range(len(prompts))]
            if step == steps - 1:
                break
            source = torch.tensor([g * beams + parents[g, k] for g in range(len(prompts)) for k in range(beams)])
            table = tables.block_tables.cpu()
            for layer in cache:
                for pages in (layer.keys, layer.values):
                    held = pages.clone()
                    for row in range(rows):
                        blocks_held = -(-tables.held[row] // page_size)
                        pages[table[row, :blocks_held].long().to(pages.device)] = held[table[source[row], :blocks_held].long().to(pages.device)]
            tables.grow()
            logits = model(torch.tensor(tokens.reshape(-1, 1), device=packed.device), cache=cache)[:, -1]
    return np.array(chosen), scores


@pytest.mark.parametrize("lengths,beams,page_size,end,patched", [
    ([21], 4, 16, None, False), ([16, 37, 5], 3, 8, None, False), ([30, 31], 5, 16, 7, True), ([9, 70], 1, 32, None, True),
])
def test_beam_search_against_one_that_shares_nothing(cuda_device, model, lengths, beams, page_size, end, patched):
    prompts = prompts_of(lengths, cuda_device, seed=6)
    steps, capacity = 24, 128

    def both():
        decoder = GraphedBeamDecoder(model, batch=len(lengths), beams=beams, capacity=capacity, page_size=page_size, end_token=end)
        with B.batch_invariant():
            tokens, scores = decoder.search(prompts, steps)
            again, _ = decoder.search(prompts, steps)      # the captured step serves the next prompts too
            expected, best = search_with_pages_of_their_own(model, prompts, beams, steps, -1 if end is None else end, capacity, page_size)
        assert torch.equal(tokens, again)
        assert decoder.tables.lengths.tolist() == decoder.tables.held == [n + steps - 1 for n in lengths for _ in range(beams)]
        assert int(decoder.tables.free_state[1]) == decoder.tables.free
        return tokens, scores, expected, best

    if patched:
        with apply_metile_to_torch_lm(model, attention=True):
            tokens, scores, expected, best = both()
    else:
        tokens, scores, expected, best = both()
    assert np.array_equal(tokens.cpu().numpy(), expected)
    # A score is rounded to 32 bits at every step, and so may differ by a step of 2^-23 of itself at each.
    assert (np.abs(scores.cpu().double().numpy() - best) <= steps * (2.0 ** -23 * np.abs(best) + 2.0 ** -20)).all()
    if end is not None:
        for row in tokens.reshape(-1, steps).tolist():
            if end in row:
                assert set(row[row.index(end):]) == {end}


def test_two_searches_side_by_side(cuda_device, model):
    """Two decoders whose captured steps run on streams of their own, at the same time."""
    decoders = [GraphedBeamDecoder(model, batch=2, beams=4, capacity=96, page_size=8) for _ in range(2)]
    prompts = [prompts_of([11, 24], cuda_device, seed=11 + i) for i in range(2)]
    with B.batch_invariant():
        apart = [decoder.search(p, 30) for decoder, p in zip(decoders, prompts)]
        streams = [torch.cuda.Stream(cuda_device) for _ in decoders]
        for stream in streams:
            stream.wait_stream(torch.cuda.current_stream())
        for decoder, p, stream in zip(decoders, prompts, streams):
            with torch.cuda.stream(stream):
                decoder.prefill(p)
        for _ in range(29):
            for decoder, stream in zip(decoders, streams):
                with torch.cuda.stream(stream):
                    decoder.step()
        for stream in streams:
            torch.cuda.current_stream().wait_stream(stream)
    for decoder, (found, scores) in zip(decoders, apart):
        assert torch.equal(decoder.scores, scores) and torch.equal(decoder.token.view(2, 4), found[:, :, -1])


def test_one_beam_is_greedy_decoding(cuda_device, model):
    prompts = prompts_of([12, 12], cuda_device, seed=8)
    decoder = GraphedBeamDecoder(model, batch=2, beams=1, capacity=64)
    greedy = GraphedDecoder(model, batch=2, capacity=64)
    with apply_metile_to_torch_lm(model, attention=True), B.batch_invariant():
        tokens, _ = decoder.search(prompts, 5)
        first = greedy.prefill(torch.stack(prompts)).argmax(-1)
        assert torch.equal(tokens[:, 0, 0], first)


def test_a_search_beyond_the_cache_is_refused(cuda_device, model):
    prompts = prompts_of([20], cuda_device, seed=9)
    decoder = GraphedBeamDecoder(model, batch=1, beams=2, capacity=32)
    with pytest.raises(ValueError, match="no room"):
        decoder.search(prompts, 20)
    decoder.search(prompts, 13)
    small = GraphedBeamDecoder(model, batch=1, beams=2, capacity=64, pages=4)
    with pytest.raises(ValueError, match="out of pages"):
        small.search(prompts, 40)
    with pytest.raises(ValueError):
        small.prefill(prompts * 2)
    with pytest.raises(ValueError):
        small.search(prompts, 0)
