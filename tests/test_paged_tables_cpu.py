"""The host's side of a paged cache, blocks.PagedTables, with the oracle in place of the kernels: what is refused is refused
before anything has changed, and no page is given to two requests that write."""

import numpy as np
import pytest
import torch

from metile_b200 import backends
from metile_b200.integrations import blocks
from oracle import paged as O


@pytest.fixture
def oracle_backends(monkeypatch):
    def paged_resize(tables, lengths, counts, ring, state, *, page_size, tokens, advance):
        out = O.resize(tables.numpy(), lengths.numpy(), counts.numpy(), ring.numpy(), state.numpy(), page_size, tokens)
        assert advance
        for own, new in zip((lengths, state, tables, ring), out[3:]):
            own.copy_(torch.tensor(new))
        return torch.tensor(out[0]), torch.tensor(out[1]), torch.tensor(out[2]), lengths, state

    def beam_reorder(tables, lengths, parents, caches):
        if parents.shape[1] > backends.MAX_BEAMS:
            raise ValueError("beams")
        pages = [p for pair in caches for p in pair]
        out, moved = O.reorder(tables.numpy(), lengths.numpy(), parents.numpy(), [p.numpy() for p in pages], pages[0].shape[2])
        for own, new in zip(pages, moved):
            own.copy_(torch.tensor(new))
        return torch.tensor(out)

    monkeypatch.setattr(backends, "paged_resize", paged_resize)
    monkeypatch.setattr(backends, "beam_reorder", beam_reorder)


def cache_of(requests, pages=24, page_size=8, width=6):
    tables = blocks.PagedTables(requests, pages, page_size, width, "cpu")
    return tables, [blocks.PagedKVCache(tables, 1, 8, torch.float16)]


def state_of(tables):
    return (tables.held[:], tables.free, tables.lengths.tolist(), tables.block_tables.tolist(), tables.free_state.tolist(), tables.free_pages.tolist())


def test_a_fork_that_is_refused_changes_nothing(oracle_backends):
    tables, caches = cache_of(66, pages=200)
    tables.grow([13] + [0] * 32 + [11] + [0] * 32)
    before = state_of(tables)
    with pytest.raises(ValueError):
        tables.fork(33, caches)
    assert state_of(tables) == before
    other = cache_of(66)[1]
    for wrong in ([], other, [None]):
        with pytest.raises(ValueError):
            tables.fork(3, wrong)
        assert state_of(tables) == before
    tables, caches = cache_of(6)
    tables.grow([13, 0, 0, 8, 0, 0])
    tables.fork(3, caches)
    assert tables.held == tables.lengths.tolist() == [13, 13, 13, 8, 8, 8] and tables.free == int(tables.free_state[1]) == 24 - 2 - 1 - 2


def test_tokens_in_shared_pages_are_not_taken_back(oracle_backends):
    """After a fork or a reordering two requests name one page: given back by both it would be handed out twice, and
    reopened by one it would be written under the other."""
    tables, caches = cache_of(3)
    tables.grow([13, 0, 0])
    tables.fork(3, caches)
    tables.grow()
    for counts in ([-14, -14, -14], [0, -7, 0], [-6, -6, -7]):
        before = state_of(tables)
        with pytest.raises(ValueError, match="share"):
            tables.grow(counts)
        assert state_of(tables) == before
    tables.grow([-6, -2, 0])  # back to the full page, and within the page in work, which is a request's own
    assert tables.held == tables.lengths.tolist() == [8, 12, 14]
    tables.grow([1, 4, 2])
    table, held = tables.block_tables.numpy(), tables.held
    own = [int(table[r, j]) for r in range(3) for j in range(1, -(-held[r] // 8))]
    free = [int(tables.free_pages[(int(tables.free_state[0]) + i) % tables.pages]) for i in range(tables.free)]
    assert len(set(own)) == len(own) and not set(own) & set(free) and len(set(free)) == len(free) and table[0, 0] not in free
    tables.grow([7, 0, 0])
    tables.reorder(torch.tensor([[0, 0, 1]], dtype=torch.int32), caches)
    assert tables.shared == [16, 16, 16]
    with pytest.raises(ValueError, match="share"):
        tables.grow([0, -1, 0])
    tables.reset()
    tables.grow([9, 8, 1])
    tables.reorder(torch.zeros((3, 1), dtype=torch.int32), caches)  # one beam each shares nothing
    tables.grow([-9, -8, -1])
    assert tables.free == 24 and np.array_equal(sorted(tables.free_pages.tolist()), range(24))
