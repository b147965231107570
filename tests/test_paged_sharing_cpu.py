"""Shared pages and pieces of prompts without a GPU: the host's side of the tables with the oracle in place of the kernels, the
oracle itself, what is refused before anything runs, and how the attention's work is cut."""

import ctypes

import numpy as np
import pytest
import torch

from metile_b200 import _lib, backends as B
from metile_b200.integrations import blocks
from oracle import paged as O

from tests import helpers


@pytest.fixture
def oracle_backends(monkeypatch):
    def paged_resize(tables, lengths, counts, ring, state, *, page_size, tokens, advance):
        out = O.resize(tables.numpy(), lengths.numpy(), counts.numpy(), ring.numpy(), state.numpy(), page_size, tokens)
        for own, new in zip((lengths, state, tables, ring), out[3:]):
            own.copy_(torch.tensor(new))
        return torch.tensor(out[0]), torch.tensor(out[1]), torch.tensor(out[2]), lengths, state

    def pages_of(caches):
        return [p for pair in caches for p in pair]

    def write(tensors, arrays):
        for own, new in zip(tensors, arrays):
            own.copy_(torch.tensor(new))

    def paged_fork(tables, lengths, sources, counts, ring, state, shares, caches, *, advance):
        pages = pages_of(caches)
        out = O.fork(*(t.numpy() for t in (tables, lengths, sources, counts, ring, state, shares)), [p.numpy() for p in pages], pages[0].shape[2])
        write([tables, lengths, state, shares] + pages, list(out[:4]) + out[4])
        return lengths, state, shares

    def paged_free(tables, lengths, ended, ring, state, shares, *, page_size, advance):
        write((lengths, state, shares, ring), O.free(*(t.numpy() for t in (tables, lengths, ended, ring, state, shares)), page_size))
        return lengths, state, shares

    def paged_compact(tables, lengths, caches):
        pages = pages_of(caches)
        out = O.compact(tables.numpy(), lengths.numpy(), [p.numpy() for p in pages], pages[0].shape[2])
        write(pages, out[4])
        return tuple(torch.tensor(a) for a in out[:4])

    def beam_reorder(tables, lengths, parents, caches):
        pages = pages_of(caches)
        out, moved = O.reorder(tables.numpy(), lengths.numpy(), parents.numpy(), [p.numpy() for p in pages], pages[0].shape[2])
        write(pages, moved)
        return torch.tensor(out)

    for name, function in dict(locals()).items():
        if name.startswith(("paged_", "beam_")):
            monkeypatch.setattr(B, name, function)


def cache_of(requests, pages=40, page_size=8, width=10):
    tables = blocks.PagedTables(requests, pages, page_size, width, "cpu")
    return tables, [blocks.PagedKVCache(tables, 1, 8, torch.float16)]


def agrees(tables):
    assert tables.lengths.tolist() == tables.held and int(tables.free_state[1]) == tables.free
    held = {}
    for r, n in enumerate(tables.held):
        for page in tables.block_tables[r, :-(-n // tables.page_size)].tolist():
            held[page] = held.get(page, 0) + 1
    ring, (first, free) = tables.free_pages.tolist(), tables.free_state.tolist()
    free = [ring[(first + i) % len(ring)] for i in range(free)]
    assert not set(held) & set(free) and len(held) + len(set(free)) == tables.pages
    assert all(tables.shares[page] == held.get(page, 1) - 1 for page in range(tables.pages))


def test_the_host_knows_what_random_lives_of_requests_leave_free(oracle_backends):
    rng = np.random.default_rng(1)
    tables, caches = cache_of(9, pages=70)
    for _ in range(120):
        kind, empty, full = rng.integers(5), [r for r in range(9) if not tables.held[r]], [r for r in range(9) if tables.held[r]]
        before = tables.held[:], tables.free, tables.block_tables.tolist(), tables.shares.tolist()
        try:
            if kind == 0:
                tables.extend(rng.integers(0, 14, 9).tolist())
            elif kind == 1:
                tables.grow(rng.integers(-6, 5, 9).tolist())
            elif kind == 2 and full and empty:
                source = int(rng.choice(full))
                tables.branch([source if r in empty[:3] else None for r in range(9)], [int(rng.integers(1, tables.held[source] + 1))] * 9, caches)
            elif kind == 3:
                tables.release(rng.permutation(9)[:rng.integers(0, 4)].tolist())
            elif kind == 4 and rng.random() < 0.4:
                tables.compact(caches)
        except ValueError:  # refused: as it was
            assert (tables.held, tables.free, tables.block_tables.tolist(), tables.shares.tolist()) == before
        agrees(tables)
    tables.release(range(9))
    agrees(tables)
    assert tables.free == 70


def test_tokens_of_branches_are_their_own(oracle_backends):
    tables, caches = cache_of(3)
    tables.extend([20, 0, 0])
    caches[0].keys[tables.block_tables[0, :3].long()] = torch.arange(3, dtype=torch.float16)[:, None, None, None]
    tables.branch([None, 0, 0], [0, 20, 11], caches)
    agrees(tables)
    assert tables.held == [20, 20, 11] and tables.shared == [16, 16, 8]
    pages = tables.block_tables
    assert pages[0, :2].tolist() == pages[1, :2].tolist() and pages[0, 0] == pages[2, 0]
    assert len({int(pages[0, 2]), int(pages[1, 2]), int(pages[2, 1])}) == 3
    assert (caches[0].keys[pages[1, 2].long(), :, :4] == 2).all() and (caches[0].keys[pages[2, 1].long(), :, :3] == 1).all()
    for counts in ([-5, 0, 0], [0, 0, -4]):
        with pytest.raises(ValueError, match="share"):
            tables.grow(counts)
    tables.grow([-4, -4, -3])  # within what is their own
    agrees(tables)


def test_what_branch_release_and_extend_refuse(oracle_backends):
    tables, caches = cache_of(4, pages=6)
    tables.extend([17, 0, 9, 0])
    before = tables.held[:], tables.free, tables.shares.tolist()
    other = cache_of(4)[1]
    for sources, counts, given in (([None, 0, None, None], [0, 18, 0, 0], caches), ([None, 0, None, None], [0, 0, 0, 0], caches),
                                   ([None, 4, None, None], [0, 1, 0, 0], caches), ([None, None, 0, None], [0, 0, 1, 0], caches),
                                   ([None, 3, None, None], [0, 1, 0, 0], caches), ([None, 1, None, None], [0, 1, 0, 0], caches),
                                   ([None, 0], [0, 1], caches), ([None, 0, None, None], [0, 1, 0, 0], []),
                                   ([None, 0, None, None], [0, 1, 0, 0], other), ([None, 0, None, 0], [0, 9, 0, 9], caches)):
        with pytest.raises(ValueError):
            tables.branch(sources, counts, given)
        assert (tables.held, tables.free, tables.shares.tolist()) == before
    for requests in ([4], [-1], [0, 9]):
        with pytest.raises(ValueError):
            tables.release(requests)
    for counts in ([1, 1, 1], [-1, 0, 0, 0], [0, 90, 0, 0], [8, 8, 8, 8]):
        with pytest.raises(ValueError):
            tables.extend(counts)
    assert (tables.held, tables.free, tables.shares.tolist()) == before
    with pytest.raises(ValueError):
        tables.compact(other)
    tables.release([])
    tables.grow([0, 1, 0, 0])
    assert tables.starts is None
    tables.extend([0, 1, 0, 0])
    assert tables.starts.tolist() == [0, 0, 1, 1, 1]


def test_beams_are_counted_again_by_compact(oracle_backends):
    tables, caches = cache_of(4)
    tables.grow([19, 0, 0, 0])
    tables.fork(4, caches)
    for _ in range(9):
        tables.grow()
        tables.reorder(torch.tensor([[1, 1, 3, 1]], dtype=torch.int32), caches)
    with pytest.raises(ValueError, match="not counted"):
        tables.release([1])
    with pytest.raises(ValueError, match="not counted"):
        tables.branch([None] * 4, [0] * 4, caches)
    tables.compact(caches)
    agrees(tables)
    tables.release([1, 2])
    agrees(tables)
    tables.reset()
    agrees(tables)


# ---- refused without a GPU ----------------------------------------------------------------------------------------------


def test_operators_refuse_what_is_not_on_a_gpu():
    table, ints = torch.zeros((2, 3), dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    pages = torch.zeros((4, 1, 8, 64), dtype=torch.bfloat16)
    query, logits = torch.zeros((3, 2, 64), dtype=torch.bfloat16), torch.zeros((2, 10))
    for call in (lambda: B.paged_attention_chunk(query, pages, pages, table, ints, torch.zeros(3, dtype=torch.int32), scale=1.0),
                 lambda: B.paged_fork(table, ints, ints, ints, ints, ints, ints, [(pages, pages)]),
                 lambda: B.paged_free(table, ints, ints.bool(), ints, ints, ints, page_size=8), lambda: B.paged_compact(table, ints, [(pages, pages)]),
                 lambda: B.token_logprobs(logits, torch.zeros(2, dtype=torch.long), top=1)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    with pytest.raises(TypeError):
        B.token_logprobs([1.0], None)
    with pytest.raises(TypeError):
        B.paged_attention_chunk(None, pages, pages, table, ints, ints, scale=1.0)


def test_the_c_interface_refuses_before_any_gpu_work():
    lib = _lib.load()
    one = ctypes.c_void_p(64)
    strides = (ctypes.c_longlong * 3)(1024, 512, 64)
    odd = (ctypes.c_longlong * 3)(1024, 512, 63)
    arrays = (ctypes.c_void_p * 1)(64)

    def chunk(q=one, ks=strides, table_stride=4, width=4, out=one, rows=3, heads=4, kv_heads=2, dim=64, pages=9, page=16, type=0, requests=2):
        return lib.mt_paged_attention_chunk(q, one, ks, one, strides, one, table_stride, width, one, one, out, None, 0, rows, requests, heads, kv_heads,
                                            dim, pages, page, type, 1.0, 0, None)

    assert chunk(rows=0) == 0
    assert {chunk(rows=-1), chunk(heads=3), chunk(dim=96), chunk(page=12), chunk(width=5), chunk(type=2), chunk(pages=0), chunk(requests=-1),
            chunk(rows=1 << 30), chunk(width=1 << 28, table_stride=1 << 28)} == {-1}
    assert chunk(q=None) == chunk(out=None) == -6
    assert chunk(q=ctypes.c_void_p(72)) == chunk(out=ctypes.c_void_p(80)) == chunk(ks=odd) == -2

    def fork(width=4, stride=4, caches=1, keys=arrays, ks=strides, pool=5, requests=2, dim=64, page=16, workspace=one, state=one, size=64):
        return lib.mt_paged_fork(one, stride, width, one, one, one, one, pool, state, one, keys, ks, arrays, strides, caches, one, one, one,
                                 workspace, size, requests, 2, dim, 9, page, None)

    assert {fork(width=0), fork(stride=3), fork(caches=-1), fork(pool=0), fork(requests=-1), fork(dim=12), fork(page=7), fork(width=1 << 30, stride=1 << 30)} == {-1}
    assert fork(state=None) == fork(keys=None) == -6 and fork(ks=odd) == -2 and fork(workspace=None) == fork(size=4) == -7

    def free(width=4, requests=2, pages=9, page=16, pool=5, ended=one, size=10 ** 4):
        return lib.mt_paged_free(one, 4, width, one, ended, one, pool, one, one, one, one, one, one, size, requests, pages, page, None)

    assert {free(width=5), free(requests=-1), free(pages=0), free(page=9), free(pool=0)} == {-1} and free(ended=None) == -6 and free(size=8) == -7

    def compact(out=ctypes.c_void_p(128), size=10 ** 4, ks=strides, requests=2, dim=64):
        return lib.mt_paged_compact(one, 4, 4, one, out, one, one, one, arrays, ks, arrays, strides, 1, one, size, requests, 2, dim, 9, 16, None)

    assert compact(out=one) == compact(requests=-1) == compact(dim=4) == -1 and compact(out=None) == -6 and compact(ks=odd) == -2 and compact(size=8) == -7

    def logprobs(rows=2, vocab=10, top=1, type=0, stride=10, logits=one, size=10 ** 4, tops=one):
        return lib.mt_token_logprobs(logits, stride, type, one, one, one, tops, one, one, size, rows, vocab, top, None)

    assert logprobs(rows=0) == 0
    assert {logprobs(rows=-1), logprobs(vocab=0), logprobs(top=11), logprobs(top=-1), logprobs(type=3), logprobs(stride=-1), logprobs(vocab=1 << 20),
            logprobs(top=65, vocab=100)} == {-1}
    assert logprobs(tops=None) == -6 and logprobs(logits=ctypes.c_void_p(65)) == -2 and logprobs(size=8) == -7


# ---- how the attention's work is counted ----------------------------------------------------------------------------------


def test_the_work_of_blocks_adds_up(tmp_path):
    """chunk_work is the sum over blocks of what their last rows see and the cost of a unit, for every length, also below the rows."""
    cases = [(0, 1, 64), (5, 5, 64), (705, 5, 42), (100, 300, 64), (300, 300, 64), (63, 200, 50), (1, 130, 64), (15093, 4093, 64), (0, 500, 2), (7, 20, 6),
             (128, 128, 64), (2 ** 31 - 70000, 70000, 256)]
    lines = "".join(f"    check({length}, {n}, {unit});\n" for length, n, unit in cases)
    rows = helpers.host_program(str(tmp_path), '#include <cstdio>\n#include "../../include/metile_b200.h"\n#include "paged_chunk.cuh"\nusing namespace mt;\n'
                                "void check(int length, int n, int unit) {\n    long long sum = 0;\n    const int blocks = chunk_blocks(n, unit);\n"
                                "    for (int b = 0; b <= blocks; ++b) {\n        printf(\"%lld %lld\\n\", chunk_work(length, n, unit, b), sum);\n"
                                "        if (b < blocks) sum += chunk_seen(length, n, unit, b) + kChunkUnitCost;\n    }\n}\n"
                                f"int main() {{\n{lines}    return 0;\n}}\n")
    assert len(rows) > 200 and all(a == b for a, b in rows)
