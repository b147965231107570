"""Forking, freeing and compacting the pages of a cache against the oracle: whole numbers and copies, equal to the bit."""

import numpy as np
import pytest
import torch

from metile_b200 import _lib, backends as B
from oracle import paged as O

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def nothing_was_recorded(cuda_device):
    yield
    ok, words = _lib.device_status()
    assert ok, [hex(w) for w in words]


def on(array, device):
    return torch.tensor(array, device=device)


def caches_of(seed, layers, pages, heads, page, dim, dtype, device, layout="head"):
    generator = torch.Generator().manual_seed(seed)

    def one():
        if layout == "token":
            return torch.randn((pages, page, heads, dim), generator=generator).to(dtype).to(device).transpose(1, 2)
        return torch.randn((pages, heads, page, dim), generator=generator).to(dtype).to(device)

    return [(one(), one()) for _ in range(layers)]


def host(caches):
    return [t.detach().cpu().view(torch.int16).numpy().copy() if t.is_contiguous() else t.contiguous().cpu().view(torch.int16).numpy().copy()
            for pair in caches for t in pair]


def shared_state(seed, groups, members, page, prompt, more, slack, ring=None):
    """Groups whose members share the full pages of a prompt, rows and ids in no order; (tables, lengths, ring, state, shares)."""
    rng = np.random.default_rng(seed)
    rows, shares, at = [], [], 0
    for _ in range(groups):
        tokens = int(rng.integers(1, prompt + 1))
        whole = tokens // page
        common = list(range(at, at + whole))
        at += whole
        shares += [members - 1] * whole
        for _ in range(members):
            n = tokens + int(rng.integers(0, more + 1))
            own = -(-n // page) - whole
            rows.append((n, common + list(range(at, at + own))))
            shares += [0] * own
            at += own
    rng.shuffle(rows)
    pool = at + slack
    names = rng.permutation(pool).astype(np.int32)
    tables = np.full((len(rows), max(len(ids) for _, ids in rows) + 2), -1, np.int32)
    for r, (_, ids) in enumerate(rows):
        tables[r, :len(ids)] = names[ids]
    counted = np.zeros(pool, np.int32)
    counted[names[:at]] = shares
    entries = pool if ring is None else ring
    start = int(rng.integers(entries))
    free = np.full(entries, -7, np.int32)
    free[(start + np.arange(slack)) % entries] = names[at:]
    return tables, np.array([n for n, _ in rows], np.int32), free, np.array([start, slack], np.int32), counted


# ---- fork ---------------------------------------------------------------------------------------------------------


def check_fork(device, arrays, caches):
    tables, lengths, sources, counts, ring, state, shares = arrays
    page = caches[0][0].shape[2]
    expected = O.fork(*arrays, host(caches), page)
    first = [on(a, device) for a in arrays]
    for _ in range(2):  # the same again
        got = B.paged_fork(*first, caches)
        for name, a, b in zip(("tables", "lengths", "state", "shares"), (first[0], *got), expected):
            assert np.array_equal(a.cpu().numpy(), b), name
        for a, b in zip(host(caches), expected[4]):
            assert np.array_equal(a, b)
    for a, b in zip(first[1:], arrays[1:]):
        assert np.array_equal(a.cpu().numpy(), b)
    second = [on(a, device) for a in arrays]
    got = B.paged_fork(*second, caches, advance=True)
    assert [t.data_ptr() for t in got] == [second[i].data_ptr() for i in (1, 5, 6)]
    for name, a, b in zip(("tables", "lengths", "state", "shares"), (second[0], *got), expected):
        assert np.array_equal(a.cpu().numpy(), b), name


def fork_case(seed, groups, children, page, prompt, free, width_slack=2):
    rng = np.random.default_rng(seed)
    held = rng.integers(1, prompt + 1, groups)
    rows = []  # (tokens, group, count)
    for g in range(groups):
        rows.append((int(held[g]), g, 0))
        rows += [(0, g, int(rng.integers(1, held[g] + 1)) if c % 2 else int(held[g])) for c in range(children)]
    rng.shuffle(rows)
    owner = {g: r for r, (n, g, _) in enumerate(rows) if n}
    blocks = [-(-n // page) for n, _, _ in rows]
    pool = sum(blocks) + free
    names = rng.permutation(pool).astype(np.int32)
    tables = np.full((len(rows), max(blocks) + width_slack), -1, np.int32)
    at = 0
    for r, count in enumerate(blocks):
        tables[r, :count] = names[at:at + count]
        at += count
    start = int(rng.integers(pool))
    ring = np.full(pool, -7, np.int32)
    ring[(start + np.arange(free)) % pool] = names[at:]
    return [tables, np.array([n for n, _, _ in rows], np.int32), np.array([-1 if n else owner[g] for n, g, _ in rows], np.int32),
            np.array([c for _, _, c in rows], np.int32), ring, np.array([start, free], np.int32), np.zeros(pool, np.int32)]


@pytest.mark.parametrize("groups,children,page,prompt,free,layers,heads,dim,dtype,layout", [
    (1, 1, 8, 5, 1, 1, 1, 8, torch.bfloat16, "head"), (1, 4, 16, 500, 9, 4, 2, 128, torch.bfloat16, "head"),
    (3, 5, 32, 100, 40, 2, 3, 64, torch.float16, "token"), (40, 7, 8, 90, 300, 1, 1, 16, torch.bfloat16, "head"),
    (2, 3, 256, 700, 8, 70, 1, 8, torch.bfloat16, "head"), (300, 5, 8, 20, 1600, 1, 1, 8, torch.float16, "head"),
    (2, 2, 64, 100, 5, 1, 2, 4096, torch.bfloat16, "head"),
])
def test_requests_go_on_from_others(cuda_device, groups, children, page, prompt, free, layers, heads, dim, dtype, layout):
    arrays = fork_case(groups + children, groups, children, page, prompt, free)
    check_fork(cuda_device, arrays, caches_of(groups, layers, len(arrays[6]), heads, page, dim, dtype, cuda_device, layout))


@pytest.mark.parametrize("free", [0, 1, 7])
def test_free_pages_do_not_reach(cuda_device, free):
    arrays = fork_case(free, 6, 5, 8, 50, free)
    check_fork(cuda_device, arrays, caches_of(1, 1, len(arrays[6]), 2, 8, 16, torch.bfloat16, cuda_device))


def test_forks_that_make_no_sense_change_nothing(cuda_device):
    arrays = fork_case(3, 4, 4, 16, 60, 40)
    lengths, sources, counts = arrays[1], arrays[2], arrays[3]
    empty = [r for r in range(20) if lengths[r] == 0]
    sources[empty[0]], sources[empty[1]], sources[empty[2]], sources[empty[3]] = 20, -5, empty[3], empty[3]
    counts[empty[4]], counts[empty[5]], counts[empty[6]] = 0, -3, 61
    sources[empty[7]] = empty[8]                                     # a source without tokens
    full = [r for r in range(20) if lengths[r]]
    sources[full[0]], counts[full[0]] = full[1], 1                   # a request that has tokens
    lengths[full[2]] = arrays[0].shape[1] * 16 + 1                   # a length its row has no room for
    check_fork(cuda_device, arrays, caches_of(1, 2, len(arrays[6]), 1, 16, 16, torch.float16, cuda_device))


def test_a_page_outside_is_recorded(cuda_device):
    arrays = fork_case(9, 1, 1, 8, 1, 3)
    arrays[1][arrays[1] > 0] = 20
    child, source = int(np.argmin(arrays[1])), int(np.argmax(arrays[1]))
    arrays[0] = np.full((2, 5), -1, np.int32)
    arrays[0][source, :3] = [0, 10 ** 6, 1]
    arrays[3][child] = 20
    caches = caches_of(1, 1, len(arrays[6]), 1, 8, 16, torch.bfloat16, cuda_device)
    tensors = [on(a, cuda_device) for a in arrays]
    got = B.paged_fork(*tensors, caches)
    ok, words = _lib.device_status()
    assert not ok and words[0] == 0x303 and words[1] == child and words[2] == 10 ** 6
    assert got[0].tolist() == [20, 20] and got[2].tolist() == [1] + [0] * (len(arrays[6]) - 1)


# ---- free ---------------------------------------------------------------------------------------------------------


def check_free(device, arrays, page):
    tables, lengths, ended, ring, state, shares = arrays
    expected = O.free(*arrays, page)
    first = [on(a, device) for a in arrays]
    for _ in range(2):
        got = B.paged_free(*first, page_size=page)
        for name, a, b in zip(("lengths", "state", "shares", "ring"), (*got, first[3]), expected):
            assert np.array_equal(a.cpu().numpy(), b), name
    for i in (0, 1, 2, 4, 5):
        assert np.array_equal(first[i].cpu().numpy(), arrays[i])
    second = [on(a, device) for a in arrays]
    got = B.paged_free(*second, page_size=page, advance=True)
    assert [t.data_ptr() for t in got] == [second[i].data_ptr() for i in (1, 4, 5)]
    for name, a, b in zip(("lengths", "state", "shares", "ring"), (*got, second[3]), expected):
        assert np.array_equal(a.cpu().numpy(), b), name
    return expected


@pytest.mark.parametrize("groups,members,page,prompt,more,share", [
    (1, 1, 8, 5, 0, 1.0), (1, 5, 16, 300, 200, 0.4), (3, 4, 32, 100, 7, 0.0), (50, 10, 16, 700, 300, 0.5), (1, 2, 16, 100000, 3000, 1.0),
    (700, 2, 8, 40, 20, 0.7), (2, 900, 8, 30, 9, 1.0), (40, 30, 8, 900, 300, 0.6),
])
def test_requests_end(cuda_device, groups, members, page, prompt, more, share):
    tables, lengths, ring, state, shares = shared_state(groups, groups, members, page, prompt, more, 11)
    ended = np.random.default_rng(members).random(len(lengths)) < share
    check_free(cuda_device, [tables, lengths, ended, ring, state, shares], page)


def test_the_last_holder_gives_the_page_back(cuda_device):
    tables, lengths, ring, state, shares = shared_state(5, 2, 6, 8, 90, 30, 4)
    before = int(state[1])
    for ended in np.array_split(np.random.default_rng(1).permutation(12), 5):
        flags = np.zeros(12, bool)
        flags[ended] = True
        lengths, state, shares, ring = check_free(cuda_device, [tables, lengths, flags, ring, state, shares], 8)
    assert state[1] == len(shares) > before and not shares.any() and not lengths.any()
    assert sorted(ring) == list(range(len(shares)))


def test_lengths_and_pages_that_make_no_sense(cuda_device):
    tables, lengths, ring, state, shares = shared_state(6, 1, 3, 8, 40, 9, 4)
    lengths[0], ended = tables.shape[1] * 8 + 1, np.array([True, True, False])
    check_free(cuda_device, [tables, lengths, ended, ring, state, shares], 8)
    lengths[0] = -4
    check_free(cuda_device, [tables, lengths, ended, ring, state, shares], 8)
    tables[1, 0] = 999
    B.paged_free(*[on(a, cuda_device) for a in (tables, lengths, ended, ring, state, shares)], page_size=8)
    ok, words = _lib.device_status()
    assert not ok and words[0] == 0x303 and words[1] == 1 and words[2] == 999


# ---- compact ------------------------------------------------------------------------------------------------------


def check_compact(device, tables, lengths, caches):
    page = caches[0][0].shape[2]
    expected = O.compact(tables, lengths, host(caches), page)
    table, held = on(tables, device), on(lengths, device)
    for _ in range(2):
        got = B.paged_compact(table, held, caches)
        for name, a, b in zip(("tables", "ring", "state", "shares"), got, expected):
            assert np.array_equal(a.cpu().numpy(), b), name
        for a, b in zip(host(caches), expected[4]):
            assert np.array_equal(a, b)
    assert np.array_equal(table.cpu().numpy(), tables) and np.array_equal(held.cpu().numpy(), lengths)
    return expected


@pytest.mark.parametrize("groups,members,page,prompt,more,slack,layers,heads,dim,dtype,layout", [
    (1, 1, 8, 5, 0, 0, 1, 1, 8, torch.bfloat16, "head"), (1, 1, 8, 5, 0, 3, 1, 1, 8, torch.bfloat16, "head"),
    (2, 4, 16, 200, 150, 90, 4, 2, 128, torch.bfloat16, "head"), (5, 3, 32, 300, 100, 20, 2, 3, 64, torch.float16, "token"),
    (30, 3, 8, 200, 60, 900, 1, 1, 16, torch.bfloat16, "head"), (1, 2, 8, 3000, 20000, 70000, 1, 1, 8, torch.bfloat16, "head"),
    (300, 2, 8, 30, 10, 500, 1, 1, 8, torch.float16, "head"), (2, 2, 64, 300, 10, 12, 67, 1, 8, torch.bfloat16, "head"),
])
def test_held_pages_move_to_the_lowest_ids(cuda_device, groups, members, page, prompt, more, slack, layers, heads, dim, dtype, layout):
    tables, lengths, _, _, shares = shared_state(groups, groups, members, page, prompt, more, slack)
    caches = caches_of(groups, layers, len(shares), heads, page, dim, dtype, cuda_device, layout)
    out = check_compact(cuda_device, tables, lengths, caches)
    assert np.array_equal(np.sort(out[3]), np.sort(shares))
    check_compact(cuda_device, out[0], lengths, caches)  # and now nothing moves


def test_nothing_held_and_pages_that_nobody_holds(cuda_device):
    tables, lengths, _, _, shares = shared_state(8, 2, 3, 8, 50, 20, 9)
    caches = caches_of(8, 1, len(shares), 1, 8, 16, torch.bfloat16, cuda_device)
    lengths[::2] = 0
    check_compact(cuda_device, tables, lengths, caches)
    out = check_compact(cuda_device, tables, np.zeros_like(lengths), caches)
    assert out[2].tolist() == [0, len(shares)] and out[1].tolist() == list(range(len(shares)))
    none = np.zeros((0, 3), np.int32)
    check_compact(cuda_device, none, np.zeros(0, np.int32), caches)


def test_entries_outside_are_recorded(cuda_device):
    tables, lengths, _, _, shares = shared_state(9, 1, 2, 8, 50, 20, 9)
    caches = caches_of(9, 1, len(shares), 1, 8, 16, torch.bfloat16, cuda_device)
    tables[1, 0] = -3
    B.paged_compact(on(tables, cuda_device), on(lengths, cuda_device), caches)
    ok, words = _lib.device_status()
    assert not ok and words[0] == 0x303 and words[1] == 1
    lengths[0] = 10 ** 6
    tables[1, 0] = 0
    got = B.paged_compact(on(tables, cuda_device), on(lengths, cuda_device), caches)
    ok, words = _lib.device_status()
    assert not ok and words[0] == 0x304 and words[1] == 0 and words[2] == 10 ** 6
    assert np.array_equal(got[0][0].cpu().numpy(), tables[0])


# ---- all three ----------------------------------------------------------------------------------------------------


def test_a_life_of_requests(cuda_device):
    """Requests grow, are forked, grow on, end and are put together, in place and against the oracle at every step."""
    page, requests, width, pages = 8, 9, 12, 60
    rng = np.random.default_rng(12)
    caches = caches_of(12, 2, pages, 2, page, 16, torch.bfloat16, cuda_device)
    tables, lengths = np.full((requests, width), -1, np.int32), np.zeros(requests, np.int32)
    ring, state, shares = rng.permutation(pages).astype(np.int32), np.array([41, pages], np.int32), np.zeros(pages, np.int32)
    mine = [on(a, cuda_device) for a in (tables, lengths, ring, state, shares)]
    own = host(caches)

    def same():
        for name, a, b in zip(("tables", "lengths", "ring", "state", "shares"), mine, (tables, lengths, ring, state, shares)):
            assert np.array_equal(a.cpu().numpy(), b), name
        for a, b in zip(host(caches), own):
            assert np.array_equal(a, b)
        held = {int(tables[r, j]) for r in range(requests) for j in range(-(-int(lengths[r]) // page))}
        free = [int(ring[(state[0] + i) % pages]) for i in range(int(state[1]))]
        assert not held & set(free) and len(set(free)) == len(free) and len(held) + len(free) == pages

    for step in range(12):
        counts = np.where(lengths > 0, rng.integers(0, 9, requests), 0).astype(np.int32)
        counts[step % requests] += 13 if lengths[step % requests] == 0 else 0
        total = int(counts.sum())
        out = O.resize(tables, lengths, counts, ring, state, page, total)
        B.paged_resize(mine[0], mine[1], on(counts, cuda_device), mine[2], mine[3], page_size=page, tokens=total, advance=True)
        lengths, state, tables, ring = out[3:]
        same()
        sources, counts = np.full(requests, -1, np.int32), np.zeros(requests, np.int32)
        for r in np.flatnonzero(lengths == 0)[:2]:
            sources[r] = rng.choice(np.flatnonzero(lengths > 0))
            counts[r] = rng.integers(1, lengths[sources[r]] + 1)
        tables, lengths, state, shares, own = O.fork(tables, lengths, sources, counts, ring, state, shares, own, page)
        B.paged_fork(mine[0], mine[1], on(sources, cuda_device), on(counts, cuda_device), mine[2], mine[3], mine[4], caches, advance=True)
        same()
        ended = rng.random(requests) < 0.3
        lengths, state, shares, ring = O.free(tables, lengths, ended, ring, state, shares, page)
        B.paged_free(mine[0], mine[1], on(ended, cuda_device), mine[2], mine[3], mine[4], page_size=page, advance=True)
        same()
        if step % 4 == 3:
            tables, ring, state, shares, own = O.compact(tables, lengths, own, page)
            out = B.paged_compact(mine[0], mine[1], caches)
            mine = [out[0], mine[1], out[1], out[2], out[3]]
            same()


def test_captured_calls(cuda_device):
    """A fork and the end of what it made, replayed from one state."""
    arrays = fork_case(30, 3, 3, 8, 60, 30)
    caches = caches_of(30, 2, len(arrays[6]), 1, 8, 16, torch.bfloat16, cuda_device)
    tensors = [on(a, cuda_device) for a in arrays]
    ended = on(arrays[1] == 0, cuda_device)

    def both():
        lengths, state, shares = B.paged_fork(*tensors, caches)
        return B.paged_free(tensors[0], lengths, ended, tensors[4], state, shares, page_size=8), lengths

    both()
    stream, graph = torch.cuda.Stream(cuda_device), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        (lengths, state, shares), between = both()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert np.array_equal(between.cpu().numpy(), O.fork(*arrays, [], 8)[1])
    assert np.array_equal(lengths.cpu().numpy(), arrays[1]) and not shares.any() and int(state[1]) == 30


def test_refusals(cuda_device):
    arrays = fork_case(31, 2, 2, 8, 40, 10)
    caches = caches_of(31, 2, len(arrays[6]), 1, 8, 16, torch.bfloat16, cuda_device)
    good = [on(a, cuda_device) for a in arrays]

    def spoiled(index, value):
        return [value if i == index else t for i, t in enumerate(good)]

    for index in range(7):
        for value, error in ((good[index].long(), (TypeError, ValueError)), (good[index].cpu(), ValueError), (good[index][:0], ValueError)):
            with pytest.raises(error):
                B.paged_fork(*spoiled(index, value), caches)
    for wrong in ([], [(caches[0][0],)], [caches[0], (caches[1][0], caches[1][1][:2])], [(caches[0][0].float(), caches[0][1].float())],
                  [(caches[0][0].cpu(), caches[0][1].cpu())]):
        with pytest.raises((TypeError, ValueError)):
            B.paged_fork(*good, wrong)
        with pytest.raises((TypeError, ValueError)):
            B.paged_compact(good[0], good[1], wrong)
    wants = [(caches[0][0].clone().requires_grad_(), caches[0][1])]
    with pytest.raises(ValueError, match="gradient"):
        B.paged_fork(*good, wants)
    with pytest.raises(ValueError, match="gradient"):
        B.paged_compact(good[0], good[1], wants)
    ended = good[1] == 0
    free = [good[0], good[1], ended, good[4], good[5], good[6]]
    for index in range(6):
        for value in (free[index].float(), free[index].cpu(), free[index][:0]):
            with pytest.raises((TypeError, ValueError)):
                B.paged_free(*[value if i == index else t for i, t in enumerate(free)], page_size=8)
    for page_size in (0, 12, 512, 8.0):
        with pytest.raises(ValueError):
            B.paged_free(*free, page_size=page_size)
    with pytest.raises(ValueError):
        B.paged_compact(good[0], good[1][:1], caches)
