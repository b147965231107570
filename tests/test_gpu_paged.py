"""The paged key-value cache against the oracle (oracle/paged.py, 64 bits): block tables and slot maps, rotary
embedding + append, decode attention.

Tolerances.  Attention: half a step of the output type, and of the weighted sum of |values| a share of: twice the
error of a score (D + 2 roundings of 2^-24 of its sum of |products|), 2^-15 for the exponential (its argument's rounding
included) and the weights' two halves, and 2^-24 for each of up to 2048 terms summed in a row.  Rotation: half a
step, and 2^-20 of |a| + |b| for sine, cosine and three roundings in 32 bits."""

import numpy as np
import pytest
import torch

from metile_b200 import _lib, backends as B
from oracle import paged as O

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


@pytest.fixture(autouse=True)
def nothing_was_recorded(cuda_device):
    yield
    ok, words = _lib.device_status()
    assert ok, [hex(w) for w in words]


def wide(tensor):
    return tensor.detach().cpu().double().numpy()


def ints(values, device, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=device)


def normal(seed, *shape, device, dtype=torch.bfloat16, std=1.0):
    generator = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=generator) * std).to(dtype).to(device)


# ---- block tables and slot maps -----------------------------------------------------------------------------------


def resize_case(seed, requests, page, width, most, free, start, device):
    rng = np.random.default_rng(seed)
    lengths = rng.integers(0, max(1, width * page - most), requests)
    counts = np.where(rng.random(requests) < 0.3, -rng.integers(0, 1 + lengths), rng.integers(0, most + 1, requests))
    used = int((-(-lengths // page)).sum())
    pool = used + free
    pages = rng.permutation(pool).astype(np.int32)
    tables = np.full((requests, width), -1, np.int32)
    at = 0
    for r, n in enumerate(lengths):
        blocks = -(-int(n) // page)
        tables[r, :blocks] = pages[at:at + blocks]
        at += blocks
    ring = np.full(max(pool, 1), -7, np.int32)
    start %= len(ring)
    ring[(start + np.arange(free)) % len(ring)] = pages[used:]
    return [tables, lengths.astype(np.int32), counts.astype(np.int32), ring, np.array([start, free], np.int32)]


def check_resize(arrays, page, tokens, device, **kwargs):
    expected = O.resize(*arrays, page, tokens)
    in_place = [torch.tensor(a, device=device) for a in arrays]
    got = B.paged_resize(*in_place, page_size=page, tokens=tokens, advance=True)
    for name, a, b in zip(("slots", "positions", "starts", "lengths", "state", "table", "ring"), (*got, in_place[0], in_place[3]), expected):
        assert np.array_equal(a.cpu().numpy(), b), name
    tensors = [torch.tensor(a, device=device) for a in arrays]
    for _ in range(2):  # a call with the same lengths and state does the same again
        got = B.paged_resize(*tensors, page_size=page, tokens=tokens, **kwargs)
        for name, a, b in zip(("slots", "positions", "starts", "lengths", "state"), got, expected):
            assert np.array_equal(a.cpu().numpy(), b), name
        assert np.array_equal(tensors[0].cpu().numpy(), expected[5]) and np.array_equal(tensors[3].cpu().numpy(), expected[6])
    assert np.array_equal(tensors[1].cpu().numpy(), arrays[1]) and np.array_equal(tensors[4].cpu().numpy(), arrays[4])


@pytest.mark.parametrize("requests,page,width,most,free,start", [
    (1, 16, 4, 1, 1, 0), (3, 8, 5, 9, 40, 17), (64, 16, 40, 1, 64, 5), (65, 32, 9, 70, 300, 1000), (1, 256, 3, 700, 3, 2),
    (1024, 16, 8, 40, 4000, 3), (300, 16, 900, 4000, 80000, 5), (2, 32, 3000, 60000, 4000, 1), (1025, 64, 4, 30, 1500, 9999), (2500, 8, 6, 20, 3000, 77),
])
def test_requests_grow_and_shrink(cuda_device, requests, page, width, most, free, start):
    arrays = resize_case(requests, requests, page, width, most, free, start, cuda_device)
    check_resize(arrays, page, int(np.maximum(arrays[2], 0).sum()) + 3, cuda_device)


@pytest.mark.parametrize("free,tokens", [(0, 500), (1, 500), (20, 500), (400, 100), (400, 0), (7, 33)])
def test_pages_or_map_do_not_reach(cuda_device, free, tokens):
    check_resize(resize_case(free + tokens, 33, 8, 12, 30, free, 11, cuda_device), 8, tokens, cuda_device)


def test_lengths_and_counts_that_make_no_sense(cuda_device):
    arrays = resize_case(5, 9, 16, 6, 8, 30, 4, cuda_device)
    tables, lengths, counts, ring, state = arrays
    lengths[:9] = [0, 90, -3, 97, 96, 16, 15, 2**31 - 1, 40]
    counts[:9] = [0, 7, 2, 1, 1, -17, 1, 2**31 - 1, -40]
    check_resize(arrays, 16, 50, cuda_device)  # the giant count takes no room: its tokens end behind the map's
    counts[7] = -2**31
    check_resize(arrays, 16, 50, cuda_device)


def test_no_request_and_no_token(cuda_device):
    tables, ring = torch.full((0, 3), -1, dtype=torch.int32, device=cuda_device), ints([4, 5], cuda_device)
    out = B.paged_resize(tables, ints([], cuda_device), ints([], cuda_device), ring, ints([1, 2], cuda_device), page_size=16, tokens=5)
    assert out[0].tolist() == [-1] * 5 and out[1].tolist() == [0] * 5 and out[2].tolist() == [0] and out[4].tolist() == [1, 2]


def test_advance_in_place_in_a_graph_until_the_pages_run_out(cuda_device):
    page, width, requests, pool = 8, 6, 5, 17
    arrays = [np.full((requests, width), -1, np.int32), np.zeros(requests, np.int32), np.array([1, 2, 0, 3, 1], np.int32),
              np.arange(pool, dtype=np.int32), np.array([9, pool], np.int32)]
    tensors = [torch.tensor(a, device=cuda_device) for a in arrays]
    stream = torch.cuda.Stream(cuda_device)
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = B.paged_resize(*tensors, page_size=page, tokens=9, advance=True)
    assert got[3].data_ptr() == tensors[1].data_ptr() and got[4].data_ptr() == tensors[4].data_ptr()
    torch.cuda.synchronize()
    for step in range(45):
        if step == 20:  # the first request ends and its pages come back
            tensors[2][0] = -int(arrays[1][0])
            arrays[2][0] = -int(arrays[1][0])
        if step == 21:
            tensors[2][0] = 0
            arrays[2][0] = 0
        graph.replay()
        out = O.resize(*arrays, page, 9)
        for a, b in zip(got, out):
            assert np.array_equal(a.cpu().numpy(), b), step
        arrays[0], arrays[1], arrays[3], arrays[4] = out[5], out[3], out[6], out[4]
        assert np.array_equal(tensors[0].cpu().numpy(), arrays[0]) and np.array_equal(tensors[3].cpu().numpy(), arrays[3])


def test_a_table_that_is_a_view_keeps_what_is_beside_it(cuda_device):
    arrays = resize_case(8, 12, 16, 7, 20, 60, 3, cuda_device)
    wider = torch.full((12, 11), 99, dtype=torch.int32, device=cuda_device)
    wider[:, 2:9] = torch.tensor(arrays[0], device=cuda_device)
    rest = [torch.tensor(a, device=cuda_device) for a in arrays[1:]]
    B.paged_resize(wider[:, 2:9], *rest, page_size=16, tokens=300)
    assert np.array_equal(wider[:, 2:9].cpu().numpy(), O.resize(*arrays, 16, 300)[5])
    assert (wider[:, :2] == 99).all() and (wider[:, 9:] == 99).all()


# ---- rotary embedding and append ----------------------------------------------------------------------------------


def pages_like(seed, layout, pages, heads, page, dim, dtype, device):
    if layout == "head":
        return normal(seed, pages, heads, page, dim, device=device, dtype=dtype)
    if layout == "token":   # [pages, page, heads, dim] seen as pages
        return normal(seed, pages, page, heads, dim, device=device, dtype=dtype).transpose(1, 2)
    return normal(seed, pages, 3, heads, page, dim, device=device, dtype=dtype)[:, 1]  # one of a pool of several


@pytest.mark.parametrize("rows,heads,kv_heads,dim,page,dtype,layout,fused", [
    (1, 1, 1, 16, 8, torch.bfloat16, "head", True), (16, 12, 2, 128, 16, torch.bfloat16, "head", True),
    (37, 4, 4, 64, 32, torch.float16, "token", False), (5, 16, 1, 256, 128, torch.bfloat16, "pool", False),
    (130, 6, 3, 96, 8, torch.float16, "pool", True), (33, 8, 8, 48, 256, torch.bfloat16, "token", True),
])
def test_rows_are_rotated_and_go_to_their_slots(cuda_device, rows, heads, kv_heads, dim, page, dtype, layout, fused):
    if fused:
        both = normal(rows, rows, (heads + 2 * kv_heads) * dim, device=cuda_device, dtype=dtype)
        q, k, v = (part.view(rows, -1, dim) for part in both.split((heads * dim, kv_heads * dim, kv_heads * dim), 1))
    else:
        q, k, v = (normal(rows + i, rows, h, dim, device=cuda_device, dtype=dtype) for i, h in enumerate((heads, kv_heads, kv_heads)))
    pool = -(-rows // page) + 3
    keys, values = (pages_like(7 + i, layout, pool, kv_heads, page, dim, dtype, cuda_device) for i in range(2))
    rng = np.random.default_rng(rows)
    slots = rng.permutation(pool * page)[:rows].astype(np.int64)
    slots[rows // 2::5] = -1
    positions = rng.integers(0, 1 << 20, rows).astype(np.int32)
    inverse = (1e6 ** (-np.arange(0, dim, 2) / dim)).astype(np.float32)
    before = wide(keys), wide(values)
    out = B.rope_kv_append_paged(q, k, v, torch.tensor(inverse, device=cuda_device), ints(positions.tolist(), cuda_device),
                                 ints(slots.tolist(), cuda_device, torch.int64), keys, values)
    assert out.shape == q.shape and out.dtype == dtype and out.is_contiguous()

    def close(got, source, what):
        a = np.abs(wide(source))
        size = a[..., :dim // 2] + a[..., dim // 2:]
        expected = O.rotate(wide(source), inverse, positions)
        bound = HALF[dtype] * np.abs(expected) + 2.0 ** -20 * np.concatenate([size, size], -1) + (2.0 ** -25 if dtype == torch.float16 else 0)
        assert (np.abs(got - expected) <= bound).all(), what

    close(wide(out), q, "query")
    there = slots >= 0
    at, row = slots[there] // page, slots[there] % page
    close_keys = wide(k)
    close_keys[there] = wide(keys)[at, :, row]
    expected_keys = O.rotate(wide(k), inverse, positions)
    close(np.where(there[:, None, None], close_keys, expected_keys), k, "keys")
    assert np.array_equal(wide(values)[at, :, row], wide(v)[there])
    untouched = np.ones((pool, page), bool)
    untouched[at, row] = False
    for now, then in ((wide(keys), before[0]), (wide(values), before[1])):
        assert np.array_equal(now.transpose(0, 2, 1, 3)[untouched], then.transpose(0, 2, 1, 3)[untouched])


def test_a_slot_outside_the_cache_is_recorded_and_left_out(cuda_device):
    q, k, v = (normal(i, 3, 2, 64, device=cuda_device) for i in range(3))
    keys, values = (normal(9 + i, 2, 2, 16, 64, device=cuda_device) for i in range(2))
    before = keys.clone(), values.clone()
    inverse = torch.ones(32, device=cuda_device)
    for slot in (32, 2**40):
        B.rope_kv_append_paged(q, k, v, inverse, ints([1, 2, 3], cuda_device), ints([-5, slot, -1], cuda_device, torch.int64), keys, values)
        ok, words = _lib.device_status()
        assert not ok and words[0] == 0x302 and words[1] == 1 and words[2] | words[3] << 32 == slot
    assert torch.equal(keys, before[0]) and torch.equal(values, before[1])


# ---- attention ----------------------------------------------------------------------------------------------------


def attention_case(seed, lengths, heads, kv_heads, dim, page, dtype, layout, device, spread=2.0, spare=3):
    rng = np.random.default_rng(seed)
    blocks = [-(-n // page) for n in lengths]
    pool = sum(blocks) + 2
    ids = rng.permutation(pool)
    tables = np.full((len(lengths), max(max(blocks), 1) + spare), -1, np.int32)
    at = 0
    for b, count in enumerate(blocks):
        tables[b, :count] = ids[at:at + count]
        at += count
    q = normal(seed, len(lengths), heads, dim, device=device, dtype=dtype, std=spread)
    keys, values = (pages_like(seed + 1 + i, layout, pool, kv_heads, page, dim, dtype, device) for i in range(2))
    return q, keys, values, tables, np.array(lengths, np.int32)


def check_attention(case, scale, device, out=None):
    q, keys, values, tables, lengths = case
    if out is None:
        out = B.paged_attention_decode(q, keys, values, torch.tensor(tables, device=device), torch.tensor(lengths, device=device), scale=scale)
    assert out.shape == q.shape and out.dtype == q.dtype
    expected, weight, reach = O.attention(wide(q), wide(keys), wide(values), tables, lengths, scale)
    share = 2 * (q.shape[-1] + 2) * 2.0 ** -24 * reach + 2.0 ** -15 + min(2048, int(lengths.max())) * 2.0 ** -24
    bound = HALF[q.dtype] * np.abs(expected) + share * weight * (1 + HALF[q.dtype]) + (2.0 ** -25 if q.dtype == torch.float16 else 0)
    error = np.abs(wide(out) - expected)
    assert (error <= bound).all(), float((error / np.maximum(bound, 1e-30)).max())
    return out


@pytest.mark.parametrize("lengths,heads,kv_heads,dim,page,dtype,layout", [
    ([1], 1, 1, 64, 8, torch.bfloat16, "head"),
    ([0, 1, 15, 16, 17, 127, 128, 129, 0], 12, 2, 128, 16, torch.bfloat16, "head"),
    ([300, 5, 64], 4, 4, 64, 32, torch.float16, "token"),
    ([1000, 1], 8, 1, 128, 8, torch.bfloat16, "pool"),
    ([513, 255, 31], 16, 1, 64, 64, torch.float16, "head"),
    ([200, 700], 27, 3, 128, 128, torch.bfloat16, "token"),
    ([333], 40, 2, 64, 16, torch.bfloat16, "pool"),
    ([257, 90], 6, 2, 256, 256, torch.float16, "head"),
    ([70, 2000], 34, 2, 256, 8, torch.bfloat16, "head"),
    ([4097, 12, 2048], 10, 2, 128, 16, torch.bfloat16, "head"),
    ([33000], 2, 2, 64, 32, torch.float16, "head"),
    ([0, 0], 3, 1, 128, 16, torch.bfloat16, "head"),
    ([700, 0, 130, 1], 20, 2, 128, 16, torch.bfloat16, "token"),
    ([900], 33, 1, 64, 8, torch.float16, "head"),
    ([400, 512], 12, 3, 256, 32, torch.bfloat16, "pool"),
    ([129] * 80, 8, 4, 128, 16, torch.bfloat16, "head"),
])
def test_paged_attention_against_the_oracle(cuda_device, lengths, heads, kv_heads, dim, page, dtype, layout):
    check_attention(attention_case(31, lengths, heads, kv_heads, dim, page, dtype, layout, cuda_device), dim ** -0.5, cuda_device)


@pytest.mark.parametrize("lengths,heads,kv_heads,dim,page,dtype", [
    ([16384, 16385, 70000, 0, 1], 8, 1, 64, 32, torch.bfloat16), ([65537], 10, 1, 128, 64, torch.float16),
    ([32769, 16500, 300], 4, 2, 64, 16, torch.bfloat16), ([20000], 16, 1, 256, 128, torch.bfloat16), ([16640], 6, 3, 64, 32, torch.float16),
])
def test_long_sequences_of_few_heads(cuda_device, lengths, heads, kv_heads, dim, page, dtype):
    """Up to 512 splits of a sequence; the bits are its own whatever the table's width and the others."""
    q, keys, values, tables, n = attention_case(37, lengths, heads, kv_heads, dim, page, dtype, "head", cuda_device)
    out = check_attention((q, keys, values, tables, n), dim ** -0.5, cuda_device)
    table = torch.tensor(tables, device=cuda_device)
    for b, count in enumerate(n):
        narrow = table[b:b + 1, :max(1, -(-int(count) // page))].contiguous()
        alone = B.paged_attention_decode(q[b:b + 1], keys, values, narrow, torch.tensor(n[b:b + 1], device=cuda_device), scale=dim ** -0.5)
        assert torch.equal(alone, out[b:b + 1]), b


def test_a_peaked_softmax_and_large_scores(cuda_device):
    check_attention(attention_case(41, [900, 60], 8, 2, 128, 16, torch.bfloat16, "head", cuda_device, spread=40.0), 128 ** -0.5, cuda_device)
    check_attention(attention_case(42, [400], 4, 4, 64, 16, torch.float16, "head", cuda_device), -0.7, cuda_device)


def test_what_lies_behind_a_sequence_is_never_used(cuda_device):
    lengths = [5, 130, 0, 64]
    case = attention_case(51, lengths, 6, 2, 128, 16, torch.bfloat16, "head", cuda_device)
    q, keys, values, tables, _ = case
    out = check_attention(case, 0.1, cuda_device)
    poisoned = keys.clone(), values.clone()
    used = np.zeros((keys.shape[0], 16), bool)
    for b, n in enumerate(lengths):
        for t in range(n):
            used[tables[b, t // 16], t % 16] = True
    free = torch.tensor(~used, device=cuda_device)[:, None, :, None].expand_as(keys)
    poisoned[0][free], poisoned[1][free] = float("nan"), float("inf")
    far = tables.copy()
    for b, n in enumerate(lengths):
        far[b, -(-n // 16):] = 2**31 - 1
    again = check_attention((q, *poisoned, far, case[4]), 0.1, cuda_device, B.paged_attention_decode(
        q, *poisoned, torch.tensor(far, device=cuda_device), ints(lengths, cuda_device), scale=0.1))
    assert torch.equal(again, out) and not again[2].any()


def test_a_request_alone_and_in_a_batch_and_in_other_pages_has_the_same_bits(cuda_device):
    lengths = [3000, 17, 129, 900, 1]
    q, keys, values, tables, n = attention_case(61, lengths, 12, 2, 128, 16, torch.bfloat16, "head", cuda_device)
    table = torch.tensor(tables, device=cuda_device)
    out = B.paged_attention_decode(q, keys, values, table, torch.tensor(n, device=cuda_device), scale=0.09)
    for b in range(len(lengths)):
        alone = B.paged_attention_decode(q[b:b + 1], keys, values, table[b:b + 1], torch.tensor(n[b:b + 1], device=cuda_device), scale=0.09)
        assert torch.equal(alone, out[b:b + 1]), b
    # Short requests by a narrow table (one launch) and by a wide one (two).
    short = B.paged_attention_decode(q[1:], keys, values, table[1:, :48].contiguous(), torch.tensor([17, 129, 700, 1], dtype=torch.int32, device=cuda_device), scale=0.09)
    again = B.paged_attention_decode(q[1:], keys, values, table[1:], torch.tensor([17, 129, 700, 1], dtype=torch.int32, device=cuda_device), scale=0.09)
    assert torch.equal(short, again)
    # The same tokens in pages of 64, in the other layout, with a wider table.
    larger = torch.full((sum(-(-x // 64) for x in lengths), 64, 2, 128), float("nan"), dtype=torch.bfloat16, device=cuda_device)
    larger = [larger.clone().transpose(1, 2) for _ in range(2)]
    wider, at = np.full((len(lengths), 90), 7, np.int32), 0
    for b, count in enumerate(lengths):
        for first in range(0, count, 64):
            wider[b, first // 64] = at
            for t in range(first, min(count, first + 64), 16):
                here = min(16, count - t)
                for old, new in ((keys, larger[0]), (values, larger[1])):
                    new[at, :, t - first:t - first + here] = old[tables[b, t // 16], :, :here]
            at += 1
    moved = B.paged_attention_decode(q, *larger, torch.tensor(wider, device=cuda_device), torch.tensor(n, device=cuda_device), scale=0.09)
    assert torch.equal(moved, out)


def test_pages_and_lengths_outside_are_recorded_and_left_out(cuda_device):
    q, keys, values, tables, n = attention_case(71, [40, 33], 4, 2, 64, 16, torch.bfloat16, "head", cuda_device, spare=0)
    for page in (-1, keys.shape[0], 2**31 - 1):
        bad = tables.copy()
        bad[1, 1] = page
        out = B.paged_attention_decode(q, keys, values, torch.tensor(bad, device=cuda_device), torch.tensor(n, device=cuda_device), scale=0.1)
        ok, words = _lib.device_status()
        assert not ok and words[:3] == (0x303, 1, page & 0xFFFFFFFF)
        rest = np.array([[tables[1, 0], tables[1, 2]]])  # its other tokens: 16 of one page, one of the last
        check_attention((q[1:], keys, values, rest, np.array([17])), 0.1, cuda_device, out[1:])
    wide_table = torch.full((2, 200), -1, dtype=torch.int32, device=cuda_device)  # as many launches as a long request takes
    wide_table[:, :3] = torch.tensor(tables, device=cuda_device)
    for length in (-4, 3201):
        B.paged_attention_decode(q, keys, values, wide_table, ints([40, length], cuda_device), scale=0.1)
        ok, words = _lib.device_status()
        assert not ok and words[0] in ((0x304,) if length < 0 else (0x303, 0x304)) and words[1] == 1
    for length in (-4, 49, 2**31 - 1):  # the table has room for 48
        out = B.paged_attention_decode(q, keys, values, torch.tensor(tables, device=cuda_device), ints([length, 33], cuda_device), scale=0.1)
        ok, words = _lib.device_status()
        assert not ok and words[:3] == (0x304, 0, length & 0xFFFFFFFF)
        if length < 0:
            assert not out[0].any()


def test_on_another_stream_in_a_graph_and_twice_at_once(cuda_device):
    cases = [attention_case(81 + i, [700, 3, 260], 12, 2, 128, 16, torch.bfloat16, "head", cuda_device) for i in range(2)]
    tensors = [[*c[:3], torch.tensor(c[3], device=cuda_device), torch.tensor(c[4], device=cuda_device)] for c in cases]
    eager = [B.paged_attention_decode(*t, scale=0.09) for t in tensors]
    torch.cuda.synchronize()
    streams, graphs, outs = [torch.cuda.Stream(cuda_device) for _ in cases], [], []
    for t, s in zip(tensors, streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs.append(B.paged_attention_decode(*t, scale=0.09))
        graphs.append(graph)
    for _ in range(20):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(eager, outs):
        assert torch.equal(a, b)
    tensors[0][4].fill_(9)  # the captured call reads its lengths from the device
    graphs[0].replay()
    torch.cuda.synchronize()
    check_attention((*cases[0][:4], np.array([9, 9, 9], np.int32)), 0.09, cuda_device, outs[0])


def test_refusals_on_the_device(cuda_device):
    q, keys, values, tables, n = attention_case(91, [40, 33], 4, 2, 64, 16, torch.bfloat16, "head", cuda_device)
    table, lengths = torch.tensor(tables, device=cuda_device), torch.tensor(n, device=cuda_device)
    good = (q, keys, values, table, lengths)
    B.paged_attention_decode(*good, scale=1)  # a whole number will do

    def refused(error, index, tensor):
        arguments = list(good)
        arguments[index] = tensor
        with pytest.raises(error):
            B.paged_attention_decode(*arguments, scale=0.1)

    refused(TypeError, 0, q.float())
    refused(ValueError, 0, q.half())
    refused(ValueError, 0, q[:1])
    refused(ValueError, 0, q[:, :3])
    refused(ValueError, 0, q[:, :, :32])
    refused(ValueError, 0, q.clone().requires_grad_())
    refused(ValueError, 1, keys[:, :, :12])
    refused(ValueError, 1, keys[:-1])
    refused(ValueError, 1, keys[:1].expand(keys.shape[0], -1, -1, -1))
    refused(ValueError, 2, values.half())
    refused(TypeError, 3, table.long())
    refused(ValueError, 3, table[:1].expand(2, -1))
    refused(ValueError, 4, lengths.long())
    refused(ValueError, 4, lengths.cpu())
    assert B.paged_attention_decode(q[:0], keys, values, table[:0], lengths[:0], scale=0.1).shape == (0, 4, 64)
    strided = torch.cat([q, q], -1)[:, :, :64]
    assert torch.equal(B.paged_attention_decode(strided, *good[1:], scale=0.1), B.paged_attention_decode(*good, scale=0.1))


def test_offsets_beyond_32_bits(cuda_device):
    """Pages that lie more than 2^31 elements behind the first: append, attention, and the copy of a page in work."""
    pages, heads, page, dim = 140000, 2, 64, 128
    keys, values = (torch.empty((pages, heads, page, dim), dtype=torch.bfloat16, device=cuda_device) for _ in range(2))
    last = [pages - 1, pages - 3, pages - 2, pages - 7]
    q, k, v = (normal(101 + i, 70, h, dim, device=cuda_device) for i, h in enumerate((4, heads, heads)))
    slots = torch.tensor([last[t // page] * page + t % page for t in range(70)], device=cuda_device)
    B.rope_kv_append_paged(q, k, v, torch.zeros(dim // 2, device=cuda_device), torch.arange(70, dtype=torch.int32, device=cuda_device), slots,
                           keys, values)
    assert torch.equal(keys[last[0]].transpose(0, 1), k[:64]) and torch.equal(values[last[1], :, :6].transpose(0, 1), v[64:])
    tables = np.array([[last[0], last[1]], [last[0], last[2]]], np.int32)
    table, lengths = torch.tensor(tables, device=cuda_device), ints([70, 70], cuda_device)
    moved = B.beam_reorder(table, lengths, ints([[0, 0]], cuda_device), [(keys, values)])
    assert moved.tolist() == [[last[0], last[1]], [last[0], last[2]]]
    assert torch.equal(keys[last[2], :, :6], keys[last[1], :, :6]) and torch.equal(values[last[2], :, :6], values[last[1], :, :6])
    out = B.paged_attention_decode(q[:2], keys, values, moved, lengths, scale=0.1)
    small = np.array([[0, 1], [0, 1]], np.int32)
    near = [torch.stack([t[last[0]], t[last[1]]]) for t in (keys, values)]
    for tensor in near:
        tensor[1, :, 6:] = 0
    check_attention((q[:2], *near, small, np.array([70, 70], np.int32)), 0.1, cuda_device, out)
