"""Attention of several new tokens per request over pages against the oracle (oracle/paged.py, 64 bits).

Tolerance: half a step of the output type, and of the weighted sum of |values| a share of: twice the error of a score (D + 2
roundings of 2^-24 of its sum of |products|), half a step of the type for each weight's rounding, 2^-15 for the
exponential with its argument and 2^-24 for each of up to 2048 terms summed in a row.  In fp16 a weight is off by
2^-25 of 2^7 at least, the smallest weight of a maximum: 2^-32 of the largest |value| for every token, and an output by half of its
smallest step, 2^-25."""

import numpy as np
import pytest
import torch

from metile_b200 import _lib, backends as B
from oracle import paged as O

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.fixture(autouse=True)
def nothing_was_recorded(cuda_device):
    yield
    ok, words = _lib.device_status()
    assert ok, [hex(w) for w in words]


def wide(tensor):
    return tensor.detach().cpu().double().numpy()


def ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def pages_like(generator, layout, pages, heads, page, dim, dtype, device):
    def normal(*shape):
        return torch.randn(shape, generator=generator).to(dtype).to(device)

    if layout == "head":
        return normal(pages, heads, page, dim)
    if layout == "token":   # [pages, page, heads, dim] seen as pages
        return normal(pages, page, heads, dim).transpose(1, 2)
    return normal(pages, 3, heads, page, dim)[:, 1]  # one of a pool of several


class Case:
    """Requests with `new` tokens behind `held` ones; what no request uses of the pages is NaN."""

    def __init__(self, device, held, new, kv_heads, group, dim, page, dtype, layout="head", scale=None, extra=0, std=2.0):
        generator = torch.Generator().manual_seed(sum(held) + 31 * sum(new) + dim)
        lengths = [h + n for h, n in zip(held, new)]
        blocks = [-(-n // page) for n in lengths]
        width, pool = max(blocks) + 2, sum(blocks) + 3
        order = torch.randperm(pool, generator=generator)
        table = torch.full((len(held), width), -1, dtype=torch.int32)
        at = 0
        for r, count in enumerate(blocks):
            table[r, :count] = order[at:at + count]
            at += count
        self.held, self.new, self.host_lengths, self.page, self.dtype = held, new, lengths, page, dtype
        self.scale = dim ** -0.5 if scale is None else scale
        self.query = (torch.randn((sum(new) + extra, kv_heads * group, dim), generator=generator) * std).to(dtype).to(device)
        self.keys, self.values = (pages_like(generator, layout, pool, kv_heads, page, dim, dtype, device) for _ in range(2))
        self.keys[order[at:].to(device)], self.values[order[at:].to(device)] = torch.nan, torch.nan
        for r, n in enumerate(lengths):
            if n % page:
                last = int(table[r, n // page])
                self.keys[last, :, n % page:], self.values[last, :, n % page:] = torch.nan, torch.inf
        self.table, self.lengths = table.to(device), ints(lengths, device)
        self.starts = ints(np.concatenate([[0], np.cumsum(new)]).tolist(), device)

    def run(self, **changes):
        a = {**self.__dict__, **changes}
        return B.paged_attention_chunk(a["query"], a["keys"], a["values"], a["table"], a["lengths"], a["starts"], scale=a["scale"])

    def slot(self, request, token):
        return int(self.table[request, token // self.page]), token % self.page

    def check(self, got=None):
        got = self.run() if got is None else got
        assert got.shape == self.query.shape and got.dtype == self.dtype and got.is_contiguous()
        keys, values = np.nan_to_num(wide(self.keys), posinf=0.0), np.nan_to_num(wide(self.values), posinf=0.0)
        expected, weight, reach = O.chunk_attention(wide(self.query), keys, values, self.table.cpu().numpy(), self.host_lengths,
                                                    self.starts.cpu().numpy(), self.scale)
        dim, half = self.query.shape[2], HALF[self.dtype]
        share = 2 * (dim + 2) * 2.0 ** -24 * reach + half + 2.0 ** -15 + 2048 * 2.0 ** -24
        bound = half * np.abs(expected) + share * weight
        if self.dtype == torch.float16:
            bound = bound + 2.0 ** -25 + max(self.host_lengths) * 2.0 ** -32 * np.abs(values).max()
        worst = float((np.abs(wide(got) - expected) / np.maximum(bound, 1e-30)).max()) if expected.size else 0.0
        assert worst <= 1.0, worst
        return got


CASES = [
    # held, new, kv_heads, group, dim, page, dtype, layout
    ([0], [1], 1, 1, 64, 8, torch.bfloat16, "head"),
    ([0], [7], 2, 3, 128, 16, torch.float16, "head"),
    ([300, 0, 17, 5], [5, 1, 0, 40], 2, 6, 128, 16, torch.bfloat16, "head"),
    ([127, 128, 129, 1000], [1, 2, 3, 130], 8, 4, 128, 16, torch.bfloat16, "token"),
    ([0, 63, 64, 65], [64, 65, 63, 64], 1, 7, 64, 8, torch.float16, "pool"),
    ([2000], [33], 1, 16, 128, 32, torch.float16, "head"),
    ([5000, 40], [3, 500], 2, 5, 64, 64, torch.bfloat16, "token"),
    ([700, 0], [100, 257], 1, 3, 256, 128, torch.bfloat16, "head"),
    ([90, 3], [66, 12], 2, 9, 256, 8, torch.float16, "pool"),
    ([1023, 255], [300, 1], 4, 1, 128, 256, torch.bfloat16, "head"),
    ([10], [21], 1, 40, 64, 16, torch.bfloat16, "head"),
    ([50, 7], [9, 3], 1, 130, 64, 16, torch.float16, "head"),
    ([9], [2], 1, 300, 128, 16, torch.bfloat16, "head"),
    ([6000], [900], 1, 4, 128, 16, torch.bfloat16, "head"),
    ([20000], [16], 1, 2, 128, 32, torch.float16, "head"),
]


@pytest.mark.parametrize("held,new,kv_heads,group,dim,page,dtype,layout", CASES)
def test_rows_see_the_tokens_up_to_their_own(cuda_device, held, new, kv_heads, group, dim, page, dtype, layout):
    case = Case(cuda_device, held, new, kv_heads, group, dim, page, dtype, layout)
    got = case.check()
    assert torch.equal(case.run(), got)  # the same again
    with B.batch_invariant():
        case.check()


@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_scales_of_any_sign(cuda_device, scale, dtype):
    Case(cuda_device, [200, 30], [40, 3], 2, 4, 64, 16, dtype, scale=scale, std=0.5).check()


def test_many_requests(cuda_device):
    rng = np.random.default_rng(3)
    held, new = rng.integers(0, 60, 1300).tolist(), rng.integers(0, 4, 1300).tolist()
    Case(cuda_device, held, new, 1, 2, 64, 8, torch.bfloat16).check()


def test_rows_of_no_request_and_rows_before_the_first_token_are_zeros(cuda_device):
    case = Case(cuda_device, [20, 0], [4, 3], 2, 2, 64, 8, torch.bfloat16, extra=9)
    got = case.check()
    assert not got[7:].any()
    # Two rows in front of request 0, and request 1 has fewer tokens than rows.
    starts, lengths = ints([2, 6, 16], cuda_device), ints([24, 3], cuda_device)
    got = case.run(starts=starts, lengths=lengths)
    assert not got[:2].any() and not got[6:13].any() and bool(got[2:6].any()) and bool((got[13:16] != 0).any(2).all())
    case.host_lengths, case.starts = [24, 3], starts
    case.check(got)
    # A request without tokens: all its rows.
    assert not case.run(lengths=ints([0, 0], cuda_device)).any()
    empty = case.run(query=case.query[:0], starts=ints([0, 0, 0], cuda_device))
    assert empty.shape == (0, 4, 64)


@pytest.mark.parametrize("dim,group,dtype", [(128, 4, torch.bfloat16), (64, 1, torch.float16), (256, 3, torch.bfloat16)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_what_a_row_does_not_see_weighs_nothing(cuda_device, dim, group, dtype, bad):
    case = Case(cuda_device, [150, 0], [200, 300], 2, group, dim, 16, dtype)
    clean = case.run()
    assert bool(torch.isfinite(clean).all())
    for token in (150, 151, 230, 255, 256, 349):  # of request 0: its own rows, at 150 on
        page, row = case.slot(0, token)
        values = case.values.clone()
        values[page, 1, row, 5] = bad
        got = case.run(values=values)
        touched = torch.zeros_like(got, dtype=torch.bool)
        touched[token - 150:200, group:, 5] = True
        assert torch.equal(got[~touched], clean[~touched]), token
        assert (torch.isnan(got[touched]) if bad != bad else got[touched] == bad).all(), token
        keys = case.keys.clone()
        keys[page, 1, row] = bad
        got = case.run(keys=keys)
        touched[token - 150:200, group:] = True
        assert torch.equal(got[~touched], clean[~touched]), token
        if bad != bad:
            assert torch.isnan(got[touched]).all(), token
    both = case.values.clone()
    for token, number in ((180, float("inf")), (190, float("-inf"))):
        page, row = case.slot(0, token)
        both[page, 0, row, 3] = number
    got = case.run(values=both)[:200, :group, 3]
    assert (got[30:40] == torch.inf).all() and torch.isnan(got[40:]).all() and torch.equal(got[:30], clean[:30, :group, 3])
    query = case.query.clone()
    query[60, 0, 7] = torch.nan
    got = case.run(query=query)
    assert torch.isnan(got[60, 0]).all()
    got[60, 0] = clean[60, 0]
    assert torch.equal(got, clean)


def test_scores_of_minus_infinity(cuda_device):
    case = Case(cuda_device, [20], [30], 1, 2, 64, 8, torch.bfloat16)
    case.query[:, :, 0], keys = 1.0, case.keys.clone()
    for token in range(0, 40):
        page, row = case.slot(0, token)
        keys[page, 0, row] = 0.0
        keys[page, 0, row, 0] = -torch.inf
    got = case.run(keys=keys)
    assert not got[:20].any() and bool(torch.isfinite(got).all()) and bool((got[20:] != 0).any(2).all())


def test_a_row_has_the_bits_of_its_own_tokens(cuda_device):
    """In the fixed order neither the other requests nor how a prompt was cut into pieces matter."""
    case = Case(cuda_device, [0, 900, 3], [700, 40, 1], 2, 3, 128, 16, torch.bfloat16)
    with B.fixed_order():
        whole = case.run()
        first = 0
        for request, n in enumerate(case.new):
            rows = slice(first, first + n)
            alone = case.run(query=case.query[rows].contiguous(), table=case.table[request:request + 1],
                             lengths=case.lengths[request:request + 1], starts=ints([0, n], cuda_device))
            assert torch.equal(alone, whole[rows]), request
            first += n
        for cuts in ((0, 1, 2, 130, 131, 700), (0, 333, 700)):
            for a, b in zip(cuts, cuts[1:]):
                piece = case.run(query=case.query[a:b].contiguous(), table=case.table[:1], lengths=ints([b], cuda_device),
                                 starts=ints([0, b - a], cuda_device))
                assert torch.equal(piece, whole[a:b]), (a, b)


def test_one_token_as_in_decoding(cuda_device):
    case = Case(cuda_device, [0, 1, 500, 3000], [1, 1, 1, 1], 2, 6, 128, 16, torch.bfloat16)
    got, decoded = case.check(), B.paged_attention_decode(case.query, case.keys, case.values, case.table, case.lengths, scale=case.scale)
    # Each within half a step, and half a step of the weights: of outputs that are averages of numbers up to 4.
    assert (got - decoded).float().abs().max() <= 2.0 ** -7 * 4


def test_a_captured_call_follows_its_lengths_on_any_stream(cuda_device):
    case = Case(cuda_device, [900, 40], [6, 90], 2, 4, 128, 16, torch.bfloat16)
    lengths, starts, stream = case.lengths.clone(), case.starts.clone(), torch.cuda.Stream(cuda_device)
    case.run()
    graphs, outs = [], []
    for _ in range(2):
        stream.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs.append(case.run(lengths=lengths, starts=starts))
        graphs.append(graph)
    torch.cuda.synchronize()
    for held, new in (([900, 40], [6, 90]), ([10, 0], [3, 93]), ([300, 129], [96, 0]), ([0, 0], [0, 0])):
        lengths.copy_(ints([h + n for h, n in zip(held, new)], cuda_device))
        starts.copy_(ints([0, new[0], sum(new)], cuda_device))
        for graph in graphs:  # one behind the other on two streams, and at once
            side = torch.cuda.Stream(cuda_device)
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                graph.replay()
        torch.cuda.synchronize()
        expected = case.run(lengths=lengths, starts=starts)
        assert torch.equal(outs[0], expected) and torch.equal(outs[1], expected)


def test_offsets_beyond_32_bits(cuda_device):
    """Pages of a pool of 4.6 GB, the ones that are used at both of its ends."""
    page, kv_heads, dim = 256, 8, 128
    pool = 9000
    keys, values = (torch.empty((pool, kv_heads, page, dim), dtype=torch.bfloat16, device=cuda_device) for _ in range(2))
    small = Case(cuda_device, [700], [80], kv_heads, 2, dim, page, torch.bfloat16)
    ids = torch.tensor([pool - 1, 0, pool - 2, 4321], device=cuda_device)
    table = small.table.clone()
    for block in range(4):
        keys[ids[block]], values[ids[block]] = small.keys[small.table[0, block].long()], small.values[small.table[0, block].long()]
        table[0, block] = ids[block]
    assert torch.equal(small.run(keys=keys, values=values, table=table), small.run())


@pytest.mark.parametrize("spoil,code", [("page", 0x303), ("length", 0x304), ("short", 0x304), ("start", 0x306), ("order", 0x306)])
def test_what_lies_outside_is_recorded_and_left_out(cuda_device, spoil, code):
    case = Case(cuda_device, [100, 30], [20, 10], 2, 4, 64, 16, torch.bfloat16)
    clean, rest = case.run(), slice(20, 30)
    table, lengths, starts = case.table.clone(), case.lengths.clone(), case.starts.clone()
    if spoil == "page":
        table[0, 3] = 10 ** 6
    elif spoil == "length":
        lengths[0] = table.shape[1] * 16 + 1
        table[0] = table[0].clamp(min=0)
    elif spoil == "short":
        lengths[0] = -5
    elif spoil == "start":
        starts[2] = 31
        rest = slice(0, 20)
    else:
        starts[0] = 25
    got = case.run(table=table, lengths=lengths, starts=starts)
    ok, words = _lib.device_status()
    assert not ok and words[0] == code, [hex(w) for w in words]
    assert torch.equal(got[rest], clean[rest])
    if spoil in ("start", "order", "short"):
        assert not got[20:30 if spoil == "start" else 20].any() and (spoil == "start" or not got[:20].any())
    if spoil == "page":  # tokens 48 to 63 weigh nothing
        keep = [t for t in range(120) if not 48 <= t < 64]
        generator = Case(cuda_device, [84], [20], 2, 4, 64, 16, torch.bfloat16)
        for i, t in enumerate(keep):
            (a, b), (c, d) = case.slot(0, t), generator.slot(0, i)
            generator.keys[c, :, d], generator.values[c, :, d] = case.keys[a, :, b], case.values[a, :, b]
        generator.query = case.query[:20].contiguous()
        generator.check(got[:20])


def test_refusals(cuda_device):
    case = Case(cuda_device, [10], [4], 2, 2, 64, 8, torch.bfloat16)
    wrong = [
        ({"query": case.query.float()}, TypeError), ({"query": case.query.cpu()}, ValueError), ({"query": case.query[0]}, ValueError),
        ({"query": case.query[:, :3]}, ValueError), ({"query": case.query.half()}, ValueError), ({"keys": case.keys[..., :32]}, ValueError),
        ({"keys": case.keys[:, :, :4]}, ValueError), ({"values": case.values[:1]}, ValueError), ({"keys": case.keys[:0], "values": case.values[:0]}, ValueError),
        ({"table": case.table.long()}, TypeError), ({"table": case.table[0]}, ValueError), ({"table": case.table[:0]}, ValueError),
        ({"table": case.table.cpu()}, ValueError), ({"lengths": case.lengths.cpu()}, ValueError), ({"lengths": case.lengths.long()}, ValueError),
        ({"starts": case.starts[:1]}, ValueError), ({"starts": case.starts.long()}, ValueError), ({"starts": None}, ValueError),
        ({"query": case.query.clone().requires_grad_()}, ValueError), ({"scale": "1"}, (TypeError, ValueError)),
    ]
    for changes, error in wrong:
        with pytest.raises(error):
            case.run(**changes)
    # What is laid out otherwise is taken all the same.
    strided = torch.empty((4, 4, 128), dtype=torch.bfloat16, device=cuda_device)[..., :64]
    strided.copy_(case.query)
    assert torch.equal(case.run(query=strided), case.run())
    with torch.no_grad():
        assert torch.equal(case.run(query=case.query.clone().requires_grad_()), case.run())


def test_no_request(cuda_device):
    case = Case(cuda_device, [10], [4], 2, 2, 64, 8, torch.bfloat16)
    none = torch.zeros((0, 3), dtype=torch.int32, device=cuda_device)
    assert not case.run(table=none, lengths=ints([], cuda_device), starts=ints([0], cuda_device)).any()
