"""Beam selection and the reordering of the paged cache against the oracle (oracle/paged.py, 64 bits).

Beams, tokens and flags have to be the oracle's; a score may be off by half a step of 32 bits and 2^-20, the most that
32-bit exponentials leave a log-sum."""

import numpy as np
import pytest
import torch

from metile_b200 import _lib, backends as B
from oracle import paged as O

pytestmark = pytest.mark.gpu

LOWEST = {torch.bfloat16: -3.3895313892515355e38, torch.float16: -65504.0, torch.float32: -3.4028234663852886e38}


@pytest.fixture(autouse=True)
def nothing_was_recorded(cuda_device):
    yield
    ok, words = _lib.device_status()
    assert ok, [hex(w) for w in words]


def wide(tensor):
    return tensor.detach().cpu().double().numpy()


def select_case(seed, groups, beams, vocab, dtype, device, ended=False, std=2.5):
    generator = torch.Generator().manual_seed(seed)
    logits = (torch.randn((groups * beams, vocab), generator=generator) * std).to(dtype).to(device)
    scores = torch.sort(torch.rand((groups, beams), generator=generator) * -20.0, dim=1, descending=True).values.to(device)
    finished = (torch.rand((groups, beams), generator=generator) < 0.3).to(device) if ended else None
    return logits, scores, finished


def check_select(logits, scores, keep, finished=None, end=None, out=None):
    if out is None:
        out = B.beam_select(logits, scores, keep=keep, finished=finished, end_token=end)
    expected = O.beam_select(wide(logits), wide(scores), keep, None if finished is None else finished.cpu().numpy(), -1 if end is None else end)
    assert [t.dtype for t in out] == [torch.float32, torch.int32, torch.int64, torch.bool]
    assert np.array_equal(out[1].cpu().numpy(), expected[1]) and np.array_equal(out[2].cpu().numpy(), expected[2])
    assert np.array_equal(out[3].cpu().numpy(), expected[3])
    got, same = wide(out[0]), expected[0] == -np.inf
    assert (got[same] == -np.inf).all()
    with np.errstate(invalid="ignore"):
        assert (np.abs(got - expected[0])[~same] <= (2.0 ** -24 * np.abs(expected[0]) + 2.0 ** -20)[~same]).all()
    return out


@pytest.mark.parametrize("groups,beams,vocab,keep,dtype,ended", [
    (1, 1, 1, 1, torch.bfloat16, False), (1, 4, 32001, 4, torch.bfloat16, False), (3, 2, 5, 7, torch.float32, False),
    (2, 8, 1000, 16, torch.float16, True), (5, 3, 8191, 3, torch.bfloat16, True), (1, 1, 8192, 64, torch.float32, False),
    (2, 5, 8193, 10, torch.float16, True), (1, 16, 50001, 32, torch.bfloat16, False), (1, 32, 777, 64, torch.float32, True),
    (9, 4, 128256, 8, torch.bfloat16, True), (40, 2, 16385, 4, torch.float16, False), (1, 3, 300007, 6, torch.float32, False),
])
def test_selection_against_the_oracle(cuda_device, groups, beams, vocab, keep, dtype, ended):
    logits, scores, finished = select_case(vocab, groups, beams, vocab, dtype, cuda_device, ended)
    check_select(logits, scores, keep, finished, min(2, vocab - 1) if ended else None)


def test_equal_candidates_go_by_beam_and_token(cuda_device):
    for dtype in (torch.bfloat16, torch.float32):
        logits = torch.zeros((6, 20000), dtype=dtype, device=cuda_device)
        check_select(logits, torch.zeros((2, 3), device=cuda_device), 40)
        logits[1, 17], logits[2, 16000:] = 3.0, 3.0
        logits[4] = -0.0
        check_select(logits, torch.zeros((2, 3), device=cuda_device), 64)
    # Beams that are the same row throughout.
    row, _, _ = select_case(3, 1, 1, 9001, torch.bfloat16, cuda_device)
    check_select(row.expand(4, -1), torch.full((1, 4), -3.25, device=cuda_device), 16)
    check_select(row.repeat(4, 1), torch.full((1, 4), -3.25, device=cuda_device), 16)


@pytest.mark.parametrize("levels,keep", [(2, 8), (3, 64), (40, 16), (4000, 5)])
def test_many_equal_logits_at_any_level(cuda_device, levels, keep):
    generator = torch.Generator().manual_seed(levels)
    logits = torch.randint(0, levels, (6, 40003), generator=generator).to(torch.float16).to(cuda_device) / 8
    logits[1] = torch.where(logits[1] > 0, logits[1], -torch.inf)
    logits[2, 16384:32768] = -torch.inf  # a span with nothing in it
    scores = torch.tensor([[-1.0, -1.25, -0.5], [-3.0, -3.0, -2.0]], device=cuda_device)
    check_select(logits, scores, keep)
    check_select(logits[:1], scores[:1, :1].contiguous(), keep)


def test_the_largest_logits_side_by_side(cuda_device):
    """All of the large ones in the vectors of few threads, more of them than a buffer takes, and in order."""
    for dtype in (torch.float32, torch.bfloat16):
        logits = torch.zeros((2, 100000), device=cuda_device)
        at = torch.arange(100000, device=cuda_device)
        near = at // (32 if dtype == torch.float32 else 64) % 32 == 5
        logits[0, near] = 1.0 + at[near].float() / 100000
        logits[1] = at.float() / 100000
        for keep in (2, 64):
            check_select(logits.to(dtype), torch.zeros((1, 2), device=cuda_device), keep)


def test_candidates_of_two_beams_closer_than_32_bits_tell(cuda_device):
    """One beam's score is moved so that its best candidate lies a hair above or below the other beam's: the order is
    the one of 64 bits."""
    for seed in range(12):
        logits, scores, _ = select_case(100 + seed, 1, 2, 4000 + 977 * seed, torch.float32, cuda_device)
        rows, s = wide(logits), wide(scores)[0]
        value = [s[k] + rows[k].max() - (np.log(np.exp(rows[k] - rows[k].max()).sum()) + rows[k].max()) for k in range(2)]
        near = np.float32(s[1] + value[0] - value[1])
        for steps in (-1, 0, 1):
            moved = near
            for _ in range(abs(steps)):
                moved = np.nextafter(moved, np.float32(steps * 1e9))
            check_select(logits, torch.tensor([[s[0], moved]], dtype=torch.float32, device=cuda_device), 6)


@pytest.mark.parametrize("vocab", [63, 64, 65, 255, 256, 257, 511, 513, 1023, 1025, 2082, 2111, 4097, 8191, 8193, 8194, 9000, 20001])
def test_short_rows_and_ends_of_rows(cuda_device, vocab):
    """Fewer logits than a span takes, at any place of a vector, with more kept than the span has buckets."""
    for dtype, beams, keep in ((torch.bfloat16, 3, 64), (torch.float16, 2, 33), (torch.float32, 4, 17)):
        logits, scores, _ = select_case(vocab, 2, beams, vocab + 3, dtype, cuda_device)
        for skip in (0, 1, 3):
            view = logits[:, skip:skip + vocab]
            check_select(view, scores, keep)
        masked = logits[:, :vocab].clone()
        masked[:, vocab // 3:vocab // 3 + vocab // 2] = -torch.inf
        masked[1] = -torch.inf
        masked[1, vocab - 40:] = 1.0
        check_select(masked, scores, keep)


@pytest.mark.parametrize("beams,vocab,keep,dtype", [
    (32, 32001, 64, torch.bfloat16), (32, 32001, 64, torch.float32), (16, 70001, 40, torch.float16), (2, 262144, 64, torch.bfloat16),
    (12, 12626, 33, torch.float32),
])
def test_one_beam_has_nearly_all_of_the_best(cuda_device, beams, vocab, keep, dtype):
    """The first entries of the other beams' lists say nothing about the keep-th best."""
    logits, scores, _ = select_case(vocab, 3, beams, vocab, dtype, cuda_device)
    scores[0, 1:] -= 100.0
    scores[1] = torch.linspace(0.0, -30.0, beams, device=cuda_device)
    scores[2] = -1.0
    check_select(logits, scores, keep)
    logits[beams:2 * beams] = (logits[beams:2 * beams] * 2).round() / 2  # many equal ones
    logits[2 * beams:] = logits[2 * beams]                               # the same beam everywhere
    check_select(logits, scores, keep)
    finished = torch.zeros((3, beams), dtype=torch.bool, device=cuda_device)
    finished[:, 0] = True
    check_select(logits, scores, keep, finished, 5)


def test_equal_and_nearly_equal_beams_wherever_their_rows_begin(cuda_device):
    """Beams with the same row and score tie at every token, and the lower beam comes first; rows of 16 bytes and an odd
    rest begin at other places of a vector.  One step of a score turns the order."""
    for dtype in LOWEST:
        for vocab, beams, keep in ((5, 2, 4), (2051, 3, 9), (32001, 8, 16), (128256, 2, 8)):
            row, _, _ = select_case(vocab, 1, 1, vocab, dtype, cuda_device)
            row[0, ::7] = -torch.inf
            logits = row.repeat(2 * beams, 1)
            scores = torch.full((2, beams), -3.25, device=cuda_device)
            scores[1, -1] = float(np.nextafter(np.float32(-3.25), np.float32(0)))
            out = check_select(logits, scores, keep)
            tied = out[0][0][1:] == out[0][0][:-1]
            assert bool((out[1][0][1:] > out[1][0][:-1])[tied & (out[2][0][1:] == out[2][0][:-1])].all())
            assert out[1][1, 0] == beams - 1


def test_masked_tokens_beams_and_rows(cuda_device):
    for dtype in LOWEST:
        logits, scores, _ = select_case(7, 3, 4, 12345, dtype, cuda_device)
        logits[0, 3:] = -torch.inf                 # three tokens left
        logits[1] = -torch.inf                     # none
        logits[2, 100:] = LOWEST[dtype]            # the type's lowest value as a mask
        logits[3] = LOWEST[dtype]                  # a whole row of it
        logits[4, 77] = torch.nan
        logits[5, 78] = torch.inf
        logits[6, ::2] = -torch.inf
        scores[1] = torch.tensor([0.0, -torch.inf, -1e30, torch.nan], device=cuda_device)
        scores[2] = torch.tensor([-torch.inf, LOWEST[torch.float32], -torch.inf, -1e9], device=cuda_device)
        check_select(logits, scores, 16)
        check_select(logits[:4], scores[:1], 64)


def test_few_allowed_tokens_leave_the_lowest_of_minus_infinity(cuda_device):
    logits = torch.full((2, 40000), -torch.inf, device=cuda_device, dtype=torch.bfloat16)
    logits[0, 39999], logits[1, 20000], logits[1, 5] = 1.0, 2.0, 0.5
    check_select(logits, torch.tensor([[-1.0, -0.5]], device=cuda_device), 9)


def test_finished_beams_offer_their_end_token_alone(cuda_device):
    logits, scores, _ = select_case(9, 2, 4, 30000, torch.bfloat16, cuda_device)
    logits[1] = torch.nan  # nobody looks at a finished beam's logits
    finished = torch.tensor([[False, True, True, False], [True] * 4], device=cuda_device)
    scores[0, 1] = -0.001
    out = check_select(logits, scores, 8, finished, 29999)
    assert out[1][0, 0] == 1 and out[2][0, 0] == 29999 and bool(out[3][0, 0])
    check_select(logits, scores, 8, finished, 0)
    check_select(logits[4:], scores[1:], 3, None, 11)  # an end token, and no beam that has finished


@pytest.mark.parametrize("dtype,offset", [(torch.bfloat16, 0), (torch.bfloat16, 3), (torch.float16, 7), (torch.float32, 1)])
def test_rows_of_a_wider_array(cuda_device, dtype, offset):
    wider, scores, _ = select_case(11, 2, 3, 9000, dtype, cuda_device)
    check_select(wider[:, offset:offset + 8500 + offset], scores, 6)
    stack = torch.stack([wider, -wider], 1)  # the last position of [rows, positions, vocabulary]
    check_select(stack[:, -1], scores, 6)
    assert all(torch.equal(a, b) for a, b in zip(B.beam_select(wider.t().contiguous().t(), scores), B.beam_select(wider, scores)))


def test_a_group_alone_and_in_a_batch_has_the_same_bits(cuda_device):
    logits, scores, _ = select_case(13, 6, 4, 20011, torch.bfloat16, cuda_device)
    together = B.beam_select(logits, scores, keep=8)
    for g in range(6):
        alone = B.beam_select(logits[4 * g:4 * g + 4].clone(), scores[g:g + 1], keep=8)
        assert all(torch.equal(a, b[g:g + 1]) for a, b in zip(alone, together)), g


def test_selection_refusals(cuda_device):
    logits, scores, finished = select_case(15, 2, 4, 100, torch.bfloat16, cuda_device, True)
    for error, call in [
        (TypeError, lambda: B.beam_select(logits.double(), scores)), (TypeError, lambda: B.beam_select(logits, scores.half())),
        (ValueError, lambda: B.beam_select(logits, scores[:1])), (ValueError, lambda: B.beam_select(logits, scores, keep=0)),
        (ValueError, lambda: B.beam_select(logits, scores, keep=65)), (ValueError, lambda: B.beam_select(logits, scores, finished=finished)),
        (ValueError, lambda: B.beam_select(logits, scores, finished=finished, end_token=100)),
        (ValueError, lambda: B.beam_select(logits, scores, end_token=-1)), (ValueError, lambda: B.beam_select(logits, scores.cpu())),
        (ValueError, lambda: B.beam_select(logits, scores, finished=finished.int(), end_token=1)),
        (ValueError, lambda: B.beam_select(logits[:, :1], scores, keep=5)),
        (ValueError, lambda: B.beam_select(logits.clone().requires_grad_(), scores)),
        (ValueError, lambda: B.beam_select(torch.zeros((33, 9), device=cuda_device), torch.zeros((1, 33), device=cuda_device))),
    ]:
        with pytest.raises(error):
            call()
    assert B.beam_select(logits[:0], scores[:0])[2].shape == (0, 4)


# ---- reordering -----------------------------------------------------------------------------------------------------


def reorder_case(seed, groups, beams, length, page, width, layers, heads, dim, dtype, layout, device):
    rng = np.random.default_rng(seed)
    block = min(length // page, width)
    pool = groups * beams * width + 2
    tables = rng.permutation(pool)[:groups * beams * width].reshape(groups, beams, width).astype(np.int32)
    for g in range(groups):  # full pages are shared as earlier steps left them
        for j in range(block):
            tables[g, :, j] = tables[g, rng.integers(0, beams, beams), j]
    parents = rng.integers(0, beams, (groups, beams)).astype(np.int32)
    generator = torch.Generator().manual_seed(seed)

    def pages():
        if layout == "token":
            return torch.randn((pool, page, heads, dim), generator=generator).to(dtype).to(device).transpose(1, 2)
        if layout == "pool":
            return torch.randn((pool, 2, heads, page, dim), generator=generator).to(dtype).to(device)[:, 0]
        return torch.randn((pool, heads, page, dim), generator=generator).to(dtype).to(device)

    caches = [(pages(), pages()) for _ in range(layers)]
    return tables.reshape(groups * beams, width), np.full(groups * beams, length, np.int32), parents, caches


@pytest.mark.parametrize("groups,beams,length,page,width,layers,heads,dim,dtype,layout", [
    (1, 1, 5, 8, 2, 1, 1, 8, torch.bfloat16, "head"), (1, 4, 37, 16, 5, 3, 2, 128, torch.bfloat16, "head"),
    (3, 8, 63, 32, 3, 2, 2, 64, torch.float16, "token"), (2, 5, 64, 16, 6, 1, 1, 40, torch.bfloat16, "pool"),
    (2, 3, 0, 16, 2, 1, 2, 64, torch.bfloat16, "head"), (1, 2, 32, 16, 2, 1, 2, 64, torch.bfloat16, "head"),
    (2, 32, 77, 64, 3, 1, 1, 64, torch.float16, "head"), (1, 6, 129, 128, 2, 70, 1, 16, torch.bfloat16, "token"),
    (4, 16, 9, 8, 4, 2, 4, 128, torch.bfloat16, "head"),
])
def test_reordering_against_the_oracle(cuda_device, groups, beams, length, page, width, layers, heads, dim, dtype, layout):
    tables, lengths, parents, caches = reorder_case(beams * 7 + length, groups, beams, length, page, width, layers, heads, dim, dtype, layout,
                                                    cuda_device)
    flat = [wide(pages) for pair in caches for pages in pair]
    expected, moved = O.reorder(tables, lengths, parents, flat, page)
    arguments = (torch.tensor(tables, device=cuda_device), torch.tensor(lengths, device=cuda_device), torch.tensor(parents, device=cuda_device))
    for _ in range(2):  # the copied pages belong to beams without children: the same call does the same again
        out = B.beam_reorder(*arguments, caches)
        assert np.array_equal(out.cpu().numpy(), expected)
        for pages, right in zip((pages for pair in caches for pages in pair), moved):
            assert np.array_equal(wide(pages), right)
    assert np.array_equal(arguments[0].cpu().numpy(), tables)


def test_the_same_parents_or_one_parent_for_all(cuda_device):
    for pattern in ([0, 1, 2, 3], [3, 2, 1, 0], [2, 2, 2, 2], [0, 0, 3, 3]):
        tables, lengths, _, caches = reorder_case(5, 2, 4, 21, 16, 3, 2, 2, 64, torch.bfloat16, "head", cuda_device)
        parents = np.array([pattern, pattern[::-1]], np.int32)
        expected, moved = O.reorder(tables, lengths, parents, [wide(p) for pair in caches for p in pair], 16)
        out = B.beam_reorder(torch.tensor(tables, device=cuda_device), torch.tensor(lengths, device=cuda_device),
                             torch.tensor(parents, device=cuda_device), caches)
        assert np.array_equal(out.cpu().numpy(), expected)
        assert all(np.array_equal(wide(p), m) for p, m in zip((p for pair in caches for p in pair), moved))


def test_parents_pages_and_lengths_outside_are_recorded(cuda_device):
    tables, lengths, _, caches = reorder_case(6, 1, 3, 21, 16, 3, 1, 2, 64, torch.bfloat16, "head", cuda_device)
    before = [p.clone() for p in caches[0]]
    device = lambda a: torch.tensor(a, device=cuda_device)  # noqa: E731

    def status():
        ok, words = _lib.device_status()
        assert not ok
        return words[:3]

    out = B.beam_reorder(device(tables), device(lengths), torch.tensor([[0, 7, 2]], dtype=torch.int32, device=cuda_device), caches)
    assert status() == (0x305, 1, 7) and np.array_equal(out.cpu().numpy(), tables)
    bad = tables.copy()
    bad[1, 1] = 10**6
    B.beam_reorder(device(bad), device(lengths), torch.tensor([[0, 0, 2]], dtype=torch.int32, device=cuda_device), caches)
    assert status() == (0x303, 1, 10**6)
    for length in (49, -1):
        out = B.beam_reorder(device(tables), device(np.full(3, length, np.int32)),
                             torch.tensor([[1, 1, 2]], dtype=torch.int32, device=cuda_device), caches)
        assert status() == (0x304, 0, length & 0xFFFFFFFF)
    assert all(torch.equal(a, b) for a, b in zip(before, caches[0]))


def test_reordering_refusals(cuda_device):
    tables, lengths, parents, caches = reorder_case(8, 2, 4, 21, 16, 3, 2, 2, 64, torch.bfloat16, "head", cuda_device)
    t, n, p = (torch.tensor(a, device=cuda_device) for a in (tables, lengths, parents))
    for error, call in [
        (ValueError, lambda: B.beam_reorder(t[:4], n, p, caches)), (ValueError, lambda: B.beam_reorder(t, n[:4], p, caches)),
        (TypeError, lambda: B.beam_reorder(t, n, p.long(), caches)), (ValueError, lambda: B.beam_reorder(t, n, p, [])),
        (ValueError, lambda: B.beam_reorder(t, n, p, [caches[0], (caches[1][0], caches[1][1][:-1])])),
        (ValueError, lambda: B.beam_reorder(t, n, p, [caches[0], tuple(c.half() for c in caches[1])])),
        (TypeError, lambda: B.beam_reorder(t, n, p, [tuple(c.float() for c in caches[1])])),
        (ValueError, lambda: B.beam_reorder(t.cpu(), n, p, caches)),
    ]:
        with pytest.raises(error):
            call()
