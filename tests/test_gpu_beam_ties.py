"""Beam selection where very many candidates are equal or nearly so: the order is the one of the exact sums, and a
group's bits are its own whatever else is in the call."""

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


def wide(tensor):
    return tensor.detach().cpu().double().numpy()


def quantised_rows(seed, rows, vocab, device, levels=40):
    """Logits of few levels (capped or quantised heads): the largest one stands in every part of a row many times over."""
    generator = torch.Generator().manual_seed(seed)
    return (torch.randint(0, levels, (rows, vocab), generator=generator) / 8).to(torch.bfloat16).to(device)


def log_sums(logits):
    rows = wide(logits)
    top = rows.max(1)
    return top, np.log(np.exp(rows - top[:, None]).sum(1))


def check(logits, scores, keep):
    out = B.beam_select(logits, scores, keep=keep)
    expected = O.beam_select(wide(logits), wide(scores), keep)
    assert np.array_equal(out[1].cpu().numpy(), expected[1]) and np.array_equal(out[2].cpu().numpy(), expected[2])
    # Half a step of 32 bits, and the bound of a log-sum of 32-bit exponentials.
    assert (np.abs(wide(out[0]) - expected[0]) <= 2.0 ** -24 * np.abs(expected[0]) + 2.0 ** -18).all()
    return out


def own_order(row, keep):
    """The tokens of one beam in the order of their logits, the lower token first among equals."""
    row = wide(row)
    return np.lexsort((np.arange(row.size), -row))[:keep]


@pytest.mark.parametrize("beams,vocab,keep,dtype", [
    (23, 524288, 4, torch.float32), (1, 524288, 4, torch.float32), (8, 128256, 16, torch.bfloat16), (2, 300, 64, torch.bfloat16),
    (32, 50001, 1, torch.float32), (5, 77777, 33, torch.float32),
])
def test_logits_that_64_bits_cannot_tell_apart(cuda_device, beams, vocab, keep, dtype):
    """Logits far below the log of their sum, or far below the largest one: all are worth the same in 64 bits and go by
    themselves.  In every part of a row but one the largest stand in front; in that one the very largest comes last."""
    generator = torch.Generator().manual_seed(vocab)
    tiny = (torch.rand((beams, vocab), generator=generator) * 2.0 ** -80).to(dtype)
    if vocab == 524288:  # 25 parts for 23 rows: the middle of the row lies inside the thirteenth
        step = torch.arange(vocab) % 20972
        tiny[0] = (torch.where(step < 4, 2.0 - step / 8, 1.0) * 2.0 ** -80).to(dtype)
        tiny[0, 262144 - 3:262144] = 2.5 * 2.0 ** -80
        tiny[0, 262144 + 9] = 3.0 * 2.0 ** -80
    logits = tiny.to(cuda_device)
    scores = torch.full((1, beams), -50.0, device=cuda_device)
    scores[0, 0] = -1.0
    for alone in (False, True):
        if alone:  # all but one token 1e30 below it; by itself, since any other beam would come before them
            logits[0, 7] = 1e30
        got, parents, tokens, _ = B.beam_select(logits[:1] if alone else logits, scores[:, :1].contiguous() if alone else scores, keep=keep)
        assert not parents.any()
        assert np.array_equal(tokens[0].cpu().numpy(), own_order(logits[0], keep))
        worth = -1.0 - (0.0 if alone else np.log(vocab))
        assert abs(float(got[0, 0]) - worth) <= 2.0 ** -24 * abs(worth) + 2.0 ** -18
    # Beams that are one row throughout tie with each other too: the lower one first.
    got, parents, tokens, _ = B.beam_select(logits[:1].expand(beams, -1), torch.zeros((1, beams), device=cuda_device), keep=keep)
    first = min(beams, keep)  # every beam's token 7 is worth 0, all others 1e30 less
    assert parents[0, :first].tolist() == list(range(first)) and tokens[0, :first].tolist() == [7] * first and not got[0, :first].any()
    assert not parents[0, first:].any() and np.array_equal(tokens[0, first:].cpu().numpy(), own_order(logits[0], keep)[1:keep - first + 1])


@pytest.mark.parametrize("beams,keep", [(2, 16), (8, 4), (3, 40)])
def test_hundreds_of_equal_candidates_in_two_beams_a_hair_apart(cuda_device, beams, keep):
    """More candidates within the margin of the sums than are collected: the beam whose exact value is larger comes first,
    by however little (64 bits leave 1e-14 here)."""
    for seed in range(4):
        logits = quantised_rows(10 * beams + seed, beams, 128256, cuda_device)
        _, sums = log_sums(logits)  # the rows have the same largest logit
        for apart in (1e-8, 3e-8, 1e-7, 3e-7, 1e-6):
            for sign in (-1.0, 1.0):
                given = sums - sums[0] - 0.1  # all beams' best are worth the same
                given[0] = 0.0
                given[1] = sums[1] - sums[0] + sign * apart
                check(logits, torch.tensor(given[None], dtype=torch.float32, device=cuda_device), keep)


@pytest.mark.parametrize("beams,keep,dtype", [(3, 16, torch.bfloat16), (8, 4, torch.bfloat16), (8, 16, torch.float32), (2, 64, torch.float16)])
def test_a_group_has_the_same_bits_however_its_rows_are_cut(cuda_device, beams, keep, dtype):
    """Alone a row is cut into sixteen parts or more, in a batch of 32 into a few.  The values lie near zero, where a score
    shows how its log-sum was taken: beams 0 and 1 have hundreds of equal candidates a hair apart, the others a few above."""
    generator = torch.Generator().manual_seed(beams)
    logits = (torch.randn((32 * beams, 128256), generator=generator) * 2.5).to(dtype).to(cuda_device)
    scores = torch.zeros((32, beams), device=cuda_device)
    for g in range(32):
        if g % 4 < 3:
            logits[g * beams:g * beams + 2] = quantised_rows(g, 2, 128256, cuda_device).to(dtype)
        _, sums = log_sums(logits[g * beams:(g + 1) * beams])
        given = sums + 0.01 * np.arange(beams)
        if g % 4 < 3:
            given[:2] = sums[:2] - (0.2 if g % 4 < 2 else 0.0)
            given[1] += (2e-8, -1e-7, 1e-5, 0.0)[g % 4]
        scores[g] = torch.tensor(given, dtype=torch.float32, device=cuda_device)
    together = B.beam_select(logits, scores, keep=keep)
    for g in range(0, 32, 3):
        rows = slice(g * beams, (g + 1) * beams)
        alone = check(logits[rows].clone(), scores[g:g + 1], keep)
        assert all(torch.equal(a, b[g:g + 1]) for a, b in zip(alone, together)), g
        few = B.beam_select(logits[:(g + 1) * beams], scores[:g + 1], keep=keep)
        assert all(torch.equal(a[g:], b[g:g + 1]) for a, b in zip(few, together)), g


def test_a_log_sum_does_not_follow_the_order_of_the_maxima(cuda_device):
    """Eight stretches of a long row whose maxima rise, fall or go up and down: every logit is weighted against the row's
    maximum through two exponentials, wherever it stands, and the rest is added in 64 bits."""
    stretches = torch.linspace(0.0, 1.0, 524288, dtype=torch.float64).float().view(8, 65536)
    scores = torch.full((4, 1), 12.7, device=cuda_device)  # the value is near zero, where 32 bits show 64
    rows = torch.stack([stretches[order].reshape(-1) for order in (
        [0, 1, 2, 3, 4, 5, 6, 7], [7, 6, 5, 4, 3, 2, 1, 0], [3, 6, 0, 7, 1, 5, 2, 4], [0, 2, 4, 6, 1, 3, 5, 7])]).to(cuda_device)
    top, sums = log_sums(rows[:1])
    scores[:] = float(np.float32(sums[0]))
    got = wide(B.beam_select(rows, scores, keep=1)[0])[:, 0]
    exact = float(scores[0]) - sums[0]
    # The two exponentials and the sums of 32 bits: 2 * 2^-22, 14 * 2^-24, and |d| * 1.33e-7 with |d| up to 1.
    assert (np.abs(got - exact) <= 2 * 2.0 ** -22 + 14 * 2.0 ** -24 + 1.33e-7).all()
    assert np.abs(got - got[0]).max() <= 1e-13  # sums of 64 bits near 13
