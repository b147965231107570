"""Log-probabilities of given tokens, entropies and alternatives against the oracle (64 bits).

Tolerance.  A term e^d of a row's sum is off by 2^-22 (ex2.approx), by |d| 2^-24 + |d| 2^-23 for d and for d log2 e rounded, and a sum
adds 2^-24 for each of up to 76 additions in a row (64 of a thread, 5 over the warp, 7 over the warps): relative to the sum
(2^-22 + 2^-22 m + 76 2^-24) where m, the mean of |d| by the weights, is the entropy at most plus log of the sum, so at most twice
the log of the vocabulary.  A log-probability is off by that and by the rounding of its result; the sum of e^d d is off by as much of
its own terms, whose size is m, so an entropy by (1 + 2 m) times it."""

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


def check(logits, tokens, top):
    got = B.token_logprobs(logits, tokens, top=top)
    rows, vocab = logits.shape
    assert [t.shape for t in got] == [(rows,), (rows,), (rows, top), (rows, top)]
    assert [t.dtype for t in got] == [torch.float32] * 3 + [torch.int64]
    logprobs, entropy, best, where = O.token_logprobs(logits.cpu().double().numpy(), tokens.cpu().numpy(), top)
    m = 2 * np.log(max(vocab, 2))
    error = 2.0 ** -22 + 2.0 ** -22 * m + 76 * 2.0 ** -24
    for what, a, b, e in (("logprobs", got[0], logprobs, error), ("entropy", got[1], entropy, error * (1 + 2 * m)), ("top", got[2], best, error)):
        a = a.cpu().double().numpy()
        same = np.isclose(a, b, rtol=2.0 ** -24, atol=e, equal_nan=True) | (a == b)
        assert same.all(), (what, np.abs(a - b)[~same].max())
    assert np.array_equal(got[3].cpu().numpy(), where)
    again = B.token_logprobs(logits, tokens, top=top)
    assert all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip(got, again))
    return got


def normal(seed, *shape, device, dtype, std=2.5):
    generator = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=generator) * std).to(dtype).to(device)


def chosen(seed, rows, vocab, device):
    return torch.randint(0, vocab, (rows,), generator=torch.Generator().manual_seed(seed)).to(device)


@pytest.mark.parametrize("rows,vocab,top,dtype", [
    (1, 1, 1, torch.bfloat16), (3, 2, 2, torch.float32), (7, 5, 0, torch.float16), (5, 63, 63, torch.bfloat16), (4, 64, 64, torch.float32),
    (9, 1000, 5, torch.float16), (8, 32001, 5, torch.bfloat16), (3, 16384, 20, torch.bfloat16), (3, 16385, 20, torch.float16),
    (2, 8193, 64, torch.float32), (5, 128256, 20, torch.bfloat16), (2, 131071, 64, torch.float32), (1, 524288, 3, torch.bfloat16),
    (300, 4097, 1, torch.float16),
])
def test_against_the_oracle(cuda_device, rows, vocab, top, dtype):
    check(normal(rows + vocab, rows, vocab, device=cuda_device, dtype=dtype), chosen(vocab, rows, vocab, cuda_device), top)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_equal_logits_go_by_the_lower_token(cuda_device, dtype):
    generator = torch.Generator().manual_seed(1)
    few = torch.randint(-2, 3, (6, 40000), generator=generator).to(dtype).to(cuda_device)
    few[3] = 1.0
    few[4, ::3], few[4, 1::3] = 0.0, -0.0
    few[5] = -1.0
    few[5, 39000:] = 5.0  # the best all lie in one stretch
    check(few, chosen(2, 6, 40000, cuda_device), 64)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_best_entries_in_few_places(cuda_device, dtype):
    """Entries 2048 (fp32: 1024) apart, and all of them side by side."""
    logits = normal(4, 2, 50000, device=cuda_device, dtype=dtype, std=1.0)
    step = 2048 if dtype == torch.bfloat16 else 1024
    logits[0, 5::step] = 20.0 + torch.arange(len(range(5, 50000, step)), device=cuda_device) % 3
    logits[1, :600] = 30.0
    check(logits, chosen(5, 2, 50000, cuda_device), 64)


@pytest.mark.parametrize("rows,vocab,top,dtype", [
    (1100, 4099, 20, torch.bfloat16), (1024, 33, 33, torch.float32), (1031, 20480, 64, torch.float16), (1025, 9001, 3, torch.bfloat16),
])
def test_many_rows(cuda_device, rows, vocab, top, dtype):
    check(normal(rows + vocab, rows, vocab, device=cuda_device, dtype=dtype), chosen(vocab, rows, vocab, cuda_device), top)


@pytest.mark.parametrize("rows", [7, 1024])
@pytest.mark.parametrize("vocab,top,dtype", [(1000, 5, torch.bfloat16), (5001, 20, torch.float16), (20479, 64, torch.bfloat16), (30003, 64, torch.float32),
                                             (33000, 1, torch.float16), (20737, 64, torch.bfloat16)])
def test_where_the_best_lie(cuda_device, rows, vocab, top, dtype):
    """Rising and falling rows, constant ones, all but a few tokens masked, and hundreds of equal ones behind a few larger ones."""
    logits = normal(vocab, rows, vocab, device=cuda_device, dtype=dtype)
    position = torch.arange(vocab, device=cuda_device)
    logits[0] = position.to(dtype) / 16
    logits[1] = -(position.to(dtype)) / 16
    logits[2] = -3.0
    logits[3] = -torch.inf
    logits[3, vocab // 3:vocab // 3 + 7] = torch.arange(7, device=cuda_device).to(dtype)
    logits[4] = torch.finfo(dtype).min
    logits[4, -9:] = 1.0
    logits[5, vocab // 4:vocab // 4 + 700] = 40.0
    logits[5, -3:] = 41.0
    logits[6] = 0.0
    logits[6, ::2] = -0.0
    logits[6, vocab - 1] = 1.0
    # (The oracle looks at some rows; the others are held to each other.)
    tokens = chosen(vocab, rows, vocab, cuda_device)
    got = check(logits[:7], tokens[:7], top)
    whole = B.token_logprobs(logits, tokens, top=top)
    assert all(torch.equal(a, b[:7]) for a, b in zip(got, whole))
    wide = torch.zeros((7, vocab + 5), dtype=dtype, device=cuda_device)
    for offset in (1, 5):
        wide[:, offset:offset + vocab] = logits[:7]
        assert all(torch.equal(a, b) for a, b in zip(got, B.token_logprobs(wide[:, offset:offset + vocab], tokens[:7], top=top)))


def test_rows_that_start_anywhere(cuda_device):
    for dtype, offset in ((torch.bfloat16, 3), (torch.float16, 1), (torch.float32, 2), (torch.bfloat16, 7)):
        whole = torch.full((6, 20011), torch.nan, dtype=dtype, device=cuda_device)
        whole[:, offset:offset + 17003] = normal(offset, 6, 17003, device=cuda_device, dtype=dtype)
        rows = whole[:, offset:offset + 17003]
        tokens = chosen(offset, 6, 17003, cuda_device)
        got = check(rows, tokens, 7)
        dense = B.token_logprobs(rows.contiguous(), tokens, top=7)
        one = B.token_logprobs(rows[2:3], tokens[2:3], top=7)
        assert all(torch.equal(a, b) for a, b in zip(got, dense)) and all(torch.equal(a[2:3], b) for a, b in zip(got, one))
    wide = normal(9, 300, 5, device=cuda_device, dtype=torch.float32).T  # the vocabulary is not dense
    check(wide, chosen(9, 5, 300, cuda_device), 4)
    same = normal(10, 1, 999, device=cuda_device, dtype=torch.bfloat16).expand(4, 999)
    check(same, chosen(10, 4, 999, cuda_device), 4)


def test_masked_logits_and_rows_without_a_distribution(cuda_device):
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        logits = normal(11, 9, 40001, device=cuda_device, dtype=dtype)
        logits[0, 1:] = -torch.inf                       # one token is left
        logits[1] = -torch.inf                           # none
        logits[2, 20000] = torch.nan
        logits[3, 39999] = torch.inf
        logits[4, :39000] = -torch.inf                   # whole parts of nothing
        logits[5] = torch.finfo(dtype).min               # a mask of the type's lowest value, everywhere
        logits[6, 7:] = torch.finfo(dtype).min
        logits[7, 5:] = -torch.inf
        tokens = torch.tensor([0, 3, 4, 39999, 39500, 8, 2, 100, -100], device=cuda_device)
        got = check(logits, tokens, 8)
        assert got[0][0] == 0 and got[1][0] == 0 and got[0][8] == 0 and got[0][7] == -torch.inf
        assert torch.isnan(got[0][1:4]).all() and torch.isnan(got[1][1:4]).all() and (got[3][1:4] == -1).all()


def test_a_token_outside_the_vocabulary_is_recorded(cuda_device):
    logits = normal(12, 3, 100, device=cuda_device, dtype=torch.bfloat16)
    got = B.token_logprobs(logits, torch.tensor([5, 100, 2 ** 40], device=cuda_device), top=1)
    ok, words = _lib.device_status()
    assert not ok and words[0] == 0x307 and words[1] in (1, 2)
    assert torch.isnan(got[0]).tolist() == [False, True, True] and torch.isfinite(got[1]).all()


def test_a_captured_call_and_another_stream(cuda_device):
    logits, tokens = normal(13, 4, 33000, device=cuda_device, dtype=torch.bfloat16), chosen(13, 4, 33000, cuda_device)
    B.token_logprobs(logits, tokens, top=3)
    stream, graph = torch.cuda.Stream(cuda_device), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        out = B.token_logprobs(logits, tokens, top=3)
    for seed in (14, 15):
        logits.copy_(normal(seed, 4, 33000, device=cuda_device, dtype=torch.bfloat16))
        tokens.copy_(chosen(seed, 4, 33000, cuda_device))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, B.token_logprobs(logits, tokens, top=3)))


def test_refusals_and_no_rows(cuda_device):
    logits, tokens = normal(16, 4, 50, device=cuda_device, dtype=torch.bfloat16), chosen(16, 4, 50, cuda_device)
    for arguments, error in (((logits.int(), tokens, 0), TypeError), ((logits.cpu(), tokens, 0), ValueError), ((logits[0], tokens, 0), ValueError),
                             ((logits, tokens.int(), 0), ValueError), ((logits, tokens[:3], 0), ValueError), ((logits, tokens.cpu(), 0), ValueError),
                             ((logits, tokens[:, None], 0), ValueError), ((logits, None, 0), TypeError), ((logits, tokens, 51), ValueError),
                             ((logits, tokens, -1), ValueError), ((logits, tokens, 1.5), ValueError), ((logits[:, :0], tokens, 0), ValueError),
                             ((logits.clone().requires_grad_(), tokens, 0), ValueError), ((logits.double(), tokens, 0), TypeError)):
        with pytest.raises(error):
            B.token_logprobs(arguments[0], arguments[1], top=arguments[2])
    got = B.token_logprobs(logits[:0], tokens[:0], top=3)
    assert [t.shape for t in got] == [(0,), (0,), (0, 3), (0, 3)]
    assert all(torch.equal(a, b) for a, b in zip(B.token_logprobs(logits, tokens.repeat_interleave(2)[::2], top=3), B.token_logprobs(logits, tokens, top=3)))
