"""Decode attention over pages: values that are not finite, and weights that 16 bits do not reach."""

import math

import numpy as np
import pytest
import torch

from metile_b200 import _lib, backends as B

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def nothing_was_recorded(cuda_device):
    yield
    ok, words = _lib.device_status()
    assert ok, [hex(w) for w in words]


def ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def case(lengths, heads, kv_heads, dim, dtype, device, page=16, width=None):
    """Pages in order: token t of request b lies in page b * width + t // page."""
    generator = torch.Generator().manual_seed(sum(lengths))
    width = width or -(-max(lengths) // page)
    shape = (len(lengths) * width, kv_heads, page, dim)
    q, keys, values = (torch.randn(s, generator=generator).to(dtype).to(device) for s in ((len(lengths), heads, dim), shape, shape))
    return q, keys, values, torch.arange(len(lengths) * width, dtype=torch.int32, device=device).view(len(lengths), width), ints(lengths, device)


# One split, the one-launch join (up to four splits) and the join kernel, with one slice and with several.
@pytest.mark.parametrize("length,width,kv_heads", [(1, 1, 2), (5, 1, 2), (129, 9, 2), (257, 64, 2), (513, 64, 4), (897, 300, 2), (20000, 1300, 1)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_nan_that_is_used_comes_out(cuda_device, length, width, kv_heads, dtype):
    heads, dim, page = 3 * kv_heads, 64, 16
    q, keys, values, table, lengths = case([length, 40], heads, kv_heads, dim, dtype, cuda_device, width=max(width, 3))
    clean = B.paged_attention_decode(q, keys, values, table, lengths, scale=0.1)
    assert bool(torch.isfinite(clean).all())

    def poisoned(query=None, key=None, value=None):
        q2, k2, v2 = q.clone(), keys.clone(), values.clone()
        if query is not None:
            q2[0, query, 3] = torch.nan
        if key is not None:
            k2[key // page, kv_heads - 1, key % page, 5] = torch.nan
        if value is not None:
            v2[value // page, kv_heads - 1, value % page, 7] = torch.nan
        return torch.isnan(B.paged_attention_decode(q2, k2, v2, table, lengths, scale=0.1)), \
            B.paged_attention_decode(q2, k2, v2, table, lengths, scale=0.1)

    last = torch.zeros((2, heads, dim), dtype=torch.bool, device=cuda_device)
    last[0, heads - 3:] = True  # the query heads of the last key head
    for at in {0, length // 2, length - 1}:
        nan, out = poisoned(key=at)
        assert torch.equal(nan, last), at
        assert torch.equal(out[~last], clean[~last])
        nan, out = poisoned(value=at)
        only = torch.zeros_like(last)
        only[0, heads - 3:, 7] = True
        assert torch.equal(nan, only), at
    nan, out = poisoned(query=1)
    only = torch.zeros_like(last)
    only[0, 1] = True
    assert torch.equal(nan, only) and torch.equal(out[~only], clean[~only])
    if length % page:  # and one behind the last token does not
        behind = keys.clone()
        behind[length // page, :, length % page:] = torch.nan
        assert torch.equal(B.paged_attention_decode(q, behind, values, table, lengths, scale=0.1), clean)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_many_small_weights_beside_a_large_one(cuda_device, dtype):
    """Token 0 has a score of 18 above all others; the 2^23 - 1 others, 2^-26 of its weight each and 65536 in a split,
    make an eighth of the sum.  Two pages serve all blocks of the table."""
    tokens, page, dim, kv_heads = 1 << 23, 256, 64, 4
    keys = torch.zeros((2, kv_heads, page, dim), dtype=dtype, device=cuda_device)
    values = torch.ones_like(keys)
    keys[0, :, 0, 0], values[0, :, 0] = 18.0, 0.0
    q = torch.zeros((1, kv_heads, dim), dtype=dtype, device=cuda_device)
    q[..., 0] = 1.0
    table = torch.ones((1, tokens // page), dtype=torch.int32, device=cuda_device)
    table[0, 0] = 0
    out = B.paged_attention_decode(q, keys, values, table, ints([tokens], cuda_device), scale=1.0).double().cpu().numpy()
    small = (tokens - 1) * math.exp(-18.0)
    expected = small / (1.0 + small)
    # Half a step of the type; 2^-22 for an exponential and 2^-24 * 26 for its argument in the small part; sums of 32 bits,
    # 4096 chunks a split one after the other and each of two products, at 2^-24 of what is there (twice a truncating sum's).
    bound = torch.finfo(dtype).eps / 2 + 2.0 ** -22 + 26 * 2.0 ** -24 + 2 * 2 * 4096 * 2.0 ** -24
    assert float(np.abs(out / expected - 1.0).max()) <= bound
