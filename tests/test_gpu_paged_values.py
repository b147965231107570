"""Decode attention over pages: values that are not finite."""

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
