"""The paged cache and beam search without a GPU: refusals of the C ABI and of the operators, and the oracle itself
against small cases worked out by hand or by brute force."""

import ctypes

import numpy as np
import pytest
import torch

from metile_b200 import _lib, backends as B
from oracle import paged as O


def strides(*values):
    return (ctypes.c_longlong * 3)(*values)


ONE, BY16, OFF = ctypes.c_void_p(16), strides(1024, 512, 64), ctypes.c_void_p(24)


def test_resize_refusals_of_the_abi():
    lib = _lib.load()

    def call(table=ONE, stride=4, width=4, ring=ONE, pool=8, state=ONE, slots=ONE, starts=ONE, requests=2, page=16, tokens=3):
        return lib.mt_paged_resize(table, stride, width, ONE, ONE, ring, pool, state, slots, ONE, starts, ONE, ONE, requests, page,
                                   tokens, None)

    for bad in (dict(page=12), dict(page=4), dict(page=512), dict(requests=-1), dict(tokens=-1), dict(width=0), dict(pool=0), dict(stride=3)):
        assert call(**bad) == -1, bad
    for bad in (dict(table=None), dict(ring=None), dict(state=None), dict(slots=None), dict(starts=None)):
        assert call(**bad) == -6, bad


def test_append_refusals_of_the_abi():
    lib = _lib.load()

    def call(q=ONE, q_stride=128, v_stride=64, key_strides=BY16, rows=2, heads=2, kv_heads=1, dim=64, pages=4, page=16, type=0):
        return lib.mt_rope_kv_append_paged(q, q_stride, ONE, 64, ONE, v_stride, ONE, ONE, ONE, ONE, ONE, key_strides, ONE, BY16, rows,
                                           heads, kv_heads, dim, pages, page, type, None)

    for bad in (dict(rows=-1), dict(heads=0), dict(kv_heads=0), dict(dim=8), dict(dim=72), dict(dim=8192), dict(pages=0), dict(page=20),
                dict(type=2), dict(type=-1)):
        assert call(**bad) == -1, bad
    assert call(q=None) == -6 and call(key_strides=None) == -6 and call(rows=0) == 0
    for bad in (dict(q=OFF), dict(q_stride=100), dict(v_stride=4), dict(key_strides=strides(1024, 500, 64)), dict(key_strides=strides(-8, 8, 8))):
        assert call(**bad) == -2, bad


def test_attention_refusals_of_the_abi():
    lib = _lib.load()
    workspace = lib.mt_paged_attention_decode_workspace_bytes(2, 8, 2, 64, 100, 16)

    def call(q=ONE, value_strides=BY16, stride=100, width=100, batch=2, heads=8, kv_heads=2, dim=64, pages=9, page=16, type=0, space=ONE,
             size=workspace):
        return lib.mt_paged_attention_decode(q, ONE, BY16, ONE, value_strides, ONE, stride, width, ONE, ONE, space, size, batch, heads,
                                             kv_heads, dim, pages, page, type, 1.0, None)

    for bad in (dict(batch=-1), dict(heads=0), dict(heads=7), dict(kv_heads=0), dict(dim=96), dict(pages=0), dict(page=1), dict(type=2),
                dict(stride=99), dict(width=0), dict(width=2**27, stride=2**27), dict(batch=2**30)):
        assert call(**bad) == -1, bad
    assert call(q=None) == -6 and call(batch=0) == 0
    assert call(q=OFF) == -2 and call(value_strides=strides(8, 4, 8)) == -2
    if workspace:
        assert call(space=None) == -7 and call(size=workspace - 1) == -7 and call(space=OFF) == -7


def test_select_and_reorder_refusals_of_the_abi():
    lib = _lib.load()
    workspace = lib.mt_beam_select_workspace_bytes(2, 4, 100, 8, 0)

    def select(logits=ONE, type=0, finished=ONE, end=3, groups=2, beams=4, vocab=100, keep=8, space=ONE, size=workspace):
        return lib.mt_beam_select(logits, vocab, type, ONE, finished, end, ONE, ONE, ONE, ONE, space, size, groups, beams, vocab, keep, None)

    for bad in (dict(groups=-1), dict(beams=0), dict(beams=33), dict(vocab=0), dict(vocab=2**19 + 1), dict(keep=0), dict(keep=65),
                dict(vocab=1, end=0, keep=5), dict(type=3), dict(end=100), dict(end=-1), dict(finished=None, end=-2), dict(groups=2**19)):
        assert select(**bad) == -1, bad
    assert select(logits=None) == -6 and select(logits=ctypes.c_void_p(17)) == -2 and select(groups=0) == 0
    if workspace:
        assert select(space=None) == -7 and select(size=workspace - 1) == -7

    def reorder(out=ctypes.c_void_p(32), keys=(16,), caches=1, groups=2, beams=4, dim=64, heads=2, pages=9, page=16, key_strides=BY16, stride=5):
        addresses = (ctypes.c_void_p * len(keys))(*keys)
        return lib.mt_beam_reorder(ONE, stride, 5, ONE, ONE, out, addresses, key_strides, addresses, BY16, caches, groups, beams, heads, dim,
                                   pages, page, None)

    for bad in (dict(groups=-1), dict(beams=0), dict(beams=33), dict(dim=12), dict(heads=0), dict(pages=0), dict(page=6), dict(stride=4),
                dict(caches=-1), dict(out=ONE)):
        assert reorder(**bad) == -1, bad
    assert reorder(keys=(None,)) == -6 and reorder(keys=(24,)) == -2 and reorder(key_strides=strides(8, 8, 9)) == -2
    assert reorder(groups=0) == 0


def test_operators_refuse_cpu_tensors():
    table, n = torch.zeros((2, 3), dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    pages, rows = torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16), torch.zeros((2, 4, 64), dtype=torch.bfloat16)
    for call in (lambda: B.paged_resize(table, n, n, n, n, page_size=16, tokens=4),
                 lambda: B.rope_kv_append_paged(rows, rows[:, :2], rows[:, :2], torch.ones(32), n, n.long(), pages, pages),
                 lambda: B.paged_attention_decode(rows, pages, pages, table, n, scale=1.0),
                 lambda: B.beam_select(torch.zeros(4, 9), torch.zeros(1, 4)),
                 lambda: B.beam_reorder(table, n, table[:1, :2].contiguous(), [(pages, pages)])):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        B.paged_resize(table.long(), n, n, n, n, page_size=16, tokens=4)
    with pytest.raises(TypeError):
        B.beam_select([1.0], torch.zeros(1, 4))


def test_the_oracle_of_block_tables():
    tables = np.array([[5, -1, -1], [2, 7, -1]], np.int32)
    out = O.resize(tables, np.array([3, 9]), np.array([7, -5]), np.array([0, 1, 3, 9], np.int32), np.array([3, 2], np.int32), 8, 9)
    assert out[0].tolist() == [43, 44, 45, 46, 47, 72, 73, -1, -1]      # the rest of page 5, then page 9
    assert out[1].tolist() == [3, 4, 5, 6, 7, 8, 9, 0, 0] and out[2].tolist() == [0, 7, 7] and out[3].tolist() == [10, 4]
    assert out[4].tolist() == [0, 2] and out[5].tolist() == [[5, 9, -1], [2, 7, -1]]
    assert out[6].tolist() == [0, 7, 3, 9]                              # page 7 came back behind page 0


def test_the_oracle_of_beam_search_by_brute_force():
    rng = np.random.default_rng(1)
    logits, scores = rng.normal(size=(6, 7)), rng.normal(size=(2, 3))
    best, parents, tokens, done = O.beam_select(logits, scores, 5, end=4)
    for g in range(2):
        every = []
        for k in range(3):
            row = logits[3 * g + k]
            every += [(scores[g, k] + row[t] - np.log(np.exp(row).sum()), k, t) for t in range(7)]
        every.sort(key=lambda c: -c[0])
        assert np.allclose(best[g], [c[0] for c in every[:5]])
        assert [(int(a), int(b)) for a, b in zip(parents[g], tokens[g])] == [c[1:] for c in every[:5]]
        assert done[g].tolist() == [c[2] == 4 for c in every[:5]]


def test_the_oracle_of_reordering():
    pages = np.arange(8 * 1 * 4 * 1, dtype=float).reshape(8, 1, 4, 1)
    tables = np.array([[0, 1, 6], [0, 2, 7], [0, 3, 5]], np.int32)
    out, (moved,) = O.reorder(tables, np.array([6, 6, 6]), np.array([[1, 1, 0]]), [pages], 4)
    assert out.tolist() == [[0, 2, 6], [0, 3, 7], [0, 1, 5]]            # beam 2 has no child: its page takes the copy
    assert moved[3, 0, :, 0].tolist() == [8, 9, 14, 15] and np.array_equal(np.delete(moved, 3, 0), np.delete(pages, 3, 0))


def test_spans_are_dealt_out_whole(tmp_path):
    """The rule by which the selection deals a row's spans to CTAs, from the header: every span in one part, no part empty or
    longer, and no row in more parts, than the kernels take."""
    from tests.helpers import host_program

    source = r"""
#include "../../include/metile_b200.h"
#include "beam_select.cuh"
#include <cstdio>
int main() {
    const int all_rows[] = {1, 2, 3, 5, 8, 31, 64, 200, 256, 333, 592, 593, 800, 4096, 100000};
    const int all_spans[] = {1, 2, 3, 4, 7, 15, 16, 17, 31, 32, 33, 64, 100, 128};
    for (int rows : all_rows)
        for (int spans : all_spans) {
            const int parts = mt::beam_parts(rows, spans, 148);
            int longest = 0, wrong = parts < 1 || mt::beam_part_start(0, spans, parts) != 0 || mt::beam_part_start(parts, spans, parts) != spans;
            for (int part = 0; part < parts; ++part) {
                const int length = mt::beam_part_start(part + 1, spans, parts) - mt::beam_part_start(part, spans, parts);
                wrong += length < 1;
                if (length > longest) longest = length;
            }
            std::printf("%d %d %d %d %d\n", rows, spans, parts, longest, wrong);
        }
    for (unsigned int n = 1; n <= 64; ++n) {
        const unsigned int r = mt::beam_reciprocal(n);
        int wrong = 0;
        for (unsigned int i = 0; i <= 65536; ++i) wrong += (r ? (unsigned int)((unsigned long long)i * r >> 32) : i) != i / n;
        std::printf("%u %d\n", n, wrong);
    }
    std::printf("%d %d\n", mt::kBeamMaxParts, mt::kBeamMostPerPart);
}
"""
    rows = host_program(str(tmp_path), source)
    (most_parts, most_per_part), plans = rows[-1], [row for row in rows if len(row) == 5]
    assert len(plans) == 15 * 14 and all(row[1] == 0 for row in rows[:-1] if len(row) == 2)
    for lines, spans, parts, longest, wrong in plans:
        assert wrong == 0 and longest <= most_per_part and parts <= min(spans, most_parts), (lines, spans, parts, longest)


def test_splits_of_a_sequence(tmp_path):
    """The cut of a sequence, from the header: by its own length alone, never more splits than the scratch has rows for."""
    from tests.helpers import host_program

    source = r"""
#include "../../include/metile_b200.h"
#include "paged_attention.cuh"
#include <cstdio>
int main() {
    for (long long capacity : {1ll, 8ll, 127ll, 128ll, 129ll, 1000ll, 16384ll, 16385ll, 100000ll, 0x7FFFFFFFll}) {
        int most = 0, wrong = 0;
        for (long long n = 0; n <= capacity; n += n < 70000 ? 1 : 65521) {
            const int shift = mt::paged_split_shift((int)n), splits = mt::paged_splits((int)n);
            if (splits > most) most = splits;
            wrong += ((long long)splits << shift) < n || (splits > 1 && ((long long)(splits - 1) << shift) >= n) || shift < 7;
        }
        std::printf("%lld %d %d %d\n", capacity, most, mt::paged_most_splits(capacity), wrong);
    }
}
"""
    for capacity, most, declared, wrong in host_program(str(tmp_path), source):
        assert wrong == 0 and most <= declared <= 128, capacity


def test_splits_of_sequences_with_few_heads(tmp_path):
    """With one, two or three KV heads a sequence has more splits, as many as the scratch and the join have room for."""
    from tests.helpers import host_program

    source = r"""
#include "../../include/metile_b200.h"
#include "paged_attention.cuh"
#include <cstdio>
int main() {
    for (int heads : {1, 2, 3, 4, 8, 64}) for (int group : {1, 9, 40}) {
        const int limit = mt::paged_split_limit(heads), floor = mt::paged_split_floor(group);
        for (long long capacity : {128ll, 129ll, 16384ll, 16385ll, 40000ll, 100000ll, 0x7FFFFFFFll}) {
            int most = 0, wrong = 0;
            for (long long n = 0; n <= capacity; n += n < 140000 ? 1 : 65521) {
                const int shift = mt::paged_split_shift((int)n, limit, floor), splits = mt::paged_splits((int)n, limit, floor);
                if (splits > most) most = splits;
                wrong += ((long long)splits << shift) < n || (splits > 1 && ((long long)(splits - 1) << shift) >= n) || shift < 7 || (splits > 128 && 1 << shift < 16 * group);
            }
            const size_t bytes = mt::paged_attention_workspace_bytes(3, heads * group, heads, 64, capacity);
            wrong += bytes != (most > 1 ? (size_t)3 * heads * group * mt::paged_most_splits(capacity, limit) * 66 * 4 : 0);
            std::printf("%d %d %d %d\n", limit * heads >= 512, most <= mt::paged_most_splits(capacity, limit), limit <= mt::kPagedSlices * mt::kPagedMostSplits, wrong);
        }
    }
}
"""
    rows = host_program(str(tmp_path), source)
    assert len(rows) == 126
    for units, fits, joined, wrong in rows:
        assert units and fits and joined and wrong == 0
