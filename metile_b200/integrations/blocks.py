"""torch modules that carry MLX-format INT4 weights: the structural targets of the patcher.

They mirror what the reference patches inside MLX-LM models (metile/integrations/mlx_lm.py):
`QuantizedLinear` (MLX's nn.QuantizedLinear: weight / scales / biases, group_size, bits, mode),
an RMSNorm, a gated MLP with gate_proj / up_proj / down_proj, a decoder block with
input_layernorm / self_attn / post_attention_layernorm / mlp, and a small causal LM used to verify
logits before and after patching.  Every INT4 projection runs the CUDA kernels; none has a CPU
path.  The UNPATCHED forward of each module is the op-by-op form native MLX computes
(metile/backends/mlx_quantized.py:883-917: each projection rounded to bf16, then silu(gate)*up,
then down, then the residual add), so that patching reproduces the reference's situation: the
fused path keeps fp32 intermediates and can differ from the op-by-op path by rounding.
"""

from __future__ import annotations

import math
import weakref

import torch
from torch import nn
from torch.nn.modules import module as torch_module

from .. import backends
from ..backends._common import stream_pointer


class QuantizedLinear(nn.Module):
    """y = x @ dequant(weight)^T (+ bias) with MLX affine INT4 weights."""

    def __init__(self, weight, scales, biases, *, group_size=64, bits=4, bias=None, mode="affine"):
        super().__init__()
        self.register_buffer("weight", weight)
        self.register_buffer("scales", scales)
        self.register_buffer("biases", biases)
        self.group_size = group_size
        self.bits = bits
        self.mode = mode
        if bias is not None:
            self.register_buffer("bias", bias)
        else:
            self.bias = None

    @property
    def in_features(self):
        return self.weight.shape[1] * 32 // self.bits

    @property
    def out_features(self):
        return self.weight.shape[0]

    @classmethod
    def from_seed(cls, seed, in_features, out_features, device="cpu"):
        from .. import synth

        return cls(*synth.affine_weight(seed, out_features, in_features, device))

    def forward(self, values):
        with backends.fixed_order():
            out = backends.mlx_affine_qmv(values, self.weight, self.scales, self.biases,
                                          group_size=self.group_size, bits=self.bits)
        return out if self.bias is None else out + self.bias


class QuantizedEmbedding(nn.Module):
    """Token embedding stored as affine INT4 rows (MLX's nn.QuantizedEmbedding: weight uint32
    [V, H/8], scales / biases [V, H/64]).  A lookup gathers the packed rows of the tokens and
    dequantises just those (w = scale * q + bias in fp32, one rounding to the scales' dtype);
    `as_linear()` serves the same triple as the tied output projection."""

    def __init__(self, weight, scales, biases, *, group_size=64, bits=4):
        super().__init__()
        self.register_buffer("weight", weight)
        self.register_buffer("scales", scales)
        self.register_buffer("biases", biases)
        self.group_size, self.bits, self.mode = group_size, bits, "affine"

    def forward(self, tokens):
        flat = tokens.reshape(-1)
        packed = self.weight.view(torch.int32)[flat]                       # [T, H/8]
        shifts = torch.arange(0, 32, 4, device=packed.device, dtype=torch.int32)
        q = ((packed[..., None] >> shifts) & 15).reshape(flat.shape[0], -1).float()   # [T, H]
        scales = self.scales[flat].float().repeat_interleave(self.group_size, dim=1)
        biases = self.biases[flat].float().repeat_interleave(self.group_size, dim=1)
        return (q * scales + biases).to(self.scales.dtype).reshape(*tokens.shape, -1)

    def as_linear(self):
        return QuantizedLinear(self.weight, self.scales, self.biases, group_size=self.group_size, bits=self.bits)


class RMSNorm(nn.Module):
    def __init__(self, weight, eps=1e-6):
        super().__init__()
        self.register_buffer("weight", weight)
        self.eps = eps

    def forward(self, values):
        # Op-by-op reference form in torch (float32 inside, one rounding at the end).
        v = values.float()
        return (v * torch.rsqrt(v.pow(2).mean(-1, keepdim=True) + self.eps) * self.weight.float()).to(values.dtype)


class GatedMLP(nn.Module):
    """down_proj(silu(gate_proj(x)) * up_proj(x)), each op rounded to the activation dtype."""

    def __init__(self, gate_proj, up_proj, down_proj):
        super().__init__()
        self.gate_proj, self.up_proj, self.down_proj = gate_proj, up_proj, down_proj

    def forward(self, values):
        return self.down_proj(nn.functional.silu(self.gate_proj(values)) * self.up_proj(values))


def _rope_frequencies(theta, dim, device):
    """theta^(-2i/D) for the pairs i of a head."""
    return 1.0 / (theta ** (torch.arange(0, dim, 2, device=device, dtype=torch.float32) / dim))


_frequency_tables = weakref.WeakKeyDictionary()  # attention module -> {(theta, dim, device, stream): table}
_MOST_FREQUENCY_TABLES = 4  # of a module; none of them is part of its state


def _current_stream(device):
    return stream_pointer(device).value


def _rope(values, positions, theta):
    """Rotary embedding over the last axis (half-split form); values [B, heads, T, D], positions [T]
    or [B, T]."""
    dim = values.shape[-1]
    inverse = _rope_frequencies(theta, dim, values.device)
    angles = positions.float()[..., None] * inverse
    if angles.ndim == 2:
        angles = angles[None]
    cos, sin = angles.cos()[:, None], angles.sin()[:, None]
    first, second = values.float()[..., : dim // 2], values.float()[..., dim // 2:]
    return torch.cat([first * cos - second * sin, second * cos + first * sin], dim=-1).to(values.dtype)


class KVCache:
    """Append-only key/value cache with room for `capacity` tokens per head, updated in place.

    The MLX-LM cache the reference's models use (`KVCache.update_and_fetch`) grows by concatenation;
    here the storage is allocated once as [batch, kv_heads, capacity, head_dim] and a step writes its
    rows at `length`, so a decode step moves only the new token's bytes."""

    def __init__(self, batch, kv_heads, capacity, head_dim, device, dtype=torch.bfloat16):
        self.keys = torch.zeros((batch, kv_heads, capacity, head_dim), dtype=dtype, device=device)
        self.values = torch.zeros_like(self.keys)
        self.length = 0
        self.positions = torch.zeros((batch,), dtype=torch.int32, device=device)

    @property
    def capacity(self):
        return self.keys.shape[2]

    def update_and_fetch(self, keys, values):
        """Write keys / values [B, H, T, D] at the current length; return views of all tokens so far."""
        steps = keys.shape[2]
        if self.length + steps > self.capacity:
            raise ValueError("KV cache capacity exceeded")
        self.keys[:, :, self.length:self.length + steps] = keys
        self.values[:, :, self.length:self.length + steps] = values
        self.advance(steps)
        return self.keys[:, :, :self.length], self.values[:, :, :self.length]

    def rotate_and_fetch(self, queries, keys, values, frequencies, only_native=False):
        """update_and_fetch with the rotary embedding in front of it, in one kernel: queries [B, T, Hq, D], keys /
        values [B, T, Hkv, D] as the projections leave them.  Returns the rotated queries and the views; with
        `only_native` None for tensors that the native call does not take, and nothing has been done."""
        steps = keys.shape[1]
        if self.length + steps > self.capacity:
            raise ValueError("KV cache capacity exceeded")
        queries = backends.rope_kv_prefill(queries, keys, values, frequencies, self.positions, self.length, self.keys,
                                           self.values, only_native=only_native)
        if queries is None:
            return None
        self.length += steps  # the kernel advanced the device-side count
        return queries, self.keys[:, :, :self.length], self.values[:, :, :self.length]

    def advance(self, steps=1):
        # The device-side count is incremented, not overwritten with the host's number, so that a
        # captured CUDA graph of a decode step advances it on every replay.
        self.length += steps
        self.positions.add_(steps)

    def reset(self, length=0):
        """Forget everything after the first `length` tokens (host and device counts together)."""
        self.length = int(length)
        self.positions.fill_(self.length)


class PagedTables:
    """Block tables, lengths and free pages of a paged cache, for the `requests` rows of a batch and all layers of a model.

    The device has the truth: a step that a CUDA graph replays takes its pages there.  The host keeps the same counts
    beside it (`held` tokens of every request, `free` pages) to refuse what would not fit before anything is queued.

    Before a forward pass the caller lets the requests `grow` or `extend`; the layers of that pass then write and read the
    new tokens.  A pass is one token of every request (grow()), the prompts of some, one after the other in a batch of one
    (grow(counts)), or the next tokens of some, likewise, whatever they hold (extend(counts)): pieces of prompts, drafts, and
    single tokens beside them.

    Requests may share what they begin with: `branch` lets empty ones go on from the first tokens of others, `release` ends
    requests, `compact` puts the pages that are held together.  `shares` counts who holds a page, which the reordering of
    beams does not: beams are ended by `reset`, or counted again by `compact`."""

    def __init__(self, requests, pages, page_size, width, device):
        if requests < 1 or pages < 1 or width < 1 or page_size not in backends.PAGE_SIZES:
            raise ValueError(f"a paged cache needs requests, pages, blocks and a page size of {backends.PAGE_SIZES}")
        self.requests, self.pages, self.page_size, self.width = int(requests), int(pages), int(page_size), int(width)
        self.block_tables = torch.zeros((self.requests, self.width), dtype=torch.int32, device=device)
        self.lengths = torch.zeros((self.requests,), dtype=torch.int32, device=device)
        self.free_pages = torch.arange(self.pages, dtype=torch.int32, device=device)
        self.free_state = torch.tensor([0, self.pages], dtype=torch.int32, device=device)
        self.shares = torch.zeros((self.pages,), dtype=torch.int32, device=device)  # requests that hold a page beyond the first
        self._ones = torch.ones((self.requests,), dtype=torch.int32, device=device)
        self.held, self.free = [0] * self.requests, self.pages
        self.shared = [0] * self.requests    # tokens of every request in pages that others may have too
        self.slots = self.positions = None   # of the tokens of the pass
        self.prompts = None                  # [(request, first row, rows)], or None: one token of every request
        self.starts = None                   # of a pass by `extend`: each request's first row
        self._forget_shares()

    @property
    def capacity(self):
        return self.width * self.page_size

    def reset(self):
        """Forget every request; all pages are free."""
        self.block_tables.zero_()
        self.lengths.zero_()
        torch.arange(self.pages, dtype=torch.int32, device=self.free_pages.device, out=self.free_pages)
        self.free_state.copy_(torch.tensor([0, self.pages], dtype=torch.int32))
        self.held, self.free = [0] * self.requests, self.pages
        self.shared = [0] * self.requests
        self.shares.zero_()
        self._forget_shares()

    def _forget_shares(self):
        # The host's own names of the pages that a request's first blocks share, and how many hold each.
        self._names, self._holders, self._next_name = [[] for _ in range(self.requests)], {}, 0
        self._counted = True  # whether `shares` says who holds what

    def fits(self, counts):
        """The host's side of a change by counts[r] tokens: (held, free) after it; refuses what does not fit."""
        def blocks(tokens):
            return -(-tokens // self.page_size)

        after = [held + count for held, count in zip(self.held, counts)]
        if len(counts) != self.requests or min(after) < 0 or max(after) > self.capacity:
            raise ValueError("paged cache: a request has no room, or fewer tokens than are taken back")
        if any(count < 0 and new < shared for count, new, shared in zip(counts, after, self.shared)):
            raise ValueError("paged cache: pages that requests share are given back by reset alone")
        changes = [blocks(new) - blocks(old) for new, old in zip(after, self.held)]
        if sum(max(0, change) for change in changes) > self.free:
            raise ValueError("paged cache: out of pages")
        return after, self.free - sum(changes)

    def account(self, counts):
        """Make the change on the host's side."""
        self.held, self.free = self.fits(counts)

    def grow(self, counts=None):
        """One new token for every request, or counts[r] for request r; negative counts give back the last tokens.

        Tokens in pages that requests share (those full at the last `fork` or `reorder`) are given back by `reset` alone: a
        page must not go back twice, nor be written by one request under another."""
        self._resize([1] * self.requests if counts is None else [int(count) for count in counts], counts is None)
        self.starts = None

    def extend(self, counts):
        """counts[r] new tokens for request r, behind those it has; the pass attends them by paged_attention_chunk."""
        counts = [int(count) for count in counts]
        if any(count < 0 for count in counts):
            raise ValueError("paged cache: a request is extended by no token or more")
        self.starts = self._resize(counts, False)

    def _resize(self, counts, ones):
        self.account(counts)
        self.prompts, first = None, 0
        if not ones:
            self.prompts = []
            for request, count in enumerate(counts):
                if count > 0:
                    self.prompts.append((request, first, count))
                    first += count
        on_device = self._ones if ones else torch.tensor(counts, dtype=torch.int32).to(self.lengths.device)
        self.slots, self.positions, starts, _, _ = backends.paged_resize(
            self.block_tables, self.lengths, on_device, self.free_pages, self.free_state, page_size=self.page_size,
            tokens=self.requests if ones else first, advance=True)
        return starts

    def share(self):
        """From now on requests may share the pages that are full, as a reordering leaves them."""
        self.shared = [max(shared, held // self.page_size * self.page_size) for shared, held in zip(self.shared, self.held)]
        self._counted = False

    def _need_counts(self, what):
        if not self._counted:
            raise ValueError(f"paged cache: beams share pages that are not counted; {what} needs a compact or a reset first")

    def branch(self, sources, counts, caches):
        """Let request r, which has no tokens, go on from the first counts[r] tokens of request sources[r]; None: r stays as it is.

        Full pages are shared, the page begun is copied, in the PagedKVCache of every layer."""
        self._need_counts("branch")
        if not caches or any(getattr(cache, "tables", None) is not self for cache in caches):
            raise ValueError("branch expects the PagedKVCache of every layer, over these tables")
        if len(sources) != self.requests or len(counts) != self.requests:
            raise ValueError("branch expects a source and a count for every request")
        chosen = [(r, int(source), int(count)) for r, (source, count) in enumerate(zip(sources, counts)) if source is not None]
        for r, source, count in chosen:
            if not 0 <= source < self.requests or source == r or self.held[r] or not 0 < count <= self.held[source]:
                raise ValueError("branch: an empty request goes on from tokens that another one has")
        begun = sum(1 for _, _, count in chosen if count % self.page_size)
        if begun > self.free:
            raise ValueError("paged cache: out of pages")
        on_device = torch.tensor([[-1] * self.requests, [0] * self.requests], dtype=torch.int32)
        for r, source, count in chosen:
            on_device[0, r], on_device[1, r] = source, count
        on_device = on_device.to(self.lengths.device)
        backends.paged_fork(self.block_tables, self.lengths, on_device[0], on_device[1], self.free_pages, self.free_state, self.shares,
                            [(cache.keys, cache.values) for cache in caches], advance=True)
        self.free -= begun
        for r, source, count in chosen:
            whole, names = count // self.page_size, self._names[source]
            while len(names) < whole:
                names.append(self._next_name)
                self._holders[self._next_name] = 1
                self._next_name += 1
            self._names[r] = names[:whole]
            for name in self._names[r]:
                self._holders[name] += 1
            self.held[r], self.shared[r] = count, whole * self.page_size
            self.shared[source] = max(self.shared[source], whole * self.page_size)

    def release(self, requests):
        """End the requests named: their pages go back, shared ones with the last request that holds them."""
        self._need_counts("release")
        ended = sorted(set(int(r) for r in requests))
        if ended and not 0 <= ended[0] <= ended[-1] < self.requests:
            raise ValueError("release expects requests of these tables")
        flags = torch.zeros((self.requests,), dtype=torch.bool)
        flags[ended] = True
        backends.paged_free(self.block_tables, self.lengths, flags.to(self.lengths.device), self.free_pages, self.free_state, self.shares,
                            page_size=self.page_size, advance=True)
        for r in ended:
            self.free += -(-self.held[r] // self.page_size) - len(self._names[r])
            for name in self._names[r]:
                self._holders[name] -= 1
                if self._holders[name] == 0:
                    del self._holders[name]
                    self.free += 1
            self.held[r], self.shared[r], self._names[r] = 0, 0, []

    def compact(self, caches):
        """Move the pages that are held to the lowest ids, in the PagedKVCache of every layer, and count who holds them from the
        tables: pages that nobody holds any more, as dropped beams leave them, are free afterwards.  Waits for the GPU, whose
        tables the host's side is taken from."""
        if not caches or any(getattr(cache, "tables", None) is not self for cache in caches):
            raise ValueError("compact expects the PagedKVCache of every layer, over these tables")
        moved = backends.paged_compact(self.block_tables, self.lengths, [(cache.keys, cache.values) for cache in caches])
        for own, new in zip((self.block_tables, self.free_pages, self.free_state, self.shares), moved):
            own.copy_(new)
        self._forget_shares()
        tables, shares = self.block_tables.tolist(), self.shares.tolist()
        self.free = int(self.free_state[1])
        for r, held in enumerate(self.held):
            ids = tables[r][:-(-held // self.page_size)]
            last = max((j for j, page in enumerate(ids) if shares[page]), default=-1)
            self._names[r] = ids[:last + 1]  # the pages' ids as they are now serve for names
            self.shared[r] = (last + 1) * self.page_size
            for page in self._names[r]:
                self._holders[page] = self._holders.get(page, 0) + 1
        self._next_name = self.pages

    def fork(self, beams, caches):
        """Every first request of `beams` in a row is continued by all of them: full pages are shared, what is begun is copied
        in the PagedKVCache of every layer."""
        groups = self.requests // max(1, beams)
        if groups * beams != self.requests or any(self.held[r] and r % beams for r in range(self.requests)):
            raise ValueError("only the first request of each group may have tokens")
        if beams > backends.MAX_BEAMS:
            raise ValueError(f"a group has up to {backends.MAX_BEAMS} beams")
        if not caches or any(getattr(cache, "tables", None) is not self for cache in caches):
            raise ValueError("fork expects the PagedKVCache of every layer, over these tables")
        held = [self.held[r - r % beams] for r in range(self.requests)]
        # The others hold the full pages in name, which cost none, and a page of their own for the rest.
        whole = [n // self.page_size * self.page_size for n in held]
        part = [0 if r % beams == 0 else held[r] - whole[r] for r in range(self.requests)]
        if sum(1 for count in part if count) > self.free:
            raise ValueError("paged cache: out of pages")
        self.held = [held[r] if r % beams == 0 else whole[r] for r in range(self.requests)]
        self.lengths.copy_(torch.tensor(self.held, dtype=torch.int32))
        self.grow(part)
        self.reorder(torch.zeros((groups, beams), dtype=torch.int32, device=self.lengths.device), caches)

    def reorder(self, parents, caches):
        """The requests of every group of beams continue those that `parents` [groups, beams] (int32) names."""
        self.block_tables.copy_(backends.beam_reorder(self.block_tables, self.lengths, parents,
                                                      [(cache.keys, cache.values) for cache in caches]))
        if parents.shape[1] > 1:
            self.share()


class PagedKVCache:
    """One layer's keys and values [pages, kv_heads, page_size, head_dim] behind the tables of the whole model."""

    def __init__(self, tables, kv_heads, head_dim, dtype=torch.bfloat16):
        self.tables = tables
        shape = (tables.pages, kv_heads, tables.page_size, head_dim)
        self.keys = torch.zeros(shape, dtype=dtype, device=tables.lengths.device)
        self.values = torch.zeros_like(self.keys)

    def append(self, queries, keys, values, frequencies):
        """Rotate the pass's rows and write keys and values to their slots; rows [tokens, heads, head_dim].  Returns the
        rotated queries."""
        tables = self.tables
        if tables.slots is None or queries.shape[0] != tables.slots.shape[0]:
            raise ValueError("paged cache: the pass does not have the tokens that its tables grew by")
        return backends.rope_kv_append_paged(queries, keys, values, frequencies, tables.positions, tables.slots, self.keys,
                                             self.values)

    def fetch(self, first, count):
        """Keys and values [count, kv_heads, head_dim] of the pass's rows `first` on, as they are stored."""
        slots = self.tables.slots[first:first + count]
        page, row = slots // self.tables.page_size, slots % self.tables.page_size
        return self.keys[page, :, row], self.values[page, :, row]


_UPDATE, _ADVANCE = KVCache.update_and_fetch, KVCache.advance


def appends_in_place(cache):
    """Whether `cache` is a KVCache whose update_and_fetch and advance are the ones above."""
    return type(cache) is KVCache and KVCache.update_and_fetch is _UPDATE and KVCache.advance is _ADVANCE \
        and "update_and_fetch" not in cache.__dict__ and "advance" not in cache.__dict__


def scaled_dot_product_attention(queries, keys, values, cache, scale, mask=None):
    """The attention primitive every Attention module here calls; the patcher replaces THIS module
    attribute (the reference replaces mlx_lm.models.base.scaled_dot_product_attention the same way,
    metile/integrations/mlx_lm.py:4607-4655).  queries [B, Hq, T, D], keys / values [B, Hkv, N, D]."""
    del cache
    causal = mask == "causal"
    return nn.functional.scaled_dot_product_attention(
        queries, keys, values, scale=scale, is_causal=causal, enable_gqa=queries.shape[1] != keys.shape[1])


class Attention(nn.Module):
    """Grouped-query attention over INT4 q/k/v/o projections with RoPE and an in-place KV cache."""

    def __init__(self, q_proj, k_proj, v_proj, o_proj, heads, kv_heads, head_dim, rope_theta=1e6):
        super().__init__()
        self.q_proj, self.k_proj, self.v_proj, self.o_proj = q_proj, k_proj, v_proj, o_proj
        self.heads, self.kv_heads, self.head_dim, self.rope_theta = heads, kv_heads, head_dim, rope_theta
        self.scale = head_dim ** -0.5

    def _frequencies_on(self, device):
        # A table serves the stream it was made on, in whose order it is also given back.  A graph that is being
        # captured makes its own, which lives as long as the graph does.
        if torch.cuda.is_current_stream_capturing():
            return _rope_frequencies(self.rope_theta, self.head_dim, device)
        tables = _frequency_tables.setdefault(self, {})
        key = self.rope_theta, self.head_dim, device, _current_stream(device)
        table = tables.get(key)
        if table is None:
            table = _rope_frequencies(self.rope_theta, self.head_dim, device)
            if len(tables) >= _MOST_FREQUENCY_TABLES:
                tables.clear()
            tables[key] = table
        return table

    def forward(self, values, cache=None):
        return self.o_proj(self.attend(self.q_proj(values), self.k_proj(values), self.v_proj(values), cache))

    def attend(self, q, k, v, cache=None):
        """Rotary embedding, cache and attention of projected rows [B, T, heads D]; returns [B, T, Hq D]."""
        if isinstance(cache, PagedKVCache):
            return self._attend_paged(q, k, v, cache)
        batch, steps, _ = q.shape
        q = q.view(batch, steps, self.heads, self.head_dim)
        k = k.view(batch, steps, self.kv_heads, self.head_dim)
        v = v.view(batch, steps, self.kv_heads, self.head_dim)
        offset = 0 if cache is None else cache.length
        if steps > 1 and offset > 0:
            raise ValueError("multi-token continuation is not supported by this harness")
        served = None
        if steps > 1 and q.is_cuda and appends_in_place(cache) and not (q.requires_grad or k.requires_grad or v.requires_grad):
            served = cache.rotate_and_fetch(q, k, v, self._frequencies_on(q.device), only_native=True)
        if served is not None:
            q, k, v = served
            q = q.transpose(1, 2)
        else:
            q, k, v = q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2)
            positions = torch.arange(offset, offset + steps, device=q.device)
            q, k = _rope(q, positions, self.rope_theta), _rope(k, positions, self.rope_theta)
            if cache is not None:
                k, v = cache.update_and_fetch(k, v)
        out = scaled_dot_product_attention(q, k, v, cache, self.scale, "causal" if steps > 1 else None)
        return out.transpose(1, 2).reshape(batch, steps, self.heads * self.head_dim)


    def _attend_paged(self, q, k, v, cache):
        batch, steps, _ = q.shape
        rows, tables = batch * steps, cache.tables
        q = q.reshape(rows, self.heads, self.head_dim)
        k = k.reshape(rows, self.kv_heads, self.head_dim)
        v = v.reshape(rows, self.kv_heads, self.head_dim)
        rotated = cache.append(q, k, v, self._frequencies_on(q.device))
        if tables.starts is not None:
            out = backends.paged_attention_chunk(rotated, cache.keys, cache.values, tables.block_tables, tables.lengths, tables.starts,
                                                 scale=self.scale)
            return out.view(batch, steps, self.heads * self.head_dim)
        if tables.prompts is None:
            out = backends.paged_attention_decode(rotated, cache.keys, cache.values, tables.block_tables, tables.lengths,
                                                  scale=self.scale)
            return out.view(batch, steps, self.heads * self.head_dim)
        out = torch.empty_like(rotated)
        for request, first, count in tables.prompts:
            if tables.held[request] != count:
                raise ValueError("multi-token continuation is not supported by this harness")
            keys, values = cache.fetch(first, count)
            attended = scaled_dot_product_attention(
                rotated[None, first:first + count].transpose(1, 2), keys[None].transpose(1, 2), values[None].transpose(1, 2),
                cache, self.scale, "causal" if count > 1 else None)
            out[first:first + count] = attended[0].transpose(0, 1)
        return out.view(batch, steps, self.heads * self.head_dim)


class DecoderBlock(nn.Module):
    """Pre-norm decoder block: x + attn(norm(x)), then h + mlp(norm(h))."""

    def __init__(self, input_layernorm, self_attn, post_attention_layernorm, mlp):
        super().__init__()
        self.input_layernorm, self.self_attn = input_layernorm, self_attn
        self.post_attention_layernorm, self.mlp = post_attention_layernorm, mlp

    def forward(self, values, cache=None):
        hidden = values + self.self_attn(self.input_layernorm(values), cache)
        return hidden + self.mlp(self.post_attention_layernorm(hidden))


_EMBEDDING_FORWARD, _EMBEDDING_CALL = nn.Embedding.forward, nn.Embedding.__call__


def _embed(module, tokens):
    """module(tokens), by the gather kernel where the module is torch's embedding and looks rows up and nothing else.
    (Of a token outside the table torch's kernel makes an assertion that ends the context; this one a row of NaN, recorded in
    the status word.)"""
    state = module.__dict__
    if type(module) is nn.Embedding and state["max_norm"] is None and nn.Embedding.forward is _EMBEDDING_FORWARD \
            and nn.Embedding.__call__ is _EMBEDDING_CALL and not (
                state["_forward_hooks"] or state["_forward_pre_hooks"] or state["_backward_hooks"]
                or state["_backward_pre_hooks"] or "forward" in state) and state.get("_compiled_call_impl") is None \
            and not torch_module._has_any_global_hook() and not torch._C._get_tracing_state():
        weight = state["_parameters"].get("weight")
        if weight is not None and weight.is_cuda:
            rows = backends.embedding(tokens, weight)
            if rows is not None:
                return rows
    return module(tokens)


class TinyCausalLM(nn.Module):
    """Embedding, a stack of DecoderBlocks, final norm and an INT4 lm_head; random initialisation."""

    def __init__(self, embed, layers, norm, lm_head, vocab_size):
        super().__init__()
        self.embed_tokens = embed
        self.layers = nn.ModuleList(layers)
        self.norm = norm
        self.lm_head = lm_head
        self.vocab_size = vocab_size

    def make_cache(self, batch=1, capacity=64):
        caches = []
        for layer in self.layers:
            attention = layer.self_attn
            caches.append(KVCache(batch, attention.kv_heads, capacity, attention.head_dim,
                                  attention.q_proj.weight.device))
        return caches

    def make_paged_cache(self, requests, pages, page_size=16, capacity=4096):
        """A PagedKVCache for every layer, over the same tables: `pages` pages for `requests` requests of up to `capacity`
        tokens each."""
        first = self.layers[0].self_attn
        tables = PagedTables(requests, pages, page_size, -(-capacity // page_size), first.q_proj.weight.device)
        return [PagedKVCache(tables, layer.self_attn.kv_heads, layer.self_attn.head_dim) for layer in self.layers]

    def forward(self, tokens, cache=None, logits_to_keep=0, logits_at=None):
        """Logits [batch, tokens, vocabulary]; with `logits_to_keep`, of that many last positions only; with `logits_at`
        (int64), of the positions it names."""
        hidden = _embed(self.embed_tokens, tokens)
        for index, layer in enumerate(self.layers):
            hidden = layer(hidden, None if cache is None else cache[index])
        if logits_at is not None or 0 < logits_to_keep < hidden.shape[1]:
            hidden = hidden[:, -logits_to_keep:].contiguous() if logits_at is None else hidden.index_select(1, logits_at)
            # The logits that all positions together would give: one row alone is else another kernel's.
            if not backends.kernel_pinned():
                with backends.batch_invariant():
                    return self.lm_head(self.norm(hidden))
        return self.lm_head(self.norm(hidden))


def random_model(seed=0, *, hidden=256, intermediate=512, heads=4, kv_heads=2, head_dim=64, layers=2, vocab=512,
                 rope_theta=1e6, eps=1e-6, device="cuda", quantized_embedding=False, tie_word_embeddings=False):
    """A seeded random-init decoder-only model in the Qwen2.5 / Llama layout with 4-bit projections
    (and, when asked, a 4-bit embedding, optionally tied to the output projection)."""
    from .. import synth

    def linear(offset, fan_in, fan_out):
        return QuantizedLinear.from_seed(seed * 1000 + offset, fan_in, fan_out, device)

    blocks = []
    for index in range(layers):
        base = 10 * index
        attention = Attention(linear(base + 1, hidden, heads * head_dim), linear(base + 2, hidden, kv_heads * head_dim),
                              linear(base + 3, hidden, kv_heads * head_dim), linear(base + 4, heads * head_dim, hidden),
                              heads, kv_heads, head_dim, rope_theta)
        mlp = GatedMLP(linear(base + 5, hidden, intermediate), linear(base + 6, hidden, intermediate),
                       linear(base + 7, intermediate, hidden))
        blocks.append(DecoderBlock(RMSNorm(synth.norm_weight(seed * 1000 + base + 8, hidden, device), eps), attention,
                                   RMSNorm(synth.norm_weight(seed * 1000 + base + 9, hidden, device), eps), mlp))
    generator = torch.Generator().manual_seed(seed * 1000 + 999)
    table = (torch.randn((vocab, hidden), generator=generator) / math.sqrt(hidden) * 4).to(torch.bfloat16)
    if quantized_embedding or tie_word_embeddings:
        from . import checkpoint

        embed = QuantizedEmbedding(*(t.to(device) for t in checkpoint.quantize_affine(table)))
    else:
        embed = nn.Embedding.from_pretrained(table.to(device), freeze=True)
    head = embed.as_linear() if tie_word_embeddings else linear(997, hidden, vocab)
    return TinyCausalLM(embed, blocks, RMSNorm(synth.norm_weight(seed * 1000 + 998, hidden, device), eps), head, vocab)
