"""The operators of the paged key-value cache and of beam search, as cases that can be timed and compared.

The kinds, and what a serving program does with them:

  tables   paged_resize: requests grow and shrink; pages come from and go back to a ring of free ones, and every new
           token is told its position and its slot in the cache
  append   rope_kv_append_paged: the new tokens' queries and keys are rotated, keys and values go to their slots
  attend   paged_attention_decode: one new token per request over the pages its row of the block table names
  select   beam_select: the best continuations over a group's beams and the vocabulary
  reorder  beam_reorder: block tables follow the surviving beams; only the page in work is copied

`run` is the plain form (elementary torch operations, 32 bits or 64 where 32 lose what matters) or, with `own`, the
framework's operators.  Head layouts and widths are those of the tests and the benchmark (2 x 6 heads of 128, heads of
64, a vocabulary of 128256, 28 layers) and others around them; lengths run from one token to a hundred thousand.
"""

from __future__ import annotations

import math

import torch

own = False

ROPE_THETA = 1e6
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}
DEAD = -1e15  # scores at or below count as no candidate: a mask, not a sum of log-probabilities

# No drawn case costs more than the largest listed one of its kind.
MOST_KV_BYTES = 1700 << 20
MOST_APPEND = 4000 * 48 * 128
MOST_LOGIT_BYTES = 31 * 8 * 128256 * 2
MOST_REORDER_BYTES = 80 << 20


def listed():
    return [
        # A decode step of 64 requests: every one grows by a token, a few enter a new page.  Latency counts.
        {"name": "tables_step", "kind": "tables", "requests": 64, "most": 1, "held": 4000, "page": 16, "shrink": 0},
        # Prompts of every length arrive while other requests decode, end, or take back a draft: the largest map.
        {"name": "tables_mixed", "kind": "tables", "requests": 501, "most": 4096, "held": 8000, "page": 16, "shrink": 7},
        # One decode step of sixteen sequences, heads as in a Qwen2.5-1.5B block.
        {"name": "append_step", "kind": "append", "tokens": 16, "padding": 0, "kv_heads": 2, "group": 6, "dim": 128,
         "page": 16, "type": "bf16", "far": 2048},
        # Prompts of several requests together, at far positions, the batch padded by a few rows.
        {"name": "append_prompt", "kind": "append", "tokens": 4093, "padding": 61, "kv_heads": 8, "group": 4, "dim": 128,
         "page": 32, "type": "bf16", "far": 120000},
        # A single short conversation: the latency of a step.
        {"name": "attend_1", "kind": "attend", "batch": 1, "kv_heads": 8, "group": 4, "dim": 128, "page": 16,
         "tokens": 301, "ragged": False, "type": "bf16"},
        # Sixteen sequences of 2048 tokens at a Qwen2.5-1.5B block's heads.
        {"name": "attend_16", "kind": "attend", "batch": 16, "kv_heads": 2, "group": 6, "dim": 128, "page": 16,
         "tokens": 2048, "ragged": False, "type": "bf16"},
        # Two very long documents, not a whole number of pages, in fp16.
        {"name": "attend_long", "kind": "attend", "batch": 2, "kv_heads": 8, "group": 4, "dim": 128, "page": 32,
         "tokens": 100003, "ragged": False, "type": "fp16"},
        # A full serving batch of requests of every length, one of them empty: the most bytes.
        {"name": "attend_serving", "kind": "attend", "batch": 100, "kv_heads": 8, "group": 4, "dim": 128, "page": 16,
         "tokens": 8191, "ragged": True, "type": "bf16"},
        # Four beams of one request; an odd vocabulary, so rows start anywhere.
        {"name": "select_4", "kind": "select", "groups": 1, "beams": 4, "keep": 4, "vocab": 32001, "type": "bf16",
         "ended": False},
        # A batch of thirty-two requests with eight beams each over a large vocabulary, twice the beams kept.
        {"name": "select_256", "kind": "select", "groups": 32, "beams": 8, "keep": 16, "vocab": 128256, "type": "bf16",
         "ended": True},
        # Four beams through four layers.
        {"name": "reorder_4", "kind": "reorder", "groups": 1, "beams": 4, "layers": 4, "kv_heads": 2, "dim": 128,
         "page": 16, "prompt": 500, "step": 37, "type": "bf16"},
        # Sixteen requests of eight beams through the 28 layers of a whole model.
        {"name": "reorder_128", "kind": "reorder", "groups": 16, "beams": 8, "layers": 28, "kv_heads": 2, "dim": 128,
         "page": 32, "prompt": 1000, "step": 55, "type": "bf16"},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("tables", "append", "attend", "attend", "select", "reorder"))
    page = rng.choice((8, 16, 32, 64, 128))
    half = rng.choice(("bf16", "fp16"))
    if kind == "tables":
        requests, most = _log_int(rng, 1, 500), rng.choice((1, 1, _log_int(rng, 2, 3500)))
        return {"kind": kind, "requests": requests, "most": most, "held": _log_int(rng, 1, 8000), "page": page,
                "shrink": rng.choice((0, 3, 7))}
    kv_heads, group, dim = rng.choice((1, 2, 4, 8)), rng.randint(1, 16), rng.choice((64, 128, 256))
    if kind == "append":
        tokens = min(_log_int(rng, 1, 4096), max(1, MOST_APPEND // ((group + 2) * kv_heads * dim)))
        return {"kind": kind, "tokens": tokens, "padding": rng.choice((0, 1, 17)), "kv_heads": kv_heads, "group": group,
                "dim": dim, "page": page, "type": half, "far": _log_int(rng, 1, 130000)}
    if kind == "attend":
        batch, tokens = _log_int(rng, 1, 100), _log_int(rng, 1, 131072)
        return {"kind": kind, "batch": batch, "kv_heads": kv_heads, "group": group, "dim": dim, "page": page,
                "tokens": max(1, min(tokens, MOST_KV_BYTES // (batch * kv_heads * dim * 4))),
                "ragged": rng.random() < 0.6, "type": half}
    if kind == "select":
        beams, vocab = rng.randint(1, 16), _log_int(rng, 100, 131072)
        name = rng.choice(("bf16", "fp16", "fp32"))
        groups = min(_log_int(rng, 1, 64), max(1, MOST_LOGIT_BYTES // (beams * vocab * SIZES[name])))
        return {"kind": kind, "groups": groups, "beams": beams, "keep": rng.choice((beams, 2 * beams)), "vocab": vocab,
                "type": name, "ended": rng.random() < 0.5}
    beams, layers = rng.randint(2, 16), rng.randint(1, 28)
    case = {"kind": kind, "groups": 1, "beams": beams, "layers": layers, "kv_heads": rng.choice((1, 2, 4)),
            "dim": rng.choice((64, 128)), "page": rng.choice((8, 16, 32)), "prompt": _log_int(rng, 1, 1000),
            "step": _log_int(rng, 1, 64), "type": half}
    return {**case, "groups": max(1, min(_log_int(rng, 1, 32), int(MOST_REORDER_BYTES // work(case)["bytes"])))}


# ---- what follows from a case alone ----------------------------------------------------------------------------


def _spread(count, low, high, step):
    """`count` whole numbers from low to high, spread evenly in an order that is not sorted."""
    return [low + (high - low) * (i * step % count) // max(1, count - 1) for i in range(count)]


def _attend_lengths(case):
    batch, tokens = case["batch"], case["tokens"]
    if not case["ragged"]:
        return [tokens] * batch
    lengths = _spread(batch, max(1, tokens // 8), tokens, 7)
    if batch >= 3:
        lengths[batch // 2] = 0  # a row of the batch that no request uses
    return lengths


def _table_requests(case):
    """(tokens held, tokens added) of every request; negative: tokens taken back."""
    requests, most, shrink = case["requests"], case["most"], case["shrink"]
    held = _spread(requests, 0, case["held"], 11)
    added = []
    for i in range(requests):
        if shrink and i % shrink == shrink - 1:
            added.append(-held[i] if i % 2 else -min(held[i], 5))  # the request has ended, or a draft was rejected
        elif most > 1 and i % 8 == 0:
            added.append(1 + (most - 1) * (i * 5 % requests) // max(1, requests - 1))
        else:
            added.append(1)
    return held, added


def _blocks(tokens, page):
    return -(-tokens // page)


def _used_block(case):
    """(tokens held, logical block in work, tokens in it) of a reorder case."""
    tokens = case["prompt"] + case["step"]
    return tokens, tokens // case["page"], tokens % case["page"]


def _surviving(beams):
    return max(1, beams * 5 // 8)


# ---- inputs --------------------------------------------------------------------------------------------------


class _Maker:
    """Seeded tensors on the GPU."""

    def __init__(self, seed):
        self.device = torch.device("cuda")
        self.generator = torch.Generator(device=self.device).manual_seed(int(seed))

    def normal(self, *shape, std=1.0, dtype=torch.bfloat16):
        out = torch.empty(shape, dtype=dtype, device=self.device)
        flat = out.view(-1)
        for first in range(0, flat.numel(), 1 << 28):
            part = flat[first:first + (1 << 28)]
            part.copy_(torch.randn(part.shape, generator=self.generator, device=self.device) * std)
        return out

    def order(self, count):
        return torch.randperm(count, generator=self.generator, device=self.device)

    def uniform(self, *shape):
        return torch.rand(shape, generator=self.generator, device=self.device)

    def ints(self, values):
        return torch.tensor(values, dtype=torch.int32, device=self.device)


def _table_of(make, lengths, page, width, pool):
    """A block table whose rows name as many distinct pages as their lengths need, in no order; the rest is unused."""
    table = torch.full((len(lengths), width), -1, dtype=torch.int32, device=make.device)
    held = make.ints([_blocks(n, page) for n in lengths])
    used = torch.arange(width, device=make.device)[None] < held[:, None]
    first = torch.cumsum(held, 0) - held
    index = (first[:, None] + torch.arange(width, device=make.device)[None]).clamp(max=pool - 1)
    return torch.where(used, make.order(pool).to(torch.int32)[index], table)


def prepare(case, seed):
    make, kind, page = _Maker(seed), case["kind"], case.get("page")
    if kind == "tables":
        held, added = _table_requests(case)
        order = make.order(len(held)).tolist()
        held, added = [held[i] for i in order], [added[i] for i in order]
        before = [_blocks(n, page) for n in held]
        after = [_blocks(n + c, page) for n, c in zip(held, added)]
        grants = sum(max(0, a - b) for a, b in zip(after, before))
        width = max(max(before), max(after)) + 2
        pool = sum(before) + grants + 16
        pages = make.order(pool).to(torch.int32)
        table = torch.full((len(held), width), -1, dtype=torch.int32, device=make.device)
        first = 0
        for row, blocks in enumerate(before):
            table[row, :blocks] = pages[first:first + blocks]
            first += blocks
        # The free pages stand somewhere in the ring, across its end as often as not.
        start = int(make.uniform(1).item() * pool)
        ring = torch.full((pool,), -1, dtype=torch.int32, device=make.device)
        ring[(torch.arange(pool - first, device=make.device) + start) % pool] = pages[first:]
        return {"kind": kind, "page": page, "tokens": sum(max(0, c) for c in added) + 5, "table": table,
                "lengths": make.ints(held), "counts": make.ints(added), "ring": ring,
                "state": make.ints([start, pool - first])}
    if kind == "append":
        tokens, dim, kv_heads, heads = case["tokens"], case["dim"], case["kv_heads"], case["kv_heads"] * case["group"]
        dtype, rows = TYPES[case["type"]], case["tokens"] + case["padding"]
        # Views into the rows of one fused q|k|v projection, as a model hands them over.
        fused = make.normal(rows, (heads + 2 * kv_heads) * dim, dtype=dtype)
        query, key, value = (part.view(rows, -1, dim) for part in fused.split((heads * dim, kv_heads * dim, kv_heads * dim), 1))
        pool = _blocks(tokens, page) + 8
        slots = torch.full((rows,), -1, dtype=torch.int64, device=make.device)
        slots[:tokens] = make.order(pool * page)[:tokens]
        positions = torch.zeros((rows,), dtype=torch.int32, device=make.device)
        positions[:tokens] = (make.uniform(tokens) * case["far"]).to(torch.int32)
        inverse = 1.0 / (ROPE_THETA ** (torch.arange(0, dim, 2, device=make.device, dtype=torch.float32) / dim))
        return {"kind": kind, "query": query, "key": key, "value": value, "inverse": inverse, "positions": positions,
                "slots": slots, "keys": make.normal(pool, kv_heads, page, dim, dtype=dtype),
                "values": make.normal(pool, kv_heads, page, dim, dtype=dtype)}
    if kind == "attend":
        lengths = _attend_lengths(case)
        lengths = [lengths[i] for i in make.order(len(lengths)).tolist()]
        dim, kv_heads, dtype = case["dim"], case["kv_heads"], TYPES[case["type"]]
        pool = sum(_blocks(n, page) for n in lengths) + 3
        width = _blocks(max(max(lengths), 1), page) + 3
        return {"kind": kind, "query": make.normal(len(lengths), kv_heads * case["group"], dim, std=2.0, dtype=dtype),
                "keys": make.normal(pool, kv_heads, page, dim, dtype=dtype),
                "values": make.normal(pool, kv_heads, page, dim, dtype=dtype),
                "table": _table_of(make, lengths, page, width, pool), "lengths": make.ints(lengths), "scale": dim ** -0.5}
    if kind == "select":
        groups, beams, vocab = case["groups"], case["beams"], case["vocab"]
        logits = make.normal(groups * beams, vocab, std=2.5, dtype=TYPES[case["type"]])
        scores = torch.sort(make.uniform(groups, beams) * -30.0, dim=1, descending=True).values
        finished = make.uniform(groups, beams) < 0.2 if case["ended"] else None
        return {"kind": kind, "logits": logits, "scores": scores, "keep": case["keep"], "finished": finished,
                "end": 2 if case["ended"] else None}
    groups, beams, width = case["groups"], case["beams"], _blocks(case["prompt"] + 128, page) + 1
    tokens, block, _ = _used_block(case)
    rows, shared = groups * beams, case["prompt"] // page
    # Pages of the prompt belong to all beams of a group; what came after it was shared or owned as earlier steps left
    # it; the page in work and those behind it are each beam's own.
    pool = groups * shared + rows * (width - shared)
    pages = make.order(pool).to(torch.int32)
    table = torch.empty((groups, beams, width), dtype=torch.int32, device=make.device)
    table[:, :, :shared] = pages[:groups * shared].view(groups, 1, shared)
    owned = pages[groups * shared:].view(groups, beams, width - shared)
    if block > shared:
        chosen = (make.uniform(groups, beams, block - shared) * beams).to(torch.int64)
        table[:, :, shared:block] = torch.gather(owned[:, :, :block - shared], 1, chosen)
    table[:, :, block:] = owned[:, :, block - shared:]
    distinct = torch.argsort(make.uniform(groups, beams), dim=1)[:, :_surviving(beams)]
    extra = (make.uniform(groups, beams - distinct.shape[1]) * distinct.shape[1]).to(torch.int64)
    parents = torch.cat([distinct, torch.gather(distinct, 1, extra)], dim=1)
    parents = torch.gather(parents, 1, torch.argsort(make.uniform(groups, beams), dim=1))
    caches = [tuple(make.normal(pool, case["kv_heads"], page, case["dim"], dtype=TYPES[case["type"]]) for _ in range(2))
              for _ in range(case["layers"])]
    return {"kind": kind, "table": table.view(rows, width), "lengths": make.ints([tokens] * rows),
            "parents": parents.to(torch.int32).contiguous(), "caches": caches}


# ---- the plain forms --------------------------------------------------------------------------------------------


def _plain_tables(state):
    table, lengths, counts, ring = state["table"], state["lengths"].long(), state["counts"].long(), state["ring"]
    page, tokens = state["page"], state["tokens"]
    pool, width, device = ring.shape[0], table.shape[1], table.device
    first, free = state["state"][0].long(), state["state"][1].long()
    after = lengths + counts
    ends = torch.cumsum(counts.clamp(min=0), 0)
    starts = torch.cat([ends.new_zeros(1), ends])
    valid = (lengths >= 0) & (after >= 0) & (lengths <= width * page) & (after <= width * page)
    valid &= (counts <= 0) | (ends <= tokens)
    old, new = (lengths + page - 1) // page, (after + page - 1) // page
    need = torch.where(valid, (new - old).clamp(min=0), 0)
    reach = torch.cumsum(need, 0)
    served = valid & ((need == 0) | (reach <= free))
    granted = torch.where(served, need, 0)
    freed = torch.where(served, (old - new).clamp(min=0), 0)
    column = torch.arange(width, device=device)[None]
    fresh = served[:, None] & (column >= old[:, None]) & (column < new[:, None])
    index = (first + (reach - need)[:, None] + column - old[:, None]) % pool
    table.copy_(torch.where(fresh, ring[index], table))
    back = served[:, None] & (column >= new[:, None]) & (column < old[:, None])
    place = (first + free + (torch.cumsum(freed, 0) - freed)[:, None] + column - new[:, None]) % pool
    place = torch.where(back, place, pool)
    longer = torch.cat([ring, ring.new_zeros(1)])
    longer[place.reshape(-1)] = table.reshape(-1)
    ring.copy_(longer[:pool])
    at = torch.arange(tokens, device=device)
    row = torch.searchsorted(ends, at, right=True)
    inside = row < lengths.shape[0]
    row = row.clamp(max=lengths.shape[0] - 1)
    inside &= served[row]
    position = torch.where(inside, lengths[row] + at - starts[row], 0)
    block = (position // page).clamp(0, width - 1)
    slot = table[row, block].long() * page + position % page
    slots = torch.where(inside, slot, -1)
    state_out = torch.stack([(first + granted.sum()) % pool, free - granted.sum() + freed.sum()])
    return {"slots": slots, "positions": position.to(torch.int32), "starts": starts.to(torch.int32),
            "lengths": torch.where(served, after, lengths).to(torch.int32), "state": state_out.to(torch.int32),
            "table": table, "ring": ring}


def _rotate(rows, cos, sin):
    half = rows.shape[-1] // 2
    first, second = rows[..., :half].float(), rows[..., half:].float()
    return torch.cat([first * cos - second * sin, second * cos + first * sin], dim=-1).to(rows.dtype)


def _plain_append(state):
    keys, values, slots = state["keys"], state["values"], state["slots"]
    page = keys.shape[2]
    angles = state["positions"].double()[:, None] * state["inverse"].double()  # 32 bits lose far positions
    cos, sin = angles.cos().float()[:, None], angles.sin().float()[:, None]
    query, key, value = _rotate(state["query"], cos, sin), _rotate(state["key"], cos, sin), state["value"]
    # Rows without a slot repeat the write of the first row that has one.
    some = torch.argmax((slots >= 0).to(torch.int8))
    source = torch.where(slots >= 0, torch.arange(slots.shape[0], device=slots.device), some)
    target = slots[source]
    keys[target // page, :, target % page] = key[source]
    values[target // page, :, target % page] = value[source]
    return {"query": query, "keys": keys, "values": values}


def _plain_attend(state):
    query, table, lengths = state["query"], state["table"], state["lengths"]
    batch, heads, dim = query.shape
    pool, kv_heads, page, _ = state["keys"].shape
    group = heads // kv_heads
    index = table.clamp(0, pool - 1).long()
    used = torch.arange(table.shape[1] * page, device=table.device)[None] < lengths[:, None]

    def gathered(pages):
        rows = pages[index].float().transpose(1, 2).reshape(batch, kv_heads, -1, dim)
        return rows.masked_fill_(~used[:, None, :, None], 0.0)

    scores = torch.matmul(query.float().view(batch, kv_heads, group, dim), gathered(state["keys"]).transpose(2, 3))
    scores = scores * state["scale"]
    scores = scores.masked_fill(~used[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights, gathered(state["values"])) / torch.where(total == 0.0, 1.0, total)
    return out.reshape(batch, heads, dim).to(query.dtype)


def _plain_select(state):
    scores, keep, finished, end = state["scores"], state["keep"], state["finished"], state["end"]
    groups, beams = scores.shape
    vocab = state["logits"].shape[1]
    # In 64 bits: two candidates of different beams may be closer than 32 bits can tell.
    logits = state["logits"].double()
    logits = logits - logits.amax(1, keepdim=True)
    logits = logits - torch.log(torch.exp(logits).sum(1, keepdim=True))
    running = scores.double().masked_fill(scores <= DEAD, -math.inf)
    found = logits.view(groups, beams, vocab) + running[:, :, None]
    if finished is not None:
        found = found.masked_fill(finished[:, :, None], -math.inf)
        found[:, :, end] = torch.where(finished, running, found[:, :, end])
    nothing = -1e300  # in place of minus infinity, which marks what has been taken
    found = torch.where(torch.isnan(found) | (found < nothing), nothing, found).view(groups, beams * vocab)
    best, where = [], []
    for _ in range(keep):
        index = torch.argmax(found, dim=1, keepdim=True)  # the first of equals
        best.append(torch.gather(found, 1, index))
        where.append(index)
        found.scatter_(1, index, -math.inf)
    best, where = torch.cat(best, 1), torch.cat(where, 1)
    parents, tokens = where // vocab, where % vocab
    done = torch.zeros_like(parents, dtype=torch.bool)
    if finished is not None:
        done = torch.gather(finished, 1, parents) | (tokens == end)
    return {"scores": torch.where(best <= nothing, -math.inf, best).float(), "parents": parents.to(torch.int32),
            "tokens": tokens, "finished": done}


def _plain_reorder(state):
    parents, caches = state["parents"].long(), state["caches"]
    groups, beams = parents.shape
    page, width = caches[0][0].shape[2], state["table"].shape[1]
    table = state["table"].view(groups, beams, width)
    length = state["lengths"].view(groups, beams)[:, :1].long()
    block, part = length // page, length % page
    followed = torch.gather(table, 1, parents[:, :, None].expand(-1, -1, width))
    column = torch.arange(width, device=table.device)[None, None]
    out = torch.where(column < block[:, :, None], followed, table)
    # The page in work: the first child keeps its parent's, the others take those of beams without children.
    here = torch.gather(table, 2, block.clamp(max=width - 1)[:, :, None].expand(-1, beams, 1))[:, :, 0]
    same = parents[:, :, None] == parents[:, None, :]
    earlier = torch.ones((beams, beams), dtype=torch.bool, device=table.device).tril(-1)
    first = ~(same & earlier).any(2)
    childless = ~(parents[:, None, :] == torch.arange(beams, device=table.device)[None, :, None]).any(2)
    spare = torch.argsort((~childless).to(torch.int8), dim=1, stable=True)
    rank = torch.cumsum((~first).long(), 1) - 1
    inherited = torch.gather(here, 1, parents)
    taken = torch.gather(here, 1, torch.gather(spare, 1, rank.clamp(min=0)))
    target = torch.where(first, inherited, taken)
    target = torch.where((part > 0) & (block < width), target, here)
    out = torch.where(column == block[:, :, None], target[:, :, None], out)
    source = torch.where((part > 0) & (block < width), inherited, target)
    moved = (torch.arange(page, device=table.device)[None, None] < part[:, :, None])[:, :, None, :, None]
    for pair in caches:
        for pages in pair:
            pages[target.long()] = torch.where(moved, pages[source.long()], pages[target.long()])
    return {"table": out.view(groups * beams, width), "pages": [pages for pair in caches for pages in pair]}


PLAIN = {"tables": _plain_tables, "append": _plain_append, "attend": _plain_attend, "select": _plain_select,
         "reorder": _plain_reorder}


# ---- the framework's operators ---------------------------------------------------------------------------------


def _own(state):
    from metile_b200 import backends

    kind = state["kind"]
    if kind == "tables":
        slots, positions, starts, lengths, free = backends.paged_resize(
            state["table"], state["lengths"], state["counts"], state["ring"], state["state"], page_size=state["page"],
            tokens=state["tokens"])
        return {"slots": slots, "positions": positions, "starts": starts, "lengths": lengths, "state": free,
                "table": state["table"], "ring": state["ring"]}
    if kind == "append":
        query = backends.rope_kv_append_paged(state["query"], state["key"], state["value"], state["inverse"],
                                              state["positions"], state["slots"], state["keys"], state["values"])
        return {"query": query, "keys": state["keys"], "values": state["values"]}
    if kind == "attend":
        return backends.paged_attention_decode(state["query"], state["keys"], state["values"], state["table"],
                                               state["lengths"], scale=state["scale"])
    if kind == "select":
        scores, parents, tokens, finished = backends.beam_select(state["logits"], state["scores"], keep=state["keep"],
                                                                 finished=state["finished"], end_token=state["end"])
        return {"scores": scores, "parents": parents, "tokens": tokens, "finished": finished}
    table = backends.beam_reorder(state["table"], state["lengths"], state["parents"], state["caches"])
    return {"table": table, "pages": [pages for pair in state["caches"] for pages in pair]}


def run(state):
    return _own(state) if own else PLAIN[state["kind"]](state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------


def work(case):
    kind, page = case["kind"], case.get("page")
    if kind == "tables":
        held, added = _table_requests(case)
        before, after = [_blocks(n, page) for n in held], [_blocks(n + c, page) for n, c in zip(held, added)]
        moved = sum(abs(a - b) for a, b in zip(after, before))
        tokens = sum(max(0, c) for c in added)
        return {"bytes": 12 * tokens + 16 * len(held) + 8 * moved, "flops": 4.0 * (tokens + len(held))}
    if kind == "append":
        values = case["tokens"] * case["kv_heads"] * (case["group"] + 2) * case["dim"]
        rotated = case["tokens"] * case["kv_heads"] * (case["group"] + 1) * case["dim"]
        return {"bytes": 2 * values * SIZES[case["type"]] + 12 * case["tokens"], "flops": 3.0 * rotated}
    if kind == "attend":
        lengths, size = _attend_lengths(case), SIZES[case["type"]]
        used, heads, dim = sum(lengths), case["kv_heads"] * case["group"], case["dim"]
        return {"bytes": size * (2 * used * case["kv_heads"] * dim + 2 * len(lengths) * heads * dim) + 4 * _blocks(used, page),
                "flops": 4.0 * used * heads * dim}
    if kind == "select":
        logits = case["groups"] * case["beams"] * case["vocab"]
        return {"bytes": logits * SIZES[case["type"]] + case["groups"] * (5 * case["beams"] + 17 * case["keep"]),
                "flops": 4.0 * logits}
    _, block, part = _used_block(case)
    extra = case["groups"] * (case["beams"] - _surviving(case["beams"]))
    moved = extra * case["layers"] * 2 * case["kv_heads"] * part * case["dim"]
    return {"bytes": 2 * moved * SIZES[case["type"]] + 8 * case["groups"] * case["beams"] * (block + 2), "flops": float(moved)}


# ---- from the definitions, in 64 bits ------------------------------------------------------------------------------


def exact(case, seed):
    kind = case["kind"]
    if kind in ("tables", "reorder"):
        return None  # whole numbers, and copies
    state = prepare(case, seed)
    if kind == "append":
        pairs = case["dim"] // 2
        turn = torch.outer(state["positions"].double(), state["inverse"].double())
        unit = torch.polar(torch.ones_like(turn), turn)[:, None, :]

        def turned(rows):
            wide = rows.double()
            spun = torch.complex(wide[..., :pairs].contiguous(), wide[..., pairs:].contiguous()) * unit
            return torch.cat([spun.real, spun.imag], dim=-1)

        keys, values = state["keys"].double(), state["values"].double()
        count = case["tokens"]
        page, row = state["slots"][:count] // case["page"], state["slots"][:count] % case["page"]
        keys[page, :, row] = turned(state["key"])[:count]
        values[page, :, row] = state["value"][:count].double()
        return {"query": turned(state["query"]), "keys": keys, "values": values}
    if kind == "attend":
        out = torch.zeros(state["query"].shape, dtype=torch.float64, device=state["query"].device)
        kv_heads, group, page = case["kv_heads"], case["group"], case["page"]
        for b, length in enumerate(state["lengths"].tolist()):
            if length == 0:
                continue
            pages = state["table"][b, :_blocks(length, page)].long()
            for h in range(kv_heads):
                k = state["keys"][pages, h].double().reshape(-1, case["dim"])[:length]
                v = state["values"][pages, h].double().reshape(-1, case["dim"])[:length]
                q = state["query"][b, h * group:(h + 1) * group].double()
                out[b, h * group:(h + 1) * group] = torch.softmax(q @ k.T * state["scale"], dim=1) @ v
        return out
    groups, beams = state["scores"].shape
    best = []
    for g in range(groups):
        rows = torch.log_softmax(state["logits"][g * beams:(g + 1) * beams].double(), dim=1)
        rows += state["scores"][g].double()[:, None]
        if state["finished"] is not None:
            for b in torch.nonzero(state["finished"][g]).flatten().tolist():
                rows[b] = -math.inf
                rows[b, state["end"]] = state["scores"][g, b].double()
        best.append(torch.sort(rows.flatten(), descending=True).values[:case["keep"]])
    return {"scores": torch.stack(best), "parents": None, "tokens": None, "finished": None}
