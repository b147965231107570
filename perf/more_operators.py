"""The operators of prompts read in pieces and of shared prompts, as cases that can be timed and compared.

The kinds, and what a serving program does with them:

  chunk    paged_attention_chunk: several new tokens per request -- a piece of a prompt, a draft to verify, one token --
           over the pages its row of the block table names, each seeing the tokens up to its own
  score    token_logprobs: log-probabilities of given tokens, the entropy and the best alternatives
  fork     paged_fork: empty requests go on from the first tokens of others; full pages are shared, begun ones copied
  free     paged_free: requests end; a page goes back when the last request that holds it has ended
  compact  paged_compact: the pages that are held move to the lowest ids

`run` is the plain form (elementary torch operations in 32 bits) or, with `own`, the framework's operators.  Head layouts
and widths are those of the tests and the benchmark (2 x 6 heads of 128, heads of 64, a vocabulary of 128256, 28
layers) and others around them; lengths run from one token to a hundred thousand.
"""

from __future__ import annotations

import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}

# No drawn case costs more than the largest listed one of its kind.
MOST_CHUNK_FLOPS = 0.9e12
MOST_CHUNK_BYTES = 700 << 20
MOST_LOGIT_BYTES = 1900 * 128256 * 2
MOST_PAGE_BYTES = 900 << 20
MOST_MOVED_BYTES = 60 << 20


def listed():
    return [
        # Drafts of five tokens verified for four short conversations: the latency of a step.
        {"name": "chunk_draft", "kind": "chunk", "requests": 4, "most": 5, "held": 700, "ragged": False, "kv_heads": 2,
         "group": 6, "dim": 128, "page": 16, "type": "bf16"},
        # A serving batch: most requests decode a token, some read a piece of their prompt, some have none.
        {"name": "chunk_mixed", "kind": "chunk", "requests": 37, "most": 500, "held": 6000, "ragged": True, "kv_heads": 8,
         "group": 4, "dim": 128, "page": 16, "type": "bf16"},
        # A question of seventeen tokens about a very long document, in fp16.
        {"name": "chunk_long", "kind": "chunk", "requests": 1, "most": 17, "held": 100003, "ragged": False, "kv_heads": 8,
         "group": 4, "dim": 128, "page": 32, "type": "fp16"},
        # A piece of 4093 tokens of a long prompt behind 11000 that are there: the most operations.
        {"name": "chunk_prompt", "kind": "chunk", "requests": 1, "most": 4093, "held": 11000, "ragged": False,
         "kv_heads": 8, "group": 4, "dim": 128, "page": 64, "type": "bf16"},
        # The tokens eight requests were given, with five alternatives; an odd vocabulary, so rows start anywhere.
        {"name": "score_8", "kind": "score", "rows": 8, "vocab": 32001, "top": 5, "type": "bf16"},
        # Every token of a prompt over a large vocabulary, twenty alternatives each.
        {"name": "score_prompt", "kind": "score", "rows": 2001, "vocab": 128256, "top": 20, "type": "bf16"},
        # Four answers to one prompt, through four layers.
        {"name": "fork_4", "kind": "fork", "groups": 1, "members": 4, "layers": 4, "kv_heads": 2, "dim": 128, "page": 16,
         "prompt": 500, "type": "bf16"},
        # Sixteen prompts with eight continuations each, through the 28 layers of a whole model.
        {"name": "fork_128", "kind": "fork", "groups": 16, "members": 8, "layers": 28, "kv_heads": 2, "dim": 128, "page": 32,
         "prompt": 1000, "type": "bf16"},
        # Two of five requests end.
        {"name": "free_5", "kind": "free", "groups": 1, "members": 5, "page": 16, "prompt": 300, "more": 200},
        # A batch of groups that share prompts; half of the requests end at once.
        {"name": "free_500", "kind": "free", "groups": 50, "members": 10, "page": 16, "prompt": 2500, "more": 900},
        # A small pool is put together after some requests have ended.
        {"name": "compact_8", "kind": "compact", "groups": 2, "members": 4, "layers": 4, "kv_heads": 2, "dim": 128,
         "page": 16, "prompt": 200, "more": 150, "type": "bf16"},
        # The pool of a whole model: half of its pages are free, and so a quarter of it moves.
        {"name": "compact_64", "kind": "compact", "groups": 16, "members": 4, "layers": 28, "kv_heads": 2, "dim": 128,
         "page": 32, "prompt": 500, "more": 250, "type": "bf16"},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("chunk", "chunk", "chunk", "score", "score", "fork", "free", "compact"))
    page = rng.choice((8, 16, 32, 64, 128, 256))
    half = rng.choice(("bf16", "fp16"))
    if kind == "chunk":
        case = {"kind": kind, "requests": _log_int(rng, 1, 64), "most": _log_int(rng, 1, 4096), "held": _log_int(rng, 1, 100000),
                "ragged": rng.random() < 0.6, "kv_heads": rng.choice((1, 2, 4, 8)), "group": rng.randint(1, 16),
                "dim": rng.choice((64, 128, 128, 256)), "page": page, "type": half}
        while work(case)["flops"] > MOST_CHUNK_FLOPS or work(case)["bytes"] > MOST_CHUNK_BYTES:
            largest = max(("requests", "most", "held"), key=lambda name: case[name] / {"requests": 8, "most": 256, "held": 4096}[name])
            case[largest] = max(1, case[largest] * 2 // 3)
        return case
    if kind == "score":
        vocab, name = _log_int(rng, 100, 131072), rng.choice(("bf16", "fp16", "fp32"))
        rows = min(_log_int(rng, 1, 4000), max(1, MOST_LOGIT_BYTES // (vocab * SIZES[name])))
        return {"kind": kind, "rows": rows, "vocab": vocab, "top": rng.choice((0, 1, 5, 20, rng.randint(1, 64))), "type": name}
    if kind == "free":
        return {"kind": kind, "groups": _log_int(rng, 1, 48), "members": rng.randint(1, 10), "page": rng.choice((16, 32, 64)),
                "prompt": _log_int(rng, 1, 2400), "more": _log_int(rng, 1, 900)}
    case = {"kind": kind, "groups": _log_int(rng, 1, 24), "members": rng.randint(1, 8), "layers": rng.randint(1, 28),
            "kv_heads": rng.choice((1, 2, 4)), "dim": rng.choice((64, 128)), "page": rng.choice((8, 16, 32)),
            "prompt": _log_int(rng, 1, 1000), "type": half}
    if kind == "compact":
        case["more"] = _log_int(rng, 1, 400)
    while _pool_bytes(case) > MOST_PAGE_BYTES or work(case)["bytes"] > 2 * MOST_MOVED_BYTES * (4 if kind == "compact" else 1):
        if case["layers"] > 1:
            case["layers"] = case["layers"] * 2 // 3
        else:
            case["groups"] = max(1, case["groups"] // 2)
    return case


# ---- what follows from a case alone ----------------------------------------------------------------------------


def _spread(count, low, high, step):
    """`count` whole numbers from low to high, spread evenly in an order that is not sorted."""
    return [low + (high - low) * (i * step % count) // max(1, count - 1) for i in range(count)]


def _blocks(tokens, page):
    return -(-tokens // page)


def _chunk_requests(case):
    """(new tokens, tokens with them) of every request."""
    requests, most, held = case["requests"], case["most"], case["held"]
    if not case["ragged"]:
        return [most] * requests, [held + most] * requests
    before, new = _spread(requests, 0, held, 7), []
    for i in range(requests):
        if requests > 2 and i == requests // 2:
            new.append(0)  # a row of the batch that has none this time
        elif i % 4 == 0:
            new.append(1 + (most - 1) * (i * 5 % requests) // max(1, requests - 1))
        else:
            new.append(1)
    return new, [b + n for b, n in zip(before, new)]


def _members(case):
    """Groups of requests that share the first `prompt` tokens or so: (prompt tokens, [tokens of each member])."""
    groups, members, more = case["groups"], case["members"], case.get("more", 0)
    prompts = _spread(groups, max(1, case["prompt"] * 2 // 3), case["prompt"], 5)
    return [(p, [p + n for n in _spread(members, 0, more, 3)]) for p in prompts]


def _fork_counts(case):
    """(prompt tokens, [tokens each new member takes]): all of the prompt, or a part."""
    return [(p, [max(1, p - (p // 3 if i % 4 == 3 else 0)) for i in range(case["members"])])
            for p in _spread(case["groups"], max(1, case["prompt"] * 2 // 3), case["prompt"], 5)]


def _held_pages(case):
    """Pages that a free or a compact case's requests hold."""
    page = case["page"]
    return sum(p // page + sum(_blocks(n, page) - p // page for n in lengths) for p, lengths in _members(case))


def _pool(case):
    page = case["page"]
    if case["kind"] == "fork":
        return sum(_blocks(p, page) + len(counts) for p, counts in _fork_counts(case)) + 9
    held = _held_pages(case)
    return held + (held if case["kind"] == "compact" else held // 3) + 7


def _pool_bytes(case):
    return 2 * case["layers"] * _pool(case) * case["kv_heads"] * case["page"] * case["dim"] * SIZES[case["type"]]


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

    def caches(self, case, pool):
        shape = pool, case["kv_heads"], case["page"], case["dim"]
        return [tuple(self.normal(*shape, dtype=TYPES[case["type"]]) for _ in range(2)) for _ in range(case["layers"])]


def _table_of(make, lengths, page, width, pool):
    """A block table whose rows name as many distinct pages as their lengths need, in no order; the rest is unused."""
    held = make.ints([_blocks(n, page) for n in lengths])
    used = torch.arange(width, device=make.device)[None] < held[:, None]
    first = torch.cumsum(held, 0) - held
    index = (first[:, None] + torch.arange(width, device=make.device)[None]).clamp(max=pool - 1)
    return torch.where(used, make.order(pool).to(torch.int32)[index], -1)


def _ring_of(make, pages, free):
    """A ring of `pages` entries with the ids `free` in it, across its end as often as not: (ring, state)."""
    start = int(make.uniform(1).item() * pages)
    ring = torch.full((pages,), -1, dtype=torch.int32, device=make.device)
    ring[(torch.arange(free.shape[0], device=make.device) + start) % pages] = free
    return ring, make.ints([start, free.shape[0]])


def _shared_state(make, case):
    """Tables of groups that share the full pages of their prompt, in an order of requests from the seed."""
    page, pool, rows, shares, at = case["page"], _pool(case), [], [], 0
    for prompt, lengths in _members(case):
        whole = prompt // page
        common = list(range(at, at + whole))
        at += whole
        shares += [len(lengths) - 1] * whole
        for n in lengths:
            count = _blocks(n, page) - whole
            rows.append((n, common + list(range(at, at + count))))
            shares += [0] * count
            at += count
    rows = [rows[i] for i in make.order(len(rows)).tolist()]
    width = max(len(ids) for _, ids in rows) + 2
    names = make.order(pool).to(torch.int32)
    index = make.ints([ids + [-1] * (width - len(ids)) for _, ids in rows])
    table = torch.where(index >= 0, names[index.clamp(min=0).long()], -1)
    counted = torch.zeros((pool,), dtype=torch.int32, device=make.device)
    counted[names[:at].long()] = make.ints(shares)
    return table, make.ints([n for n, _ in rows]), counted, names[at:], pool


def prepare(case, seed):
    make, kind, page = _Maker(seed), case["kind"], case.get("page")
    if kind == "chunk":
        new, lengths = _chunk_requests(case)
        order = make.order(len(new)).tolist()
        new, lengths = [new[i] for i in order], [lengths[i] for i in order]
        dim, kv_heads, dtype = case["dim"], case["kv_heads"], TYPES[case["type"]]
        pool = sum(_blocks(n, page) for n in lengths) + 3
        width = _blocks(max(max(lengths), 1), page) + 3
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        return {"kind": kind, "query": make.normal(starts[-1], kv_heads * case["group"], dim, std=2.0, dtype=dtype),
                "keys": make.normal(pool, kv_heads, page, dim, dtype=dtype),
                "values": make.normal(pool, kv_heads, page, dim, dtype=dtype),
                "table": _table_of(make, lengths, page, width, pool), "lengths": make.ints(lengths), "starts": make.ints(starts),
                "scale": dim ** -0.5, "host_new": new, "host_lengths": lengths}
    if kind == "score":
        logits = make.normal(case["rows"], case["vocab"], std=2.5, dtype=TYPES[case["type"]])
        tokens = (make.uniform(case["rows"]) * case["vocab"]).long().clamp(max=case["vocab"] - 1)
        return {"kind": kind, "logits": logits, "tokens": tokens, "top": min(case["top"], case["vocab"])}
    if kind == "fork":
        requests = []  # (tokens held, group or -1, tokens to take)
        for group, (prompt, counts) in enumerate(_fork_counts(case)):
            requests.append((prompt, group, 0))
            requests += [(0, group, count) for count in counts]
        requests = [requests[i] for i in make.order(len(requests)).tolist()]
        owner = {group: row for row, (held, group, _) in enumerate(requests) if held}
        lengths, pool = [held for held, _, _ in requests], _pool(case)
        width = _blocks(max(lengths), page) + 2
        table = _table_of(make, lengths, page, width, pool)
        used = torch.zeros((pool + 1,), dtype=torch.bool, device=make.device)
        used[torch.where(table < 0, pool, table).long().view(-1)] = True
        order = make.order(pool)
        ring, state = _ring_of(make, pool, order[~used[order]].to(torch.int32))
        return {"kind": kind, "table": table, "lengths": make.ints(lengths),
                "sources": make.ints([-1 if held else owner[group] for held, group, _ in requests]),
                "counts": make.ints([count for _, _, count in requests]), "ring": ring, "state": state,
                "shares": torch.zeros((pool,), dtype=torch.int32, device=make.device), "caches": make.caches(case, pool)}
    table, lengths, shares, free, pool = _shared_state(make, case)
    if kind == "free":
        ring, state = _ring_of(make, pool, free)
        # Of one group the first two requests, of several every other one on the whole: some shared pages lose all who hold them.
        ended = torch.arange(lengths.shape[0], device=make.device) < 2 if case["groups"] == 1 else make.uniform(lengths.shape[0]) < 0.5
        return {"kind": kind, "table": table, "lengths": lengths, "ended": ended, "ring": ring, "state": state, "shares": shares,
                "page": page}
    return {"kind": kind, "table": table, "lengths": lengths, "caches": make.caches(case, pool)}


# ---- the plain forms --------------------------------------------------------------------------------------------


def _plain_chunk(state):
    query, keys, values, table, scale = state["query"], state["keys"], state["values"], state["table"], state["scale"]
    rows, heads, dim = query.shape
    _, kv_heads, page, _ = keys.shape
    group = heads // kv_heads
    out, first = torch.zeros_like(query), 0
    for request, (new, length) in enumerate(zip(state["host_new"], state["host_lengths"])):
        if new == 0:
            continue
        index = table[request, :_blocks(length, page)].long()
        k = keys[index].float().transpose(0, 1).reshape(kv_heads, -1, dim)[:, :length]
        v = values[index].float().transpose(0, 1).reshape(kv_heads, -1, dim)[:, :length]
        step = max(1, (1 << 28) // (heads * length))  # rows at once
        for at in range(0, new, step):
            n = min(step, new - at)
            q = query[first + at:first + at + n].float().view(n, kv_heads, group, dim).permute(1, 2, 0, 3).reshape(kv_heads, group * n, dim)
            scores = torch.matmul(q, k.transpose(1, 2)).view(kv_heads, group, n, length) * scale
            position = torch.arange(length - new + at, length - new + at + n, device=query.device)
            scores.masked_fill_(torch.arange(length, device=query.device)[None] > position[:, None], -math.inf)
            scores -= scores.amax(-1, keepdim=True)
            scores.exp_()
            total = scores.sum(-1, keepdim=True)
            found = torch.matmul(scores.view(kv_heads, group * n, length), v).view(kv_heads, group, n, dim) / total
            out[first + at:first + at + n] = found.permute(2, 0, 1, 3).reshape(n, heads, dim).to(query.dtype)
        first += new
    return out


def _plain_score(state):
    logits, tokens, top = state["logits"].float(), state["tokens"], state["top"]
    logits = logits - logits.amax(1, keepdim=True)
    logits = logits - torch.log(torch.exp(logits).sum(1, keepdim=True))
    logprobs = torch.gather(logits, 1, tokens[:, None])[:, 0]
    entropy = -(torch.exp(logits) * logits).sum(1)
    left, best, where = state["logits"].float(), [], []  # ordered as the logits are
    for _ in range(top):
        index = torch.argmax(left, dim=1, keepdim=True)  # the first of equals
        best.append(torch.gather(logits, 1, index))
        where.append(index)
        left.scatter_(1, index, -math.inf)
    empty = logits.new_zeros((logits.shape[0], 0))
    return {"logprobs": logprobs, "entropy": entropy, "top_logprobs": torch.cat([empty, *best], 1),
            "top_tokens": torch.cat([empty.long(), *where], 1)}


def _plain_fork(state):
    table, lengths, sources, counts = state["table"], state["lengths"].long(), state["sources"].long(), state["counts"].long()
    ring, caches = state["ring"], state["caches"]
    page, pool, width, requests = caches[0][0].shape[2], ring.shape[0], table.shape[1], table.shape[0]
    first, free = state["state"][0].long(), state["state"][1].long()
    source = sources.clamp(0, requests - 1)
    valid = (sources >= 0) & (sources < requests) & (source != torch.arange(requests, device=table.device))
    valid &= (lengths == 0) & (counts > 0) & (counts <= lengths[source]) & (lengths[source] <= width * page)
    whole, part = counts // page, counts % page
    need = (valid & (part > 0)).long()
    reach = torch.cumsum(need, 0)
    served = valid & ((need == 0) | (reach <= free))
    granted = torch.where(served, need, 0).sum()
    column = torch.arange(width, device=table.device)[None]
    shared = served[:, None] & (column < whole[:, None])
    taken = ring[(first + reach - need) % pool]
    begun = served & (part > 0)
    old = torch.gather(table[source], 1, whole.clamp(0, width - 1)[:, None])[:, 0]  # the page each begun one is a copy of
    new = torch.where(shared, table[source], table)
    new = torch.where(begun[:, None] & (column == whole[:, None]), taken[:, None], new)
    shares = torch.cat([state["shares"], state["shares"].new_zeros(1)])
    shares.index_put_((torch.where(shared, table[source], pool).long().view(-1),), torch.ones((), dtype=torch.int32, device=table.device),
                      accumulate=True)
    table.copy_(new)
    # A request without a page of its own to fill repeats the copy of one that has.
    some = torch.argmax(begun.to(torch.int8))
    pick = torch.where(begun, torch.arange(requests, device=table.device), some)
    to, of, rows = taken[pick].long(), old[pick].long(), part[pick]
    moved = (torch.arange(page, device=table.device)[None] < rows[:, None])[:, None, :, None] & begun[some]
    to, of = torch.where(begun[some], to, 0), torch.where(begun[some], of, 0)
    for pair in caches:
        for pages in pair:
            pages[to] = torch.where(moved, pages[of], pages[to])
    return {"table": table, "lengths": torch.where(served, counts, lengths).to(torch.int32),
            "state": torch.stack([(first + granted) % pool, free - granted]).to(torch.int32), "shares": shares[:pool],
            "pages": [pages for pair in caches for pages in pair]}


def _plain_free(state):
    table, lengths, ended, ring, shares = state["table"], state["lengths"], state["ended"], state["ring"], state["shares"]
    page, pool, width = state["page"], ring.shape[0], table.shape[1]
    first, free = state["state"][0].long(), state["state"][1].long()
    held = (lengths.long() + page - 1) // page
    dropped = (ended[:, None] & (torch.arange(width, device=table.device)[None] < held[:, None])).view(-1)
    ids = torch.where(dropped, table.view(-1), pool).long()
    place = torch.arange(ids.shape[0], device=table.device)
    drops = torch.zeros((pool + 1,), dtype=torch.long, device=table.device).scatter_add_(0, ids, torch.ones_like(ids))
    earliest = torch.full((pool + 1,), ids.shape[0], dtype=torch.long, device=table.device).scatter_reduce_(0, ids, place, "amin")
    longer = torch.cat([shares, shares.new_zeros(1)]).long()
    gone = drops > longer
    back = dropped & gone[ids] & (earliest[ids] == place)
    rank = torch.cumsum(back.long(), 0)
    target = torch.where(back, (first + free + rank - 1) % pool, pool)
    kept = torch.cat([ring, ring.new_zeros(1)])
    kept[target] = ids.to(torch.int32)
    ring.copy_(kept[:pool])
    return {"lengths": torch.where(ended, 0, lengths), "state": torch.stack([first, free + rank[-1]]).to(torch.int32),
            "shares": torch.where(gone, 0, longer - drops)[:pool].to(torch.int32), "ring": ring}


def _plain_compact(state):
    table, lengths, caches = state["table"], state["lengths"].long(), state["caches"]
    pool, page, width = caches[0][0].shape[0], caches[0][0].shape[2], table.shape[1]
    held = (lengths + page - 1) // page
    inside = torch.arange(width, device=table.device)[None] < held[:, None]
    ids = torch.where(inside, table, pool).long()
    holders = torch.zeros((pool + 1,), dtype=torch.long, device=table.device)
    holders.scatter_add_(0, ids.view(-1), torch.ones_like(ids.view(-1)))
    holders = holders[:pool]
    used = holders > 0
    count = used.sum()
    page_id = torch.arange(pool, device=table.device)
    moves, holes = used & (page_id >= count), ~used & (page_id < count)
    # The n-th page that moves goes to the n-th hole; there are as many of one as of the other.
    order = torch.argsort((~holes).to(torch.int8), stable=True)
    rank = torch.cumsum(moves.long(), 0) - 1
    place = torch.where(moves, order[rank.clamp(min=0)], page_id)
    # Every page is written where it goes; one that is not held and not in a hole stays what it is.
    source = torch.arange(pool + 1, device=table.device)
    source[torch.where(moves, place, pool)] = page_id
    source = source[:pool]
    for pair in caches:
        for pages in pair:
            for start in range(0, pool, 256):
                # Sources lie behind the last hole, so nothing is read that has been written.
                pages[start:start + 256] = pages[source[start:start + 256]]
    shares = torch.zeros((pool + 1,), dtype=torch.long, device=table.device)
    shares[torch.where(used, place, pool)] = (holders - 1).clamp(min=0)
    longer = torch.cat([place, place.new_zeros(1)])
    return {"table": torch.where(inside, longer[ids].to(torch.int32), table), "ring": ((count + page_id) % pool).to(torch.int32),
            "state": torch.stack([torch.zeros_like(count), pool - count]).to(torch.int32), "shares": shares[:pool].to(torch.int32),
            "pages": [pages for pair in caches for pages in pair]}


PLAIN = {"chunk": _plain_chunk, "score": _plain_score, "fork": _plain_fork, "free": _plain_free, "compact": _plain_compact}


# ---- the framework's operators ---------------------------------------------------------------------------------


def _own(state):
    from metile_b200 import backends

    kind = state["kind"]
    if kind == "chunk":
        return backends.paged_attention_chunk(state["query"], state["keys"], state["values"], state["table"], state["lengths"],
                                              state["starts"], scale=state["scale"])
    if kind == "score":
        logprobs, entropy, best, where = backends.token_logprobs(state["logits"], state["tokens"], top=state["top"])
        return {"logprobs": logprobs, "entropy": entropy, "top_logprobs": best, "top_tokens": where}
    if kind == "fork":
        lengths, free, shares = backends.paged_fork(state["table"], state["lengths"], state["sources"], state["counts"],
                                                    state["ring"], state["state"], state["shares"], state["caches"])
        return {"table": state["table"], "lengths": lengths, "state": free, "shares": shares,
                "pages": [pages for pair in state["caches"] for pages in pair]}
    if kind == "free":
        lengths, free, shares = backends.paged_free(state["table"], state["lengths"], state["ended"], state["ring"],
                                                    state["state"], state["shares"], page_size=state["page"])
        return {"lengths": lengths, "state": free, "shares": shares, "ring": state["ring"]}
    table, ring, free, shares = backends.paged_compact(state["table"], state["lengths"], state["caches"])
    return {"table": table, "ring": ring, "state": free, "shares": shares,
            "pages": [pages for pair in state["caches"] for pages in pair]}


def run(state):
    return _own(state) if own else PLAIN[state["kind"]](state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------


def work(case):
    kind, page = case["kind"], case.get("page")
    if kind == "chunk":
        new, lengths = _chunk_requests(case)
        size, dim, kv_heads, heads = SIZES[case["type"]], case["dim"], case["kv_heads"], case["kv_heads"] * case["group"]
        used = sum(length for n, length in zip(new, lengths) if n)
        seen = sum(n * (length - n) + n * (n + 1) // 2 for n, length in zip(new, lengths))
        return {"bytes": size * (2 * used * kv_heads * dim + 2 * sum(new) * heads * dim) + 4 * _blocks(used, page),
                "flops": 4.0 * dim * heads * seen}
    if kind == "score":
        logits = case["rows"] * case["vocab"]
        return {"bytes": logits * SIZES[case["type"]] + case["rows"] * (16 + 12 * case["top"]), "flops": 5.0 * logits}
    if kind == "fork":
        parts = sum(count % page for _, counts in _fork_counts(case) for count in counts)
        entries = sum(_blocks(count, page) for _, counts in _fork_counts(case) for count in counts)
        moved = parts * case["layers"] * 2 * case["kv_heads"] * case["dim"]
        return {"bytes": 2 * moved * SIZES[case["type"]] + 16 * entries, "flops": float(moved + entries)}
    if kind == "free":
        dropped = sum(_blocks(n, page) for _, lengths in _members(case) for n in lengths) // 2
        return {"bytes": 16 * dropped + 8 * _pool(case), "flops": float(2 * dropped)}
    entries = sum(_blocks(n, page) for _, lengths in _members(case) for n in lengths)
    held, pool = _held_pages(case), _pool(case)
    moved = held * (pool - held) // pool * page * case["layers"] * 2 * case["kv_heads"] * case["dim"]  # those above, on the whole
    return {"bytes": 2 * moved * SIZES[case["type"]] + 8 * entries + 8 * pool, "flops": float(moved + entries)}


# ---- from the definitions, in 64 bits ------------------------------------------------------------------------------


def exact(case, seed):
    kind = case["kind"]
    if kind in ("fork", "free", "compact"):
        return None  # whole numbers, and copies
    state = prepare(case, seed)
    if kind == "score":
        rows, top = state["logits"].shape[0], state["top"]
        chosen, entropy, best = [], [], []
        for at in range(0, rows, 256):
            logs = torch.log_softmax(state["logits"][at:at + 256].double(), dim=1)
            chosen.append(logs[torch.arange(logs.shape[0], device=logs.device), state["tokens"][at:at + 256]])
            entropy.append(-(logs.exp() * logs).sum(1))
            best.append(torch.sort(logs, dim=1, descending=True).values[:, :top])
        return {"logprobs": torch.cat(chosen), "entropy": torch.cat(entropy), "top_logprobs": torch.cat(best), "top_tokens": None}
    out = torch.zeros(state["query"].shape, dtype=torch.float64, device=state["query"].device)
    page, group = case["page"], case["group"]
    starts, lengths = state["starts"].tolist(), state["lengths"].tolist()
    for b, length in enumerate(lengths):
        first, last = starts[b], starts[b + 1]
        if first == last:
            continue
        ids = state["table"][b, :_blocks(length, page)].long()
        for head in range(case["kv_heads"] * group):
            k = state["keys"][ids, head // group].double().reshape(-1, case["dim"])[:length]
            v = state["values"][ids, head // group].double().reshape(-1, case["dim"])[:length]
            logits = state["query"][first:last, head].double() @ k.T * state["scale"]
            hidden = torch.ones_like(logits, dtype=torch.bool).triu(length - (last - first) + 1)
            out[first:last, head] = torch.softmax(logits.masked_fill(hidden, -math.inf), dim=1) @ v
    return out
