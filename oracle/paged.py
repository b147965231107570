"""The paged key-value cache and beam search in numpy, in 64 bits, request by request: the oracle of metile_b200's
paged_resize, rope_kv_append_paged, paged_attention_decode, paged_attention_chunk, paged_fork, paged_free, paged_compact,
token_logprobs, beam_select and beam_reorder."""

import numpy as np


def resize(tables, lengths, counts, ring, state, page, tokens):
    """Returns (slots, positions, starts, lengths, state, tables, ring); nothing is changed in place."""
    tables, ring = tables.copy(), ring.copy()
    width, pool = tables.shape[1], len(ring)
    first, free = int(state[0]), int(state[1])
    slots, positions = np.full(tokens, -1, np.int64), np.zeros(tokens, np.int32)
    starts, out = [0], [int(n) for n in lengths]
    asked = granted = freed = 0
    for r, (length, count) in enumerate(zip(out[:], (int(c) for c in counts))):
        begin, after = starts[-1], length + count
        starts.append(begin + max(count, 0))
        valid = 0 <= length <= width * page and 0 <= after <= width * page and (count <= 0 or starts[-1] <= tokens)
        old, new = -(-length // page), -(-after // page)
        served = valid
        if valid and new > old:
            asked += new - old
            served = asked <= free
            if served:
                for i, block in enumerate(range(old, new)):
                    tables[r, block] = ring[(first + asked - (new - old) + i) % pool]
                granted += new - old
        if valid and new < old:
            for block in range(new, old):
                ring[(first + free + freed) % pool] = tables[r, block]
                freed += 1
        for i in range(max(count, 0)):
            if begin + i >= tokens:
                break
            if served:
                at = positions[begin + i] = length + i
                page_id = int(tables[r, at // page])
                slots[begin + i] = page_id * page + at % page if page_id >= 0 else -1
        if served:
            out[r] = after
    state = np.array([(first + granted) % pool, free - granted + freed], np.int32)
    return slots, positions, np.minimum(starts, 2**31 - 1).astype(np.int32), np.array(out, np.int32), state, tables, ring


def rotate(rows, inverse, positions):
    """rows [R, H, D] float64, pair (i, i + D/2) of row r turned by positions[r] * inverse[i]."""
    half = rows.shape[-1] // 2
    angle = positions.astype(np.float64)[:, None] * inverse.astype(np.float64)[None]
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    a, b = rows[..., :half], rows[..., half:]
    return np.concatenate([a * c - b * s, b * c + a * s], axis=-1)


def attention(query, keys, values, tables, lengths, scale):
    """query [B, Hq, D], pages [P, Hkv, page, D], all float64; returns (out, sum of weight * |value|, largest sum of
    |products| behind a score)."""
    batch, heads, dim = query.shape
    _, kv_heads, page, _ = keys.shape
    group = heads // kv_heads
    out, weight, reach = np.zeros_like(query), np.zeros_like(query), 0.0
    for b in range(batch):
        n = int(lengths[b])
        if n == 0:
            continue
        ids = tables[b, :-(-n // page)]
        for h in range(kv_heads):
            k = keys[ids, h].reshape(-1, dim)[:n]
            v = values[ids, h].reshape(-1, dim)[:n]
            q = query[b, h * group:(h + 1) * group]
            score = q @ k.T * scale
            reach = max(reach, float((np.abs(q) @ np.abs(k).T).max() * abs(scale)))
            p = np.exp(score - score.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            out[b, h * group:(h + 1) * group] = p @ v
            weight[b, h * group:(h + 1) * group] = p @ np.abs(v)
    return out, weight, reach


def beam_select(logits, scores, keep, finished=None, end=-1):
    """logits [G * K, V] and scores [G, K] float64; returns (scores, parents, tokens, finished).  Equal candidates: the lower
    beam, then the larger logit, then the lower token."""
    groups, beams = scores.shape
    vocab = logits.shape[1]
    best, parents, tokens, done = [], [], [], []
    for g in range(groups):
        found, own = np.full((beams, vocab), -np.inf), np.zeros((beams, vocab))
        for k in range(beams):
            score, row = scores[g, k], logits[g * beams + k]
            if not score > -1e9:
                continue
            if finished is not None and finished[g, k]:
                found[k, end] = score
                continue
            top = row.max()
            if not np.isfinite(top):  # NaN, +inf, or nothing above -inf
                continue
            found[k], own[k] = score + ((row - top) - np.log(np.exp(row - top).sum())), row
        flat = found.reshape(-1)
        order = np.lexsort((np.arange(flat.size), -own.reshape(-1), np.arange(flat.size) // vocab, -flat))[:keep]
        best.append(flat[order])
        parents.append(order // vocab)
        tokens.append(order % vocab)
        done.append([bool((finished is not None and finished[g, o // vocab]) or o % vocab == end) for o in order])
    return np.array(best), np.array(parents, np.int32), np.array(tokens, np.int64), np.array(done)


def reorder(tables, lengths, parents, caches, page):
    """Returns (tables, caches); nothing is changed in place.  Caches: list of arrays [P, H, page, D]."""
    out, moved = tables.copy(), [pages.copy() for pages in caches]
    groups, beams = parents.shape
    for g in range(groups):
        base = g * beams
        block, part = divmod(int(lengths[base]), page)
        spare = [j for j in range(beams) if j not in parents[g]]
        seen = set()
        for k in range(beams):
            parent = int(parents[g, k])
            out[base + k, :block] = tables[base + parent, :block]
            if part == 0:
                continue
            owner = parent
            if parent in seen:
                owner = spare.pop(0)
                source, target = tables[base + parent, block], tables[base + owner, block]
                for old, new in zip(caches, moved):
                    new[target, :, :part] = old[source, :, :part]
            seen.add(parent)
            out[base + k, block] = tables[base + owner, block]
    return out, moved


def chunk_attention(query, keys, values, tables, lengths, starts, scale):
    """query [rows, Hq, D], pages [P, Hkv, page, D], all float64; rows starts[r] .. starts[r + 1] are the last tokens of request r,
    each seeing the tokens up to its own.  Returns (out, sum of weight * |value|, largest sum of |products| behind a score)."""
    rows, heads, dim = query.shape
    _, kv_heads, page, _ = keys.shape
    group = heads // kv_heads
    out, weight, reach = np.zeros_like(query), np.zeros_like(query), 0.0
    for r in range(len(lengths)):
        first, end, n = int(starts[r]), int(starts[r + 1]), int(lengths[r])
        if first == end:
            continue
        ids = tables[r, :-(-n // page)]
        for h in range(kv_heads):
            k = keys[ids, h].reshape(-1, dim)[:n]
            v = values[ids, h].reshape(-1, dim)[:n]
            q = query[first:end, h * group:(h + 1) * group]                   # [tokens, group, D]
            position = n - (end - first) + np.arange(end - first)
            for i in range(end - first):
                seen = int(position[i]) + 1
                if seen <= 0:
                    continue
                score = q[i] @ k[:seen].T * scale
                reach = max(reach, float((np.abs(q[i]) @ np.abs(k[:seen]).T).max() * abs(scale)))
                p = np.exp(score - score.max(1, keepdims=True))
                p /= p.sum(1, keepdims=True)
                out[first + i, h * group:(h + 1) * group] = p @ v[:seen]
                weight[first + i, h * group:(h + 1) * group] = p @ np.abs(v[:seen])
    return out, weight, reach


def fork(tables, lengths, sources, counts, ring, state, shares, caches, page):
    """Returns (tables, lengths, state, shares, caches); nothing is changed in place.  Caches: list of arrays [P, H, page, D]."""
    new, held, counted, moved = tables.copy(), lengths.copy(), shares.copy(), [pages.copy() for pages in caches]
    first, free, asked, granted = int(state[0]), int(state[1]), 0, 0
    for r in range(len(lengths)):
        source, count = int(sources[r]), int(counts[r])
        if not 0 <= source < len(lengths) or source == r or lengths[r] != 0 or not 0 < count <= lengths[source] \
                or lengths[source] > tables.shape[1] * page:
            continue
        whole, part = divmod(count, page)
        if part:
            asked += 1
            if asked > free:
                continue
            granted += 1
            new[r, whole] = ring[(first + asked - 1) % len(ring)]
            for old, pages in zip(caches, moved):
                pages[new[r, whole], :, :part] = old[tables[source, whole], :, :part]
        for j in range(whole):
            new[r, j] = tables[source, j]
            counted[tables[source, j]] += 1
        held[r] = count
    return new, held, np.array([(first + granted) % len(ring), free - granted], np.int32), counted, moved


def free(tables, lengths, ended, ring, state, shares, page):
    """Returns (lengths, state, shares, ring); nothing is changed in place."""
    held, ring, counted = lengths.copy(), ring.copy(), shares.copy()
    first, available = int(state[0]), int(state[1])
    order, drops = [], {}
    for r in range(len(lengths)):
        if not ended[r] or not 0 <= lengths[r] <= tables.shape[1] * page:
            continue
        for j in range(-(-int(lengths[r]) // page)):
            one = int(tables[r, j])
            if one not in drops:
                order.append(one)
            drops[one] = drops.get(one, 0) + 1
        held[r] = 0
    returned = 0
    for one in order:
        if drops[one] > shares[one]:
            ring[(first + available + returned) % len(ring)] = one
            returned += 1
        counted[one] = max(0, shares[one] - drops[one])
    return held, np.array([first, available + returned], np.int32), counted, ring


def compact(tables, lengths, caches, page):
    """Returns (tables, ring, state, shares, caches); nothing is changed in place."""
    pages = len(caches[0])
    holders = np.zeros(pages, np.int64)
    inside = np.arange(tables.shape[1])[None] < -(-lengths.astype(np.int64) // page)[:, None]
    np.add.at(holders, tables[inside], 1)
    held = int((holders > 0).sum())
    place, moved = np.arange(pages), [one.copy() for one in caches]
    for source, target in zip([i for i in range(held, pages) if holders[i]], [i for i in range(held) if not holders[i]]):
        place[source] = target
        for old, new in zip(caches, moved):
            new[target] = old[source]
    out, shares = tables.copy(), np.zeros(pages, np.int32)
    out[inside] = place[tables[inside]]
    for i in range(pages):
        if holders[i]:
            shares[place[i]] = holders[i] - 1
    return out, ((held + np.arange(pages)) % pages).astype(np.int32), np.array([0, pages - held], np.int32), shares, moved


def token_logprobs(logits, tokens, top):
    """logits [R, V] float64; returns (logprobs, entropy, top_logprobs, top_tokens), the largest first, the lower token among equals."""
    rows, vocab = logits.shape
    chosen, entropy, best, where = np.full(rows, np.nan), np.full(rows, np.nan), np.full((rows, top), np.nan), np.full((rows, top), -1, np.int64)
    for r in range(rows):
        largest = logits[r].max()
        if np.isfinite(largest):
            d = logits[r] - largest
            logs = d - np.log(np.exp(d).sum())
            p = np.exp(logs)
            entropy[r] = -(p * np.where(p > 0, logs, 0.0)).sum()
            if 0 <= tokens[r] < vocab:
                chosen[r] = logs[tokens[r]]
            where[r] = np.lexsort((np.arange(vocab), -logits[r]))[:top]
            best[r] = logs[where[r]]
        if tokens[r] < 0:
            chosen[r] = 0.0
    return chosen, entropy, best, where
