"""The paged key-value cache and beam search in numpy, in 64 bits, request by request: the oracle of metile_b200's
paged_resize, rope_kv_append_paged, paged_attention_decode, beam_select and beam_reorder."""

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
