"""The full-attention layers' operators restated on the CPU: page tables by a
loop over requests, attention row by row in 64 bits."""
from __future__ import annotations

import numpy as np

STATUS_SPAN, STATUS_PAGES, STATUS_TABLE = 1, 8, 16


def page_plan(prefix_len, new_len, block_table, held, free_pages, free_pos, *, page_size, rows, trim=False, depth=None):
    """One request after the other.  Arrays in, dict of arrays out; the table
    and the ring come back as copies."""
    table, ring = np.array(block_table), np.array(free_pages)
    B, cols, cap = table.shape[0], table.shape[1], len(ring)
    head, tail = int(free_pos[0]), int(free_pos[1])
    free = min(max(tail - head, 0), cap)
    out = dict(slots=np.full(rows, -1, np.int64), positions=np.zeros(rows, np.int64), cu_seqlens=np.zeros(B + 1, np.int32),
               seq_len=np.zeros(B, np.int32), held=np.zeros(B, np.int32), status=np.zeros(B, np.int32))
    row = asked = taken = returned = given = 0
    for b in range(B):
        prefix, n = max(int(prefix_len[b]), 0), max(int(new_len[b]), 0)
        n = min(n, rows - row)
        status = STATUS_SPAN if n != new_len[b] or prefix_len[b] < 0 else 0
        have, want = min(max(int(held[b]), 0), cols), -(-(prefix + n) // page_size)
        end = have
        if want > cols:
            status |= STATUS_TABLE
        elif want > have:
            asked += want - have
            if asked > free:
                status |= STATUS_PAGES
            else:
                for c in range(have, want):
                    table[b, c] = free_pages[(head + taken) % cap]
                    taken += 1
                end = want
        elif trim and want < have:
            returned += have - want
            if returned > cap - free:
                status |= STATUS_PAGES
            else:
                for c in range(want, have):
                    ring[(tail + given) % cap] = block_table[b][c]
                    given += 1
                end = want
        served = not status & (STATUS_PAGES | STATUS_TABLE)
        for i in range(n):
            place = prefix + i
            out["positions"][row + i] = prefix + depth[row + i] if depth is not None else place
            if served:
                page = int(table[b, place // page_size])
                out["slots"][row + i] = page * page_size + place % page_size if page >= 0 else -1
        row += n
        out["cu_seqlens"][b + 1] = row
        out["seq_len"][b] = prefix + n if served else 0
        out["held"][b], out["status"][b] = end, status
    return out | {"free_pos": np.array([head + taken, tail + given]), "block_table": table, "free_pages": ring}


def kv_append(k, v, key_cache, value_cache, slots, rows=None):
    """Copies of the caches [pages, page_size, heads, d] with the rows in their slots, and the status word."""
    key_cache, value_cache, status = np.array(key_cache), np.array(value_cache), 0
    pages, ps = key_cache.shape[:2]
    for i, s in enumerate(slots):
        r = i if rows is None else int(rows[i])
        if s < 0 or r < 0:
            continue
        if s >= pages * ps or r >= len(k):
            status = 1
            continue
        key_cache[s // ps, s % ps], value_cache[s // ps, s % ps] = k[r], v[r]
    return key_cache, value_cache, status


def attend(q, k, v, sees, scale):
    """q [n, hq, d] over k, v [L, hkv, d]; sees [n, L].  Returns (o, lse,
    weight [n, hq, d] = sum_j p_j |v_j|, reach [n, hq] = the largest |scale| *
    sum |q| |k| of a visible key): the last two scale the rounding bounds.
    A key that a row does not see takes no part, whatever it holds."""
    n, hq, d = q.shape
    hkv = k.shape[1]
    o, lse = np.zeros((n, hq, d)), np.full((n, hq), -np.inf)
    weight, reach = np.zeros((n, hq, d)), np.zeros((n, hq))
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    for i in range(n):
        at = np.flatnonzero(sees[i])
        if not len(at):
            continue
        for h in range(hq):
            g = h * hkv // hq
            with np.errstate(invalid="ignore", over="ignore"):
                s = scale * (k[at, g] @ q[i, h])
                top = s.max()
                p = np.exp(s - top)
                total = p.sum()
                lse[i, h] = top + np.log(total)
                o[i, h] = (p / total) @ v[at, g]
                weight[i, h] = (p / total) @ np.abs(v[at, g])
                reach[i, h] = abs(scale) * (np.abs(k[at, g]) @ np.abs(q[i, h])).max()
    return o, lse, weight, reach


def sees_causal(n, keys):
    """Row i of the last n of `keys` tokens sees the ones up to its own."""
    return np.arange(keys) <= (keys - n + np.arange(n))[:, None]


def sees_tree(words, keys):
    """words: the nodes' ancestor-or-self bits (uint64); the nodes are the last tokens."""
    words = np.asarray(words).astype(np.uint64)
    n = len(words)
    at = np.arange(keys) - (keys - n)
    bit = (words[:, None] >> np.clip(at, 0, 63).astype(np.uint64)) & np.uint64(1)
    return (at < 0) | (bit == 1)


def paged_keys(cache, table_row, keys):
    """One request's tokens of a cache [pages, page_size, heads, d], and which
    of them are there: none of a page outside the cache or past the table."""
    pages, ps = cache.shape[:2]
    out, there = np.zeros((keys, *cache.shape[2:]), cache.dtype), np.zeros(keys, bool)
    for j in range(min(keys, len(table_row) * ps)):
        page = int(table_row[j // ps])
        if 0 <= page < pages:
            out[j], there[j] = cache[page, j % ps], True
    return out, there
