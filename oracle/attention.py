"""Attention over a paged cache, token weights and eviction, row by row in float64 (numpy)."""

from __future__ import annotations

import numpy as np


def gather(cache: np.ndarray, row: np.ndarray, n: int, part: int) -> np.ndarray:
    """The first ``n`` tokens' keys (part 0) or values (1) of a table row: [n, heads, dim]."""
    block = cache.shape[2]
    ids = row[: -(-n // block)]
    x = cache[ids, part].reshape(len(ids) * block, cache.shape[3], cache.shape[4])
    return x[:n].astype(np.float64)


def attend(query, cache, table, lens, scale, query_start=None, pool_ok=None):
    """out [tokens, q_heads, dim], lse [tokens, q_heads] and per row the weights [kv_heads, n] it gives its tokens.

    Tokens of no row are NaN in both. ``pool_ok`` [rows, width] marks the table entries that may be read."""
    tokens, q_heads, dim = query.shape
    block, heads = cache.shape[2], cache.shape[3]
    group = q_heads // heads
    out = np.full((tokens, q_heads, dim), np.nan)
    lse = np.full((tokens, q_heads), np.nan)
    weights = []
    for r in range(len(table)):
        a, b = (r, r + 1) if query_start is None else (int(query_start[r]), int(query_start[r + 1]))
        n = int(min(max(lens[r], 0), table.shape[1] * block))
        ids = table[r].copy()
        seen = np.ones(n, dtype=bool)
        if pool_ok is not None:
            seen = np.repeat(pool_ok[r], block)[:n]
            ids[~pool_ok[r]] = 0
        k, v = gather(cache, ids, n, 0), gather(cache, ids, n, 1)
        received = np.zeros((heads, n))
        for i in range(b - a):
            limit = n - (b - a) + i + 1
            mask = seen & (np.arange(n) < limit)
            for h in range(q_heads):
                if not mask.any():
                    out[a + i, h], lse[a + i, h] = 0.0, -np.inf
                    continue
                x = k[mask, h // group] @ query[a + i, h].astype(np.float64) * scale
                top = x.max()
                e = np.exp(x - top)
                lse[a + i, h] = top + np.log(e.sum())
                out[a + i, h] = (e / e.sum()) @ v[mask, h // group]
                received[h // group, mask] += e / e.sum()
        weights.append(received)
    return out, lse, weights


def accumulate(scores, slots, lens, queries, weights, fresh=None, decay=1.0):
    """``scores`` [slots, heads, capacity] after ``weights`` (``attend``'s) have been added, in float64."""
    scores = scores.astype(np.float64)
    for r, w in enumerate(weights):
        if queries[r] == 0 or slots[r] < 0:
            continue
        n = w.shape[1]
        old = max(n - (int(fresh[r]) if fresh is not None else queries[r]), 0)
        row = scores[slots[r]]
        if decay != 0:
            row[:, :old] = decay * row[:, :old] + w[:, :old]
        else:
            row[:, :old] = w[:, :old]
        row[:, old:n] = w[:, old:]
    return scores


def select(scores, lens, keep, first, recent, slots):
    """kept [rows, heads, capacity] and new_lens [rows]."""
    heads, capacity = scores.shape[1:]
    kept = np.full((len(lens), heads, capacity), -1, dtype=np.int32)
    new = np.zeros(len(lens), dtype=np.int32)
    for r, n in enumerate(np.clip(lens, 0, capacity)):
        n, k = int(n), int(keep[r])
        whole = k < 0 or k >= n or slots[r] < 0 or slots[r] >= len(scores)
        new[r] = n if whole else max(k, min(n, first + recent))
        for h in range(heads):
            at = np.arange(n)
            if whole:
                kept[r, h, :n] = at
                continue
            pinned = (at < first) | (at >= n - recent)
            x = scores[slots[r], h, :n].astype(np.float64)
            x = np.where(np.isnan(x), -np.inf, x) + 0.0
            free = at[~pinned]
            best = free[np.argsort(-x[free], kind="stable")][: new[r] - pinned.sum()]
            kept[r, h, : new[r]] = np.sort(np.concatenate([at[pinned], best]))
    return kept, new


def compact(cache, scores, table, lens, kept, new_lens, slots):
    """The cache and the scores after every row's kept tokens moved to its front (copies)."""
    cache, scores = cache.copy(), None if scores is None else scores.copy()
    block = cache.shape[2]
    for r, (n, m) in enumerate(zip(lens, new_lens)):
        if not 0 <= m < n:
            continue
        to = np.arange(m)
        for h in range(cache.shape[3]):
            old = kept[r, h, :m]
            cache[table[r, to // block], :, to % block, h] = cache[table[r, old // block], :, old % block, h]
            if scores is not None and slots[r] >= 0:
                scores[slots[r], h, :m] = scores[slots[r], h, old]
    return cache, scores
