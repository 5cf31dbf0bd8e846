"""cache_ref's attention and weights by whole requests, for batches that its rows would take minutes for."""
import numpy as np

import cache_ref as C


def scores(q, k, scale):
    """(s, sum of magnitudes) of rows q [n, Hd] and keys k [m, Hd]."""
    return q @ k.T * scale, np.abs(q) @ np.abs(k).T * abs(scale)


def shared_attention(q, k_cache, v_cache, prefix_tables, prefix_lens, group_starts, tables, starts, key_lens, out, lse, scale, kind=0,
                     window=-1, sinks=0):
    """C.shared_attention for lengths in order, finite values and rows that see a key."""
    T, Nq, _ = q.shape
    nkv = k_cache.shape[1]
    out, lse = out.astype(np.float64).copy(), lse.astype(np.float64).copy()
    mag, spread, count = np.zeros_like(out), np.zeros((T, Nq, 1)), np.ones((T, Nq, 1))
    held = {}
    for r in range(len(tables)):
        a, n, length, g = starts[r], starts[r + 1] - starts[r], key_lens[r], C.group_of(r, group_starts)
        if n == 0:
            continue
        first = 0 if g is None else prefix_lens[g]
        if g is not None and g not in held:
            held = {g: [C.rows_of(c, prefix_tables[g], first)[0] for c in (k_cache, v_cache)]}
        own = [C.rows_of(c, tables[r], length)[0] for c in (k_cache, v_cache)]
        k, v = own if g is None else (np.concatenate(x, 1) for x in zip(held[g], own))
        at, o = np.arange(first + length), (length - n + np.arange(n))[:, None]
        see = np.full((n, first + length), kind == 2) | (at < first) | (at - first <= o)
        if kind == 1:
            see &= (first + np.maximum(o, 0) - at < window) | (at < sinks)
        rows = slice(a, a + n)
        for h in range(Nq):
            kv = h // (Nq // nkv)
            s, size = scores(q[rows, h].astype(np.float64), k[kv], scale)
            s = np.where(see, s, -np.inf)
            top = s.max(1, keepdims=True)
            w = np.exp(s - top)
            total = w.sum(1, keepdims=True)
            lse[rows, h] = (top + np.log(total))[:, 0]
            w /= total
            out[rows, h], mag[rows, h] = w @ v[kv], w @ np.abs(v[kv])
            spread[rows, h, 0] = np.where(see, size, 0.0).max(1)
            count[rows, h, 0] = see.sum(1)
    return out, lse, (mag, spread, count)


def weights(q, k_cache, tables, starts, key_lens, lse, old, scale, kind=0, last_rows=0):
    """C.weights for lengths in order and tables of pages that the cache holds; with lse None the requests' own logarithms, rounded to f32, NaN for the
    rows that do not count.
    (weights, bound, the logarithms)"""
    T, Nq, hd = q.shape
    nkv, page, u = k_cache.shape[1], k_cache.shape[2], 2.0 ** -24
    new, bound = old.astype(np.float64).copy(), np.zeros(old.shape)
    logs = np.full((T, Nq), np.nan, np.float32) if lse is None else lse
    for r in range(len(tables)):
        b, n, length = starts[r + 1], starts[r + 1] - starts[r], key_lens[r]
        pages, at = np.unique(tables[r, :-(-length // page)], return_inverse=True)  # (each page's scores once, however often a table names it)
        of = (at.reshape(-1)[:, None] * page + np.arange(page)).reshape(-1)[:length]
        k = k_cache[pages].transpose(1, 0, 2, 3).reshape(nkv, -1, hd).astype(np.float64)
        rows = min(n, last_rows or n)
        see = (np.arange(length) <= (length - rows + np.arange(rows))[:, None]) | (kind == 2)
        for h in range(Nq):
            kv = h // (Nq // nkv)
            s, spread = (x[:, of] for x in scores(q[b - rows:b, h].astype(np.float64), k[kv], scale))
            s[~see] = -np.inf
            top = s.max(1, keepdims=True)
            w = np.exp(s - top)
            if lse is None:
                logs[b - rows:b, h] = (top + np.log(w.sum(1, keepdims=True)))[:, 0]
            mine = logs[b - rows:b, h, None].astype(np.float64)
            w *= np.exp(top - mine)
            new[r, kv, :length] += w.sum(0)
            bound[r, kv, :length] += (hd + 6) * u * np.einsum("ik,ik->k", w, spread)
            bound[r, kv, :length] += ((3 * u * np.abs(mine) + 2.0 ** -22 + (n * Nq // nkv + 4) * u).T @ w)[0]
    return new, bound + 2 * u * np.abs(old), logs
