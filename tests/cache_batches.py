"""cache_ref's attention and weights by whole requests, for batches that its rows would take minutes for."""
import numpy as np

import cache_ref as C


def scores(q, k, scale):
    """(s, sum of magnitudes) of rows q [n, Hd] and keys k [m, Hd]."""
    return q @ k.T * scale, np.abs(q) @ np.abs(k).T * abs(scale)


def part(q, k, v, see, scale):
    """Of rows q and keys k: the highest score, the sum of exponentials from it, those times v and times |v|, the largest magnitude and
    how many keys are seen (0 and no score where none is)."""
    s, size = scores(q, k, scale)
    s[~see], size[~see] = -np.inf, 0.0
    top = s.max(1, keepdims=True, initial=-np.inf)
    s -= np.where(np.isneginf(top), 0.0, top)
    w = np.exp(s, out=s)
    return top, w.sum(1, keepdims=True), w @ v, w @ np.abs(v), size.max(1, keepdims=True, initial=0.0), see.sum(1, keepdims=True)


def shared_attention(q, k_cache, v_cache, prefix_tables, prefix_lens, group_starts, tables, starts, key_lens, out, lse, scale, kind=0,
                     window=-1, sinks=0):
    """C.shared_attention for lengths in order, finite values and rows that see a key."""
    T, Nq, hd = q.shape
    nkv, G = k_cache.shape[1], Nq // k_cache.shape[1]
    out, lse = out.astype(np.float64).copy(), lse.astype(np.float64).copy()
    mag, spread, count = np.zeros_like(out), np.zeros((T, Nq, 1)), np.ones((T, Nq, 1))
    inside = [C.group_of(r, group_starts) for r in range(len(tables))]
    groups = [(g, [r for r, x in enumerate(inside) if x == g]) for g in range(len(prefix_lens))]
    groups += [(None, [r]) for r, x in enumerate(inside) if x is None]
    for g, rs in groups:
        if not rs:
            continue
        a, b = starts[rs[0]], starts[rs[-1] + 1]
        first = 0 if g is None else prefix_lens[g]
        pk, pv = (C.rows_of(c, [] if g is None else prefix_tables[g], first)[0] for c in (k_cache, v_cache))
        own = [[C.rows_of(c, tables[r], key_lens[r])[0] for c in (k_cache, v_cache)] for r in rs]
        o = np.concatenate([key_lens[r] - (starts[r + 1] - starts[r]) + np.arange(starts[r + 1] - starts[r]) for r in rs])[:, None]

        def sees(o, at, behind):  # keys `at` of the whole sequence, `behind` the prefix or in it
            see = np.full((len(o), len(at)), kind == 2) | ((at - first <= o) if behind else True)
            return see & ((first + np.maximum(o, 0) - at < window) | (at < sinks)) if kind == 1 else see

        for kv in range(nkv):
            rows = q[a:b, kv * G:(kv + 1) * G].astype(np.float64).reshape(-1, hd)
            parts = [part(rows, pk[kv], pv[kv], np.repeat(sees(o, np.arange(first), False), G, 0), scale)]
            mine = []
            for r, (k, v) in zip(rs, own):
                x, y = starts[r] - a, starts[r + 1] - a
                mine.append(part(rows[x * G:y * G], k[kv], v[kv], np.repeat(sees(o[x:y], first + np.arange(key_lens[r]), True), G, 0), scale))
            parts.append([np.concatenate(x) for x in zip(*mine)])
            top = np.maximum(parts[0][0], parts[1][0])
            total, up, size = (sum(x[i] * np.exp(x[0] - top) for x in parts) for i in (1, 2, 3))
            heads = lambda x: x.reshape(b - a, G, -1)  # noqa: E731
            at = (slice(a, b), slice(kv * G, (kv + 1) * G))
            lse[at] = heads(top + np.log(total))[..., 0]
            out[at], mag[at] = heads(up / total), heads(size / total)
            spread[at], count[at] = heads(np.maximum(parts[0][4], parts[1][4])), heads(parts[0][5] + parts[1][5])
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
