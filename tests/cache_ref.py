"""64-bit references of shared-prefix attention, attention weights, eviction and page release, written from their
definitions, and the bounds on what a kernel may be off."""
import numpy as np

from serving_ref import HALF, attention_bound  # noqa: F401 (the bound of `out` is attention's)


def rows_of(cache, table, keys):
    """(keys [Nkv, n, Hd] of a table's row, which of them a page holds)"""
    pages = np.asarray(table, np.int64)[:-(-keys // cache.shape[2])]
    ok = (pages >= 0) & (pages < cache.shape[0])
    x = cache[np.where(ok, pages, 0)].transpose(1, 0, 2, 3).reshape(cache.shape[1], -1, cache.shape[3])[:, :keys]
    return x.astype(np.float64), np.repeat(ok, cache.shape[2])[:keys]


def group_of(r, group_starts):
    return next((g for g in range(len(group_starts) - 1) if group_starts[g] <= r < group_starts[g + 1]), None)


def shared_attention(q, k_cache, v_cache, prefix_tables, prefix_lens, group_starts, tables, starts, key_lens, out, lse, scale, kind=0,
                     window=-1, sinks=0):
    """(out, lse, parts for the bounds), rows of no request as they were."""
    T, Nq, _ = q.shape
    page, nkv = k_cache.shape[2], k_cache.shape[1]
    out, lse = out.astype(np.float64).copy(), lse.astype(np.float64).copy()
    mag, spread, count = np.zeros_like(out), np.zeros((T, Nq, 1)), np.ones((T, Nq, 1))
    for r in range(len(tables)):
        a, b = min(max(starts[r], 0), T), min(max(starts[r + 1], 0), T)
        n, length, g = max(b - a, 0), max(key_lens[r], 0), group_of(r, group_starts)
        first = min(max(prefix_lens[g], 0), len(prefix_tables[g]) * page) if g is not None else 0
        keys = min(length, tables.shape[1] * page)
        both = [[rows_of(c, t, m) for t, m in (([], 0) if g is None else (prefix_tables[g], first), (tables[r], keys))] for c in (k_cache, v_cache)]
        k, v = (np.concatenate([x[0] for x in y], 1) for y in both)
        ok = np.concatenate([x[1] for x in both[0]])
        at = np.arange(first + keys)
        for i in range(n):
            o = length - n + i
            see = ok.copy()
            if kind != 2:
                see &= (at < first) | (at - first <= o)
            if kind == 1:
                see &= (first + max(o, 0) - at < window) | (at < sinks)
            for h in range(Nq):
                kv = h // (Nq // nkv)
                if not see.any():
                    out[a + i, h], lse[a + i, h] = 0.0, -np.inf
                    continue
                ks, vs, qr = k[kv][see], v[kv][see], q[a + i, h].astype(np.float64)
                s = ks @ qr * scale
                with np.errstate(invalid="ignore"):
                    w = np.exp(s - s.max())
                    lse[a + i, h] = s.max() + np.log(w.sum())
                    w /= w.sum()
                    out[a + i, h] = w @ vs
                    mag[a + i, h] = w @ np.abs(vs)
                spread[a + i, h] = (np.abs(ks) @ np.abs(qr)).max() * abs(scale)
                count[a + i, h] = see.sum()
    return out, lse, (mag, spread, count)


def lse_bound(lse, parts, hd):
    """The scores' errors as attention_bound has them, 2^-22 of each exponential and the sum's `count` roundings (all relative to the
    sum, so absolute in its logarithm), and in units of 2^-24 four roundings of numbers no larger than the
    score, the logarithm in base 2 and its parts (the reference that a maximum is kept by may be 16 away from it)."""
    _, spread, count = (x[..., 0] for x in parts)
    u = 2.0 ** -24
    with np.errstate(invalid="ignore"):
        return (hd + 3) * u * spread + 2.0 ** -22 + (count + 8) * u + 4 * u * 1.5 * (np.abs(lse) + np.log(count) + spread + 16)


def weights(q, k_cache, tables, starts, key_lens, lse, old, scale, kind=0, last_rows=0):
    """(weights, bound)"""
    T, Nq, hd = q.shape
    page, nkv = k_cache.shape[2], k_cache.shape[1]
    new, bound, u = old.astype(np.float64).copy(), np.zeros(old.shape), 2.0 ** -24
    for r in range(len(tables)):
        a, b = min(max(starts[r], 0), T), min(max(starts[r + 1], 0), T)
        n, length = max(b - a, 0), max(key_lens[r], 0)
        keys = min(length, tables.shape[1] * page)
        k, ok = rows_of(k_cache, tables[r], keys)
        for i in range(max(n - last_rows, 0) if last_rows else 0, n):
            see = ok & ((np.arange(keys) <= length - n + i) | (kind == 2))
            for h in range(Nq):
                kv, of = h // (Nq // nkv), float(lse[a + i, h])
                if of == -np.inf or not see.any():
                    continue
                ks, qr = k[kv][see], q[a + i, h].astype(np.float64)
                with np.errstate(invalid="ignore"):
                    s = ks @ qr * scale
                    w = np.exp(s - of)
                    spread = np.abs(ks) @ np.abs(qr) * abs(scale)
                    at = np.flatnonzero(see)
                    new[r, kv, at] += w
                    # a score's error as attention's, with 3 more roundings in its exponent; lse in base 2 has two; 2^-22 of exp2;
                    # then no more additions than rows
                    bound[r, kv, at] += w * ((hd + 6) * u * spread + 3 * u * abs(of) + 2.0 ** -22 + (n * Nq // nkv + 4) * u)
    return new, bound + 2 * u * np.abs(old)


def evict(weights, k_cache, v_cache, tables, key_lens, budgets, kept, first, last):
    """(kept, kept_weights, k_cache, v_cache, new lengths)"""
    R, nkv, room = weights.shape
    P, _, page, _ = k_cache.shape
    kept, kept_w = kept.copy(), np.zeros_like(weights)
    caches = [c.copy() for c in (k_cache, v_cache)]
    lens = []
    for r in range(R):
        keys = min(max(int(key_lens[r]), 0), room)
        n = min(keys, max(int(budgets[r]), 0))
        f = min(first, n)
        e = min(last, n - f)
        lens.append(n)
        for h in range(nkv):
            w = weights[r, h]
            middle = sorted(range(f, keys - e), key=lambda i: (w[i] != w[i], -w[i] if w[i] == w[i] else 0.0, i))
            mine = sorted(list(range(f)) + middle[:n - f - e] + list(range(keys - e, keys)))
            kept[r, h, :n] = mine
            kept_w[r, h, :n] = w[mine]
            for new, old in zip(caches, (k_cache, v_cache)):
                for j, i in enumerate(mine):
                    a, b = tables[r, i // page], tables[r, j // page]
                    if 0 <= a < P and 0 <= b < P and i != j:
                        new[b, h, j % page] = old[a, h, i % page]
    return kept, kept_w, caches[0], caches[1], np.array(lens)


def release(key_lens, budgets, tables, page, freed):
    """(new lengths, freed, number of pages)"""
    freed, at, lens = freed.copy(), 0, []
    for r in range(len(tables)):
        keys = min(max(int(key_lens[r]), 0), tables.shape[1] * page)
        n = min(keys, max(int(budgets[r]), 0))
        lens.append(n)
        for c in range(-(-n // page), -(-keys // page)):
            freed[at] = tables[r, c]
            at += 1
    return np.array(lens, np.int64), freed, at
