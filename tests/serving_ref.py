"""64-bit references of the operators over a paged cache and of the token draw,
written from their definitions, and the bounds on what a kernel may be off."""
import numpy as np

HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # of a rounding, relative to the value
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}  # of a rounding to a subnormal


def page_tables(past, new, free, tables, page_size, tokens):
    """The outputs of Kernels.PageTables, token by token."""
    tables = tables.astype(np.int64).copy()
    R, M = tables.shape
    past, new = (np.maximum(np.asarray(x, np.int64), 0) for x in (past, new))
    starts, keys = [0], []
    positions, slots = np.zeros(tokens, np.int64), np.full(tokens, -1, np.int64)
    used = t = 0
    for r in range(R):
        held = -(-past[r] // page_size)
        for i in range(new[r]):
            if t + i >= tokens:
                break
            pos = past[r] + i
            col, row = divmod(pos, page_size)
            page = -1
            if col < M:
                if col < held:
                    page = tables[r, col]
                else:
                    k = used + col - held
                    page = max(free[k], -1) if k < len(free) else -1
                    if row == 0:
                        tables[r, col] = page
            positions[t + i] = min(pos, 2 ** 31 - 1)
            slot = page * page_size + row
            slots[t + i] = slot if page >= 0 and slot < 2 ** 31 else -1
        used += -(-(past[r] + new[r]) // page_size) - held
        t += new[r]
        starts.append(min(t, tokens))
        keys.append(min(past[r] + new[r], 2 ** 31 - 1))
    return tables, np.array(starts), np.array(keys, np.int64), positions, slots, np.array([t, used])


def visible(pos, keys, kind, window, sinks):
    j = np.arange(keys)
    if kind == 2:
        return np.ones(keys, bool)
    see = j <= pos
    return see if kind == 0 else see & ((pos - j < window) | (j < sinks))


def attention(q, k_cache, v_cache, tables, starts, key_lens, out, scale, kind=0, window=-1, sinks=0):
    """(out, bound / error unit): out in 64 bits with the rows of no request as they were, and for each element
    sum of weights times |V| and the largest sum of |q k| of the row, for `bound`."""
    T, Nq, Hd = q.shape
    P, Nkv, page, _ = k_cache.shape
    out = out.astype(np.float64).copy()
    mag, spread, count = np.zeros_like(out), np.zeros((T, Nq, 1)), np.ones((T, Nq, 1))
    for r in range(tables.shape[0]):
        a, b = min(max(starts[r], 0), T), min(max(starts[r + 1], 0), T)
        n = max(b - a, 0)
        length = max(key_lens[r], 0)
        keys = min(length, tables.shape[1] * page)
        pages = tables[r, :-(-keys // page)]
        ok = np.repeat((pages >= 0) & (pages < P), page)[:keys]
        safe = np.where((pages >= 0) & (pages < P), pages, 0)
        k = k_cache[safe].transpose(1, 0, 2, 3).reshape(Nkv, -1, Hd)[:, :keys].astype(np.float64)
        v = v_cache[safe].transpose(1, 0, 2, 3).reshape(Nkv, -1, Hd)[:, :keys].astype(np.float64)
        for i in range(n):
            see = visible(length - n + i, keys, kind, window, sinks) & ok
            for h in range(Nq):
                row, kv = a + i, h // (Nq // Nkv)
                if not see.any():
                    out[row, h] = 0.0
                    continue
                ks, vs, qr = k[kv][see], v[kv][see], q[row, h].astype(np.float64)
                s = ks @ qr * scale
                with np.errstate(invalid="ignore"):
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    out[row, h] = w @ vs
                    mag[row, h] = w @ np.abs(vs)
                spread[row, h] = (np.abs(ks) @ np.abs(qr)).max() * abs(scale)
                count[row, h] = see.sum()
    return out, (mag, spread, count)


def attention_bound(out, parts, dtype, hd):
    """A score is a sum of hd products of f32 (or of 16-bit values, exact in f32): off by at most hd 2^-24 times the
    sum of their magnitudes, and its product with scale and log2(e) adds 3 roundings; a weight's relative error is
    that of its exponent plus 2^-22 of the exp2, and the ratio of weights to their sum doubles it. The weights enter
    the product with V with at least 11 bits (one f16) or 16 (two bf16), and up to `count` additions, rescalings
    and merges round once each. Then the result is rounded to the dtype."""
    mag, spread, count = parts
    weight = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -16}[dtype]
    eps = 2.0 * ((hd + 3) * 2.0 ** -24 * spread + 2.0 ** -22) + weight + (count + 8) * 2.0 ** -24
    # a few terms' errors line up, all of them do not: the bound holds as it stands, without a factor
    return HALF[dtype] * np.abs(out) + TINY[dtype] + mag * eps * (1.0 + HALF[dtype])


ONE = 2 ** 40


def sample(logits, uniforms, temperature=None, top_k=None, top_p=None, min_p=None):
    """Kernels.Sample, in whole numbers of any size."""
    out = []
    for r in range(logits.shape[0]):
        x = logits[r].astype(np.float64)
        fine = x > -np.inf
        if not fine.any():
            out.append(-1)
            continue
        top = x[fine].max()
        t = 1.0 if temperature is None else float(np.float32(temperature[r]))
        k = 0 if top_k is None else int(top_k[r])
        if not t > 0:
            t, k = 1.0, 1
        with np.errstate(all="ignore"):
            d = np.where(x == top, 0.0, (x - top) / t)
            w = np.where(fine & (d > -40.0), np.rint(np.exp(np.minimum(d, 0.0)) * ONE), 0.0)
        w = [int(v) for v in w]
        order = sorted(range(x.size), key=lambda i: (-x[i] if x[i] == x[i] else np.inf, x[i] != x[i], i))
        if k > 0:
            order = order[:k]
        if top_p is not None and np.float32(top_p[r]) < 1:
            share = int(max(float(np.float32(top_p[r])), 0.0) * 2 ** 31)
            z, run, kept = sum(w[i] for i in order), 0, []
            for i in order:
                if kept and not run * 2 ** 31 < share * z:
                    break
                kept.append(i)
                run += w[i]
            order = kept
        if min_p is not None and np.float32(min_p[r]) > 0:
            order = [i for i in order if w[i] >= min(float(np.float32(min_p[r])), 1.0) * ONE]
        u = float(np.float32(uniforms[r]))
        u31 = min(int(min(u, 1.0) * 2 ** 31), 2 ** 31 - 1) if u > 0 else 0
        z = sum(w[i] for i in order)
        target, run = u31 * z >> 31, 0
        for i in sorted(order):
            run += w[i]
            if run > target:
                out.append(i)
                break
    return np.array(out)
