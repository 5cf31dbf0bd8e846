"""CPU test of the references by whole requests against those row by row."""
import numpy as np
import pytest

import cache_batches as B
import cache_ref as C


def batch(seed):
    g = np.random.default_rng(seed)
    page, nkv, nq, hd = 16, 2, 4, 8
    lens = [(20, 3), (0, 40), (50, 1), (7, 0), (33, 5)]
    own, prefixes = np.array([p + n for p, n in lens]), [37, 5]
    starts = np.concatenate([[0], np.cumsum([n for _, n in lens])])
    k, v = g.standard_normal((2, 12, nkv, page, hd))
    tables, prefix = g.integers(0, 12, (5, 4)), g.integers(0, 12, (2, 3))
    q = g.standard_normal((int(starts[-1]) + 3, nq, hd))
    return q, k, v, prefix, prefixes, [0, 2, 4], tables, starts, own


@pytest.mark.parametrize("kind,window,sinks", [(0, -1, 0), (1, 30, 3), (2, -1, 0)])
def test_attention(kind, window, sinks):
    c = batch(1)
    out, lse = np.full(c[0].shape, 7.0), np.full(c[0].shape[:2], 7.0)
    a, b = (f(*c, out, lse, 0.4, kind, window, sinks) for f in (B.shared_attention, C.shared_attention))
    for x, y in zip((*a[:2], *a[2]), (*b[:2], *b[2])):
        np.testing.assert_allclose(x, y, 1e-12, 1e-12)


@pytest.mark.parametrize("kind,last_rows", [(0, 0), (2, 0), (0, 2), (2, 4)])
def test_weights(kind, last_rows):
    q, k, v, _, _, _, tables, starts, own = batch(2)
    old = np.random.default_rng(3).random((5, 2, 64)).astype(np.float32)
    _, logs, _ = C.shared_attention(q, k, v, [], [], [0], tables, starts, own, np.zeros(q.shape), np.zeros(q.shape[:2]), 0.4, kind)
    logs = logs.astype(np.float32)
    ref = C.weights(q, k, tables, starts, own, logs, old, 0.4, kind, last_rows)
    for lse in (None, logs):
        got = B.weights(q, k, tables, starts, own, lse, old, 0.4, kind, last_rows)
        counts = ~np.isnan(got[2])
        assert lse is not None or counts.sum() == sum(min(n, last_rows or n) for n in np.diff(starts)) * 4
        np.testing.assert_array_equal(got[2][counts], logs[counts])
        for x, y in zip(got, ref):
            np.testing.assert_allclose(x, y, 1e-9, 1e-12)
