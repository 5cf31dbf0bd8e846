"""GPU tests of the paged cache: tables, writes and attention against 64-bit
references (serving_ref), at the lengths, masks and pages where they can go wrong."""
import numpy as np
import pytest

import serving_ref as R
from gpu_util import download, gpu_env, rounded, upload

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    return gpu_env()


def i32(pa, x):
    return pa.Tensor.from_numpy(np.asarray(x, np.int32), "i32")


# ---- page tables -------------------------------------------------------------------


def run_tables(env, past, new, free, table, page, tokens):
    pa, _, stream, enc = env
    n = len(past)
    out = [i32(pa, np.full(s, -77)) for s in (n + 1, n, tokens, tokens, 2)]
    tt = i32(pa, table)
    enc.encode(pa.Kernels.PageTables(i32(pa, past), i32(pa, new), i32(pa, free), tt, page_size=page, query_starts=out[0],
                                     key_lens=out[1], positions=out[2], slots=out[3], counts=out[4]))
    stream.synchronize()
    got = [tt.numpy(stream)] + [t.numpy(stream) for t in out]
    for a, b in zip(got, R.page_tables(past, new, free, np.asarray(table), page, tokens)):
        np.testing.assert_array_equal(a, b)
    return got


@pytest.mark.parametrize("requests,page,seed", [(1, 16, 0), (3, 16, 1), (255, 48, 2), (257, 16, 3), (1023, 1, 4), (1024, 64, 5),
                                                (1025, 16, 6), (2500, 7, 7)])
def test_page_tables(env, requests, page, seed):
    g = np.random.default_rng(seed)
    past = g.integers(0, 5 * page, requests) * g.integers(0, 2, requests)
    new = g.choice([0, 1, 1, 2, page - 1, page, page + 1, 3 * page], requests)
    held = -(-past // page)
    columns = int((-(-(past + new) // page)).max()) + 1
    ids = g.permutation(int(held.sum() + (past + new).sum()) + 5)
    table = np.full((requests, columns), -1)
    at = 0
    for r in range(requests):
        table[r, :held[r]] = ids[at:at + held[r]]
        at += held[r]
    run_tables(env, past, new, ids[at:], table, page, int(new.sum()) + int(g.integers(0, 40)))


def test_page_tables_one_long_prompt(env):
    run_tables(env, [33], [20000], np.arange(2000)[::-1], np.full((1, 1300), 5), 16, 20000)


def test_page_tables_runs_out(env):
    # pages, columns and room for tokens each run out; lengths below zero and at the type's end
    table = np.arange(6 * 3).reshape(6, 3)
    run_tables(env, [5, 0, 30, 16, 0, 40], [10, 40, 60, 0, 3, 1], [100, -4, 102], table, 16, 200)
    run_tables(env, [5, 0, 30, 16, 0, 40], [10, 40, 60, 0, 3, 1], [], table, 16, 200)
    run_tables(env, [5, 0, 30, 16, 0, 40], [10, 40, 60, 0, 3, 1], np.arange(50), table, 16, 47)
    run_tables(env, [-3, 2 ** 31 - 1, 7], [2, 5, -8], np.arange(50), np.full((3, 2), 2 ** 31 - 1), 16, 12)
    run_tables(env, [4], [3], np.arange(5), np.zeros((1, 0)), 16, 3)
    run_tables(env, [4, 5], [0, 0], np.arange(5), np.zeros((2, 3)), 16, 0)
    run_tables(env, [], [], np.arange(5), np.zeros((0, 3)), 16, 4)


def test_page_tables_sums_past_32_bits(env):
    pa, _, stream, enc = env
    out = [i32(pa, np.zeros(n)) for n in (4, 3, 8, 8, 2)]
    big = 2 ** 31 - 1
    enc.encode(pa.Kernels.PageTables(i32(pa, [0, 0, 9]), i32(pa, [5, big, big]), i32(pa, [3, 4]), i32(pa, np.zeros((3, 2))), page_size=16,
                                     query_starts=out[0], key_lens=out[1], positions=out[2], slots=out[3], counts=out[4]))
    stream.synchronize()
    starts, keys, positions, slots, counts = (t.numpy(stream) for t in out)
    assert list(starts) == [0, 5, 8, 8] and list(keys) == [5, big, big]
    assert list(positions) == [0, 1, 2, 3, 4, 0, 1, 2] and list(slots) == [48, 49, 50, 51, 52, 64, 65, 66]
    assert list(counts) == [big, min(big, 1 + 2 * (2 ** 27) + 0)]


# ---- cache write -------------------------------------------------------------------


@pytest.mark.parametrize("src,dst", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "bf16")])
@pytest.mark.parametrize("tokens,nkv,hd,page,offset", [(1, 1, 8, 1, 0), (5, 2, 64, 16, 0), (70, 3, 80, 48, 0), (9, 2, 13, 16, 0),
                                                       (33, 4, 256, 32, 0), (6, 2, 64, 16, 1)])
def test_paged_write(env, src, dst, tokens, nkv, hd, page, offset):
    pa, _, stream, enc = env
    g = np.random.default_rng(tokens)
    pages = -(-tokens // page) + 3
    rows = [rounded(g.standard_normal((tokens, nkv, hd)), src) for _ in range(2)]
    old = [rounded(g.standard_normal((pages, nkv, page, hd)), dst) for _ in range(2)]
    slots = g.permutation(pages * page)[:tokens].astype(np.int64)
    bad = [-1, -2 ** 31, pages * page, 2 ** 31 - 1]
    for i, b in zip(range(0, tokens, 4), bad):
        if tokens > 4:
            slots[i] = b
    size = {"f32": 4, "f16": 2, "bf16": 2}

    def shifted(x, dtype):  # data `offset` elements behind an aligned address
        flat = np.concatenate([np.zeros(offset), x.ravel()])
        t = upload(pa, flat, dtype)
        return pa.Tensor(t.ptr + offset * size[dtype], x.shape, dtype, owner=t)

    k, v = (shifted(x, src) for x in rows)
    kc, vc = (shifted(x, dst) for x in old)
    enc.encode(pa.Kernels.PagedKVCacheWrite(k, v, i32(pa, slots), kc, vc))
    stream.synchronize()
    for x, cache, was in ((rows[0], kc, old[0]), (rows[1], vc, old[1])):
        want = was.copy()
        for t in range(tokens):
            if 0 <= slots[t] < pages * page:
                want[slots[t] // page, :, slots[t] % page] = rounded(x[t], dst)
        np.testing.assert_array_equal(download(cache, stream), want)


# ---- attention ---------------------------------------------------------------------


class Batch:
    """A cache with the pages of requests of given (past, new) lengths in any order; what no request holds is NaN."""

    def __init__(self, lens, nq, nkv, hd, dtype, page, seed, pad=0, spare=1, fill=np.nan):
        g = np.random.default_rng(seed)
        self.lens, self.dtype, self.hd = lens, dtype, hd
        held = [-(-(p + n) // page) for p, n in lens]
        pages = sum(held) + 2
        ids = g.permutation(pages)
        self.table = np.full((len(lens), max(held + [0]) + spare), -1, np.int64)
        self.k, self.v = (rounded(g.standard_normal((pages, nkv, page, hd)), dtype) for _ in range(2))
        live = np.zeros((pages, page), bool)
        at = 0
        for r, ((p, n), h) in enumerate(zip(lens, held)):
            self.table[r, :h] = ids[at:at + h]
            for j in range(p + n):
                live[ids[at + j // page], j % page] = True
            at += h
        self.live = live
        self.fill(fill)
        self.starts = np.concatenate([[0], np.cumsum([n for _, n in lens])]).astype(np.int64)
        self.keys = np.array([p + n for p, n in lens], np.int64)
        tokens = int(self.starts[-1]) + pad
        self.q = rounded(g.standard_normal((tokens, nq, hd)), dtype)
        self.old = rounded(g.standard_normal((tokens, nq, hd)), dtype)
        self.scale = float(np.float32(hd ** -0.5))

    def fill(self, value):
        for x in (self.k, self.v):
            np.copyto(x, value, where=~self.live[:, None, :, None])

    def run(self, env, mask=(0, -1), sinks=0, hint=None, enc=None):
        pa, _, stream, own = env
        t = [upload(pa, x, self.dtype) for x in (self.q, self.k, self.v)]
        out = upload(pa, self.old, self.dtype)
        hint = max([n for _, n in self.lens] + [0]) if hint is None else hint
        (enc or own).encode(pa.Kernels.PagedAttention(*t, i32(pa, self.table), i32(pa, self.starts), i32(pa, self.keys), out,
                                                      scale=self.scale, mask=pa.AttentionMask(*mask), sinks=sinks, max_query_len=hint))
        stream.synchronize()
        return download(out, stream)

    def check(self, env, mask=(0, -1), sinks=0, hint=None):
        got = self.run(env, mask, sinks, hint)
        want, parts = R.attention(self.q, self.k, self.v, self.table, self.starts, self.keys, self.old, self.scale, mask[0], mask[1], sinks)
        assert np.isfinite(want).all()
        off = np.abs(got - want)
        bound = R.attention_bound(want, parts, self.dtype, self.hd)
        bad = ~(off <= bound)
        assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], want[bad][:4], bound[bad][:4])
        return got


LENS = {
    "decode": [(0, 1), (1, 1), (15, 1), (16, 1), (31, 1), (32, 1), (200, 1), (1000, 1)],
    "one": [(700, 1)],
    "few": [(0, 2), (5, 5), (64, 3), (333, 8), (31, 17), (0, 1)],
    "chunk": [(0, 150), (77, 130), (300, 64)],
    "mixed": [(40, 1), (0, 0), (0, 90), (513, 1), (9, 200), (0, 0), (127, 3)],
}
HEADS = [(4, 4, 64), (8, 2, 128), (8, 4, 256), (6, 2, 80), (8, 2, 512), (20, 1, 128), (3, 1, 24), (2, 1, 36)]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("lens", list(LENS))
@pytest.mark.parametrize("heads", HEADS, ids=str)
def test_attention(env, dtype, lens, heads):
    page = {64: 16, 128: 48, 256: 32, 80: 16, 512: 64, 24: 256, 36: 16}[heads[2]]
    Batch(LENS[lens], *heads, dtype, page, seed=heads[2] + len(lens), pad=3).check(env)


@pytest.mark.parametrize("dtype,heads", [("bf16", (8, 4, 256)), ("f16", (8, 2, 128)), ("f32", (4, 2, 64)), ("bf16", (4, 1, 512)),
                                         ("f16", (6, 2, 80))])
@pytest.mark.parametrize("mask,sinks", [((2, -1), 0), ((1, 1), 0), ((1, 16), 0), ((1, 33), 1), ((1, 100), 4), ((1, 70), 64),
                                        ((1, 50), 2000), ((1, 5000), 3)])
@pytest.mark.parametrize("lens", ["decode", "mixed"])
def test_attention_masks(env, dtype, heads, mask, sinks, lens):
    Batch(LENS[lens], *heads, dtype, 16, seed=7 + sinks, pad=1).check(env, mask, sinks)


@pytest.mark.parametrize("hint", [0, 1, 2, 5, 1000])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_attention_hint_changes_nothing(env, hint, dtype):
    Batch(LENS["mixed"], 8, 2, 128, dtype, 16, seed=3).check(env, hint=hint)
    Batch(LENS["decode"], 8, 4, 256, dtype, 16, seed=4).check(env, (1, 64), 2, hint=hint)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("lens", ["decode", "mixed"])
def test_attention_rows_without_keys(env, dtype, lens):
    # a window of nothing; with sinks the sinks alone
    b = Batch(LENS[lens], 8, 2, 128, dtype, 16, seed=5, pad=2)
    got = b.check(env, (1, 0))
    assert not got[:b.starts[-1]].any()
    b.check(env, (1, 0), 3)
    b.check(env, (1, -9), 40)
    # fewer keys than new tokens: the first tokens see nothing
    b.keys[:] = [max(n - 2, 0) for _, n in b.lens]
    b.live[:] = True
    b.fill(0)
    b.check(env)


@pytest.mark.parametrize("dtype,heads", [("bf16", (8, 4, 256)), ("f16", (8, 2, 128)), ("f32", (4, 2, 64))])
@pytest.mark.parametrize("lens", ["decode", "mixed", "few"])
def test_attention_bad_tables(env, dtype, heads, lens):
    # entries that name no page are left out, wherever they are; more keys than the table has columns
    b = Batch(LENS[lens], *heads, dtype, 16, seed=6)
    g = np.random.default_rng(1)
    b.table[g.random(b.table.shape) < 0.3] = -1
    b.table[g.random(b.table.shape) < 0.1] = 2 ** 31 - 1
    b.table[-1] = -2 ** 31
    b.table[0, 0] = len(b.k)
    b.check(env)
    b.check(env, (2, -1))
    b.check(env, (1, 40), 20)
    b.live[:] = True
    b.fill(0)
    b.k[np.isnan(b.k)] = 0
    b.v[np.isnan(b.v)] = 0
    b.keys[1:] += 3000
    b.check(env)
    b.check(env, (2, -1))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_attention_bad_starts(env, dtype):
    # ranges past the rows, and below them: what is in range is computed, the other rows stay
    b = Batch([(20, 4), (3, 5), (50, 6)], 8, 2, 128, dtype, 16, seed=8, pad=4, fill=0)
    for starts in ([-7, 4, 9, 40], [2, 2, 9, 15], [0, 4, 4, 4], [30, 40, 50, 60], [-9, -8, -7, -6]):
        b.starts = np.array(starts)
        b.check(env)


@pytest.mark.parametrize("dtype,heads", [("bf16", (8, 4, 256)), ("f16", (8, 2, 128)), ("f32", (4, 2, 64)), ("bf16", (8, 2, 512))])
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("lens", ["decode", "mixed"])
def test_attention_unseen_infinities(env, dtype, heads, value, lens):
    # infinities and NaN in keys and values that a row does not see, of the same chunk and outside the window
    b = Batch(LENS[lens], *heads, dtype, 16, seed=9)
    mask, sinks = (1, 30), 4
    want, parts = R.attention(b.q, b.k, b.v, b.table, b.starts, b.keys, b.old, b.scale, *mask, sinks)
    touched = np.zeros(len(b.q), bool)
    for r, (past, n) in enumerate(b.lens):
        for key in {past + n - 1, past + n // 2, 10, 4} & set(range(past + n)):
            page, row = b.table[r, key // 16], key % 16
            b.v[page, :, row, 3::7] = value
            b.k[page, :, row, ::5] = value
            for i in range(n):
                if R.visible(past + i, past + n, *mask, sinks)[key]:
                    touched[b.starts[r] + i] = True
    got = b.run(env, mask, sinks)
    clean = ~touched
    assert clean[:b.starts[-1]].any() or lens == "decode"
    off = np.abs(got - want)
    assert (off <= R.attention_bound(want, parts, dtype, b.hd))[clean].all()
    if value != value:
        assert np.isnan(got[touched]).any(axis=-1).all()


def test_attention_infinite_values(env):
    # an infinity in V that a row sees reaches its dims only, in both signs
    for dtype in ("bf16", "f16", "f32"):
        for lens in ([(100, 1), (300, 1)], [(100, 70), (5, 40)]):
            b = Batch(lens, 8, 2, 128, dtype, 16, seed=10)
            page = b.table[0, 1]
            b.v[page, :, 2, 5], b.v[page, :, 3, 9] = np.inf, -np.inf
            want, parts = R.attention(b.q, b.k, b.v, b.table, b.starts, b.keys, b.old, b.scale)
            got = b.run(env)
            fin = np.isfinite(want)
            assert (~fin).any()
            np.testing.assert_array_equal(got[~fin], want[~fin])
            with np.errstate(invalid="ignore"):
                ok = np.abs(got - want) <= R.attention_bound(np.where(fin, want, 0), [np.where(np.isfinite(p), p, 0) for p in parts], dtype, b.hd)
            assert ok[fin].all()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_attention_large_scores(env, dtype):
    # scores of +-200 and more: the running maximum moves, late and early
    for lens in ([(400, 1), (90, 1)], [(150, 80)]):
        b = Batch(lens, 8, 2, 128, dtype, 16, seed=11)
        ramp = np.linspace(-3, 3, b.k.shape[0])[:, None, None, None].astype(np.float32)
        b.k = rounded(b.k * ramp * 4, dtype)
        b.check(env)
        b.scale = -b.scale  # a negative scale turns the order round
        b.check(env)
        b.scale = 0.0
        b.check(env)


def test_attention_unaligned(env):
    pa, _, stream, enc = env
    for dtype in ("bf16", "f32"):
        b = Batch(LENS["mixed"], 4, 2, 64, dtype, 16, seed=12)
        size = {"bf16": 2, "f32": 4}[dtype]

        def shifted(x):
            t = upload(pa, np.concatenate([[0.0], x.ravel()]), dtype)
            return pa.Tensor(t.ptr + size, x.shape, dtype, owner=t)

        t = [shifted(x) for x in (b.q, b.k, b.v, b.old)]
        enc.encode(pa.Kernels.PagedAttention(*t[:3], i32(pa, b.table), i32(pa, b.starts), i32(pa, b.keys), t[3], scale=b.scale))
        stream.synchronize()
        want, parts = R.attention(b.q, b.k, b.v, b.table, b.starts, b.keys, b.old, b.scale)
        assert (np.abs(download(t[3], stream) - want) <= R.attention_bound(want, parts, dtype, 64)).all()


def test_attention_empty_calls(env):
    pa, _, stream, enc = env
    e = lambda *s: pa.Tensor.empty(s, "bf16")
    z = lambda *s: i32(pa, np.zeros(s))
    old = upload(pa, np.ones((5, 4, 64)), "bf16")
    for tokens, pages, requests, columns in ((0, 3, 2, 2), (5, 3, 0, 2), (5, 3, 2, 0), (5, 0, 2, 2)):
        out = old.view([tokens, 4, 64])
        enc.encode(pa.Kernels.PagedAttention(e(tokens, 4, 64), e(pages, 2, 16, 64), e(pages, 2, 16, 64), z(requests, columns),
                                             z(requests + 1), z(requests), out, scale=1.0))
    stream.synchronize()
    assert (download(old, stream) == 1).all()
    # every key on a page that is not there
    q = upload(pa, np.ones((2, 4, 64)), "bf16")
    enc.encode(pa.Kernels.PagedAttention(q, e(0, 2, 16, 64), e(0, 2, 16, 64), z(2, 3), i32(pa, [0, 1, 2]), i32(pa, [40, 1]),
                                         old.view([2, 4, 64]), scale=1.0))
    stream.synchronize()
    got = download(old, stream)
    assert not got[:2].any() and (got[2:] == 1).all()


def test_attention_cache_past_4_gib(env):
    # two pages at either end of caches of 4.5 GiB each: offsets past 32 bits
    pa, _, stream, enc = env
    nq, nkv, hd, page = 4, 2, 128, 16
    pages = (9 << 29) // (nkv * page * hd * 2)
    g = np.random.default_rng(13)
    k, v = pa.Tensor.empty([pages, nkv, page, hd], "bf16"), pa.Tensor.empty([pages, nkv, page, hd], "bf16")
    rows = [rounded(g.standard_normal((40, nkv, hd)), "bf16") for _ in range(2)]
    ids = [pages - 1, 0, pages - 2]
    slots = [ids[j // page] * page + j % page for j in range(40)]
    q = rounded(g.standard_normal((3, nq, hd)), "bf16")
    out = pa.Tensor.empty([3, nq, hd], "bf16")
    enc.encode(pa.Kernels.PagedKVCacheWrite(upload(pa, rows[0], "bf16"), upload(pa, rows[1], "bf16"), i32(pa, slots), k, v),
               pa.Kernels.PagedAttention(upload(pa, q, "bf16"), k, v, i32(pa, [ids]), i32(pa, [0, 3]), i32(pa, [40]), out, scale=0.088))
    stream.synchronize()
    small = [np.zeros((3, nkv, page, hd), np.float32) for _ in range(2)]
    for x, r in zip(small, rows):
        for j in range(40):
            x[j // page, :, j % page] = r[j]
    want, parts = R.attention(q, *small, np.array([[0, 1, 2]]), [0, 3], [40], np.zeros((3, nq, hd)), np.float32(0.088))
    assert (np.abs(download(out, stream) - want) <= R.attention_bound(want, parts, "bf16", hd)).all()


def test_attention_many_requests(env):
    # more tiles than a block lays out by itself
    g = np.random.default_rng(14)
    lens = [(int(p), int(n)) for p, n in zip(g.integers(0, 60, 1500), g.integers(0, 3, 1500))]
    for dtype in ("bf16", "f32"):
        Batch(lens, 4, 2, 64, dtype, 16, seed=15, pad=2).check(env)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,requests", [((16, 8, 128), 66), ((8, 8, 64), 70), ((12, 4, 256), 65), ((2, 1, 128), 520)], ids=str)
@pytest.mark.parametrize("mask,sinks", [((0, -1), 0), ((1, 40), 3)])
def test_attention_few_rows_beside_tiles(env, dtype, heads, requests, mask, sinks):
    # as many units as blocks: requests of few rows and of many in launches of their own, short and long in turn
    g = np.random.default_rng(16)
    lens = [(int(p), int(n)) for p, n in zip(g.integers(0, 200, requests), g.integers(0, 5, requests))]
    lens[0], lens[7], lens[40], lens[-1] = (5, 90), (130, 17), (0, 70), (64, 150)
    Batch(lens, *heads, dtype, 16, seed=17, pad=2).check(env, mask, sinks)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads", [(8, 2, 64), (4, 1, 128), (8, 2, 256)], ids=str)
@pytest.mark.parametrize("rows", [32, 36, 64, 68, 128, 132])
def test_attention_one_request_of_few_rows(env, dtype, heads, rows):
    # either side of the rows at which tiles take over
    Batch([(700, rows // (heads[0] // heads[1]))], *heads, dtype, 32, seed=rows).check(env)


@pytest.mark.parametrize("dtype,hd", [("bf16", 36), ("f16", 33), ("f32", 62), ("bf16", 500)])
def test_attention_odd_rows_of_an_empty_cache(env, dtype, hd):
    # every key on a page that is not there, rows that are no 16-byte runs
    pa, _, stream, enc = env
    e = lambda *s: pa.Tensor.empty(s, dtype)
    q, out = (upload(pa, np.ones((3, 4, hd)), dtype) for _ in range(2))
    enc.encode(pa.Kernels.PagedAttention(q, e(0, 2, 16, hd), e(0, 2, 16, hd), i32(pa, np.zeros((2, 3))), i32(pa, [0, 1, 2]), i32(pa, [40, 1]),
                                         out, scale=1.0))
    stream.synchronize()
    got = download(out, stream)
    assert not got[:2].any() and (got[2:] == 1).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads", [(4, 2, 33), (2, 1, 250), (3, 3, 510)], ids=str)
@pytest.mark.parametrize("mask,sinks", [((0, -1), 0), ((2, -1), 0), ((1, 40), 3)])
def test_attention_odd_rows(env, dtype, heads, mask, sinks):
    Batch([(500, 1), (0, 1), (0, 7), (30, 2), (15, 0), (64, 33)], *heads, dtype, 16, seed=heads[2], pad=2).check(env, mask, sinks)


@pytest.mark.parametrize("dtype,heads,mask,sinks", [("bf16", (16, 16, 64), (0, -1), 0), ("f16", (8, 8, 256), (1, 18000), 70)])
def test_attention_long_keys_in_tiles(env, dtype, heads, mask, sinks):
    # one new token in a tile beside a chunk, and more steps for a block than it looks up pages for at once
    Batch([(20000, 1), (19900, 40)], *heads, dtype, 64, seed=18).check(env, mask, sinks)


# ---- plans laid out in memory: more tiles or requests than a block lays out by itself ----------------------


def launches(b, hint=None):
    """The kernels of a batch's call, in order."""
    import popcorn_amd as pa

    fake = lambda i, shape, t: pa.Tensor(0x7F0000000000 + (i << 44), list(shape), t)  # (descriptors only validate)
    k = pa.Kernels.PagedAttention(fake(1, b.q.shape, b.dtype), fake(2, b.k.shape, b.dtype), fake(3, b.v.shape, b.dtype),
                                  fake(4, b.table.shape, "i32"), fake(5, [len(b.lens) + 1], "i32"), fake(6, [len(b.lens)], "i32"),
                                  fake(7, b.q.shape, b.dtype), scale=b.scale,
                                  max_query_len=max(n for _, n in b.lens) if hint is None else hint)
    return [n.replace("paged_attention_", "").replace("paged_", "").split("_")[0] for n in k.function_names]


@pytest.mark.parametrize("dtype,hd", [("bf16", 64), ("f16", 128), ("bf16", 256)])
def test_planned_few_and_tiles(env, dtype, hd):
    # more requests than a block lays out: both launches read plans, each its own
    g = np.random.default_rng(40)
    lens = [(int(p), int(n)) for p, n in zip(g.integers(0, 60, 1100), g.integers(0, 3, 1100))]
    for r, x in ((0, (70, 50)), (500, (0, 90)), (501, (33, 17)), (777, (130, 40)), (1099, (5, 66))):
        lens[r] = x
    b = Batch(lens, 4, 2, hd, dtype, 16, seed=41, pad=2)
    assert launches(b) == ["plan", "few", "plan", "tile", "merge"]
    b.check(env)
    b.check(env, (1, 40), 3)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_planned_few_beside_tiles_of_the_blocks(env, dtype):
    # more tiles of 16 rows than a block lays out, fewer of 128 rows: a plan for one launch only
    g = np.random.default_rng(42)
    lens = [(int(p), int(n)) for p, n in zip(g.integers(0, 90, 520), g.integers(1, 5, 520))]
    lens[3], lens[100], lens[519] = (64, 100), (0, 300), (17, 60)
    b = Batch(lens, 16, 2, 64, dtype, 16, seed=43, pad=1)
    assert launches(b) == ["plan", "few", "tile", "merge"]
    b.check(env)
    b.check(env, (1, 30), 20)


@pytest.mark.parametrize("dtype,heads", [("bf16", (16, 1, 64)), ("f16", (16, 1, 64)), ("f16", (16, 1, 128))], ids=str)
def test_planned_tiles_of_a_long_prompt(env, dtype, heads):
    # one prompt of more tiles than a block lays out; a window keeps the reference small
    b = Batch([(20, 8250)], *heads, dtype, 64, seed=44, pad=3)
    assert launches(b) == ["plan", "tile", "merge"]
    got = b.run(env, (1, 24), 2)
    rows = np.r_[0:40, 4000:4030, 8220:8250]
    want, parts = sampled_rows(b, rows, (1, 24), 2)
    assert (np.abs(got[rows] - want) <= R.attention_bound(want, parts, dtype, b.hd)).all()
    np.testing.assert_array_equal(got[8250:], b.old[8250:])
    assert np.isfinite(got).all()


def sampled_rows(b, rows, mask, sinks):
    """The reference of some new tokens of a batch of one request: each as a request of its own over the same pages."""
    past, n = b.lens[0]
    keys = np.array([past + r + 1 for r in rows])
    return R.attention(b.q[rows], b.k, b.v, np.repeat(b.table, len(rows), 0), np.arange(len(rows) + 1), keys, b.old[rows], b.scale,
                       mask[0], mask[1], sinks)


@pytest.mark.parametrize("dtype,hd", [("bf16", 512), ("f32", 256)])
def test_planned_few_of_other_kinds(env, dtype, hd):
    # requests of a row and a prompt without tiles
    g = np.random.default_rng(45)
    lens = [(int(p), int(n)) for p, n in zip(g.integers(0, 40, 1060), g.integers(0, 2, 1060))]
    lens[9] = (30, 70)
    b = Batch(lens, 4, 2, hd, dtype, 16, seed=46, pad=2)
    assert launches(b) == ["plan", "few", "merge"]
    b.check(env)


# ---- the bits of a weight in its product with V ---------------------------------------------


def words_of(w, dtype, words):
    """A weight as the sum of `words` numbers of the type."""
    left, total = np.array(w, np.float64), 0.0
    for _ in range(words):
        part = rounded(left, dtype).astype(np.float64)
        total, left = total + part, left - part
    return total


def against_each_other(dtype, lens, heads, page, seed):
    """Keys of two scores in turn, whose weights meet values that take each other away: what a weight loses in its
    rounding is left, where in a sum of random values the rounding of the result hides it."""
    b = Batch(lens, *heads, dtype, page, seed=seed)
    b.scale = 1.0
    b.q[:], b.q[..., 0] = 0.0, 1.0
    # the score whose weight has the largest remainder behind one word (the maximum's weight is a power of two)
    scores = np.arange(1, 129) / 64.0
    lost = np.abs(words_of(np.exp(-scores), dtype, 1) - np.exp(-scores)) * np.exp(scores)
    low = -scores[np.argmax(lost)]
    for r, (p, n) in enumerate(b.lens):
        for j in range(p + n):
            at = (b.table[r, j // page], slice(None), j % page)
            b.k[at] = 0.0
            b.k[at + (0,)] = low if j % 2 else 0.0
            b.v[at] = rounded(-np.exp(-low) if j % 2 else 1.0, dtype)
    return b, low


@pytest.mark.parametrize("dtype,lens,heads,kind,words", [
    ("f16", [(255, 1), (600, 1)], (4, 2, 64), "few", 2), ("f16", [(128, 4)], (8, 2, 128), "few", 2), ("f16", [(201, 1)], (8, 4, 256), "few", 2),
    ("f16", [(99, 9)], (2, 1, 512), "few", 2), ("bf16", [(255, 1), (600, 1)], (4, 2, 64), "few", 2), ("bf16", [(201, 1)], (8, 4, 256), "few", 2),
    ("bf16", [(99, 9)], (2, 1, 512), "few", 2), ("bf16", [(128, 72)], (8, 2, 64), "tile", 2), ("bf16", [(100, 60)], (8, 2, 128), "tile", 2),
    ("bf16", [(64, 90)], (4, 2, 256), "tile", 2), ("f16", [(128, 72)], (8, 2, 64), "tile", 1), ("f16", [(64, 90)], (4, 2, 256), "tile", 1)])
def test_attention_weights_keep_their_bits(env, dtype, lens, heads, kind, words):
    b, low = against_each_other(dtype, lens, heads, 16, seed=50)
    assert launches(b)[0] == kind
    got = b.run(env)
    want, (mag, spread, count) = R.attention(b.q, b.k, b.v, b.table, b.starts, b.keys, b.old, b.scale)
    # as R.attention_bound, with the words of this kernel: 11 bits in an f16, 8 in a bf16, and as many in the second
    weight = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}[dtype] ** words
    eps = 2.0 * ((heads[2] + 3) * 2.0 ** -24 * spread + 2.0 ** -22) + weight + (count + 8) * 2.0 ** -24
    bound = R.HALF[dtype] * np.abs(want) + R.TINY[dtype] + mag * eps * (1.0 + R.HALF[dtype])
    assert (np.abs(got - want) <= bound).all()
    if words == 2:  # a kernel that lost the second word would not pass
        last = b.starts[1:] - 1
        n = b.keys // 2
        w = np.exp(low)
        lost = n * abs(words_of([w], dtype, 1)[0] - w) * np.exp(-low) / (b.keys - n + n * w)
        assert (lost > 2 * bound[last].max(axis=(1, 2))).all(), (lost, bound[last].max(axis=(1, 2)))
