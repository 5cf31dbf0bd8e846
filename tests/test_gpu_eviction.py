"""GPU tests of attention weights, eviction by them and the pages that it frees, against 64-bit references, at the lengths, masks,
ties and pages where they can go wrong; and of a server's steps with all of them, eagerly and from a graph."""
import numpy as np
import pytest

import cache_ref as C
from gpu_util import download, gpu_env, rounded, upload
from test_gpu_shared_prefix import Batch, i32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    return gpu_env()


def f32(pa, x):
    return pa.Tensor.from_numpy(np.asarray(x, np.float32), "f32")


# ---- weights -----------------------------------------------------------------------


def logarithms(b, scale, kind):
    """What the attention before would give, rounded to f32; odd ones where no row looks."""
    _, lse, _ = C.shared_attention(b.q, b.k, b.v, [], [], [0], b.table, b.starts, b.keys, b.out, b.lse, scale, kind)
    return lse.astype(np.float32)


def weigh(env, b, scale, kind=0, last_rows=0, hint=0, lse=None, kinds=None, t=None):
    pa, _, stream, enc = env
    scale = float(np.float32(scale))
    lse = logarithms(b, scale, kind) if lse is None else lse
    page, nkv = b.k.shape[2], b.k.shape[1]
    old = np.random.default_rng(1).random((len(b.lens), nkv, b.table.shape[1] * page)).astype(np.float32)
    t = t or b.tensors(pa)[0]
    w = f32(pa, old)
    k = pa.Kernels.PagedAttentionWeights(t[0], t[1], *t[6:9], f32(pa, lse), w, scale=scale, last_rows=last_rows, max_query_len=hint,
                                         mask=pa.AttentionMask.bidirectional if kind == 2 else pa.AttentionMask.causal)
    if kinds is not None:
        assert {n.split("_")[2] for n in k.function_names} - {"plan"} == kinds
    enc.encode(k)
    stream.synchronize()
    got = download(w, stream)
    ref, bound = C.weights(b.q, b.k, b.table, b.starts, b.keys, lse, old, scale, kind, last_rows)
    untouched = ref == old
    np.testing.assert_array_equal(got[untouched], old[untouched])
    with np.errstate(invalid="ignore"):
        off = np.abs(got - ref)
        assert (off <= bound).all(), np.nanmax(off / bound)
    return got


ALONE = [(None, [(0, 1), (5, 1), (40, 1), (16, 1), (0, 0), (200, 0), (31, 2), (17, 1), (255, 1), (1000, 1)])]
PROMPTS = [(None, [(0, 40), (5, 1), (70, 3), (0, 0), (20, 165), (9, 33), (300, 64)])]
SHAPES = [(8, 4, 256, 16), (8, 2, 128, 48), (4, 2, 64, 32), (6, 2, 80, 16), (4, 1, 512, 16), (4, 2, 36, 16), (3, 3, 7, 16), (24, 1, 64, 16)]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("nq,nkv,hd,page", SHAPES)
@pytest.mark.parametrize("kind", [0, 2])
def test_weights_of_single_tokens(env, dtype, nq, nkv, hd, page, kind):
    weigh(env, Batch(ALONE, nq, nkv, hd, dtype, page, hd, pad=3), hd ** -0.5, kind, hint=2)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("nq,nkv,hd,page", SHAPES)
@pytest.mark.parametrize("kind,last_rows", [(0, 0), (2, 0), (0, 1), (0, 32), (2, 33)])
def test_weights_of_prompts(env, dtype, nq, nkv, hd, page, kind, last_rows):
    weigh(env, Batch(PROMPTS, nq, nkv, hd, dtype, page, hd, pad=3), hd ** -0.5, kind, last_rows)


@pytest.mark.parametrize("hint", [1, 5, 200])
def test_a_wrong_hint_chooses_kernels_alone(env, hint):
    weigh(env, Batch(PROMPTS, 8, 2, 128, "bf16", 16, 1), 0.1, hint=hint)
    weigh(env, Batch(ALONE, 8, 2, 128, "bf16", 16, 1), 0.1, hint=hint)


@pytest.mark.parametrize("requests", [1, 300, 1024, 1100])
def test_weights_of_many_requests(env, requests):
    g = np.random.default_rng(requests)
    b = Batch([(None, [(int(p), 1) for p in g.integers(0, 60, requests)])], 4, 2, 64, "f16", 16, 2)
    weigh(env, b, 0.125, hint=1)
    if requests < 1024:
        weigh(env, b, 0.125)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_weights_where_nothing_counts(env, dtype):
    # rows that saw no key, keys of no page, NaN and infinities in rows and keys that do not count
    for groups in (ALONE, PROMPTS):
        b = Batch(groups, 4, 2, 64, dtype, 16, 3)
        lse = logarithms(b, 0.125, 0)
        lse[::3] = -np.inf
        b.q[::3] = np.nan
        b.table[2, 0] = -1
        b.table[6, 1] = 2 ** 31 - 1
        b.keys[0] = 0
        weigh(env, b, 0.125, 0, lse=lse)
        b = Batch(PROMPTS, 4, 2, 64, dtype, 16, 4)
        lse = logarithms(b, 0.125, 0)
        for r in (0, 4, 6):  # all but the last two rows of a request do not count
            a, e = b.starts[r], b.starts[r + 1]
            b.q[a:e - 2], lse[a:e - 2] = np.nan, np.nan
        weigh(env, b, 0.125, 0, last_rows=2, lse=lse)


def test_weights_of_a_shared_prefix(env):
    # the logarithms hold the prefix's share, so that the own keys' weights and the prefix's add up to the rows
    pa, _, stream, enc = env
    b = Batch([(90, [(20 + i, 1 + i % 2) for i in range(6)])], 8, 2, 128, "bf16", 16, 5)
    t, lse = b.tensors(pa)
    enc.encode(pa.Kernels.SharedPrefixAttention(*t, scale=0.1, lse=lse))
    stream.synchronize()
    w = weigh(env, b, 0.1, lse=download(lse, stream).astype(np.float32), t=t)
    got = w - np.random.default_rng(1).random(w.shape).astype(np.float32)
    rows = np.diff(b.starts) * 4
    assert (got.sum(-1) < rows[:, None]).all() and (got.sum(-1) > 0.05 * rows[:, None]).all()


def test_weights_are_the_same_twice(env):
    b = Batch(PROMPTS, 8, 2, 128, "bf16", 16, 6, std=3.0)
    np.testing.assert_array_equal(weigh(env, b, 0.1), weigh(env, b, 0.1))


def test_weights_of_data_that_is_not_aligned(env):
    pa = env[0]
    b = Batch(PROMPTS, 4, 2, 64, "f16", 16, 7)
    t, _ = b.tensors(pa)
    flat = upload(pa, np.concatenate([[0.0], b.k.ravel()]), "f16")
    t[1] = pa.Tensor(flat.ptr + 2, b.k.shape, "f16", owner=flat)
    weigh(env, b, 0.125, t=t, kinds={"plain"})


# ---- eviction ----------------------------------------------------------------------


def evict(env, lens, budgets, first, last, nkv, hd, page, dtype, seed, weights="ties", spare=1, offset=0, bad=()):
    pa, _, stream, enc = env
    g = np.random.default_rng(seed)
    held = [-(-max(n, 0) // page) for n in lens]
    pages = sum(held) + 2
    ids = g.permutation(pages)
    table = np.full((len(lens), max(held) + spare), -1, np.int64)
    at = 0
    for r, h in enumerate(held):
        table[r, :h] = ids[at:at + h]
        at += h
    for r, c, v in bad:
        table[r, c] = v
    room = table.shape[1] * page
    shape = (len(lens), nkv, room)
    if weights == "ties":
        w = g.integers(0, 4, shape) / 4
    elif weights == "special":
        w = g.choice([np.nan, np.inf, -np.inf, 0.0, -0.0, 1e-45, -1e-45, 1.0, -1.0, 3e38], shape)
    else:
        w = np.exp(3 * g.standard_normal(shape))
    w = w.astype(np.float32)
    k, v = (rounded(g.standard_normal((pages, nkv, page, hd)), dtype) for _ in range(2))
    size = {"f32": 4, "f16": 2, "bf16": 2}[dtype]

    def shifted(x):
        t = upload(pa, np.concatenate([np.zeros(offset), x.ravel()]), dtype)
        return pa.Tensor(t.ptr + offset * size, x.shape, dtype, owner=t)

    kt, vt = shifted(k), shifted(v)
    kept, kept_w = i32(pa, np.full(shape, -7)), f32(pa, np.full(shape, 7.0))
    wt, lt, bt, tt = f32(pa, w), i32(pa, lens), i32(pa, budgets), i32(pa, table)
    enc.encode(pa.Kernels.PagedEviction(wt, kt, vt, tt, lt, bt, kept, kept_w, first=first, last=last))
    new, freed, counts = i32(pa, np.full(len(lens), -7)), i32(pa, np.full(table.size, -7)), i32(pa, [-7])
    enc.encode(pa.Kernels.ReleasePages(lt, bt, tt, page_size=page, new_lens=new, freed=freed, counts=counts))
    stream.synchronize()
    ref = C.evict(w, k, v, table, lens, budgets, np.full(shape, -7), first, last)
    np.testing.assert_array_equal(kept.numpy(stream), ref[0])
    np.testing.assert_array_equal(kept_w.numpy(stream), ref[1])
    np.testing.assert_array_equal(download(kt, stream), ref[2])
    np.testing.assert_array_equal(download(vt, stream), ref[3])
    np.testing.assert_array_equal(wt.numpy(stream), w)
    lens_, freed_, n = C.release(lens, budgets, table, page, np.full(table.size, -7))
    np.testing.assert_array_equal(new.numpy(stream), lens_)
    np.testing.assert_array_equal(freed.numpy(stream), freed_)
    assert list(counts.numpy(stream)) == [n]


LENS = [0, 1, 15, 16, 17, 100, 255, 256, 257, 300]


@pytest.mark.parametrize("weights", ["ties", "special", "spread"])
@pytest.mark.parametrize("budget", [0, 1, 16, 31, 100, 256, 5000])
@pytest.mark.parametrize("first,last", [(0, 0), (4, 8), (1, 0), (0, 40), (200, 200)])
def test_eviction(env, weights, budget, first, last):
    evict(env, LENS, [budget] * len(LENS), first, last, 2, 16, 16, "f16", budget, weights)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("nkv,hd,page,offset", [(4, 256, 16, 0), (2, 128, 48, 0), (1, 80, 7, 0), (2, 36, 16, 0), (3, 13, 16, 0), (2, 64, 16, 1),
                                                (1, 512, 128, 2), (2, 1, 1, 0)])
def test_eviction_of_any_rows(env, dtype, nkv, hd, page, offset):
    g = np.random.default_rng(hd)
    lens = [int(x) for x in g.integers(0, 400, 5)]
    evict(env, lens, [int(x) for x in g.integers(0, 300, 5)], 3, 5, nkv, hd, page, dtype, hd, "spread", offset=offset)


@pytest.mark.parametrize("length,budget,weights", [(9000, 4096, "spread"), (9000, 4095, "ties"), (5000, 4999, "spread"), (20011, 12345, "ties"),
                                                   (70000, 30000, "special")])
def test_eviction_of_long_requests(env, length, budget, weights):
    # several of the block's passes and chunks; rows that move by one place and by many
    evict(env, [length, length // 3], [budget, budget // 2], 4, 100, 2, 32, 16, "bf16", length, weights)


def test_eviction_at_odd_lengths(env):
    # lengths and budgets below 0 and past the table, entries of no page
    big = 2 ** 31 - 1
    evict(env, [-5, 40, 60, 33], [3, -9, big, 0], 1, 1, 2, 16, 16, "f16", 1)
    evict(env, [100, 90, 64], [40, 30, 20], 2, 2, 2, 16, 16, "f16", 2, bad=[(0, 2, -1), (1, 0, 2 ** 31 - 1), (2, 3, -1)])
    evict(env, [100, 90, 64], [40, 30, 20], big, big, 2, 16, 16, "f16", 3)
    pa, _, stream, enc = env
    # longer than its table
    w = f32(pa, np.arange(32)[::-1].reshape(1, 1, 32))
    k = upload(pa, np.arange(64).reshape(2, 1, 16, 2), "f32")
    v = upload(pa, np.arange(64).reshape(2, 1, 16, 2), "f32")
    kept, kw = i32(pa, np.zeros((1, 1, 32))), f32(pa, np.zeros((1, 1, 32)))
    enc.encode(pa.Kernels.PagedEviction(w, k, v, i32(pa, [[1, 0]]), i32(pa, [big]), i32(pa, [4]), kept, kw, first=0, last=1))
    stream.synchronize()
    assert list(kept.numpy(stream)[0, 0, :4]) == [0, 1, 2, 31]
    assert list(k.numpy(stream)[1, 0, 3]) == [30.0, 31.0]


@pytest.mark.parametrize("requests", [0, 1, 15, 17, 255, 257, 5000])
def test_release(env, requests):
    pa, _, stream, enc = env
    g = np.random.default_rng(requests)
    lens, budgets = g.integers(-3, 300, requests), g.integers(-3, 300, requests)
    table = g.integers(-1, 10 ** 6, (requests, 20))
    new, freed, counts = i32(pa, np.full(requests, -7)), i32(pa, np.full(table.size, -7)), i32(pa, [-7])
    enc.encode(pa.Kernels.ReleasePages(i32(pa, lens), i32(pa, budgets), i32(pa, table), page_size=13, new_lens=new, freed=freed, counts=counts))
    stream.synchronize()
    lens_, freed_, n = C.release(lens, budgets, table, 13, np.full(table.size, -7))
    np.testing.assert_array_equal(new.numpy(stream), lens_)
    np.testing.assert_array_equal(freed.numpy(stream), freed_)
    assert list(counts.numpy(stream)) == [n]


def test_weights_of_starts_out_of_order(env):
    # within the tensors whatever the lengths say: what lies around the weights is as it was
    pa, _, stream, enc = env
    g = np.random.default_rng(17)
    for i in range(6):
        for hd, dtype in ((64, "bf16"), (64, "f32"), (36, "f16")):
            b = Batch(PROMPTS, 4, 2, hd, dtype, 16, 18, pad=4)
            t, _ = b.tensors(pa)
            starts = g.permutation(b.starts) if i % 2 else g.integers(-5, 400, b.starts.size)
            R_, room = len(b.lens), b.table.shape[1] * 16
            big = f32(pa, np.full((R_ + 2, 2, room), 5.0))
            w = pa.Tensor(big.ptr + 2 * room * 4, (R_, 2, room), "f32", owner=big)
            lse = f32(pa, np.full(b.q.shape[:2], 3.0))
            enc.encode(pa.Kernels.PagedAttentionWeights(t[0], t[1], t[6], i32(pa, starts), i32(pa, g.integers(-9, 900, R_)), lse, w, scale=0.1))
            stream.synchronize()
            x = download(big, stream)
            assert (x[0] == 5.0).all() and (x[-1] == 5.0).all()


def test_caches_past_32_bits(env):
    # the requests' pages lie more than 2^32 elements behind the cache's first
    pa, _, stream, enc = env
    nkv, hd, page = 1, 512, 16
    pages = 2 ** 32 // (nkv * hd * page) + 64
    b = Batch([(100, [(60, 1), (5, 1)]), (None, [(200, 1), (33, 20)])], 4, nkv, hd, "bf16", page, 19)
    used = len(b.k)
    first = pages - used
    caches = []
    for x in (b.k, b.v):
        big = pa.Tensor.empty([pages, nkv, page, hd], "bf16")
        view = pa.Tensor(big.ptr + first * nkv * page * hd * 2, x.shape, "bf16", owner=big)
        import oracle as O

        view.copy_from(O.to_bits(x, O.BF16), stream)
        caches.append((big, view))
    t, lse = b.tensors(pa)
    for i, x in ((3, b.prefix_table), (6, b.table)):
        t[i] = i32(pa, np.where(x >= 0, x + first, -1))
    t[1], t[2] = caches[0][0], caches[1][0]
    enc.encode(pa.Kernels.SharedPrefixAttention(*t, scale=0.05, lse=lse))
    stream.synchronize()
    b.check(download(t[-1], stream), download(lse, stream), 0.05)
    weigh(env, b, 0.05, t=t, lse=download(lse, stream).astype(np.float32))
    lens = b.keys
    w = np.random.default_rng(3).random((4, nkv, b.table.shape[1] * page)).astype(np.float32)
    kept, kept_w = i32(pa, np.full(w.shape, -7)), f32(pa, w)
    enc.encode(pa.Kernels.PagedEviction(f32(pa, w), t[1], t[2], t[6], i32(pa, lens), i32(pa, [20] * 4), kept, kept_w, first=2, last=3))
    stream.synchronize()
    ref = C.evict(w, b.k, b.v, b.table, lens, [20] * 4, np.full(w.shape, -7), 2, 3)
    np.testing.assert_array_equal(kept.numpy(stream), ref[0])
    for (_, view), x in zip(caches, ref[2:4]):
        np.testing.assert_array_equal(download(view, stream), x)


@pytest.mark.parametrize("dtype,hd,last_rows", [("bf16", 128, 0), ("f16", 256, 0), ("bf16", 64, 40)])
def test_weights_of_prompts_among_many_single_tokens(env, dtype, hd, last_rows):
    # a launch for requests of few rows beside the tiles'
    lens = [(int(p), 1) for p in np.random.default_rng(hd).integers(0, 90, 40)]
    lens[7], lens[30] = (33, 130), (0, 70)
    weigh(env, Batch([(None, lens)], 8, 2, hd, dtype, 16, 20), hd ** -0.5, last_rows=last_rows, kinds={"few", "tile", "join"})


def test_weights_of_more_tiles_than_a_block_lays_out(env):
    lens = [(int(p), 1 + 40 * (i % 50 == 0)) for i, p in enumerate(np.random.default_rng(4).integers(0, 60, 1100))]
    weigh(env, Batch([(None, lens)], 4, 2, 64, "bf16", 16, 21), 0.125, kinds={"few", "tiles", "tile", "join"})
