"""GPU tests of attention over prefixes that requests share, against a 64-bit reference: every kernel it is made of, the groups,
lengths, masks and pages where it can go wrong, its logarithms, graphs and streams."""
import numpy as np
import pytest

import cache_ref as C
from gpu_util import download, gpu_env, rounded, upload
from test_gpu_serving import Graph

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    return gpu_env()


def i32(pa, x):
    return pa.Tensor.from_numpy(np.asarray(x, np.int32), "i32")


class Batch:
    """Groups of requests: groups = [(prefix keys, [(past, new), ...]), ...], prefix None for requests of no group; a cache whose pages stand
    in any order, with NaN wherever no key is."""

    def __init__(self, groups, nq, nkv, hd, dtype, page, seed, pad=0, spare=1, fill=np.nan, std=1.0):
        g = np.random.default_rng(seed)
        self.dtype, self.hd = dtype, hd
        self.lens = [x for _, rs in groups for x in rs]
        self.group_starts, self.prefix_lens = [], []
        at = 0
        for prefix, rs in groups:  # (a stretch without a prefix is a group whose prefix has no key, or behind the last group)
            self.group_starts.append(at)
            self.prefix_lens.append(prefix or 0)
            at += len(rs)
        self.group_starts.append(at)
        if groups[-1][0] is None:
            self.group_starts.pop()
            self.prefix_lens.pop()
        own = [p + n for p, n in self.lens]
        need = [-(-x // page) for x in self.prefix_lens + own]
        pages = sum(need) + 2
        ids = g.permutation(pages)
        tables, live, at = [], np.zeros((pages, page), bool), 0
        for x, m in zip(self.prefix_lens + own, need):
            tables.append(ids[at:at + m])
            for j in range(x):
                live[ids[at + j // page], j % page] = True
            at += m

        def table(rows):
            t = np.full((len(rows), max([len(x) for x in rows] + [0]) + spare), -1, np.int64)
            for i, x in enumerate(rows):
                t[i, :len(x)] = x
            return t

        n = len(self.prefix_lens)
        self.prefix_table, self.table = table(tables[:n]), table(tables[n:])
        self.k, self.v = (rounded(g.standard_normal((pages, nkv, page, hd)), dtype) for _ in range(2))
        for c in (self.k, self.v):
            c[~np.broadcast_to(live[:, None, :, None], c.shape)] = fill
        self.starts = np.concatenate([[0], np.cumsum([m for _, m in self.lens])])
        self.keys = np.array(own)
        T = int(self.starts[-1]) + pad
        self.q = rounded(g.standard_normal((T, nq, hd)) * std, dtype)
        self.out = rounded(g.standard_normal((T, nq, hd)), dtype)
        self.lse = rounded(g.standard_normal((T, nq)), "f32")

    def tensors(self, pa):
        u = lambda x: upload(pa, x, self.dtype)  # noqa: E731
        return [u(self.q), u(self.k), u(self.v), i32(pa, self.prefix_table), i32(pa, self.prefix_lens), i32(pa, self.group_starts),
                i32(pa, self.table), i32(pa, self.starts), i32(pa, self.keys), u(self.out)], upload(pa, self.lse, "f32")

    def check(self, out, lse, scale, kind=0, window=-1, sinks=0):
        ref, ref_lse, parts = C.shared_attention(self.q, self.k, self.v, self.prefix_table, self.prefix_lens, self.group_starts, self.table,
                                                 self.starts, self.keys, self.out, self.lse, float(np.float32(scale)), kind, window, sinks)
        off, most = np.abs(out - ref), C.attention_bound(ref, parts, self.dtype, self.hd)
        live = np.zeros(len(self.q), bool)
        for a, b in zip(self.starts, self.starts[1:]):
            live[max(a, 0):max(b, 0)] = True
        same = (out == ref) | (np.isnan(out) & np.isnan(ref))
        assert same[~live].all() and (lse[~live] == ref_lse[~live]).all(), "rows of no request"
        assert (same | (off <= most)).all(), np.nanmax(np.where(same, 0, off / most))
        empty = np.isneginf(ref_lse)
        np.testing.assert_array_equal(np.isneginf(lse), empty)
        with np.errstate(invalid="ignore"):
            off, most = np.abs(lse - ref_lse), C.lse_bound(ref_lse, parts, self.hd)
        assert (empty | (off <= most))[live].all(), np.nanmax((off / most)[live & ~empty.all(1)])


def attend(env, b, scale, kind=0, window=-1, sinks=0, hint=0, kinds=None, with_lse=True):
    pa, _, stream, enc = env
    t, lse = b.tensors(pa)
    mask = {0: pa.AttentionMask.causal, 1: pa.AttentionMask.causal_sliding_window(window), 2: pa.AttentionMask.bidirectional}[kind]
    k = pa.Kernels.SharedPrefixAttention(*t, scale=scale, mask=mask, sinks=sinks, max_query_len=hint, lse=lse if with_lse else None)
    if kinds is not None:
        assert {n.split("_")[2] for n in k.function_names} - {"merge", "plan", "positions"} == kinds
    enc.encode(k)
    stream.synchronize()
    got = download(t[-1], stream), download(lse, stream)
    if with_lse:
        b.check(*got, scale, kind, window, sinks)
    else:
        np.testing.assert_array_equal(got[1], b.lse)
    return got


# prefixes that end inside a page and at its end, of one key, of none; a group without requests; requests without tokens, with more
# of them than keys in the cache, without past keys, of no group
GROUPS = [(77, [(0, 1), (5, 1), (40, 1)]), (0, [(3, 1)]), (33, []), (1, [(16, 1), (0, 1), (200, 0)]), (160, [(31, 1)] * 4), (None, [(18, 1), (0, 1)])]
MASKS = [(0, -1, 0), (1, 50, 3), (1, 24, 0), (1, 1, 90), (2, -1, 0)]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("nq,nkv,hd,page", [(8, 4, 256, 16), (8, 2, 128, 48), (4, 2, 64, 32), (6, 2, 80, 16), (4, 1, 512, 16), (4, 2, 36, 16),
                                            (3, 3, 7, 16)])
@pytest.mark.parametrize("kind,window,sinks", MASKS)
def test_single_tokens(env, dtype, nq, nkv, hd, page, kind, window, sinks):
    attend(env, Batch(GROUPS, nq, nkv, hd, dtype, page, hd + page, pad=3), hd ** -0.5, kind, window, sinks, hint=1)


CHUNKS = [(130, [(0, 40), (5, 1), (70, 3)]), (17, [(0, 1), (20, 65)]), (None, [(9, 30), (0, 2)])]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("nq,nkv,hd,page", [(8, 4, 256, 16), (8, 2, 128, 48), (4, 2, 64, 32), (6, 2, 80, 16), (4, 1, 512, 16), (4, 2, 36, 16)])
@pytest.mark.parametrize("kind,window,sinks", MASKS)
def test_chunks(env, dtype, nq, nkv, hd, page, kind, window, sinks):
    tile = dtype != "f32" and hd <= 256 and hd % 8 == 0
    attend(env, Batch(CHUNKS, nq, nkv, hd, dtype, page, 3 * hd + page, pad=5), hd ** -0.5, kind, window, sinks,
           kinds={"few", "many"} if tile and hd == 256 else {"both"} if tile else {"plain"} if hd == 36 and dtype != "f32" else {"few"})


@pytest.mark.parametrize("dtype,nq,nkv,hd", [("bf16", 16, 4, 128), ("f16", 8, 4, 256), ("bf16", 4, 2, 64), ("f16", 16, 4, 128)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (700, 4)])
def test_many_rows_many_pieces(env, dtype, nq, nkv, hd, window, sinks):
    # 45 requests' rows fill tiles of 128 and a part of one; the prefix is cut into pieces for most of the blocks
    b = Batch([(2000, [(7 * i % 60, 1) for i in range(45)]), (300, [(3, 1)] * 2)], nq, nkv, hd, dtype, 32, hd, std=2.0)
    attend(env, b, hd ** -0.5, 1 if window else 0, window or -1, sinks, hint=1,
           kinds={"few", "many"} if hd == 256 else {"both"})


def test_requests_of_few_rows_apart(env):
    b = Batch([(90, [(i % 40, 1) for i in range(300)]), (20, [(i % 9, 1 + i % 3) for i in range(40)])], 8, 2, 128, "bf16", 16, 5)
    attend(env, b, 0.1, kinds={"both"}, hint=3)


@pytest.mark.parametrize("window", [0, 40])
def test_plans_in_memory(env, window):
    # more requests than a block lays out by itself
    b = Batch([(64, [(i % 20, 1) for i in range(700)]), (None, [(i % 5, 1) for i in range(500)])], 4, 2, 64, "f16", 16, 6)
    pa = env[0]
    t, lse = b.tensors(pa)
    assert "shared_prefix_plan" in pa.Kernels.SharedPrefixAttention(*t, scale=0.1, lse=lse).function_names
    attend(env, b, 0.125, 1 if window else 0, window or -1, 2 if window else 0, hint=1)


@pytest.mark.parametrize("dtype,hd", [("bf16", 128), ("f16", 64), ("f32", 64), ("f16", 36)])
def test_without_prefixes_it_is_paged_attention(env, dtype, hd):
    pa, _, stream, enc = env
    for rs in ([(100, 1), (0, 3), (2000, 1), (7, 0)], [(50, 90), (0, 1)]):
        b = Batch([(None, rs)], 4, 2, hd, dtype, 16, 8, pad=2)
        b.prefix_lens, b.group_starts = [], [0]
        t, lse = b.tensors(pa)
        plain = upload(pa, b.out, dtype)
        a = pa.Kernels.PagedAttention(t[0], t[1], t[2], *t[6:9], t[9], scale=0.2, lse=lse)
        enc.encode(a, pa.Kernels.PagedAttention(t[0], t[1], t[2], *t[6:9], plain, scale=0.2))
        stream.synchronize()
        b.check(download(t[9], stream), download(lse, stream), 0.2)
        b.check(download(plain, stream), download(lse, stream), 0.2)


def test_logarithms_may_be_left_out(env):
    for hd in (64, 36):
        b = Batch(GROUPS, 4, 2, hd, "bf16", 16, 9)
        with_lse = attend(env, b, 0.2, hint=1)[0]
        np.testing.assert_array_equal(with_lse, attend(env, b, 0.2, hint=1, with_lse=False)[0])


@pytest.mark.parametrize("scale", [0.0, -0.3])
def test_scales(env, scale):
    for groups in (GROUPS, CHUNKS):
        attend(env, Batch(groups, 4, 2, 64, "bf16", 16, 10), scale)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_infinities_and_nan_where_no_row_looks(env, dtype):
    # keys behind a causal row that other rows of the tile see, and keys outside the window
    for groups in (CHUNKS, GROUPS):
        b = Batch(groups, 4, 2, 64, dtype, 16, 11)
        last = [(r, k) for r, k in enumerate(b.keys) if k > 0 and b.lens[r][1] > 1]
        for i, (r, k) in enumerate(last):
            row = (b.table[r, (k - 1) // 16], slice(None), (k - 1) % 16)
            b.v[row] = [np.inf, np.nan, -np.inf][i % 3]
            b.k[row] = np.nan if i % 2 else b.k[row]
        for p, n in zip(b.prefix_table, b.prefix_lens):
            if n > 30:
                b.v[p[0], :, 4] = np.nan
                b.k[p[0], :, 4] = np.inf
        t, lse = b.tensors(env[0])
        with np.errstate(invalid="ignore"):
            ref, ref_lse, parts = C.shared_attention(b.q, b.k, b.v, b.prefix_table, b.prefix_lens, b.group_starts, b.table, b.starts, b.keys,
                                                     b.out, b.lse, 0.125, 1, 12, 2)
        pa, _, stream, enc = env
        enc.encode(pa.Kernels.SharedPrefixAttention(*t, scale=0.125, mask=pa.AttentionMask.causal_sliding_window(12), sinks=2, lse=lse))
        stream.synchronize()
        out, got = download(t[-1], stream), download(lse, stream)
        fine = np.isfinite(ref).all(-1) & np.isfinite(ref_lse)
        assert fine.sum() > fine.size // 3
        with np.errstate(invalid="ignore"):
            assert (np.abs(out - ref) <= C.attention_bound(ref, parts, dtype, 64))[fine].all()
            assert (np.abs(got - ref_lse) <= C.lse_bound(ref_lse, parts, 64))[fine].all()


def test_pages_that_no_cache_holds_and_short_lengths(env):
    # table entries of no page are left out; a request with fewer keys than new tokens; lengths past the tables
    for groups in (GROUPS, CHUNKS):
        for kind, window, sinks in MASKS:
            b = Batch(groups, 4, 2, 64, "bf16", 16, 12)
            b.prefix_table[0, 1] = -1
            b.prefix_table[-1, 0] = len(b.k)
            b.table[2, 0] = 2 ** 31 - 1
            b.keys[0] = 0
            b.keys[1] = max(0, b.lens[1][1] - 2)
            for t in (b.prefix_table, b.table):
                assert t.max() >= len(b.k)
            attend(env, b, 0.125, kind, window, sinks)
            b.keys[3] = 2 ** 31 - 1  # (its table ends long before)
            b.k = np.nan_to_num(b.k)
            b.v = np.nan_to_num(b.v)
            if kind == 2:
                attend(env, b, 0.125, kind, window, sinks)


@pytest.mark.parametrize("hd", [64, 36])
def test_data_that_is_not_aligned(env, hd):
    pa, _, stream, enc = env
    b = Batch(GROUPS, 4, 2, hd, "f16", 16, 13)
    t, lse = b.tensors(pa)
    flat = upload(pa, np.concatenate([[0.0], b.v.ravel()]), "f16")
    t[2] = pa.Tensor(flat.ptr + 2, b.v.shape, "f16", owner=flat)
    k = pa.Kernels.SharedPrefixAttention(*t, scale=0.2, lse=lse)
    assert k.function_names == ["shared_prefix_plain_f16_any"]
    enc.encode(k)
    stream.synchronize()
    b.check(download(t[-1], stream), download(lse, stream), 0.2)


def test_nothing_to_do(env):
    pa, _, stream, enc = env
    for T, R, G in ((0, 2, 1), (3, 0, 0), (2, 2, 0)):
        q, out = (upload(pa, np.ones((T, 4, 64)), "bf16") for _ in range(2))
        k = upload(pa, np.ones((2, 2, 16, 64)), "bf16")
        starts = [0] * R + [0 if R == 0 else T]
        lse = upload(pa, np.ones((T, 4)), "f32")
        enc.encode(pa.Kernels.SharedPrefixAttention(q, k, k, i32(pa, np.zeros((G, 2))), i32(pa, [5] * G), i32(pa, [0] + [1] * G),
                                                    i32(pa, np.ones((R, 1))), i32(pa, starts), i32(pa, [4] * R), out, scale=1.0, lse=lse))
        stream.synchronize()
        assert np.isfinite(download(out, stream)).all()


def test_graph_replays_with_other_lengths(env):
    pa, lib, stream, enc = env
    sets = [Batch([(p, [(a + i, 1) for i in range(6)]), (33, [(a, 1)])], 8, 2, 128, "bf16", 16, s, std=2.0) for s, (p, a) in
            enumerate(((400, 5), (390, 20), (31, 0), (400, 60)))]
    size = max(len(b.k) for b in sets)
    for b in sets:  # of one shape
        b.k, b.v = (np.concatenate([x, np.full((size - len(x),) + x.shape[1:], np.nan, np.float32)]) for x in (b.k, b.v))
        b.prefix_table, b.table = (np.pad(x, ((0, 0), (0, w - x.shape[1])), constant_values=-1)
                                   for x, w in ((b.prefix_table, 30), (b.table, 9)))
    for mask, args in ((pa.AttentionMask.causal, (0, -1, 0)), (pa.AttentionMask.causal_sliding_window(50), (1, 50, 2))):
        t, lse = sets[0].tensors(pa)
        k = pa.Kernels.SharedPrefixAttention(*t, scale=0.1, mask=mask, sinks=args[2], max_query_len=1, lse=lse)
        enc.encode(k)  # scratch is there
        stream.synchronize()
        graph = Graph(pa, stream, lambda: enc.encode(k))
        for b in sets + sets[::-1]:
            u, w = b.tensors(pa)
            import oracle as O

            for x, y in zip((b.q, b.k, b.v, b.out), (t[0], t[1], t[2], t[9])):
                y.copy_from(O.to_bits(x, O.BF16), stream)
            lse.copy_from(b.lse.astype(np.float32), stream)
            for x, y in ((b.prefix_table, t[3]), (b.prefix_lens, t[4]), (b.group_starts, t[5]), (b.table, t[6]), (b.starts, t[7]), (b.keys, t[8])):
                y.copy_from(np.asarray(x, np.int32), stream)
            graph.launch()
            stream.synchronize()
            got = download(t[9], stream), download(lse, stream)
            b.check(*got, 0.1, *args)
            enc.encode(pa.Kernels.SharedPrefixAttention(*u, scale=0.1, mask=mask, sinks=args[2], max_query_len=1, lse=w))
            stream.synchronize()
            np.testing.assert_array_equal(got[0], download(u[9], stream))
            np.testing.assert_array_equal(got[1], download(w, stream))


def test_two_streams(env):
    pa, lib, stream, enc = env
    other = pa.Stream()
    enc2 = pa.KernelCommandEncoder(lib, other)
    bs = [Batch([(700 + 100 * s, [(3 * i, 1) for i in range(30)])], 8, 2, 128, "f16", 16, s) for s in range(2)]
    ts = [b.tensors(pa) for b in bs]
    for _ in range(3):
        for e, (t, lse) in zip((enc, enc2), ts):
            e.encode(pa.Kernels.SharedPrefixAttention(*t, scale=0.1, max_query_len=1, lse=lse))
    for s, b, (t, lse) in zip((stream, other), bs, ts):
        s.synchronize()
        b.check(download(t[-1], s), download(lse, s), 0.1)


@pytest.mark.parametrize("groups", [64, 65, 150])
@pytest.mark.parametrize("window", [0, 30])
def test_many_groups(env, groups, window):
    # as many as a wave's lanes hold, and more
    g = np.random.default_rng(groups)
    stretches = [(int(g.integers(0, 40)), [(int(g.integers(0, 20)), 1)] * int(g.integers(0, 4))) for _ in range(groups)] + [(None, [(3, 1)])]
    for hd, dtype in ((64, "bf16"), (64, "f32"), (36, "f16")):
        attend(env, Batch(stretches, 4, 2, hd, dtype, 16, groups), 0.2, 1 if window else 0, window or -1, 3 if window else 0, hint=1)


@pytest.mark.parametrize("window,sinks", [(0, 0), (200, 4)])
def test_long_chunks_behind_prefixes(env, window, sinks):
    # more tokens than a block of the plan places; prefixes that the window leaves
    b = Batch([(250, [(40, 1300), (900, 1)]), (60, [(0, 70), (5, 1)])], 2, 1, 64, "bf16", 16, 14, pad=9)
    attend(env, b, 0.125, 1 if window else 0, window or -1, sinks)


def test_positions_for_plans_in_memory(env):
    # few rows alone, under a window, in f32
    b = Batch([(40, [(i % 30, 1) for i in range(900)]), (17, [(i % 3, 1) for i in range(300)])], 2, 1, 64, "f32", 16, 15)
    pa = env[0]
    t, lse = b.tensors(pa)
    k = pa.Kernels.SharedPrefixAttention(*t, scale=0.2, mask=pa.AttentionMask.causal_sliding_window(25), sinks=1, lse=lse)
    assert k.function_names[:2] == ["shared_prefix_positions", "shared_prefix_plan"]
    attend(env, b, 0.2, 1, 25, 1, hint=1)


@pytest.mark.parametrize("dtype,hd", [("bf16", 64), ("f16", 256), ("f32", 64), ("bf16", 36)])
def test_starts_and_groups_out_of_order(env, dtype, hd):
    # what they give is not said, but it stays within the tensors: tables, caches and what lies around the outputs are as they were
    pa, _, stream, enc = env
    g = np.random.default_rng(16)
    for i in range(6):
        b = Batch([(40, [(7, 3)] * 5), (70, [(20, 9)] * 4), (None, [(2, 2)])], 4, 2, hd, dtype, 16, 16, pad=4)
        b.starts = g.permutation(b.starts) if i % 2 else g.integers(-5, 80, b.starts.size)
        b.group_starts = list(g.integers(-3, 14, len(b.group_starts)))
        b.prefix_lens = [int(x) for x in g.integers(-9, 2000, len(b.prefix_lens))]
        b.keys = g.integers(-9, 300, b.keys.size)
        for window in (0, 33):
            t, lse = b.tensors(pa)
            T, nq = b.q.shape[:2]
            big, logs = upload(pa, np.full((T + 64, nq, hd), 5.0), dtype), upload(pa, np.full((T + 64, nq), 5.0), "f32")
            size = 4 if dtype == "f32" else 2
            out = pa.Tensor(big.ptr + 32 * nq * hd * size, (T, nq, hd), dtype, owner=big)
            lse = pa.Tensor(logs.ptr + 32 * nq * 4, (T, nq), "f32", owner=logs)
            mask = pa.AttentionMask.causal_sliding_window(window) if window else pa.AttentionMask.causal
            enc.encode(pa.Kernels.SharedPrefixAttention(*t[:9], out, scale=0.1, mask=mask, lse=lse))
            stream.synchronize()
            for x in (download(big, stream), download(logs, stream)):
                assert (x[:32] == 5.0).all() and (x[32 + T:] == 5.0).all()
