"""GPU tests of a server's steps over shared prefixes with a bounded cache: tables, the new rows' write, attention with its
logarithms, the keys' weights, and now and then an eviction in every layer and the release of its pages; eagerly, from captured
graphs, and two servers at once."""
import numpy as np
import pytest

import cache_ref as C
import oracle as O
import serving_ref as R
from gpu_util import download, gpu_env, rounded, upload
from test_gpu_serving import Graph

pytestmark = pytest.mark.gpu

NQ, NKV, HD, PAGE, LAYERS = 8, 2, 64, 16, 2
PREFIXES, GROUPS = [70, 33], [0, 2, 4]  # the last request has none
BUDGETS, FIRST, LAST = [40, 24, 64, 17, 33], 2, 6
SCALE = float(np.float32(0.15))


@pytest.fixture(scope="module")
def env():
    return gpu_env()


def i32(pa, x):
    return pa.Tensor.from_numpy(np.asarray(x, np.int32), "i32")


class Server:
    def __init__(self, pa, stream, seed, requests=5, tokens=150, pages=70, columns=14):
        self.pa, self.stream, self.g = pa, stream, np.random.default_rng(seed)
        g, K = self.g, pa.Kernels
        ids = list(g.permutation(pages))
        held = [-(-n // PAGE) for n in PREFIXES]
        self.prefix_tables = np.full((len(PREFIXES), max(held)), -1, np.int64)
        for i, h in enumerate(held):
            self.prefix_tables[i, :h] = [ids.pop() for _ in range(h)]
        self.free, self.past, self.columns, self.T = ids, np.zeros(requests, np.int64), columns, tokens
        self.tables = np.full((requests, columns), -1, np.int64)
        shape = (pages, NKV, PAGE, HD)
        # nothing is known of pages that hold no key
        self.k, self.v = ([np.full(shape, np.nan, np.float32) for _ in range(LAYERS)] for _ in range(2))
        for x in self.k + self.v:
            for row, n in zip(self.prefix_tables, PREFIXES):
                for j in range(n):
                    x[row[j // PAGE], :, j % PAGE] = rounded(g.standard_normal((NKV, HD)), "bf16")
        self.caches = [[upload(pa, x, "bf16") for x in xs] for xs in (self.k, self.v)]
        self.d = {n: i32(pa, np.zeros(s)) for n, s in dict(past=requests, new=requests, free=pages, starts=requests + 1, keys=requests,
                                                           positions=tokens, slots=tokens, counts=2, lens=requests, gone=1,
                                                           freed=requests * columns).items()}
        self.d.update(tables=i32(pa, self.tables), budgets=i32(pa, BUDGETS), prefix=i32(pa, self.prefix_tables), prefix_lens=i32(pa, PREFIXES),
                      groups=i32(pa, GROUPS))
        room = (requests, NKV, columns * PAGE)
        self.layers = []
        d = self.d
        for i in range(LAYERS):
            L = {n: upload(pa, np.zeros((tokens, h, HD)), "bf16") for n, h in (("q", NQ), ("k", NKV), ("v", NKV), ("out", NQ))}
            L["lse"] = upload(pa, np.zeros((tokens, NQ)), "f32")
            L["weights"] = [upload(pa, np.zeros(room), "f32") for _ in range(2)]
            L["kept"] = i32(pa, np.full(room, -7))
            L["now"] = np.zeros(room, np.float32)
            self.layers.append(L)
        self.side = 0  # which of the two weights is current
        self.step_kernels, self.evict_kernels = [], []
        for side in range(2):
            step = [K.PageTables(d["past"], d["new"], d["free"], d["tables"], page_size=PAGE, query_starts=d["starts"], key_lens=d["keys"],
                                 positions=d["positions"], slots=d["slots"], counts=d["counts"])]
            evict = []
            for i, L in enumerate(self.layers):
                kc, vc = self.caches[0][i], self.caches[1][i]
                step += [K.PagedKVCacheWrite(L["k"], L["v"], d["slots"], kc, vc),
                         K.SharedPrefixAttention(L["q"], kc, vc, d["prefix"], d["prefix_lens"], d["groups"], d["tables"], d["starts"], d["keys"],
                                                 L["out"], scale=SCALE, lse=L["lse"]),
                         K.PagedAttentionWeights(L["q"], kc, d["tables"], d["starts"], d["keys"], L["lse"], L["weights"][side], scale=SCALE)]
                evict += [K.PagedEviction(L["weights"][side], kc, vc, d["tables"], d["keys"], d["budgets"], L["kept"], L["weights"][1 - side],
                                          first=FIRST, last=LAST)]
            evict.append(K.ReleasePages(d["keys"], d["budgets"], d["tables"], page_size=PAGE, new_lens=d["lens"], freed=d["freed"],
                                        counts=d["gone"]))
            self.step_kernels.append(step)
            self.evict_kernels.append(evict)

    def feed(self, new):
        g, s, T = self.g, self.stream, self.T
        self.want = R.page_tables(self.past, np.asarray(new), np.array(self.free), self.tables, PAGE, T)
        self.tables = self.want[0]
        self.before = []
        for i, L in enumerate(self.layers):
            x = {n: rounded(g.standard_normal((T, h, HD)) * (2 if n == "q" else 1), "bf16") for n, h in
                 (("q", NQ), ("k", NKV), ("v", NKV), ("out", NQ))}
            for n, a in x.items():
                L[n].copy_from(O.to_bits(a, O.BF16), s)
            old = g.random((T, NQ)).astype(np.float32)
            L["lse"].copy_from(old, s)
            for cache, rows in ((self.k[i], x["k"]), (self.v[i], x["v"])):
                for t, slot in enumerate(self.want[4]):
                    if slot >= 0:
                        cache[slot // PAGE, :, slot % PAGE] = rows[t]
            self.before.append((x, old))
        for n, a in (("past", self.past), ("new", new), ("free", self.free + [-1] * (70 - len(self.free)))):
            self.d[n].copy_from(np.asarray(a, np.int32), s)

    def check(self):
        s, d = self.stream, self.d
        for n, a in zip(("tables", "starts", "keys", "positions", "slots", "counts"), self.want):
            np.testing.assert_array_equal(d[n].numpy(s), a)
        starts, keys = self.want[1], self.want[2]
        for i, (L, (x, old)) in enumerate(zip(self.layers, self.before)):
            out, lse, parts = C.shared_attention(x["q"], self.k[i], self.v[i], self.prefix_tables, PREFIXES, GROUPS, self.tables, starts, keys,
                                                 x["out"], old, SCALE)
            got, logs = download(L["out"], s), download(L["lse"], s)
            assert (np.abs(got - out) <= C.attention_bound(out, parts, "bf16", HD)).all()
            assert (np.abs(logs - lse) <= C.lse_bound(lse, parts, HD)).all()
            want, bound = C.weights(x["q"], self.k[i], self.tables, starts, keys, logs.astype(np.float32), L["now"], SCALE)
            L["now"] = download(L["weights"][self.side], s).astype(np.float32)
            assert (np.abs(L["now"] - want) <= bound).all()
        used = self.want[5][1]
        self.free, self.past = self.free[used:], keys.copy()

    def check_eviction(self):
        s, d = self.stream, self.d
        for i, L in enumerate(self.layers):
            kept, weights, self.k[i], self.v[i], lens = C.evict(L["now"], self.k[i], self.v[i], self.tables, self.past, BUDGETS,
                                                                L["kept_before"], FIRST, LAST)
            np.testing.assert_array_equal(L["kept"].numpy(s), kept)
            L["now"] = download(L["weights"][1 - self.side], s).astype(np.float32)
            np.testing.assert_array_equal(L["now"], weights)
            np.testing.assert_array_equal(download(self.caches[0][i], s), self.k[i])
            np.testing.assert_array_equal(download(self.caches[1][i], s), self.v[i])
        new, freed, n = C.release(self.past, BUDGETS, self.tables, PAGE, np.zeros(self.tables.size))
        np.testing.assert_array_equal(d["lens"].numpy(s), new)
        assert list(d["gone"].numpy(s)) == [n]
        np.testing.assert_array_equal(d["freed"].numpy(s)[:n], freed[:n])
        self.free += [int(x) for x in freed[:n]]
        self.past, self.side = new.astype(np.int64), 1 - self.side

    def hold(self):
        for L in self.layers:
            L["kept_before"] = L["kept"].numpy(self.stream).astype(np.int64)


STEPS = [[60, 0, 20, 1, 50], [1, 30, 1, 0, 1], "evict", [1, 1, 1, 1, 1], [2, 1, 40, 1, 1], "evict", [0, 1, 0, 0, 5], "evict", [1, 1, 1, 1, 1]]


def test_steps(env):
    pa, lib, stream, enc = env
    server = Server(pa, stream, 1)
    for new in STEPS:
        if new == "evict":
            server.hold()
            enc.encode(server.evict_kernels[server.side])
            stream.synchronize()
            server.check_eviction()
        else:
            server.feed(new)
            enc.encode(server.step_kernels[server.side])
            stream.synchronize()
            server.check()


def test_steps_from_graphs(env):
    # captured once, replayed with other lengths, with eager work of another server between the replays
    pa, lib, _, _ = env
    stream = pa.Stream()
    enc = pa.KernelCommandEncoder(lib, stream)
    server, other = Server(pa, stream, 2), Server(pa, stream, 3)
    step = [Graph(pa, stream, lambda: enc.encode(server.step_kernels[i])) for i in range(2)]
    evict = [Graph(pa, stream, lambda: enc.encode(server.evict_kernels[i])) for i in range(2)]
    for new in STEPS:
        for who, run in ((server, [g.launch for g in (step if new != "evict" else evict)]),
                         (other, [lambda i=i: enc.encode((other.step_kernels if new != "evict" else other.evict_kernels)[i]) for i in range(2)])):
            if new == "evict":
                who.hold()
            else:
                who.feed(new)
            run[who.side]()
            stream.synchronize()
            who.check_eviction() if new == "evict" else who.check()
    for graph in step + evict:
        graph.close()


def test_steps_on_two_streams(env):
    # an encoder (and its scratch) per stream
    pa, lib, _, _ = env
    streams = [pa.Stream() for _ in range(2)]
    encs = [pa.KernelCommandEncoder(lib, s) for s in streams]
    servers = [Server(pa, s, 4 + i) for i, s in enumerate(streams)]
    for new in STEPS:
        for s in servers:
            s.hold() if new == "evict" else s.feed(new)
        for s, e in zip(servers, encs):
            e.encode((s.evict_kernels if new == "evict" else s.step_kernels)[s.side])
        for s, t in zip(servers, streams):
            t.synchronize()
            s.check_eviction() if new == "evict" else s.check()
