"""GPU tests of the serving operators together, as a step of a server runs them:
tables from the lengths, the new rows into their slots, attention over the pages,
a token from the logits; eagerly, from a captured graph, on two streams at once."""
import ctypes

import numpy as np
import pytest

import serving_ref as R
from gpu_util import download, gpu_env, rounded, upload

pytestmark = pytest.mark.gpu

NQ, NKV, HD, PAGE, VOCAB = 8, 2, 128, 16, 5003


@pytest.fixture(scope="module")
def env():
    return gpu_env()


def i32(pa, x):
    return pa.Tensor.from_numpy(np.asarray(x, np.int32), "i32")


class Server:
    """Caches and tensors of up to `requests` requests and `tokens` new tokens a step, and the step's kernels."""

    def __init__(self, pa, stream, requests, tokens, pages, columns, seed):
        self.pa, self.stream = pa, stream
        self.g = np.random.default_rng(seed)
        self.pages = pages
        self.host_tables = np.full((requests, columns), -1, np.int64)
        self.free = list(self.g.permutation(pages))
        self.past = np.zeros(requests, np.int64)
        shape = [pages, NKV, PAGE, HD]
        self.k_cache, self.v_cache = (upload(pa, np.zeros(shape), "bf16") for _ in range(2))
        self.host = [np.zeros(shape, np.float32) for _ in range(2)]
        self.d = {n: i32(pa, np.zeros(s)) for n, s in dict(past=requests, new=requests, free=pages, tables=(requests, columns),
                                                           starts=requests + 1, keys=requests, positions=tokens, slots=tokens,
                                                           counts=2, tokens=requests).items()}
        self.d["tables"].copy_from(self.host_tables.astype(np.int32))
        self.q, self.out = (upload(pa, np.zeros((tokens, NQ, HD)), "bf16") for _ in range(2))
        self.k, self.v = (upload(pa, np.zeros((tokens, NKV, HD)), "bf16") for _ in range(2))
        self.logits = upload(pa, np.zeros((requests, VOCAB)), "bf16")
        self.u = pa.Tensor.from_numpy(np.zeros(requests, np.float32))
        self.top_p = pa.Tensor.from_numpy(np.full(requests, 0.9, np.float32))
        self.top_k = i32(pa, np.full(requests, 40))
        d, K = self.d, pa.Kernels
        self.kernels = [
            K.PageTables(d["past"], d["new"], d["free"], d["tables"], page_size=PAGE, query_starts=d["starts"], key_lens=d["keys"],
                         positions=d["positions"], slots=d["slots"], counts=d["counts"]),
            K.PagedKVCacheWrite(self.k, self.v, d["slots"], self.k_cache, self.v_cache),
            K.PagedAttention(self.q, self.k_cache, self.v_cache, d["tables"], d["starts"], d["keys"], self.out, scale=0.09,
                             mask=pa.AttentionMask.causal_sliding_window(48), sinks=4),
            K.Sample(self.logits, self.u, d["tokens"], top_k=self.top_k, top_p=self.top_p)]

    def feed(self, new):
        """The step's inputs; what the step has to give."""
        g, past, new = self.g, self.past, np.asarray(new)
        T = self.q.shape[0]
        free = np.array(self.free + [-1] * (self.pages - len(self.free)))
        want = R.page_tables(past, new, np.array(self.free), self.host_tables, PAGE, T)
        x = {n: rounded(g.standard_normal((T, h, HD)), "bf16") for n, h in (("q", NQ), ("k", NKV), ("v", NKV))}
        logits, u, old = rounded(g.standard_normal((len(past), VOCAB)) * 2, "bf16"), g.random(len(past)), rounded(g.standard_normal((T, NQ, HD)), "bf16")
        import oracle as O

        s = self.stream
        for t, a in ((self.q, x["q"]), (self.k, x["k"]), (self.v, x["v"]), (self.logits, logits), (self.out, old)):
            t.copy_from(O.to_bits(a, O.BF16), s)
        self.u.copy_from(u.astype(np.float32), s)
        for n, a in (("past", past), ("new", new), ("free", free)):
            self.d[n].copy_from(a.astype(np.int32), s)
        self.host_tables = want[0]
        for cache, rows in zip(self.host, (x["k"], x["v"])):
            for t, slot in enumerate(want[4]):
                if slot >= 0:
                    cache[slot // PAGE, :, slot % PAGE] = rows[t]
        att, parts = R.attention(x["q"], *self.host, want[0], want[1], want[2], old, float(np.float32(0.09)), 1, 48, 4)
        self.free = self.free[want[5][1]:]
        self.past = past + new
        return want, att, parts, R.sample(logits, u, top_k=np.full(len(past), 40), top_p=np.full(len(past), 0.9))

    def check(self, expected):
        want, att, parts, tokens = expected
        s, d = self.stream, self.d
        for n, a in zip(("tables", "starts", "keys", "positions", "slots", "counts"), want):
            np.testing.assert_array_equal(d[n].numpy(s), a)
        for t, a in zip((self.k_cache, self.v_cache), self.host):
            np.testing.assert_array_equal(download(t, s), a)
        got = download(self.out, s)
        assert (np.abs(got - att) <= R.attention_bound(att, parts, "bf16", HD)).all()
        np.testing.assert_array_equal(d["tokens"].numpy(s), tokens)


STEPS = [[70, 0, 33, 1, 200], [1, 16, 1, 0, 1], [1, 1, 1, 1, 1], [0, 0, 0, 0, 0], [90, 1, 1, 40, 1]]


def test_steps(env):
    pa, lib, stream, enc = env
    server = Server(pa, stream, 5, 310, 60, 24, seed=1)
    for new in STEPS:
        expected = server.feed(new)
        enc.encode(server.kernels)
        stream.synchronize()
        server.check(expected)


class Graph:
    """A capture of `body` on `stream` into an executable graph."""

    def __init__(self, pa, stream, body):
        self.hip = pa.lib()  # the HIP runtime that it is linked to (another package may have loaded one of its own)
        self.stream = ctypes.c_void_p(stream.handle)
        graph, self.exec = ctypes.c_void_p(), ctypes.c_void_p()
        assert self.hip.hipStreamBeginCapture(self.stream, 0) == 0
        body()
        assert self.hip.hipStreamEndCapture(self.stream, ctypes.byref(graph)) == 0
        assert self.hip.hipGraphInstantiate(ctypes.byref(self.exec), graph, None, None, ctypes.c_size_t(0)) == 0
        self.hip.hipGraphDestroy(graph)

    def launch(self):
        assert self.hip.hipGraphLaunch(self.exec, self.stream) == 0

    def close(self):
        self.hip.hipGraphExecDestroy(self.exec)


def test_steps_from_a_graph(env):
    # captured once, replayed with other lengths, with eager work of another server between the replays
    pa, lib, _, _ = env
    stream = pa.Stream()
    enc = pa.KernelCommandEncoder(lib, stream)
    server, other = (Server(pa, stream, 5, 310, 60, 24, seed=s) for s in (2, 3))
    graph = Graph(pa, stream, lambda: enc.encode(server.kernels))
    for new in STEPS:
        expected = server.feed(new)
        graph.launch()
        stream.synchronize()
        server.check(expected)
        expected = other.feed(new[::-1])
        enc.encode(other.kernels)
        stream.synchronize()
        other.check(expected)
    graph.close()


def test_steps_on_two_streams(env):
    # an encoder (and its scratch) per stream: two servers' steps at once
    pa, lib, _, _ = env
    servers = []
    for seed in (4, 5):
        stream = pa.Stream()
        servers.append((Server(pa, stream, 5, 310, 60, 24, seed=seed), pa.KernelCommandEncoder(lib, stream)))
    for new in STEPS:
        expected = [s.feed(new if i else new[::-1]) for i, (s, _) in enumerate(servers)]
        for _ in range(3):  # (a step run again gives the same)
            for s, enc in servers:
                enc.encode(s.kernels)
        for s, _ in servers:
            s.stream.synchronize()
        for e, (s, _) in zip(expected, servers):
            s.check(e)


def test_decoding_agrees_with_the_contiguous_cache(env):
    # one request: FlashAttention over a contiguous cache gives what the pages give
    pa, lib, stream, enc = env
    g = np.random.default_rng(6)
    n, keys = 5, 333
    k, v = (rounded(g.standard_normal((1, NKV, keys, HD)), "bf16") for _ in range(2))
    q = rounded(g.standard_normal((n, NQ, HD)), "bf16")
    pages = -(-keys // PAGE)
    ids = g.permutation(pages)
    paged = []
    for x in (k, v):
        p = np.zeros((pages, NKV, PAGE, HD), np.float32)
        for j in range(keys):
            p[ids[j // PAGE], :, j % PAGE] = x[0, :, j]
        paged.append(upload(pa, p, "bf16"))
    o1, o2 = pa.Tensor.empty([1, NQ, n, HD], "bf16"), pa.Tensor.empty([n, NQ, HD], "bf16")
    enc.encode(pa.Kernels.FlashAttention(upload(pa, q.transpose(1, 0, 2)[None], "bf16"), upload(pa, k, "bf16"), upload(pa, v, "bf16"), out=o1,
                                         scale=0.09, batch=1, query_heads=NQ, kv_heads=NKV, query_len=n, key_len=keys, head_dim=HD),
               pa.Kernels.PagedAttention(upload(pa, q, "bf16"), *paged, i32(pa, [ids]), i32(pa, [0, n]), i32(pa, [keys]), o2, scale=0.09))
    stream.synchronize()
    a, b = download(o1, stream)[0].transpose(1, 0, 2), download(o2, stream)
    # two results within half a step of the value each, and near it before: at most a step of bf16 apart, or two at a border
    assert (np.abs(a - b) <= 2 * 2.0 ** -8 * np.abs(a) + 1e-5).all()


def test_scratch_that_is_refused(env):
    # an allocator with nothing to give: the encode fails with its status, and nothing is left running
    pa, lib, stream, _ = env

    class Nothing(pa.KernelScratchAllocator):
        def borrow(self, length):
            raise MemoryError("none")

    enc = pa.KernelCommandEncoder(lib, stream, Nothing())
    server = Server(pa, stream, 5, 310, 60, 24, seed=7)
    for kernel in server.kernels[2:]:
        with pytest.raises(pa.PopcornError) as e:
            enc.encode(kernel)
        assert e.value.code == pa.PopcornError.TENSOR_ALLOCATION_FAILED
    stream.synchronize()


@pytest.mark.parametrize("room", [15, 3, 0, 26])
def test_step_without_room_for_its_tokens(env, room):
    # T cuts a request: those before it are as in a step with room, nothing of another request is written, and the
    # step run again with room (or with the tokens that had it) gives everything
    pa, lib, stream, enc = env
    K = pa.Kernels
    g = np.random.default_rng(30 + room)
    past, new, columns, pages = np.array([21, 0, 16, 40, 5]), np.array([3, 20, 9, 5, 0]), 5, 40
    total = int(new.sum())
    held = -(-past // PAGE)
    ids = g.permutation(pages)
    table = np.full((5, columns), -1)
    at = 0
    for r in range(5):
        table[r, :held[r]] = ids[at:at + held[r]]
        at += held[r]
    free = ids[at:]
    host = [rounded(g.standard_normal((pages, NKV, PAGE, HD)), "bf16") for _ in range(2)]
    caches = [upload(pa, x, "bf16") for x in host]
    tables = i32(pa, table)
    rows = {n: rounded(g.standard_normal((total, h, HD)), "bf16") for n, h in (("q", NQ), ("k", NKV), ("v", NKV))}
    old = rounded(g.standard_normal((total, NQ, HD)), "bf16")

    def step(T, lens):
        d = [i32(pa, np.full(n, -77)) for n in (6, 5, T, T, 2)]
        q, k, v, out = (upload(pa, x[:T], "bf16") for x in (rows["q"], rows["k"], rows["v"], old))
        enc.encode([K.PageTables(i32(pa, past), i32(pa, lens), i32(pa, free), tables, page_size=PAGE, query_starts=d[0], key_lens=d[1],
                                 positions=d[2], slots=d[3], counts=d[4]),
                    K.PagedKVCacheWrite(k, v, d[3], *caches),
                    K.PagedAttention(q, *caches, tables, d[0], d[1], out, scale=0.09)])
        stream.synchronize()
        return [t.numpy(stream) for t in d], download(out, stream), [download(c, stream) for c in caches], tables.numpy(stream)

    def check(T, lens, upto):
        want = R.page_tables(past, lens, free, table, PAGE, T)
        d, out, cache, got_table = step(T, lens)
        np.testing.assert_array_equal(got_table, want[0])
        for a, b in zip(d, want[1:]):
            np.testing.assert_array_equal(a, b)
        assert d[4][0] == lens.sum()  # what the host looks at
        for x, c, n in zip(host, cache, "kv"):
            w = x.copy()
            for t, s in enumerate(want[4]):
                w[s // PAGE, :, s % PAGE] = rows[n][t]
            np.testing.assert_array_equal(c, w)
        filled = [c.copy() for c in cache]
        att, parts = R.attention(rows["q"][:upto], *filled, want[0], np.minimum(want[1], upto), want[2], old[:upto], float(np.float32(0.09)))
        assert (np.abs(out[:upto] - att) <= R.attention_bound(att, parts, "bf16", HD)).all()

    starts = np.concatenate([[0], np.cumsum(new)])
    check(room, new, int(starts[starts <= room].max()))
    if room:  # the tokens that had room, as a step of their own
        check(room, np.clip(room - starts[:-1], 0, new), room)
    check(total, new, total)


def test_step_to_its_tokens_from_a_graph(env):
    # tables, rows, attention, the last row of each request, logits and tokens in one graph, replayed with other lengths
    pa, lib, _, _ = env
    import oracle as O

    stream = pa.Stream()
    enc = pa.KernelCommandEncoder(lib, stream)
    K, R_, T, H, vocab = pa.Kernels, 5, 310, NQ * HD, 6000
    server, other = (Server(pa, stream, R_, T, 60, 24, seed=s) for s in (8, 9))
    g = np.random.default_rng(10)
    head = rounded(g.standard_normal((vocab, H)) * 0.5, "bf16")
    lm_head, hidden = upload(pa, head, "bf16"), upload(pa, np.zeros((T + 1, H)), "bf16")
    last, logits = pa.Tensor.empty([R_, H], "bf16"), pa.Tensor.empty([R_, vocab], "bf16")
    u, t, m = (pa.Tensor.from_numpy(np.zeros(R_, np.float32)) for _ in range(3))
    d = server.d
    step = [server.kernels[0], server.kernels[1],
            K.PagedAttention(server.q, server.k_cache, server.v_cache, d["tables"], d["starts"], d["keys"],
                             hidden.view([T, NQ, HD], offset_elements=H), scale=0.09),
            K.EmbeddingGather(d["starts"].view([R_], offset_elements=1), hidden, last),
            K.Matmul(last, lm_head, logits, True),
            K.Sample(logits, u, d["tokens"], temperature=t, top_k=server.top_k, top_p=server.top_p, min_p=m)]
    enc.encode(step)  # once before the capture
    graph = Graph(pa, stream, lambda: enc.encode(step))
    for new in STEPS:
        want, _, _, _ = server.feed(new)
        hidden.copy_from(O.to_bits(np.zeros((T + 1, H), np.float32), O.BF16), stream)
        uv, tv, mv = g.random(R_).astype(np.float32), g.uniform(0.5, 2, R_).astype(np.float32), g.uniform(0, 0.02, R_).astype(np.float32)
        for x, a in ((u, uv), (t, tv), (m, mv)):
            x.copy_from(a, stream)
        graph.launch()
        stream.synchronize()
        np.testing.assert_array_equal(d["starts"].numpy(stream), want[1])
        rows, x = download(hidden, stream), download(logits, stream)
        np.testing.assert_array_equal(download(last, stream), rows[want[1][1:]])
        ends = np.flatnonzero(new)
        assert rows[want[1][1:]][ends].any(axis=1).all() and not rows[0].any() and not rows[1 + want[1][-1]:].any()
        exact = rows[want[1][1:]].astype(np.float64) @ head.T.astype(np.float64)
        # sums of H products of 16-bit values in f32, then one rounding
        mag = np.abs(rows[want[1][1:]]).astype(np.float64) @ np.abs(head.T).astype(np.float64)
        assert (np.abs(x - exact) <= 2.0 ** -8 * np.abs(exact) + (H + 1) * 2.0 ** -24 * mag).all()
        options = dict(temperature=tv, top_k=np.full(R_, 40), top_p=np.full(R_, 0.9), min_p=mv)
        np.testing.assert_array_equal(d["tokens"].numpy(stream), R.sample(x, uv, **options))
        expected = other.feed(new[::-1])
        enc.encode(other.kernels)
        stream.synchronize()
        other.check(expected)
    graph.close()
