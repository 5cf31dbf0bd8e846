"""CPU tests of the descriptors of shared prefixes, attention weights, eviction and page release: what they refuse, and
their index arithmetic, compiled for the host, over bad lengths."""
import ctypes
import itertools
import os
import subprocess

import numpy as np
import pytest

import popcorn_amd as pa
import serving_ref
from test_serving_abi import LENGTHS, ROOT, E, T, refused

WINDOW = pa.AttentionMask.causal_sliding_window(8)


def share(q=(6, 4, 64), cache=(9, 2, 16, 64), vcache=None, prefix=(2, 7), plens=(2,), groups=(3,), table=(3, 5), starts=(4,), lens=(3,),
          out=None, lse=(6, 4), t="bf16", kt=None, ot=None, it="i32", lt="f32", qptr=None, pt="i32", **kw):
    kw.setdefault("scale", 0.125)
    opt = [x and T(x, pt) for x in (prefix, plens, groups)]
    return pa.Kernels.SharedPrefixAttention(T(q, t, qptr), T(cache, kt or t), T(vcache or cache, kt or t), *opt, T(table, it), T(starts, "i32"),
                                            T(lens, "i32"), T(out or q, ot or t), lse=lse and T(lse, lt), **kw)


def test_shared_prefix_refusals():
    for t in ("f32", "f16", "bf16"):
        assert all(n.startswith("shared_prefix_") for n in share(t=t).function_names)
    share(lse=None)
    share(prefix=None, plens=None, groups=None)
    share(prefix=(0, 7), plens=(0,), groups=(1,))
    share(sinks=4, mask=WINDOW)
    for kw in (dict(t="i32"), dict(kt="f16"), dict(ot="f32"), dict(it="i64"), dict(lt="bf16"), dict(pt="f32")):
        refused(E.UNSUPPORTED_DATA_TYPE_COMBINATION, share, **kw)
    for kw in (dict(q=(6, 3, 64)), dict(q=(6, 4, 32)), dict(cache=(9, 2, 24, 64)), dict(vcache=(8, 2, 16, 64)), dict(starts=(3,)), dict(lens=(4,)),
               dict(out=(5, 4, 64)), dict(q=(6, 4, 520), cache=(9, 2, 16, 520)), dict(lse=(6, 2)), dict(plens=(3,)), dict(groups=(2,)),
               dict(q=(2 ** 22, 4, 64), lse=(2 ** 22, 4)), dict(prefix=(2 ** 31 - 4, 0), plens=(2 ** 31 - 4,), groups=(2 ** 31 - 3,))):
        refused(E.TENSOR_SHAPE_MISMATCH, share, **kw)
    for kw in (dict(prefix=(14,)), dict(q=(1, 6, 4, 64)), dict(lse=(24,)), dict(plens=(2, 1)), dict(groups=(3, 1))):
        refused(E.TENSOR_INVALID_RANK, share, **kw)
    for kw in (dict(qptr=0), dict(mask=pa.AttentionMask(3)), dict(sinks=4), dict(sinks=-1, mask=WINDOW), dict(max_query_len=-1),
               dict(prefix=None), dict(plens=None), dict(groups=None), dict(prefix=None, plens=None)):
        refused(E.INVALID_ARGUMENT, share, **kw)


def test_shared_prefix_kernels():
    def kinds(R, tokens, nq, nkv, hd, hint=1, t="bf16", groups=True, **kw):
        k = share(q=(tokens, nq, hd), cache=(9, nkv, 16, hd), table=(R, 5), starts=(R + 1,), lens=(R,), lse=(tokens, nq), t=t, max_query_len=hint,
                  **({} if groups else dict(prefix=None, plens=None, groups=None)), **kw)
        return {n.split("_")[2] for n in k.function_names} - {"merge"}

    # a group's rows are one request's: many of them are tiles, whatever the requests bring
    assert kinds(64, 64, 8, 2, 128) == {"plan", "both"} and kinds(64, 64, 8, 2, 128, groups=False) == {"few"}
    assert kinds(8, 8, 8, 2, 128) == {"few"} and kinds(33, 33, 8, 2, 128) == {"plan", "both"} and kinds(17, 17, 8, 2, 256) == {"plan", "few", "many"}
    for kw in (dict(t="f32"), dict(scale=0.0), dict(scale=float("nan")), dict()):
        assert kinds(64, 64, 8, 2, 128 if kw else 512, **kw) == {"few"}
    assert kinds(64, 64, 8, 2, 36) == {"plain"}
    assert kinds(64, 64, 8, 2, 128, mask=WINDOW) == {"plan", "both"} and kinds(8, 8, 8, 2, 128, mask=WINDOW) == {"positions", "few"}
    assert kinds(64, 64, 8, 2, 128, mask=WINDOW, groups=False) == {"few"}
    assert kinds(1100, 1100, 8, 2, 128, t="f32") == {"plan", "few"}  # (more than a block lays out)


def weigh(q=(6, 4, 64), cache=(9, 2, 16, 64), table=(3, 5), starts=(4,), lens=(3,), lse=(6, 4), weights=(3, 2, 80), t="bf16", kt=None, lt="f32",
          wt="f32", it="i32", wptr=None, **kw):
    kw.setdefault("scale", 0.125)
    return pa.Kernels.PagedAttentionWeights(T(q, t), T(cache, kt or t), T(table, it), T(starts, "i32"), T(lens, "i32"), T(lse, lt),
                                            T(weights, wt, wptr), **kw)


def test_weights_refusals():
    for t in ("f32", "f16", "bf16"):
        assert all(n.startswith("attention_weights_") for n in weigh(t=t).function_names)
    weigh(mask=pa.AttentionMask.bidirectional, last_rows=5)
    for kw in (dict(t="i32"), dict(kt="f16"), dict(it="i64"), dict(lt="bf16"), dict(wt="f16")):
        refused(E.UNSUPPORTED_DATA_TYPE_COMBINATION, weigh, **kw)
    for kw in (dict(q=(6, 3, 64)), dict(cache=(9, 2, 24, 64)), dict(starts=(3,)), dict(lse=(6, 3)), dict(weights=(3, 2, 79)), dict(weights=(3, 4, 80)),
               dict(weights=(2, 2, 80)), dict(q=(6, 4, 520), cache=(9, 2, 16, 520)), dict(q=(2 ** 22, 4, 64), lse=(2 ** 22, 4))):
        refused(E.TENSOR_SHAPE_MISMATCH, weigh, **kw)
    refused(E.TENSOR_INVALID_RANK, weigh, weights=(6, 80))
    for kw in (dict(mask=WINDOW), dict(mask=pa.AttentionMask(3)), dict(last_rows=-1), dict(max_query_len=-1), dict(wptr=0)):
        refused(E.INVALID_ARGUMENT, weigh, **kw)


def evict(weights=(3, 2, 80), k=(9, 2, 16, 64), v=None, table=(3, 5), lens=(3,), budgets=(3,), kept=(3, 2, 80), kept_w=(3, 2, 80), t="bf16", vt=None,
          wt="f32", it="i32", kt="i32", kw_t="f32", ptr=None, **kw):
    return pa.Kernels.PagedEviction(T(weights, wt), T(k, t, ptr), T(v or k, vt or t), T(table, it), T(lens, "i32"), T(budgets, "i32"), T(kept, kt),
                                    T(kept_w, kw_t), **kw)


def test_eviction_refusals():
    big = 2 ** 31
    assert evict(first=4, last=big - 1).function_names == ["evict_select", "evict_move_b128"]
    assert evict(k=(9, 2, 16, 12)).function_names[1] == "evict_move_b64"
    assert evict(k=(9, 2, 16, 2)).function_names[1] == "evict_move_b32"
    assert evict(k=(9, 2, 16, 7)).function_names[1] == "evict_move_b16"
    assert evict(ptr=0x7F0000000002 + (99 << 44)).function_names[1] == "evict_move_b16"
    evict(k=(9, 2, 5, 64), weights=(3, 2, 25), kept=(3, 2, 25), kept_w=(3, 2, 25))  # (pages of any size)
    for kw in (dict(t="i32"), dict(vt="f16"), dict(wt="bf16"), dict(it="i64"), dict(kt="f32"), dict(kw_t="i32")):
        refused(E.UNSUPPORTED_DATA_TYPE_COMBINATION, evict, **kw)
    for kw in (dict(weights=(3, 2, 79)), dict(kept=(3, 1, 80)), dict(kept_w=(2, 2, 80)), dict(v=(8, 2, 16, 64)), dict(lens=(4,)), dict(budgets=(2,)),
               dict(k=(9, 2, 0, 64)), dict(table=(3, 2 ** 27)), dict(k=(9, 2, 16, 2 ** 20))):
        refused(E.TENSOR_SHAPE_MISMATCH, evict, **kw)
    refused(E.TENSOR_INVALID_RANK, evict, k=(9, 16, 64))
    for kw in (dict(first=-1), dict(last=-1), dict(first=big), dict(last=big), dict(ptr=0)):
        refused(E.INVALID_ARGUMENT, evict, **kw)


def release(lens=(3,), budgets=(3,), table=(3, 5), new=(3,), freed=(15,), counts=(1,), it="i32", page_size=16):
    return pa.Kernels.ReleasePages(T(lens, it), T(budgets, "i32"), T(table, "i32"), page_size=page_size, new_lens=T(new, "i32"),
                                   freed=T(freed, "i32"), counts=T(counts, "i32"))


def test_release_refusals():
    assert release().function_names == ["release_pages"]
    release(page_size=7)
    refused(E.UNSUPPORTED_DATA_TYPE_COMBINATION, release, it="f32")
    for kw in (dict(lens=(4,)), dict(budgets=(2,)), dict(new=(2,)), dict(freed=(14,)), dict(counts=(2,)), dict(page_size=2 ** 30)):
        refused(E.TENSOR_SHAPE_MISMATCH, release, **kw)
    refused(E.TENSOR_INVALID_RANK, release, table=(15,))
    for size in (0, -1, 2 ** 31):
        refused(E.INVALID_ARGUMENT, release, page_size=size)


def test_overlaps_are_refused():
    K = pa.Kernels
    f = lambda: T([3, 2, 80], "f32")  # noqa: E731
    i = lambda n=3: T([n], "i32")  # noqa: E731
    shapes = dict(weights=([3, 2, 80], "f32"), k=([9, 2, 16, 64], "bf16"), v=([9, 2, 16, 64], "bf16"), table=([3, 5], "i32"), lens=([3], "i32"),
                  budgets=([3], "i32"), kept=([3, 2, 80], "i32"), kept_w=([3, 2, 80], "f32"))
    outputs = {"k", "v", "kept", "kept_w"}
    for a, b in itertools.combinations(shapes, 2):
        ptr = T([1], "f32").ptr
        args = [T(*shapes[n], *([ptr] if n in (a, b) else [])) for n in shapes]
        if {a, b} & outputs:
            refused(E.INVALID_ARGUMENT, K.PagedEviction, *args)
        else:
            K.PagedEviction(*args)
    q, cache, lse = T([6, 4, 64]), T([9, 2, 16, 64]), T([6, 4], "f32")
    common = [T([3, 5], "i32"), i(4), i()]
    for kw in (dict(out=q), dict(out=T([6, 4, 64], ptr=cache.ptr)), dict(lse=T([6, 4], "f32", q.ptr))):
        refused(E.INVALID_ARGUMENT, K.SharedPrefixAttention, q, cache, cache, T([1, 2], "i32"), i(1), i(2), *common, kw.get("out", T([6, 4, 64])),
                scale=1.0, lse=kw.get("lse", lse))
    out = T([6, 4, 64])
    refused(E.INVALID_ARGUMENT, K.SharedPrefixAttention, q, cache, cache, T([1, 2], "i32"), i(1), i(2), *common, out, scale=1.0,
            lse=T([6, 4], "f32", out.ptr))
    refused(E.INVALID_ARGUMENT, K.SharedPrefixAttention, q, cache, cache, T([1, 2], "i32", out.ptr), i(1), i(2), *common, out, scale=1.0)
    for other in (q, cache, lse):
        refused(E.INVALID_ARGUMENT, K.PagedAttentionWeights, q, cache, *common, lse, T([3, 2, 80], "f32", other.ptr), scale=1.0)
    K.PagedAttentionWeights(q, cache, *common, lse, f(), scale=1.0)
    lens = i()
    for n in ("new_lens", "freed", "counts"):
        kw = dict(new_lens=i(), freed=i(15), counts=i(1))
        kw[n] = T(kw[n].shape, "i32", lens.ptr)
        refused(E.INVALID_ARGUMENT, K.ReleasePages, lens, i(), T([3, 5], "i32"), page_size=16, **kw)


def test_null_arguments():
    lib, h, mask = pa.lib(), ctypes.c_void_p(), pa.AttentionMask(0).desc()
    d = [ctypes.byref(T([3], "i32").desc()) for _ in range(11)]
    assert lib.popcorn_kernel_shared_prefix_attention(None, *d[:10], 1.0, mask, 0, 0, ctypes.byref(h)) == E.INVALID_ARGUMENT
    assert lib.popcorn_kernel_paged_attention_weights(*d[:6], None, 1.0, mask, 0, 0, ctypes.byref(h)) == E.INVALID_ARGUMENT
    assert lib.popcorn_kernel_paged_eviction(*d[:7], None, 0, 0, ctypes.byref(h)) == E.INVALID_ARGUMENT
    assert lib.popcorn_kernel_release_pages(*d[:3], 16, None, *d[:2], ctypes.byref(h)) == E.INVALID_ARGUMENT
    assert h.value is None


HOST = r"""
#include <cstdint>
#include "paged.hpp"
static PagedAttentionConstants P(uint32_t T, uint32_t R, uint32_t columns, uint32_t page, uint32_t kind, int32_t window, uint32_t sinks) {
    PagedAttentionConstants p{};
    p.T = T, p.R = R, p.Nq = 4, p.Nkv = 2, p.columns = columns, p.pageSize = page, p.maskKind = kind, p.slidingWindow = window, p.sinks = sinks;
    return p;
}
// out: prefix, start, n, pos0, keys, before, then r0, r1, sinks, first, n of the steps of every tile, and their number in front of them
extern "C" int shared(uint32_t v, const int32_t *starts, const int32_t *keyLens, const int32_t *prefixLens, const int32_t *groupStarts,
                      const int32_t *positions, uint32_t T, uint32_t R, uint32_t columns, uint32_t page, uint32_t groups, uint32_t prefixColumns,
                      uint32_t kind, int32_t window, uint32_t sinks, uint32_t rows, uint32_t step, int32_t *out) {
    const PagedAttentionConstants p = P(T, R, columns, page, kind, window, sinks);
    SharedPrefixConstants s{};
    s.groups = groups, s.columns = prefixColumns, s.windowed = positions != nullptr;
    const pk::SharedRequest q = pk::paged_shared(v, starts, keyLens, prefixLens, groupStarts, positions, p, s);
    out[0] = q.prefix, out[1] = q.start, out[2] = q.n, out[3] = q.pos0, out[4] = q.keys, out[5] = q.before;
    PagedWorkConstants w{};
    w.rows = rows, w.stepKeys = step;
    const uint32_t tiles = ((uint32_t)q.n * 2 + rows - 1) / rows;
    for (uint32_t t = 0; t < tiles; ++t) {
        const pk::PagedSteps x = pk::paged_shared_steps(q, t, p, w);
        int32_t *o = out + 6 + 5 * t;
        o[0] = x.r0, o[1] = x.r1, o[2] = x.sinks, o[3] = x.first, o[4] = x.n;
    }
    return tiles;
}
extern "C" int sees(uint32_t v, const int32_t *starts, const int32_t *keyLens, const int32_t *prefixLens, const int32_t *groupStarts,
                    const int32_t *positions, uint32_t T, uint32_t R, uint32_t columns, uint32_t page, uint32_t groups, uint32_t prefixColumns,
                    uint32_t kind, int32_t window, uint32_t sinks, int32_t pos, int32_t key) {
    const PagedAttentionConstants p = P(T, R, columns, page, kind, window, sinks);
    SharedPrefixConstants s{};
    s.groups = groups, s.columns = prefixColumns, s.windowed = positions != nullptr;
    return pk::paged_sees(pos, key, pk::paged_shared_mask(pk::paged_shared(v, starts, keyLens, prefixLens, groupStarts, positions, p, s), p));
}
extern "C" int place(int32_t start, int32_t pos0, int32_t t, int32_t prefix) {
    pk::PagedRequest r{};
    r.start = start, r.pos0 = pos0;
    return pk::paged_place(r, t, prefix);
}
extern "C" uint32_t span_of(const int32_t *at, uint32_t n, int32_t x) { return pk::paged_span_of(at, n, x); }
extern "C" void keep(int32_t len, int32_t budget, uint32_t columns, uint32_t page, uint32_t first, uint32_t last, uint32_t *out) {
    EvictConstants e{};
    e.columns = columns, e.pageSize = page, e.first = first, e.last = last;
    const pk::EvictKeep k = pk::evict_keep(len, budget, e);
    out[0] = k.keys, out[1] = k.n, out[2] = k.first, out[3] = k.last;
}
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    d = tmp_path_factory.mktemp("shared")
    (d / "h.cpp").write_text(HOST)
    subprocess.run(["g++", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I", os.path.join(ROOT, "include"), "-I",
                    os.path.join(ROOT, "popcorn_amd", "csrc", "kernels"), "-o", str(d / "h.so"), str(d / "h.cpp")], check=True)
    return ctypes.CDLL(str(d / "h.so"))


def ints(x):
    return (ctypes.c_int32 * max(len(x), 1))(*x)


def test_units_stay_in_range(host):
    g = np.random.default_rng(0)
    out = (ctypes.c_int32 * 4000)()
    for _ in range(3000):
        R, G, tokens = int(g.integers(1, 6)), int(g.integers(0, 4)), int(g.integers(1, 60))
        odd = lambda n, hi: [int(g.choice(LENGTHS)) if g.random() < 0.3 else int(g.integers(0, hi)) for _ in range(n)]  # noqa: E731
        starts, lens, plens, groups = odd(R + 1, tokens + 1), odd(R, 90), odd(G, 90), odd(G + 1, R + 1)
        positions = odd(tokens + G, 200)
        kind, window, sinks = int(g.integers(0, 3)), int(g.choice([-5, 0, 1, 20, 2 ** 31 - 1])), int(g.integers(0, 40))
        for v in range(G + R):
            tiles = host.shared(v, ints(starts), ints(lens), ints(plens), ints(groups), ints(positions) if kind == 1 else None, tokens, R, 5, 16, G,
                                4, kind, window, sinks, 32, 16, out)
            prefix, start, n, _, keys, before = out[:6]
            assert prefix == (v < G) and 0 <= start and 0 <= n and start + n <= tokens
            assert 0 <= keys <= (64 if prefix else 80) and 0 <= before <= 64
            assert tiles == -(-2 * n // 32)
            for t in range(tiles):
                r0, r1, s, first, steps = out[6 + 5 * t:11 + 5 * t]
                assert r0 == 32 * t and r0 < r1 <= min(r0 + 32, 2 * n)
                # (the one step of a tile without a visible key may lie behind the keys, where the kernels read none)
                assert 0 <= s <= first and 1 <= steps and ((first + steps - s) * 16 <= max(keys, 1) + 15 or steps == 1 and first * 16 <= keys + 15)


def test_units_hold_every_visible_key(host):
    g = np.random.default_rng(1)
    out = (ctypes.c_int32 * 4000)()
    for _ in range(150):
        R, G = int(g.integers(1, 6)), int(g.integers(1, 3))
        n = g.integers(0, 20, R)
        starts = np.concatenate([[0], np.cumsum(n)])
        lens, plens = [int(x) + int(g.integers(-2, 50)) for x in n], [int(g.integers(0, 65)) for _ in range(G)]
        groups = sorted(int(x) for x in g.integers(0, R + 1, G + 1))
        kind, window, sinks = int(g.integers(0, 3)), int(g.choice([0, 1, 20, 70])), int(g.integers(0, 40))
        tokens = int(starts[-1])
        if tokens == 0:
            continue
        positions, least = [0] * tokens, [2 ** 31 - 1] * G
        group = [next((k for k in range(G) if groups[k] <= r < groups[k + 1]), None) for r in range(R)]
        own = [max(x, 0) for x in lens]
        for r in range(R):
            for t in range(starts[r], starts[r + 1]):
                first = plens[group[r]] if group[r] is not None else 0
                positions[t] = host.place(int(starts[r]), own[r] - int(n[r]), t, first)
                assert positions[t] == first + max(own[r] - n[r] + t - starts[r], 0)
                if group[r] is not None:
                    least[group[r]] = min(least[group[r]], positions[t])
        args = [ints(starts.tolist()), ints(lens), ints(plens), ints(groups), ints(positions + least) if kind == 1 else None, tokens, R, 5, 16, G, 5, kind,
                window, sinks]
        for v in range(G + R):
            tiles = host.shared(v, *args, 32, 16, out)
            prefix, start, m, pos0, keys, before = out[:6]
            for t in range(tiles):
                r0, r1, s, first, steps = out[6 + 5 * t:11 + 5 * t]
                held = set(range(16 * s)) | set(range(16 * first, 16 * (first + steps - s)))
                for row in range(r0, r1):
                    token = start + row // 2
                    r = int(np.searchsorted(starts, token, side="right")) - 1
                    o = own[r] - int(n[r]) + token - int(starts[r])
                    pre = plens[group[r]] if group[r] is not None else 0
                    pos = positions[token] if prefix else pos0 + row // 2
                    if prefix:
                        assert group[r] == v and keys == pre
                        want = [kind != 1 or positions[token] - j < window or j < sinks for j in range(keys)]
                    else:
                        assert r == v - G and before == pre
                        want = [bool(x) and (kind != 1 or o - j < window or pre + j < sinks)
                                for j, x in enumerate(serving_ref.visible(o, keys, 2 if kind == 2 else 0, 0, 0))]
                    got = [bool(host.sees(v, *args, pos, j)) for j in range(keys)]
                    assert got == want
                    assert {j for j in range(keys) if got[j]} <= held


def test_searches(host):
    g = np.random.default_rng(2)
    for n in range(1, 20):
        at = sorted(int(x) for x in g.integers(-3, 15, n + 1))
        for x in range(-5, 20):
            want = [i for i in range(n) if at[i] <= x < at[i + 1]]
            assert host.span_of(ints(at), n, x) == (want[0] if want else n)
    assert host.span_of(ints([]), 0, 3) == 0


def test_what_stays(host):
    out = (ctypes.c_uint32 * 4)()
    for length, budget, first, last in itertools.product(LENGTHS, LENGTHS, (0, 1, 20, 2 ** 31 - 1), (0, 1, 20, 2 ** 31 - 1)):
        host.keep(length, budget, 3, 16, first, last, out)
        keys, n, f, e = out
        assert keys == min(max(length, 0), 48) and n == min(keys, max(budget, 0))
        assert f == min(first, n) and e == min(last, n - f)
