"""CPU tests of the paged-cache and token-draw descriptors: what they refuse, and
the index arithmetic of the kernels, compiled for the host, over bad lengths."""
import ctypes
import itertools
import os
import subprocess

import numpy as np
import pytest

import popcorn_amd as pa

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FAKE = 0x7F0000000000  # never dereferenced: descriptors only validate
APART = itertools.count(1)  # tensors of up to 2^44 bytes with no byte in common
E = pa.PopcornError


def T(shape, dtype="bf16", ptr=None):
    return pa.Tensor(FAKE + (next(APART) << 44) if ptr is None else ptr, shape, dtype)


def refused(code, fn, *args, **kw):
    with pytest.raises(E) as e:
        fn(*args, **kw)
    assert e.value.code == code, e.value


def tables(**kw):
    a = dict(past=T([3], "i32"), new=T([3], "i32"), free=T([9], "i32"), table=T([3, 4], "i32"), page_size=16,
             query_starts=T([4], "i32"), key_lens=T([3], "i32"), positions=T([7], "i32"), slots=T([7], "i32"), counts=T([2], "i32"))
    a.update(kw)
    return pa.Kernels.PageTables(a.pop("past"), a.pop("new"), a.pop("free"), a.pop("table"), **a)


def test_page_tables_refusals():
    assert tables().function_names == ["page_tables"]
    for name in ("past", "new", "free", "table", "query_starts", "key_lens", "positions", "slots", "counts"):
        shape = {"table": [3, 4], "free": [9], "query_starts": [4], "positions": [7], "slots": [7], "counts": [2]}.get(name, [3])
        refused(E.UNSUPPORTED_DATA_TYPE_COMBINATION, tables, **{name: T(shape, "f32")})
        refused(E.INVALID_ARGUMENT, tables, **{name: T(shape, "i32", 0)})
        refused(E.INVALID_ARGUMENT, tables, **{name: T(shape, "i32", FAKE + 2)})
        refused(E.TENSOR_INVALID_RANK, tables, **{name: T([1] + shape, "i32")})
    for name, shape in (("new", [4]), ("table", [2, 4]), ("query_starts", [3]), ("key_lens", [2]), ("slots", [6]), ("counts", [1])):
        refused(E.TENSOR_SHAPE_MISMATCH, tables, **{name: T(shape, "i32")})
    for size in (0, -16, 2 ** 31):
        refused(E.INVALID_ARGUMENT, tables, page_size=size)
    refused(E.TENSOR_SHAPE_MISMATCH, tables, free=T([2 ** 31], "i32"))


def write(k="bf16", v=None, c="bf16", kshape=(5, 2, 64), vshape=None, slots=(5,), cache=(7, 2, 16, 64), vcache=None, stype="i32"):
    return pa.Kernels.PagedKVCacheWrite(T(kshape, k), T(vshape or kshape, v or k), T(slots, stype), T(cache, c), T(vcache or cache, c))


def test_paged_write_refusals():
    assert [write(a, c=b).function_names[0] for a, b in (("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "bf16"))] == [
        "paged_kv_write_f32", "paged_kv_write_f16", "paged_kv_write_bf16", "paged_kv_write_f32_to_bf16"]
    for a, b in (("bf16", "f32"), ("f16", "bf16"), ("f32", "f16"), ("i32", "i32")):
        refused(E.UNSUPPORTED_DATA_TYPE_COMBINATION, write, a, c=b)
    refused(E.UNSUPPORTED_DATA_TYPE_COMBINATION, write, "bf16", v="f16")
    refused(E.UNSUPPORTED_DATA_TYPE_COMBINATION, write, stype="i64")
    for kw in (dict(kshape=(5, 3, 64)), dict(kshape=(5, 2, 32)), dict(vshape=(4, 2, 64)), dict(slots=(4,)), dict(vcache=(8, 2, 16, 64)),
               dict(cache=(7, 2, 0, 64)), dict(cache=(2 ** 28, 2, 16, 64))):
        refused(E.TENSOR_SHAPE_MISMATCH, write, **kw)
    refused(E.TENSOR_INVALID_RANK, write, kshape=(5, 128))
    refused(E.TENSOR_INVALID_RANK, write, cache=(7, 16, 64))


def attend(q=(6, 4, 64), cache=(9, 2, 16, 64), vcache=None, table=(3, 5), starts=(4,), lens=(3,), out=None, t="bf16", kt=None, ot=None,
           it="i32", qptr=None, **kw):
    kw.setdefault("scale", 0.125)
    return pa.Kernels.PagedAttention(T(q, t, qptr), T(cache, kt or t), T(vcache or cache, kt or t), T(table, it), T(starts, "i32"),
                                     T(lens, "i32"), T(out or q, ot or t), **kw)


def test_paged_attention_refusals():
    for t in ("f32", "f16", "bf16"):
        assert all(n.startswith("paged_") for n in attend(t=t).function_names)
    refused(E.UNSUPPORTED_DATA_TYPE_COMBINATION, attend, t="i32")
    refused(E.UNSUPPORTED_DATA_TYPE_COMBINATION, attend, kt="f16")
    refused(E.UNSUPPORTED_DATA_TYPE_COMBINATION, attend, ot="f32")
    refused(E.UNSUPPORTED_DATA_TYPE_COMBINATION, attend, it="i64")
    for kw in (dict(q=(6, 3, 64)), dict(q=(6, 4, 32)), dict(cache=(9, 2, 24, 64)), dict(cache=(9, 2, 0, 64)), dict(vcache=(8, 2, 16, 64)),
               dict(starts=(3,)), dict(lens=(4,)), dict(out=(5, 4, 64)), dict(q=(6, 4, 520), cache=(9, 2, 16, 520)),
               dict(q=(6, 0, 64)), dict(cache=(9, 0, 16, 64)), dict(q=(6, 4, 0), cache=(9, 2, 16, 0)), dict(q=(2 ** 29, 4, 64))):
        refused(E.TENSOR_SHAPE_MISMATCH, attend, **kw)
    refused(E.TENSOR_INVALID_RANK, attend, q=(1, 6, 4, 64))
    refused(E.TENSOR_INVALID_RANK, attend, cache=(9, 16, 64))
    refused(E.TENSOR_INVALID_RANK, attend, table=(15,))
    refused(E.INVALID_ARGUMENT, attend, qptr=0)
    refused(E.INVALID_ARGUMENT, attend, mask=pa.AttentionMask(3))
    refused(E.INVALID_ARGUMENT, attend, sinks=4)
    refused(E.INVALID_ARGUMENT, attend, sinks=-1, mask=pa.AttentionMask.causal_sliding_window(8))
    refused(E.INVALID_ARGUMENT, attend, max_query_len=-1)
    attend(sinks=4, mask=pa.AttentionMask.causal_sliding_window(8))


def test_paged_attention_kernels():
    def kinds(R, T, nq, nkv, hd, hint, t="bf16", scale=0.1):
        k = attend(q=(T, nq, hd), cache=(9, nkv, 16, hd), table=(R, 5), starts=(R + 1,), lens=(R,), t=t, max_query_len=hint, scale=scale)
        return {n.split("_")[2] for n in k.function_names if n.split("_")[1] == "attention"} - {"merge"}

    assert kinds(8, 8, 8, 2, 128, 1) == {"few"}  # decode
    assert kinds(8, 72, 8, 2, 128, 9) == {"tile"}  # 36 rows of one request
    assert kinds(8, 72, 8, 2, 128, 8) == {"few"}
    assert kinds(1, 32, 8, 2, 128, 32) == {"few"} and kinds(1, 33, 8, 2, 128, 33) == {"tile"}
    assert kinds(1, 16, 8, 2, 256, 16) == {"few"} and kinds(1, 17, 8, 2, 256, 17) == {"tile"}
    assert kinds(257, 300, 8, 2, 128, 40) == {"few", "tile"} and kinds(256, 300, 8, 2, 128, 40) == {"tile"}
    assert kinds(129, 300, 8, 2, 256, 40) == {"few", "tile"} and kinds(128, 300, 8, 2, 256, 40) == {"tile"}
    for kw in (dict(t="f32"), dict(scale=0.0), dict(scale=float("nan"))):
        assert kinds(4, 500, 8, 2, 128, 200, **kw) == {"few"}
    assert kinds(4, 500, 8, 2, 512, 200) == {"few"}
    for t, hd, rows in (("f32", 256, "r1"), ("f32", 128, "r2"), ("bf16", 256, "r2"), ("f16", 512, "r1")):
        names = attend(q=(32, 8, hd), cache=(9, 2, 16, hd), table=(4, 5), starts=(5,), lens=(4,), t=t, max_query_len=8).function_names
        assert names[0].endswith(f"_d{hd}_{rows}")
    assert kinds(4, 500, 8, 2, 36, 200) == {"plain"}


def draw(logits=(3, 100), t="f32", rows=3, ut="f32", kt="i32", **kw):
    o = dict(temperature=T([3], "f32"), top_k=T([3], kt), top_p=T([3], "f32"), min_p=T([3], "f32"))
    o.update(kw)
    return pa.Kernels.Sample(T(logits, t), T([rows], ut), T([3], "i32"), **o)


def test_sample_refusals():
    for t in ("f32", "f16", "bf16"):
        assert all(n.startswith("sample_") for n in draw(t=t).function_names)
    draw(temperature=None, top_k=None, top_p=None, min_p=None)
    refused(E.UNSUPPORTED_DATA_TYPE_COMBINATION, draw, t="i32")
    refused(E.UNSUPPORTED_DATA_TYPE_COMBINATION, draw, ut="bf16")
    refused(E.UNSUPPORTED_DATA_TYPE_COMBINATION, draw, kt="f32")
    refused(E.TENSOR_SHAPE_MISMATCH, draw, rows=2)
    refused(E.TENSOR_SHAPE_MISMATCH, draw, top_p=T([1], "f32"))
    refused(E.TENSOR_SHAPE_MISMATCH, draw, logits=(3, 0))
    refused(E.TENSOR_SHAPE_MISMATCH, draw, logits=(3, 2 ** 22 + 1))
    refused(E.TENSOR_INVALID_RANK, draw, logits=(300,))
    refused(E.INVALID_ARGUMENT, draw, min_p=T([3], "f32", 0))


def test_sample_launches():
    none = dict(temperature=None, top_k=None, top_p=None, min_p=None)
    t, k = T([3], "f32"), T([3], "i32")

    def names(**kw):
        return [n.split("_")[1] for n in draw(logits=(3, 50000), **dict(none, **kw)).function_names]

    # the histogram serves top-k and top-p alone
    for kw in ({}, dict(temperature=t), dict(min_p=t), dict(temperature=t, min_p=T([3], "f32"))):
        assert names(**kw) == ["top", "gather", "finish"]
    for kw in (dict(top_k=k), dict(top_p=t), dict(temperature=t, top_k=k)):
        assert names(**kw) == ["top", "hist", "gather", "finish"]
    assert draw(logits=(3, 4096)).function_names == ["sample_small_f32"]


def test_overlaps_are_refused():
    lens, names = T([3], "i32"), ("past", "new", "free", "table", "query_starts", "key_lens", "positions", "slots", "counts")
    shapes = dict(past=[3], new=[3], free=[9], table=[3, 4], query_starts=[4], key_lens=[3], positions=[7], slots=[7], counts=[2])
    for a, b in itertools.combinations(names, 2):
        kw = {n: T(shapes[n], "i32", lens.ptr) for n in (a, b)}
        if b in ("new", "free"):  # two inputs
            tables(**kw)
        else:
            refused(E.INVALID_ARGUMENT, tables, **kw)
    # the last element of one is the first of the other; next to each other is apart
    refused(E.INVALID_ARGUMENT, tables, past=lens, key_lens=T([3], "i32", lens.ptr + 8))
    tables(past=lens, key_lens=T([3], "i32", lens.ptr + 12))
    tables(free=T([0], "i32", lens.ptr), past=lens, positions=T([0], "i32", lens.ptr), slots=T([0], "i32", 0))
    rows, cache = T([5, 2, 64]), T([7, 2, 16, 64])
    slots = T([5], "i32")
    W = pa.Kernels.PagedKVCacheWrite
    refused(E.INVALID_ARGUMENT, W, rows, rows, slots, cache, cache)
    refused(E.INVALID_ARGUMENT, W, rows, rows, slots, T([7, 2, 16, 64], ptr=rows.ptr), cache)
    W(rows, rows, slots, cache, T([7, 2, 16, 64]))
    q, starts, lens = T([6, 4, 64]), T([4], "i32"), T([3], "i32")
    for x, k, v, o in ((q, cache, cache, q), (q, cache, cache, T([6, 4, 64], ptr=cache.ptr + 128))):
        refused(E.INVALID_ARGUMENT, pa.Kernels.PagedAttention, x, k, v, T([3, 5], "i32"), starts, lens, o, scale=1.0)
    pa.Kernels.PagedAttention(q, cache, cache, T([3, 5], "i32"), starts, lens, T([6, 4, 64]), scale=1.0)
    k, x = T([3], "i32"), T([3, 100], "f32")
    for kw in (dict(top_k=k), dict(temperature=T([3], "f32", k.ptr)), dict(top_p=T([3], "f32", k.ptr + 4)), dict(min_p=T([3], "f32", k.ptr))):
        refused(E.INVALID_ARGUMENT, pa.Kernels.Sample, x, T([3], "f32"), into=k, **kw)
    refused(E.INVALID_ARGUMENT, pa.Kernels.Sample, x, T([3], "f32"), into=T([3], "i32", x.ptr + 396))


def test_too_many_rows_are_refused():
    n = 2 ** 22
    refused(E.TENSOR_SHAPE_MISMATCH, pa.Kernels.Sample, T([n, 64], "f16"), T([n], "f32"), into=T([n], "i32"))
    pa.Kernels.Sample(T([n - 1, 64], "f16"), T([n - 1], "f32"), into=T([n - 1], "i32"))
    refused(E.TENSOR_SHAPE_MISMATCH, attend, q=(2 ** 22, 4, 64))


def test_null_arguments():
    lib = pa.lib()
    h = ctypes.c_void_p()
    d = [ctypes.byref(T([3], "i32").desc()) for _ in range(9)]
    assert lib.popcorn_kernel_page_tables(None, *d[:3], 16, *d[:5], ctypes.byref(h)) == E.INVALID_ARGUMENT
    assert lib.popcorn_kernel_paged_kv_cache_write(*d[:4], None, ctypes.byref(h)) == E.INVALID_ARGUMENT
    assert lib.popcorn_kernel_sample(None, *d[:6], ctypes.byref(h)) == E.INVALID_ARGUMENT
    assert lib.popcorn_kernel_paged_attention(*d[:6], None, 1.0, pa.AttentionMask(0).desc(), 0, 0, ctypes.byref(h)) == E.INVALID_ARGUMENT


HOST = r"""
#include <cstdint>
#include "paged.hpp"
extern "C" int request(const int32_t *in, uint32_t T, uint32_t columns, uint32_t pageSize, int32_t *out) {
    PagedAttentionConstants p{};
    p.T = T, p.columns = columns, p.pageSize = pageSize;
    const pk::PagedRequest r = pk::paged_request(in[0], in[1], in[2], p);
    out[0] = r.start, out[1] = r.n, out[2] = r.pos0, out[3] = r.keys;
    return 0;
}
extern "C" void span(int32_t first, int32_t last, int32_t keys, uint32_t kind, int32_t window, uint32_t sinks, int32_t *out) {
    PagedAttentionConstants p{};
    p.maskKind = kind, p.slidingWindow = window, p.sinks = sinks;
    const pk::PagedSpan s = pk::paged_span(first, last, keys, p);
    out[0] = s.sinkEnd, out[1] = s.lo, out[2] = s.hi;
}
extern "C" int sees(int32_t pos, int32_t key, uint32_t kind, int32_t window, uint32_t sinks) {
    PagedAttentionConstants p{};
    p.maskKind = kind, p.slidingWindow = window, p.sinks = sinks;
    return pk::paged_sees(pos, key, p);
}
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    d = tmp_path_factory.mktemp("paged")
    (d / "h.cpp").write_text(HOST)
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-I", os.path.join(ROOT, "include"), "-I",
                    os.path.join(ROOT, "popcorn_amd", "csrc", "kernels"), "-o", str(d / "h.so"), str(d / "h.cpp")], check=True)
    return ctypes.CDLL(str(d / "h.so"))


LENGTHS = [-2 ** 31, -5, -1, 0, 1, 2, 15, 16, 17, 31, 32, 33, 100, 2 ** 31 - 1]


def test_requests_stay_in_range(host):
    out = (ctypes.c_int32 * 4)()
    for a in LENGTHS:
        for b in LENGTHS:
            for length in LENGTHS:
                for T_, columns, page in ((40, 4, 16), (1, 1, 16), (2 ** 31 - 1, 2 ** 20, 2 ** 20), (7, 0, 32)):
                    host.request((ctypes.c_int32 * 3)(a, b, length), T_, columns, page, out)
                    start, n, pos0, keys = out
                    assert 0 <= start and 0 <= n and start + n <= T_
                    assert 0 <= keys <= columns * page and keys <= max(length, 0)
                    assert pos0 + n == max(length, 0)


def test_spans_hold_every_visible_key(host):
    out = (ctypes.c_int32 * 3)()
    for first in (-3, -1, 0, 5, 16, 40):
        for rows in (1, 3, 16):
            for keys in (0, 1, 30, 57):
                for kind, window, sinks in ((0, -1, 0), (2, -1, 0), (1, 8, 0), (1, 1, 3), (1, 0, 5), (1, -7, 0), (1, 200, 4), (1, 8, 500),
                                            (1, 2 ** 31 - 1, 1), (1, -2 ** 31, 2)):
                    host.span(first, first + rows - 1, keys, kind, window, sinks, out)
                    sink, lo, hi = out
                    assert 0 <= sink <= lo <= hi <= keys
                    inside = set(range(sink)) | set(range(lo, hi))
                    seen = {j for pos in range(first, first + rows) for j in range(keys) if host.sees(pos, j, kind, window, sinks)}
                    assert seen <= inside
                    for pos in range(first, first + rows):
                        import serving_ref

                        want = serving_ref.visible(pos, keys, kind, window, sinks)
                        assert [bool(host.sees(pos, j, kind, window, sinks)) for j in range(keys)] == list(want)
