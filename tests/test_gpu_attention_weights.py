"""GPU tests of attention weights against a 64-bit reference: rows whose logarithm is NaN, and launches whose waves and blocks have
long stretches of keys and rows."""
import numpy as np
import pytest

import cache_batches as B
import cache_ref as C
from gpu_util import download, gpu_env, rounded, upload
from test_gpu_eviction import PROMPTS, f32, logarithms
from test_gpu_shared_prefix import Batch, i32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    return gpu_env()


@pytest.mark.parametrize("dtype,nq,nkv,hd", [("bf16", 4, 2, 64), ("f16", 8, 2, 128), ("bf16", 8, 4, 256), ("f32", 4, 2, 64), ("bf16", 4, 1, 512),
                                             ("f16", 4, 2, 36)])
@pytest.mark.parametrize("kind", [0, 2])
def test_a_row_of_nan_gives_it_to_the_keys_that_it_sees_alone(env, dtype, nq, nkv, hd, kind):
    pa, _, stream, enc = env
    b = Batch(PROMPTS, nq, nkv, hd, dtype, 16, hd)
    scale = float(np.float32(hd ** -0.5))
    lse = logarithms(b, scale, kind)
    for r, i in ((0, 3), (2, 0), (4, 60), (4, 61), (6, 20)):  # row i of request r, in one of its heads
        row = b.starts[r] + i
        b.q[row, r % nq], lse[row, r % nq] = np.nan, np.nan
    old = np.random.default_rng(1).random((len(b.lens), nkv, b.table.shape[1] * 16)).astype(np.float32)
    t, w = b.tensors(pa)[0], f32(pa, old)
    enc.encode(pa.Kernels.PagedAttentionWeights(t[0], t[1], *t[6:9], f32(pa, lse), w, scale=scale,
                                                mask=pa.AttentionMask.bidirectional if kind == 2 else pa.AttentionMask.causal))
    stream.synchronize()
    got = download(w, stream)
    ref, bound = C.weights(b.q, b.k, b.table, b.starts, b.keys, lse, old, scale, kind, 0)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(ref))
    fine = ~np.isnan(ref)
    assert (np.abs(got - ref) <= bound)[fine].all()
    if kind == 0:
        assert np.isnan(ref[4, :, :82]).all(-1).any() and not np.isnan(ref[4, :, 82:]).any()


# ---- launches whose waves and blocks have long stretches --------------------------------

CUS = 256


class Loose:
    """Requests [(past, new), ...] whose tables name the same few pages again and again, so that long ones need no large cache."""

    def __init__(self, lens, nq, nkv, hd, dtype, page, seed, std=1.0):
        g = np.random.default_rng(seed)
        self.keys = np.array([p + n for p, n in lens])
        self.starts = np.concatenate([[0], np.cumsum([n for _, n in lens])])
        self.k = rounded(g.standard_normal((40, nkv, page, hd)), dtype)
        self.table = g.integers(0, 40, (len(lens), -(-int(self.keys.max()) // page) + 1))
        self.q = rounded(g.standard_normal((int(self.starts[-1]), nq, hd), np.float32) * std, dtype)
        self.old = g.random((len(lens), nkv, self.table.shape[1] * page), np.float32)


def weigh_loose(env, b, dtype, kind=0, last_rows=0, hint=0, kinds=None):
    pa, _, stream, enc = env
    scale = float(np.float32(b.q.shape[2] ** -0.5))
    ref, bound, lse = B.weights(b.q, b.k, b.table, b.starts, b.keys, None, b.old, scale, kind, last_rows)
    w = f32(pa, b.old)
    k = pa.Kernels.PagedAttentionWeights(upload(pa, b.q, dtype), upload(pa, b.k, dtype), i32(pa, b.table), i32(pa, b.starts), i32(pa, b.keys),
                                         f32(pa, lse), w, scale=scale, last_rows=last_rows, max_query_len=hint,
                                         mask=pa.AttentionMask.bidirectional if kind == 2 else pa.AttentionMask.causal)
    assert {n.split("_")[2] for n in k.function_names} - {"plan", "tiles"} == kinds
    enc.encode(k)
    stream.synchronize()
    got = download(w, stream)
    np.testing.assert_array_equal(got[ref == b.old], b.old[ref == b.old])
    off = np.abs(got - ref)
    assert (off <= bound).all(), (off / bound).max()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("nq,new,kind", [(8, 2, 0), (24, 2, 2)])
def test_waves_that_take_more_keys_than_their_lanes_hold_pages_of(env, dtype, hd, nq, new, kind):
    # a wave's stretch is over 64 groups of 16 keys; 24 rows are two tiles of 16, whose second one adds to what the first left
    nkv, waves = 2, 4 * CUS * {64: 3 + (dtype != "f32"), 128: 2 + (dtype != "f32"), 256: 2, 512: 1 + (dtype != "f32")}[hd]
    keys = 70 * 16 * waves // (3 * nkv)
    lens = [(keys + 5, 1), (keys - 100, new), (keys // 2 + 17, new), (0, 1), (keys // 2 + 1300, 1)]
    b = Loose(lens, nq, nkv, hd, dtype, 16, hd)
    assert sum(-(-int(x) // 16) for x in b.keys) * nkv > 68 * waves
    weigh_loose(env, b, dtype, kind, hint=new, kinds={"few"})


def tile_share(b, nq, nkv, hd, kind, last_rows, few):
    """Counted steps of a block (a unit's steps of 64 rows, and 10), and the units' steps."""
    G, units = nq // nkv, []
    for keys, n in zip(b.keys, np.diff(b.starts)):
        n = min(n, last_rows or n)
        if n * G > few:
            rows = -(-n * G // 64)
            units += [rows - (0 if kind == 2 else max(t - (keys - n), 0) * G // 64) for t in range(0, keys, 256)] * nkv
    return -(-(sum(units) + 10 * len(units)) // (CUS * (1 if hd > 128 else 2))), units


@pytest.mark.parametrize("dtype,nq,nkv,hd,past,new,kind,last_rows", [
    ("bf16", 8, 4, 256, 0, 3000, 0, 0), ("f16", 16, 4, 128, 133, 3000, 0, 0), ("bf16", 12, 4, 64, 7, 3500, 0, 0), ("f16", 12, 4, 80, 0, 2500, 2, 0),
    ("bf16", 20, 4, 256, 500, 1300, 0, 0), ("bf16", 16, 8, 128, 2000, 1500, 2, 1333)])
def test_blocks_that_go_round_their_ring_of_rows(env, dtype, nq, nkv, hd, past, new, kind, last_rows):
    # a block's piece is many more steps than Q has places in LDS; heads to a KV head that divide a step's 64 rows, and 3, 5 that do not
    b = Loose([(past, new)], nq, nkv, hd, dtype, 32, hd)
    share, units = tile_share(b, nq, nkv, hd, kind, last_rows, 0)
    assert share >= 10 and max(units) >= 20
    weigh_loose(env, b, dtype, kind, last_rows, kinds={"tile", "join"})


@pytest.mark.parametrize("dtype,nq,nkv,hd,requests,last_rows", [("bf16", 8, 8, 64, 100, 0), ("f16", 4, 4, 256, 60, 0), ("f16", 12, 4, 128, 110, 160)])
def test_blocks_that_take_several_units(env, dtype, nq, nkv, hd, requests, last_rows):
    g = np.random.default_rng(hd)
    lens = [(int(p), int(n)) for p, n in zip(g.integers(0, 300, requests), g.integers(250, 500, requests))]
    lens[::9] = [(700, 1)] * len(lens[::9])
    b = Loose(lens, nq, nkv, hd, dtype, 16, hd)
    share, units = tile_share(b, nq, nkv, hd, 0, last_rows, 32)
    assert share > 1.5 * (np.mean(units) + 10)
    weigh_loose(env, b, dtype, 0, last_rows, kinds={"few", "tile", "join"})


@pytest.mark.parametrize("dtype,nq,nkv,hd,keys", [("f16", 16, 8, 128, 9000), ("bf16", 8, 2, 256, 9000), ("bf16", 8, 4, 64, 9000)])
def test_long_caches_of_single_tokens_beside_a_prompt(env, dtype, nq, nkv, hd, keys):
    # few requests, whose keys are read by the kernel that streams them and not by tiles
    b = Loose([(0, 300)] + [(keys - 500 * i, 1) for i in range(7)], nq, nkv, hd, dtype, 16, hd)
    weigh_loose(env, b, dtype, kinds={"few", "tile", "join"})
    b = Loose([(0, 300)] + [(300 - 50 * i, 1) for i in range(5)], nq, nkv, hd, dtype, 16, hd)
    weigh_loose(env, b, dtype, kinds={"tile", "join"})
