"""GPU tests of attention behind shared prefixes where the merge takes a wave per row and blocks have long stretches of steps and
several units, against a 64-bit reference by whole requests."""
import numpy as np
import pytest

import cache_batches as B
import cache_ref as C
from gpu_util import download, gpu_env
from test_gpu_shared_prefix import Batch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    return gpu_env()


def attend(env, b, kinds, window=0, sinks=0, hint=0):
    pa, _, stream, enc = env
    t, lse = b.tensors(pa)
    scale = float(np.float32(b.hd ** -0.5))
    mask = pa.AttentionMask.causal_sliding_window(window) if window else pa.AttentionMask.causal
    k = pa.Kernels.SharedPrefixAttention(*t, scale=scale, mask=mask, sinks=sinks, max_query_len=hint, lse=lse)
    assert {n.split("_")[2] for n in k.function_names} - {"merge", "plan", "positions"} == kinds
    enc.encode(k)
    stream.synchronize()
    out, logs = download(t[-1], stream), download(lse, stream)
    ref, ref_lse, parts = B.shared_attention(b.q, b.k, b.v, b.prefix_table, b.prefix_lens, b.group_starts, b.table, b.starts, b.keys, b.out,
                                             b.lse, scale, 1 if window else 0, window or -1, sinks)
    end = int(b.starts[-1])
    np.testing.assert_array_equal(out[end:], b.out[end:])
    np.testing.assert_array_equal(logs[end:], b.lse[end:])
    for got, x, most in ((out, ref, C.attention_bound(ref, parts, b.dtype, b.hd)), (logs, ref_lse, C.lse_bound(ref_lse, parts, b.hd))):
        off = np.abs(got - x)[:end] / most[:end]
        assert (off <= 1).all(), off.max()


@pytest.mark.parametrize("dtype,nq,nkv,hd,kinds", [
    ("bf16", 32, 8, 64, {"both"}), ("f16", 32, 8, 128, {"both"}), ("bf16", 32, 4, 80, {"both"}), ("bf16", 32, 8, 256, {"few", "many"}),
    ("f16", 32, 4, 512, {"few"}), ("bf16", 32, 8, 480, {"few"}), ("f32", 32, 8, 128, {"few"}), ("f32", 32, 4, 256, {"few"}), ("f32", 32, 8, 512, {"few"})])
@pytest.mark.parametrize("window,sinks", [(0, 0), (150, 3)])
def test_rows_that_a_wave_merges_alone(env, dtype, nq, nkv, hd, kinds, window, sinks):
    # 4096 rows and more; rows behind a prefix and not, pieces of one state and of many
    b = Batch([(700, [(13 * i % 90, 1) for i in range(100)]), (40, [(3, 1), (0, 30)]), (None, [(260, 1), (5, 1)])], nq, nkv, hd, dtype, 16, hd,
              pad=2, std=2.0)
    assert b.starts[-1] * nq >= 4096
    attend(env, b, kinds, window, sinks, hint=30)


def shares(b, nq, nkv, hd):
    """Counted steps (of 64 keys, and 6 a unit) of a block with tiles, if all blocks had some, and of a prefix's unit."""
    rows = [(b.starts[y] - b.starts[x]) * nq // nkv for x, y in zip(b.group_starts, b.group_starts[1:])]
    units = [(-(-n // 64) + 6, -(-int(r) // 128) * nkv) for n, r in zip(b.prefix_lens, rows)]
    return sum(s * n for s, n in units) / (256 if hd > 128 else 512), units[0][0]


@pytest.mark.parametrize("dtype,nq,nkv,hd,tokens,prefix", [("bf16", 32, 8, 64, 220, 12500), ("f16", 32, 8, 128, 190, 14000), ("bf16", 16, 8, 80, 400, 12500),
                                                           ("f16", 16, 4, 256, 190, 14000)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (9000, 70)])
def test_blocks_of_many_steps(env, dtype, nq, nkv, hd, tokens, prefix, window, sinks):
    # more steps than a lane's quad holds the pages of (16); under the window rows whose first keys lie in different steps
    b = Batch([(prefix, [(61 * i % 90, 1) for i in range(tokens - 3)] + [(0, 3)])], nq, nkv, hd, dtype, 32, hd, std=2.0)
    share, unit = shares(b, nq, nkv, hd)
    assert min(share, unit) > 20
    attend(env, b, {"few", "many"} if hd == 256 else {"both"}, window, sinks, hint=3)


@pytest.mark.parametrize("dtype,nq,nkv,hd,tokens,prefix", [("f16", 32, 8, 64, 1900, 330), ("bf16", 32, 8, 128, 1900, 200), ("bf16", 16, 4, 256, 1500, 150)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (120, 5)])
def test_blocks_of_several_units(env, dtype, nq, nkv, hd, tokens, prefix, window, sinks):
    b = Batch([(prefix, [(17 * i % 40, 1) for i in range(tokens)]), (prefix // 2, [(5, 9)] * (tokens // 10))], nq, nkv, hd, dtype, 16, hd, std=2.0)
    share, unit = shares(b, nq, nkv, hd)
    assert share > 1.3 * unit
    attend(env, b, {"few", "many"} if hd == 256 else {"both"}, window, sinks, hint=1 if hd == 64 else 9)
