"""GPU tests of attention weights beyond small batches, against a 64-bit reference: rows whose logarithm is NaN."""
import numpy as np
import pytest

import cache_ref as C
from gpu_util import download, gpu_env
from test_gpu_eviction import PROMPTS, f32, logarithms
from test_gpu_shared_prefix import Batch

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
