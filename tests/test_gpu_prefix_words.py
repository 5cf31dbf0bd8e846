"""GPU test of the weights' bits in attention behind shared prefixes: f16 weights enter the product with V as two words wherever they
do in PagedAttention of the same max_query_len, however many rows a group has."""
import numpy as np
import pytest

import cache_ref as C
from gpu_util import download, gpu_env, rounded
from test_gpu_shared_prefix import Batch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    return gpu_env()


def two_word_bound(out, parts, hd):
    """attention_bound with weights of two f16 words. The first is off by 2^-11 of the weight at most, its rest is exact in f32 and off by
    2^-11 of itself: 2^-22 (scores here are so near each other that neither word leaves f16's normal range)."""
    mag, spread, count = parts
    eps = 2.0 * ((hd + 3) * 2.0 ** -24 * spread + 2.0 ** -22) + 2.0 ** -22 + (count + 8) * 2.0 ** -24
    return 2.0 ** -11 * np.abs(out) + 2.0 ** -25 + mag * eps * (1.0 + 2.0 ** -11)


# single tokens; single tokens of so many requests that PagedAttention has a launch for them beside a prompt's tiles, in its group and not
STEPS = [([(64, [(0, 1)] * 70)], 1), ([(64, [(0, 1)] * 300 + [(64, 40)])], 40), ([(64, [(0, 1)] * 300), (0, [(64, 70)])], 0)]


@pytest.mark.parametrize("nq,nkv,hd", [(8, 2, 64), (8, 2, 128), (6, 2, 80), (8, 4, 256)])
@pytest.mark.parametrize("groups,hint", STEPS)
def test_f16_weights_behind_prefixes_have_two_words(env, nq, nkv, hd, groups, hint):
    # V's rows in pairs that cancel, so that a result is small beside the terms whose rounding it shows
    pa, _, stream, enc = env
    b = Batch(groups, nq, nkv, hd, "f16", 16, hd, fill=0.0, std=0.02)
    g = np.random.default_rng(7)
    for table, n in [*zip(b.prefix_table, b.prefix_lens), *zip(b.table, b.keys)]:
        for p in table[:-(-n // 16)]:
            v = g.standard_normal((nkv, 8, hd))
            b.v[p] = rounded(np.stack([v, -v], 2).reshape(nkv, 16, hd), "f16")
        if n == 1:
            b.v[table[0], :, 0] = 0.0
    t, lse = b.tensors(pa)
    scale = float(np.float32(hd ** -0.5))
    mask = pa.AttentionMask.bidirectional
    k = pa.Kernels.SharedPrefixAttention(*t, scale=scale, mask=mask, max_query_len=hint, lse=lse)
    alone = pa.Kernels.PagedAttention(*t[:3], *t[6:], scale=scale, mask=mask, max_query_len=hint)
    assert {"both", "many"} & {n.split("_")[2] for n in k.function_names}
    assert any("_few_" in n for n in alone.function_names)
    enc.encode(k)
    stream.synchronize()
    ref, _, parts = C.shared_attention(b.q, b.k, b.v, b.prefix_table, b.prefix_lens, b.group_starts, b.table, b.starts, b.keys, b.out, b.lse,
                                       scale, 2)
    off = np.abs(download(t[-1], stream) - ref) / two_word_bound(ref, parts, hd)
    assert (off <= 1).all(), off.max()
