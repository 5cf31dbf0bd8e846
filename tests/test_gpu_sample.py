"""GPU tests of the token draw: equal, token for token, to the definition in
whole numbers (serving_ref.sample)."""
import numpy as np
import pytest

import serving_ref as R
from gpu_util import gpu_env, rounded, upload

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    return gpu_env()


def run(env, logits, dtype, uniforms, **options):
    pa, _, stream, enc = env
    rows = len(logits)
    as_dtype = {"temperature": "f32", "top_k": "i32", "top_p": "f32", "min_p": "f32"}
    o = {n: pa.Tensor.from_numpy(np.asarray(v, np.int32 if n == "top_k" else np.float32), as_dtype[n]) for n, v in options.items()}
    out = pa.Tensor.from_numpy(np.full(rows, -77, np.int32), "i32")
    enc.encode(pa.Kernels.Sample(upload(pa, logits, dtype), pa.Tensor.from_numpy(np.asarray(uniforms, np.float32)), out, **o))
    stream.synchronize()
    return out.numpy(stream)


def check(env, logits, dtype, uniforms, **options):
    logits = rounded(logits, dtype)
    got = run(env, logits, dtype, uniforms, **options)
    np.testing.assert_array_equal(got, R.sample(logits, uniforms, **options))
    return got


OPTIONS = {
    "plain": {},
    "temperature": dict(temperature=[0.7, 1.3, 0.05, 40.0, 1.0]),
    "top_k": dict(top_k=[1, 2, 50, 700, 10 ** 6]),
    "top_p": dict(top_p=[0.1, 0.5, 0.9, 0.999, 1.0]),
    "min_p": dict(min_p=[0.0, 0.001, 0.05, 0.5, 1.0]),
    "all": dict(temperature=[0.7, 1.3, 0.9, 2.0, 1.0], top_k=[3, 40, 0, 333, 100], top_p=[0.95, 0.5, 0.8, 0.99, 0.3],
                min_p=[0.01, 0.0, 0.1, 0.002, 0.05]),
    "edges": dict(temperature=[0.0, -1.0, np.nan, np.inf, 1e-30], top_k=[-5, 0, 7, 9, 3], top_p=[0.0, -1.0, np.nan, 2.0, 1e-20],
                  min_p=[-1.0, np.nan, 3.0, 0.0, 1.0]),
}


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("options", list(OPTIONS))
@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 65, 1000, 1025, 5003, 17000])
def test_sample(env, dtype, options, vocab):
    g = np.random.default_rng(vocab)
    for spread in (0.3, 3.0):
        check(env, g.standard_normal((5, vocab)) * spread, dtype, g.random(5), **OPTIONS[options])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_sample_large(env, dtype):
    g = np.random.default_rng(1)
    x = g.standard_normal((3, 256000)) * 1.5
    check(env, x, dtype, g.random(3), top_p=[0.9, 0.99, 0.5])
    check(env, x, dtype, g.random(3), top_k=[50, 20000, 200000], top_p=[0.9, 0.95, 1.0], temperature=[0.8, 1.0, 1.5])
    check(env, x, dtype, g.random(3), min_p=[0.1, 0.01, 0.5])
    check(env, x, dtype, g.random(3))


@pytest.mark.parametrize("vocab", [5, 1024, 9000, 65537])
def test_sample_ties(env, vocab):
    # few distinct logits: the cut falls among equals, by index
    g = np.random.default_rng(vocab)
    x = g.integers(-2, 3, (8, vocab)).astype(np.float32) * 0.5
    check(env, x, "f32", g.random(8), top_k=g.integers(1, vocab + 1, 8))
    check(env, x, "bf16", g.random(8), top_p=g.random(8))
    check(env, np.zeros((8, vocab)), "f16", g.random(8), top_k=g.integers(1, vocab + 1, 8), top_p=g.random(8))
    signed = np.where(g.random((8, vocab)) < 0.5, 0.0, -0.0).astype(np.float32)  # both zeros are one logit
    check(env, signed, "f32", g.random(8), top_k=g.integers(1, vocab + 1, 8))
    check(env, signed, "f32", g.random(8), temperature=np.zeros(8))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_sample_special_logits(env, dtype):
    g = np.random.default_rng(2)
    low = {"f32": np.finfo(np.float32).min, "f16": -65504.0, "bf16": -3.3895313892515355e38}[dtype]
    x = g.standard_normal((9, 3000)).astype(np.float32)
    x[0, g.random(3000) < 0.9] = -np.inf
    x[1, g.random(3000) < 0.9] = low
    x[2] = -np.inf
    x[3] = np.nan
    x[4, g.random(3000) < 0.5] = np.nan
    x[5, [7, 2000, 2999]] = np.inf
    x[6] = -np.inf
    x[6, 1234] = low
    x[7] = low
    x[8, :2] = np.nan, np.inf
    got = check(env, x, dtype, g.random(9))
    assert got[2] == got[3] == -1 and got[6] == 1234 and got[8] == 1 and got[5] in (7, 2000, 2999)
    check(env, x, dtype, g.random(9), top_k=[5] * 9, top_p=[0.7] * 9, min_p=[0.05] * 9, temperature=[0.5] * 9)
    check(env, x, dtype, g.random(9), top_k=[2990] * 9, top_p=[0.999] * 9)
    check(env, x, dtype, g.random(9), temperature=[0.0] * 9)
    check(env, x, dtype, g.random(9), temperature=[np.inf] * 9)
    check(env, x, dtype, g.random(9), temperature=[1e30] * 9)


def test_sample_uniform_ends(env):
    x = np.random.default_rng(3).standard_normal((8, 777))
    u = [0.0, -1.0, 1.0 - 2.0 ** -24, 1.0, 5.0, np.nan, np.inf, 2.0 ** -40]
    check(env, x, "f32", u)
    check(env, x, "f32", u, top_k=[10] * 8, top_p=[0.8] * 8)


def test_sample_frequencies(env):
    # 20000 draws from 6 weights: each count within 5 standard deviations of its share
    n = 20000
    logits = np.tile(np.log(np.array([1, 2, 3, 4, 5, 85.0])).astype(np.float32), (n, 1))
    got = run(env, logits, "f32", np.random.default_rng(4).random(n))
    p = np.array([1, 2, 3, 4, 5, 85]) / 100
    assert (np.abs(np.bincount(got, minlength=6) - n * p) < 5 * np.sqrt(n * p * (1 - p))).all()


def test_sample_unaligned_rows(env):
    pa, _, stream, enc = env
    g = np.random.default_rng(5)
    x = rounded(g.standard_normal((3, 4001)), "bf16")
    t = upload(pa, np.concatenate([[9.0], x.ravel()]), "bf16")
    u = g.random(3)
    out = pa.Tensor.empty([3], "i32")
    enc.encode(pa.Kernels.Sample(pa.Tensor(t.ptr + 2, [3, 4001], "bf16", owner=t), pa.Tensor.from_numpy(u.astype(np.float32)), out))
    stream.synchronize()
    np.testing.assert_array_equal(out.numpy(stream), R.sample(x, u))


def test_sample_no_rows(env):
    pa, _, stream, enc = env
    z = pa.Tensor.empty([0], "f32")
    enc.encode(pa.Kernels.Sample(pa.Tensor.empty([0, 50], "f32"), z, pa.Tensor.empty([0], "i32")))
    stream.synchronize()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_sample_special_logits_in_slices(env, dtype):
    g = np.random.default_rng(20)
    n = 30001
    low = {"f32": np.finfo(np.float32).min, "f16": -65504.0, "bf16": -3.3895313892515355e38}[dtype]
    x = g.standard_normal((9, n)).astype(np.float32)
    x[0, g.random(n) < 0.99] = -np.inf
    x[1, g.random(n) < 0.9] = low
    x[2] = -np.inf
    x[3] = np.nan
    x[4, g.random(n) < 0.5] = np.nan
    x[5, [7, 20000, n - 1]] = np.inf
    x[6] = -np.inf
    x[6, n - 1] = low
    x[7] = low
    x[8, :2] = np.nan, np.inf
    for options in (dict(), dict(top_k=[5] * 9, top_p=[0.7] * 9, min_p=[0.05] * 9, temperature=[0.5] * 9), dict(top_k=[n - 3] * 9),
                    dict(top_k=[n - 10] * 9, top_p=[0.999] * 9), dict(temperature=[0.0] * 9), dict(temperature=[np.inf] * 9, top_p=[0.6] * 9),
                    dict(temperature=[0.0, 1.0, np.inf] * 3, top_k=[0, 50, n] * 3, top_p=[1.0] * 5 + [0.5] * 4)):
        got = check(env, x, dtype, g.random(9), **options)
        assert got[2] == got[3] == -1 and got[6] == n - 1 and got[8] == 1 and got[5] in (7, 20000, n - 1)


@pytest.mark.parametrize("dtype,options", [("f32", dict(top_k=[3000], top_p=[0.95])), ("bf16", dict(min_p=[0.001]))])
def test_sample_longest_row(env, dtype, options):
    x = np.random.default_rng(21).standard_normal((1, 2 ** 22)).astype(np.float32) * 2
    check(env, x, dtype, [1.0 - 2.0 ** -24], **options)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("least", [1, 2, 3, 7, 19, 20, 100])
def test_sample_min_p_at_its_least_weights(env, dtype, least):
    # Many tokens whose weights round to the least whole number that min-p keeps, from just below it (min-p's
    # border in the logits is at least - 1/2), behind one heavy token; top-k is on and cuts nothing.
    n, many = 250000, 200000
    x = np.full((3, n), -60.0, np.float32)
    x[:, 0] = 0.0
    g = np.random.default_rng(least)
    at = 1 + g.permutation(n - 1)[:many]
    x[:, at] = np.log((least - np.array([0.45, 0.3, 0.1]))[:, None] / 2.0 ** 40)
    if dtype != "f32":  # the nearest logits of the type whose weights are the same
        steps = {"f16": 2.0 ** -6, "bf16": 2.0 ** -3}[dtype]
        x[:, at] = np.floor(x[:, at] / steps + 0.5) * steps
    u = np.array([1.0 - 2.0 ** -24, 1.0 - 2.0 ** -23, 1.0 - 2.0 ** -22])
    p = [(least - 0.5) / 2.0 ** 40] * 3
    got = check(env, x, dtype, u, min_p=p, top_k=[n - 1] * 3)
    if dtype == "f32" and least <= 3:
        assert got[0] > 0  # (not the heavy token)


@pytest.mark.parametrize("temperature,logits", [
    (1e38, [3e38, 1e38, -1e38, -3e38, -3.4e38]),  # distances past the largest number
    (3e38, [3.4e38, 0.0, -3.4e38]),
    (1e-38, [0.0, -4e-39, -1e-38, -2e-38, -1e-37]),  # more bins in a unit than the largest number
    (1.1e-41, [0.0, -1e-41, -3e-41]),  # numbers below the smallest normal one
], ids=str)
@pytest.mark.parametrize("vocab", [1000, 9001])
def test_sample_min_p_at_extreme_temperatures(env, temperature, logits, vocab):
    g = np.random.default_rng(vocab)
    x = np.array(logits, np.float32)[g.integers(0, len(logits), (6, vocab))]
    x[g.random((6, vocab)) < 0.5] = -np.inf
    t = [temperature] * 6
    check(env, x, "f32", g.random(6), temperature=t, min_p=[0.001, 0.05, 0.2, 0.5, 0.9, 1.0], top_k=[vocab - 1] * 6)
    check(env, x, "f32", g.random(6), temperature=t, min_p=[0.001, 0.05, 0.2, 0.5, 0.9, 1.0], top_p=[0.9999] * 6)
    # few tokens with weight, so that the candidates fit their list
    x[g.random((6, vocab)) < 0.9] = -np.inf
    check(env, x, "f32", g.random(6), temperature=t, min_p=[0.001, 0.05, 0.2, 0.5, 0.9, 1.0], top_k=[vocab - 1] * 6)
    check(env, x, "f32", g.random(6), temperature=t, top_k=[vocab // 30] * 6)


@pytest.mark.parametrize("vocab", [70, 4096, 4097, 30001])
def test_sample_greedy_rows_among_others(env, vocab):
    # a temperature of 0 (or less, or NaN) takes the first of the highest, whatever the other options; beside rows that draw
    g = np.random.default_rng(vocab)
    x = g.integers(-5, 3, (8, vocab)).astype(np.float32)
    x[3], x[5, 9:] = -np.inf, np.nan
    x[6, [11, 60]] = np.inf
    t = np.array([0.0, 1.0, -1.0, 0.0, np.nan, 0.0, 0.0, 1e-30], np.float32)
    u = np.full(8, 1.0 - 2.0 ** -24)
    for kw in (dict(), dict(min_p=[1.0] * 8), dict(top_k=[7] * 8), dict(top_p=[0.99] * 8), dict(top_k=[40] * 8, top_p=[0.3] * 8, min_p=[0.2] * 8)):
        got = check(env, x, "f32", u, temperature=t, **kw)
        want = [int(np.nanargmax(np.where(np.isnan(r), -np.inf, r))) for r in x]
        assert got[3] == -1 and all(got[r] == want[r] for r in (0, 2, 4, 5, 6))


def most_in_a_bin(x, t):
    """The tokens in the fullest of the bins, 72 to a temperature, that the cuts are looked for in."""
    return np.bincount(np.minimum((x.max() - x) * (72.0 / t), 2047).astype(np.int64)).max()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("options", [dict(top_p=[0.5, 0.6, 0.7]), dict(top_k=[60000, 128000, 150000]),
                                     dict(top_k=[200000] * 3, top_p=[0.5, 0.7, 0.6], min_p=[0.0, 0.001, 0.3])], ids=lambda o: "-".join(o))
def test_sample_flat_rows(env, dtype, options):
    # distinct logits that lie close together: the bin with the cut holds more candidates than their list
    g = np.random.default_rng(22)
    x = rounded(g.standard_normal((3, 256000)) * 0.5, dtype)
    x[:, 0] = x.max()  # rows of one highest logit and one temperature
    assert all(most_in_a_bin(r, 2.0) > 5000 for r in x)
    assert dtype == "bf16" or len(np.unique(x[0])) > 250000
    for u in (g.random(3), [0.0, 0.5, 1.0 - 2.0 ** -24]):
        check(env, x, dtype, u, temperature=[2.0] * 3, **options)
