"""CPU test of a token's weight in the draw (sample.hpp, compiled for the host)
against 50-digit arithmetic: what is promised is a whole number at most 0.51 from
2^40 exp((logit - highest) / temperature)."""
import ctypes
import os
import subprocess
from decimal import Decimal, getcontext

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HOST = r"""
#include "sample.hpp"
extern "C" void weights(const float *v, const float *top, const float *temperature, uint64_t *out, long n) {
    for (long i = 0; i < n; ++i) out[i] = pk::sample_weight(v[i], top[i], pk::sample_rate(temperature[i]));
}
"""


@pytest.fixture(scope="module")
def weights(tmp_path_factory):
    d = tmp_path_factory.mktemp("sample")
    (d / "h.cpp").write_text(HOST)
    # (libm's fma rounds once, as the GPU's does)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", os.path.join(ROOT, "popcorn_amd", "csrc", "kernels"), "-o",
                    str(d / "h.so"), str(d / "h.cpp"), "-lm"], check=True)
    lib = ctypes.CDLL(str(d / "h.so"))

    def run(v, top, t):
        v, top, t = (np.ascontiguousarray(np.broadcast_to(np.asarray(x, np.float32), np.shape(v))) for x in (v, top, t))
        out = np.zeros(v.size, np.uint64)
        lib.weights(*[ctypes.c_void_p(x.ctypes.data) for x in (v, top, t, out)], ctypes.c_long(v.size))
        return out

    return run


def off(v, top, t, w):
    """The largest distance of a weight from the real number that it stands for."""
    getcontext().prec = 50
    worst = Decimal(0)
    for a, b, c, u in zip(*(np.broadcast_to(np.asarray(x, np.float32), np.shape(v)).tolist() for x in (v, top, t)), w.tolist()):
        real = ((Decimal(a) - Decimal(b)) / Decimal(c)).exp() * 2 ** 40
        worst = max(worst, abs(Decimal(u) - real))
    return float(worst)


@pytest.mark.parametrize("temperature", [1.0, 0.7, 1.3, 0.05, 40.0, 1e-20, 1e30, 1e-38, 3.4e38])
def test_weights_over_distances(weights, temperature):
    g = np.random.default_rng(1)
    top = np.float32(g.standard_normal() * 3 * min(max(temperature, 1e-30), 1e37))
    # distances of up to 30 temperatures, most of them small, where a unit is the smallest part of a weight
    d = np.concatenate([g.uniform(0, 30, 3000), g.uniform(0, 1, 3000), np.arange(0, 43) * np.log(2), (np.arange(0, 43) + 0.5) * np.log(2)])
    v = top - d * temperature
    v = v[np.abs(v) < 3.4e38].astype(np.float32)
    assert off(v, top, temperature, weights(v, top, temperature)) <= 0.51


def test_weights_of_16_bit_logits(weights):
    # every step of a bf16 and an f16 row near its highest logit
    for top, step in ((8.0, 2.0 ** -5), (3.0, 2.0 ** -9), (0.0, 2.0 ** -10)):
        v = np.float32(top) - np.arange(0, 3000, dtype=np.float32) * np.float32(step)
        for t in (1.0, 0.8, 1.7):
            assert off(v, top, t, weights(v, top, t)) <= 0.51


def test_weights_where_there_is_no_distance(weights):
    inf, nan, one = np.inf, np.nan, 2 ** 40
    low = np.finfo(np.float32).min
    v = [2.0, 1.0, -inf, nan, low, -inf, inf, 5.0, nan, -0.0]
    top = [2.0, 2.0, 2.0, 2.0, 2.0, low, inf, inf, inf, 0.0]
    for t, second in ((1.0, round(one / np.e)), (inf, one), (0.0, 0), (1e-30, 0)):
        w = weights(v, top, t)
        assert w[0] == w[6] == w[9] == one and w[1] == second
        assert not w[[2, 3, 5, 7, 8]].any()
        assert w[4] == (one if t == inf else 0)
    # a temperature of 0, less or NaN leaves weight to the highest alone
    for t in (0.0, -0.0, -3.0, nan):
        assert list(weights([1.0, 0.99999994, 1.0], 1.0, t)) == [one, 0, one]
