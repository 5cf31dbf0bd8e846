"""CPU tests of how paged attention cuts its work up (paged.hpp, compiled for the
host): the steps of a tile hold every visible key once, the pieces that workers are
dealt hold every step of every unit once, and the merge is told who shares a unit."""
import ctypes
import itertools
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HOST = r"""
#include <algorithm>
#include <cstdint>
#include <vector>
#include "paged.hpp"
using namespace pk;
struct Call {
    PagedAttentionConstants p;
    PagedWorkConstants w;
};
static Call call(const int32_t *c) {
    Call x{};
    x.p.T = c[0], x.p.R = c[1], x.p.Nq = c[2], x.p.Nkv = c[3], x.p.pageSize = c[4], x.p.columns = c[5];
    x.p.maskKind = c[6], x.p.slidingWindow = c[7], x.p.sinks = c[8];
    x.w.rows = c[9], x.w.stepKeys = c[10], x.w.fewRows = c[11], x.w.manyRows = c[12], x.w.workers = c[13], x.w.minSteps = c[14], x.w.unitSteps = c[15];
    return x;
}
struct Tile {
    uint64_t before;
    uint32_t request, tile;
    PagedSteps steps;
};
static std::vector<Tile> tiles_of(const Call &x, const int32_t *starts, const int32_t *lens, uint64_t &total) {
    std::vector<Tile> tiles;
    total = 0;
    for (uint32_t r = 0; r < x.p.R; ++r) {
        const PagedRequest q = paged_request(starts[r], starts[r + 1], lens[r], x.p);
        const uint32_t rows = (uint32_t)q.n * (x.p.Nq / x.p.Nkv);
        if (rows <= x.w.fewRows || rows > x.w.manyRows) continue;
        for (uint32_t t = 0; t * x.w.rows < rows; ++t) {
            const PagedSteps s = paged_steps(q, t, x.p, x.w);
            tiles.push_back(Tile{total, r, t, s});
            total += s.n + x.w.unitSteps;
        }
    }
    return tiles;
}
// (request, tile, r0, r1, n) of each tile, and after them the first keys of its steps
extern "C" long tiles(const int32_t *c, const int32_t *starts, const int32_t *lens, int64_t *out, int64_t *keys, long most) {
    const Call x = call(c);
    uint64_t total;
    long i = 0, k = 0;
    for (const Tile &t : tiles_of(x, starts, lens, total)) {
        for (uint32_t v : {t.request, t.tile, t.steps.r0, t.steps.r1, t.steps.n}) out[i++] = v;
        for (uint32_t s = 0; s < t.steps.n && k < most; ++s) keys[k++] = paged_step_key(t.steps, s, x.w);
    }
    return i / 5;
}
// (worker, tile, head, lo, hi, workers that share the unit) of each piece
extern "C" long deal(const int32_t *c, const int32_t *starts, const int32_t *lens, int64_t *out) {
    const Call x = call(c);
    uint64_t total;
    const std::vector<Tile> tiles = tiles_of(x, starts, lens, total);
    total *= x.p.Nkv;
    const uint64_t share = paged_share(total, x.w);
    long i = 0;
    for (uint32_t worker = 0; worker < x.w.workers; ++worker) {
        uint64_t at = worker * share;
        const uint64_t end = std::min(at + share, total);
        size_t tile = 0;
        if (at < end)
            while (tile + 1 < tiles.size() && tiles[tile + 1].before * x.p.Nkv <= at) ++tile;
        while (at < end) {
            const Tile &t = tiles[tile];
            const PagedPiece p = paged_piece(at - t.before * x.p.Nkv, end - at, t.steps.n, x.w);
            at += p.taken;
            const int64_t v[] = {worker, (int64_t)tile, p.hkv, p.lo, p.hi, at == end ? paged_sharers(p, t.steps.n, end, share, worker) : 0};
            out[i++] = v[0], out[i++] = v[1], out[i++] = v[2], out[i++] = v[3], out[i++] = v[4], out[i++] = v[5];
            if (p.behind == 0 && p.hkv + 1 == x.p.Nkv) ++tile;
        }
    }
    return i / 6;
}
extern "C" uint32_t worker_of(uint64_t at, uint64_t share) { return paged_worker(at, share); }
// the piece at `in` of units of n steps, in wide numbers
extern "C" void piece(uint64_t in, uint64_t left, uint32_t n, uint32_t unitSteps, uint32_t *out) {
    PagedWorkConstants w{};
    w.unitSteps = unitSteps;
    const PagedPiece p = paged_piece(in, left, n, w);
    out[0] = p.hkv, out[1] = p.lo, out[2] = p.hi, out[3] = p.taken, out[4] = p.behind;
}
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "h.cpp").write_text(HOST)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", os.path.join(ROOT, "include"), "-I",
                    os.path.join(ROOT, "popcorn_amd", "csrc", "kernels"), "-o", str(d / "h.so"), str(d / "h.cpp")], check=True)
    lib = ctypes.CDLL(str(d / "h.so"))
    lib.tiles.restype = lib.deal.restype = ctypes.c_long
    return lib


def ptr(a):
    return ctypes.c_void_p(a.ctypes.data)


class Plan:
    """A launch over requests of (past, new) lengths."""

    FIELDS = ("T", "R", "Nq", "Nkv", "page", "columns", "mask", "window", "sinks", "rows", "step", "few", "many", "workers", "least", "unit")

    def __init__(self, lens, **kw):
        base = dict(T=sum(n for _, n in lens), R=len(lens), Nq=8, Nkv=2, page=16, columns=10 ** 4, mask=0, window=-1, sinks=0, rows=16, step=32,
                    few=0, many=2 ** 31 - 1, workers=64, least=4, unit=12)
        self.lens, self.k = lens, dict(base, **kw)
        self.c = np.array([self.k[f] for f in self.FIELDS], np.int32)
        self.starts = np.concatenate([[0], np.cumsum([n for _, n in lens])]).astype(np.int32)
        self.keys = np.array([p + n for p, n in lens], np.int32)

    def tiles(self, host):
        out, keys = np.zeros((100000, 5), np.int64), np.zeros(2000000, np.int64)
        n = host.tiles(ptr(self.c), ptr(self.starts), ptr(self.keys), ptr(out), ptr(keys), ctypes.c_long(keys.size))
        out = out[:n]
        ends = np.cumsum(out[:, 4])
        assert not n or ends[-1] <= keys.size
        return out, [keys[e - s:e] for e, s in zip(ends, out[:, 4])]

    def deal(self, host):
        out = np.zeros((400000, 6), np.int64)
        return out[:host.deal(ptr(self.c), ptr(self.starts), ptr(self.keys), ptr(out))]

    def seen(self, pos):
        """(sink keys, first key, end) that a token sees of a request's keys (before they end)."""
        if self.k["mask"] == 2:
            return 0, 0, 2 ** 31
        if self.k["mask"] == 0:
            return 0, 0, pos + 1
        lo = max(pos - self.k["window"] + 1, 0)
        return min(self.k["sinks"], pos + 1), lo, pos + 1


MASKS = [dict(), dict(mask=2), dict(mask=1, window=40, sinks=3), dict(mask=1, window=1), dict(mask=1, window=0, sinks=70), dict(mask=1, window=-5),
         dict(mask=1, window=100, sinks=64), dict(mask=1, window=10 ** 6, sinks=500)]
LENS = {
    "decode": [(0, 1), (1, 1), (15, 1), (16, 1), (777, 1), (64, 1), (0, 0), (2000, 1)],
    "mixed": [(40, 1), (0, 0), (0, 90), (513, 1), (9, 200), (0, 0), (127, 3), (1500, 33)],
    "one": [(4096, 1)],
    "chunk": [(700, 300)],
}
WORK = [dict(rows=16, step=32, least=4, unit=12), dict(rows=32, step=16, least=8, unit=24), dict(rows=128, step=64, least=2, unit=6),
        dict(rows=128, step=64, least=2, unit=6, few=32), dict(rows=16, step=32, least=4, unit=12, many=32)]


@pytest.mark.parametrize("mask", MASKS, ids=str)
@pytest.mark.parametrize("lens", list(LENS))
def test_steps_hold_every_visible_key_once(host, lens, mask):
    for work in WORK:
        check_steps(host, lens, mask, work)


def check_steps(host, lens, mask, work):
    plan = Plan(LENS[lens], **mask, **work)
    G, step = plan.k["Nq"] // plan.k["Nkv"], plan.k["step"]
    tiles, steps = plan.tiles(host)
    rows = {r: n * G for r, (_, n) in enumerate(plan.lens) if plan.k["few"] < n * G <= plan.k["many"]}
    covered = {r: np.zeros(n, int) for r, n in rows.items()}
    for (r, t, r0, r1, n), first in zip(tiles, steps):
        assert r0 == t * plan.k["rows"] and r0 < r1 <= min(r0 + plan.k["rows"], rows[r])
        covered[r][r0:r1] += 1
        past, new = plan.lens[r]
        assert n >= 1 and (first % step == 0).all()
        # increasing, so no key is in two steps
        assert (np.diff(first) >= step).all()
        held = np.zeros(past + new + 2 * step + first.max(), bool)
        for f in first:
            held[f:f + step] = True
        for token in range(r0 // G, (r1 - 1) // G + 1):
            sink, lo, hi = plan.seen(past + token)
            hi = min(hi, past + new)
            assert held[:min(sink, hi)].all() and held[min(lo, hi):hi].all()
    assert all((c == 1).all() for c in covered.values())


@pytest.mark.parametrize("workers", [1, 2, 7, 64, 512])
@pytest.mark.parametrize("lens", list(LENS))
def test_pieces_hold_every_step_once(host, lens, workers):
    for work, heads, mask in itertools.product(WORK, [(8, 2), (3, 3), (5, 1), (64, 16)], (MASKS[0], MASKS[2], MASKS[4])):
        plan = Plan(LENS[lens], **mask, **work, Nq=heads[0], Nkv=heads[1], workers=workers)
        tiles, _ = plan.tiles(host)
        units = {(t, h): [] for t in range(len(tiles)) for h in range(heads[1])}
        states = set()
        told = {}
        for worker, tile, head, lo, hi, sharers in plan.deal(host).tolist():
            n = tiles[tile][4]
            assert 0 <= lo <= hi <= n
            if sharers:
                told[worker] = ((tile, head), sharers)
            if lo == hi:
                assert not sharers
                continue
            units[tile, head].append((lo, hi, worker))
            if (lo, hi) != (0, n):  # its state goes to one of its worker's two places
                place = (worker, lo == 0)
                assert place not in states
                states.add(place)
        shared = {}
        for (tile, head), pieces in units.items():
            assert [p[0] for p in pieces] == [0] + [p[1] for p in pieces[:-1]] and pieces[-1][1] == tiles[tile][4]
            by = [p[2] for p in pieces]
            assert by == list(range(by[0], by[0] + len(by)))
            if len(pieces) > 1:
                shared[by[0]] = ((tile, head), len(by))
        assert told == shared


def test_deals_of_random_calls(host):
    g = np.random.default_rng(3)
    for _ in range(150):
        lens = [(int(p), int(n)) for p, n in zip(np.exp(g.uniform(0, 8, 40)).astype(int), g.choice([0, 1, 1, 1, 2, 9, 60], 40))]
        nkv = int(g.integers(1, 9))
        w = WORK[g.integers(len(WORK))]
        plan = Plan(lens, **MASKS[g.integers(len(MASKS))], **w, Nkv=nkv, Nq=nkv * int(g.integers(1, 9)), workers=int(g.integers(1, 600)))
        tiles, _ = plan.tiles(host)
        steps = {}
        load = np.zeros(plan.k["workers"])
        for worker, tile, head, lo, hi, _ in plan.deal(host).tolist():
            steps[tile, head] = steps.get((tile, head), 0) + hi - lo
            load[worker] += hi - lo
        assert {k: v for k, v in steps.items() if v} == {(t, h): tiles[t][4] for t in range(len(tiles)) for h in range(nkv)}
        total = (tiles[:, 4] + plan.k["unit"]).sum() * nkv
        assert load.max(initial=0) <= max(-(-total // plan.k["workers"]), plan.k["least"])


def test_wide_numbers(host):
    out = (ctypes.c_uint32 * 5)()
    u64, u32 = ctypes.c_uint64, ctypes.c_uint32
    big = 2 ** 31 // 16 + 3  # steps of a unit of 2^31 keys
    for units in (0, 1, 1000, 2 ** 24):
        for into in (0, 5, 24, 25, big + 23):
            for left in (1, 30, big, 2 ** 40):
                host.piece(u64(units * (big + 24) + into), u64(left), u32(big), u32(24), out)
                hi = min(into + left, big + 24)
                assert list(out) == [units, max(into, 24) - 24, max(hi, 24) - 24, hi - into, big + 24 - hi]
    for at in (0, 5, 2 ** 32 - 1, 2 ** 32, 2 ** 45 + 7):
        for share in (1, 3, 2 ** 32 - 1, 2 ** 33):
            if at // share < 2 ** 32:
                assert host.worker_of(u64(at), u64(share)) & 0xffffffff == at // share
