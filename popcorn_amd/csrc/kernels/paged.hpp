// Index arithmetic of the paged cache, shared by its kernels and (compiled
// for the host) their tests. Lengths and tables come from device memory and
// are not checked before a launch, so every number read is brought into range
// here: no value of theirs leads outside the tensors.
#pragma once

#include <stdint.h>

#include "popcorn_kernel_types.h"

#if defined(__HIPCC__)
#define PAGED_FN __host__ __device__ inline
#else
#define PAGED_FN inline
#endif

namespace pk {

PAGED_FN int32_t paged_min(int32_t a, int32_t b) { return a < b ? a : b; }
PAGED_FN int32_t paged_max(int32_t a, int32_t b) { return a > b ? a : b; }

// One request of a paged attention call: its new tokens are rows start ..
// start + n - 1, token i at position pos0 + i (negative where the request has
// fewer keys than new tokens), and its first `keys` keys lie in its pages.
struct PagedRequest {
    int32_t start, n, pos0, keys;
};

PAGED_FN PagedRequest paged_request(int32_t first, int32_t next, int32_t keyLen, const PagedAttentionConstants &p) {
    PagedRequest r;
    r.start = paged_min(paged_max(first, 0), (int32_t)p.T);
    r.n = paged_min(paged_max(next, r.start), (int32_t)p.T) - r.start;
    const int32_t len = paged_max(keyLen, 0);
    const uint64_t room = (uint64_t)p.columns * p.pageSize;
    r.pos0 = len - r.n;
    r.keys = (uint64_t)len < room ? len : (int32_t)room;
    return r;
}

// Keys that some of the positions first .. last see: [0, sinkEnd) and [lo, hi).
struct PagedSpan {
    int32_t sinkEnd, lo, hi;
};

PAGED_FN PagedSpan paged_span(int32_t first, int32_t last, int32_t keys, const PagedAttentionConstants &p) {
    PagedSpan s;
    s.hi = p.maskKind == 2u || last >= keys ? keys : paged_max(last + 1, 0);
    s.lo = 0;
    s.sinkEnd = 0;
    if (p.maskKind == 1u) {
        const int64_t lo = (int64_t)first - p.slidingWindow + 1;
        s.lo = lo <= 0 ? 0 : lo < s.hi ? (int32_t)lo : s.hi;
        s.sinkEnd = p.sinks < (uint32_t)s.lo ? (int32_t)p.sinks : s.lo;
    }
    return s;
}

PAGED_FN bool paged_sees(int32_t pos, int32_t key, const PagedAttentionConstants &p) {
    return (p.maskKind == 2u) | ((key <= pos) & ((p.maskKind == 0u) | ((int64_t)pos - key < p.slidingWindow) | ((uint32_t)key < p.sinks)));
}

// The plan of a launch: entry 0 holds the counted steps of all tiles (of one
// KV head) and the number of tiles, entry 1 + i tile i with those before it.
struct PagedTile {
    uint64_t before;
    uint32_t request, tile;
};

// Tile `tile` of request r: rows r0 .. r1 - 1 of its n * G, and its steps: sink
// steps from key 0, then the others from step `first`. A tile without a visible key has one
// step, so that its rows are written.
struct PagedSteps {
    uint32_t r0, r1, sinks, first, n;
};

PAGED_FN PagedSteps paged_steps(const PagedRequest &r, uint32_t tile, const PagedAttentionConstants &p, const PagedWorkConstants &w) {
    const uint32_t G = p.Nq / p.Nkv, rows = (uint32_t)r.n * G;
    PagedSteps s;
    s.r0 = tile * w.rows;
    s.r1 = rows - s.r0 < w.rows ? rows : s.r0 + w.rows;
    const PagedSpan k = paged_span(r.pos0 + (int32_t)(s.r0 / G), r.pos0 + (int32_t)((s.r1 - 1) / G), r.keys, p);
    const uint32_t step = w.stepKeys;
    s.sinks = ((uint32_t)k.sinkEnd + step - 1) / step;
    s.first = (uint32_t)k.lo / step > s.sinks ? (uint32_t)k.lo / step : s.sinks;
    const uint32_t end = k.hi > k.lo ? ((uint32_t)k.hi + step - 1) / step : 0u;
    s.n = s.sinks + (end > s.first ? end - s.first : 0u);
    if (s.n == 0) s.n = 1;
    return s;
}

// First key of step `step` of a tile.
PAGED_FN uint32_t paged_step_key(const PagedSteps &s, uint32_t step, const PagedWorkConstants &w) {
    return (step < s.sinks ? step : step - s.sinks + s.first) * w.stepKeys;
}

// Steps per worker, for `total` steps of all units.
PAGED_FN uint64_t paged_share(uint64_t total, const PagedWorkConstants &w) {
    const uint64_t q = (total + w.workers - 1) / w.workers;
    return q > w.minSteps ? q : w.minSteps;
}

// The worker of counted step `at` of all units. (A division of 64 bits takes ten times as long as one of 32.)
PAGED_FN uint32_t paged_worker(uint64_t at, uint64_t share) {
    return (at | share) >> 32 ? (uint32_t)(at / share) : (uint32_t)at / (uint32_t)share;
}

// What a worker takes next of a tile's units, one per KV head: steps lo .. hi - 1 of head hkv's, none where it reaches the unit's
// extra count only. `in`: counted steps of the units before the worker's place; `left`: counted steps to the end of its stretch;
// n: steps of a unit.
struct PagedPiece {
    uint32_t hkv, lo, hi;
    uint32_t taken, behind;  // counted steps of it, and of the unit behind it
};

// (hi as it stands: compared in 32 bits it made the few-row kernels 300 instructions longer, 64 requests' decode 137.5 -> 139.6 us.)
PAGED_FN PagedPiece paged_piece(uint64_t in, uint64_t left, uint32_t n, const PagedWorkConstants &w) {
    const uint32_t all = n + w.unitSteps;
    PagedPiece c;
    c.hkv = in >> 32 ? (uint32_t)(in / all) : (uint32_t)in / all;
    const uint32_t lo = (uint32_t)(in - (uint64_t)c.hkv * all), hi = (uint32_t)(lo + left < all ? lo + left : all);
    c.lo = (lo > w.unitSteps ? lo : w.unitSteps) - w.unitSteps;
    c.hi = (hi > w.unitSteps ? hi : w.unitSteps) - w.unitSteps;
    c.taken = hi - lo;
    c.behind = all - hi;
    return c;
}

// How many workers share the unit of a worker's last piece, where the piece begins the unit and leaves some of it (its stretch
// ends at `end`); else 0.
PAGED_FN uint32_t paged_sharers(const PagedPiece &c, uint32_t n, uint64_t end, uint64_t share, uint32_t worker) {
    return c.lo == 0 && c.hi > 0 && c.hi < n ? paged_worker(end + c.behind - 1, share) - worker + 1 : 0u;
}

}  // namespace pk
