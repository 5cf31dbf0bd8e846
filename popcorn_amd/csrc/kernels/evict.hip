// Eviction from a paged cache by weight, and the pages that it leaves empty.
//   n = min(keys, budget), first' = min(first, n), last' = min(last, n - first'): a KV head of a request keeps its first' first
//   and last' last keys and, of those between, the n - first' - last' of the highest weight (ties: the lowest index; NaN is
//   the lowest weight). evict_select says which, in index order, and evict_move brings their rows to the front.
// The choice is bound by its passes, the moves by rows that lie apart: 48 requests of 300 to 8000 keys cut to 1000, 8 heads of 128 in
// 16 bits take 14 us and 58 (120 MB read, 115 MB written: 4.1 TB/s, where a copy of 2 GiB reaches 4.85).
#include "paged.hpp"
#include "scan.hpp"

namespace {

// Whole numbers in the order of the weights: NaN 0, then from -infinity on, both zeros alike.
__device__ inline uint32_t rank_key(float x) {
    if (x != x) return 0u;
    const uint32_t b = __float_as_uint(x + 0.0f);  // (-0 + 0 is 0)
    return b >> 31 ? ~b : b | 0x80000000u;
}

constexpr uint32_t kBins = 2048;
constexpr uint32_t kTile = 4096;  // weights of a block's pass, four in a row to a thread
constexpr uint32_t kHeld = 4;     // passes whose weights a block holds in registers
// Counters of a bin, the even threads' and the odd ones': additions of a wave to one word take a cycle each. (One request of 4 heads
// of 8191 weights, uniform in 0 to 1, in 1 to 1.05, all equal: 16, 18 and 23 us with short rows' moves; with one counter 17, 22 and 33;
// with four 17, 17 and 18, but 48 requests' 8 heads 16 us instead of 15.) For more weights than a block holds
// eight (8 heads of 100000, the choice alone: 78, 80 and 83 us; with two 76, 106 and 171).
constexpr uint32_t kHeldCopies = 2, kLongCopies = 8, kBinStride = kBins + 8;

struct SelectSpace {
    __attribute__((aligned(16))) uint32_t bins[kBinStride * kLongCopies];
    uint32_t sums[16], found[3][2];
};

// HELD: all weights are read once, into registers, a thread's in a row; else again for each count and for the choice, tile by tile.
template <bool HELD>
__device__ inline void select_kept(const float *__restrict__ w, const pk::EvictKeep &k, int32_t *__restrict__ to, float *__restrict__ toW,
                                   SelectSpace &sp) {
    constexpr uint32_t kCopies = HELD ? kHeldCopies : kLongCopies;
    const uint32_t tid = threadIdx.x, tiles = (k.keys + kTile - 1) / kTile;
    struct Four {
        float v[4];
    };
    auto first_of = [&](uint32_t tile) { return HELD ? (tid * tiles + tile) * 4 : tile * kTile + tid * 4; };
    // read without a branch, so that the next read need not wait for it; the last weights, where a thread has fewer than four, again
    auto read = [&](uint32_t tile) {
        Four f{};
        if (k.keys >= 4) __builtin_memcpy(&f, w + min(first_of(tile), k.keys - 4), sizeof(f));
        return f;
    };
    auto whole = [&](uint32_t tile, Four &f) {
        const uint32_t i = first_of(tile);
        if (i + 4 > k.keys) {
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) f.v[j] = i + j < k.keys ? w[i + j] : 0.0f;
        }
    };
    Four held[HELD ? kHeld : 1];
    if constexpr (HELD) {
#pragma unroll
        for (uint32_t t = 0; t < kHeld; ++t)
            if (t < tiles) held[t] = read(t);
#pragma unroll
        for (uint32_t t = 0; t < kHeld; ++t)
            if (t < tiles) whole(t, held[t]);
    }
    auto each = [&](auto &&body) {  // body(first index, its four weights)
        if constexpr (HELD) {
#pragma unroll
            for (uint32_t t = 0; t < kHeld; ++t)
                if (t < tiles) body(first_of(t), held[t]);
        } else {
            Four next = read(0);
            for (uint32_t t = 0; t < tiles; ++t) {
                Four f = next;
                if (t + 1 < tiles) next = read(t + 1);
                whole(t, f);
                body(first_of(t), f);
            }
        }
    };
    // a thread's two bins, in order from the highest
    pk::u32x2 *mine2 = reinterpret_cast<pk::u32x2 *>(sp.bins + kBins - 2 - 2 * tid);
    auto clear = [&] {
#pragma unroll
        for (uint32_t c = 0; c < kCopies; ++c) mine2[c * (kBinStride / 2)] = pk::u32x2{0u, 0u};
    };
    const uint32_t lo = k.first, hi = k.keys - k.last;  // between them `need` are kept
    uint32_t need = k.n - k.first - k.last, least = 0, shift = 32;
    if (need > 0) {
        clear();
        __syncthreads();
    }
    // (unrolled, so that its shifts are constants: 48 requests' 8 heads 13.7 us, and 15.1)
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
        if (need == 0) break;
        const uint32_t bits = pass < 2 ? 11u : 10u, above = shift;
        shift -= bits;
        each([&](uint32_t base, const Four &f) {
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                const uint32_t i = base + j, x = rank_key(f.v[j]);
                if (i >= lo && i < hi && (above == 32 || x >> above == least >> above))
                    atomicAdd(&sp.bins[(x >> shift & ((1u << bits) - 1)) + tid % kCopies * kBinStride], 1u);
            }
        });
        __syncthreads();
        // from the highest bin down: the bin where the need is met
        uint32_t a = 0, b = 0;
#pragma unroll
        for (uint32_t c = 0; c < kCopies; ++c) {
            const pk::u32x2 x = mine2[c * (kBinStride / 2)];
            a += x[1];
            b += x[0];
        }
        clear();
        const pk::Scan<uint32_t> s = pk::block_scan<16>(a + b, sp.sums);
        const uint32_t beforeA = s.upto - a - b, beforeB = beforeA + a;
        if (beforeA < need && need <= beforeB) {
            sp.found[pass][0] = kBins - 1 - 2 * tid;
            sp.found[pass][1] = need - beforeA;
        }
        if (beforeB < need && need <= s.upto) {
            sp.found[pass][0] = kBins - 2 - 2 * tid;
            sp.found[pass][1] = need - beforeB;
        }
        __syncthreads();
        least |= sp.found[pass][0] << shift;
        need = sp.found[pass][1];
    }
    // `need` of those at `least` are kept, the lowest indices; where none between is, nothing is above
    const bool none = k.n == k.first + k.last;
    auto is_kept = [&](uint32_t i, float v, bool &sure, bool &tie) {
        const bool between = i >= lo && i < hi;
        const uint32_t x = rank_key(v);
        sure = i < k.keys && (!between || (!none && x > least));
        tie = between && !none && x == least;
    };
    auto count = [&](uint32_t base, const Four &f) {  // of both, 16 bits each (a block's are at most 16384)
        uint32_t n = 0;
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            bool sure, tie;
            is_kept(base + j, f.v[j], sure, tie);
            n += (uint32_t)sure | (uint32_t)tie << 16;
        }
        return n;
    };
    // a, b: of both, those before it
    auto write = [&](uint32_t base, const Four &f, uint32_t &a, uint32_t &b) {
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            bool sure, tie;
            is_kept(base + j, f.v[j], sure, tie);
            if (sure || (tie && b < need)) {
                const uint32_t at = a + min(b, need);
                to[at] = (int32_t)(base + j);
                toW[at] = f.v[j];
            }
            a += sure;
            b += tie;
        }
    };
    if constexpr (HELD) {
        uint32_t mine = 0;
        each([&](uint32_t base, const Four &f) { mine += count(base, f); });
        const uint32_t before = pk::block_scan<16>(mine, sp.sums).upto - mine;
        uint32_t a = before & 0xffffu, b = before >> 16;
        each([&](uint32_t base, const Four &f) { write(base, f, a, b); });
    } else {
        uint32_t sure = 0, ties = 0;  // before this tile
        each([&](uint32_t base, const Four &f) {
            const uint32_t mine = count(base, f);
            const pk::Scan<uint32_t> s = pk::block_scan<16>(mine, sp.sums);
            uint32_t a = sure + ((s.upto - mine) & 0xffffu), b = ties + ((s.upto - mine) >> 16);
            write(base, f, a, b);
            sure += s.total & 0xffffu;
            ties += s.total >> 16;
        });
    }
}

}  // namespace

// A block per (request, KV head). The least kept weight by three counts of its bits (11, 11 and 10), then one pass in
// order that numbers what is kept: no sort, and no atomics but the counts', so equal weights leave the lowest index whatever
// the order of waves. Up to 16384 weights stay in registers between the passes (8191 of them: 9 us; read for each pass, 14). One request's
// 4 heads leave 252 CUs idle; several blocks to a head would have to wait for each other's counts three times (one of 100000 keys, cut to
// a quarter: 80 us).
POPCORN_KERNEL void __launch_bounds__(1024, 8)
    evict_select(const float *weights, const int32_t *keyLens, const int32_t *budgets, int32_t *kept, float *keptWeights, EvictConstants e) {
    __shared__ SelectSpace space;
    const uint32_t tid = threadIdx.x, r = blockIdx.x / e.Nkv;
    const uint64_t room = (uint64_t)e.columns * e.pageSize;
    const pk::EvictKeep k = pk::evict_keep(keyLens[r], budgets[r], e);
    const float *w = weights + blockIdx.x * room;
    int32_t *to = kept + blockIdx.x * room;
    float *toW = keptWeights + blockIdx.x * room;
    if (k.n == k.keys) {
        for (uint32_t i = tid; i < k.n; i += 1024) {
            to[i] = (int32_t)i;
            toW[i] = w[i];
        }
    } else if (k.keys <= kHeld * kTile) {
        select_kept<true>(w, k, to, toW, space);
    } else {
        select_kept<false>(w, k, to, toW, space);
    }
    for (uint64_t i = k.n + tid; i < room; i += 1024) toW[i] = 0.0f;
}

namespace {

// In place, since a step has no spare cache: a kept row only ever moves to the front.
// A block takes e.units units of U (its slice) of the rows of one (request, KV head) in K or V. Row j becomes row kept[j] >= j, in chunks from
// the front: a chunk's rows are all read before one of them is written, and what later chunks read lies behind what it
// writes (kept rises, so kept[j] >= j for them too).
template <typename U>
__device__ void evict_move(const int32_t *__restrict__ kept, const int32_t *__restrict__ tables, const int32_t *__restrict__ keyLens,
                           const int32_t *__restrict__ budgets, U *kCache, U *vCache, const EvictConstants &e) {
    constexpr uint32_t kDeep = 4;
    const uint32_t rows = 1024 / e.units, chunk = rows * kDeep;
    const uint32_t of = blockIdx.x, r = of / e.Nkv, hkv = of % e.Nkv;
    const pk::EvictKeep k = pk::evict_keep(keyLens[r], budgets[r], e);
    if (k.n == k.keys) return;
    const uint64_t room = (uint64_t)e.columns * e.pageSize;
    const int32_t *from = kept + of * room, *table = tables + (uint64_t)r * e.columns;
    U *cache = blockIdx.z ? vCache : kCache;
    const uint32_t unit = blockIdx.y * e.units + threadIdx.x % e.units, row = threadIdx.x / e.units;
    const bool mine = unit < e.rowUnits;
    auto page_of = [&](uint32_t i) { return (uint32_t)table[i / e.pageSize]; };
    auto at = [&](uint32_t page, uint32_t i) {
        return cache + (((uint64_t)page * e.Nkv + hkv) * e.pageSize + i % e.pageSize) * e.rowUnits + unit;
    };
    for (uint32_t base = k.first; base < k.n; base += chunk) {
        // step by step for all kDeep rows, so that their reads stand side by side (row by row 69 us, and 58; with the next chunk's rows read
        // before these are written, in registers that leave a CU one block, 104)
        U v[kDeep];
        uint32_t i[kDeep], page[kDeep], to[kDeep];  // `to`: the page; none where the row stays
#pragma unroll
        for (uint32_t d = 0; d < kDeep; ++d) i[d] = (uint32_t)from[min(base + d * rows + row, k.n - 1)];
#pragma unroll
        for (uint32_t d = 0; d < kDeep; ++d) {
            // (what is kept lies at or behind its place; a list that another call has left leads nowhere else)
            i[d] = min(i[d], k.keys - 1);
            page[d] = page_of(i[d]);
            to[d] = page_of(min(base + d * rows + row, k.n - 1));
        }
#pragma unroll
        for (uint32_t d = 0; d < kDeep; ++d) {
            const uint32_t j = base + d * rows + row;
            if (!(mine && j < k.n && i[d] > j && page[d] < e.pages && to[d] < e.pages)) to[d] = ~0u;
            if (to[d] != ~0u) v[d] = *at(page[d], i[d]);
        }
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): the rows have been read
        __syncthreads();
#pragma unroll
        for (uint32_t d = 0; d < kDeep; ++d)
            if (to[d] != ~0u) *at(to[d], base + d * rows + row) = v[d];
    }
}

}  // namespace

#define EVICT_MOVE(name, U)                                                                                                   \
    POPCORN_KERNEL void __launch_bounds__(1024, 8) name(const int32_t *kept, const int32_t *tables, const int32_t *keyLens,      \
                                                     const int32_t *budgets, U *kCache, U *vCache, EvictConstants e) {        \
        evict_move<U>(kept, tables, keyLens, budgets, kCache, vCache, e);                                                     \
    }
EVICT_MOVE(evict_move_b128, pk::u32x4)
EVICT_MOVE(evict_move_b64, pk::u32x2)
EVICT_MOVE(evict_move_b32, uint32_t)
EVICT_MOVE(evict_move_b16, uint16_t)

// The lengths after an eviction, and the pages from ceil(n / pageSize) on of each request that it left empty, in request order.
// Every block sums what the requests before its own free.
POPCORN_KERNEL void __launch_bounds__(256)
    release_pages(const int32_t *keyLens, const int32_t *budgets, const int32_t *tables, int32_t *newLens, int32_t *freed, int32_t *counts,
                  EvictConstants e) {
    __shared__ uint32_t sums[4], sBefore[256], sFrom[256], sCount[256];
    const uint32_t tid = threadIdx.x;
    const uint32_t lo = (uint32_t)((uint64_t)e.R * blockIdx.x / gridDim.x), hi = (uint32_t)((uint64_t)e.R * (blockIdx.x + 1) / gridDim.x);
    auto pages = [&](uint32_t keys) { return keys / e.pageSize + (keys % e.pageSize != 0); };
    uint32_t run = 0;
    auto wave_total = [&](uint32_t v) {
        const pk::Scan<uint32_t> s = pk::block_scan<4>(v, sums);
        return s;
    };
    {
        uint32_t mine = 0;
        for (uint32_t r = tid; r < lo; r += 256) {
            const pk::EvictKeep k = pk::evict_keep(keyLens[r], budgets[r], e);
            mine += pages(k.keys) - pages(k.n);
        }
        run = wave_total(mine).total;
    }
    for (uint32_t base = lo; base < hi; base += 256) {
        const uint32_t r = base + tid;
        uint32_t count = 0, from = 0;
        if (r < hi) {
            const pk::EvictKeep k = pk::evict_keep(keyLens[r], budgets[r], e);
            from = pages(k.n);
            count = pages(k.keys) - from;
            newLens[r] = (int32_t)k.n;
        }
        const pk::Scan<uint32_t> s = wave_total(count);
        sBefore[tid] = run + s.upto - count;
        sFrom[tid] = from;
        sCount[tid] = count;
        __syncthreads();
        for (uint32_t i = tid / 64; i < min(256u, hi - base); i += 4)
            for (uint32_t c = tid % 64; c < sCount[i]; c += 64) freed[sBefore[i] + c] = tables[(uint64_t)(base + i) * e.columns + sFrom[i] + c];
        run += s.total;
        __syncthreads();
    }
    if (blockIdx.x == gridDim.x - 1 && tid == 0) counts[0] = (int32_t)run;
}
