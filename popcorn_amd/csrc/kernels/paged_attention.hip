// Attention of the new tokens of a batch of requests over a paged cache
// [pages, Nkv, pageSize, Hd]: out = softmax(scale q K^T | visible keys) V per
// request, query heads in groups per KV head, with the lengths and the pages
// read on the GPU.
#include <type_traits>

#include "mfma.hpp"
#include "paged.hpp"
#include "scan.hpp"

namespace {

constexpr float kLog2e = 1.4426950408889634f;

// One row's O, m (log2 units) and l over those of the keys [k0, k1) that it
// sees, in f32 on the vector ALUs with weights of at most 1. 16 lanes per
// row, lane t's dims 4 t + 64 j; VEC: rows in whole, aligned fours. Of `of`
// such groups of lanes, this one takes every of-th run of keys, from the nth on.
// U keys in flight.
template <typename T, int NJ, bool VEC, uint32_t U>
__device__ inline void paged_row(const pk::f32x4 (&q)[NJ], const typename T::storage *__restrict__ K,
                                 const typename T::storage *__restrict__ V, const int32_t *__restrict__ table, uint32_t hkv,
                                 int pos, int k0, int k1, const PagedAttentionConstants &p, pk::f32x4 (&o)[NJ], float &m, float &l,
                                 uint32_t nth = 0, uint32_t of = 1) {
    const uint32_t D = p.Hd;
    uint32_t td = threadIdx.x % 16 * 4;
    asm volatile("" : "+v"(td));  // (what follows from it is computed here, and held through no caller's loop)
    const float c2 = p.scale * kLog2e;
    using Four = std::conditional_t<sizeof(typename T::storage) == 4, pk::f32x4, pk::u32x2>;
    // (past the row's end its last elements again, so that no load waits for a branch, and zeros instead of them)
    auto load = [&](const typename T::storage *row, int j) {
        const uint32_t d = td + 64 * j;
        Four v;
        if constexpr (VEC) {
            v = *reinterpret_cast<const Four *>(row + min(d, D - 4));
        } else {
            typename T::storage e[4];
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) e[i] = row[min(d + i, D - 1)];
            __builtin_memcpy(&v, e, sizeof(v));
        }
        return v;
    };
    auto value = [&](const Four &v, int j, int i) {
        float x;
        if constexpr (sizeof(typename T::storage) == 4) x = v[i];
        else x = pk::from_bits16<T>(i % 2 ? v[i / 2] >> 16 : v[i / 2] & 0xffffu);
        return td + 64 * j + i < D ? x : 0.0f;
    };
    if (p.pages == 0) return;  // (a key that no page holds is read from page 0, and left out)
    for (uint64_t at = (uint64_t)(uint32_t)k0 + nth * U; at < (uint32_t)k1; at += of * U) {
        const uint32_t k = (uint32_t)at;
        Four kv[U][NJ], vv[U][NJ];
        bool in[U];
        uint32_t page[U], left[U];
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            const uint32_t key = min(k + u, (uint32_t)k1 - 1), column = key / p.pageSize;
            page[u] = (uint32_t)table[column];
            left[u] = key - column * p.pageSize;
        }
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            in[u] = page[u] < p.pages && k + u < (uint32_t)k1;
            const uint64_t row = (((uint64_t)(page[u] < p.pages ? page[u] : 0u) * p.Nkv + hkv) * p.pageSize + left[u]) * D;
#pragma unroll
            for (int j = 0; j < NJ; ++j)
                if (64u * j < D) {
                    kv[u][j] = load(K + row, j);
                    vv[u][j] = load(V + row, j);
                }
        }
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            float s = 0.0f;
#pragma unroll
            for (int j = 0; j < NJ; ++j)
                if (64u * j < D)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s = fmaf(q[j][i], value(kv[u][j], j, i), s);
            s = pk::group_sum<16>(s) * c2;
            if (!in[u] || !pk::paged_sees(pos, (int)(k + u), p)) continue;  // a row's lanes together
            const float mn = fmaxf(m, s);
            if (mn == -INFINITY && s == -INFINITY) continue;  // (a NaN is not left out)
            const float alpha = __builtin_amdgcn_exp2f(m - mn), w = __builtin_amdgcn_exp2f(s - mn);
            l = l * alpha + w;
            m = mn;
#pragma unroll
            for (int j = 0; j < NJ; ++j)
                if (64u * j < D)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[j][i] = fmaf(value(vv[u][j], j, i), w, o[j][i] * alpha);
        }
    }
}


// ---- the plan ----------------------------------------------------------------------

__device__ inline uint32_t first_lane(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ inline uint64_t first_lane64(uint64_t v) {
    return (uint64_t)first_lane((uint32_t)(v >> 32)) << 32 | first_lane((uint32_t)v);
}

template <uint32_t N, typename U>
struct PlanSpace {  // of a block of N threads
    U sums[N / 64];
    uint32_t tile[N];
    pk::PagedRequest req[N];
};

// The tiles of every request, in request order: put(tile, steps before, request, tile of it).
template <uint32_t N, typename U, typename Put>
__device__ inline void lay_tiles(const int32_t *starts, const int32_t *keyLens, PlanSpace<N, U> &sp, const PagedAttentionConstants &p,
                                 const PagedWorkConstants &w, U &steps, uint32_t &tiles, Put &&put) {
    const uint32_t tid = threadIdx.x, G = p.Nq / p.Nkv;
    steps = 0;
    tiles = 0;
    for (uint32_t base = 0; base < p.R; base += N) {
        const uint32_t r = base + tid;
        pk::PagedRequest q{0, 0, 0, 0};
        if (r < p.R) q = pk::paged_request(starts[r], starts[r + 1], keyLens[r], p);
        const uint32_t rows = (uint32_t)q.n * G;
        const uint32_t mine = rows > w.fewRows && rows <= w.manyRows ? (rows + w.rows - 1) / w.rows : 0u;
        const pk::Scan<U> of = pk::block_scan<N / 64>((U)mine, sp.sums);
        const U upto = of.upto, total = of.total;
        // overlapping ranges of requests could hold more rows than there are: what passes the plan's room is left out
        const uint32_t here = (uint32_t)min(total, (U)(w.maxTiles - tiles));
        sp.tile[tid] = (uint32_t)min(upto - mine, (U)here);
        sp.req[tid] = q;
        __syncthreads();
        for (uint32_t t0 = 0; t0 < here; t0 += N) {
            const uint32_t t = t0 + tid;
            uint32_t i = 0, n = 0;
            if (t < here) {
#pragma unroll
                for (uint32_t d = N / 2; d; d >>= 1)
                    if (sp.tile[i + d] <= t) i += d;
                n = pk::paged_steps(sp.req[i], t - sp.tile[i], p, w).n + w.unitSteps;
            }
            const pk::Scan<U> sum = pk::block_scan<N / 64>((U)n, sp.sums);
            if (t < here) put(tiles + t, steps + sum.upto - n, base + i, t - sp.tile[i]);
            steps += sum.total;
        }
        tiles += here;
        __syncthreads();
    }
}

typedef uint64_t u64;

}  // namespace

POPCORN_KERNEL void __launch_bounds__(1024)
    paged_plan(const int32_t *starts, const int32_t *keyLens, pk::PagedTile *plan, PagedAttentionConstants p, PagedWorkConstants w) {
    __shared__ PlanSpace<1024, u64> space;
    u64 steps;
    uint32_t tiles;
    lay_tiles<1024, u64>(starts, keyLens, space, p, w, steps, tiles, [&](uint32_t at, u64 before, uint32_t request, uint32_t tile) {
        plan[1 + at] = pk::PagedTile{before, request, tile};
    });
    if (threadIdx.x == 0) plan[0] = pk::PagedTile{steps, tiles, 0};
}

namespace {

// ---- a few rows per KV head: decode and drafts ------------------------------------------------

constexpr int kWaves = 4;
constexpr float kRescaleGap = 8.0f * kLog2e;  // log2 units, as the maxima
constexpr int kOutOfRange = (int)0x80000000u;  // past every page: zeros

typedef __attribute__((address_space(3))) void lds_void;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
using pk::f32x16;
using pk::u32x2;
using pk::u32x4;

__device__ inline float quad16_max(float v) { return pk::pair32_max(pk::pair16_max(v)); }
__device__ inline float quad16_sum(float v) { return pk::pair32_sum(pk::pair16_sum(v)); }

template <int N>
__device__ inline void wait_vmcnt() {
    static_assert(N >= 0 && N < 64, "vmcnt range");
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}

// Tiles that a block lays out by itself, in LDS.
constexpr uint32_t kOwnTiles = 1024;
struct OwnTile {
    uint32_t before, place;  // request << 16 | tile
};

// The tile whose units hold step x: the last with before * Nkv <= x. A wave's
// lanes look at 64 entries at once.
template <typename Before>
__device__ inline uint32_t find_tile(uint32_t tiles, uint64_t at, Before &&before) {
    uint32_t lo = 0, n = tiles;
    while (n > 1) {
        const uint32_t stride = (n + 63) / 64, i = (threadIdx.x & 63) * stride;
        const bool in = i < n && before(lo + i) <= at;
        const uint32_t last = 63 - __clzll(__ballot(in));  // lane 0's entry is always at or before x
        const uint32_t from = last * stride;
        n = min(stride, n - from);
        lo += from;
    }
    return first_lane(lo);
}

// A stretch [lo, hi) of one unit's steps, empty where it is of the unit's extra
// count only.
struct Piece {
    pk::PagedRequest req;
    pk::PagedSteps steps;
    uint32_t request, hkv, lo, hi;
};

// What a worker's last piece leaves to the merge: nothing (pieces 0), or the
// rows r0 .. r1 - 1 of a unit that it begins and `pieces` workers share. Worker
// w's two states are `rows` rows each, from row base + 2 w rows on.
struct Shared {
    uint32_t pieces, start, hkv, r0, r1, rows, base, worker;
};

// Deals a block of NT threads its pieces.
template <uint32_t NT>
struct Dealer {
    const pk::PagedTile *plan;
    const OwnTile *own;
    const int32_t *starts, *keyLens;
    Shared *shared;
    uint64_t share, x, end;
    uint32_t tile;

    // `space` is free again afterwards.
    __device__ inline Dealer(const int32_t *st, const int32_t *kl, const pk::PagedTile *pl, OwnTile *ow, PlanSpace<NT, uint32_t> &space,
                             Shared *sh, const PagedAttentionConstants &p, const PagedWorkConstants &w)
        : plan(pl), own(ow), starts(st), keyLens(kl), shared(sh + blockIdx.x) {
        uint32_t tiles;
        uint64_t total;
        if (w.ownPlan) {
            uint32_t steps;
            lay_tiles<NT, uint32_t>(starts, keyLens, space, p, w, steps, tiles, [&](uint32_t at, uint32_t before, uint32_t request, uint32_t t) {
                ow[at] = OwnTile{before, request << 16 | t};
            });
            total = (uint64_t)first_lane(steps) * p.Nkv;
            tiles = first_lane(tiles);
        } else {
            total = plan[0].before * p.Nkv;
            tiles = plan[0].request;
        }
        share = pk::paged_share(total, w);
        x = first_lane64(blockIdx.x * share);
        end = first_lane64(min(x + share, total));
        if (x < end) {
            tile = w.ownPlan ? find_tile(tiles, x >> 32 ? x / p.Nkv : (uint32_t)x / p.Nkv, [&](uint32_t i) { return own[i].before; })
                             : find_tile(tiles, x >> 32 ? x / p.Nkv : (uint32_t)x / p.Nkv, [&](uint32_t i) { return plan[1 + i].before; });
        } else if (threadIdx.x == 0) {
            shared->pieces = 0;
        }
    }

    // False at the end of the block's stretch.
    __device__ inline bool next(Piece &c, const PagedAttentionConstants &p, const PagedWorkConstants &w) {
        while (x < end) {
            pk::PagedTile t;
            if (w.ownPlan) {
                const OwnTile o = own[tile];
                t = pk::PagedTile{first_lane(o.before), first_lane(o.place >> 16), first_lane(o.place & 0xffffu)};
            } else {
                t = plan[1 + tile];
                t = pk::PagedTile{first_lane64(t.before), first_lane(t.request), first_lane(t.tile)};
            }
            c.request = t.request;
            c.req = pk::paged_request(starts[t.request], starts[t.request + 1], keyLens[t.request], p);
            c.steps = pk::paged_steps(c.req, t.tile, p, w);
            const pk::PagedPiece piece = pk::paged_piece(x - t.before * p.Nkv, end - x, c.steps.n, w);
            c.hkv = piece.hkv;
            c.lo = piece.lo;
            c.hi = piece.hi;
            x += piece.taken;
            if (piece.behind == 0 && c.hkv + 1 == p.Nkv) ++tile;
            if (x == end && threadIdx.x == 0) {
                Shared sh{0, (uint32_t)c.req.start, c.hkv, c.steps.r0, c.steps.r1, w.rows, w.stateBase, blockIdx.x};
                sh.pieces = pk::paged_sharers(piece, c.steps.n, end, share, blockIdx.x);
                *shared = sh;
            }
            if (c.lo < c.hi) return true;
        }
        return false;
    }
};

// The result of one row's lane of 4 dims, rounded.
template <typename T>
__device__ inline void store4(typename T::storage *dst, const pk::f32x4 &o, float l) {
    pk::f32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = l != 0.0f ? o[i] / l : 0.0f;
    if constexpr (sizeof(typename T::storage) == 4) {
        *reinterpret_cast<pk::f32x4 *>(dst) = v;
    } else {
        *reinterpret_cast<u32x2 *>(dst) = u32x2{pk::bits16<T>(v[0]) | pk::bits16<T>(v[1]) << 16, pk::bits16<T>(v[2]) | pk::bits16<T>(v[3]) << 16};
    }
}

// Tiles of 16 or 32 rows: S^T = K . Q^T on 16x16 products, so that a row's
// scores lie in four lanes and its weights are the next product's operand as
// they are. The block's waves take steps in turn (16 keys in f32, else 32),
// each with a softmax state of its own: K goes from memory to fragments, a step
// ahead, V into the wave's own LDS and from there by ds_read_b64_tr_b16, so
// waves wait for nobody until they are merged. 16-bit weights enter P . V as
// two numbers, which leaves out 2^-16 (bf16) or 2^-22 (f16) of each.
// What bounds it: reading K and V where there is enough of them (766 MB of 64
// requests in 136 us, 5.6 TB/s, with the merge), else the chain from lengths to
// table to keys to merge: one request of 4096 keys on 4 heads of 256 takes 12 us
// and 6 in the merge, and its 17 MB would take 3. Keys shared out among waves
// instead of rows because decoding has few rows; 32 rows only from 17 on (both
// sides where the kernel is chosen).
// A piece's partial state goes to one of its worker's two slots: 2 w + 1 if
// the piece begins its unit, else 2 w.
template <typename T, int HD, int RT>
__device__ void paged_few(const typename T::storage *__restrict__ Q, const typename T::storage *__restrict__ K,
                          const typename T::storage *__restrict__ V, const int32_t *__restrict__ tables,
                          const int32_t *__restrict__ starts, const int32_t *__restrict__ keyLens,
                          const pk::PagedTile *__restrict__ plan, float *__restrict__ pO, float *__restrict__ pML,
                          Shared *__restrict__ shared, typename T::storage *__restrict__ out, const PagedAttentionConstants &p,
                          const PagedWorkConstants &w) {
    using S = typename T::storage;
    constexpr bool kWide = sizeof(S) == 4;
    constexpr int KM = kWide ? 1 : 2;          // 16-key groups per step
    constexpr int BKV = 16 * KM, E = 16 / sizeof(S);
    constexpr int KS = HD / (4 * E);           // 16-byte pieces of a lane's K and Q rows
    constexpr int DT = HD / 16;                // 16-row tiles of O^T
    constexpr int CH = HD / E;                 // 16-byte chunks per row
    constexpr int kRowsPer = CH > 64 ? 1 : 64 / CH;  // V rows per copy instruction
    constexpr int kHalves = CH > 64 ? CH / 64 : 1;   // copy instructions per row
    constexpr int kParts = kWide ? 1 : 2;
    constexpr float kLead = std::is_same<T, pk::F16>::value ? 4.0f : 0.0f;  // max over reference when it moves
    constexpr int LDO = HD + 4;                // merged-state row, in floats
    constexpr int kStage = kWaves * BKV * HD * (int)sizeof(S), kMerge = kWaves * 16 * LDO * 4;
    __shared__ __attribute__((aligned(16))) uint8_t smem[kStage > kMerge ? kStage : kMerge];
    __shared__ float sm_m[kWaves][RT * 16], sm_l[kWaves][RT * 16];
    __shared__ OwnTile sm_plan[kOwnTiles];
    __shared__ uint32_t sm_bad;
    // Q of 512 dims in 16 bits is kept in LDS: in registers 60 of 512 spilled, so 4 (32 requests of 100 to 8000 keys, 8 heads
    // on 2: 48 us, and 99; 1000 tokens behind as many 148 and 438)
    constexpr bool kQInLds = HD == 512 && !kWide;
    // and in 32 bits, where LDS has no room for it, read again for each step (19 spilled; the same call 135 us, and 325)
    constexpr bool kQAgain = HD == 512 && kWide;
    __shared__ __attribute__((aligned(16))) u32x4 sm_q[kQInLds ? KS * 64 : 1];
    static_assert(sizeof(PlanSpace<64 * kWaves, uint32_t>) <= sizeof(smem), "the plan is laid out where V goes");

    const uint32_t lane = threadIdx.x & 63, g = lane >> 4, c16 = lane & 15;
    const uint32_t wave = first_lane(threadIdx.x >> 6);
    const uint32_t D = p.Hd, G = p.Nq / p.Nkv;
    const float c2 = p.scale * kLog2e;
    Dealer<64 * kWaves> dealer(starts, keyLens, plan, sm_plan, *reinterpret_cast<PlanSpace<64 * kWaves, uint32_t> *>(smem), shared, p, w);
    Piece c;
    while (dealer.next(c, p, w)) {
        const int32_t *table = tables + (uint64_t)c.request * p.columns;
        const uint32_t keys = (uint32_t)c.req.keys;
        auto q_row = [&](uint32_t r) { return ((uint64_t)(uint32_t)c.req.start + r / G) * p.Nq + c.hkv * G + r % G; };

        // rows past the tile's last repeat it and are not stored
        u32x4 qf[RT][kQInLds || kQAgain ? 1 : KS];
        const S *qAgain = Q;
        int posQ[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const uint32_t r = min(c.steps.r0 + rt * 16 + c16, c.steps.r1 - 1);
            posQ[rt] = c.req.pos0 + (int)(r / G);
            const S *row = Q + q_row(r) * D + g * E;
            auto piece = [&](int s) { return s * 4 * E + g * E < D ? *reinterpret_cast<const u32x4 *>(row + s * 4 * E) : u32x4{0u, 0u, 0u, 0u}; };
            if constexpr (kQInLds) {
                for (int s = wave; s < KS; s += kWaves) sm_q[s * 64 + lane] = piece(s);
            } else if constexpr (kQAgain) {
                qAgain = Q + q_row(r) * D;
            } else {
#pragma unroll
                for (int s = 0; s < KS; ++s) qf[rt][s] = piece(s);
            }
        }
        if constexpr (kQInLds) __syncthreads();

        // The wave's steps are c.lo + wave + kWaves i. Lane l holds page and row in it
        // of group l % KM of the wave's step `page0` + l / KM; a group that no
        // page holds has none (-1): its keys are left out and read as zeros.
        constexpr uint32_t kHeld = 64 / KM;
        uint32_t page0 = 0, heldPage = 0, heldRow = 0;
        auto hold = [&](uint32_t i) {
            const uint32_t step = c.lo + wave + kWaves * (i + lane / KM);
            page0 = i;
            heldPage = ~0u;
            heldRow = 0;
            if (step < c.hi) {
                const uint32_t key = pk::paged_step_key(c.steps, step, w) + lane % KM * 16, column = key / p.pageSize;
                if (key < keys) {
                    heldPage = (uint32_t)table[column];
                    heldRow = key - column * p.pageSize;
                }
            }
        };
        struct Group {
            __amdgpu_buffer_rsrc_t k, v;
            bool ok;
        };
        auto group = [&](uint32_t i, int mt, uint32_t key) {
            const uint32_t at = (i - page0) * KM + mt;
            const uint32_t page = (uint32_t)__builtin_amdgcn_readlane((int)heldPage, (int)at);
            const uint32_t row = (uint32_t)__builtin_amdgcn_readlane((int)heldRow, (int)at);
            Group gr;
            gr.ok = page < p.pages;
            const uint64_t off = gr.ok ? (((uint64_t)page * p.Nkv + c.hkv) * p.pageSize + row) * D : 0;
            const int bytes = gr.ok ? (int)(min(16u, keys - key) * D * (uint32_t)sizeof(S)) : 0;
            gr.k = __builtin_amdgcn_make_buffer_rsrc(const_cast<S *>(K + off), 0, bytes, 0x00020000);
            gr.v = __builtin_amdgcn_make_buffer_rsrc(const_cast<S *>(V + off), 0, bytes, 0x00020000);
            return gr;
        };

        u32x4 kf[KM][KS];
        Group gr[KM];
        auto loadK = [&](uint32_t i, uint32_t step) {
            const uint32_t key = step < c.hi ? pk::paged_step_key(c.steps, step, w) : keys;
#pragma unroll
            for (int mt = 0; mt < KM; ++mt) {
                gr[mt] = group(i, mt, key + mt * 16);
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    const uint32_t d = s * 4 * E + g * E;
                    const int off = d < D ? (int)((c16 * D + d) * sizeof(S)) : kOutOfRange;
                    kf[mt][s] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(gr[mt].k, off, 0, 0));
                }
            }
        };
        // V goes row-major into the wave's own tile, 16-byte chunks swizzled by the row (`swz`)
        uint8_t *sV = smem + wave * (BKV * HD * sizeof(S));
        auto swz = [](uint32_t row) { return kWide ? ((row >> 2) & 3u) << 2 : 2u * (row % 8u) % CH; };
        auto copyV = [&](const Group *from) {
#pragma unroll
            for (int mt = 0; mt < KM; ++mt)
#pragma unroll
                for (int i = 0; i < 16 / kRowsPer * kHalves; ++i) {
                    const uint32_t row = i / kHalves * kRowsPer + (kHalves > 1 ? 0u : lane / CH);
                    const uint32_t chunk = ((i % kHalves) * 64 + lane % CH) ^ swz(row);
                    const int off = chunk * E < D ? (int)((row * D + chunk * E) * sizeof(S)) : kOutOfRange;
                    lds_void *to = (lds_void *)(sV + (mt * 16 / kRowsPer * kHalves + i) * 1024);
                    if (w.stream) __builtin_amdgcn_raw_ptr_buffer_load_lds(from[mt].v, to, 16, off, 0, 0, 2);  // (not to be kept)
                    else __builtin_amdgcn_raw_ptr_buffer_load_lds(from[mt].v, to, 16, off, 0, 0, 0);
                }
        };

        pk::f32x4 acc[RT][DT];
        float m[RT], l[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            m[rt] = -INFINITY;
            l[rt] = 0.0f;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) acc[rt][dt] = pk::f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }

        hold(0);
        uint32_t i = 0;
        loadK(0, c.lo + wave);
        for (uint32_t step = c.lo + wave; step < c.hi; step += kWaves, ++i) {
            const uint32_t k0 = pk::paged_step_key(c.steps, step, w);
            bool ok[KM];
#pragma unroll
            for (int mt = 0; mt < KM; ++mt) ok[mt] = gr[mt].ok;
            if constexpr (!kQInLds) copyV(gr);
            pk::f32x4 st[RT][KM];
            if constexpr (kQInLds) {
                static_assert(RT == 1, "one tile's rows");
#pragma unroll
                for (int mt = 0; mt < KM; ++mt) st[0][mt] = pk::f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    const u32x4 q = sm_q[s * 64 + lane];
#pragma unroll
                    for (int mt = 0; mt < KM; ++mt) st[0][mt] = pk::Mma16<T>::run(kf[mt][s], q, st[0][mt]);
                }
                copyV(gr);  // (the compiler has a read of LDS wait for copies into it)
            } else if constexpr (kQAgain) {
                static_assert(RT == 1 && KM == 1, "one tile's rows, 16 keys");
                st[0][0] = pk::f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                uint32_t d0 = g * E;
                asm volatile("" : "+v"(d0));  // (no load of this is the loop's)
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    const uint32_t d = s * 4 * E + d0;
                    u32x4 q = *reinterpret_cast<const u32x4 *>(qAgain + min(d, D - E));
                    if (d >= D) q = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        st[0][0] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kf[0][s][e]), __uint_as_float(q[e]), st[0][0], 0, 0, 0);
                }
            } else {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int mt = 0; mt < KM; ++mt) {
                    st[rt][mt] = pk::f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int s = 0; s < KS; ++s) {
                        if constexpr (kWide) {
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                st[rt][mt] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kf[mt][s][e]), __uint_as_float(qf[rt][s][e]),
                                                                                  st[rt][mt], 0, 0, 0);
                        } else {
                            st[rt][mt] = pk::Mma16<T>::run(kf[mt][s], qf[rt][s], st[rt][mt]);
                        }
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            if (i + 1 - page0 == kHeld) hold(i + 1);
            loadK(i + 1, step + kWaves);
            __builtin_amdgcn_sched_barrier(0);
            float pw[RT][4 * KM];
            u32x4 pf[RT][kParts];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                float mx = -INFINITY, ps = 0.0f, alpha = 1.0f;
#pragma unroll
                for (int j = 0; j < 4 * KM; ++j) {
                    const int key = (int)k0 + (j / 4) * 16 + (int)g * 4 + j % 4;
                    const bool seen = ok[j / 4] & (key < (int)keys) & pk::paged_sees(posQ[rt], key, p);
                    pw[rt][j] = seen ? st[rt][j / 4][j % 4] * c2 : -INFINITY;
                    mx = fmaxf(mx, pw[rt][j]);
                }
                mx = quad16_max(mx);
                const bool move = mx > m[rt] + (kRescaleGap + kLead);
                if (move) {
                    alpha = __builtin_amdgcn_exp2f(m[rt] - (mx - kLead));
                    m[rt] = mx - kLead;
                }
                if (__ballot(move)) {
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) acc[rt][dt] *= alpha;
                }
                // a row that has seen no key yet: every weight 0
                const float mref = m[rt] == -INFINITY ? 0.0f : m[rt];
#pragma unroll
                for (int j = 0; j < 4 * KM; ++j) {
                    pw[rt][j] = __builtin_amdgcn_exp2f(pw[rt][j] - mref);
                    ps += pw[rt][j];
                }
                if constexpr (!kWide) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int e = 0; e < kParts; ++e) {
                            const uint32_t v = pk::pack2<T>(pw[rt][2 * j], pw[rt][2 * j + 1]);
                            pf[rt][e][j] = v;
                            pw[rt][2 * j] -= pk::from_bits16<T>(v & 0xffffu);  // exact
                            pw[rt][2 * j + 1] -= pk::from_bits16<T>(v >> 16);
                        }
                }
                l[rt] = l[rt] * alpha + quad16_sum(ps);
            }
            wait_vmcnt<(KM * KS < 63 ? KM * KS : 63)>();  // the V copies; the next step's K loads stay in flight
            asm volatile("" ::: "memory");
            // V's fragments, kAhead of them before their products
            constexpr int kAhead = HD <= 64 ? 3 : HD <= 128 ? 4 : 0;  // (0: the registers are taken)
            u32x4 va[kAhead + 1];
            auto readV = [&](int dt) {
                auto four = [&](uint32_t key) {
                    const uint32_t chunk = (2 * dt + (c16 & 3) / 2) ^ swz(key);
                    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(sV + (key * CH + chunk) * 16 + (c16 & 1) * 8)));
                };
                const u32x2 a = four(4 * g + c16 / 4), b = four(16 + 4 * g + c16 / 4);
                return u32x4{a.x, a.y, b.x, b.y};
            };
            if constexpr (!kWide && kAhead > 0) {
#pragma unroll
                for (int dt = 0; dt < kAhead; ++dt) va[dt] = readV(dt);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                if constexpr (kWide) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t key = 4 * g + e, chunk = (dt * 4 + c16 / 4) ^ swz(key);
                        const float va = *reinterpret_cast<const float *>(sV + (key * CH + chunk) * 16 + c16 % 4 * 4);
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt) acc[rt][dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(va, pw[rt][e], acc[rt][dt], 0, 0, 0);
                    }
                } else {
                    if (dt + kAhead < DT) va[(dt + kAhead) % (kAhead + 1)] = readV(dt + kAhead);
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                        for (int e = 0; e < kParts; ++e) acc[rt][dt] = pk::Mma16<T>::run(va[dt % (kAhead + 1)], pf[rt][e], acc[rt][dt]);
                    if constexpr (kAhead > 0) __builtin_amdgcn_sched_barrier(0);
                }
            }
            __builtin_amdgcn_s_waitcnt(0xC07F);  // this wave's reads of its V tile are done before it is overwritten
            asm volatile("" ::: "memory");
        }
        wait_vmcnt<0>();  // the last K loads (zeros), before their registers go

        // merge the waves' states, one tile of 16 rows at a time: O through LDS,
        // thread t takes row t / 16, dims 4 (t % 16) + 64 j
        if (g == 0) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                sm_m[wave][rt * 16 + c16] = m[rt];
                sm_l[wave][rt * 16 + c16] = l[rt];
            }
        }
        if (threadIdx.x == 0) sm_bad = 0;
        float *sO = reinterpret_cast<float *>(smem);
        const uint32_t tr = threadIdx.x / 16, td = threadIdx.x % 16 * 4;
        const bool whole = c.lo == 0 && c.hi == c.steps.n;
        const uint64_t slot = w.stateBase + (2 * (uint64_t)blockIdx.x + (c.lo == 0)) * (RT * 16);
        auto store = [&](uint32_t r, uint32_t d, const pk::f32x4 &o, float L) {
            if (whole) store4<T>(out + q_row(r) * D + d, o, L);
            else *reinterpret_cast<pk::f32x4 *>(pO + (slot + r - c.steps.r0) * HD + d) = o;
        };
        auto storeML = [&](uint32_t r, float M, float L) {
            if (!whole && td == 0) *reinterpret_cast<float2 *>(pML + 2 * (slot + r - c.steps.r0)) = float2{M, L};
        };
        bool bad = false;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            __syncthreads();  // V tiles and the previous tile's state are read
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
                *reinterpret_cast<pk::f32x4 *>(&sO[(wave * 16 + c16) * LDO + dt * 16 + g * 4]) = acc[rt][dt];
            __syncthreads();
            const uint32_t r = c.steps.r0 + rt * 16 + tr;
            if (r >= c.steps.r1) continue;
            float M = -INFINITY, wt[kWaves], L = 0.0f;
#pragma unroll
            for (int v = 0; v < kWaves; ++v) M = fmaxf(M, sm_m[v][rt * 16 + tr]);
#pragma unroll
            for (int v = 0; v < kWaves; ++v) {
                const float mv = sm_m[v][rt * 16 + tr];
                wt[v] = mv == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mv - M);
                L += wt[v] * sm_l[v][rt * 16 + tr];
            }
            bad |= !(fabsf(L) < INFINITY);
            for (uint32_t d = td; d < D; d += 64) {
                pk::f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int v = 0; v < kWaves; ++v) o += *reinterpret_cast<const pk::f32x4 *>(&sO[(v * 16 + tr) * LDO + d]) * wt[v];
#pragma unroll
                for (int e = 0; e < 4; ++e) bad |= !(fabsf(o[e]) < INFINITY);
                store(r, d, o, L);
            }
            storeML(r, M, L);
        }
        if (bad) sm_bad = 1;
        __syncthreads();
        if (sm_bad) {
            // A matrix product adds 0 x V for a key that a row does not see, which an infinity or
            // NaN in V turns into NaN: the rows again, over the keys that each sees.
            const uint32_t s0 = min(c.lo, c.steps.sinks), s1 = min(c.hi, c.steps.sinks);
            const uint32_t t0 = max(c.lo, c.steps.sinks), t1 = max(c.hi, c.steps.sinks);
            auto key_at = [&](uint32_t k) { return (int)min(k * w.stepKeys, keys); };
            for (uint32_t r = c.steps.r0 + tr; r < c.steps.r1; r += 16) {
                constexpr int NJ = HD / 64;
                pk::f32x4 qv[NJ], o[NJ];
                float M = -INFINITY, L = 0.0f;
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    o[j] = qv[j] = pk::f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                    if (td + 64 * j < D)
#pragma unroll
                        for (int e = 0; e < 4; ++e) qv[j][e] = T::load(Q[q_row(r) * D + td + 64 * j + e]);
                }
                const int pos = c.req.pos0 + (int)(r / G);
                paged_row<T, NJ, true, 1>(qv, K, V, table, c.hkv, pos, key_at(s0), key_at(s1), p, o, M, L);
                paged_row<T, NJ, true, 1>(qv, K, V, table, c.hkv, pos, key_at(t0 - c.steps.sinks + c.steps.first),
                                       key_at(t1 - c.steps.sinks + c.steps.first), p, o, M, L);
#pragma unroll
                for (int j = 0; j < NJ; ++j)
                    if (td + 64 * j < D) store(r, td + 64 * j, o[j], L);
                storeML(r, M, L);
            }
        }
        __syncthreads();  // the state is read before the next piece's V tiles
    }
}

// ---- many rows: chunks of prompts --------------------------------------------------------
// Tiles of 128 rows, 32 to a wave, on v_mfma_f32_32x32x16: S^T = K . Q^T has a
// row's scores in two lanes (mfma.hpp), so maxima and sums take one lane swap,
// and a lane's weights are its P^T operand of O^T += V^T . P^T as they are.
// Steps are 64 keys; wave w copies group w's 16 keys (of one page) of K and V
// from the page straight into LDS, K two steps ahead and V one. K is read by
// rows, V by ds_read_b64_tr_b16 (four keys of a dim to a lane); 16-byte chunks
// are swizzled so that the rows of one read fall in different banks.
// What bounds it: products and softmax take about as long (HD 128: 1024 cycles
// of MFMA and 960 of VALU for a step), so step i + 1's scores are computed
// beside step i's exponentials, and step i's product with V beside the
// maximum of step i + 1. 2048 tokens behind 8192 keys, 8 heads of 256 in f16:
// 186 to 199 us with the merge, 780 to 830 TFLOP/s, where a large product reaches
// 1250 to 1414. A pass is 3500 cycles, 1500 of them with scores, 1350 with V (1024
// of MFMA in each), 300 at the barrier. Counted at 2.04 GHz: a wave lives 321000
// cycles, 72 passes and 69000 for its starts, states and stores; 148000 (46%) are MFMA.
constexpr int kTileRows = 128;

template <typename T, int HD>
__device__ void paged_tile(const typename T::storage *__restrict__ Q, const typename T::storage *__restrict__ K,
                           const typename T::storage *__restrict__ V,
                           const int32_t *__restrict__ tables, const int32_t *__restrict__ starts, const int32_t *__restrict__ keyLens,
                           const pk::PagedTile *__restrict__ plan, float *__restrict__ pO, float *__restrict__ pML,
                           Shared *__restrict__ shared, typename T::storage *__restrict__ out, const PagedAttentionConstants &p,
                           const PagedWorkConstants &w) {
    using S = typename T::storage;
    constexpr int BKV = 64, KS = HD / 16, DT = HD / 32, CH = HD / 8;
    constexpr int kRowsPer = 64 / CH;       // rows per copy instruction
    constexpr int kCopies = 16 / kRowsPer;  // instructions for a wave's 16 rows of K (or V) of a step
    // The words of a weight in the product with V. One bf16 has 8 bits, so there are two, 2^-16 off. One f16 has 11, as many as
    // the result: 2048 tokens behind 8192 keys, 8 heads of 256 on 4, are 2.9e-4 off (2-norm, against 64 bits) in 193 us; with two
    // words 2.1e-4, which the rounding of the result alone makes, in 250 (1000 tokens of 128 dims 70 and 88). As FlashAttention.
    constexpr bool kTwo = std::is_same<T, pk::BF16>::value;
    constexpr float kLead = kTwo ? 0.0f : 4.0f;
    constexpr uint32_t kTileBytes = BKV * HD * 2;
    // K's two places, V's two, the plan (one array: with two, the compiler has every read of LDS wait for the latest copy)
    __shared__ __attribute__((aligned(256))) uint8_t smem[4 * kTileBytes + kOwnTiles * sizeof(OwnTile)];
    static_assert(sizeof(PlanSpace<256, uint32_t>) <= 4 * kTileBytes, "the plan is laid out where K and V go");
    OwnTile *sm_plan = reinterpret_cast<OwnTile *>(smem + 4 * kTileBytes);

    const uint32_t lane = threadIdx.x & 63, h = lane >> 5, c32 = lane & 31;
    const uint32_t wave = first_lane(threadIdx.x >> 6);
    const uint32_t D = p.Hd, G = p.Nq / p.Nkv;
    const float c2 = fabsf(p.scale) * kLog2e;
    const uint32_t flip = p.scale < 0.0f ? 0x80008000u : 0u;  // -scale K . Q = scale K . -Q
    auto swzK = [](uint32_t row) { return CH >= 16 ? row % 16u : row / 2u % 8u; };
    auto swzV = [](uint32_t row) { return CH >= 16 ? row % 4u * 4u : row / 2u % 2u * 4u; };

    Dealer<256> dealer(starts, keyLens, plan, sm_plan, *reinterpret_cast<PlanSpace<256, uint32_t> *>(smem), shared, p, w);
    Piece c;
    while (dealer.next(c, p, w)) {
        const int32_t *table = tables + (uint64_t)c.request * p.columns;
        const uint32_t keys = (uint32_t)c.req.keys;
        auto q_row = [&](uint32_t r) { return ((uint64_t)(uint32_t)c.req.start + r / G) * p.Nq + c.hkv * G + r % G; };
        // the wave's rows; those past the tile's last repeat it and are not stored
        const uint32_t w0 = c.steps.r0 + wave * 32, myRow = w0 + c32, rowAt = min(myRow, c.steps.r1 - 1);
        const int pos = c.req.pos0 + (int)(rowAt / G);
        const int posLo = c.req.pos0 + (int)(min(w0, c.steps.r1 - 1) / G), posHi = c.req.pos0 + (int)(min(w0 + 31, c.steps.r1 - 1) / G);
        // Lane l holds, of group l % 4 of the piece's step held0 + l / 4, the bytes from K's (V's) start and the rows that
        // a page holds (0: none); of the step, all four groups' rows (a byte each) and whether all rows of the wave see all keys.
        const uint32_t n = c.hi - c.lo;
        uint32_t held0 = 0, heldLo = 0, heldHi = 0, heldRows = 0, heldAll = 0;
        uint64_t heldSee = 0;
        auto hold = [&](uint32_t i) {
            const uint32_t at = i + lane / 4;
            held0 = i;
            uint64_t off = 0;
            heldRows = 0;
            const uint32_t key0 = pk::paged_step_key(c.steps, c.lo + at, w), key = key0 + lane % 4 * 16;
            if (at < n && key < keys) {
                const uint32_t column = key / p.pageSize, page = (uint32_t)table[column];
                if (page < p.pages) {
                    off = (((uint64_t)page * p.Nkv + c.hkv) * p.pageSize + (key - column * p.pageSize)) * (D * 2);
                    heldRows = min(16u, keys - key);
                }
            }
            heldLo = (uint32_t)off;
            heldHi = (uint32_t)(off >> 32);
            auto of_quad = [&](auto ctrl) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)heldRows, decltype(ctrl)::value, 0xf, 0xf, false); };
            heldAll = of_quad(std::integral_constant<int, 0x00>{}) | of_quad(std::integral_constant<int, 0x55>{}) << 8 |
                      of_quad(std::integral_constant<int, 0xaa>{}) << 16 | of_quad(std::integral_constant<int, 0xff>{}) << 24;
            const bool see = heldAll == 0x10101010u &&
                             (p.maskKind == 2u || ((int)key0 + BKV - 1 <= posLo && (p.maskKind == 0u || (int64_t)posHi - key0 < p.slidingWindow ||
                                                                                    key0 + BKV - 1 < p.sinks)));
            heldSee = __ballot(see);
        };
        // The wave's group of step i of K (V); of a step behind the last, nothing. Rows that no page holds are read as zeros.
        auto group = [&](const S *from, uint32_t i) {
            const int at = (int)(((i < n ? i : held0) - held0) * 4 + wave);
            const uint64_t off = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)heldHi, at) << 32 |
                                 (uint32_t)__builtin_amdgcn_readlane((int)heldLo, at);
            const int bytes = i < n ? __builtin_amdgcn_readlane((int)heldRows, at) * (int)(D * 2) : 0;
            return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<uint8_t *>(const_cast<S *>(from)) + off, 0, bytes, 0x00020000);
        };
        // Instruction j of kCopies of a group's copy into the place at `to`.
        auto copy = [&](__amdgpu_buffer_rsrc_t rs, uint32_t to, int j, auto &&swz) {
            const uint32_t row = j * kRowsPer + lane / CH, chunk = lane % CH ^ swz(row);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void *)(smem + to + (wave * 16 + j * kRowsPer) * HD * 2), 16,
                                                     chunk * 8 < D ? (int)((row * D + chunk * 8) * 2) : kOutOfRange, 0, 0, 0);
        };
        auto copyK = [&](__amdgpu_buffer_rsrc_t rs, uint32_t i, int j) { copy(rs, i % 2 * kTileBytes, j, swzK); };
        auto copyV = [&](__amdgpu_buffer_rsrc_t rs, uint32_t i, int j) { copy(rs, (2 + i % 2) * kTileBytes, j, swzV); };
        struct Ahead {
            uint32_t rows;  // a byte per group
            bool see;
        };
        auto ahead_of = [&](uint32_t i) {
            return Ahead{(uint32_t)__builtin_amdgcn_readlane((int)heldAll, (int)((i - held0) * 4)), (heldSee >> ((i - held0) * 4) & 1) != 0};
        };

        u32x4 qf[KS];
        f32x16 acc[DT];
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[dt][i] = 0.0f;
        float m = -INFINITY, l = 0.0f;

        // LDS offsets of this lane's K and V, in a place: the other fragments' are these with bits 5 to 7 turned over
        // (a row's 16-byte chunks s and s + 8 are 256 bytes apart), and constant distances. Kept from being computed
        // once for all fragments (48 registers).
        const uint32_t kAt = c32 * (HD * 2) + (h ^ swzK(c32)) * 16;
        const uint32_t s16 = lane & 15, swz4 = CH >= 16 ? s16 / 4 : s16 / 8;
        const uint32_t vAt = 2 * kTileBytes + (h * 4 + s16 / 4) * (HD * 2) + swz4 * 64 + (lane >> 4 & 1) * 32 + (s16 & 3) * 8;
        auto in_place = [](uint32_t lane0, uint32_t i) {
            uint32_t x = lane0 + i % 2 * kTileBytes;
            asm volatile("" : "+v"(x));
            return x;
        };
        // fragment f: dims 16 (f % KS) .. + 15 of keys 32 (f / KS) + c32
        auto readK = [&](uint32_t x, int f) {
            const int s = f % KS;
            return *reinterpret_cast<const u32x4 *>(smem + ((x ^ (s & 7) * 32u) + (s >> 3) * 256u + f / KS * (32 * HD * 2)));
        };
        // fragment f: this lane's 4 + 4 keys of the 16 from 16 (f % 4) on, one dim of 32 (f / 4) .. + 31
        auto readV = [&](uint32_t x, int f) {
            const int dt = f / 4;
            const uint32_t y = (x ^ (dt & 3) * 64u) + (dt >> 2) * 256u + f % 4 * (16 * HD * 2);
            const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(smem + y)));
            const u32x2 b = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(smem + y + 8 * HD * 2)));
            return u32x4{a.x, a.y, b.x, b.y};
        };
        struct Scores {
            f32x16 half[2];  // of 32 keys each
        };
        // Hides what the rows do not see of step i.
        auto mask = [&](Scores &s, uint32_t i, uint32_t rows) {
            const uint32_t key0 = pk::paged_step_key(c.steps, c.lo + i, w);
#pragma unroll
            for (int j = 0; j < 32; ++j) {
                const uint32_t in = (j >> 2) * 8 + h * 4 + (j & 3);  // groups of 16: j / 8
                const bool seen = (in % 16 < (rows >> j / 8 * 8 & 0xffu)) & pk::paged_sees(pos, (int)(key0 + in), p);
                s.half[j / 16][j % 16] = seen ? s.half[j / 16][j % 16] : -INFINITY;
            }
        };
        // Moves the rows' reference to a maximum that passes it by more than the gap.
        auto follow = [&](float highest) {
            const float mx = pk::pair32_max(highest) * c2;
            const bool move = mx > m + (kRescaleGap + kLead);
            if (!__ballot(move)) return;
            float alpha = 1.0f;
            if (move) {
                alpha = __builtin_amdgcn_exp2f(m - (mx - kLead));
                m = mx - kLead;
            }
            l *= alpha;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) acc[dt] *= alpha;
        };
        Scores st;
        u32x4 pf[4], pr[4];
        float mref = 0.0f, ps = 0.0f;
        // The weights of two of st's scores, as a word of the P^T operands.
        auto weigh = [&](int pair) {
            const int e = pair % 8 * 2;
            const f32x16 &x = st.half[pair / 8];
            const float p0 = __builtin_amdgcn_exp2f(fmaf(x[e], c2, -mref)), p1 = __builtin_amdgcn_exp2f(fmaf(x[e + 1], c2, -mref));
            ps += p0 + p1;
            uint32_t v = pk::pack2<T>(p0, p1);
            if constexpr (kTwo) {
                uint32_t r = pk::pack2<T>(p0 - __uint_as_float(v << 16), p1 - __uint_as_float(v & 0xffff0000u));
                asm volatile("" : "+v"(r));
                pr[pair / 4][pair % 4] = r;
            }
            asm volatile("" : "+v"(v));  // here, and not where it is used
            pf[pair / 4][pair % 4] = v;
        };
        auto start_weights = [&] {
            mref = m == -INFINITY ? 0.0f : m;
            ps = 0.0f;
        };
        // acc += V^T . P^T of step i, with `beside(f)` next to the product of fragment f. V is read kAheadV
        // fragments before its product.
        constexpr int kFragV = DT * 4, kAheadV = 4, kFragK = KS * 2, kAheadK = 4;
        auto multiply = [&](uint32_t i, auto &&beside) {
            const uint32_t x = in_place(vAt, i);
            u32x4 va[kAheadV];
#pragma unroll
            for (int f = 0; f < kAheadV; ++f) va[f] = readV(x, f);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int f = 0; f < kFragV; ++f) {
                acc[f / 4] = pk::Mma<T>::run(va[f % kAheadV], pf[f % 4], acc[f / 4]);
                if constexpr (kTwo) acc[f / 4] = pk::Mma<T>::run(va[f % kAheadV], pr[f % 4], acc[f / 4]);
                if (f + kAheadV < kFragV) va[f % kAheadV] = readV(x, f + kAheadV);
                beside(f);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        // The scores of step i, with `beside(f)` next to the product of fragment f.
        auto score = [&](uint32_t i, auto &&beside) {
            Scores s;
            const uint32_t x = in_place(kAt, i);
            u32x4 kf[kAheadK];
#pragma unroll
            for (int f = 0; f < kAheadK; ++f) kf[f] = readK(x, f);
#pragma unroll
            for (int j = 0; j < 32; ++j) s.half[j / 16][j % 16] = 0.0f;
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int f = 0; f < kFragK; ++f) {
                s.half[f / KS] = pk::Mma<T>::run(kf[f % kAheadK], qf[f % KS], s.half[f / KS]);
                if (f + kAheadK < kFragK) kf[f % kAheadK] = readK(x, f + kAheadK);
                beside(f);
                __builtin_amdgcn_sched_barrier(0);
            }
            return s;
        };

        hold(0);
        {
            const S *row = Q + q_row(rowAt) * D + h * 8;
#pragma unroll
            for (int s = 0; s < KS; ++s) qf[s] = s * 16 + h * 8 < D ? *reinterpret_cast<const u32x4 *>(row + s * 16) : u32x4{0u, 0u, 0u, 0u};
        }
        {
            const __amdgpu_buffer_rsrc_t k0 = group(K, 0), v0 = group(V, 0), k1 = group(K, 1);
#pragma unroll
            for (int j = 0; j < kCopies; ++j) {
                copyK(k0, 0, j);
                copyV(v0, 0, j);
                copyK(k1, 1, j);
            }
        }
        if (w0 >= c.steps.r1) {  // a wave without rows copies its part of K and V, and leaves LDS and the matrix cores to the others
            wait_vmcnt<0>();
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
#pragma unroll 1
            for (uint32_t i = 0; i + 1 < n; ++i) {
                wait_vmcnt<0>();
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                const __amdgpu_buffer_rsrc_t rv = group(V, i + 1);
                if (i + 2 < n && i + 2 - held0 == 16) hold(i + 2);
                const __amdgpu_buffer_rsrc_t rk = group(K, i + 2);
#pragma unroll
                for (int j = 0; j < kCopies; ++j) {
                    copyK(rk, i + 2, j);
                    copyV(rv, i + 1, j);
                }
            }
            wait_vmcnt<0>();
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            continue;
        }
        Ahead next = ahead_of(0), next2 = n > 1 ? ahead_of(1) : next;
#pragma unroll
        for (int s = 0; s < KS; ++s) qf[s] ^= flip;
        wait_vmcnt<0>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        st = score(0, [](int) {});
        if (!next.see) mask(st, 0, next.rows);
        {
            float mx = st.half[0][0];
#pragma unroll
            for (int j = 1; j < 32; ++j) mx = fmaxf(mx, st.half[j / 16][j % 16]);
            follow(mx);
        }
        // Pass i: step i + 1's scores beside step i's weights, then step i's product with V beside the maximum of step
        // i + 1, in chunks that keep their order: products run while the vector instructions behind them issue.
        for (uint32_t i = 0; i + 1 < n; ++i) {
            // K of step i + 1 and V of step i are in LDS (copied in pass i - 1), and every wave has read what is copied over
            wait_vmcnt<0>();
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            next = next2;
            const __amdgpu_buffer_rsrc_t rv = group(V, i + 1);
            if (i + 2 < n) {
                if (i + 2 - held0 == 16) hold(i + 2);
                next2 = ahead_of(i + 2);
            }
            const __amdgpu_buffer_rsrc_t rk = group(K, i + 2);
            start_weights();
            Scores sn = score(i + 1, [&](int f) {
                // the copies, spread over the products: a CU takes 16 cycles for each, so the four waves' would wait in a row
                constexpr int kEvery = kFragK / (2 * kCopies);
                if (f % kEvery == 0) {
                    const int j = f / kEvery;
                    if (j < kCopies) copyK(rk, i + 2, j);
                    else copyV(rv, i + 1, j - kCopies);
                }
                // the 16 pairs over the kFragK products
                if constexpr (kFragK >= 16) {
                    if (f % (kFragK / 16) == 0) weigh(f / (kFragK / 16));
                } else {
#pragma unroll
                    for (int j = 0; j < 16 / kFragK; ++j) weigh(f * (16 / kFragK) + j);
                }
            });
            if (!next.see) mask(sn, i + 1, next.rows);
            float mx = sn.half[0][0];
            multiply(i, [&](int f) {
                constexpr int kEach = 32 / kFragV;
#pragma unroll
                for (int j = f * kEach; j < (f + 1) * kEach; ++j) mx = fmaxf(mx, sn.half[j / 16][j % 16]);
            });
            l += pk::pair32_sum(ps);
            follow(mx);
            st = sn;
        }
        wait_vmcnt<0>();  // V of the last step
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        start_weights();
#pragma unroll
        for (int j = 0; j < 16; ++j) weigh(j);
        l += pk::pair32_sum(ps);
        multiply(n - 1, [](int) {});
        // every wave has read its last tiles before the next piece's copies
        __builtin_amdgcn_s_waitcnt(0xC07F);
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");

        const bool whole = c.lo == 0 && c.hi == c.steps.n;
        const uint64_t slot = w.stateBase + (2 * (uint64_t)blockIdx.x + (c.lo == 0)) * kTileRows;
        auto store = [&](uint32_t r, uint32_t d, const pk::f32x4 &o, float L) {
            if (whole) store4<T>(out + q_row(r) * D + d, o, L);
            else *reinterpret_cast<pk::f32x4 *>(pO + (slot + r - c.steps.r0) * HD + d) = o;
        };
        bool bad = !(fabsf(l) < INFINITY);
        uint32_t d0 = h * 4;
        asm volatile("" : "+v"(d0));  // (computed here)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int i4 = 0; i4 < 4; ++i4) {
                const uint32_t d = dt * 32 + i4 * 8 + d0;
                const pk::f32x4 o = {acc[dt][4 * i4], acc[dt][4 * i4 + 1], acc[dt][4 * i4 + 2], acc[dt][4 * i4 + 3]};
#pragma unroll
                for (int e = 0; e < 4; ++e) bad |= !(fabsf(o[e]) < INFINITY) & (d < D);
                if (myRow < c.steps.r1 && d < D) store(myRow, d, o, l);
            }
        if (!whole && myRow < c.steps.r1 && h == 0) *reinterpret_cast<float2 *>(pML + 2 * (slot + myRow - c.steps.r0)) = float2{m, l};
        if (!__ballot(bad)) continue;
        wait_vmcnt<0>();  // the rows' stores, before other lanes store them again
        // as in paged_few: an infinity or NaN in V that a row does not see
        const uint32_t s0 = min(c.lo, c.steps.sinks), s1 = min(c.hi, c.steps.sinks);
        const uint32_t t0 = max(c.lo, c.steps.sinks), t1 = max(c.hi, c.steps.sinks);
        auto key_at = [&](uint32_t k) { return (int)min(k * w.stepKeys, keys); };
        uint32_t row16 = lane;
        asm volatile("" : "+v"(row16));  // (computed here)
        const uint32_t td = row16 % 16 * 4;
        for (uint32_t r = w0 + row16 / 16; r < min(w0 + 32, c.steps.r1); r += 4) {
            constexpr int NJ = HD / 64;
            pk::f32x4 qv[NJ], o[NJ];
            float M = -INFINITY, L = 0.0f;
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                o[j] = qv[j] = pk::f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                if (td + 64 * j < D)
#pragma unroll
                    for (int e = 0; e < 4; ++e) qv[j][e] = T::load(Q[q_row(r) * D + td + 64 * j + e]);
            }
            const int rp = c.req.pos0 + (int)(r / G);
            paged_row<T, NJ, true, 1>(qv, K, V, table, c.hkv, rp, key_at(s0), key_at(s1), p, o, M, L);
            paged_row<T, NJ, true, 1>(qv, K, V, table, c.hkv, rp, key_at(t0 - c.steps.sinks + c.steps.first),
                                   key_at(t1 - c.steps.sinks + c.steps.first), p, o, M, L);
#pragma unroll
            for (int j = 0; j < NJ; ++j)
                if (td + 64 * j < D) store(r, td + 64 * j, o[j], L);
            if (!whole && td == 0) *reinterpret_cast<float2 *>(pML + 2 * (slot + r - c.steps.r0)) = float2{M, L};
        }
    }
}

// The units that several workers shared: the first one's state is in its slot
// 2 w + 1, the following ones' in theirs 2 w'. 16 lanes take a row's dims; with
// fewer than 16 rows, several groups of lanes share a row's pieces. Bound by its
// launch and two reads that wait for each other (5 us), for tiles by the states
// (8 to 13 us, of up to 67 MB).
template <typename T, int HD>
__device__ void paged_merge(const float *__restrict__ pO, const float *__restrict__ pML, const Shared *__restrict__ shared,
                            typename T::storage *__restrict__ out, const PagedAttentionConstants &p) {
    constexpr int NJ = HD / 64;
    __shared__ __attribute__((aligned(16))) float sO[16][HD];
    __shared__ float sM[16], sL[16];
    const uint32_t D = p.Hd, G = p.Nq / p.Nkv;
    const Shared c = shared[blockIdx.x];
    if (c.pieces == 0) return;
    const uint32_t r0 = c.r0 + blockIdx.y * 16;
    if (r0 >= c.r1) return;
    const uint32_t rows = min(c.r1 - r0, 16u), each = rows <= 8 ? 16u >> (32 - __clz(rows - 1)) : 1u;  // groups per row
    const uint32_t td = threadIdx.x % 16 * 4, group = threadIdx.x / 16, in = group / each, sub = group % each;
    const uint32_t r = r0 + in;
    const bool live = in < rows;
    pk::f32x4 o[NJ];
    float m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int j = 0; j < NJ; ++j) o[j] = pk::f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    auto add = [&](float mi, float li, const pk::f32x4 (&v)[NJ]) {
        if (mi == -INFINITY && li == 0.0f) return;  // no key seen
        const float mn = fmaxf(m, mi);
        const float a = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn), b = __builtin_amdgcn_exp2f(mi - mn);
        l = l * a + li * b;
        m = mn;
#pragma unroll
        for (int j = 0; j < NJ; ++j) o[j] = o[j] * a + v[j] * b;
    };
    constexpr uint32_t U = NJ > 4 ? 2 : 4;  // pieces in flight
    if (live)
        for (uint32_t i0 = sub; i0 < c.pieces; i0 += U * each) {
            float2 ml[U];
            pk::f32x4 v[U][NJ];
#pragma unroll
            for (uint32_t u = 0; u < U; ++u) {
                const uint32_t i = min(i0 + u * each, c.pieces - 1);
                const uint64_t row = c.base + (2 * ((uint64_t)c.worker + i) + (i == 0)) * c.rows + (r - c.r0);
                ml[u] = *reinterpret_cast<const float2 *>(pML + 2 * row);
#pragma unroll
                for (int j = 0; j < NJ; ++j) v[u][j] = td + 64 * j < D ? *reinterpret_cast<const pk::f32x4 *>(pO + row * HD + td + 64 * j) : o[j];
            }
#pragma unroll
            for (uint32_t u = 0; u < U; ++u)
                if (i0 + u * each < c.pieces) add(ml[u].x, ml[u].y, v[u]);
        }
    if (each > 1) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) *reinterpret_cast<pk::f32x4 *>(&sO[group][td + 64 * j]) = o[j];
        if (td == 0) {
            sM[group] = m;
            sL[group] = l;
        }
        __syncthreads();
        if (sub != 0) return;
        for (uint32_t e = 1; e < each; ++e) {
            pk::f32x4 v[NJ];
#pragma unroll
            for (int j = 0; j < NJ; ++j) v[j] = *reinterpret_cast<const pk::f32x4 *>(&sO[group + e][td + 64 * j]);
            add(sM[group + e], sL[group + e], v);
        }
    }
    if (!live) return;
    const uint64_t row = ((uint64_t)c.start + r / G) * p.Nq + c.hkv * G + r % G;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
        if (td + 64 * j < D) store4<T>(out + row * D + td + 64 * j, o[j], l);
}

// Any head dim up to 512 and any alignment: a block per row of the T * Nq
// (token, head) pairs, whose 16 groups of 16 lanes take runs of keys in turn
// and are merged. Bound by the loads of one row's keys, which each row reads
// again: 8 heads on 4 over 4096 keys of 100 dims (f16) 186 us, 64 requests of
// 100 to 4000 keys 213 us, 300 tokens behind 2000 keys 545 us. (A row per 16
// lanes took 11.8 ms for 4096 keys of 256, which the kernels below read in 18 us.)
template <typename T, bool VEC>
__device__ void paged_plain(const typename T::storage *__restrict__ Q, const typename T::storage *__restrict__ K,
                            const typename T::storage *__restrict__ V, const int32_t *__restrict__ tables,
                            const int32_t *__restrict__ starts, const int32_t *__restrict__ keyLens,
                            typename T::storage *__restrict__ out, const PagedAttentionConstants &p) {
    constexpr int NJ = 8;
    __shared__ float sO[16][NJ * 64], sM[16], sL[16];
    const uint32_t row = blockIdx.x, part = threadIdx.x / 16, td = threadIdx.x % 16 * 4;
    const int32_t t = (int32_t)(row / p.Nq);
    const uint32_t hkv = row % p.Nq / (p.Nq / p.Nkv);
    // the last request that starts at or before t
    uint32_t a = 0, b = p.R;  // starts[a] <= t < starts[b], if any does
    while (b - a > 1) {
        const uint32_t mid = (a + b) / 2;
        if (starts[mid] <= t) a = mid;
        else b = mid;
    }
    const pk::PagedRequest r = pk::paged_request(starts[a], starts[a + 1], keyLens[a], p);
    if (t < r.start || t >= r.start + r.n) return;
    const int pos = r.pos0 + (t - r.start);
    const pk::PagedSpan s = pk::paged_span(pos, pos, r.keys, p);
    pk::f32x4 q[NJ], o[NJ];
    const typename T::storage *qr = Q + (uint64_t)row * p.Hd;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
        o[j] = q[j] = pk::f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (td + 64 * j + i < p.Hd) q[j][i] = T::load(qr[td + 64 * j + i]);
    }
    float m = -INFINITY, l = 0.0f;
    const int32_t *table = tables + (uint64_t)a * p.columns;
    paged_row<T, NJ, VEC, 2>(q, K, V, table, hkv, pos, 0, s.sinkEnd, p, o, m, l, part, 16);
    paged_row<T, NJ, VEC, 2>(q, K, V, table, hkv, pos, s.lo, s.hi, p, o, m, l, part, 16);
#pragma unroll
    for (int j = 0; j < NJ; ++j) *reinterpret_cast<pk::f32x4 *>(&sO[part][td + 64 * j]) = o[j];
    if (td == 0) {
        sM[part] = m;
        sL[part] = l;
    }
    __syncthreads();
    float M = -INFINITY, L = 0.0f, wt[16];
#pragma unroll
    for (int v = 0; v < 16; ++v) M = fmaxf(M, sM[v]);
#pragma unroll
    for (int v = 0; v < 16; ++v) {
        wt[v] = sM[v] == -INFINITY && sL[v] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(sM[v] - M);
        L += wt[v] * sL[v];
    }
    for (uint32_t d = threadIdx.x; d < p.Hd; d += 256) {
        float x = 0.0f;
#pragma unroll
        for (int v = 0; v < 16; ++v) x = fmaf(sO[v][d], wt[v], x);
        out[(uint64_t)row * p.Hd + d] = T::store(L != 0.0f ? x / L : 0.0f);
    }
}

}  // namespace

#define PAGED_PLAIN(name, T, VEC)                                                                                         \
    POPCORN_KERNEL void __launch_bounds__(256)                                                                            \
        name(const T::storage *q, const T::storage *k, const T::storage *v, const int32_t *tables, const int32_t *starts, \
             const int32_t *keyLens, T::storage *out, PagedAttentionConstants p) {                                        \
        paged_plain<T, VEC>(q, k, v, tables, starts, keyLens, out, p);                                                    \
    }

using pk::BF16;
using pk::F16;
using pk::F32;

PAGED_PLAIN(paged_attention_plain_f32, F32, true)
PAGED_PLAIN(paged_attention_plain_f16, F16, true)
PAGED_PLAIN(paged_attention_plain_bf16, BF16, true)
PAGED_PLAIN(paged_attention_plain_f32_any, F32, false)
PAGED_PLAIN(paged_attention_plain_f16_any, F16, false)
PAGED_PLAIN(paged_attention_plain_bf16_any, BF16, false)

#define PAGED_FEW(name, T, HD, RT, PER_CU)                                                                                \
    POPCORN_KERNEL void __launch_bounds__(256, PER_CU)                                                                    \
        name(const T::storage *q, const T::storage *k, const T::storage *v, const int32_t *tables, const int32_t *starts, \
             const int32_t *keyLens, const pk::PagedTile *plan, float *pO, float *pML, Shared *shared, T::storage *out,   \
             PagedAttentionConstants p, PagedWorkConstants w) {                                                           \
        paged_few<T, HD, RT>(q, k, v, tables, starts, keyLens, plan, pO, pML, shared, out, p, w);                         \
    }
#define PAGED_TILE(name, T, HD, PER_CU)                                                                                   \
    POPCORN_KERNEL void __launch_bounds__(256, PER_CU)                                                                    \
        name(const T::storage *q, const T::storage *k, const T::storage *v, const int32_t *tables, const int32_t *starts,       \
             const int32_t *keyLens, const pk::PagedTile *plan, float *pO, float *pML, Shared *shared, T::storage *out,     \
             PagedAttentionConstants p, PagedWorkConstants w) {                                                           \
        paged_tile<T, HD>(q, k, v, tables, starts, keyLens, plan, pO, pML, shared, out, p, w);                            \
    }
#define PAGED_MERGE(name, T, HD)                                                                                          \
    POPCORN_KERNEL void __launch_bounds__(256) name(const float *pO, const float *pML, const Shared *shared, T::storage *out, \
                                                    PagedAttentionConstants p) {                                          \
        paged_merge<T, HD>(pO, pML, shared, out, p);                                                                      \
    }
// The blocks per CU limit the registers. Most kernels hold everything in them; of a lane's VGPRs these spill to scratch memory:
// 11 in tile_bf16_d128 (and 48 bytes of it per lane in all), 2 in tile_f16_d128, 4 in few_f32_d128_r1, 4 in the 16-bit
// few_d512_r1, 19 in few_f32_d512_r1.
#define PAGED_FEW_D(t, T, PER256)                                   \
    PAGED_FEW(paged_attention_few_##t##_d64_r1, T, 64, 1, 4)   \
    PAGED_FEW(paged_attention_few_##t##_d64_r2, T, 64, 2, 3)   \
    PAGED_FEW(paged_attention_few_##t##_d128_r1, T, 128, 1, 3) \
    PAGED_FEW(paged_attention_few_##t##_d128_r2, T, 128, 2, 2) \
    PAGED_FEW(paged_attention_few_##t##_d256_r1, T, 256, 1, PER256) \
    PAGED_FEW(paged_attention_few_##t##_d512_r1, T, 512, 1, 1) \
    PAGED_MERGE(paged_attention_merge_##t##_d64, T, 64)        \
    PAGED_MERGE(paged_attention_merge_##t##_d128, T, 128)      \
    PAGED_MERGE(paged_attention_merge_##t##_d256, T, 256)      \
    PAGED_MERGE(paged_attention_merge_##t##_d512, T, 512)

PAGED_FEW_D(f32, F32, 1)
PAGED_FEW_D(f16, F16, 2)
PAGED_FEW_D(bf16, BF16, 2)
PAGED_FEW(paged_attention_few_f16_d256_r2, F16, 256, 2, 1)
PAGED_FEW(paged_attention_few_bf16_d256_r2, BF16, 256, 2, 1)

PAGED_TILE(paged_attention_tile_f16_d64, F16, 64, 2)
PAGED_TILE(paged_attention_tile_f16_d128, F16, 128, 2)
PAGED_TILE(paged_attention_tile_f16_d256, F16, 256, 1)
PAGED_TILE(paged_attention_tile_bf16_d64, BF16, 64, 2)
PAGED_TILE(paged_attention_tile_bf16_d128, BF16, 128, 2)
PAGED_TILE(paged_attention_tile_bf16_d256, BF16, 256, 1)
