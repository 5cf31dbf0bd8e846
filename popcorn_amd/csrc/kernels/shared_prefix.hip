// Attention of a batch whose requests share prefixes. A group is a stretch of
// requests with a prefix in pages of its own; a row's keys are its group's
// prefix and, behind it, its request's own pages:
//   out = softmax(scale q (Kp, Ko)^T) (Vp, Vo), lse = log of the row's sum of exponentials.
// The rows of all the group's requests stand in a row in q, so to the prefix they are
// one request of many rows: a call's units (paged_attention.hpp) are first
// the groups' rows against the prefixes, then each request's rows against its
// pages, so the prefix's keys are read once for 128 rows and not once for each request.
// A row has two units, each in one piece or several; a row's record of a unit (u32x4) says
// where the states of its pieces lie, and the merge adds them all:
//   O = sum O_i 2^(m_i - M) / L, L = sum l_i 2^(m_i - M), lse = (M + log2 L) ln 2.
// What bounds it: small calls their chain of dependent reads (lengths 3 us, the piece 2, table and q 1, two steps 6, the store 2) and
// the merge's launch (4): 2 requests behind up to 1024 keys 20 us in all, where their bytes take 1; large batches the cold reads of
// many short stretches of pages (64 requests of 50 to 1500 own keys behind 8192, 142 MB: 47 us, 3.0 TB/s, beside 14 for the plan and
// the merge; torch.sum reads 111 MB at 3.0), and the products with weights of two words (256 behind 16384, bf16, 35 GFLOP: 80 to 90 us).
#include "paged_attention.hpp"

namespace {

constexpr float kLn2 = 0.6931471805599453f;
constexpr uint32_t kBehindPrefix = 1u << 31;  // in the last word of a row's record of its own keys: it has one of its prefix too

// The groups of a call, a lane of every wave for each where there are up to 64 (else read where they are asked for): a unit's
// group would take loads that wait for each other. Not in LDS: beside another array there the compiler has every read of LDS wait
// for the latest copy into it (256 requests behind 16384 keys, the prefix alone: 95 us, and 65).
struct HeldGroups {
    int32_t end, len, first;  // of the lane's group; first: where group 0 begins, in every lane
    uint32_t n;

    __device__ inline HeldGroups(const int32_t *groupStarts, const int32_t *prefixLens, const SharedPrefixConstants &s) {
        const uint32_t lane = threadIdx.x & 63;
        n = s.groups <= 64 ? s.groups : 0u;
        end = lane < n ? groupStarts[lane + 1] : 0;
        len = lane < n ? prefixLens[lane] : 0;
        first = n ? groupStarts[0] : 0;
    }
    // Group g's requests and its prefix's keys. (Lanes that ask for a group are among those that hold one, or all ask for the same.)
    __device__ inline void group(uint32_t g, int32_t &a, int32_t &b, int32_t &keys) const {
        const int32_t before = __shfl(end, (int)(g ? g - 1 : 0u));
        a = g ? before : first;
        b = __shfl(end, (int)g);
        keys = __shfl(len, (int)g);
    }
    // Keys of the prefix of request r's group.
    __device__ inline int32_t before(int32_t r) const {
        int32_t from = first, keys = 0;
        for (uint32_t g = 0; g < n; ++g) {
            const int32_t to = __builtin_amdgcn_readlane(end, (int)g);
            if (from <= r && r < to) keys = __builtin_amdgcn_readlane(len, (int)g);
            from = to;
        }
        return keys;
    }
};

template <bool Planned, bool TwoWords = false>
struct SharedPages {
    static constexpr bool kShared = true, kPlanned = Planned, kTwoWords = TwoWords;
    using Request = pk::SharedRequest;
    using Tile = pk::SharedTile;
    using Left = pk::u32x4;  // the rows' records, of prefixes and then of own keys
    struct More {
        const int32_t *prefixTables, *prefixLens, *groupStarts;
        const int32_t *positions;  // under a window: of each token, then each group's least
        float *lse;
        const HeldGroups &held;
        const SharedPrefixConstants &s;
        uint32_t firstBlock;  // of a launch's blocks, the first that takes this work
    };
    const int32_t *tables, *starts, *keyLens;
    Left *left;
    const More &more;
    const uint32_t firstBlock = more.firstBlock;

    __device__ inline uint32_t requests(const PagedAttentionConstants &p) const { return more.s.groups + p.R; }
    __device__ inline Request request(uint32_t v, const PagedAttentionConstants &p) const {
        const SharedPrefixConstants &s = more.s;
        if (s.groups > 64) return pk::paged_shared(v, starts, keyLens, more.prefixLens, more.groupStarts, more.positions, p, s);
        // The request's own numbers are asked for before the groups' are waited for: cold lines take over a microsecond each.
        const uint32_t r = v < s.groups ? 0u : v - s.groups;
        const int32_t from = starts[r], to = starts[r + 1], keys = keyLens[r];
        Request q{};
        q.prefix = v < s.groups;
        if (s.groups) {
            int32_t a, b, len;
            more.held.group(q.prefix ? v : 0u, a, b, len);
            if (q.prefix) {
                a = pk::paged_min(pk::paged_max(a, 0), (int32_t)p.R);
                b = pk::paged_min(pk::paged_max(b, a), (int32_t)p.R);
                static_cast<pk::PagedRequest &>(q) = pk::paged_request(starts[a], starts[b], 0, p);
                q.keys = pk::paged_prefix_keys(len, p, s);
                if (a == b || q.keys == 0) q.n = 0;
                q.lo = s.windowed ? more.positions[p.T + v] : q.keys;
                return q;
            }
        }
        static_cast<pk::PagedRequest &>(q) = pk::paged_request(from, to, keys, p);
        q.before = pk::paged_prefix_keys(more.held.before((int32_t)r), p, s);
        return q;
    }
    __device__ inline PagedAttentionConstants mask(const Request &q, const PagedAttentionConstants &p) const { return pk::paged_shared_mask(q, p); }
    __device__ inline uint32_t tiles(const Request &q, uint32_t G, const PagedWorkConstants &w) const { return row_tiles(q, G, w); }
    __device__ inline pk::PagedSteps steps(const Request &q, uint32_t tile, const PagedAttentionConstants &p, const PagedWorkConstants &w) const {
        return pk::paged_shared_steps(q, tile, p, w);
    }
    __device__ inline const int32_t *table(uint32_t v, const PagedAttentionConstants &p) const {
        return v < more.s.groups ? more.prefixTables + (uint64_t)v * more.s.columns : tables + (uint64_t)(v - more.s.groups) * p.columns;
    }
    __device__ inline int pos(const Request &q, uint32_t r, uint32_t G) const {
        return !q.prefix ? q.pos0 + (int)(r / G) : more.s.windowed ? more.positions[(uint32_t)q.start + r / G] : q.keys;
    }
    __device__ inline void pos_range(const Request &q, uint32_t first, uint32_t last, uint32_t G, int mine, int &lo, int &hi) const {
        lo = q.prefix ? mine : q.pos0 + (int)(first / G);
        hi = q.prefix ? mine : q.pos0 + (int)(last / G);
        if (!q.prefix || !more.s.windowed) return;
#pragma unroll
        for (int d = 32; d; d >>= 1) {
            lo = min(lo, __shfl_xor(lo, d));
            hi = max(hi, __shfl_xor(hi, d));
        }
        lo = (int)first_lane((uint32_t)lo);
        hi = (int)first_lane((uint32_t)hi);
    }

    // The same request, in scalar registers. (Where the compiler took its keys for the lanes' own, each load through a descriptor
    // became a loop over the lanes' descriptors: 256 requests of 20 to 800 own keys 50 us, and 49, beside other waves; alone a step 3.3 us, and 2.4.)
    __device__ static inline Request uniform(const Request &q) {
        Request u;
        u.start = (int32_t)first_lane((uint32_t)q.start);
        u.n = (int32_t)first_lane((uint32_t)q.n);
        u.pos0 = (int32_t)first_lane((uint32_t)q.pos0);
        u.keys = (int32_t)first_lane((uint32_t)q.keys);
        u.prefix = first_lane(q.prefix);
        u.before = (int32_t)first_lane((uint32_t)q.before);
        u.lo = (int32_t)first_lane((uint32_t)q.lo);
        return u;
    }
    // Where a unit's state goes that one worker has whole.
    __device__ inline uint64_t own_row(const Request &q, uint64_t row) const { return more.s.rowBase + (q.prefix ? 0u : more.s.rows) + row; }
    // Of a piece that begins its unit: the rows' records. True where the piece is all that its rows have: they go to `out`.
    template <typename Row>
    __device__ inline bool begin(const Piece<Request> &c, bool whole, Row &&row, const PagedWorkConstants &w, uint32_t worker, uint32_t thread,
                                 uint32_t threads) const {
        const bool direct = whole && !c.req.prefix && c.req.before == 0;
        if (c.lo != 0) return false;
        for (uint32_t r = c.steps.r0 + thread; r < c.steps.r1; r += threads) {
            const uint64_t at = row(r);
            const uint32_t next = w.stateBase + 2 * worker * w.rows + (r - c.steps.r0);
            const uint32_t behind = !c.req.prefix && c.req.before > 0 ? kBehindPrefix : 0u;
            left[(c.req.prefix ? 0u : more.s.rows) + at] =
                whole ? pk::u32x4{(uint32_t)own_row(c.req, at), 0u, 0u, direct ? 0u : 1u | behind}
                      : pk::u32x4{next + w.rows, next, 2 * w.rows, c.sharers | behind};
        }
        return direct;
    }
    __device__ inline void store_lse(uint64_t row, float m, float l) const {
        if (more.s.hasLse) more.lse[row] = l == 0.0f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2;  // (logf: of base 2)
    }
};

// Under a window, a group's least position, by one wave; and a token's position (behind its group's prefix; a token that its
// request's keys do not hold counts as the first behind it).
__device__ inline int32_t group_least(uint32_t g, const int32_t *starts, const int32_t *keyLens, const int32_t *prefixLens, const int32_t *groupStarts,
                                      const PagedAttentionConstants &p, const SharedPrefixConstants &s) {
    const int32_t a = min(max(groupStarts[g], 0), (int32_t)p.R), b = min(max(groupStarts[g + 1], a), (int32_t)p.R);
    int32_t least = 0x7fffffff;
    for (int32_t r = a + (int32_t)(threadIdx.x & 63); r < b; r += 64) {
        const pk::PagedRequest q = pk::paged_request(starts[r], starts[r + 1], keyLens[r], p);
        if (q.n > 0) least = min(least, pk::paged_place(q, q.start, pk::paged_prefix_keys(prefixLens[g], p, s)));
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) least = min(least, __shfl_xor(least, d));
    return least;
}

__device__ inline void token_position(uint32_t t, const int32_t *starts, const int32_t *keyLens, const int32_t *prefixLens,
                                      const int32_t *groupStarts, int32_t *positions, const PagedAttentionConstants &p,
                                      const SharedPrefixConstants &s) {
    if (t >= p.T) return;
    const uint32_t r = pk::paged_span_of(starts, p.R, (int32_t)t);
    int32_t pos = 0;
    if (r < p.R) {
        const uint32_t g = pk::paged_span_of(groupStarts, s.groups, (int32_t)r);
        const pk::PagedRequest q = pk::paged_request(starts[r], starts[r + 1], keyLens[r], p);
        pos = pk::paged_place(q, (int32_t)t, g < s.groups ? pk::paged_prefix_keys(prefixLens[g], p, s) : 0);
    }
    positions[t] = pos;
}

}  // namespace

// The plan, before a launch that two kinds of work share: 5 us, reads that wait for each other and the scan. (Each block
// by itself would take as long, and its lists the LDS of the copies.)
// Block 0 lays out the tiles of many rows, block 1 those of few (of the few-row kernel alone there is just block 0: many is few). Each
// plan's entry 0: the counted steps, the number of tiles. Under a window both write each group's least position first, behind the
// tokens' positions, which the blocks behind them write.
POPCORN_KERNEL void __launch_bounds__(1024)
    shared_prefix_plan(const int32_t *starts, const int32_t *keyLens, const int32_t *prefixLens, const int32_t *groupStarts, int32_t *positions,
                       pk::SharedTile *plan, PagedAttentionConstants p, PagedWorkConstants many, PagedWorkConstants few, SharedPrefixConstants s) {
    if (blockIdx.x > 1) {
        token_position((blockIdx.x - 2) * 1024 + threadIdx.x, starts, keyLens, prefixLens, groupStarts, positions, p, s);
        return;
    }
    __shared__ PlanSpace<1024, u64, pk::SharedRequest> space;
    if (s.windowed) {
        for (uint32_t g = threadIdx.x >> 6; g < s.groups; g += 16) {
            const int32_t least = group_least(g, starts, keyLens, prefixLens, groupStarts, p, s);
            if ((threadIdx.x & 63) == 0) positions[p.T + g] = least;
        }
        __threadfence_block();
        __syncthreads();
    }
    const HeldGroups held(groupStarts, prefixLens, s);
    using Pages = SharedPages<true>;
    const Pages::More more{nullptr, prefixLens, groupStarts, positions, nullptr, held, s, 0};
    const Pages batch{nullptr, starts, keyLens, nullptr, more};
    u64 steps;
    uint32_t tiles;
    const PagedWorkConstants w = blockIdx.x ? few : many;
    pk::SharedTile *to = plan + (blockIdx.x ? many.maxTiles + 1 : 0u);
    lay_tiles<1024, u64>(batch, space, p, w, steps, tiles,
                         [&](uint32_t at, u64 before, uint32_t request, uint32_t tile, const pk::SharedRequest &req) {
                             to[1 + at] = pk::SharedTile{{before, request, tile}, req, 0};
                         });
    if (threadIdx.x == 0) to[0] = pk::SharedTile{{steps, tiles, 0}, {}, 0};
}

// The same for the few-row kernel alone, which lays out its plan by itself: blocks take tokens, or those past them four groups. A
// launch (24 requests 4 us), since a prefix's rows belong to many requests: a wave would search for each of its rows.
POPCORN_KERNEL void __launch_bounds__(256)
    shared_prefix_positions(const int32_t *starts, const int32_t *keyLens, const int32_t *prefixLens, const int32_t *groupStarts,
                            int32_t *positions, PagedAttentionConstants p, SharedPrefixConstants s) {
    const uint32_t tokenBlocks = (p.T + 255) / 256;
    if (blockIdx.x < tokenBlocks) return token_position(blockIdx.x * 256 + threadIdx.x, starts, keyLens, prefixLens, groupStarts, positions, p, s);
    const uint32_t g = (blockIdx.x - tokenBlocks) * 4 + (threadIdx.x >> 6);
    if (g >= s.groups) return;
    const int32_t least = group_least(g, starts, keyLens, prefixLens, groupStarts, p, s);
    if ((threadIdx.x & 63) == 0) positions[p.T + g] = least;
}

namespace {

// The launch's blocks are shared out by the counted steps, a wave's counted a quarter of a block's.
__device__ inline uint32_t tile_blocks(u64 many, u64 few) {
    const u64 fewSteps = first_lane64((few + 3) / 4), all = first_lane64(many) + fewSteps;
    const uint32_t blocks = all ? (uint32_t)((gridDim.x * fewSteps + all - 1) / all) : 0u;
    return first_lane(gridDim.x - (many ? min(blocks, gridDim.x - 1) : blocks));
}

// A row's pieces, of its prefix and of its own keys, by one wave or the block's four (s.parts): their maximum and sum first,
// a lane for a piece, then their O, HD / 4 lanes for a piece. Bound by its launch and two rounds of reads, the records and what they
// lead to: a row's own record says that there is a prefix's. (Looked up in starts and groups it took two rounds more: 16 rows 5.0 us, and
// 4.2; 6000 rows 10, and 9.) The rest is the states themselves, of 512 bytes each in 128 dims (2048 rows behind 8192 keys: 9 us).
template <typename T, int HD>
__device__ void shared_prefix_merge(const float *__restrict__ pO, const float *__restrict__ pML, const pk::u32x4 *__restrict__ records,
                                    const int32_t *__restrict__ starts, typename T::storage *__restrict__ out, float *__restrict__ lse,
                                    const PagedAttentionConstants &p, const SharedPrefixConstants &s) {
    constexpr uint32_t kLanes = HD >= 256 ? 64 : HD / 4, kAtOnce = 64 / kLanes;
    constexpr int NJ = HD > 256 ? HD / 256 : 1;
    constexpr uint32_t U = NJ > 1 ? 2 : 4;  // pieces in flight
    __shared__ __attribute__((aligned(16))) float sO[4][HD];
    const uint32_t lane = threadIdx.x & 63, wave = first_lane(threadIdx.x >> 6);
    const uint32_t part = wave % s.parts, row = blockIdx.x * (4 / s.parts) + wave / s.parts;
    if (row >= s.rows) return;  // (with four parts the whole block)
    const int32_t token = (int32_t)(row / p.Nq), from = starts[0], end = starts[p.R];
    const pk::u32x4 own = records[s.rows + row], pre = records[row];
    if (token < from || token >= end) return;  // a row of no request
    if (own.w == 0) return;                    // its piece has stored it
    // (what lengths out of order could leave here leads to no row past the states)
    const uint32_t nPre = own.w & kBehindPrefix ? min(pre.w, s.most) : 0u, n = nPre + min(own.w & ~kBehindPrefix, s.most);
    auto at = [&](uint32_t i) {
        const bool mine = i >= nPre;
        const uint32_t j = mine ? i - nPre : i;
        return (uint64_t)min(j == 0 ? (mine ? own.x : pre.x) : (mine ? own.y + j * own.z : pre.y + j * pre.z), s.states - 1);
    };
    float m = -INFINITY, l = 0.0f;
    auto weight = [&](float mi, float li, float M) { return mi == -INFINITY && li == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(mi - M); };
    const uint32_t d0 = lane % kLanes * 4, step = s.parts * kAtOnce;
    pk::f32x4 v[U][NJ];
    float2 ml[U];
    auto read = [&](uint32_t i0) {
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            const uint64_t a = at(min(i0 + u * step, n - 1));
            ml[u] = *reinterpret_cast<const float2 *>(pML + 2 * a);
#pragma unroll
            for (int j = 0; j < NJ; ++j)
                v[u][j] = d0 + 256 * j < p.Hd ? *reinterpret_cast<const pk::f32x4 *>(pO + a * HD + d0 + 256 * j) : pk::f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    };
    uint32_t i0 = part * kAtOnce + lane / kLanes;
    read(i0);  // the first of them beside the maximum's
    for (uint32_t i = lane; i < n; i += 64) {
        const float2 x = *reinterpret_cast<const float2 *>(pML + 2 * at(i));
        const float mn = fmaxf(m, x.x);
        l = (m == -INFINITY ? 0.0f : l * __builtin_amdgcn_exp2f(m - mn)) + x.y * weight(x.x, x.y, mn);
        m = mn;
    }
    const float M = pk::wave_max(m);
    const float L = pk::wave_sum(weight(m, l, M) * l);
    pk::f32x4 o[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) o[j] = pk::f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (; i0 < n;) {
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            const float w = i0 + u * step < n ? weight(ml[u].x, ml[u].y, M) : 0.0f;
            if (w != 0.0f)
#pragma unroll
                for (int j = 0; j < NJ; ++j) o[j] += v[u][j] * w;
        }
        i0 += U * step;
        if (i0 < n) read(i0);
    }
    if constexpr (kAtOnce > 1)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (kAtOnce > 2) o[0][e] = pk::pair16_sum(o[0][e]);
            o[0][e] = pk::pair32_sum(o[0][e]);
        }
    if (s.parts > 1) {
        if (lane < kLanes)
#pragma unroll
            for (int j = 0; j < NJ; ++j) *reinterpret_cast<pk::f32x4 *>(&sO[wave][d0 + 256 * j]) = o[j];
        __syncthreads();
        if (part != 0) return;
#pragma unroll
        for (int j = 0; j < NJ; ++j)
            for (uint32_t v = 1; v < s.parts; ++v) o[j] += *reinterpret_cast<const pk::f32x4 *>(&sO[v][d0 + 256 * j]);
    }
    if (lane < kLanes)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
            if (d0 + 256 * j < p.Hd) store4<T>(out + (uint64_t)row * p.Hd + d0 + 256 * j, o[j], L);
    if (lane == 0 && s.hasLse) lse[row] = L == 0.0f ? -INFINITY : (M + __builtin_amdgcn_logf(L)) * kLn2;
}

// Any head dim up to 512 and any alignment, as paged_attention_plain: a block per row, whose 16 groups of 16 lanes take runs of
// keys in turn, of the prefix and then of the row's own.
template <typename T, bool VEC>
__device__ void shared_prefix_plain(const typename T::storage *__restrict__ Q, const typename T::storage *__restrict__ K,
                                    const typename T::storage *__restrict__ V, const SharedPages<false> &batch, typename T::storage *__restrict__ out,
                                    const PagedAttentionConstants &p) {
    constexpr int NJ = 8;
    __shared__ float sO[16][NJ * 64], sM[16], sL[16];
    const SharedPrefixConstants &s = batch.more.s;
    const uint32_t row = blockIdx.x, part = threadIdx.x / 16, td = threadIdx.x % 16 * 4;
    const int32_t t = (int32_t)(row / p.Nq);
    const uint32_t hkv = row % p.Nq / (p.Nq / p.Nkv);
    const uint32_t own = pk::paged_span_of(batch.starts, p.R, t);
    if (own >= p.R) return;
    const uint32_t g = pk::paged_span_of(batch.more.groupStarts, s.groups, (int32_t)own);
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
    const pk::SharedRequest r = batch.request(s.groups + own, p);
    const int pos = r.pos0 + (t - r.start);
    if (r.before > 0) {
        const int32_t *table = batch.table(g, p);
        pk::SharedRequest pre{};
        pre.prefix = 1;
        const PagedAttentionConstants mp = batch.mask(pre, p);
        const int at = pk::paged_place(r, t, r.before);
        const pk::PagedSpan k = pk::paged_span(at, at, r.before, mp);
        paged_row<T, NJ, VEC, 2>(q, K, V, table, hkv, at, 0, k.sinkEnd, mp, o, m, l, part, 16);
        paged_row<T, NJ, VEC, 2>(q, K, V, table, hkv, at, k.lo, k.hi, mp, o, m, l, part, 16);
    }
    const PagedAttentionConstants mo = batch.mask(r, p);
    const pk::PagedSpan k = pk::paged_span(pos, pos, r.keys, mo);
    const int32_t *table = batch.table(s.groups + own, p);
    paged_row<T, NJ, VEC, 2>(q, K, V, table, hkv, pos, 0, k.sinkEnd, mo, o, m, l, part, 16);
    paged_row<T, NJ, VEC, 2>(q, K, V, table, hkv, pos, k.lo, k.hi, mo, o, m, l, part, 16);
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
    if (threadIdx.x == 0) batch.store_lse(row, M, L);
}

}  // namespace

#define SHARED_PARAMS(T)                                                                                                     \
    const T::storage *q, const T::storage *k, const T::storage *v, const int32_t *tables, const int32_t *starts,             \
        const int32_t *keyLens, const int32_t *prefixTables, const int32_t *prefixLens, const int32_t *groupStarts
// (Rows of a tile and keys of a step are the kernels' own, as the plan has them: known here they are shifts, not divisions.)
// Few rows alone.
#define SHARED_FEW(t, T, HD, RT, PER_CU)                                                                                     \
    POPCORN_KERNEL void __launch_bounds__(256, PER_CU)                                                                       \
        shared_prefix_few_##t##_d##HD##_r##RT(SHARED_PARAMS(T), const int32_t *positions, const pk::SharedTile *plan, float *pO, \
                                              float *pML, pk::u32x4 *records, T::storage *out, float *lse,                   \
                                              PagedAttentionConstants p, PagedWorkConstants w, SharedPrefixConstants s) {    \
        w.rows = 16 * RT;                                                                                                    \
        w.stepKeys = sizeof(T::storage) == 4 ? 16 : 32;                                                                      \
        const HeldGroups held(groupStarts, prefixLens, s);                                                                   \
        const SharedPages<false>::More more{prefixTables, prefixLens, groupStarts, positions, lse, held, s, 0};              \
        paged_few<T, HD, RT, SharedPages<false>, HD == 512 ? kWaves : 1>(q, k, v, tables, starts, keyLens, plan, pO, pML, records, \
                                                                         out, p, w, more);                                   \
    }
// WORDS, TWO: whether weights of the tiles have two words.
// Many rows and few in one launch: the first blocks take tiles of many rows, which the matrix cores bound, the others, a wave each,
// the requests of few, which memory bounds; so both are busy at once.
#define SHARED_BOTH(t, T, HD, PER_CU, WORDS, TWO)                                                                            \
    POPCORN_KERNEL void __launch_bounds__(256, PER_CU)                                                                       \
        shared_prefix_both_##t##_d##HD##WORDS(SHARED_PARAMS(T), const int32_t *positions, const pk::SharedTile *plan, float *pO, float *pML, \
                                       pk::u32x4 *records, T::storage *out, float *lse, PagedAttentionConstants p,           \
                                       PagedWorkConstants many, PagedWorkConstants few, SharedPrefixConstants s) {           \
        __shared__ __attribute__((aligned(256))) uint8_t lds[4 * 64 * HD * 2];                                               \
        using Pages = SharedPages<true, TWO>;                                                                                \
        const pk::SharedTile *planFew = plan + many.maxTiles + 1;                                                            \
        const uint32_t tileBlocks = tile_blocks(plan[0].before, planFew[0].before);                                          \
        many.rows = 128;                                                                                                     \
        many.stepKeys = 64;                                                                                                  \
        few.rows = 16;                                                                                                       \
        few.stepKeys = 32;                                                                                                   \
        const HeldGroups held(groupStarts, prefixLens, s);                                                                   \
        if (blockIdx.x < tileBlocks) {                                                                                       \
            many.workers = tileBlocks;                                                                                       \
            const Pages::More more{prefixTables, prefixLens, groupStarts, positions, lse, held, s, 0};                       \
            paged_tile<T, HD, Pages>(q, k, v, tables, starts, keyLens, plan, pO, pML, records, out, p, many, more, lds);     \
        } else {                                                                                                             \
            few.workers = 4 * (gridDim.x - tileBlocks);                                                                      \
            const Pages::More more{prefixTables, prefixLens, groupStarts, positions, lse, held, s, tileBlocks};              \
            paged_few<T, HD, 1, Pages, 1>(q, k, v, tables, starts, keyLens, planFew, pO, pML, records, out, p, few, more, lds); \
        }                                                                                                                    \
    }
// Many rows alone: beside the few-row kernel's code those of 256 dims, which take all registers, spilled 51 to 65 of them (a prompt of
// 2048 tokens behind 8192 keys, bf16: 332 us, and 251).
#define SHARED_MANY(t, T, HD, PER_CU, WORDS, TWO)                                                                            \
    POPCORN_KERNEL void __launch_bounds__(256, PER_CU)                                                                       \
        shared_prefix_many_##t##_d##HD##WORDS(SHARED_PARAMS(T), const int32_t *positions, const pk::SharedTile *plan, float *pO, float *pML, \
                                       pk::u32x4 *records, T::storage *out, float *lse, PagedAttentionConstants p,           \
                                       PagedWorkConstants w, SharedPrefixConstants s) {                                      \
        __shared__ __attribute__((aligned(256))) uint8_t lds[4 * 64 * HD * 2];                                               \
        w.rows = 128;                                                                                                        \
        w.stepKeys = 64;                                                                                                     \
        const HeldGroups held(groupStarts, prefixLens, s);                                                                   \
        const SharedPages<true, TWO>::More more{prefixTables, prefixLens, groupStarts, positions, lse, held, s, 0};          \
        paged_tile<T, HD, SharedPages<true, TWO>>(q, k, v, tables, starts, keyLens, plan, pO, pML, records, out, p, w, more, lds); \
    }
#define SHARED_MERGE(t, T, HD)                                                                                               \
    POPCORN_KERNEL void __launch_bounds__(256)                                                                               \
        shared_prefix_merge_##t##_d##HD(const float *pO, const float *pML, const pk::u32x4 *records, const int32_t *starts,  \
                                        T::storage *out, float *lse, PagedAttentionConstants p, SharedPrefixConstants s) {   \
        shared_prefix_merge<T, HD>(pO, pML, records, starts, out, lse, p, s);                                                \
    }
#define SHARED_PLAIN(name, T, VEC)                                                                                           \
    POPCORN_KERNEL void __launch_bounds__(256) name(SHARED_PARAMS(T), T::storage *out, float *lse, PagedAttentionConstants p, \
                                                    SharedPrefixConstants s) {                                               \
        const HeldGroups held(groupStarts, prefixLens, s);                                                                   \
        const SharedPages<false>::More more{prefixTables, prefixLens, groupStarts, nullptr, lse, held, s, 0};                \
        shared_prefix_plain<T, VEC>(q, k, v, SharedPages<false>{tables, starts, keyLens, nullptr, more}, out, p);            \
    }

using pk::BF16;
using pk::F16;
using pk::F32;

#define SHARED_ALL(t, T, PER256)                    \
    SHARED_FEW(t, T, 64, 1, 4)                      \
    SHARED_FEW(t, T, 64, 2, 3)                      \
    SHARED_FEW(t, T, 128, 1, 3)                     \
    SHARED_FEW(t, T, 128, 2, 2)                     \
    SHARED_FEW(t, T, 256, 1, PER256)                \
    SHARED_FEW(t, T, 512, 1, 1)                     \
    SHARED_MERGE(t, T, 64)                          \
    SHARED_MERGE(t, T, 128)                         \
    SHARED_MERGE(t, T, 256)                         \
    SHARED_MERGE(t, T, 512)                         \
    SHARED_PLAIN(shared_prefix_plain_##t, T, true)  \
    SHARED_PLAIN(shared_prefix_plain_##t##_any, T, false)

SHARED_ALL(f32, F32, 1)
SHARED_ALL(f16, F16, 2)
SHARED_ALL(bf16, BF16, 2)
SHARED_FEW(f16, F16, 256, 2, 1)
SHARED_FEW(bf16, BF16, 256, 2, 1)
SHARED_BOTH(f16, F16, 64, 2, , false)
SHARED_BOTH(f16, F16, 128, 2, , false)
SHARED_MANY(f16, F16, 256, 1, , false)
SHARED_BOTH(f16, F16, 64, 2, _two, true)
SHARED_BOTH(f16, F16, 128, 2, _two, true)
SHARED_MANY(f16, F16, 256, 1, _two, true)
SHARED_BOTH(bf16, BF16, 64, 2, , true)
SHARED_BOTH(bf16, BF16, 128, 2, , true)
SHARED_MANY(bf16, BF16, 256, 1, , true)
