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
#include "paged_attention.hpp"

namespace {

constexpr float kLn2 = 0.6931471805599453f;

// A wave's search: its lanes look at 64 entries at once.
__device__ inline uint32_t wave_span_of(const int32_t *at, uint32_t n, int32_t x) {
    if (n == 0 || at[0] > x) return n;
    const uint32_t a = find_tile(n, (uint64_t)(uint32_t)x, [&](uint32_t i) { return at[i] < 0 ? 0u : (uint32_t)at[i]; });
    return x < at[a + 1] ? a : n;
}

struct SharedPages {
    static constexpr bool kShared = true;
    using Request = pk::SharedRequest;
    using Left = pk::u32x4;  // the rows' records, of prefixes and then of own keys
    struct More {
        const int32_t *prefixTables, *prefixLens, *groupStarts;
        const int32_t *positions;  // under a window: of each token, then each group's least
        float *lse;
        const SharedPrefixConstants &s;
    };
    const int32_t *tables, *starts, *keyLens;
    Left *left;
    const More &more;

    __device__ inline uint32_t requests(const PagedAttentionConstants &p) const { return more.s.groups + p.R; }
    __device__ inline Request request(uint32_t v, const PagedAttentionConstants &p) const {
        return pk::paged_shared(v, starts, keyLens, more.prefixLens, more.groupStarts, more.positions, p, more.s);
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

    // Where a unit's state goes that one worker has whole.
    __device__ inline uint64_t own_row(const Request &q, uint64_t row) const { return more.s.rowBase + (q.prefix ? 0u : more.s.rows) + row; }
    // Of a piece that begins its unit: the rows' records. True where the piece is all that its rows have: they go to `out`.
    template <typename Row>
    __device__ inline bool begin(const Piece<Request> &c, bool whole, Row &&row, const PagedAttentionConstants &p, const PagedWorkConstants &w) const {
        const bool direct = whole && !c.req.prefix && c.req.before == 0;
        if (c.lo != 0) return false;
        for (uint32_t r = c.steps.r0 + threadIdx.x; r < c.steps.r1; r += 256) {
            const uint64_t at = row(r);
            const uint32_t next = w.stateBase + 2 * blockIdx.x * w.rows + (r - c.steps.r0);
            left[(c.req.prefix ? 0u : more.s.rows) + at] =
                whole ? pk::u32x4{(uint32_t)own_row(c.req, at), 0u, 0u, direct ? 0u : 1u} : pk::u32x4{next + w.rows, next, 2 * w.rows, c.sharers};
        }
        return direct;
    }
    __device__ inline void store_lse(uint64_t row, float m, float l) const {
        if (more.s.hasLse) more.lse[row] = l == 0.0f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2;  // (logf: of base 2)
    }
};

}  // namespace

POPCORN_KERNEL void __launch_bounds__(1024)
    shared_prefix_plan(const int32_t *starts, const int32_t *keyLens, const int32_t *prefixLens, const int32_t *groupStarts,
                       const int32_t *positions, pk::PagedTile *plan, PagedAttentionConstants p, PagedWorkConstants w,
                       SharedPrefixConstants s) {
    __shared__ PlanSpace<1024, u64, SharedPages::Request> space;
    u64 steps;
    uint32_t tiles;
    const SharedPages::More more{nullptr, prefixLens, groupStarts, positions, nullptr, s};
    const SharedPages batch{nullptr, starts, keyLens, nullptr, more};
    lay_tiles<1024, u64>(batch, space, p, w, steps, tiles, [&](uint32_t at, u64 before, uint32_t request, uint32_t tile) {
        plan[1 + at] = pk::PagedTile{before, request, tile};
    });
    if (threadIdx.x == 0) plan[0] = pk::PagedTile{steps, tiles, 0};
}

// Under a window: each token's position (behind its group's prefix; a token that its request's keys do not hold counts as the
// first behind it), and behind the tokens each group's least. A block's threads take tokens, or the blocks past them one group.
POPCORN_KERNEL void __launch_bounds__(256)
    shared_prefix_positions(const int32_t *starts, const int32_t *keyLens, const int32_t *prefixLens, const int32_t *groupStarts,
                            int32_t *positions, PagedAttentionConstants p, SharedPrefixConstants s) {
    const uint32_t tokenBlocks = (p.T + 255) / 256;
    if (blockIdx.x < tokenBlocks) {
        const uint32_t t = blockIdx.x * 256 + threadIdx.x;
        if (t >= p.T) return;
        const uint32_t r = pk::paged_span_of(starts, p.R, (int32_t)t);
        int32_t pos = 0;
        if (r < p.R) {
            const uint32_t g = pk::paged_span_of(groupStarts, s.groups, (int32_t)r);
            const pk::PagedRequest q = pk::paged_request(starts[r], starts[r + 1], keyLens[r], p);
            pos = pk::paged_place(q, (int32_t)t, g < s.groups ? pk::paged_prefix_keys(prefixLens[g], p, s) : 0);
        }
        positions[t] = pos;
        return;
    }
    __shared__ int32_t sLeast[4];
    const uint32_t g = blockIdx.x - tokenBlocks;
    if (g >= s.groups) return;
    const int32_t a = min(max(groupStarts[g], 0), (int32_t)p.R), b = min(max(groupStarts[g + 1], a), (int32_t)p.R);
    int32_t least = 0x7fffffff;
    for (int32_t r = a + (int32_t)threadIdx.x; r < b; r += 256) {
        const pk::PagedRequest q = pk::paged_request(starts[r], starts[r + 1], keyLens[r], p);
        if (q.n > 0) least = min(least, pk::paged_place(q, q.start, pk::paged_prefix_keys(prefixLens[g], p, s)));
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) least = min(least, __shfl_xor(least, d));
    if ((threadIdx.x & 63) == 0) sLeast[threadIdx.x >> 6] = least;
    __syncthreads();
    if (threadIdx.x != 0) return;
    positions[p.T + g] = min(min(sLeast[0], sLeast[1]), min(sLeast[2], sLeast[3]));
}

namespace {

// A row's pieces, of its prefix and of its own keys, by one wave or the block's four (s.parts): their maximum and sum first,
// a lane for a piece, then their O, HD / 4 lanes for a piece.
template <typename T, int HD>
__device__ void shared_prefix_merge(const float *__restrict__ pO, const float *__restrict__ pML, const pk::u32x4 *__restrict__ records,
                                    const int32_t *__restrict__ starts, const int32_t *__restrict__ prefixLens,
                                    const int32_t *__restrict__ groupStarts, typename T::storage *__restrict__ out, float *__restrict__ lse,
                                    const PagedAttentionConstants &p, const SharedPrefixConstants &s) {
    constexpr uint32_t kLanes = HD >= 256 ? 64 : HD / 4, kAtOnce = 64 / kLanes;
    constexpr int NJ = HD > 256 ? HD / 256 : 1;
    constexpr uint32_t U = NJ > 1 ? 2 : 4;  // pieces in flight
    __shared__ __attribute__((aligned(16))) float sO[4][HD];
    const uint32_t lane = threadIdx.x & 63, wave = first_lane(threadIdx.x >> 6);
    const uint32_t part = wave % s.parts, row = blockIdx.x * (4 / s.parts) + wave / s.parts;
    if (row >= s.rows) return;  // (with four parts the whole block)
    const uint32_t r = wave_span_of(starts, p.R, (int32_t)(row / p.Nq));
    if (r >= p.R) return;
    const uint32_t g = wave_span_of(groupStarts, s.groups, (int32_t)r);
    const bool shared = g < s.groups && pk::paged_prefix_keys(prefixLens[g], p, s) > 0;
    const pk::u32x4 own = records[s.rows + row];
    if (!shared && own.w == 0) return;  // its piece has stored it
    const pk::u32x4 pre = shared ? records[row] : pk::u32x4{0u, 0u, 0u, 0u};
    // (what lengths out of order could leave here leads to no row past the states)
    const uint32_t nPre = min(pre.w, s.most), n = nPre + min(own.w, s.most);
    auto at = [&](uint32_t i) {
        const bool mine = i >= nPre;
        const uint32_t j = mine ? i - nPre : i;
        return (uint64_t)min(j == 0 ? (mine ? own.x : pre.x) : (mine ? own.y + j * own.z : pre.y + j * pre.z), s.states - 1);
    };
    float m = -INFINITY, l = 0.0f;
    auto weight = [&](float mi, float li, float M) { return mi == -INFINITY && li == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(mi - M); };
    for (uint32_t i = lane; i < n; i += 64) {
        const float2 ml = *reinterpret_cast<const float2 *>(pML + 2 * at(i));
        const float mn = fmaxf(m, ml.x);
        l = (m == -INFINITY ? 0.0f : l * __builtin_amdgcn_exp2f(m - mn)) + ml.y * weight(ml.x, ml.y, mn);
        m = mn;
    }
    const float M = pk::wave_max(m);
    const float L = pk::wave_sum(weight(m, l, M) * l);
    pk::f32x4 o[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) o[j] = pk::f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const uint32_t d0 = lane % kLanes * 4, step = s.parts * kAtOnce;
    for (uint32_t i0 = part * kAtOnce + lane / kLanes; i0 < n; i0 += U * step) {
        pk::f32x4 v[U][NJ];
        float2 ml[U];
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            const uint64_t a = at(min(i0 + u * step, n - 1));
            ml[u] = *reinterpret_cast<const float2 *>(pML + 2 * a);
#pragma unroll
            for (int j = 0; j < NJ; ++j) v[u][j] = d0 + 256 * j < p.Hd ? *reinterpret_cast<const pk::f32x4 *>(pO + a * HD + d0 + 256 * j) : o[j];
        }
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            const float w = i0 + u * step < n ? weight(ml[u].x, ml[u].y, M) : 0.0f;
            if (w != 0.0f)
#pragma unroll
                for (int j = 0; j < NJ; ++j) o[j] += v[u][j] * w;
        }
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
                                    const typename T::storage *__restrict__ V, const SharedPages &batch, typename T::storage *__restrict__ out,
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
    const SharedPages::Request r = batch.request(s.groups + own, p);
    const int pos = r.pos0 + (t - r.start);
    if (r.before > 0) {
        const int32_t *table = batch.table(g, p);
        SharedPages::Request pre{};
        pre.prefix = true;
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
#define SHARED_WORK(name, T, PER_CU, CALL)                                                                                   \
    POPCORN_KERNEL void __launch_bounds__(256, PER_CU)                                                                       \
        name(SHARED_PARAMS(T), const int32_t *positions, const pk::PagedTile *plan, float *pO, float *pML, pk::u32x4 *records, \
             T::storage *out, float *lse, PagedAttentionConstants p, PagedWorkConstants w, SharedPrefixConstants s) {        \
        const SharedPages::More more{prefixTables, prefixLens, groupStarts, positions, lse, s};                              \
        CALL(q, k, v, tables, starts, keyLens, plan, pO, pML, records, out, p, w, more);                                     \
    }
#define SHARED_FEW(t, T, HD, RT, PER_CU) \
    SHARED_WORK(shared_prefix_few_##t##_d##HD##_r##RT, T, PER_CU, (paged_few<T, HD, RT, SharedPages>))
#define SHARED_TILE(t, T, HD, PER_CU) SHARED_WORK(shared_prefix_tile_##t##_d##HD, T, PER_CU, (paged_tile<T, HD, SharedPages>))
#define SHARED_MERGE(t, T, HD)                                                                                               \
    POPCORN_KERNEL void __launch_bounds__(256)                                                                               \
        shared_prefix_merge_##t##_d##HD(const float *pO, const float *pML, const pk::u32x4 *records, const int32_t *starts,  \
                                        const int32_t *prefixLens, const int32_t *groupStarts, T::storage *out, float *lse,  \
                                        PagedAttentionConstants p, SharedPrefixConstants s) {                                \
        shared_prefix_merge<T, HD>(pO, pML, records, starts, prefixLens, groupStarts, out, lse, p, s);                       \
    }
#define SHARED_PLAIN(name, T, VEC)                                                                                           \
    POPCORN_KERNEL void __launch_bounds__(256) name(SHARED_PARAMS(T), T::storage *out, float *lse, PagedAttentionConstants p, \
                                                    SharedPrefixConstants s) {                                               \
        const SharedPages::More more{prefixTables, prefixLens, groupStarts, nullptr, lse, s};                                \
        shared_prefix_plain<T, VEC>(q, k, v, SharedPages{tables, starts, keyLens, nullptr, more}, out, p);                   \
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
SHARED_TILE(f16, F16, 64, 2)
SHARED_TILE(f16, F16, 128, 2)
SHARED_TILE(f16, F16, 256, 1)
SHARED_TILE(bf16, BF16, 64, 2)
SHARED_TILE(bf16, BF16, 128, 2)
SHARED_TILE(bf16, BF16, 256, 1)
