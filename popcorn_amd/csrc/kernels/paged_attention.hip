// PagedAttention's kernels: the plan, paged_few and paged_tile over every request's own pages, the merge of what several blocks
// shared, and the form for any head dim and alignment.
#include "paged_attention.hpp"

POPCORN_KERNEL void __launch_bounds__(1024)
    paged_plan(const int32_t *starts, const int32_t *keyLens, pk::PagedTile *plan, PagedAttentionConstants p, PagedWorkConstants w) {
    __shared__ PlanSpace<1024, u64, pk::PagedRequest> space;
    u64 steps;
    uint32_t tiles;
    const OwnPages batch{nullptr, starts, keyLens, nullptr, {}};
    lay_tiles<1024, u64>(batch, space, p, w, steps, tiles, [&](uint32_t at, u64 before, uint32_t request, uint32_t tile, const auto &) {
        plan[1 + at] = pk::PagedTile{before, request, tile};
    });
    if (threadIdx.x == 0) plan[0] = pk::PagedTile{steps, tiles, 0};
}

namespace {

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
        paged_few<T, HD, RT, OwnPages>(q, k, v, tables, starts, keyLens, plan, pO, pML, shared, out, p, w, {});                         \
    }
#define PAGED_TILE(name, T, HD, PER_CU)                                                                                   \
    POPCORN_KERNEL void __launch_bounds__(256, PER_CU)                                                                    \
        name(const T::storage *q, const T::storage *k, const T::storage *v, const int32_t *tables, const int32_t *starts,       \
             const int32_t *keyLens, const pk::PagedTile *plan, float *pO, float *pML, Shared *shared, T::storage *out,     \
             PagedAttentionConstants p, PagedWorkConstants w) {                                                           \
        paged_tile<T, HD, OwnPages>(q, k, v, tables, starts, keyLens, plan, pO, pML, shared, out, p, w, {});                            \
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
