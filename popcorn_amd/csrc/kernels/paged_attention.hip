// Attention of the new tokens of a batch of requests over a paged cache
// [pages, Nkv, pageSize, Hd]: out = softmax(scale q K^T | visible keys) V per
// request, query heads in groups per KV head, with the lengths and the pages
// read on the GPU.
#include "mfma.hpp"
#include "paged.hpp"

namespace {

constexpr float kLog2e = 1.4426950408889634f;

// One row's O, m (log2 units) and l over those of the keys [k0, k1) that it
// sees, in f32 on the vector ALUs with weights of at most 1. 16 lanes per
// row, lane t's dims 4 t + 64 j; VEC: rows in whole, aligned fours.
template <typename T, int NJ, bool VEC>
__device__ inline void paged_row(const pk::f32x4 (&q)[NJ], const typename T::storage *__restrict__ K,
                                 const typename T::storage *__restrict__ V, const int32_t *__restrict__ table, uint32_t hkv,
                                 int pos, int k0, int k1, const PagedAttentionConstants &p, pk::f32x4 (&o)[NJ], float &m, float &l) {
    constexpr int U = NJ > 4 ? 2 : 4;  // keys in flight
    const uint32_t D = p.Hd, td = threadIdx.x % 16 * 4;
    const float c2 = p.scale * kLog2e;
    auto load = [&](const typename T::storage *row, int j) {
        pk::f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
        const uint32_t d = td + 64 * j;
        if constexpr (VEC && sizeof(typename T::storage) == 4) {
            if (d < D) x = *reinterpret_cast<const pk::f32x4 *>(row + d);
        } else if constexpr (VEC) {
            if (d < D) {
                const pk::u32x2 v = *reinterpret_cast<const pk::u32x2 *>(row + d);
                x = pk::f32x4{pk::from_bits16<T>(v.x & 0xffffu), pk::from_bits16<T>(v.x >> 16), pk::from_bits16<T>(v.y & 0xffffu),
                              pk::from_bits16<T>(v.y >> 16)};
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (d + i < D) x[i] = T::load(row[d + i]);
        }
        return x;
    };
    for (int k = k0; k < k1; k += U) {
        pk::f32x4 kv[U][NJ], vv[U][NJ];
        bool in[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t key = (uint32_t)min(k + u, k1 - 1), column = key / p.pageSize;
            const uint32_t page = (uint32_t)table[column];
            in[u] = page < p.pages && k + u < k1;
            const uint64_t row = (((uint64_t)(page < p.pages ? page : 0u) * p.Nkv + hkv) * p.pageSize + (key - column * p.pageSize)) * D;
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                kv[u][j] = load(K + row, j);
                vv[u][j] = load(V + row, j);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float s = 0.0f;
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) s = fmaf(q[j][i], kv[u][j][i], s);
            s = pk::group_sum<16>(s) * c2;
            if (!in[u] || !pk::paged_sees(pos, k + u, p)) continue;  // a row's lanes together
            const float mn = fmaxf(m, s);
            if (mn == -INFINITY && s == -INFINITY) continue;  // (a NaN is not left out)
            const float alpha = __builtin_amdgcn_exp2f(m - mn), w = __builtin_amdgcn_exp2f(s - mn);
            l = l * alpha + w;
            m = mn;
#pragma unroll
            for (int j = 0; j < NJ; ++j) o[j] = o[j] * alpha + vv[u][j] * w;
        }
    }
}

// Any head dim up to 512 and any alignment: 16 rows per block, row b * 16 + i
// of the T * Nq (token, head) pairs.
template <typename T, bool VEC>
__device__ void paged_plain(const typename T::storage *__restrict__ Q, const typename T::storage *__restrict__ K,
                            const typename T::storage *__restrict__ V, const int32_t *__restrict__ tables,
                            const int32_t *__restrict__ starts, const int32_t *__restrict__ keyLens,
                            typename T::storage *__restrict__ out, const PagedAttentionConstants &p) {
    constexpr int NJ = 8;
    const uint64_t row = (uint64_t)blockIdx.x * 16 + threadIdx.x / 16;
    const int32_t t = (int32_t)min(row / p.Nq, (uint64_t)p.T - 1);
    const uint32_t hq = (uint32_t)(row % p.Nq), hkv = hq / (p.Nq / p.Nkv), td = threadIdx.x % 16 * 4;
    // the last request that starts at or before t
    uint32_t a = 0, b = p.R;  // starts[a] <= t < starts[b], if any does
    while (b - a > 1) {
        const uint32_t mid = (a + b) / 2;
        if (starts[mid] <= t) a = mid;
        else b = mid;
    }
    const pk::PagedRequest r = pk::paged_request(starts[a], starts[a + 1], keyLens[a], p);
    const bool live = row < (uint64_t)p.T * p.Nq && t >= r.start && t < r.start + r.n;
    if (!live) return;  // (a row's lanes together)
    const int pos = r.pos0 + (t - r.start);
    const pk::PagedSpan s = pk::paged_span(pos, pos, r.keys, p);
    pk::f32x4 q[NJ], o[NJ];
    const typename T::storage *qr = Q + row * p.Hd;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
        o[j] = q[j] = pk::f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (td + 64 * j + i < p.Hd) q[j][i] = T::load(qr[td + 64 * j + i]);
    }
    float m = -INFINITY, l = 0.0f;
    const int32_t *table = tables + (uint64_t)a * p.columns;
    paged_row<T, NJ, VEC>(q, K, V, table, hkv, pos, 0, s.sinkEnd, p, o, m, l);
    paged_row<T, NJ, VEC>(q, K, V, table, hkv, pos, s.lo, s.hi, p, o, m, l);
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t d = td + 64 * j + i;
            if (d < p.Hd) out[row * p.Hd + d] = T::store(l != 0.0f ? o[j][i] / l : 0.0f);
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
