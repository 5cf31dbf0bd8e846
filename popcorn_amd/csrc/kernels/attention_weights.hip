// What a step's attention gives each cached key:
//   weights[r, hkv, k] += sum of exp(scale q.k - lse) over request r's rows (its last lastRows new tokens, and the query heads
//   of KV head hkv) that see key k,
// with the rows' lse from the attention before. K is read once more, V is not, and a key's sum belongs to one
// wave, so that no order of atomics shows in it.
#include "paged_attention.hpp"

namespace {

// A request of the call: the rows that count are tokens start .. start + n - 1, token i at position pos0 + i.
__device__ inline pk::PagedRequest weights_request(const int32_t *starts, const int32_t *keyLens, uint32_t r, const PagedAttentionConstants &p,
                                                   const AttentionWeightsConstants &w) {
    pk::PagedRequest q = pk::paged_request(starts[r], starts[r + 1], keyLens[r], p);
    if (w.lastRows && (uint32_t)q.n > w.lastRows) {
        q.pos0 += q.n - (int32_t)w.lastRows;
        q.start += q.n - (int32_t)w.lastRows;
        q.n = (int32_t)w.lastRows;
    }
    return q;
}

// Groups of 16 keys that a launch reads of a request, for one KV head.
__device__ inline uint32_t weights_groups(const pk::PagedRequest &q, const PagedAttentionConstants &p, const AttentionWeightsConstants &w) {
    const uint32_t rows = (uint32_t)q.n * (p.Nq / p.Nkv);
    if (rows <= w.fewRows || rows > w.manyRows) return 0;
    const int32_t last = q.pos0 + q.n - 1;  // (a key behind the last row is nobody's)
    const int32_t keys = p.maskKind == 2u ? q.keys : min(q.keys, max(last, -1) + 1);
    return ((uint32_t)keys + 15) / 16;
}

constexpr uint32_t kOwn = 1024;  // requests that a block sums by itself

}  // namespace

// before[r]: groups of the requests before r; before[R]: of all.
POPCORN_KERNEL void __launch_bounds__(1024)
    attention_weights_plan(const int32_t *starts, const int32_t *keyLens, uint64_t *before, PagedAttentionConstants p, AttentionWeightsConstants w) {
    __shared__ uint64_t sums[16];
    uint64_t run = 0;
    for (uint32_t base = 0; base < p.R; base += 1024) {
        const uint32_t r = base + threadIdx.x;
        const uint64_t n = r < p.R ? weights_groups(weights_request(starts, keyLens, r, p, w), p, w) : 0u;
        const pk::Scan<uint64_t> s = pk::block_scan<16>(n, sums);
        if (r < p.R) before[r] = run + s.upto - n;
        run += s.total;
    }
    if (threadIdx.x == 0) before[p.R] = run;
}

namespace {

// A few rows: a wave takes a stretch of the groups of all (request, KV head), 16 KM keys at a time: S^T = K . Q^T on 16x16
// products, so that a key's scores lie in the 16 lanes of a row of lanes, K from memory to fragments a step ahead. Memory bounds it, K
// being read once and nothing else to speak of: 48 requests of 100 to 12000 keys, 8 heads of 128, 234 MB in 54 us, 4.3 TB/s.
template <typename T, int HD, int KM>
__device__ void weights_few(const typename T::storage *__restrict__ Q, const typename T::storage *__restrict__ K,
                            const int32_t *__restrict__ tables, const int32_t *__restrict__ starts, const int32_t *__restrict__ keyLens,
                            const float *__restrict__ lse, const uint64_t *__restrict__ plan, float *__restrict__ weights,
                            const PagedAttentionConstants &p, const AttentionWeightsConstants &w) {
    using S = typename T::storage;
    constexpr bool kWide = sizeof(S) == 4;
    constexpr int E = 16 / sizeof(S), KS = HD / (4 * E);
    __shared__ uint32_t sBefore[kOwn + 1];
    __shared__ uint32_t sSums[4];
    const uint32_t lane = threadIdx.x & 63, g = lane >> 4, c16 = lane & 15, wave = first_lane(threadIdx.x >> 6);
    const uint32_t D = p.Hd, G = p.Nq / p.Nkv;
    const float c2 = p.scale * kLog2e;
    const uint64_t room = (uint64_t)p.columns * p.pageSize;
    if (w.ownPlan) {
        uint32_t run = 0;
        for (uint32_t base = 0; base < p.R; base += 256) {
            const uint32_t r = base + threadIdx.x;
            const uint32_t n = r < p.R ? weights_groups(weights_request(starts, keyLens, r, p, w), p, w) : 0u;
            const pk::Scan<uint32_t> s = pk::block_scan<4>(n, sSums);
            if (r < p.R) sBefore[r] = run + s.upto - n;
            run += s.total;
        }
        if (threadIdx.x == 0) sBefore[p.R] = run;
        __syncthreads();
    }
    auto before = [&](uint32_t r) { return w.ownPlan ? (uint64_t)sBefore[r] : plan[r]; };
    const uint64_t total = before(p.R) * p.Nkv, workers = (uint64_t)gridDim.x * 4;
    // steps of KM groups, so that a wave's stretch begins where a step of the whole does
    const uint64_t share = ((total + workers - 1) / workers + KM - 1) / KM * KM;
    uint64_t x = ((uint64_t)blockIdx.x * 4 + wave) * share;
    const uint64_t end = min(x + share, total);
    if (x >= end) return;
    uint32_t r;
    {
        uint32_t a = 0, b = p.R;  // the last request that begins at or before x
        while (b - a > 1) {
            const uint32_t mid = (a + b) / 2;
            if (before(mid) * p.Nkv <= x) a = mid;
            else b = mid;
        }
        r = first_lane(a);
    }
    while (x < end) {
        const uint64_t from = before(r) * p.Nkv;
        const uint32_t groups = first_lane((uint32_t)(before(r + 1) - before(r)));
        if (groups == 0) {
            ++r;
            continue;
        }
        const uint32_t in = (uint32_t)(x - from), hkv = first_lane(in / groups), g0 = first_lane(in - hkv * groups);
        const uint32_t g1 = (uint32_t)min((uint64_t)groups, g0 + (end - x));
        const pk::PagedRequest q = weights_request(starts, keyLens, r, p, w);
        const int32_t *table = tables + (uint64_t)r * p.columns;
        const uint32_t keys = (uint32_t)q.keys, rows = (uint32_t)q.n * G;
        float *to = weights + ((uint64_t)r * p.Nkv + hkv) * room;
        for (uint32_t r0 = 0; r0 < rows; r0 += 16) {
            // this lane's row; those past the last give nothing
            const uint32_t row = min(r0 + c16, rows - 1);
            const uint64_t at = ((uint64_t)(uint32_t)q.start + row / G) * p.Nq + hkv * G + row % G;
            const int pos = q.pos0 + (int)(row / G);
            const float of = lse[at] * kLog2e;
            const bool counts = r0 + c16 < rows && of != -INFINITY;
            u32x4 qf[KS];
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const uint32_t d = (s * 4 + g) * E;
                qf[s] = d < D ? *reinterpret_cast<const u32x4 *>(Q + at * D + d) : u32x4{0u, 0u, 0u, 0u};
            }
            u32x4 kf[KM][KS];
            float old[KM];
            bool ok[KM];
            // lane l holds the page of group held0 + l, so that no read of K waits for its page (54.5 us above, and 53.8)
            uint32_t held0 = 0, heldPage = 0;
            auto hold = [&](uint32_t grp) {
                held0 = grp;
                heldPage = grp + lane < g1 ? (uint32_t)table[(grp + lane) * 16 / p.pageSize] : ~0u;
            };
            auto load = [&](uint32_t grp) {
#pragma unroll
                for (int m = 0; m < KM; ++m) {
                    const uint32_t key = (grp + m) * 16, column = key / p.pageSize;
                    const bool in = grp + m < g1;
                    const uint32_t page = (uint32_t)__builtin_amdgcn_readlane((int)heldPage, (int)(grp + m - held0));
                    ok[m] = page < p.pages;
                    const uint64_t off = ok[m] ? (((uint64_t)page * p.Nkv + hkv) * p.pageSize + (key - column * p.pageSize)) * D : 0;
                    const int bytes = ok[m] ? (int)(min(16u, keys - key) * D * (uint32_t)sizeof(S)) : 0;
                    const auto rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<S *>(K + off), 0, bytes, 0x00020000);
#pragma unroll
                    for (int s = 0; s < KS; ++s) {
                        const uint32_t d = (s * 4 + g) * E;
                        kf[m][s] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                                                 rs, d < D ? (int)((c16 * D + d) * sizeof(S)) : kOutOfRange, 0, 0));
                    }
                    old[m] = 0.0f;
                    if (in && c16 < 4 && key + 4 * g + c16 < keys) old[m] = to[key + 4 * g + c16];
                }
            };
            hold(g0);
            load(g0);
            for (uint32_t grp = g0; grp < g1; grp += KM) {
                pk::f32x4 st[KM];
                float was[KM];
                bool held[KM];
#pragma unroll
                for (int m = 0; m < KM; ++m) {
                    st[m] = pk::f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int s = 0; s < KS; ++s) {
                        if constexpr (kWide) {
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                st[m] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kf[m][s][e]), __uint_as_float(qf[s][e]), st[m], 0, 0, 0);
                        } else {
                            st[m] = pk::Mma16<T>::run(kf[m][s], qf[s], st[m]);
                        }
                    }
                    was[m] = old[m];
                    held[m] = ok[m];
                }
                if (grp + KM < g1) {
                    if (grp + KM - held0 == 64) hold(grp + KM);
                    load(grp + KM);
                }
#pragma unroll
                for (int m = 0; m < KM; ++m) {
                    const uint32_t key0 = (grp + m) * 16 + 4 * g;
                    float mine = 0.0f;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const bool seen = counts & (p.maskKind == 2u || (int)(key0 + j) <= pos);
                        const float sum = pk::row16_sum(seen ? __builtin_amdgcn_exp2f(fmaf(st[m][j], c2, -of)) : 0.0f);
                        if (c16 == (uint32_t)j) mine = sum;
                    }
                    if (held[m] && grp + m < g1 && c16 < 4 && key0 + c16 < keys) to[key0 + c16] = was[m] + mine;
                }
            }
        }
        x += g1 - g0;
        if (x >= from + (uint64_t)groups * p.Nkv) ++r;
    }
}

// ---- many rows: prompts -------------------------------------------------------------------
// A unit is 256 keys of a request for one KV head, 64 to a wave, whose fragments stay in registers, on v_mfma_f32_32x32x16: S^T =
// K . Q^T has a row's scores in a lane of each half, so a key's sum over rows is added up in its own register, and over the
// lanes once at the end. Steps are 64 rows of Q, copied straight into LDS, three steps ahead. The units' steps
// in a row are dealt out as for attention; of a unit that several blocks share each leaves 256 partial sums.
// K stays and Q streams, since a key's sum is what is wanted: with Q held, each key's would go through LDS or atomics. The products bound
// it, an exponential and a sum beside each of their outputs: 16384 tokens, 8 heads on 4 of 256, 852 TFLOP/s causal, 1127 with every key
// seen; 4096 tokens 637 (54 us, 15 of them the blocks' starts and 5 the join).
constexpr uint32_t kKeys = 256, kStageRows = 64;

struct WeightsBatch {
    static constexpr bool kShared = false, kPlanned = false;
    using Request = pk::PagedRequest;
    using Tile = pk::PagedTile;
    struct Left {  // a unit that its block shares with others behind it
        uint32_t pieces, request, hkv, key0, keys, pad[3];
    };
    const int32_t *starts, *keyLens;
    Left *left;
    const AttentionWeightsConstants &a;

    __device__ inline uint32_t requests(const PagedAttentionConstants &p) const { return p.R; }
    __device__ inline Request request(uint32_t r, const PagedAttentionConstants &p) const { return weights_request(starts, keyLens, r, p, a); }
    __device__ inline uint32_t tiles(const Request &q, uint32_t G, const PagedWorkConstants &w) const {
        const uint32_t rows = (uint32_t)q.n * G;
        if (rows <= w.fewRows || rows > w.manyRows) return 0;
        const int32_t keys = a.everyKey ? q.keys : min(q.keys, max(q.pos0 + q.n - 1, -1) + 1);
        return ((uint32_t)keys + kKeys - 1) / kKeys;
    }
    // Steps of rows from the first that sees a key.
    __device__ inline pk::PagedSteps steps(const Request &q, uint32_t tile, const PagedAttentionConstants &p, const PagedWorkConstants &) const {
        const uint32_t G = p.Nq / p.Nkv;
        pk::PagedSteps s{};
        s.first = a.everyKey ? 0u : (uint32_t)max((int64_t)tile * kKeys - q.pos0, (int64_t)0) * G / kStageRows;
        s.n = ((uint32_t)q.n * G + kStageRows - 1) / kStageRows - s.first;
        return s;
    }
    __device__ static inline void idle(Left *to) { to->pieces = 0; }
    __device__ static inline void close(Left *to, const Piece<Request> &c, uint32_t sharers, const PagedWorkConstants &) {
        *to = Left{sharers, c.request, c.hkv, c.tile * kKeys, (uint32_t)c.req.keys, {}};
    }
};

template <typename T, int HD>
__device__ void weights_tile(const typename T::storage *__restrict__ Q, const typename T::storage *__restrict__ K,
                             const int32_t *__restrict__ tables, const int32_t *__restrict__ starts, const int32_t *__restrict__ keyLens,
                             const float *__restrict__ lse, const pk::PagedTile *__restrict__ plan, float *__restrict__ partial,
                             WeightsBatch::Left *__restrict__ left, float *__restrict__ weights, const PagedAttentionConstants &p,
                             const PagedWorkConstants &w, const AttentionWeightsConstants &a) {
    using S = typename T::storage;
    constexpr int KS = HD / 16, CH = HD / 8;
    constexpr int kRowsPer = 64 / CH;       // rows per copy instruction
    constexpr int kCopies = 16 / kRowsPer;  // instructions for a wave's 16 rows of a stage
    // A step takes less than a copy's latency, so copies run three steps ahead: four places for 64 rows and, for each wave, their
    // logarithms.
    constexpr uint32_t kPlaces = 4, kStageBytes = kStageRows * HD * 2, kLse = kPlaces * kStageBytes, kPlan = kLse + kPlaces * 4 * 256;
    __shared__ __attribute__((aligned(256))) uint8_t smem[kPlan + kOwnTiles * sizeof(OwnTile)];
    using Space = PlanSpace<256, uint32_t, pk::PagedRequest>;
    static_assert(sizeof(Space) <= kLse, "the plan is laid out where Q goes");
    OwnTile *sm_plan = reinterpret_cast<OwnTile *>(smem + kPlan);
    const uint32_t lane = threadIdx.x & 63, h = lane >> 5, c32 = lane & 31, wave = first_lane(threadIdx.x >> 6);
    const uint32_t D = p.Hd, G = p.Nq / p.Nkv;
    const float c2 = fabsf(p.scale) * kLog2e;
    const uint32_t flip = p.scale < 0.0f ? 0x80008000u : 0u;  // -scale K . Q = scale -K . Q
    auto swz = [](uint32_t row) { return CH >= 16 ? row % 16u : row / 2u % 8u; };
    // row / G: rows are below 2^24 and G at most 256, so that row (ceil(2^32 / G) G - 2^32) stays below 2^32
    const uint32_t inverse = G == 1 ? 0u : (uint32_t)((0x100000000ull + G - 1) / G), single = G == 1 ? ~0u : 0u;
    auto token_of = [&](uint32_t row) { return __umulhi(row, inverse) + (row & single); };
    const WeightsBatch batch{starts, keyLens, left, a};
    Dealer<256, WeightsBatch> dealer(batch, plan, sm_plan, reinterpret_cast<Space *>(smem), p, w);
    Piece<pk::PagedRequest> c;
    while (dealer.next(c, p, w)) {
        const int32_t *table = tables + (uint64_t)c.request * p.columns;
        const uint32_t keys = (uint32_t)c.req.keys, rows = (uint32_t)c.req.n * G, key0 = c.tile * kKeys + wave * 64;
        auto page_of = [&](uint32_t key) { return key < keys ? (uint32_t)table[key / p.pageSize] : ~0u; };
        // Q's rows of a step and their logarithms. Those past the request's last give nothing, whatever they hold; those past the
        // tensor's are zeros. (Always as many instructions.) Where G divides a step its rows lie alike in every step.
        const uint32_t n = c.hi - c.lo, row0 = (c.steps.first + c.lo) * kStageRows;
        const bool alike = kStageRows % G == 0;
        uint32_t at[kCopies], lseAt = 0;
        auto lay = [&](uint32_t first) {
            const uint32_t token = token_of(first);
            auto behind = [&](uint32_t row) {  // the first token, in rows of Q
                const uint32_t of = token_of(row);
                return (of - token) * p.Nq + (row - of * G);
            };
#pragma unroll
            for (int j = 0; j < kCopies; ++j) {
                const uint32_t in = wave * 16 + j * kRowsPer + lane / CH, chunk = lane % CH ^ swz(in);
                const uint32_t x = (behind(first + in) * D + chunk * 8) * 2;
                at[j] = chunk * 8 < D ? x : (uint32_t)kOutOfRange;
            }
            lseAt = behind(first + lane) * 4;
        };
        lay(row0);
        struct Rows {
            __amdgpu_buffer_rsrc_t q, lse;
            uint32_t place;
        };
        auto rows_of = [&](uint32_t i) {
            const uint32_t first = row0 + i * kStageRows;
            if (!alike) lay(first);
            const uint64_t at0 = ((uint64_t)(uint32_t)c.req.start + first_lane(token_of(first))) * p.Nq + c.hkv * G, all = (uint64_t)p.T * p.Nq;
            const uint64_t left = at0 < all ? all - at0 : 0;
            Rows r;
            r.q = __builtin_amdgcn_make_buffer_rsrc(const_cast<S *>(Q + (at0 < all ? at0 : 0) * D), 0, (int)min(left * D * 2, (uint64_t)0x7fffffff),
                                                    0x00020000);
            r.lse = __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(lse + (at0 < all ? at0 : 0)), 0, (int)min(left * 4, (uint64_t)0x7fffffff),
                                                      0x00020000);
            r.place = i % kPlaces;
            return r;
        };
        constexpr int kParts = kCopies + 1;
        auto copy_part = [&](const Rows &r, int j) {
            if (j < kCopies)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(r.q, (lds_void *)(smem + r.place * kStageBytes + (wave * 16 + j * kRowsPer) * HD * 2), 16,
                                                         (int)at[j], 0, 0, 0);
            else
                __builtin_amdgcn_raw_ptr_buffer_load_lds(r.lse, (lds_void *)(smem + kLse + (r.place * 4 + wave) * 256), 4, (int)lseAt, 0, 0, 0);
        };
        auto copy = [&](uint32_t i) {
            const Rows r = rows_of(i);
#pragma unroll
            for (int j = 0; j < kParts; ++j) copy_part(r, j);
        };
#pragma unroll
        for (uint32_t i = 0; i + 1 < kPlaces; ++i) copy(i);
        u32x4 kf[2][KS];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const uint32_t key = key0 + t * 32 + c32, page = page_of(key);
            const S *row = K + (((uint64_t)(page < p.pages ? page : 0u) * p.Nkv + c.hkv) * p.pageSize + key % p.pageSize) * D;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const uint32_t d = s * 16 + h * 8;
                kf[t][s] = (page < p.pages && d < D ? *reinterpret_cast<const u32x4 *>(row + d) : u32x4{0u, 0u, 0u, 0u}) ^ flip;
            }
        }
        f32x16 sum[2], st[2][2];  // scores of a step's first and second 32 rows, 32 keys each
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                sum[t][e] = 0.0f;
                st[1][t][e] = -INFINITY;  // (none before the first)
            }
        const uint32_t qAt = c32 * (HD * 2) + (h ^ swz(c32)) * 16;
        float ofs[2] = {0.0f, 0.0f};
        // What scores e and e + 16 j of rows rt give their keys.
        auto weigh = [&](int rt, int at) {
            const int t = at / 16, e = at % 16;
            float v = sum[t][e] + __builtin_amdgcn_exp2f(fmaf(st[rt][t][e], c2, -ofs[rt]));
            asm volatile("" : "+v"(v));  // here, beside the product
            sum[t][e] = v;
        };
        // The scores of 32 rows, with the weights of the 32 before beside the products.
        auto score = [&](uint32_t x, int rt, const Rows *ahead) {
            // Beside product i stand the sum of its scores - 2, the exponential of its scores - 1 and the exponent of its own: in a row of
            // their own each would wait for the one before it.
            constexpr int kEach = 32 / (KS * 2), kAhead = 4;
            float x0[kEach], x1[kEach];
            auto beside = [&](int i) {
#pragma unroll
                for (int j = 0; j < kEach; ++j) {
                    if (i >= 2) {
                        const int at = (i - 2) * kEach + j;
                        float to = sum[at / 16][at % 16] + x1[j];
                        asm volatile("" : "+v"(to));
                        sum[at / 16][at % 16] = to;
                    }
                    if (i >= 1 && i <= 2 * KS) {
                        x1[j] = __builtin_amdgcn_exp2f(x0[j]);
                        asm volatile("" : "+v"(x1[j]));
                    }
                    if (i < 2 * KS) {
                        x0[j] = fmaf(st[1 - rt][(i * kEach + j) / 16][(i * kEach + j) % 16], c2, -ofs[1 - rt]);
                        asm volatile("" : "+v"(x0[j]));
                    }
                }
            };
            u32x4 q[kAhead];
            auto read = [&](int i) {
                return *reinterpret_cast<const u32x4 *>(smem + ((x ^ (i & 7) * 32u) + (i >> 3) * 256u + rt * (32 * HD * 2)));
            };
#pragma unroll
            for (int i = 0; i < kAhead; ++i) q[i] = read(i);
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 16; ++e) st[rt][t][e] = 0.0f;
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < KS; ++i) {
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    st[rt][t] = pk::Mma<T>::run(kf[t][i], q[i % kAhead], st[rt][t]);
                    if (t == 1 && i + kAhead < KS) q[i % kAhead] = read(i + kAhead);
                    beside(i * 2 + t);
                    // the copies of a later step between the products: a CU takes 16 cycles for each, so four waves' would wait in a row
                    constexpr int kEvery = 2 * KS / kParts;
                    if (ahead && (i * 2 + t) % kEvery == 0 && (i * 2 + t) / kEvery < kParts) copy_part(*ahead, (i * 2 + t) / kEvery);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            beside(2 * KS);
            beside(2 * KS + 1);
        };
        // Hides what rows do not see, and rows that give nothing.
        auto mask = [&](int rt, uint32_t first) {
            const int posLo = c.req.pos0 + (int)token_of(first);
            if (__ballot(ofs[rt] != ofs[rt])) {  // a NaN is its row's scores, so that keys which the row does not see can be told from them
                const bool nan = ofs[rt] != ofs[rt];
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int e = 0; e < 16; ++e) st[rt][t][e] = nan ? __builtin_nanf("") : st[rt][t][e];
                ofs[rt] = nan ? 0.0f : ofs[rt];
            }
            if (__ballot(ofs[rt] == INFINITY) == 0 && (p.maskKind == 2u || (int)key0 + 63 <= posLo)) return;
            const int pos = ofs[rt] == INFINITY ? -1 : p.maskKind == 2u ? 0x7fffffff : c.req.pos0 + (int)token_of(min(first + c32, rows - 1));
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int key = (int)(key0 + t * 32 + (e >> 2) * 8 + h * 4 + (e & 3));
                    st[rt][t][e] = key <= pos ? st[rt][t][e] : -INFINITY;
                }
        };
        int last = 1;  // the rows whose weights are still to be taken
        for (uint32_t i = 0; i < n; ++i) {
            // this step's rows are in LDS, and every wave has read those that are copied over
            wait_vmcnt<(int)(kPlaces - 2) * (kCopies + 1)>();
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            if (key0 >= keys) {
                copy(i + kPlaces - 1);
                continue;
            }
            const Rows later = rows_of(i + kPlaces - 1);
            const uint32_t first = row0 + i * kStageRows, place = i % kPlaces;
            uint32_t x = qAt + place * kStageBytes;
            asm volatile("" : "+v"(x));
            // in base 2; infinity: the row gives nothing
            auto logarithm = [&](int rt) {
                const float v = *reinterpret_cast<const float *>(smem + kLse + (place * 4 + wave) * 256 + (rt * 32 + c32) * 4);
                return v == -INFINITY || first + rt * 32 + c32 >= rows ? INFINITY : v * kLog2e;
            };
            ofs[0] = logarithm(0);
            score(x, 0, &later);
            mask(0, first);
            last = 0;
            if (first + 32 >= rows) break;
            ofs[1] = logarithm(1);
            score(x, 1, nullptr);
            mask(1, first + 32);
            last = 1;
        }
        if (last) {
#pragma unroll
            for (int e = 0; e < 32; ++e) weigh(1, e);
        } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) weigh(0, e);
        }
        // every wave has read its last rows before the next piece's copies
        wait_vmcnt<0>();
        __builtin_amdgcn_s_waitcnt(0xC07F);
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const bool whole = c.lo == 0 && c.hi == c.steps.n;
        float *to = weights + ((uint64_t)c.request * p.Nkv + c.hkv) * ((uint64_t)p.columns * p.pageSize);
        float *slot = partial + (2 * (uint64_t)blockIdx.x + (c.lo == 0)) * kKeys + wave * 64;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            float mine = 0.0f;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float v = pk::half32_sum(sum[t][e]);
                if (c32 == (uint32_t)e) mine = v;
            }
            if (c32 < 16) {
                const uint32_t in = t * 32 + (c32 >> 2) * 8 + h * 4 + (c32 & 3);
                if (!whole) slot[in] = mine;
                else if (page_of(key0 + in) < p.pages) to[key0 + in] += mine;
            }
        }
    }
}

}  // namespace

// The partial sums of the units that several blocks shared, in their order. Bound by its launch and two rounds of loads: all that
// hang on the unit are asked for before any is looked at.
POPCORN_KERNEL void __launch_bounds__(256)
    attention_weights_join(const int32_t *tables, const float *partial, const WeightsBatch::Left *left, float *weights,
                           PagedAttentionConstants p) {
    const WeightsBatch::Left c = left[blockIdx.x];
    if (c.pieces == 0) return;
    const uint32_t key = c.key0 + threadIdx.x, in = min(key, c.keys - 1);  // (a unit has keys)
    const uint32_t page = (uint32_t)tables[(uint64_t)c.request * p.columns + in / p.pageSize];
    float *to = weights + ((uint64_t)c.request * p.Nkv + c.hkv) * ((uint64_t)p.columns * p.pageSize) + in;
    const float old = *to;
    auto piece = [&](uint32_t i) { return partial[(2 * ((uint64_t)blockIdx.x + i) + (i == 0)) * kKeys + threadIdx.x]; };
    float x = piece(0), next = piece(1);  // (shared by two at least)
    for (uint32_t i = 1; i < c.pieces; ++i) {
        const float v = next;
        if (i + 1 < c.pieces) next = piece(i + 1);
        x += v;
    }
    if (key < c.keys && page < p.pages) *to = old + x;
}

POPCORN_KERNEL void __launch_bounds__(1024)
    attention_weights_tiles(const int32_t *starts, const int32_t *keyLens, pk::PagedTile *plan, PagedAttentionConstants p, PagedWorkConstants w,
                            AttentionWeightsConstants a) {
    __shared__ PlanSpace<1024, u64, pk::PagedRequest> space;
    u64 steps;
    uint32_t tiles;
    const WeightsBatch batch{starts, keyLens, nullptr, a};
    lay_tiles<1024, u64>(batch, space, p, w, steps, tiles, [&](uint32_t at, u64 before, uint32_t request, uint32_t tile, const auto &) {
        plan[1 + at] = pk::PagedTile{before, request, tile};
    });
    if (threadIdx.x == 0) plan[0] = pk::PagedTile{steps, tiles, 0};
}

namespace {

// Any head dim and alignment: 16 lanes take a key at a time, for every row in turn.
template <typename T>
__device__ void weights_plain(const typename T::storage *__restrict__ Q, const typename T::storage *__restrict__ K,
                              const int32_t *__restrict__ tables, const int32_t *__restrict__ starts, const int32_t *__restrict__ keyLens,
                              const float *__restrict__ lse, float *__restrict__ weights, const PagedAttentionConstants &p,
                              const AttentionWeightsConstants &w) {
    const uint32_t r = blockIdx.x / p.Nkv, hkv = blockIdx.x % p.Nkv, G = p.Nq / p.Nkv, t = threadIdx.x % 16;
    const float c2 = p.scale * kLog2e;
    const pk::PagedRequest q = weights_request(starts, keyLens, r, p, w);
    const uint32_t rows = (uint32_t)q.n * G;
    if (rows == 0) return;
    float *to = weights + ((uint64_t)r * p.Nkv + hkv) * ((uint64_t)p.columns * p.pageSize);
    for (uint64_t k = blockIdx.y * 16 + threadIdx.x / 16; k < (uint32_t)q.keys; k += (uint64_t)gridDim.y * 16) {
        const uint32_t key = (uint32_t)k, page = (uint32_t)tables[(uint64_t)r * p.columns + key / p.pageSize];
        if (page >= p.pages) continue;
        const typename T::storage *kr = K + (((uint64_t)page * p.Nkv + hkv) * p.pageSize + key % p.pageSize) * p.Hd;
        float sum = 0.0f;
        for (uint32_t row = 0; row < rows; ++row) {
            if (p.maskKind != 2u && (int)key > q.pos0 + (int)(row / G)) continue;
            const uint64_t at = ((uint64_t)(uint32_t)q.start + row / G) * p.Nq + hkv * G + row % G;
            const float of = lse[at] * kLog2e;
            if (of == -INFINITY) continue;
            float s = 0.0f;
            for (uint32_t d = t; d < p.Hd; d += 16) s = fmaf(T::load(Q[at * p.Hd + d]), T::load(kr[d]), s);
            sum += __builtin_amdgcn_exp2f(fmaf(pk::row16_sum(s), c2, -of));
        }
        if (t == 0) to[key] += sum;
    }
}

}  // namespace

#define WEIGHTS_FEW(t, T, HD, KM, PER_CU)                                                                                     \
    POPCORN_KERNEL void __launch_bounds__(256, PER_CU)                                                                        \
        attention_weights_few_##t##_d##HD(const T::storage *q, const T::storage *k, const int32_t *tables, const int32_t *starts, \
                                          const int32_t *keyLens, const float *lse, const uint64_t *plan, float *weights,     \
                                          PagedAttentionConstants p, AttentionWeightsConstants w) {                           \
        weights_few<T, HD, KM>(q, k, tables, starts, keyLens, lse, plan, weights, p, w);                                      \
    }
#define WEIGHTS_TILE(t, T, HD)                                                                                                \
    POPCORN_KERNEL void __launch_bounds__(256, HD > 128 ? 1 : 2)                                                              \
        attention_weights_tile_##t##_d##HD(const T::storage *q, const T::storage *k, const int32_t *tables, const int32_t *starts, \
                                           const int32_t *keyLens, const float *lse, const pk::PagedTile *plan, float *partial, \
                                           WeightsBatch::Left *left, float *weights, PagedAttentionConstants p,               \
                                           PagedWorkConstants w, AttentionWeightsConstants a) {                               \
        weights_tile<T, HD>(q, k, tables, starts, keyLens, lse, plan, partial, left, weights, p, w, a);                       \
    }
#define WEIGHTS_PLAIN(t, T)                                                                                                   \
    POPCORN_KERNEL void __launch_bounds__(256)                                                                                \
        attention_weights_plain_##t(const T::storage *q, const T::storage *k, const int32_t *tables, const int32_t *starts,   \
                                    const int32_t *keyLens, const float *lse, float *weights, PagedAttentionConstants p,      \
                                    AttentionWeightsConstants w) {                                                            \
        weights_plain<T>(q, k, tables, starts, keyLens, lse, weights, p, w);                                                  \
    }

using pk::BF16;
using pk::F16;
using pk::F32;

#define WEIGHTS_16(t, T)          \
    WEIGHTS_FEW(t, T, 64, 4, 4)   \
    WEIGHTS_FEW(t, T, 128, 4, 3)  \
    WEIGHTS_FEW(t, T, 256, 2, 2)  \
    WEIGHTS_FEW(t, T, 512, 1, 2)  \
    WEIGHTS_TILE(t, T, 64)        \
    WEIGHTS_TILE(t, T, 128)       \
    WEIGHTS_TILE(t, T, 256)       \
    WEIGHTS_PLAIN(t, T)
WEIGHTS_16(f16, F16)
WEIGHTS_16(bf16, BF16)
WEIGHTS_FEW(f32, F32, 64, 4, 3)
WEIGHTS_FEW(f32, F32, 128, 2, 2)
WEIGHTS_FEW(f32, F32, 256, 1, 2)
WEIGHTS_FEW(f32, F32, 512, 1, 1)
WEIGHTS_PLAIN(f32, F32)
