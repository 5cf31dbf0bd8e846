// The paged cache's bookkeeping: page_tables (tables, slots and positions of a
// step's new tokens from the requests' lengths) and paged_kv_write_* (the new
// tokens' K and V rows into their slots).
#include "scan.hpp"

namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kPer = 4;                  // requests per thread and pass
constexpr uint32_t kPass = kThreads * kPer;   // requests per pass

__device__ inline int32_t saturate(uint64_t v) { return v < 0x7fffffffu ? (int32_t)v : 0x7fffffff; }

__device__ inline uint32_t ceil_div(uint32_t a, uint32_t b) { return a / b + (a % b != 0); }

}  // namespace

// Tokens are numbered through the requests in order, so token t belongs to the
// request r with start[r] <= t < start[r + 1] (start: sums of new lengths), has
// position past[r] + t - start[r], and lies in table column position /
// pageSize. Columns from ceil(past / pageSize) on are new: the k-th new page
// of the whole step is free_pages[k], k counted by the sums of ceil((past +
// new) / pageSize) - ceil(past / pageSize). The token at a page's first row
// writes the table's entry.
//
// Every block sums all requests by itself (they are few beside the tokens'
// reads and writes, and it saves a launch and a round trip between blocks) and
// serves its share of the tokens; block 0 also writes what belongs to requests.
// Bound by its launch and one round of reads: 4.0 us for 256 requests of a token,
// 5.0 for 48 of 24000 tokens in all.
POPCORN_KERNEL void __launch_bounds__(256)
    page_tables(const int32_t *past, const int32_t *fresh, const int32_t *freePages, int32_t *tables, int32_t *queryStarts,
                int32_t *keyLens, int32_t *positions, int32_t *slots, int32_t *counts, PageTablesConstants p) {
    __shared__ int32_t sStart[kPass + 1], sPast[kPass];
    __shared__ uint64_t sTaken[kPass], sWave[2][kThreads / 64];
    const uint32_t tid = threadIdx.x, wave = tid >> 6;
    const uint32_t lo = (uint32_t)((uint64_t)p.T * blockIdx.x / gridDim.x);
    const uint32_t hi = (uint32_t)((uint64_t)p.T * (blockIdx.x + 1) / gridDim.x);
    uint64_t tokens = 0, taken = 0;  // of the passes before
    for (uint32_t base = 0; base < p.R; base += kPass) {
        if (blockIdx.x != 0 && tokens >= hi) return;  // this block's tokens are served
        uint32_t n[kPer], pages[kPer];
        int32_t at[kPer];
        uint64_t a = 0, b = 0;
#pragma unroll
        for (uint32_t j = 0; j < kPer; ++j) {
            const uint32_t r = base + tid * kPer + j;
            at[j] = r < p.R ? max(past[r], 0) : 0;
            n[j] = r < p.R ? (uint32_t)max(fresh[r], 0) : 0u;
            pages[j] = ceil_div((uint32_t)at[j] + n[j], p.pageSize) - ceil_div((uint32_t)at[j], p.pageSize);
            a += n[j];
            b += pages[j];
        }
        const uint64_t sa = pk::wave_scan(a), sb = pk::wave_scan(b);
        __syncthreads();  // the pass before has read the sums and the tables
        if ((tid & 63) == 63) {
            sWave[0][wave] = sa;
            sWave[1][wave] = sb;
        }
        __syncthreads();
        uint64_t ra = tokens + sa - a, rb = taken + sb - b;
#pragma unroll
        for (uint32_t w = 0; w < kThreads / 64; ++w) {
            const uint64_t x = sWave[0][w], y = sWave[1][w];
            if (w < wave) {
                ra += x;
                rb += y;
            }
            tokens += x;
            taken += y;
        }
#pragma unroll
        for (uint32_t j = 0; j < kPer; ++j) {
            const uint32_t r = base + tid * kPer + j;
            sStart[tid * kPer + j] = saturate(ra);
            sPast[tid * kPer + j] = at[j];
            sTaken[tid * kPer + j] = rb;
            if (blockIdx.x == 0 && r < p.R) {
                queryStarts[r] = min(saturate(ra), (int32_t)p.T);
                keyLens[r] = saturate((uint64_t)(uint32_t)at[j] + n[j]);
            }
            ra += n[j];
            rb += pages[j];
        }
        if (tid == 0) sStart[kPass] = saturate(tokens);
        __syncthreads();
        const uint32_t t0 = max(lo, (uint32_t)sStart[0]), t1 = min(hi, (uint32_t)sStart[kPass]);
        for (uint32_t t = t0 + tid; t < t1; t += kThreads) {
            // the last request of the pass that starts at or before t (empty ones start there too, before it)
            uint32_t i = 0;
#pragma unroll
            for (uint32_t d = kPass / 2; d; d >>= 1)
                if (i + d < kPass && (uint32_t)sStart[i + d] <= t) i += d;
            const uint32_t r = base + i, first = (uint32_t)sPast[i];
            const uint32_t pos = first + (t - (uint32_t)sStart[i]);
            const uint32_t column = pos / p.pageSize, held = ceil_div(first, p.pageSize), row = pos - column * p.pageSize;
            int32_t page = -1;
            if (column < p.columns) {
                int32_t *entry = tables + (uint64_t)r * p.columns + column;
                if (column < held) {
                    page = *entry;
                } else {
                    const uint64_t k = sTaken[i] + (column - held);
                    if (k < p.F) page = freePages[k];
                    if (row == 0) *entry = page < 0 ? -1 : page;
                }
            }
            const uint64_t slot = (uint64_t)(uint32_t)max(page, 0) * p.pageSize + row;
            positions[t] = saturate(pos);
            slots[t] = page < 0 || slot > 0x7fffffffu ? -1 : (int32_t)slot;
        }
    }
    for (uint32_t t = max((uint64_t)lo, min(tokens, (uint64_t)hi)) + tid; t < hi; t += kThreads) {
        positions[t] = 0;
        slots[t] = -1;
    }
    if (blockIdx.x == 0 && tid == 0) {
        queryStarts[p.R] = min(saturate(tokens), (int32_t)p.T);
        counts[0] = saturate(tokens);
        counts[1] = saturate(taken);
    }
}

namespace {

// One run of up to kRun elements per thread and step (16 bytes of the source), as in
// kv_cache_write; blocks take consecutive stretches of kStretch runs, and only a
// stretch's start is divided in 64 bits. Bound by the copy: 8000 tokens of 4 heads of
// 256 in bf16, 66 MB read and written, in 13.5 us (4.9 TB/s); 64 tokens in 3.
constexpr uint32_t kStretch = 1024;

template <typename S, typename C>
__device__ void paged_write(const typename S::storage *__restrict__ k, const typename S::storage *__restrict__ v,
                            const int32_t *__restrict__ slots, typename C::storage *__restrict__ kc,
                            typename C::storage *__restrict__ vc, const PagedKVWriteConstants &p) {
    constexpr uint32_t kRun = 16 / sizeof(typename S::storage);
    const uint32_t runsPerRow = (p.Hd + kRun - 1) / kRun, runsPerToken = runsPerRow * p.Nkv;
    const uint64_t total = (uint64_t)p.T * runsPerToken;
    const uint64_t begin = (uint64_t)blockIdx.x * kStretch;
    const uint64_t t0 = begin / runsPerToken;
    const uint32_t r0 = (uint32_t)(begin - t0 * runsPerToken);
    const typename S::storage *src = blockIdx.y ? v : k;
    typename C::storage *dst = blockIdx.y ? vc : kc;
    const bool vec = p.Hd % kRun == 0 && reinterpret_cast<uintptr_t>(src) % 16 == 0 &&
                     reinterpret_cast<uintptr_t>(dst) % (kRun * sizeof(typename C::storage)) == 0;
#pragma unroll
    for (uint32_t i = 0; i < kStretch; i += kThreads) {
        if (begin + i + threadIdx.x >= total) return;
        const uint32_t at = r0 + i + threadIdx.x, dt = at / runsPerToken, in = at - dt * runsPerToken;
        const uint32_t h = in / runsPerRow, d0 = (in - h * runsPerRow) * kRun;
        const uint64_t t = t0 + dt;
        const int32_t slot = slots[t];
        const uint32_t page = (uint32_t)slot / p.pageSize, row = (uint32_t)slot - page * p.pageSize;
        if (slot < 0 || page >= p.pages) continue;
        const typename S::storage *s = src + (t * p.Nkv + h) * p.Hd + d0;
        typename C::storage *c = dst + (((uint64_t)page * p.Nkv + h) * p.pageSize + row) * p.Hd + d0;
        if (!vec) {
            for (uint32_t d = 0; d < kRun && d0 + d < p.Hd; ++d) c[d] = C::store(S::load(s[d]));
        } else if constexpr (S::kTag == C::kTag) {
            *reinterpret_cast<pk::u32x4 *>(c) = __builtin_nontemporal_load(reinterpret_cast<const pk::u32x4 *>(s));
        } else {
            pk::Vec<S> x;
            x.load(s);
            typename C::storage out[kRun];
#pragma unroll
            for (uint32_t d = 0; d < kRun; ++d) out[d] = C::store(x.get(d));
            *reinterpret_cast<pk::u32x2 *>(c) = *reinterpret_cast<const pk::u32x2 *>(out);
        }
    }
}

}  // namespace

#define PAGED_WRITE(name, S, C)                                                                          \
    POPCORN_KERNEL void __launch_bounds__(256) name(const S::storage *k, const S::storage *v, const int32_t *slots, \
                                                    C::storage *kc, C::storage *vc, PagedKVWriteConstants p) {      \
        paged_write<S, C>(k, v, slots, kc, vc, p);                                                       \
    }

using pk::BF16;
using pk::F16;
using pk::F32;

PAGED_WRITE(paged_kv_write_f32, F32, F32)
PAGED_WRITE(paged_kv_write_f16, F16, F16)
PAGED_WRITE(paged_kv_write_bf16, BF16, BF16)
PAGED_WRITE(paged_kv_write_f32_to_bf16, F32, BF16)
