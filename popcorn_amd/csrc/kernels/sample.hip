// One token a row of logits, drawn with a given uniform random number.
//
// Tokens rank by logit, ties by index; a token's weight is the whole number
// rint(2^40 exp((logit - highest) / temperature)), computed in 64 bits, so
// sums of weights are exact whatever their order, and a vocabulary of up to
// 2^22 tokens sums below 2^62. Each option keeps a prefix of the ranking, so
// what is kept is one cut (a logit and an index) and a least weight.
//
// Sorting the row is not needed to find the cut. Four launches, a row cut into slices:
//  1. sample_top: each slice's highest logit;
//  2. sample_hist (top-k, top-p): number and weight of the tokens in 2048
//     bins of the distance from the highest;
//  3. sample_gather: the bins in which the cuts must fall, from the bins'
//     running sums; their tokens (the candidates, a few hundred of a large
//     vocabulary) go to a list, the weight before them is summed by slice;
//  4. sample_finish: sorts the candidates, finds the cuts among them, the
//     slice where the running weight passes the draw, and the token in it.
// A row of up to 4096 logits is one launch (sample_small): all are candidates.
// More candidates than the list holds (thousands of equal logits at the cut)
// are counted digit by digit of their logits instead (cut_by_digits).
#include "common.hpp"

namespace {

constexpr uint32_t kSlice = 256;                        // threads of a slice's block
constexpr uint32_t kRow = 1024, kRowWaves = kRow / 64;  // threads of a row's block
constexpr uint32_t E = 8;                               // consecutive logits per thread and step
constexpr double kOne = 1099511627776.0;                // 2^40
constexpr uint32_t kBins = SAMPLE_BINS, kList = SAMPLE_CANDIDATES;
constexpr uint32_t kPerThread = kBins / kSlice;
typedef unsigned long long u64;

// A logit's place in the ranking: greater for greater logits, 0 for NaN, equal
// for both zeros.
__device__ inline uint32_t rank_key(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    if (v != v) return 0u;
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ inline float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// Coefficients ln(2)^k / k! of 2^f: for |f| <= 1/2 the terms left out are below 2^-47 of it.
struct Exp2Terms {
    double c[12];
    constexpr Exp2Terms() : c() {
        c[0] = 1.0;
        for (int k = 1; k < 12; ++k) c[k] = c[k - 1] * 0.69314718055994530942 / k;
    }
};

// One row's options, and its highest logit.
struct Row {
    float top, bins;  // bins per unit of distance
    double rate;      // log2(e) / temperature
    u64 least;
    float p;
    uint32_t k;
    bool live, useK, useP;

    __device__ inline u64 weight(float v) const {
        constexpr Exp2Terms terms;
        if (!(v > -INFINITY)) return 0;
        const double t = ((double)v - (double)top) * rate;
        const double n = __builtin_rint(t), f = t - n;
        double s = terms.c[11];
#pragma unroll
        for (int k = 10; k >= 0; --k) s = __builtin_fma(s, f, terms.c[k]);
        // adding 2^52 rounds to a whole number and leaves it in the low bits
        const double w = __builtin_ldexp(s, (int)n + 40) + 4503599627370496.0;
        const u64 u = t > -42.0 ? __builtin_bit_cast(u64, w) & 0xfffffffffffffull : 0;  // (a NaN is 0)
        return v == top ? (u64)1 << 40 : u;
    }
    // Grows, if anything, from a logit to the next in the ranking.
    __device__ inline uint32_t bin(float v) const {
        return v == top ? 0u : (uint32_t)fminf((top - v) * bins, (float)(kBins - 1));
    }
};

struct Options {
    const float *uniforms, *temperature;
    const int32_t *topK;
    const float *topP, *minP;
};

__device__ inline Row row_of(const Options &o, uint32_t r, uint32_t topKey, const SampleConstants &c) {
    Row w;
    w.top = key_value(topKey);
    w.live = topKey != 0 && w.top > -INFINITY;
    const float t = c.hasTemperature ? o.temperature[r] : 1.0f;
    const int32_t k = c.hasTopK ? o.topK[r] : 0;
    const float p = c.hasTopP ? o.topP[r] : 1.0f, least = c.hasMinP ? o.minP[r] : 0.0f;
    const bool greedy = !(t > 0.0f);
    w.rate = 1.4426950408889634074 / (greedy ? 1.0 : (double)t);
    w.bins = 72.0f / (greedy ? 1.0f : t);  // weights end at a distance of 28.5 temperatures
    w.k = greedy ? 1u : k > 0 ? (uint32_t)k : 0u;
    w.useK = w.k > 0 && w.k < c.vocab;
    w.useP = p < 1.0f;  // (not where it is NaN)
    w.p = fmaxf(p, 0.0f);
    w.least = least > 0.0f ? (u64)__builtin_ceil((double)fminf(least, 1.0f) * kOne) : 0;
    return w;
}

// floor(m z / 2^31), and whether a part is left over, for m <= 2^31 and z < 2^62.
__device__ inline u64 share(uint32_t m, u64 z, bool &more) {
    const u64 low = (z & 0x7fffffffu) * m;
    more = (low & 0x7fffffffu) != 0;
    return (z >> 31) * m + (low >> 31);
}
// The weight at which top-p stops: kept are tokens before which less lies.
__device__ inline u64 limit_of(float p, u64 z) {
    bool more;
    const u64 s = share((uint32_t)((double)p * 2147483648.0), z, more);
    return max(s + more, (u64)1);
}

__device__ inline uint32_t wave_max_u32(uint32_t v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, d));
    return v;
}
__device__ inline u64 wave_sum64(u64 v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

// Inclusive sums over the block of NT threads, and the total.
template <uint32_t NT, typename U>
__device__ inline U block_scan(U v, U *sums, U &total) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) {
        const U x = __shfl_up(v, d);
        if (lane >= d) v += x;
    }
    __syncthreads();
    if (lane == 63) sums[wave] = v;
    __syncthreads();
    U before = 0;
    total = 0;
#pragma unroll
    for (uint32_t w = 0; w < NT / 64; ++w) {
        if (w == wave) before = total;
        total += sums[w];
    }
    return before + v;
}

// f(index, logit) for this thread's logits of [lo, hi), eight in a row at a time.
template <typename T, uint32_t NT, typename F>
__device__ inline void each_logit(const typename T::storage *__restrict__ x, uint32_t lo, uint32_t hi, F &&f) {
    struct Eight {
        typename T::storage v[E];
    };
    for (uint32_t i = lo + threadIdx.x * E; i < hi; i += NT * E) {
        if (i + E <= hi) {
            Eight e;
            __builtin_memcpy(&e, x + i, sizeof(e));
#pragma unroll
            for (uint32_t j = 0; j < E; ++j) f(i + j, T::load(e.v[j]));
        } else {
            for (uint32_t j = i; j < hi; ++j) f(j, T::load(x[j]));
        }
    }
}

template <typename T>
__device__ void sample_top(const typename T::storage *__restrict__ logits, SampleRow *__restrict__ rows, const SampleConstants &c) {
    __shared__ uint32_t sTop[kSlice / 64];
    const uint32_t r = blockIdx.x / c.slices, slice = blockIdx.x % c.slices;
    SampleRow &row = rows[r];
    const uint32_t lo = slice * c.sliceLen, hi = min(lo + c.sliceLen, c.vocab);
    uint32_t best = 0;
    each_logit<T, kSlice>(logits + (uint64_t)r * c.vocab, lo, hi, [&](uint32_t, float v) { best = max(best, rank_key(v)); });
    best = wave_max_u32(best);
    if ((threadIdx.x & 63) == 0) sTop[threadIdx.x >> 6] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (uint32_t w = 1; w < kSlice / 64; ++w) best = max(best, sTop[w]);
        row.sliceTop[slice] = best;
        if (slice == 0) row.candidates = 0;
    }
    // the next launch adds to these
    for (uint32_t b = slice * kSlice + threadIdx.x; b < kBins; b += c.slices * kSlice) {
        row.weight[b] = 0;
        row.count[b] = 0;
    }
}

// The row's highest logit, of up to 256 slices.
template <uint32_t NT>
__device__ inline uint32_t top_of(const SampleRow &row, uint32_t slices, uint32_t *shared) {
    const uint32_t best = wave_max_u32(threadIdx.x < slices ? row.sliceTop[threadIdx.x] : 0u);
    if ((threadIdx.x & 63) == 0 && threadIdx.x < 256) shared[threadIdx.x >> 6] = best;
    __syncthreads();
    return max(max(shared[0], shared[1]), max(shared[2], shared[3]));
}

template <typename T>
__device__ void sample_hist(const typename T::storage *__restrict__ logits, const Options &o, SampleRow *__restrict__ rows,
                            const SampleConstants &c) {
    __shared__ u64 sWeight[kBins];
    __shared__ uint32_t sCount[kBins], sTop[4];
    const uint32_t r = blockIdx.x / c.histBlocks, part = blockIdx.x % c.histBlocks;
    SampleRow &row = rows[r];
    const Row w = row_of(o, r, top_of<kSlice>(row, c.slices, sTop), c);
    if (!w.live || !(w.useK || w.useP)) return;
    for (uint32_t b = threadIdx.x; b < kBins; b += kSlice) {
        sWeight[b] = 0;
        sCount[b] = 0;
    }
    __syncthreads();
    const uint32_t per = (c.slices + c.histBlocks - 1) / c.histBlocks * c.sliceLen;
    const uint32_t lo = min(part * per, c.vocab), hi = min(lo + per, c.vocab);
    each_logit<T, kSlice>(logits + (uint64_t)r * c.vocab, lo, hi, [&](uint32_t, float v) {
        const u64 u = w.weight(v);
        if (u == 0) return;
        const uint32_t b = w.bin(v);
        if (w.useP) atomicAdd(&sWeight[b], u);
        if (w.useK) atomicAdd(&sCount[b], 1u);
    });
    __syncthreads();
    for (uint32_t b = threadIdx.x; b < kBins; b += kSlice) {
        if (sWeight[b]) atomicAdd(reinterpret_cast<u64 *>(&row.weight[b]), sWeight[b]);
        if (sCount[b]) atomicAdd(&row.count[b], sCount[b]);
    }
}

template <typename T>
__device__ void sample_gather(const typename T::storage *__restrict__ logits, const Options &o, SampleRow *__restrict__ rows,
                              const SampleConstants &c) {
    __shared__ u64 sSums[kSlice / 64], sAbove[2];
    __shared__ uint32_t sCounts[kSlice / 64], sTop[4], sBin[3], sNeed;
    const uint32_t r = blockIdx.x / c.slices, slice = blockIdx.x % c.slices;
    SampleRow &row = rows[r];
    const uint32_t tid = threadIdx.x, lane = tid & 63;
    const Row w = row_of(o, r, top_of<kSlice>(row, c.slices, sTop), c);
    if (!w.live) return;
    // bins before `first` are kept; candidates are the bins first .. lastP and binK
    uint32_t first = kBins, lastP = 0, binK = kBins;
    if (w.useK || w.useP) {
        u64 bw[kPerThread], mine = 0, total;
        uint32_t bc[kPerThread], here = 0, counted;
#pragma unroll
        for (uint32_t j = 0; j < kPerThread; ++j) {
            bw[j] = row.weight[tid * kPerThread + j];
            bc[j] = row.count[tid * kPerThread + j];
            mine += bw[j];
            here += bc[j];
        }
        const u64 wend = block_scan<kSlice>(mine, sSums, total);
        const uint32_t cend = block_scan<kSlice>(here, sCounts, counted);
        if (tid == 0) {
            sBin[0] = sBin[1] = sBin[2] = kBins;
            sAbove[0] = sAbove[1] = 0;
            sNeed = 0;
        }
        __syncthreads();
        // calls at(bin, weight before it) for the one bin of this thread's that `in(before, with)` names
        auto find = [&](auto &&in, auto &&at) {
            u64 before = wend - mine;
            uint32_t cb = cend - here;
#pragma unroll
            for (uint32_t j = 0; j < kPerThread; ++j) {
                if (in(before, before + bw[j], cb, cb + bc[j])) at(tid * kPerThread + j, before, cb);
                before += bw[j];
                cb += bc[j];
            }
        };
        u64 zLo = total, zHi = total;
        if (w.useK) {
            find([&](u64, u64, uint32_t a, uint32_t b) { return a < w.k && w.k <= b; },
                 [&](uint32_t b, u64 before, uint32_t cb) {
                     sBin[0] = b;
                     sAbove[0] = before;
                     sNeed = w.k - cb;
                 });
            __syncthreads();
            binK = sBin[0];
            if (binK < kBins) {
                zLo = sAbove[0];
                zHi = zLo + row.weight[binK];
            }
        }
        if (w.useP) {
            // top-p's share is of a weight between zLo and zHi
            const u64 lo = limit_of(w.p, zLo), hi = limit_of(w.p, zHi);
            find([&](u64 a, u64 b, uint32_t, uint32_t) { return a < lo && lo <= b; },
                 [&](uint32_t b, u64 before, uint32_t) {
                     sBin[1] = b;
                     sAbove[1] = before;
                 });
            find([&](u64 a, u64 b, uint32_t, uint32_t) { return a < hi && hi <= b; }, [&](uint32_t b, u64, uint32_t) { sBin[2] = b; });
            __syncthreads();
            first = sBin[1];
            lastP = sBin[2];
        } else {
            first = lastP = binK;
        }
        if (slice == 0 && tid == 0) {
            row.binK = binK;
            row.needK = sNeed;
            row.aboveK = sAbove[0];
            row.aboveP = sAbove[1];
            row.total = total;
            row.lastP = lastP;
        }
    }
    const uint32_t lo = slice * c.sliceLen, hi = min(lo + c.sliceLen, c.vocab);
    u64 sum = 0;
    each_logit<T, kSlice>(logits + (uint64_t)r * c.vocab, lo, hi, [&](uint32_t i, float v) {
        const u64 u = w.weight(v);
        if (u == 0) return;
        const uint32_t b = first < kBins ? w.bin(v) : 0u;
        if (b < first) {
            sum += u >= w.least ? u : 0;
        } else if (b <= lastP || b == binK) {
            const uint32_t at = atomicAdd(&row.candidates, 1u);
            if (at < kList) row.candidate[at] = (u64)rank_key(v) << 32 | (uint32_t)~i;
        }
    });
    sum = wave_sum64(sum);
    __syncthreads();
    if (lane == 0) sSums[tid >> 6] = sum;
    __syncthreads();
    if (tid == 0) row.sliceWeight[slice] = sSums[0] + sSums[1] + sSums[2] + sSums[3];
}

struct RowSpace {
    u64 list[kList];
    u64 sums[kRowWaves], slice[SAMPLE_MAX_SLICES], pick;
    uint32_t counts[kRowWaves], hist[256], bin;
    u64 weights[256];
};

// Sorts list[0, n), n a power of two, from the greatest.
__device__ inline void sort_list(u64 *list, uint32_t n) {
    for (uint32_t size = 2; size <= n; size <<= 1)
        for (uint32_t d = size >> 1; d; d >>= 1) {
            __syncthreads();
            for (uint32_t t = threadIdx.x; t < n / 2; t += kRow) {
                const uint32_t i = 2 * t - (t & (d - 1)), j = i + d;
                const u64 a = list[i], b = list[j];
                if ((a < b) == ((i & size) == 0)) {
                    list[i] = b;
                    list[j] = a;
                }
            }
        }
    __syncthreads();
}

// The last token that top-k and top-p keep, of n candidates in the list (in any order): rank key << 32 | ~index.
__device__ inline u64 cut_in_list(RowSpace &s, const Row &w, uint32_t n, uint32_t binK, uint32_t needK, uint32_t lastP, u64 aboveK,
                                  u64 aboveP, u64 total) {
    const uint32_t tid = threadIdx.x;
    uint32_t n2 = 64;
    while (n2 < n) n2 <<= 1;
    for (uint32_t i = n + tid; i < n2; i += kRow) s.list[i] = 0;
    sort_list(s.list, n2);
    constexpr uint32_t P = kList / kRow;  // a thread's candidates, in a row
    const uint32_t per = (n2 + kRow - 1) / kRow;
    u64 u[P], mine = 0, all;
    uint32_t b[P], before = 0, beforeK;
#pragma unroll
    for (uint32_t j = 0; j < P; ++j) {
        const uint32_t i = tid * per + j;
        const bool in = j < per && i < n;
        const float v = in ? key_value((uint32_t)(s.list[i] >> 32)) : 0.0f;
        u[j] = in ? w.weight(v) : 0;
        b[j] = in ? w.bin(v) : kBins;
        before += in && b[j] < binK;
    }
    uint32_t kept = n;
    if (binK < kBins) {
        (void)block_scan<kRow>(before, s.counts, beforeK);
        kept = min(n, beforeK + needK);
        u64 part = 0;
#pragma unroll
        for (uint32_t j = 0; j < P; ++j) {
            const uint32_t i = tid * per + j;
            if (j < per && i >= beforeK && i < kept) part += u[j];
            if (i >= kept) u[j] = 0;
        }
        (void)block_scan<kRow>(part, s.sums, total);
        total += aboveK;
    }
    if (w.useP) {
        const u64 limit = limit_of(w.p, total);
#pragma unroll
        for (uint32_t j = 0; j < P; ++j) mine += u[j];
        u64 run = aboveP + block_scan<kRow>(mine, s.sums, all) - mine;
        uint32_t keep = 0, sum;
#pragma unroll
        for (uint32_t j = 0; j < P; ++j) {
            const uint32_t i = tid * per + j;
            keep += j < per && i < kept && b[j] <= lastP && run < limit;
            run += u[j];
        }
        (void)block_scan<kRow>(keep, s.counts, sum);
        kept = sum;
    }
    __syncthreads();
    return kept ? s.list[kept - 1] : 0;
}

// The same cut for any number of candidates: the running measure over the
// ranking, 8 bits of the rank key at a time.
template <typename T>
__device__ u64 cut_by_digits(RowSpace &s, const typename T::storage *__restrict__ x, const Row &w, uint32_t n) {
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    u64 cut = 0;
    auto rank = [](float v, uint32_t i) { return (u64)rank_key(v) << 32 | (uint32_t)~i; };
    // Moves the cut to the token at which the running measure reaches `want`
    // (at least 1, at most the measure of what is kept).
    auto move = [&](u64 want, auto &&measure) {
        uint32_t prefix = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) s.weights[tid] = 0;
            __syncthreads();
            each_logit<T, kRow>(x, 0, n, [&](uint32_t i, float v) {
                const uint32_t key = rank_key(v);
                if (shift < 24 && (key >> (shift + 8)) != prefix) return;
                if (rank(v, i) >= cut) atomicAdd(&s.weights[(key >> shift) & 255u], measure(v));
            });
            __syncthreads();
            // thread t takes digit 255 - t
            u64 all;
            const u64 mine = tid < 256 ? s.weights[255 - tid] : 0, run = block_scan<kRow>(mine, s.sums, all);
            if (run - mine < want && want <= run) {
                s.bin = 255 - tid;
                s.pick = run - mine;
            }
            __syncthreads();
            want -= s.pick;
            prefix = prefix << 8 | s.bin;
        }
        // equal logits measure the same: the nth of them in index order
        const u64 each = measure(key_value(prefix)), nth = each ? (want + each - 1) / each : 1;
        const uint32_t lo = (uint32_t)((uint64_t)n * wave / kRowWaves), hi = (uint32_t)((uint64_t)n * (wave + 1) / kRowWaves);
        auto tie = [&](uint32_t i) {
            const float v = T::load(x[min(i, n - 1)]);
            return i < hi && rank_key(v) == prefix && rank(v, i) >= cut;
        };
        u64 count = 0, all;
        for (uint32_t i0 = lo; i0 < hi; i0 += 64) count += __popcll(__ballot(tie(i0 + lane)));
        u64 before = block_scan<kRow>(lane == 0 ? count : 0, s.sums, all) - count;  // the same in the wave's lanes
        if (before < nth && nth <= before + count) {
            for (uint32_t i0 = lo; i0 < hi; i0 += 64) {
                const u64 ties = __ballot(tie(i0 + lane)), here = __popcll(ties);
                if (before + here >= nth) {
                    if ((ties >> lane & 1) && before + __popcll(ties & ((2ull << lane) - 1)) == nth) s.pick = (u64)prefix << 32 | (uint32_t)~(i0 + lane);
                    break;
                }
                before += here;
            }
        }
        __syncthreads();
        cut = s.pick;
        __syncthreads();
    };
    if (w.useK) move(w.k, [](float) { return (u64)1; });
    if (w.useP) {
        u64 z = 0, total;
        each_logit<T, kRow>(x, 0, n, [&](uint32_t i, float v) { z += rank(v, i) >= cut ? w.weight(v) : 0; });
        (void)block_scan<kRow>(z, s.sums, total);
        move(limit_of(w.p, total), [&](float v) { return w.weight(v); });
    }
    return cut;
}

// The first kept index of [lo, hi) whose running weight, from `before` on, passes `target`.
template <typename T>
__device__ inline void find_token(RowSpace &s, const typename T::storage *__restrict__ x, const Row &w, u64 cut, uint32_t lo, uint32_t hi,
                                  u64 before, u64 target, int32_t *token) {
    for (uint32_t i0 = lo; i0 < hi; i0 += kRow * E) {
        u64 u[E], mine = 0, all;
#pragma unroll
        for (uint32_t j = 0; j < E; ++j) u[j] = 0;
        const uint32_t from = i0 + threadIdx.x * E;
#pragma unroll
        for (uint32_t j = 0; j < E; ++j)
            if (from + j < hi) {
                const float v = T::load(x[from + j]);
                const u64 m = w.weight(v);
                u[j] = m >= w.least && ((u64)rank_key(v) << 32 | (uint32_t)~(from + j)) >= cut ? m : 0;
                mine += u[j];
            }
        u64 run = before + block_scan<kRow>(mine, s.sums, all) - mine;
        if (run <= target && target < run + mine) {
            for (uint32_t j = 0; j < E; ++j) {
                run += u[j];
                if (run > target) {
                    *token = (int32_t)(from + j);
                    break;
                }
            }
        }
        before += all;
        if (before > target) return;  // (the same in every thread)
    }
}

__device__ inline u64 target_of(float u, u64 z) {
    bool more;
    return share(u > 0.0f ? (uint32_t)fmin((double)u * 2147483648.0, 2147483647.0) : 0u, z, more);
}

template <typename T>
__device__ void sample_finish(const typename T::storage *__restrict__ logits, const Options &o, const SampleRow *__restrict__ rows,
                              int32_t *__restrict__ tokens, const SampleConstants &c) {
    __shared__ RowSpace s;
    __shared__ uint32_t sTop[4];
    const uint32_t r = blockIdx.x, tid = threadIdx.x;
    const SampleRow &row = rows[r];
    const typename T::storage *x = logits + (uint64_t)r * c.vocab;
    const Row w = row_of(o, r, top_of<kRow>(row, c.slices, sTop), c);
    if (!w.live) {
        if (tid == 0) tokens[r] = -1;
        return;
    }
    if (tid < c.slices) s.slice[tid] = row.sliceWeight[tid];
    u64 cut = 0;
    if ((w.useK || w.useP) && row.candidates > kList) {
        cut = cut_by_digits<T>(s, x, w, c.vocab);
        u64 z = 0, all;
        each_logit<T, kRow>(x, 0, c.vocab, [&](uint32_t i, float v) {
            const u64 m = w.weight(v);
            z += m >= w.least && ((u64)rank_key(v) << 32 | (uint32_t)~i) >= cut ? m : 0;
        });
        (void)block_scan<kRow>(z, s.sums, all);
        find_token<T>(s, x, w, cut, 0, c.vocab, 0, target_of(o.uniforms[r], all), tokens + r);
        return;
    }
    if (w.useK || w.useP) {
        const uint32_t n = row.candidates;
        for (uint32_t i = tid; i < n; i += kRow) s.list[i] = row.candidate[i];
        __syncthreads();
        cut = cut_in_list(s, w, n, row.binK, row.needK, row.lastP, row.aboveK, row.aboveP, row.total);
        for (uint32_t i = tid; i < n; i += kRow)
            if (s.list[i] >= cut) {
                const u64 m = w.weight(key_value((uint32_t)(s.list[i] >> 32)));
                if (m >= w.least) atomicAdd(&s.slice[~(uint32_t)s.list[i] / c.sliceLen], m);
            }
    }
    __syncthreads();
    u64 z;
    const u64 mine = tid < c.slices ? s.slice[tid] : 0, run = block_scan<kRow>(mine, s.sums, z);
    const u64 target = target_of(o.uniforms[r], z);
    if (run - mine <= target && target < run) {
        s.bin = tid;
        s.pick = run - mine;
    }
    __syncthreads();
    const uint32_t lo = s.bin * c.sliceLen;
    find_token<T>(s, x, w, cut, lo, min(lo + c.sliceLen, c.vocab), s.pick, target, tokens + r);
}

template <typename T>
__device__ void sample_small(const typename T::storage *__restrict__ logits, const Options &o, int32_t *__restrict__ tokens,
                             const SampleConstants &c) {
    __shared__ RowSpace s;
    const uint32_t r = blockIdx.x, tid = threadIdx.x, n = c.vocab;
    const typename T::storage *x = logits + (uint64_t)r * n;
    uint32_t best = 0;
    for (uint32_t i = tid; i < n; i += kRow) {
        const uint32_t key = rank_key(T::load(x[i]));
        s.list[i] = (u64)key << 32 | (uint32_t)~i;
        best = max(best, key);
    }
    best = wave_max_u32(best);
    if ((tid & 63) == 0) s.counts[tid >> 6] = best;
    __syncthreads();
    for (uint32_t v = 0; v < kRowWaves; ++v) best = max(best, s.counts[v]);
    __syncthreads();
    const Row w = row_of(o, r, best, c);
    if (!w.live) {
        if (tid == 0) tokens[r] = -1;
        return;
    }
    u64 cut = 0, z = 0, all;
    if (w.useK || w.useP) {
        u64 total = 0;
        for (uint32_t i = tid; i < n; i += kRow) z += w.weight(T::load(x[i]));
        (void)block_scan<kRow>(z, s.sums, total);
        // every token a candidate: top-k's bin is then the one that nothing lies before
        cut = cut_in_list(s, w, n, w.useK ? 0u : kBins, w.k, kBins, 0, 0, total);
        z = 0;
    }
    for (uint32_t i = tid; i < n; i += kRow) {
        const float v = T::load(x[i]);
        const u64 m = w.weight(v);
        z += m >= w.least && ((u64)rank_key(v) << 32 | (uint32_t)~i) >= cut ? m : 0;
    }
    (void)block_scan<kRow>(z, s.sums, all);
    find_token<T>(s, x, w, cut, 0, n, 0, target_of(o.uniforms[r], all), tokens + r);
}

}  // namespace

#define SAMPLE(t, T)                                                                                                              \
    POPCORN_KERNEL void __launch_bounds__(256) sample_top_##t(const T::storage *logits, SampleRow *rows, SampleConstants c) {     \
        sample_top<T>(logits, rows, c);                                                                                           \
    }                                                                                                                             \
    POPCORN_KERNEL void __launch_bounds__(256)                                                                                    \
        sample_hist_##t(const T::storage *logits, const float *uniforms, const float *temperature, const int32_t *topK,           \
                        const float *topP, const float *minP, SampleRow *rows, SampleConstants c) {                               \
        sample_hist<T>(logits, Options{uniforms, temperature, topK, topP, minP}, rows, c);                                        \
    }                                                                                                                             \
    POPCORN_KERNEL void __launch_bounds__(256)                                                                                    \
        sample_gather_##t(const T::storage *logits, const float *uniforms, const float *temperature, const int32_t *topK,         \
                          const float *topP, const float *minP, SampleRow *rows, SampleConstants c) {                             \
        sample_gather<T>(logits, Options{uniforms, temperature, topK, topP, minP}, rows, c);                                      \
    }                                                                                                                             \
    POPCORN_KERNEL void __launch_bounds__(1024)                                                                                   \
        sample_finish_##t(const T::storage *logits, const float *uniforms, const float *temperature, const int32_t *topK,         \
                          const float *topP, const float *minP, const SampleRow *rows, int32_t *tokens, SampleConstants c) {      \
        sample_finish<T>(logits, Options{uniforms, temperature, topK, topP, minP}, rows, tokens, c);                              \
    }                                                                                                                             \
    POPCORN_KERNEL void __launch_bounds__(1024)                                                                                   \
        sample_small_##t(const T::storage *logits, const float *uniforms, const float *temperature, const int32_t *topK,          \
                         const float *topP, const float *minP, int32_t *tokens, SampleConstants c) {                              \
        sample_small<T>(logits, Options{uniforms, temperature, topK, topP, minP}, tokens, c);                                     \
    }

SAMPLE(f32, pk::F32)
SAMPLE(f16, pk::F16)
SAMPLE(bf16, pk::BF16)
