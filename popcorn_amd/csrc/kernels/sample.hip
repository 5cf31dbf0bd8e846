// One token a row of logits, drawn with a given uniform random number.
//
// Tokens rank by logit, ties by index; a token's weight is 2^40 exp((logit -
// highest) / temperature) as a whole number (sample.hpp), so sums of weights are
// exact whatever their order, and a vocabulary of up to 2^22 tokens sums below
// 2^62. Each option keeps a prefix of the ranking, so
// what is kept is one cut (a logit and an index) and a least weight.
//
// Sorting the row is not needed to find the cut. Four launches, a row cut into slices:
//  1. sample_top: the highest logit;
//  2. sample_hist: number and weight of the tokens of each slice in 2048
//     bins of the distance from the highest, and their sums over the row;
//  3. sample_gather: the bins in which the cuts must fall, from the bins'
//     running sums; their tokens (the candidates, a few hundred where a model
//     has its preferences) go to a list, and of each slice the weight of what lies before;
//  4. sample_finish: the cuts among the candidates, by selection, the
//     slice where the running weight passes the draw, and the token in it.
// Only the second evaluates the whole row's weights, which bounds it (24 us of
// 64 rows of 256000 bf16 logits, 49 instructions a logit; the others 8, 18
// and 18, the last with one block to a row). A row that neither top-k
// nor top-p cuts has its slices' weights summed by the third instead; a call
// without either has no second launch (64 x 256000 in 40 us).
// A row of up to 4096 logits is one launch (sample_small): all are candidates.
// More candidates than the list holds are counted digit by digit of their
// logits instead (cut_by_digits): thousands of equal logits at the cut, or a flat
// row, where a bin's 1/72 of a temperature is wide enough for thousands of
// different ones (256000 normal logits of spread 0.5 at temperature 2 put about
// 5500 in top-p's bin). So is min-p at temperatures that lead the bins out of
// f32's range. One block then reads the row 6 to 11 times: 64 such rows of
// 256000 take 0.65 ms instead of 0.07, 0.90 with top-k too, one 0.47; 64 of equal
// logits, whose additions all meet in one word, 1.37.
#include "sample.hpp"
#include "scan.hpp"

namespace {

constexpr uint32_t kThreads = 1024, kWaves = kThreads / 64;
constexpr uint32_t E = 8;                               // consecutive logits per thread and step
constexpr double kOne = 1099511627776.0;                // 2^40
constexpr uint32_t kBins = SAMPLE_BINS, kList = SAMPLE_CANDIDATES;
constexpr uint32_t kPerThread = kBins / kThreads, kEach = kList / kThreads, kFew = 128;
constexpr uint32_t kFound = 1024;                       // candidates that a block of sample_gather collects
typedef uint64_t u64;
using pk::Scan;
using pk::wave_max_u32;
using pk::wave_sum64;

__device__ inline void add64(u64 *at, u64 v) { atomicAdd(reinterpret_cast<unsigned long long *>(at), (unsigned long long)v); }

// A logit's place in the ranking: greater for greater logits, 0 for NaN, equal
// for both zeros.
__device__ inline uint32_t rank_key(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    if (v != v) return 0u;
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ inline float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

struct Options {
    const float *uniforms, *temperature;
    const int32_t *topK;
    const float *topP, *minP;
};

// One row's options, and its highest logit.
struct Row {
    float top, bins;  // bins per unit of distance
    double rate;      // pk::sample_rate
    u64 least;
    float p;
    uint32_t k;
    bool live, useK, useP;
    bool binned;  // bins are as the definition has them; else they only keep the order

    __device__ inline u64 weight(float v) const { return pk::sample_weight(v, top, rate); }
    __device__ inline float uniform(const Options &o, uint32_t r) const { return rate < INFINITY ? o.uniforms[r] : 0.0f; }
    // Grows, if anything, from a logit to the next in the ranking.
    __device__ inline uint32_t bin(float v) const {
        return v == top ? 0u : (uint32_t)fminf((top - v) * bins, (float)(kBins - 1));
    }
};

__device__ inline Row row_of(const Options &o, uint32_t r, uint32_t topKey, const SampleConstants &c) {
    Row w;
    w.top = key_value(topKey);
    w.live = topKey != 0 && w.top > -INFINITY;
    const float t = c.hasTemperature ? o.temperature[r] : 1.0f;
    const int32_t k = c.hasTopK ? o.topK[r] : 0;
    const float p = c.hasTopP ? o.topP[r] : 1.0f, least = c.hasMinP ? o.minP[r] : 0.0f;
    // a temperature of 0 leaves weight to the highest logit alone, of which a uniform of 0 draws the first: no cut
    const bool greedy = !(t > 0.0f);
    w.rate = pk::sample_rate(greedy ? 0.0f : t);
    w.bins = 72.0f / t;  // weights end at a distance of 28.5 temperatures
    w.binned = t > 3e-37f && t < 1e37f;  // neither 72 / t nor a distance of 28.5 t passes the largest number
    w.k = k > 0 ? (uint32_t)k : 0u;
    w.useK = w.k > 0 && w.k < c.vocab && !greedy;
    w.useP = p < 1.0f && !greedy;  // (not where it is NaN)
    w.p = fmaxf(p, 0.0f);
    w.least = least > 0.0f && !greedy ? (u64)__builtin_ceil((double)fminf(least, 1.0f) * kOne) : 0;
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

// f(index, its place among the eight, logit) for this thread's logits of [lo, hi), eight in a row at a time;
// after each eight done(index of the first).
template <typename T, typename F, typename D>
__device__ inline void each_logit(const typename T::storage *__restrict__ x, uint32_t lo, uint32_t hi, F &&f, D &&done) {
    struct Eight {
        typename T::storage v[E];
    };
#pragma unroll 1
    for (uint32_t i = lo + threadIdx.x * E; i < hi; i += kThreads * E) {
        if (i + E <= hi) {
            Eight e;
            __builtin_memcpy(&e, x + i, sizeof(e));
#pragma unroll
            for (uint32_t j = 0; j < E; ++j) f(i + j, j, T::load(e.v[j]));
        } else {
#pragma unroll 1
            for (uint32_t j = i; j < hi; ++j) f(j, j - i, T::load(x[j]));
        }
        done(i);
    }
}
template <typename T, typename F>
__device__ inline void each_logit(const typename T::storage *__restrict__ x, uint32_t lo, uint32_t hi, F &&f) {
    each_logit<T>(x, lo, hi, f, [](uint32_t) {});
}

// Clears what the launches after it add to.
__device__ inline void clear_row(SampleRow &row, uint32_t at, uint32_t step) {
    for (uint32_t b = at; b < kBins; b += step) {
        row.weight[b] = 0;
        row.count[b] = 0;
    }
    if (at == 0) row.candidates = 0;
}

template <typename T>
__device__ void sample_top(const typename T::storage *__restrict__ logits, SampleRow *__restrict__ rows, const SampleConstants &c) {
    __shared__ uint32_t sTop[kWaves];
    const uint32_t r = blockIdx.x / c.slices, slice = blockIdx.x % c.slices;
    const uint32_t lo = slice * c.sliceLen, hi = min(lo + c.sliceLen, c.vocab);
    uint32_t best = 0;
    each_logit<T>(logits + (uint64_t)r * c.vocab, lo, hi, [&](uint32_t, uint32_t, float v) { best = max(best, rank_key(v)); });
    best = wave_max_u32(best);
    if ((threadIdx.x & 63) == 0) sTop[threadIdx.x >> 6] = best;
    __syncthreads();
    if (threadIdx.x < 64) {
        best = wave_max_u32(threadIdx.x < kWaves ? sTop[threadIdx.x] : 0u);
        if (threadIdx.x == 0) rows[r].sliceTop[slice] = best;
    }
    clear_row(rows[r], slice * kThreads + threadIdx.x, c.slices * kThreads);
}

// The row's highest logit, of up to 64 slices: each wave by itself.
__device__ inline uint32_t top_of(const SampleRow &row, uint32_t slices) {
    const uint32_t lane = threadIdx.x & 63;
    return wave_max_u32(lane < slices ? row.sliceTop[lane] : 0u);
}

template <typename T>
__device__ void sample_hist(const typename T::storage *__restrict__ logits, const Options &o, SampleRow *__restrict__ rows,
                            uint64_t *__restrict__ bins, const SampleConstants &c) {
    __shared__ u64 sWeight[kBins];
    __shared__ uint32_t sCount[kBins];
    const uint32_t r = blockIdx.x / c.slices, slice = blockIdx.x % c.slices;
    SampleRow &row = rows[r];
    const Row w = row_of(o, r, top_of(row, c.slices), c);
    if (!w.live || !(w.useK || w.useP)) return;
    for (uint32_t b = threadIdx.x; b < kBins; b += kThreads) {
        sWeight[b] = 0;
        sCount[b] = 0;
    }
    __syncthreads();
    const uint32_t lo = slice * c.sliceLen, hi = min(lo + c.sliceLen, c.vocab);
    each_logit<T>(logits + (uint64_t)r * c.vocab, lo, hi, [&](uint32_t, uint32_t, float v) {
        const u64 u = w.weight(v);
        if (u == 0) return;
        const uint32_t b = w.bin(v);
        add64(&sWeight[b], u);
        if (w.useK) atomicAdd(&sCount[b], 1u);
    });
    __syncthreads();
    uint64_t *mine = bins + (uint64_t)blockIdx.x * kBins;
    for (uint32_t b = threadIdx.x; b < kBins; b += kThreads) {
        mine[b] = sWeight[b];
        if (sWeight[b]) add64(&row.weight[b], sWeight[b]);
        if (sCount[b]) atomicAdd(&row.count[b], sCount[b]);
    }
}

// Whether min-p may cut in a bin: the bin where e^-distance is least - 1/2 (from
// there on a weight is rounded to `least`), and one to either side for the
// roundings of bin and weight (a bin's weights span 1.4%).
__device__ inline bool least_bin(const Row &w, uint32_t b, float at) {
    return (w.least != 0) & (fabsf((float)b + 0.5f - at) < 2.0f);
}
__device__ inline float least_at(const Row &w) {
    return w.least ? (40.0f - __log2f((float)w.least - 0.5f)) * (72.0f * 0.69314718f) : 1e9f;
}

template <typename T>
__device__ void sample_gather(const typename T::storage *__restrict__ logits, const Options &o, SampleRow *__restrict__ rows,
                              const uint64_t *__restrict__ bins, const SampleConstants &c) {
    __shared__ u64 sSums[kWaves], sAbove[2], sWith, sList[kFound], sKept[SAMPLE_MAX_SLICES];
    __shared__ uint32_t sCounts[kWaves], sBin[3], sNeed, sFound, sBase;
    const uint32_t r = blockIdx.x / c.parts, part = blockIdx.x % c.parts;
    SampleRow &row = rows[r];
    const uint32_t tid = threadIdx.x;
    const Row w = row_of(o, r, top_of(row, c.slices), c);
    if (!w.live) return;
    const typename T::storage *x = logits + (uint64_t)r * c.vocab;
    if (!(w.useK || w.useP)) {
        for (uint32_t slice = part; slice < c.slices; slice += c.parts) {
            const uint32_t lo = slice * c.sliceLen, hi = min(lo + c.sliceLen, c.vocab);
            u64 sum = 0;
            each_logit<T>(x, lo, hi, [&](uint32_t, uint32_t, float v) {
                const u64 u = w.weight(v);
                sum += u >= w.least ? u : 0;
            });
            sum = pk::block_scan<kWaves>(sum, sSums).total;
            if (tid == 0) row.weight[slice] = sum;
        }
        return;
    }
    if (w.least && !w.binned) {  // no bin is known to hold min-p's border: the row is counted by digits
        if (part == 0 && tid == 0) row.candidates = kList + 1;
        return;
    }
    // bins before `first` are kept; candidates are the bins first .. lastP and binK
    u64 bw[kPerThread], mine = 0;
    uint32_t bc[kPerThread], here = 0;
#pragma unroll
    for (uint32_t j = 0; j < kPerThread; ++j) {
        bw[j] = row.weight[tid * kPerThread + j];
        bc[j] = row.count[tid * kPerThread + j];
        mine += bw[j];
        here += bc[j];
    }
    const Scan<u64> weights = pk::block_scan<kWaves>(mine, sSums);
    const u64 wend = weights.upto, total = weights.total;
    const uint32_t cend = pk::block_scan<kWaves>(here, sCounts).upto;
    if (tid < SAMPLE_MAX_SLICES) sKept[tid] = 0;
    if (tid == 0) {
        sFound = 0;
        sBin[0] = sBin[1] = sBin[2] = kBins;
        sAbove[0] = sAbove[1] = 0;
        sNeed = 0;
    }
    __syncthreads();
    // calls at(bin, weight before it, with it, tokens before it) for the one bin of this thread's that `in` names
    auto find = [&](auto &&in, auto &&at) {
        u64 before = wend - mine;
        uint32_t cb = cend - here;
#pragma unroll
        for (uint32_t j = 0; j < kPerThread; ++j) {
            if (in(before, before + bw[j], cb, cb + bc[j])) at(tid * kPerThread + j, before, before + bw[j], cb);
            before += bw[j];
            cb += bc[j];
        }
    };
    u64 zLo = total, zHi = total;
    uint32_t first, lastP, binK = kBins;
    if (w.useK) {
        find([&](u64, u64, uint32_t a, uint32_t b) { return a < w.k && w.k <= b; },
             [&](uint32_t b, u64 before, u64 with, uint32_t cb) {
                 sBin[0] = b;
                 sAbove[0] = before;
                 sWith = with;
                 sNeed = w.k - cb;
             });
        __syncthreads();
        binK = sBin[0];
        if (binK < kBins) {
            zLo = sAbove[0];
            zHi = sWith;
        }
    }
    if (w.useP) {
        // top-p's share is of a weight between zLo and zHi
        const u64 a0 = limit_of(w.p, zLo), a1 = limit_of(w.p, zHi);
        find([&](u64 a, u64 b, uint32_t, uint32_t) { return a < a0 && a0 <= b; },
             [&](uint32_t b, u64 before, u64, uint32_t) {
                 sBin[1] = b;
                 sAbove[1] = before;
             });
        find([&](u64 a, u64 b, uint32_t, uint32_t) { return a < a1 && a1 <= b; }, [&](uint32_t b, u64, u64, uint32_t) { sBin[2] = b; });
        __syncthreads();
        first = sBin[1];
        lastP = sBin[2];
    } else {
        first = lastP = binK;
    }
    if (part == 0 && tid == 0) {
        row.first = first;
        row.binK = binK;
        row.needK = sNeed;
        row.aboveK = sAbove[0];
        row.aboveP = sAbove[1];
        row.total = total;
    }
    const float at = least_at(w);
    // the part's slices are next to each other
    const uint32_t each = (c.slices + c.parts - 1) / c.parts, s0 = min(part * each, c.slices), s1 = min(s0 + each, c.slices);
    // each slice's weight of the bins that are kept whatever the cuts
    for (uint32_t sl = s0; sl < s1; ++sl) {
        const uint64_t *b = bins + ((uint64_t)r * c.slices + sl) * kBins + tid * kPerThread;
        u64 sum = 0;
#pragma unroll
        for (uint32_t j = 0; j < kPerThread; ++j) {
            const uint32_t i = tid * kPerThread + j;
            const u64 v = b[j];
            sum += (i < first) & !least_bin(w, i, at) & ((float)i < at) ? v : 0;
        }
        sum = wave_sum64(sum);
        if ((tid & 63) == 0) add64(&sKept[sl - s0], sum);
    }
    auto put = [&](uint32_t slot, u64 v) {
        if (slot < kList) row.candidate[slot] = v;
    };
    uint32_t found = 0;  // of a thread's eight, a bit each
    auto collect = [&](uint32_t i0) {
#pragma unroll 1
        for (; found; found &= found - 1) {
            const uint32_t i = i0 + (uint32_t)__ffs((int)found) - 1;
            const u64 c = (u64)rank_key(T::load(x[i])) << 32 | (uint32_t)~i;
            const uint32_t n = atomicAdd(&sFound, 1u);
            if (n < kFound) sList[n] = c;
            else put(atomicAdd(&row.candidates, 1u), c);
        }
    };
    const uint32_t hi = min(s1 * c.sliceLen, c.vocab);
    each_logit<T>(
        x, s0 * c.sliceLen, hi,
        [&](uint32_t, uint32_t j, float v) {
            const uint32_t b = w.bin(v);
            found |= (uint32_t)((v > -INFINITY) & (b < first ? least_bin(w, b, at) : (b <= lastP) | (b == binK))) << j;
        },
        collect);
    __syncthreads();
    // the row's counter is one address for all its blocks: one addition each
    const uint32_t n = min(sFound, kFound);
    if (tid < s1 - s0) row.kept[s0 + tid] = sKept[tid];
    if (tid == 0) sBase = n ? atomicAdd(&row.candidates, n) : 0;
    __syncthreads();
    for (uint32_t i = tid; i < n; i += kThreads) put(sBase + i, sList[i]);
}

struct RowSpace {
    u64 list[kList];
    u64 sums[kWaves], slice[SAMPLE_MAX_SLICES], pick, bits[2];
    u64 weights[kThreads], few[kFew], measure[kFew];
    uint32_t counts[kWaves], bin, left;
};

// The entry at which the running measure m, over entries e (all distinct) from the greatest, reaches `want`: at
// least 1, at most the sum. Entries of measure 0 are not looked at. While more than kFew are left, a pass keeps one
// of 1024 values of the 10 bits from the highest in which they differ; the few are compared with each other.
// (A sort by merging made sample_finish 34 us of 64 rows of 256000 bf16 logits, this 20; counting every entry's
// greater ones was 1.5 us faster for 100 candidates.)
__device__ inline u64 select(RowSpace &s, const u64 (&e)[kEach], const u64 (&m)[kEach], u64 want) {
    const uint32_t tid = threadIdx.x;
    uint32_t left = 0;
#pragma unroll
    for (uint32_t j = 0; j < kEach; ++j) left |= (uint32_t)(m[j] != 0) << j;
    while (true) {
        s.weights[tid] = 0;
        if (tid < 2) s.bits[tid] = 0;
        if (tid == 0) s.left = 0;
        u64 ones = 0, zeros = 0;
        __syncthreads();
#pragma unroll
        for (uint32_t j = 0; j < kEach; ++j)
            if (left >> j & 1) {
                ones |= e[j];
                zeros |= ~e[j];
                const uint32_t at = atomicAdd(&s.left, 1u);
                if (at < kFew) {
                    s.few[at] = e[j];
                    s.measure[at] = m[j];
                }
            }
        if (__ballot(left != 0)) {
            ones = pk::wave_or64(ones);
            zeros = pk::wave_or64(zeros);
            if ((tid & 63) == 0) {
                atomicOr(reinterpret_cast<unsigned long long *>(&s.bits[0]), (unsigned long long)ones);
                atomicOr(reinterpret_cast<unsigned long long *>(&s.bits[1]), (unsigned long long)zeros);
            }
        }
        __syncthreads();
        if (s.left <= kFew) break;
        const int shift = max(63 - __clzll((long long)(s.bits[0] & s.bits[1])) - 9, 0);
#pragma unroll
        for (uint32_t j = 0; j < kEach; ++j)
            if (left >> j & 1) add64(&s.weights[e[j] >> shift & 1023u], m[j]);
        __syncthreads();
        const uint32_t digit = 1023 - tid;
        const u64 mine = s.weights[digit], run = pk::block_scan<kWaves>(mine, s.sums).upto;
        if (run - mine < want && want <= run) {
            s.bin = digit;
            s.pick = run - mine;
        }
        __syncthreads();
        want -= s.pick;
#pragma unroll
        for (uint32_t j = 0; j < kEach; ++j) left &= ~((uint32_t)((e[j] >> shift & 1023u) != s.bin) << j);
    }
    // s.weights, cleared: each of the few's running measure, of a part of the others by each of its threads
    const uint32_t few = s.left, at = tid % kFew;
    const u64 mine = at < few ? s.few[at] : ~(u64)0;
    u64 run = 0;
#pragma unroll 4
    for (uint32_t j = tid / kFew; j < few; j += kThreads / kFew) run += s.few[j] >= mine ? s.measure[j] : 0;
    if (run) add64(&s.weights[at], run);
    __syncthreads();
    run = s.weights[at];
    if (tid < few && run - s.measure[at] < want && want <= run) s.pick = mine;
    __syncthreads();
    return s.pick;
}

// The last token that top-k and top-p keep, of n candidates in the list (in any order): rank key << 32 | ~index; 0
// keeps all. (Tokens of bins before `first` are in the list for min-p's sake, and kept.)
__device__ inline u64 cut_in_list(RowSpace &s, const Row &w, uint32_t n, uint32_t first, uint32_t binK, uint32_t needK, u64 aboveK,
                                  u64 aboveP, u64 total) {
    u64 e[kEach], u[kEach], m[kEach], cut = 0, sum = 0;
    uint32_t bins[kEach], count = 0;
    __syncthreads();
#pragma unroll
    for (uint32_t j = 0; j < kEach; ++j) {
        const uint32_t i = threadIdx.x + j * kThreads;
        e[j] = u[j] = m[j] = 0;
        bins[j] = 0;
        if (i < n) {
            e[j] = s.list[i];
            const float v = key_value((uint32_t)(e[j] >> 32));
            u[j] = w.weight(v);
            bins[j] = w.bin(v);
            m[j] = bins[j] >= binK;
            count += (uint32_t)m[j];
        }
    }
    if (binK < kBins) {
        if (pk::block_scan<kWaves>(count, s.counts).total >= needK) cut = select(s, e, m, needK);
#pragma unroll
        for (uint32_t j = 0; j < kEach; ++j) sum += m[j] && e[j] >= cut ? u[j] : 0;
        total = aboveK + pk::block_scan<kWaves>(sum, s.sums).total;
    }
    if (w.useP) {
        sum = 0;
#pragma unroll
        for (uint32_t j = 0; j < kEach; ++j) {
            m[j] = bins[j] >= first && e[j] >= cut ? u[j] : 0;
            sum += m[j];
        }
        const u64 want = limit_of(w.p, total) - aboveP;
        if (pk::block_scan<kWaves>(sum, s.sums).total >= want) cut = select(s, e, m, want);
    }
    return cut;
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
            each_logit<T>(x, 0, n, [&](uint32_t i, uint32_t, float v) {
                const uint32_t key = rank_key(v);
                if (shift < 24 && (key >> (shift + 8)) != prefix) return;
                if (rank(v, i) >= cut) add64(&s.weights[(key >> shift) & 255u], measure(v));
            });
            __syncthreads();
            // thread t takes digit 255 - t
            const u64 mine = tid < 256 ? s.weights[255 - tid] : 0, run = pk::block_scan<kWaves>(mine, s.sums).upto;
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
        const uint32_t lo = (uint32_t)((uint64_t)n * wave / kWaves), hi = (uint32_t)((uint64_t)n * (wave + 1) / kWaves);
        auto tie = [&](uint32_t i) {
            const float v = T::load(x[min(i, n - 1)]);
            return i < hi && rank_key(v) == prefix && rank(v, i) >= cut;
        };
        u64 count = 0;
        for (uint32_t i0 = lo; i0 < hi; i0 += 64) count += __popcll(__ballot(tie(i0 + lane)));
        u64 before = pk::block_scan<kWaves>(lane == 0 ? count : 0, s.sums).upto - count;  // the same in the wave's lanes
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
        u64 z = 0;
        each_logit<T>(x, 0, n, [&](uint32_t i, uint32_t, float v) { z += rank(v, i) >= cut ? w.weight(v) : 0; });
        move(limit_of(w.p, pk::block_scan<kWaves>(z, s.sums).total), [&](float v) { return w.weight(v); });
    }
    return cut;
}

// The first kept index of [lo, hi) whose running weight, from `before` on, passes `target`.
template <typename T>
__device__ inline void find_token(RowSpace &s, const typename T::storage *__restrict__ x, const Row &w, u64 cut, uint32_t lo, uint32_t hi,
                                  u64 before, u64 target, int32_t *token) {
    for (uint32_t i0 = lo; i0 < hi; i0 += kThreads * E) {
        const uint32_t from = i0 + threadIdx.x * E;
        struct Eight {
            typename T::storage v[E];
        } e;
        if (from + E <= hi) {
            __builtin_memcpy(&e, x + from, sizeof(e));
        } else {
#pragma unroll
            for (uint32_t j = 0; j < E; ++j) e.v[j] = x[min(from + j, hi - 1)];
        }
        u64 u[E], mine = 0;
#pragma unroll
        for (uint32_t j = 0; j < E; ++j) {
            const float v = T::load(e.v[j]);
            const bool in = (from + j < hi) & (((u64)rank_key(v) << 32 | (uint32_t)~(from + j)) >= cut);
            u[j] = 0;
            if (__ballot(in)) {  // (top-k leaves most waves none)
                const u64 m = w.weight(v);
                u[j] = in & (m >= w.least) ? m : 0;
            }
            mine += u[j];
        }
        const Scan<u64> scan = pk::block_scan<kWaves>(mine, s.sums);
        u64 run = before + scan.upto - mine;
        if (run <= target && target < run + mine) {
            uint32_t at = 0;
#pragma unroll
            for (uint32_t j = 0; j < E; ++j) {
                run += u[j];
                at += run <= target;
            }
            *token = (int32_t)(from + at);
        }
        before += scan.total;
        if (before > target) return;  // (the same in every thread)
    }
}

__device__ inline u64 target_of(float u, u64 z) {
    bool more;
    return share(u > 0.0f ? (uint32_t)fmin((double)u * 2147483648.0, 2147483647.0) : 0u, z, more);
}

template <typename T>
__device__ __attribute__((noinline)) void finish_by_digits(RowSpace &s, const typename T::storage *__restrict__ x, Row w, uint32_t n, float u,
                                                           int32_t *token) {
    const u64 cut = cut_by_digits<T>(s, x, w, n);
    u64 z = 0;
    each_logit<T>(x, 0, n, [&](uint32_t i, uint32_t, float v) {
        const u64 m = w.weight(v);
        z += m >= w.least && ((u64)rank_key(v) << 32 | (uint32_t)~i) >= cut ? m : 0;
    });
    find_token<T>(s, x, w, cut, 0, n, 0, target_of(u, pk::block_scan<kWaves>(z, s.sums).total), token);
}

template <typename T>
__device__ void sample_finish(const typename T::storage *__restrict__ logits, const Options &o, const SampleRow *__restrict__ rows,
                              int32_t *__restrict__ tokens, const SampleConstants &c) {
    __shared__ RowSpace s;
    const uint32_t r = blockIdx.x, tid = threadIdx.x;
    const SampleRow &row = rows[r];
    const typename T::storage *x = logits + (uint64_t)r * c.vocab;
    const Row w = row_of(o, r, top_of(row, c.slices), c);
    if (!w.live) {
        if (tid == 0) tokens[r] = -1;
        return;
    }
    u64 cut = 0;
    const bool cuts = w.useK || w.useP;
    if (cuts && row.candidates > kList) {
        finish_by_digits<T>(s, x, w, c.vocab, w.uniform(o, r), tokens + r);
        return;
    }
    if (cuts) {
        const uint32_t n = row.candidates;
        for (uint32_t i = tid; i < n; i += kThreads) s.list[i] = row.candidate[i];
        if (tid < c.slices) s.slice[tid] = row.kept[tid];
        __syncthreads();
        cut = cut_in_list(s, w, n, row.first, row.binK, row.needK, row.aboveK, row.aboveP, row.total);
        for (uint32_t i = tid; i < n; i += kThreads)
            if (s.list[i] >= cut) {
                const u64 m = w.weight(key_value((uint32_t)(s.list[i] >> 32)));
                if (m >= w.least) add64(&s.slice[~(uint32_t)s.list[i] / c.sliceLen], m);
            }
    } else if (tid < c.slices) {
        s.slice[tid] = row.weight[tid];
    }
    __syncthreads();
    const u64 mine = tid < c.slices ? s.slice[tid] : 0;
    const Scan<u64> scan = pk::block_scan<kWaves>(mine, s.sums);
    const u64 run = scan.upto, target = target_of(w.uniform(o, r), scan.total);
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
    for (uint32_t i = tid; i < n; i += kThreads) {
        const uint32_t key = rank_key(T::load(x[i]));
        s.list[i] = (u64)key << 32 | (uint32_t)~i;
        best = max(best, key);
    }
    best = wave_max_u32(best);
    if ((tid & 63) == 0) s.counts[tid >> 6] = best;
    __syncthreads();
    for (uint32_t v = 0; v < kWaves; ++v) best = max(best, s.counts[v]);
    __syncthreads();
    const Row w = row_of(o, r, best, c);
    if (!w.live) {
        if (tid == 0) tokens[r] = -1;
        return;
    }
    u64 cut = 0, z = 0;
    if (w.useK || w.useP) {
        for (uint32_t i = tid; i < n; i += kThreads) z += w.weight(T::load(x[i]));
        // every token a candidate: top-k's bin is then the one that nothing lies before
        cut = cut_in_list(s, w, n, 0, w.useK ? 0u : kBins, w.k, 0, 0, pk::block_scan<kWaves>(z, s.sums).total);
        z = 0;
    }
    for (uint32_t i = tid; i < n; i += kThreads) {
        const float v = T::load(x[i]);
        const u64 m = w.weight(v);
        z += m >= w.least && ((u64)rank_key(v) << 32 | (uint32_t)~i) >= cut ? m : 0;
    }
    find_token<T>(s, x, w, cut, 0, n, 0, target_of(w.uniform(o, r), pk::block_scan<kWaves>(z, s.sums).total), tokens + r);
}

}  // namespace

#define SAMPLE_OPTIONS const float *uniforms, const float *temperature, const int32_t *topK, const float *topP, const float *minP
#define SAMPLE(t, T)                                                                                                           \
    POPCORN_KERNEL void __launch_bounds__(1024)                                                                                 \
        sample_top_##t(const T::storage *logits, SampleRow *rows, SampleConstants c) {                         \
        sample_top<T>(logits, rows, c);                                                                                  \
    }                                                                                                                          \
    POPCORN_KERNEL void __launch_bounds__(1024) sample_hist_##t(const T::storage *logits, SAMPLE_OPTIONS, \
                                                                SampleRow *rows, uint64_t *bins, SampleConstants c) {          \
        sample_hist<T>(logits, Options{uniforms, temperature, topK, topP, minP}, rows, bins, c);                         \
    }                                                                                                                          \
    POPCORN_KERNEL void __launch_bounds__(1024, 8)                                                                              \
        sample_gather_##t(const T::storage *logits, SAMPLE_OPTIONS, SampleRow *rows, const uint64_t *bins, SampleConstants c) {    \
        sample_gather<T>(logits, Options{uniforms, temperature, topK, topP, minP}, rows, bins, c);                             \
    }                                                                                                                          \
    POPCORN_KERNEL void __launch_bounds__(1024)                                                                                \
        sample_finish_##t(const T::storage *logits, SAMPLE_OPTIONS, const SampleRow *rows, int32_t *tokens, SampleConstants c) {   \
        sample_finish<T>(logits, Options{uniforms, temperature, topK, topP, minP}, rows, tokens, c);                           \
    }                                                                                                                          \
    POPCORN_KERNEL void __launch_bounds__(1024)                                                                                \
        sample_small_##t(const T::storage *logits, SAMPLE_OPTIONS, int32_t *tokens, SampleConstants c) {                       \
        sample_small<T>(logits, Options{uniforms, temperature, topK, topP, minP}, tokens, c);                                  \
    }

SAMPLE(f32, pk::F32)
SAMPLE(f16, pk::F16)
SAMPLE(bf16, pk::BF16)
