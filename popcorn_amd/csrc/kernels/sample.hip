// One token a row of logits, drawn with a given uniform random number.
//
// Tokens rank by logit, ties by index; a token's weight is the whole number
// rint(2^40 exp((logit - highest) / temperature)), exponent and rounding in 64
// bits, so sums of weights are exact whatever their order and a vocabulary of
// up to 2^22 tokens sums below 2^62. Each option keeps a prefix of the
// ranking, so what is kept is one cut: every token of a greater logit, and of
// the cut's logit those up to an index.
#include "common.hpp"

namespace {

constexpr uint32_t kThreads = 1024, kWaves = kThreads / 64;
constexpr double kOne = 1099511627776.0;  // 2^40
typedef unsigned long long u64;

// A logit's place in the ranking: greater for greater logits, 0 for NaN, equal
// for both zeros.
__device__ inline uint32_t rank_key(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    if (v != v) return 0u;
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ inline float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

__device__ inline u64 weight(float v, float top, double t) {
    if (!(v > -INFINITY)) return 0;
    if (v == top) return (u64)1 << 40;
    const double d = ((double)v - (double)top) / t;
    return d > -40.0 ? (u64)__builtin_rint(exp(d) * kOne) : 0;  // (a NaN is 0 too)
}

// floor(m z / 2^31), and whether a part is left over, for m <= 2^31 and z < 2^62.
__device__ inline u64 share(uint32_t m, u64 z, bool &more) {
    const u64 low = (z & 0x7fffffffu) * m;
    more = (low & 0x7fffffffu) != 0;
    return (z >> 31) * m + (low >> 31);
}

__device__ inline u64 wave_sum64(u64 v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

template <typename T>
__device__ void sample_row(const typename T::storage *__restrict__ x, uint32_t n, float u, float temperature, int32_t topK,
                           float topP, float minP, int32_t *token) {
    __shared__ u64 sHist[256], sSum[kWaves], sTotal;
    __shared__ uint32_t sMax[kWaves], sBin;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // wave w's stretch of the row, in index order
    const uint32_t lo = (uint32_t)((uint64_t)n * wave / kWaves), hi = (uint32_t)((uint64_t)n * (wave + 1) / kWaves);
    uint32_t best = 0;
    for (uint32_t i = tid; i < n; i += kThreads) best = max(best, rank_key(T::load(x[i])));
#pragma unroll
    for (int d = 32; d; d >>= 1) best = max(best, (uint32_t)__shfl_xor((int)best, d));
    if (lane == 0) sMax[wave] = best;
    __syncthreads();
    for (uint32_t w = 0; w < kWaves; ++w) best = max(best, sMax[w]);
    const float top = key_value(best);
    if (!(top > -INFINITY) || best == 0) {
        if (tid == 0) *token = -1;
        return;
    }
    const bool greedy = !(temperature > 0.0f);
    if (greedy) topK = 1;
    const double t = greedy ? 1.0 : (double)temperature;

    // the cut: kept are keys above cutKey, and of cutKey the indexes up to cutIndex
    uint32_t cutKey = 0, cutIndex = 0xffffffffu;
    auto kept = [&](uint32_t key, uint32_t i) { return key > cutKey || (key == cutKey && i <= cutIndex); };
    auto block_sum = [&](u64 v) {
        v = wave_sum64(v);
        __syncthreads();
        if (lane == 0) sSum[wave] = v;
        __syncthreads();
        u64 s = 0;
        for (uint32_t w = 0; w < kWaves; ++w) s += sSum[w];
        return s;
    };
    // Moves the cut to the token at which the running measure over the ranking
    // reaches `want` (1 <= want <= the measure of what is kept).
    auto cut = [&](u64 want, auto &&measure) {
        uint32_t prefix = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (uint32_t b = tid; b < 256; b += kThreads) sHist[b] = 0;
            __syncthreads();
            for (uint32_t i = tid; i < n; i += kThreads) {
                const float v = T::load(x[i]);
                const uint32_t key = rank_key(v);
                if (shift < 24 && (key >> (shift + 8)) != prefix) continue;
                if (kept(key, i)) atomicAdd(&sHist[(key >> shift) & 255u], measure(v));
            }
            __syncthreads();
            if (tid == 0) {
                u64 above = 0;
                uint32_t b = 255;
                for (; b > 0 && above + sHist[b] < want; --b) above += sHist[b];
                sBin = b;
                sTotal = above;
            }
            __syncthreads();
            want -= sTotal;
            prefix = prefix << 8 | sBin;
            __syncthreads();
        }
        // of the ties: each measures the same, so the nth of them in index order
        const u64 each = measure(key_value(prefix));
        const u64 nth = each ? (want + each - 1) / each : 1;
        u64 before = 0;
        uint32_t c = 0;
        for (uint32_t i = lo + lane; i < hi; i += 64) c += rank_key(T::load(x[i])) == prefix && kept(prefix, i);
        const u64 mine = wave_sum64(c);
        if (lane == 0) sSum[wave] = mine;
        if (tid == 0) sBin = 0xffffffffu;
        __syncthreads();
        for (uint32_t w = 0; w < wave; ++w) before += sSum[w];
        if (before < nth && nth <= before + mine) {  // (a wave's lanes together)
            for (uint32_t i0 = lo; i0 < hi; i0 += 64) {
                const uint32_t i = i0 + lane;
                const u64 tie = __ballot(i < hi && rank_key(T::load(x[min(i, hi - 1)])) == prefix && kept(prefix, i));
                const uint32_t count = (uint32_t)__popcll(tie);
                if (before + count >= nth) {
                    if ((tie >> lane & 1) && before + __popcll(tie & ((2ull << lane) - 1)) == nth) sBin = i;
                    break;
                }
                before += count;
            }
        }
        __syncthreads();
        cutKey = prefix;
        cutIndex = sBin;
        __syncthreads();
    };
    auto weigh = [&](float v) { return weight(v, top, t); };
    if (topK > 0 && (uint32_t)topK < n) cut((u64)topK, [](float) { return (u64)1; });
    if (topP < 1.0f) {  // (not where it is NaN)
        u64 z = 0;
        for (uint32_t i = tid; i < n; i += kThreads) {
            const float v = T::load(x[i]);
            if (kept(rank_key(v), i)) z += weigh(v);
        }
        z = block_sum(z);
        bool more;
        u64 limit = share((uint32_t)((double)max(topP, 0.0f) * 2147483648.0), z, more);
        limit += more;
        cut(limit ? limit : 1, weigh);
    }
    const u64 least = minP > 0.0f ? (u64)__builtin_ceil((double)min(minP, 1.0f) * kOne) : 0;
    // the draw, in index order
    auto mass = [&](uint32_t i) {
        const float v = T::load(x[i]);
        if (!kept(rank_key(v), i)) return (u64)0;
        const u64 w = weigh(v);
        return w >= least ? w : (u64)0;
    };
    u64 mine = 0;
    for (uint32_t i = lo + lane; i < hi; i += 64) mine += mass(i);
    mine = wave_sum64(mine);
    __syncthreads();
    if (lane == 0) sSum[wave] = mine;
    __syncthreads();
    u64 z = 0, before = 0;
    for (uint32_t w = 0; w < kWaves; ++w) {
        if (w == wave) before = z;
        z += sSum[w];
    }
    const double ud = u > 0.0f ? min((double)u * 2147483648.0, 2147483647.0) : 0.0;
    bool more;
    const u64 target = share((uint32_t)ud, z, more);
    if (before <= target && target < before + mine) {  // one wave's lanes
        for (uint32_t i0 = lo; i0 < hi; i0 += 64) {
            const u64 w = i0 + lane < hi ? mass(i0 + lane) : 0;
            u64 run = w;
#pragma unroll
            for (uint32_t d = 1; d < 64; d <<= 1) {
                const u64 y = __shfl_up(run, d);
                if (lane >= d) run += y;
            }
            const u64 past = __ballot(before + run > target);
            if (past) {
                if (lane == (uint32_t)__ffsll(past) - 1) *token = (int32_t)(i0 + lane);
                break;
            }
            before += __shfl(run, 63);
        }
    }
}

}  // namespace

// A block per row.
#define SAMPLE(name, T)                                                                                                   \
    POPCORN_KERNEL void __launch_bounds__(1024)                                                                           \
        name(const T::storage *logits, const float *uniforms, const float *temperature, const int32_t *topK, const float *topP, \
             const float *minP, int32_t *tokens, SampleConstants p) {                                                     \
        const uint32_t r = blockIdx.x;                                                                                    \
        sample_row<T>(logits + (uint64_t)r * p.vocab, p.vocab, uniforms[r], p.hasTemperature ? temperature[r] : 1.0f,     \
                      p.hasTopK ? topK[r] : 0, p.hasTopP ? topP[r] : 1.0f, p.hasMinP ? minP[r] : 0.0f, tokens + r);       \
    }

SAMPLE(sample_f32, pk::F32)
SAMPLE(sample_f16, pk::F16)
SAMPLE(sample_bf16, pk::BF16)
