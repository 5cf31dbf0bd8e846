// A token's weight in a draw, shared by the kernels of sample.hip and (compiled
// for the host) their test.
#pragma once

#include <math.h>
#include <stdint.h>

#if defined(__HIPCC__)
#define SAMPLE_FN __host__ __device__ inline
#else
#define SAMPLE_FN inline
#endif

namespace pk {

// Coefficients ln(2)^k / k! of 2^f: for |f| <= 1/2 the terms left out are below 2^-47 of it.
struct Exp2Terms {
    double c[12];
    constexpr Exp2Terms() : c() {
        c[0] = 1.0;
        for (int k = 1; k < 12; ++k) c[k] = c[k - 1] * 0.69314718055994530942 / k;
    }
};

// a * b + c of a c that is the same in all lanes, kept in scalar registers (the compiler's own choice adds into c,
// which takes a copy of each constant first).
SAMPLE_FN double fma_uniform(double a, double b, double c) {
#if defined(__HIP_DEVICE_COMPILE__)
    double d;
    asm("v_fma_f64 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "s"(c));
    return d;
#else
    return __builtin_fma(a, b, c);
#endif
}

// log2(e) / temperature; infinite for a temperature of 0, which leaves weight to the highest logit alone.
SAMPLE_FN double sample_rate(float temperature) { return temperature > 0.0f ? 1.4426950408889634074 / (double)temperature : INFINITY; }

// 2^40 exp((v - top) / temperature), rounded to a whole number: at most 0.51 off. What is rounded is off by
// 2^40 times 6.3e-15 of the terms left out, 4 roundings of 2^-53 in the sum, and 2^t |t| <= 0.54 times 3.5 of them in
// the exponent: less than 0.008 in all. 0 for -infinity and NaN.
SAMPLE_FN uint64_t sample_weight(float v, float top, double rate) {
    constexpr Exp2Terms terms;
    const double t = __builtin_fmax(((double)v - (double)top) * rate, -64.0);  // (a NaN is -64 too: weights end at -41)
    const double n = __builtin_rint(t), f = t - n;
    double s = terms.c[11];
#if defined(__clang__)
#pragma unroll
#endif
    for (int k = 10; k >= 0; --k) s = fma_uniform(s, f, terms.c[k]);
    // adding 2^52 rounds to a whole number and leaves it in the low bits
    const double w = __builtin_ldexp(s, (int)n + 40) + 4503599627370496.0;
    uint64_t u;
    __builtin_memcpy(&u, &w, sizeof(u));
    u &= 0xfffffffffffffull;
    return v == top ? (uint64_t)1 << 40 : u;
}

}  // namespace pk
