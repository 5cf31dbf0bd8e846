// Index arithmetic of the paged cache, shared by its kernels and (compiled
// for the host) their tests. Lengths and tables come from device memory and
// are not checked before a launch, so every number read is brought into range
// here: no value of theirs leads outside the tensors.
#pragma once

#include <stdint.h>

#include "popcorn_kernel_types.h"

#if defined(__HIPCC__)
#define PAGED_FN __host__ __device__ inline
#else
#define PAGED_FN inline
#endif

namespace pk {

PAGED_FN int32_t paged_min(int32_t a, int32_t b) { return a < b ? a : b; }
PAGED_FN int32_t paged_max(int32_t a, int32_t b) { return a > b ? a : b; }

// One request of a paged attention call: its new tokens are rows start ..
// start + n - 1, token i at position pos0 + i (negative where the request has
// fewer keys than new tokens), and its first `keys` keys lie in its pages.
struct PagedRequest {
    int32_t start, n, pos0, keys;
};

PAGED_FN PagedRequest paged_request(int32_t first, int32_t next, int32_t keyLen, const PagedAttentionConstants &p) {
    PagedRequest r;
    r.start = paged_min(paged_max(first, 0), (int32_t)p.T);
    r.n = paged_min(paged_max(next, r.start), (int32_t)p.T) - r.start;
    const int32_t len = paged_max(keyLen, 0);
    const uint64_t room = (uint64_t)p.columns * p.pageSize;
    r.pos0 = len - r.n;
    r.keys = (uint64_t)len < room ? len : (int32_t)room;
    return r;
}

// Keys that some of the positions first .. last see: [0, sinkEnd) and [lo, hi).
struct PagedSpan {
    int32_t sinkEnd, lo, hi;
};

PAGED_FN PagedSpan paged_span(int32_t first, int32_t last, int32_t keys, const PagedAttentionConstants &p) {
    PagedSpan s;
    s.hi = p.maskKind == 2u || last >= keys ? keys : paged_max(last + 1, 0);
    s.lo = 0;
    s.sinkEnd = 0;
    if (p.maskKind == 1u) {
        const int64_t lo = (int64_t)first - p.slidingWindow + 1;
        s.lo = lo <= 0 ? 0 : lo < s.hi ? (int32_t)lo : s.hi;
        s.sinkEnd = p.sinks < (uint32_t)s.lo ? (int32_t)p.sinks : s.lo;
    }
    return s;
}

PAGED_FN bool paged_sees(int32_t pos, int32_t key, const PagedAttentionConstants &p) {
    return (p.maskKind == 2u) | ((key <= pos) & ((p.maskKind == 0u) | ((int64_t)pos - key < p.slidingWindow) | ((uint32_t)key < p.sinks)));
}

}  // namespace pk
