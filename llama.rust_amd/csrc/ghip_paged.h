// ghip_paged.h -- which rows and keys attention over a paged KV cache deals
// with: index arithmetic alone, the same for the kernels and for a host build.
#pragma once
#include <stdint.h>

#ifdef __HIPCC__
#define PAGED_FN static __device__ __forceinline__
#else
#define PAGED_FN static inline
#endif

// One sequence as its table row describes it, cut to what there is: rows q0 ..
// q0 + nq - 1 of q (those inside q, at most max_q), row i at position pos0 + i.
// Nothing a table holds leads out of q, of dst or of the table: a sequence that
// starts below row 0 has none, and keys past the table are on no page.
struct PagedSeq {
    int q0, nq;
    int64_t pos0;
};
PAGED_FN PagedSeq paged_seq(int q0, int nq, int nkv, int T, int max_q) {
    PagedSeq s;
    s.q0 = q0;
    s.pos0 = (int64_t)nkv - nq;
    int n = nq < max_q ? nq : max_q;
    if (q0 < 0 || q0 >= T || n < 0) n = 0;
    else if (n > T - q0) n = T - q0;
    s.nq = n;
    return s;
}

// The keys that rows at positions p0 .. p1 see between them, as two ranges:
// [0, first) and [lo, hi), first <= lo.  Every key of [lo, hi) is seen by one of
// the rows, and so is every key of [0, first).  window 0: all keys up to a row's
// own.  hi may lie past the table; p1 < 0: nothing.
struct PagedKeys {
    int64_t first, lo, hi;
};
PAGED_FN PagedKeys paged_keys(int64_t p0, int64_t p1, int window, int n_first) {
    PagedKeys k;
    k.hi = p1 + 1 > 0 ? p1 + 1 : 0;
    k.lo = 0;
    if (window && p0 - window + 1 > 0) k.lo = p0 - window + 1;
    if (k.lo > k.hi) k.lo = k.hi;
    k.first = n_first < k.lo ? n_first : k.lo;
    return k;
}
// does the row at position p see key j >= 0?
PAGED_FN bool paged_seen(int64_t p, int64_t j, int window, int n_first) {
    return j <= p && (!window || j > p - window || j < n_first);
}

// n / d for any 32-bit n by a product (Granlund and Montgomery's division by an
// invariant integer); paged_divisor works the factors out on the host.
struct PagedDiv {
    uint32_t mul, sh1, sh2;
};
static inline PagedDiv paged_divisor(uint32_t d) {
    uint32_t l = 0;
    while (l < 32 && (1ull << l) < d) l++;
    PagedDiv r;
    r.mul = (uint32_t)((((1ull << l) - d) << 32) / d + 1);
    r.sh1 = l < 1 ? l : 1;
    r.sh2 = l < 1 ? 0 : l - 1;
    return r;
}
PAGED_FN uint32_t paged_div(uint32_t n, PagedDiv d) {
#ifdef __HIPCC__
    const uint32_t t = __umulhi(d.mul, n);
#else
    const uint32_t t = (uint32_t)(((uint64_t)d.mul * n) >> 32);
#endif
    return (t + ((n - t) >> d.sh1)) >> d.sh2;
}

// The tiles of `kt` keys that a block of rows at positions p0 .. p1 goes through
// in [from, to) of the keys (a pass over the shared prefix: [0, n_shared), one
// over what is a sequence's own: from n_shared on): na of them over [a0, a1),
// which are the keys seen whatever the window, then those over [b0, b1).
struct PagedTiles {
    int a0, a1, b0, b1, na, n;
};
PAGED_FN PagedTiles paged_tiles(int64_t p0, int64_t p1, int window, int n_first, int from, int to, int kt) {
    const PagedKeys k = paged_keys(p0, p1, window, n_first);
    PagedTiles t;
    t.a0 = from;
    t.a1 = k.first < to ? (int)k.first : to;
    if (t.a1 < t.a0) t.a1 = t.a0;
    t.b0 = k.lo > from ? (k.lo < to ? (int)k.lo : to) : from;
    t.b1 = k.hi < to ? (int)k.hi : to;
    if (t.b1 < t.b0) t.b1 = t.b0;
    t.na = (int)(((int64_t)t.a1 - t.a0 + kt - 1) / kt);
    t.n = t.na + (int)(((int64_t)t.b1 - t.b0 + kt - 1) / kt);
    return t;
}
// Split z of `nz` takes tiles [z c, z c + c) of n.
PAGED_FN int paged_share(int n, int nz) { return (int)(((int64_t)n + nz - 1) / nz); }
