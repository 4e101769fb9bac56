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
