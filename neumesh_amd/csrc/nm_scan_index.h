// nm_scan_index.h -- host + device: which rows belong to which sequence in packed recurrences (nm_scan.hip).  The borders `cu` are device values that no
// host code reads, so every index made from them is bounded HERE, whatever they hold.
#pragma once

#ifndef NM_HD
#ifdef __HIPCC__
#define NM_HD __host__ __device__ __forceinline__
#else
#define NM_HD static inline
#endif
#endif

// the sequence of a row: the last one that starts at or before it, -1 before the first and behind the last.  In [-1, S).
NM_HD int nm_scan_sequence(const int* cu, long long S, long long row) {
    long long lo = 0, hi = S + 1;        // first index with cu > row
    while (lo < hi) {
        const long long mid = (lo + hi) >> 1;
        if (cu[mid] > row) hi = mid;
        else lo = mid + 1;
    }
    return lo >= 1 && lo <= S ? (int)(lo - 1) : -1;
}

// Of a range [c0, c1) of steps (step i is row i, or row L - 1 - i): where a reduction from the left may start, given the sequence q of the range's last
// step: at that sequence's first step.  In [c0, c1).
NM_HD long long nm_scan_reduce_from(const int* cu, int q, int reverse, long long L, long long c0, long long c1) {
    const long long s = q < 0 ? c1 - 1 : reverse ? L - cu[q + 1] : (long long)cu[q];
    return s < c0 ? c0 : s >= c1 ? c1 - 1 : s;
}

// ... and where a reduction from the right may end, given the sequence q of the range's first step: at that sequence's last step.  In [c0, c1).
NM_HD long long nm_scan_reduce_to(const int* cu, int q, int reverse, long long L, long long c0, long long c1) {
    const long long e = q < 0 ? c0 : reverse ? L - 1 - cu[q] : cu[q + 1] - 1LL;
    return e < c0 ? c0 : e >= c1 ? c1 - 1 : e;
}
