// vw_window.cuh -- the pages and tokens that a sliding window with sinks leaves
// visible, shared by the decode, its combine grid and the prefill.
//
// A query at position p sees the keys j <= p with p - j < window or j < sinks.
// For queries at positions p0 .. p1 no key in [sinks, lo), lo = p0 - window + 1,
// is visible to any of them, so the pages between page ceil(sinks/16) and page
// lo/16 are neither resolved nor read: their block-table entries may hold
// anything.  The visited pages are numbered by ordinals 0 .. n-1, the sink pages
// first; page() maps an ordinal to the logical page.  Every visited page holds
// a visible token, so the first page of a running softmax has a finite maximum.
#pragma once
#include "vw_internal.h"

namespace vw {

// Pages of seq_len tokens; unsigned, since seq_len + 15 may not fit 31 bits.  (Callers
// discard the result for lengths below 1.)
__device__ __forceinline__ int pages_of(int seq_len) { return (int)(((uint32_t)seq_len + 15u) >> 4); }

struct PageSpan {
    int n;          // pages visited
    int ns;         // sink pages: ordinals below ns are the logical pages themselves
    int skip;       // pages left out after them
    int lo;         // first position of the window (0: everything is visible)
    int sinks;

    __device__ __forceinline__ int page(int ord) const { return ord < ns ? ord : ord + skip; }
    // rows [a, b) of a logical page that no query sees (a >= b: none)
    __device__ __forceinline__ void hidden(int pg, int& a, int& b) const {
        a = max(0, sinks - pg * kBlockSize);
        b = min(kBlockSize, lo - pg * kBlockSize);
    }
};

// Queries from position `first` on over `np` pages (np >= 1, first < np * 16).
__device__ __forceinline__ PageSpan page_span(int np, int first, uint32_t window, uint32_t sinks) {
    PageSpan s;
    s.lo = max(0, first + 1 - (int)window);
    s.sinks = (int)sinks;
    s.ns = (min(s.sinks, s.lo) + kBlockSize - 1) / kBlockSize;
    s.skip = max(0, s.lo / kBlockSize - s.ns);
    s.n = np - s.skip;
    return s;
}

// A decode's span: seq_len tokens, the query at the last one.  A seq_len beyond
// the block-table row (flagged by the decode) counts as the row's last token.
__device__ __forceinline__ PageSpan decode_span(int seq_len, int bt_stride, uint32_t window, uint32_t sinks) {
    const int np = min(pages_of(seq_len), bt_stride);
    return page_span(np, min(seq_len - 1, (np - 1) * kBlockSize + kBlockSize - 1), window, sinks);
}

}  // namespace vw
