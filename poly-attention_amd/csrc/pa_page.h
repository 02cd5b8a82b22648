// pa_page.h -- the pages of a paged cache as its kernels see them: rows, chunks, tokens and places.
#pragma once

#include "pa_common.h"
#include "pa_draft_partial.h"
#include "pa_launch.h"

namespace pa {

constexpr int kPageThreads = 256;
// workgroups of a grid's first dimension, at most: its threads are counted in 32 bits
constexpr int64_t kPageGroups = (int64_t(1) << 32) / 1024 - 1;

struct PageDev {
    int32_t rows, pages, lg, max_pages;  // lg: log2 of the page size
    int32_t tokens, packed;              // of the step's inputs: per row, or in all
    const int32_t* table;
    const int32_t* counts;
    const int32_t* fresh;
    const int32_t* starts;
};

// A row's chunk: positions [p0, p0 + len) are new, token i is place `start` + i of the inputs.  Whatever the counts
// hold, the positions lie inside the table and the tokens inside the inputs.
struct PageRow {
    int n;      // positions with the chunk's
    int p0;     // the first of them that is new
    int len;    // new tokens
    int start;  // of packed inputs
};
__device__ __forceinline__ int page_count(const PageDev& P, int b) {
    const int n = P.counts[b], cap = P.max_pages << P.lg;
    return n < 0 ? 0 : min(n, cap);
}
__device__ __forceinline__ PageRow page_row(const PageDev& P, int b) {
    PageRow r;
    r.n = page_count(P, b);
    const int want = min(max(P.fresh[b], 0), r.n);
    r.start = P.packed ? P.starts[b] : 0;
    if (r.start < 0 || r.start > P.tokens) r.start = P.tokens;
    r.p0 = r.n - want;
    r.len = min(want, P.tokens - r.start);
    return r;
}

// Place `page place` of position p of row b, in positions of the pool; -1 for a page outside it.
__device__ __forceinline__ int64_t page_place(const PageDev& P, int b, int p) {
    const int id = P.table[(int64_t)b * P.max_pages + (p >> P.lg)];
    return (unsigned)id < (unsigned)P.pages ? ((int64_t)id << P.lg) + (p & ((1 << P.lg) - 1)) : -1;
}

// The row whose packed tokens `tok` belongs to: the last one that starts at or before it, by the whole wave.
__device__ __forceinline__ int page_find(const PageDev& P, int tok, int lane) {
    int lo = 0, n = P.rows;  // starts[lo] <= tok, as starts[0] is 0
    while (n > 1) {
        const int step = (n + 63) >> 6;
        const int r = lo + lane * step;
        const uint64_t below = __ballot(lane * step < n && P.starts[min(r, P.rows)] <= tok);
        // starts do not fall, so the lanes are the first ones; none: a table that was never extended
        const int k = max(__popcll(below) - 1, 0);
        lo += k * step;
        n = min(step, n - k * step);
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

inline int page_lg(int size) {
    int lg = 0;
    while ((1 << lg) < size) ++lg;
    return lg;
}

// PA_OK where a table's description holds together
inline int page_check(const pa_page_table& t) {
    if (t.rows < 1 || t.pages < 1 || t.max_pages < 1 || !t.table || !t.counts || !t.refs || !t.fresh || !t.starts)
        return PA_EINVAL;
    if (t.page_size < 16 || t.page_size > 4096 || (t.page_size & (t.page_size - 1))) return PA_EUNSUPPORTED;
    if (t.rows > PA_MAX_PAGE_ROWS || (int64_t)t.max_pages * t.page_size > (1 << 30) || t.pages > (1 << 30))
        return PA_EUNSUPPORTED;
    return PA_OK;
}

inline PageDev page_dev(const pa_page_table& t, int tokens, int packed) {
    PageDev P;
    P.rows = t.rows;
    P.pages = t.pages;
    P.lg = page_lg(t.page_size);
    P.max_pages = t.max_pages;
    P.tokens = tokens;
    P.packed = packed;
    P.table = t.table;
    P.counts = t.counts;
    P.fresh = t.fresh;
    P.starts = t.starts;
    return P;
}

// the types, head dims and inputs that the calls take
inline bool page_dtype(int d) { return d == PA_F32 || d == PA_F16 || d == PA_BF16; }
inline bool page_dim(int d) { return d >= 8 && d <= 256 && d % 8 == 0 && (d <= 128 || d % 16 == 0); }
inline bool page_rows16(const pa_view& v) {
    const int E = v.dtype == PA_F32 ? 4 : 8;
    return (uintptr_t)v.ptr % 16 == 0 && v.sb % E == 0 && v.sh % E == 0 && v.sn % E == 0;
}
inline DraftRow page_view(const pa_view& v) {
    DraftRow r;
    r.p = static_cast<char*>(v.ptr);
    r.sb = v.sb;
    r.sh = v.sh;
    r.sn = v.sn;
    return r;
}

}  // namespace pa
