// pa_draft.h -- attention of drafted tokens over the poly KV cache: what its kernels share.
//
// A step looks at T nodes per batch row (T <= 64) behind n_b cached positions.  A level's query rows
// of one key head are R = T * G (G query heads per key head: 1 below the final level), and all of
// them read the same keys and values, so the scores and the weighted sums are matrix products with
// R rows: the cached positions are read from memory once for all nodes and heads of a group.
//
// Two launches.  k_draft_partial covers the cached positions of every level: they do not depend on the
// step's results, so all levels run at once, split over positions ("units": chunks of one size in
// all rows, whose number follows the counts on the device); it leaves (max, sum, weighted values)
// per unit.  k_draft_combine walks the levels, deepest first: it joins the units and adds the tree
// part, where the deeper level's result is the bias and the value.  Values enter linearly, column by
// column, and the scores need no values: a workgroup of the combine owns some columns of the head
// and repeats the (small) scores of the tree, so no workgroup waits for another.
#pragma once

#include "pa_common.h"
#include "pa_launch.h"

namespace pa {

constexpr int kDraftThreads = 256;
constexpr int kDraftChunk = 128;  // a unit covers a multiple of this many positions (4 waves x 32)
constexpr float kDraftTau = 8.f;  // lazy-rescale headroom of the running maximum (log2 units)

struct DraftRow {  // a [B, h, n, dim] array: base and element strides
    char* p;
    int64_t sb, sh, sn;
    template <typename T> __device__ __forceinline__ T* at(int b, int h) const {
        return reinterpret_cast<T*>(p) + (int64_t)b * sb + (int64_t)h * sh;
    }
};

struct DraftLevelDev {
    DraftRow k, v, m, bias, q, dk, dv, out, lse;
    int32_t rows, rep, row0;  // rows per key head, heads per key head, first row in a unit's record
};

struct DraftDev {
    int32_t batch, kv_heads, T, dim, order, capacity;
    int32_t target;      // units aimed at over the whole batch
    int32_t row_blocks;  // partial: blocks of rows per key head (of the level that has most)
    int32_t rec_rows;    // rows of a unit's record, all levels
    int32_t cols;        // combine: columns per workgroup
    float scale, softclamp;
    const int32_t* counts;
    const int32_t* parents;
    int64_t parents_stride;
    float* ws_o;   // [unit][kv head][rec_rows][dim]
    float2* ws_s;  // [unit][kv head][rec_rows]: running maximum (log2 units) and sum
    DraftLevelDev L[PA_MAX_ORDER];
};

__device__ __forceinline__ int draft_count(const DraftDev& P, int b) {
    const int n = P.counts[b];
    return n < 0 ? 0 : (n > P.capacity ? P.capacity : n);
}

// Positions per unit: the batch's positions over the units aimed at, in whole kDraftChunk.  The sum
// of ceil(n_b / size) is then at most target + batch.
__device__ __forceinline__ int64_t draft_unit_size(const DraftDev& P, int lane) {
    int64_t total = 0;
    for (int b = lane; b < P.batch; b += 64) total += draft_count(P, b);
    for (int off = 32; off > 0; off >>= 1) total += __shfl_xor(total, off);
    const int64_t c = (total + P.target - 1) / P.target;
    const int64_t size = (c + kDraftChunk - 1) / kDraftChunk * kDraftChunk;
    return size > 0 ? size : kDraftChunk;
}

// number of units of the rows before b (the whole wave takes part)
__device__ __forceinline__ int draft_first_unit(const DraftDev& P, int64_t size, int b, int lane) {
    int sum = 0;
    for (int r = lane; r < b; r += 64) sum += (int)((draft_count(P, r) + size - 1) / size);
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
    return sum;
}

// the row of unit u and its place among that row's units; false past the last unit
__device__ __forceinline__ bool draft_find_unit(const DraftDev& P, int64_t size, int u, int lane, int& b,
                                                int& place) {
    int before = 0;
    for (int r0 = 0; r0 < P.batch; r0 += 64) {
        const int r = r0 + lane;
        const int mine = r < P.batch ? (int)((draft_count(P, r) + size - 1) / size) : 0;
        int incl = mine;
        for (int off = 1; off < 64; off <<= 1) {
            const int y = __shfl_up(incl, off);
            if (lane >= off) incl += y;
        }
        const uint64_t past = __ballot(before + incl > u);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            b = r0 + l;
            place = u - (before + __shfl(incl, l) - __shfl(mine, l));
            return true;
        }
        before += __shfl(incl, 63);
    }
    return false;
}

// Lane t's ancestors and itself as a bit mask, 0 for an absent node (and lanes past T): pointer
// doubling, six steps for up to 64 nodes.  Every value of a parent is safe.
__device__ __forceinline__ uint64_t draft_ancestors(const int32_t* parents, int T, int lane) {
    const int p = lane < T ? (parents ? parents[lane] : lane - 1) : -2;
    const bool inner = p >= 0 && p < lane;
    int dead = (inner || p == -1) ? 0 : 1;
    int up = inner ? p : lane;
    uint32_t lo = lane < 32 ? 1u << lane : 0u, hi = lane < 32 ? 0u : 1u << (lane - 32);
    for (int s = 0; s < 6; ++s) {
        const uint32_t l2 = __shfl(lo, up), h2 = __shfl(hi, up);
        const int d2 = __shfl(dead, up), u2 = __shfl(up, up);
        lo |= l2;
        hi |= h2;
        dead |= d2;
        up = u2;
    }
    return dead ? 0ull : ((uint64_t)hi << 32) | lo;
}

template <typename T> void launch_draft_partial(const DraftDev& P, int units, bool vmul, hipStream_t s);
// in source files of their own
extern template void launch_draft_partial<bf16>(const DraftDev& P, int units, bool vmul, hipStream_t s);
extern template void launch_draft_partial<f16>(const DraftDev& P, int units, bool vmul, hipStream_t s);
extern template void launch_draft_partial<float>(const DraftDev& P, int units, bool vmul, hipStream_t s);
template <typename T> constexpr int draft_row_tiles(int D) {
    // 16-row tiles that a wave's accumulators hold
    return D > 128 ? 1 : sizeof(T) == 4 ? 2 : 4;
}

}  // namespace pa
