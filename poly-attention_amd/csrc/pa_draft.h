// pa_draft.h -- attention of drafted tokens over the poly KV cache: what its kernels share.
//
// A step looks at T nodes per batch row (T <= 64) behind n_b cached positions.  A level's query rows
// of one key head are R = T * G (G query heads per key head: 1 below the final level), and all of
// them read the same keys and values, so the scores and the weighted sums are matrix products with
// R rows: the cached positions are read from memory once for all nodes and heads of a group.
//
// Two launches.  k_draft_partial covers what does not depend on the step's results, so all levels run
// at once: the cached positions, split into units (chunks of one size in all rows, whose number
// follows the counts on the device), each leaving (max, sum, weighted values), and the scores of
// the drafted tokens among themselves.  k_draft_combine walks the levels, deepest first: it joins the
// units and the tree part, where the deeper level's result is the bias and the value.  Values enter
// linearly, column by column, and the scores need no values: a workgroup of the combine owns some
// columns of the head and repeats the (few) weights, so no workgroup waits for another.
#pragma once

#include <type_traits>

#include "pa_common.h"
#include "pa_launch.h"

namespace pa {

constexpr int kDraftThreads = 256;
constexpr int kDraftChunk = 128;  // a unit covers a multiple of this many positions (4 waves x 32)
// tickets of different rows lie on cache lines of their own: atomics on one line follow one another (432 of
// them on one line took 4 us)
constexpr int kTicketStride = PA_TICKET_STRIDE;
// A row's weights are exp2(score - m), log2 units, with m its running maximum or less: m is raised where a score passes
// it by more than draft_tau, to draft_lift below that score.  fp16's smallest number is 2^-24: against a largest
// weight of 1 those below 2^-25 vanish, of which a long cache holds as many as to matter (20000 of 2^-25.5 beside
// one of 1: 0.04%, times their values).  Against a largest weight of 2^7 to 2^15 those below 2^-32 do.
template <typename T> __device__ constexpr float draft_lift() { return std::is_same_v<T, f16> ? 7.f : 0.f; }
template <typename T> __device__ constexpr float draft_tau() { return std::is_same_v<T, f16> ? 15.f : 8.f; }

struct DraftRow {  // a [B, h, n, dim] array: base and element strides
    char* p;
    int64_t sb, sh, sn;
    template <typename T> __device__ __forceinline__ T* at(int b, int h) const {
        return reinterpret_cast<T*>(p) + (int64_t)b * sb + (int64_t)h * sh;
    }
};

// What the two launches share.
struct DraftCommon {
    int32_t batch, kv_heads, T, dim, order, capacity;
    int32_t rec_rows;    // rows of a unit's record, all levels
    int32_t t16;         // T in whole sixteens
    int32_t target;      // units aimed at over the whole batch ...
    int32_t target_min;  // ... or this many, where units are smaller than
    int32_t least;       // this many chunks
    const int32_t* counts;
    const int32_t* parents;
    int64_t parents_stride;
    float* ws_o;   // [unit][kv head][rec_rows][dim]
    float2* ws_s;  // [unit][kv head][rec_rows]: running maximum (log2 units) and sum
    int64_t none;  // the record behind those of the units: maximum -inf, sum and values 0
    float* ws_t;   // [row][kv head][rec_rows][t16]: scores of the tree without biases (log2 units), -inf
                   // where a node does not see another
    int4* ws_u;    // [row]: the row's first unit, its units, and which of its nodes are there (64 bits)
};

struct DraftLevelDev {
    DraftRow q, k, v, bias, m, dk;
    int32_t rows, rep, row0;  // rows per key head, heads per key head, first row in a unit's record
};
struct DraftDev : DraftCommon {
    int32_t row_blocks;  // blocks of rows per key head (of the level that has most)
    float scale, softclamp;
    DraftLevelDev L[PA_MAX_ORDER];
};

struct DraftJoinLevel {
    DraftRow dv, out;
    float* lse;
    int64_t lse_sb, lse_sh;
};
struct DraftJoin : DraftCommon {
    int32_t lgcols;  // log2 of the columns per workgroup
    int32_t rep;     // heads per key head at the final level
    DraftJoinLevel L[PA_MAX_ORDER];
};

__device__ __forceinline__ int draft_count(const DraftCommon& P, int b) {
    const int n = P.counts[b];
    return n < 0 ? 0 : (n > P.capacity ? P.capacity : n);
}
__device__ __forceinline__ int draft_chunks(const DraftCommon& P, int b) {
    return (int)(((unsigned)draft_count(P, b) + kDraftChunk - 1) / kDraftChunk);
}

// How the cached positions are split: units of at most so many chunks in all rows that there are about
// `target` of them (at most target + batch), counted on the device; a row's units are of one size.
struct DraftUnits {
    int size;    // chunks per unit of row b
    int b;       // the row of the unit asked for
    int place;   // its place among the row's units
    int first;   // the first unit of row b
    int number;  // the units of row b
};

__device__ __forceinline__ unsigned draft_ceil(unsigned n, unsigned d) { return d == 1 ? n : (n + d - 1) / d; }

// chunks per unit for a batch of `total` chunks
__device__ __forceinline__ int draft_unit_size(const DraftCommon& P, unsigned total) {
    const unsigned many = draft_ceil(total, P.target), few = draft_ceil(total, P.target_min);
    return max(max(1u, many), min(few, (unsigned)P.least));
}

// The units of row `want` (want >= 0), or the row of unit u (want < 0; false past the last unit).
// The whole wave takes part.  One row needs no sums.
__device__ __forceinline__ bool draft_units(const DraftCommon& P, int want, int u, int lane, DraftUnits& r) {
    if (P.batch == 1) {
        const unsigned n = draft_chunks(P, 0);
        r.size = draft_unit_size(P, n);
        r.b = 0;
        r.first = 0;
        r.place = u;
        r.number = draft_ceil(n, r.size);
        if (r.number > 0) r.size = draft_ceil(n, r.number);
        return want >= 0 || u < r.number;
    }
    unsigned total = 0, n0 = 0;  // n0: this lane's row of the first 64
    for (int b = lane; b < P.batch; b += 64) {
        const unsigned n = draft_chunks(P, b);
        total += n;
        if (b < 64) n0 = n;
    }
    for (int off = 32; off > 0; off >>= 1) total += __shfl_xor(total, off);
    r.size = draft_unit_size(P, total);
    int before = 0;
    for (int r0 = 0; r0 < P.batch; r0 += 64) {
        const int row = r0 + lane;
        const unsigned n = r0 == 0 ? n0 : row < P.batch ? draft_chunks(P, row) : 0;
        const int mine = draft_ceil(n, r.size);
        int incl = mine;
        for (int off = 1; off < 64; off <<= 1) {
            const int y = __shfl_up(incl, off);
            if (lane >= off) incl += y;
        }
        const uint64_t past = want >= 0 ? (want < r0 + 64 ? 1ull << (want - r0) : 0ull)
                                        : __ballot(before + incl > u);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            r.b = __builtin_amdgcn_readfirstlane(r0 + l);
            r.number = __builtin_amdgcn_readlane(mine, l);
            r.first = before + __builtin_amdgcn_readlane(incl, l) - r.number;
            r.place = u - r.first;
            if (r.number > 0) r.size = draft_ceil(__builtin_amdgcn_readlane(n, l), r.number);
            return true;
        }
        before += __builtin_amdgcn_readlane(incl, 63);
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

// The record of no unit, by one wave: the join reads it where it has fewer units than loads.  A unit's record in its
// place would do for finite values, but 0 times an infinite one is no 0.
__device__ __forceinline__ void draft_none(const DraftCommon& P, int lane) {
    for (int d = lane; d < P.dim; d += 64) P.ws_o[P.none * P.dim + d] = 0.f;
    if (lane == 0) P.ws_s[P.none] = make_float2(-INFINITY, 0.f);
}

template <typename T> void launch_draft_partial(const DraftDev& P, int units, int tiles, bool vmul, hipStream_t s);
// in source files of their own
extern template void launch_draft_partial<bf16>(const DraftDev& P, int units, int tiles, bool vmul, hipStream_t s);
extern template void launch_draft_partial<f16>(const DraftDev& P, int units, int tiles, bool vmul, hipStream_t s);
extern template void launch_draft_partial<float>(const DraftDev& P, int units, int tiles, bool vmul, hipStream_t s);
// the same for 16-bit types where draft_wide says so
template <typename T> void launch_draft_wide(const DraftDev& P, int units, bool vmul, hipStream_t s);
extern template void launch_draft_wide<bf16>(const DraftDev& P, int units, bool vmul, hipStream_t s);
extern template void launch_draft_wide<f16>(const DraftDev& P, int units, bool vmul, hipStream_t s);
// its waves, and their 16-row tiles: what two waves per SIMD have registers for
constexpr int kDraftWideWaves = 4;
// Whether a group of `rows` rows at the final level goes to k_draft_wide (D: the padded head dim).  Both, in
// us, behind cold caches: 40 rows of 128, 8 x 4096 positions 87 here, 73 there, 64 rows 94 and 76, 48 rows 20 x 500
// 42 and 40; 64 rows of 64, 8 x 4096 61 and 53, 48 rows 20 x 500 34 and 29.  With a middle level (order 3, 8 x 2048)
// 64 rows of 64 50 and 61, 128 rows 66 and 68; 64 rows of 128 102 and 100.
constexpr bool draft_wide(int D, bool f32, bool middle, int rows) {
    return !f32 && D <= 128 && rows > (D == 64 && middle ? 64 : 32);
}
constexpr int draft_wide_tiles(int D) { return D <= 64 ? 4 : 2; }
// Waves per SIMD that the first launch's registers are held to, with RT tiles of 16 rows and, for a middle
// level, a third stream: two where they fit, which hide each other's waits and ends.
constexpr int draft_waves(int D, int RT, bool middle) {
    return D <= 128 && D * RT <= (middle && D == 128 ? 128 : 256) ? 2 : 1;
}
// 16-row tiles of a workgroup of that kernel, at most: what a wave's accumulators leave room for, and 16-bit
// blocks of more rows are the other kernel's (draft_wide); `middle` with a middle level's third stream
template <typename T> constexpr int draft_row_tiles(int D, bool middle) {
    return D > 128 ? 1 : sizeof(T) == 2 && D == 64 && middle ? 4 : 2;
}

}  // namespace pa
