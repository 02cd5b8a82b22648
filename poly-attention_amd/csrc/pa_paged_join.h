// pa_paged_join.h -- the end of a level's tiles of many rows: the join of their units, and rows that are formed again.
#pragma once

#include "pa_paged.h"

namespace pa {

// A query row position by position in fp32, by the workgroup: its waves take 64 positions at a time in turn, a lane's
// score each, then a lane's features.  A position that the row does not see takes no part.
struct SlowRow {
    float top[4], sum[4], y[4][256];
};
template <typename T>
__device__ __forceinline__ void paged_slow(const PagedDev& P, const PagedUnit& U, int hk, int r, SlowRow& S) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const T* const q = paged_query<T>(P, U, hk, r);
    const int see = U.row.p0 + r / P.rep + 1;
    float top = -INFINITY, sum = 0.f, y[4] = {0.f, 0.f, 0.f, 0.f};  // features lane + 64 i
    for (int j0 = 64 * wave; j0 < see; j0 += 256) {
        const int64_t place = page_place(P.p, U.b, min(j0 + lane, see - 1));
        int64_t at = -1;
        float s = 0.f;
        if (place >= 0) {
            at = paged_base(P, (int)(place >> P.p.lg), hk) + (place & ((1 << P.p.lg) - 1));
            const T* const k = reinterpret_cast<const T*>(P.keys) + at * P.dim;
            if (q)
                for (int d = 0; d < P.dim; ++d) s = fmaf(to_f(q[d]), to_f(k[d]), s);
        }
        s *= P.scale;
        if (P.softclamp > 0.f) s = P.softclamp * tanhf(s / P.softclamp);
        if (P.bias && at >= 0) s += P.bias[at];
        s = j0 + lane < see ? s * kLog2e : -INFINITY;
        float t = fmaxf(top, s);
        for (int off = 32; off > 0; off >>= 1) t = fmaxf(t, __shfl_xor(t, off));
        const float f = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - t);
        top = t;
        const float w = s == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s - t);
        float add = w;
        for (int off = 32; off > 0; off >>= 1) add += __shfl_xor(add, off);
        sum = sum * f + add;
        for (int i = 0; i < 4; ++i) y[i] *= f;
        for (int k = 0; k < min(64, see - j0); ++k) {
            const float wk = __shfl(w, k);
            const int64_t ak = __shfl(at, k);
            if (wk == 0.f || ak < 0) continue;
            const T* const v = reinterpret_cast<const T*>(P.values) + ak * P.dim;
            for (int i = 0; i < 4; ++i)
                if (lane + 64 * i < P.dim) y[i] = fmaf(wk, to_f(v[lane + 64 * i]), y[i]);
        }
    }
    __syncthreads();  // S has been read
    if (lane == 0) {
        S.top[wave] = top;
        S.sum[wave] = sum;
    }
    for (int i = 0; i < 4; ++i) S.y[wave][lane + 64 * i] = y[i];
    __syncthreads();
    if (wave) return;
    // a maximum that is no number is passed over above, and shows in the sums, also of a wave that has no other
    const float t = fmaxf(fmaxf(S.top[0], S.top[1]), fmaxf(S.top[2], S.top[3]));
    sum = 0.f;
    for (int i = 0; i < 4; ++i) y[i] = 0.f;
    for (int w = 0; w < 4; ++w) {
        if (64 * w >= see) break;  // had no position
        const float f = S.top[w] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(S.top[w] - t);
        sum += S.sum[w] * f;
        if (f == 0.f) continue;
        for (int i = 0; i < 4; ++i) y[i] += S.y[w][lane + 64 * i] * f;
    }
    const PagedTo to = paged_to<T>(P, U, hk, r);
    if (lane == 0 && to.lse) *to.lse = (t + log2f(sum)) * kLn2;
    for (int i = 0; i < 4; ++i)
        if (to.out && lane + 64 * i < P.dim) {
            float x = y[i] / sum;
            if (to.mul) x *= to_f(reinterpret_cast<const T*>(to.mul)[lane + 64 * i]);
            reinterpret_cast<T*>(to.out)[lane + 64 * i] = from_f<T>(x);
        }
}

// Blocks of rows of tiles that were split, a workgroup each.
template <typename T>
__device__ __forceinline__ void paged_join_tiles(const PagedDev& P, int group, int groups, float (*s_red)[6], SlowRow& S) {
    for (int64_t item = group;; item += groups) {
        const int hk = (int)(item % P.kv_heads);
        PagedUnit U;
        if (!paged_find<kRows>(P, item / P.kv_heads, threadIdx.x & 63, U)) return;
        if (!paged_recorded(P, U)) continue;
        const int n = min(1 << P.lgr, U.rows - U.at);
        const int live = min(U.splits, (paged_keys(P, U) + U.size * kPagedChunk - 1) / (U.size * kPagedChunk));
        if (__syncthreads_or(paged_join<T, 1, false>(P, U, hk, 0, 1, live, true, U.at, n, P.lgr, s_red)))
            for (int r = U.at; r < U.at + n; ++r) paged_slow<T>(P, U, hk, r, S);
    }
}

// The tiles of one unit that asked to be formed again.
template <typename T>
__device__ __forceinline__ void paged_again(const PagedDev& P, int group, int groups, SlowRow& S) {
    const int64_t all = (int64_t)P.units * P.kv_heads;
    for (int64_t x = group; x < all; x += groups) {
        if (reinterpret_cast<const uint64_t*>(P.flags)[x] == 0) continue;
        PagedUnit U;
        if (!paged_find<kUnits>(P, x / P.kv_heads, threadIdx.x & 63, U)) continue;
        for (int r = U.tile * P.tile; r < min((U.tile + 1) * P.tile, U.rows); ++r)
            paged_slow<T>(P, U, (int)(x % P.kv_heads), r, S);
    }
}

}  // namespace pa
