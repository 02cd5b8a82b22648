// pa_paged.h -- attention of chunks of new tokens over a paged cache: what its kernels share.
//
// A level's query rows of one key head are its new tokens, at the final level times the query heads of
// the group: row r of a chunk is token r / rep, head r % rep, so that a tile of rows covers few positions
// and its causal ends lie together.  A tile's keys are the row's positions up to its last token; they are
// split into units of `size` chunks of 128 positions where there are few tiles.  The rows' counts are known
// on the device only: every workgroup finds its unit from them (a scan over the rows by a wave), and the
// grid is the most units there can be (one without a unit is gone after 2 us; a launch of such 4.7).  A tile of one unit
// is finished where it is computed; the others leave records (maximum, sum, weighted values), which few rows' last unit
// joins, and workgroups of the next launch those of many rows: a workgroup reads some 25 GB/s, as each CU does that has work of its own,
// so 256 rows of 8 units took 20 us in the last unit and take 9 in a launch of their own, 28 rows of 9 units 10.
// The levels follow one another, as each reads what the one below left in the cache.
#pragma once

#include "pa_page.h"

namespace pa {

constexpr int kPagedChunk = 128;
constexpr int kPagedMost = (1 << 30) / kPagedChunk;  // chunks of a row, at most

struct PagedDev {
    PageDev p;
    int32_t kv_heads, dim, rep;
    int32_t last;              // the final level: queries from q, results to out
    int32_t over, most;        // rows of a chunk, more than `over` and at most `most`, that a launch takes
    int32_t tile;              // rows of its tiles
    int32_t target;            // units aimed at over all rows ...
    int32_t target_min, least; // ... or this many, where units are of at most so many chunks
    int32_t fewest;            // chunks of a unit, at least
    int64_t recs;              // records there are
    float scale, softclamp;
    SoftClampDev sc;           // of the logits
    DraftRow q, out, vmul;     // of the inputs; vmul: the next level's projected values, where it is a middle one
    const char* keys;
    const char* values;
    const float* bias;         // the logsumexps of the level below, or null
    const char* queries;       // not at the final level: the next level's keys, new tokens' queries
    char* next;                // the next level's values
    float* lses;
    float* ws_o;               // [record][kv head][tile][dim]
    float2* ws_s;              // [record][kv head][tile]: maximum (log2 units) and sum
    uint8_t* flags;            // [unit][kv head][8]: its waves'
    int32_t* tickets;          // [record][kv head][kTicketStride], 0 between launches
    int32_t units;             // at most
    int32_t lgr;               // log2 of the rows that a workgroup of k_paged_join takes at once
};

__device__ __forceinline__ int64_t paged_base(const PagedDev& P, int id, int hk) {  // in positions
    return ((int64_t)id * P.kv_heads + hk) << P.p.lg;
}

struct PagedUnit {
    PageRow row;
    int b, rows;         // the batch row, its query rows per key head
    int tiles, tile;     // of the row, and the one asked for
    int splits, split;   // units of a tile, and the one asked for
    int size;            // chunks of the row's units
    int rec;             // the record of the tile's first unit (splits > 1)
    int at;              // what was asked for, from the row's first (kRows: its first row)
};

// Chunks per unit for `tiles` tiles of `total` chunks together: P.target units in all, or P.target_min where
// those are of at most P.least chunks.  Each tile's last unit is half one on
// average: there are total / size + tiles / 2 or so.
__device__ __forceinline__ int paged_size(const PagedDev& P, uint64_t total, int tiles) {
    auto chunks = [&](int target) __attribute__((always_inline)) -> uint32_t {
        const uint32_t aim = max(target - tiles / 2, target / 2 + 1);
        const uint64_t n = total >> 31 ? (total + aim - 1) / aim : (uint64_t)(((uint32_t)total + aim - 1) / aim);
        return (uint32_t)min(n, (uint64_t)kPagedMost);
    };
    return (int)max(max(chunks(P.target), min(chunks(P.target_min), (uint32_t)P.least)), (uint32_t)P.fewest);
}

// sums of the lanes up to each, whole waves
__device__ __forceinline__ int paged_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // rows of 16 lanes: shifted by 1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // a row's last into the next row
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // the second row's into the upper half
    return x;
}

// One row's tiles and chunks, 0 for a row that the launch does not take.
__device__ __forceinline__ void paged_tiles(const PagedDev& P, const PageRow& r, int& rows, int& tiles, int& chunks) {
    rows = r.len * P.rep;
    tiles = rows > P.over && rows <= P.most ? (rows + P.tile - 1) / P.tile : 0;
    chunks = (r.n + kPagedChunk - 1) / kPagedChunk;
}

// What a row has of the things that are counted: kUnits, its units, or (kRows) blocks of 2^P.lgr query rows of tiles that
// are to be joined.
enum { kUnits, kRows };

// Finds unit (or block of rows) `want` over all rows of the batch, by the whole wave; false past the last one.  What it finds
// is held in scalar registers, so that the branches and loops over it are scalar ones.
template <int WHAT>
__device__ __forceinline__ bool paged_find(const PagedDev& P, int want, int lane, PagedUnit& U) {
    uint64_t total = 0;
    int all_tiles = 0;
    PageRow r0;
    int rows0 = 0, tiles0 = 0, chunks0 = 0;  // this lane's row of the first 64
    for (int b = lane; b < P.p.rows; b += 64) {
        const PageRow r = page_row(P.p, b);
        int rows, tiles, chunks;
        paged_tiles(P, r, rows, tiles, chunks);
        total += (uint64_t)tiles * chunks;
        all_tiles += tiles;
        if (b < 64) {
            r0 = r;
            rows0 = rows;
            tiles0 = tiles;
            chunks0 = chunks;
        }
    }
    const int all = __builtin_amdgcn_readlane(paged_scan(all_tiles), 63);
    if (!__any(total >> 25 != 0)) {  // the sum is below 2^31
        total = (uint32_t)__builtin_amdgcn_readlane(paged_scan((int)total), 63);
    } else {
        for (int off = 32; off > 0; off >>= 1) total += __shfl_xor((unsigned long long)total, off);
        total = ((uint64_t)__builtin_amdgcn_readfirstlane((int)(total >> 32)) << 32) | (uint32_t)__builtin_amdgcn_readfirstlane((int)total);
    }
    U.size = __builtin_amdgcn_readfirstlane(paged_size(P, total, all));
    int before = 0, recs = 0;  // units are at most the grid's, and blocks of rows fewer than memory holds outputs of
    for (int b0 = 0; b0 < P.p.rows; b0 += 64) {
        const int b = b0 + lane;
        PageRow r = r0;
        int rows = rows0, tiles = tiles0, chunks = chunks0;
        if (b0 > 0) {
            tiles = 0;
            chunks = 0;
            rows = 0;
            if (b < P.p.rows) {
                r = page_row(P.p, b);
                paged_tiles(P, r, rows, tiles, chunks);
            }
        }
        const int splits = (int)(((unsigned)chunks + U.size - 1) / U.size);
        const int units = tiles * splits, rec = splits > 1 ? units : 0;
        const int mine = WHAT == kUnits ? units : splits > 1 && tiles > 0 ? (rows + (1 << P.lgr) - 1) >> P.lgr : 0;
        const int incl = paged_scan(mine), incl_rec = paged_scan(rec);
        const uint64_t past = __ballot(before + incl > want);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            U.b = __builtin_amdgcn_readfirstlane(b0 + l);
            U.row.n = __builtin_amdgcn_readlane(r.n, l);
            U.row.p0 = __builtin_amdgcn_readlane(r.p0, l);
            U.row.len = __builtin_amdgcn_readlane(r.len, l);
            U.row.start = __builtin_amdgcn_readlane(r.start, l);
            U.rows = __builtin_amdgcn_readlane(rows, l);
            U.tiles = __builtin_amdgcn_readlane(tiles, l);
            U.splits = __builtin_amdgcn_readlane(splits, l);
            // the row's units of one size
            U.size = __builtin_amdgcn_readfirstlane((int)(((unsigned)__builtin_amdgcn_readlane(chunks, l) + U.splits - 1) / U.splits));
            U.rec = recs + __builtin_amdgcn_readlane(incl_rec - rec, l);
            U.at = want - before - __builtin_amdgcn_readlane(incl - mine, l);
            if (WHAT == kUnits) {
                // the last tiles, which have most keys, first
                const int t = __builtin_amdgcn_readfirstlane(U.at / U.splits);
                U.split = U.at - t * U.splits;
                U.tile = U.tiles - 1 - t;
            } else {
                U.at <<= P.lgr;  // the first of the rows
                U.tile = __builtin_amdgcn_readfirstlane(U.at / P.tile);
                U.split = 0;
            }
            U.rec += U.tile * U.splits;
            return true;
        }
        before += __builtin_amdgcn_readlane(incl, 63);
        recs += __builtin_amdgcn_readlane(incl_rec, 63);
    }
    return false;
}

// the positions that a tile's last token sees
__device__ __forceinline__ int paged_keys(const PagedDev& P, const PagedUnit& U) {
    return U.row.p0 + __builtin_amdgcn_readfirstlane((min((U.tile + 1) * P.tile, U.rows) - 1) / P.rep) + 1;
}
// whether there is a record for each of the tile's units: there are as many as there can be
__device__ __forceinline__ bool paged_recorded(const PagedDev& P, const PagedUnit& U) {
    return U.rec >= 0 && (int64_t)U.rec + U.splits <= P.recs;
}

// Where a query row's results go.
struct PagedTo {
    char* out;        // its features
    const char* mul;  // or null
    float* lse;       // or null
};
template <typename T>
__device__ __forceinline__ PagedTo paged_to(const PagedDev& P, const PagedUnit& U, int hk, int r) {
    PagedTo to = {nullptr, nullptr, nullptr};
    const int i = r / P.rep, src_b = P.p.packed ? 0 : U.b, tok = U.row.start + i;
    if (P.last) {
        to.out = reinterpret_cast<char*>(P.out.at<T>(src_b, hk * P.rep + r - i * P.rep) + (int64_t)tok * P.out.sn);
        return to;
    }
    const int64_t place = page_place(P.p, U.b, U.row.p0 + i);
    if (place < 0) return to;
    const int64_t at = paged_base(P, (int)(place >> P.p.lg), hk) + (place & ((1 << P.p.lg) - 1));
    to.out = P.next + at * P.dim * (int64_t)sizeof(T);
    to.lse = P.lses + at;
    if (P.vmul.p) to.mul = reinterpret_cast<const char*>(P.vmul.at<T>(src_b, hk) + (int64_t)tok * P.vmul.sn);
    return to;
}

// four features of a result
template <typename T>
__device__ __forceinline__ void paged_store(const PagedTo& to, int d, float4 y) {
    if constexpr (sizeof(T) == 4) {
        if (to.mul) {
            const float4 m = *reinterpret_cast<const float4*>(to.mul + 4 * d);
            y = make_float4(y.x * m.x, y.y * m.y, y.z * m.z, y.w * m.w);
        }
        *reinterpret_cast<float4*>(to.out + 4 * d) = y;
    } else {
        if (to.mul) {
            typedef T t4 __attribute__((ext_vector_type(4)));
            const t4 m = *reinterpret_cast<const t4*>(to.mul + 2 * d);
            y = make_float4(y.x * (float)m[0], y.y * (float)m[1], y.z * (float)m[2], y.w * (float)m[3]);
        }
        u32x2_d w;
        w[0] = draft_pack2<T>(y.x, y.y);
        w[1] = draft_pack2<T>(y.z, y.w);
        *reinterpret_cast<u32x2_d*>(to.out + 2 * d) = w;
    }
}

// The first features of query row r: q at the final level, else the next level's keys at its position; null for
// a page outside the pool.
template <typename T>
__device__ __forceinline__ const T* paged_query(const PagedDev& P, const PagedUnit& U, int hk, int r) {
    const int i = r / P.rep;
    if (P.last)
        return P.q.at<T>(P.p.packed ? 0 : U.b, hk * P.rep + r - i * P.rep) + (int64_t)(U.row.start + i) * P.q.sn;
    const int64_t place = page_place(P.p, U.b, U.row.p0 + i);
    if (place < 0) return nullptr;
    const int64_t at = paged_base(P, (int)(place >> P.p.lg), hk) + (place & ((1 << P.p.lg) - 1));
    return reinterpret_cast<const T*>(P.queries) + at * P.dim;
}

// acc, no number once a word of two 16-bit numbers (of one of 32 bits) held one that is not finite.
template <typename T>
__device__ __forceinline__ float paged_odd(uint32_t w, float acc) {
    if constexpr (sizeof(T) == 4) {
        return fmaf(__uint_as_float(w), 0.f, acc);
    } else if constexpr (std::is_same_v<T, f16>) {
        typedef _Float16 v2 __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(v2, w), __builtin_bit_cast(v2, 0u), acc, false);
    } else {
        typedef __bf16 v2 __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2, w), __builtin_bit_cast(v2, 0u), acc, false);
    }
}

// Records that the same launch reads (GPU) are written and read at the GPU's level, past their XCD's cache.
constexpr int kPagedGpu = 16;  // sc1
// a tile's records, from its first unit's
template <bool GPU>
struct PagedRecords {
    __amdgpu_buffer_rsrc_t o;
    float2* s;
    int step;  // rows from a unit's record to the next one's
    int dim;
    __device__ __forceinline__ PagedRecords(const PagedDev& P, const PagedUnit& U, int hk) {
        const int64_t first = ((int64_t)U.rec * P.kv_heads + hk) * P.tile;
        step = P.kv_heads * P.tile;
        dim = P.dim;
        s = P.ws_s + first;
        o = draft_buffer(reinterpret_cast<const char*>(P.ws_o + first * P.dim), (int64_t)U.splits * step * P.dim * 4);
    }
    __device__ __forceinline__ float4 get(int row, int d) const {
        return __builtin_bit_cast(float4, __builtin_amdgcn_raw_buffer_load_b128(o, (row * dim + d) * 4, 0, GPU ? kPagedGpu : 0));
    }
    __device__ __forceinline__ void put(int row, int d, float4 y) const {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_d, y), o, (row * dim + d) * 4, 0, GPU ? kPagedGpu : 0);
    }
    __device__ __forceinline__ float2 get_sum(int row) const {
        if (!GPU) return s[row];
        return __builtin_bit_cast(float2, __hip_atomic_load(reinterpret_cast<const uint64_t*>(s + row), __ATOMIC_RELAXED,
                                                            __HIP_MEMORY_SCOPE_AGENT));
    }
    __device__ __forceinline__ void put_sum(int row, float top, float sum) const {
        if (!GPU)
            s[row] = make_float2(top, sum);
        else
            __hip_atomic_store(reinterpret_cast<uint64_t*>(s + row), __builtin_bit_cast(uint64_t, make_float2(top, sum)),
                               __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
};

// Joins `count` records, `first` and every `ustep`-th after it, of n query rows of a tile, r first, by the workgroup:
// M 2^lgr rows at a time, M of them and four features a thread, the records dealt out over what is left of the
// threads, so that 8 to 16 loads are under way.  The rows are finished, or the first record takes what was
// joined.  True where a record's sum is no number.
template <typename T, int M, bool GPU>
__device__ __forceinline__ bool paged_join(const PagedDev& P, const PagedUnit& U, int hk, int first, int ustep, int count, bool finish,
                                           int r, int n, int lgr, float (*s_red)[6]) {
    constexpr int N = M >= 2 ? 4 : 6;
    const PagedRecords<GPU> R(P, U, hk);
    const int tid = threadIdx.x;
    const int quads = P.dim >> 2;
    int lgq = 0;
    while ((1 << lgq) < quads) ++lgq;  // at most 64
    const int lgp = lgq + lgr, parts = kPageThreads >> lgp, part = tid >> lgp, d = (tid & ((1 << lgq) - 1)) * 4;
    const int row0 = first * R.step + r - U.tile * P.tile;
    bool none = false;
    for (int i0 = 0; i0 < n; i0 += M << lgr) {
        const int i = i0 + ((tid >> lgq) & ((1 << lgr) - 1));
        float top[M], sum[M];
        float4 y[M];
#pragma unroll
        for (int q = 0; q < M; ++q) {
            top[q] = -INFINITY;
            sum[q] = 0.f;
            y[q] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        if (d < P.dim)
            for (int u0 = part; u0 < count; u0 += N * parts) {
                float2 ms[M][N];
                float4 z[M][N];
#pragma unroll
                for (int k = 0; k < N; ++k)
#pragma unroll
                    for (int q = 0; q < M; ++q) {
                        const int at = row0 + min(i + (q << lgr), n - 1) + min(u0 + k * parts, count - 1) * ustep * R.step;
                        ms[q][k] = R.get_sum(at);
                        z[q][k] = R.get(at, d);
                    }
#pragma unroll
                for (int q = 0; q < M; ++q) {
                    float t = top[q];
#pragma unroll
                    for (int k = 0; k < N; ++k) t = u0 + k * parts < count ? fmaxf(t, ms[q][k].x) : t;
                    const float f = top[q] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top[q] - t);
                    top[q] = t;
                    sum[q] *= f;
                    y[q] = make_float4(y[q].x * f, y[q].y * f, y[q].z * f, y[q].w * f);
#pragma unroll
                    for (int k = 0; k < N; ++k) {
                        if (u0 + k * parts >= count) continue;
                        if (ms[q][k].x == -INFINITY) {  // its sum is 0, or no number as its scores are
                            sum[q] += ms[q][k].y;
                            continue;
                        }
                        const float w = __builtin_amdgcn_exp2f(ms[q][k].x - t);
                        sum[q] += ms[q][k].y * w;
                        y[q] = make_float4(fmaf(z[q][k].x, w, y[q].x), fmaf(z[q][k].y, w, y[q].y), fmaf(z[q][k].z, w, y[q].z),
                                           fmaf(z[q][k].w, w, y[q].w));
                    }
                }
            }
        if (!finish) __syncthreads();  // the first record has been read
        auto end = [&](float top, float sum, float4 y, int row) __attribute__((always_inline)) {
            none = none || sum != sum;
            if (row - i + i0 < n && parts > 1) {  // a row in some thread
                float* const mine = s_red[tid];
                mine[0] = top;
                mine[1] = sum;
                mine[2] = y.x;
                mine[3] = y.y;
                mine[4] = y.z;
                mine[5] = y.w;
                __syncthreads();
                if (part == 0) {
                    float t = top;
                    for (int k = 1; k < parts; ++k) t = fmaxf(t, s_red[(k << lgp) + tid][0]);
                    const float f0 = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - t);
                    top = t;
                    sum *= f0;
                    y = make_float4(y.x * f0, y.y * f0, y.z * f0, y.w * f0);
                    for (int k = 1; k < parts; ++k) {
                        const float* z = s_red[(k << lgp) + tid];
                        if (z[0] == -INFINITY) {
                            sum += z[1];
                            continue;
                        }
                        const float w = __builtin_amdgcn_exp2f(z[0] - t);
                        sum += z[1] * w;
                        y = make_float4(fmaf(z[2], w, y.x), fmaf(z[3], w, y.y), fmaf(z[4], w, y.z), fmaf(z[5], w, y.w));
                    }
                }
                __syncthreads();  // s_red is written again
            }
            if (part != 0 || row >= n || d >= P.dim) return;
            if (finish) {
                const PagedTo to = paged_to<T>(P, U, hk, r + row);
                const float inv = 1.f / sum;
                if (to.out) paged_store<T>(to, d, make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv));
                if (d == 0 && to.lse) *to.lse = (top + log2f(sum)) * kLn2;
            } else {
                R.put(row0 + row, d, y);
                if (d == 0) R.put_sum(row0 + row, top, sum);
            }
        };
        end(top[0], sum[0], y[0], i);
        if constexpr (M > 1) end(top[1], sum[1], y[1], i + (1 << lgr));
        if constexpr (M > 2) {
            end(top[2], sum[2], y[2], i + (2 << lgr));
            end(top[3], sum[3], y[3], i + (3 << lgr));
        }
    }
    return none;
}

// The end of a unit of the tile's n query rows, r first, its records written: the last one of its tile joins them, as a
// ticket says.  More than eight units, or than 128 rows of records, join in two steps, groups of about the square root of
// their number first, as one workgroup reads but 25 GB/s or so: one row of 65536 positions 116 us in one step, 110 in two; 32
// query rows behind up to 4096 59 with groups of eight, 57 so.
template <typename T, int M>
__device__ __forceinline__ void paged_end(const PagedDev& P, const PagedUnit& U, int hk, int r, int n, float (*s_red)[6], int& s_last) {
    const int live = min(U.splits, (paged_keys(P, U) + U.size * kPagedChunk - 1) / (U.size * kPagedChunk));
    int size = live;  // of a group
    if (live > 8 || live * n > 128)
        for (size = 2; size * size < live;) ++size;
    const int first = U.split - U.split % size, groups = (live + size - 1) / size, in = min(size, live - first);
    int lgr = 0;  // rows at once, as there are rows, and threads for four features each
    while ((1 << lgr) < n && (((P.dim >> 2) - 1) >> (7 - lgr)) == 0) ++lgr;
    for (bool whole = groups == 1;; whole = true) {
        int32_t* const ticket = P.tickets + ((int64_t)(U.rec + (whole ? 0 : first)) * P.kv_heads + hk) * kTicketStride + (whole ? 0 : 1);
        const int all = groups == 1 ? live : whole ? groups : in;
        // the records are there once the waves' stores have returned; a release would write the cache back, at several us
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (threadIdx.x == 0) {
            const int drawn = __hip_atomic_fetch_add(ticket, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            s_last = drawn == all - 1;
            if (drawn == all - 1) __hip_atomic_store(ticket, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (!__builtin_amdgcn_readfirstlane(s_last)) return;
        paged_join<T, M, true>(P, U, hk, whole ? 0 : first, whole && groups > 1 ? size : 1, all, whole, r, n, lgr, s_red);
        if (whole) return;
    }
}

// Where values that are not finite lie behind some row's own position, the products of k_paged_tiles are no numbers: a
// weight of 0 times such a value.  A unit says so by a sum that is no number, in its records, or where it is its tile's
// only one by a byte for each of its waves; the join then forms the rows again, one after another.
__device__ __forceinline__ uint8_t* paged_flag(const PagedDev& P, int wave) {
    return P.flags + 8 * (int64_t)blockIdx.x + wave;
}

// Outputs of tokens behind their chunk: 0.  A wave per token, workgroup `group` of `groups`.
template <typename T>
__device__ __forceinline__ void paged_clear(const PagedDev& P, int group, int groups) {
    const int lane = threadIdx.x & 63;
    const int64_t all = (int64_t)P.p.tokens * (P.p.packed ? 1 : P.p.rows), step = (int64_t)groups * (kPageThreads / 64);
    for (int64_t x = (int64_t)group * (kPageThreads / 64) + (threadIdx.x >> 6); x < all; x += step) {
        const int b = P.p.packed ? page_find(P.p, (int)x, lane) : (int)(x / P.p.tokens);
        const int i = (int)(P.p.packed ? x : x - (int64_t)b * P.p.tokens);
        const PageRow r = page_row(P.p, b);
        if (i >= r.start && i - r.start < r.len) continue;
        const int quads = P.dim >> 2, items = P.kv_heads * P.rep * quads;
        PagedTo at = {nullptr, nullptr, nullptr};
        for (int k = lane; k < items; k += 64) {
            const int h = k / quads, d = (k - h * quads) * 4;
            at.out = reinterpret_cast<char*>(P.out.at<T>(P.p.packed ? 0 : b, h) + (int64_t)i * P.out.sn);
            paged_store<T>(at, d, make_float4(0.f, 0.f, 0.f, 0.f));
        }
    }
}

// 16-row tiles of the workgroup's rows: what its registers hold
template <typename T> constexpr int paged_row_tiles(int D) { return D > 128 ? 1 : 2; }
// Waves per SIMD that the registers are held to
constexpr int paged_waves(int D, int RT) { return D <= 128 && D * RT <= 256 ? 2 : 1; }

// joins: workgroups that join the tiles of B; clear: those that clear outputs
template <typename T> void launch_paged_rows(const PagedDev& P, const PagedDev& B, int64_t units, int joins, int clear, int tiles, hipStream_t s);
// in source files of their own
extern template void launch_paged_rows<bf16>(const PagedDev& P, const PagedDev& B, int64_t units, int joins, int clear, int tiles, hipStream_t s);
extern template void launch_paged_rows<f16>(const PagedDev& P, const PagedDev& B, int64_t units, int joins, int clear, int tiles, hipStream_t s);
extern template void launch_paged_rows<float>(const PagedDev& P, const PagedDev& B, int64_t units, int joins, int clear, int tiles, hipStream_t s);
// 16-bit chunks of more rows (k_paged_tiles), head dims up to 128
constexpr int kTileRows = 256;  // of a tile
template <typename T> void launch_paged_tiles(const PagedDev& P, int64_t units, hipStream_t s);
extern template void launch_paged_tiles<bf16>(const PagedDev& P, int64_t units, hipStream_t s);
extern template void launch_paged_tiles<f16>(const PagedDev& P, int64_t units, hipStream_t s);

}  // namespace pa
