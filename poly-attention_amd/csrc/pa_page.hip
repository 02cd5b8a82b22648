// pa_page.hip -- the pages of a paged cache: which row has which (k_page_extend, k_page_select,
// k_page_plan), their copies (k_page_copy), and the norms and rotary of a chunk's tokens into them
// (k_page_append).
//
// A page is free where nothing refers to it, and the free pages are found by a scan in their order: no
// list has to agree with the counts of references, and which page a row gets does not depend on the
// order in which atomics arrive.
#include <algorithm>

#include "pa_page.h"

namespace pa {

constexpr int kPlanThreads = 1024;  // of the kernels of one workgroup
constexpr int kPlanWaves = kPlanThreads / 64;
constexpr int kCopyParts = 64;  // of a page's copy, at most

struct PagePlan {  // a table, and a call's arguments
    int32_t rows, pages, lg, max_pages;
    int32_t* table;
    int32_t* counts;
    int32_t* refs;
    int32_t* fresh;
    int32_t* starts;
    int32_t* overflow;
    const int32_t* index;
    const int32_t* lengths;
    const int32_t* more;
    // scratch
    int32_t* head;   // [4]: moves, ...
    int4* moves;     // [max(rows, pages / 2 + 1)]: from, to, positions
    int32_t* list;   // [pages]: the free pages that are handed out, or where a page went
    int32_t* need;   // [rows]
    int32_t* copy;   // [rows, max_pages]
    const pa_page_array* arrays;
    int32_t count;
};

// Exclusive prefix sums of two numbers over the workgroup, and their totals.
// In 64 bits: a step may ask for any number of pages and tokens.
struct Sums {
    int64_t a, b, all_a, all_b;
};
__device__ __forceinline__ Sums block_sums(int a, int b, int64_t (*part)[2], int tid) {
    const int lane = tid & 63, wave = tid >> 6;
    int64_t x = a, y = b;
    for (int off = 1; off < 64; off <<= 1) {
        const int64_t u = __shfl_up(x, off), v = __shfl_up(y, off);
        if (lane >= off) {
            x += u;
            y += v;
        }
    }
    __syncthreads();  // the last call's sums have been read
    if (lane == 63) {
        part[wave][0] = x;
        part[wave][1] = y;
    }
    __syncthreads();
    Sums s = {x - a, y - b, 0, 0};
    for (int w = 0; w < kPlanWaves; ++w) {
        if (w == wave) {
            s.a += s.all_a;
            s.b += s.all_b;
        }
        s.all_a += part[w][0];
        s.all_b += part[w][1];
    }
    return s;
}

// 16 references from place `first`, a multiple of 16; `none` past the last page
__device__ __forceinline__ void plan_refs(const PagePlan& P, int64_t first, int none, int (&r)[16]) {
    if (first + 16 <= P.pages && (uintptr_t)P.refs % 16 == 0) {
#pragma unroll
        for (int k = 0; k < 16; k += 4) {
            const int4 x = *reinterpret_cast<const int4*>(P.refs + first + k);
            r[k] = x.x, r[k + 1] = x.y, r[k + 2] = x.z, r[k + 3] = x.w;
        }
    } else {
#pragma unroll
        for (int k = 0; k < 16; ++k) r[k] = first + k < P.pages ? P.refs[first + k] : none;
    }
}

// the free ones among them, a bit each
__device__ __forceinline__ uint32_t plan_free(const int (&r)[16]) {
    uint32_t free = 0;
#pragma unroll
    for (int k = 0; k < 16; ++k) free |= (uint32_t)(r[k] == 0) << k;
    return free;
}

__device__ __forceinline__ int plan_count(const PagePlan& P, int b) {
    return min(max(P.counts[b], 0), P.max_pages << P.lg);
}
__device__ __forceinline__ bool plan_page(const PagePlan& P, int id) { return (unsigned)id < (unsigned)P.pages; }

// What row b asks for: m positions (0 where they pass the table), behind n.
__device__ __forceinline__ void plan_asked(const PagePlan& P, int b, int& n, int& m, bool& past) {
    n = plan_count(P, b);
    m = max(P.more[b], 0);
    past = m > (P.max_pages << P.lg) - n;
    if (past) m = 0;
}

// Pages for the rows' next positions, by one workgroup.  Latency: the rows' state, a scan of the references
// that ends when enough free pages are found, the writes of the table: 7.6 us for one user, 10.5 for 32 rows.
__global__ __launch_bounds__(kPlanThreads) void k_page_extend(const PagePlan P) {
    __shared__ int64_t s_part[kPlanWaves][2];
    __shared__ int s_tail[PA_MAX_PAGE_ROWS];  // the partly filled page that a row is about to write, or -1
    __shared__ int s_need[PA_MAX_PAGE_ROWS], s_upto[PA_MAX_PAGE_ROWS], s_after[PA_MAX_PAGE_ROWS];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int size = 1 << P.lg;
    int r[16];
    plan_refs(P, (int64_t)tid * 16, 1, r);
    uint32_t free = plan_free(r);  // nothing below writes them before they have been looked at
    for (int b = tid; b < P.rows; b += kPlanThreads) {
        int n, m;
        bool past;
        plan_asked(P, b, n, m, past);
        int tail = -1;
        if (m > 0 && (n & (size - 1))) {
            tail = P.table[(int64_t)b * P.max_pages + (n >> P.lg)];
            if (!plan_page(P, tail)) tail = -1;
        }
        s_tail[b] = tail;
    }
    __syncthreads();
    // a row's pages, and how many the rows up to it need
    int64_t needed = 0, tokens = 0;
    auto clip = [](int64_t x) __attribute__((always_inline)) -> int { return (int)min(x, (int64_t)INT32_MAX); };
    for (int b0 = 0; b0 < P.rows; b0 += kPlanThreads) {
        const int b = b0 + tid;
        int n = 0, m = 0, want = 0, flags = 0, after = -1;
        bool past = false;
        if (b < P.rows) {
            plan_asked(P, b, n, m, past);
            if (m > 0) want = ((n + m + size - 1) >> P.lg) - ((n + size - 1) >> P.lg);
            const int tail = s_tail[b];
            if (tail >= 0) {
                const int refs = P.refs[tail];
                if (refs > 1) {  // all but the last of the rows that write a shared page copy it
                    int before = 0;
                    for (int r = 0; r < b; ++r)
                        if (s_tail[r] == tail) {
                            ++before;
                            after = r;
                        }
                    if (refs - before > 1) {
                        flags |= 1;
                        ++want;
                    }
                }
            }
            if (past) flags |= 4;
        }
        const int asked = b < P.rows ? max(P.more[b], 0) : 0;
        const Sums s = block_sums(want, asked, s_part, tid);
        if (b < P.rows) {
            s_need[b] = want << 3 | flags;
            s_after[b] = after;
            s_upto[b] = clip(needed + s.a + want);
            P.starts[b] = clip(tokens + s.b);
        }
        needed += s.all_a;
        tokens += s.all_b;
    }
    if (tid == 0) {
        P.starts[P.rows] = clip(tokens);
        P.head[0] = 0;
    }
    // the first `needed` free pages
    int64_t found = 0;
    constexpr int U = 16;
    for (int64_t p0 = 0; p0 < P.pages && found < needed; p0 += kPlanThreads * U) {
        const int64_t first = p0 + (int64_t)tid * U;
        if (p0 > 0) {
            plan_refs(P, first, 1, r);
            free = plan_free(r);
        }
        const Sums s = block_sums(__popc(free), 0, s_part, tid);
        int64_t at = found + s.a;
        for (; free && at < needed; free &= free - 1, ++at) P.list[at] = (int)(first + __ffs(free) - 1);
        found += s.all_a;
    }
    __syncthreads();
    // a wave per row
    for (int b = wave; b < P.rows; b += kPlanWaves) {
        int n, m;
        bool past;
        plan_asked(P, b, n, m, past);
        const int need = s_need[b], want = need >> 3;
        const int first = s_upto[b] - want;
        // a row that keeps a page needs the last of those that copied it to have got theirs, and so the others
        const int after = s_after[b];
        const bool ok = m > 0 && (want > 0 ? s_upto[b] <= found : after < 0 || s_upto[after] <= found);
        const bool copies = need & 1;
        if (ok) {
            const int at = copies ? n >> P.lg : (n + size - 1) >> P.lg;
            int32_t* row = P.table + (int64_t)b * P.max_pages + at;
            for (int k = lane; k < want; k += 64) {
                const int id = P.list[first + k];
                row[k] = id;
                P.refs[id] = 1;
            }
            if (copies && lane == 0) {
                const int tail = s_tail[b];
                atomicSub(P.refs + tail, 1);
                // which of the moves comes first does not matter: they go to pages of their own
                P.moves[atomicAdd(P.head, 1)] = make_int4(tail, P.list[first], n & (size - 1), 0);
            }
        }
        // every lane has read the row's count
        __builtin_amdgcn_wave_barrier();
        if (lane == 0) {
            P.counts[b] = n + (ok ? m : 0);
            P.fresh[b] = ok ? m : 0;
            if (P.overflow && ((need & 4) || (m > 0 && !ok))) *P.overflow = 1;
        }
    }
}

// Rows as the beginnings of other rows: what the rows become, beside the references; then, when all rows have been
// read, into the table.  A workgroup per row in two launches, or one for a small table, which saves the second
// launch's 4 us or so.
__device__ __forceinline__ void select_new(const PagePlan& P, int b, int tid, int threads) {
    const int size = 1 << P.lg, old_pages = (plan_count(P, b) + size - 1) >> P.lg;
    int src = P.index[b], n = 0;
    if (src < 0 || src >= P.rows) {
        src = -1;
    } else {
        n = plan_count(P, src);
        if (P.lengths) n = min(n, max(P.lengths[b], 0));
    }
    const int used = (n + size - 1) >> P.lg, most = max(used, old_pages);
    const int32_t* from = P.table + (int64_t)max(src, 0) * P.max_pages;
    const int32_t* own = P.table + (int64_t)b * P.max_pages;
    int32_t* to = P.copy + (int64_t)b * P.max_pages;
    for (int k = tid; k < most; k += threads) {
        const int was = k < old_pages ? own[k] : -1, is = k < used ? from[k] : -1;
        to[k] = is;
        if (was != is) {
            if (plan_page(P, was)) atomicSub(P.refs + was, 1);
            if (plan_page(P, is)) atomicAdd(P.refs + is, 1);
        }
    }
    if (tid == 0) P.need[b] = n;
}
// the count, which the callers write when all threads of the row have read it
__device__ __forceinline__ int select_row(const PagePlan& P, int b, int tid, int threads) {
    const int size = 1 << P.lg;
    const int n = P.need[b], old = plan_count(P, b);
    const int most = max((n + size - 1) >> P.lg, (old + size - 1) >> P.lg);
    int32_t* row = P.table + (int64_t)b * P.max_pages;
    const int32_t* from = P.copy + (int64_t)b * P.max_pages;
    for (int k = tid; k < most; k += threads) row[k] = from[k];
    return n;
}
__global__ __launch_bounds__(kPageThreads) void k_page_select(const PagePlan P) {
    select_new(P, blockIdx.x, threadIdx.x, kPageThreads);
}
__global__ __launch_bounds__(kPageThreads) void k_page_selected(const PagePlan P) {
    const int b = blockIdx.x, n = select_row(P, b, threadIdx.x, kPageThreads);
    __syncthreads();
    if (threadIdx.x == 0) {
        P.counts[b] = n;
        P.fresh[b] = 0;
    }
}
__global__ __launch_bounds__(kPlanThreads) void k_page_select_all(const PagePlan P) {  // a wave per row
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int b = wave; b < P.rows; b += kPlanWaves) select_new(P, b, lane, 64);
    __syncthreads();
    for (int b = wave; b < P.rows; b += kPlanWaves) {
        const int n = select_row(P, b, lane, 64);
        __builtin_amdgcn_wave_barrier();
        if (lane == 0) {
            P.counts[b] = n;
            P.fresh[b] = 0;
        }
    }
}

// Where the pages in use go: the k-th that lies behind the first `used` places into the k-th free of those.
// One workgroup, two scans of the references, 16 a thread at a time: 7.8 to 8.5 us.
__global__ __launch_bounds__(kPlanThreads) void k_page_plan(const PagePlan P) {
    __shared__ int64_t s_part[kPlanWaves][2];
    const int tid = threadIdx.x;
    constexpr int U = 16;
    int used = 0;
    for (int64_t p0 = 0; p0 < P.pages; p0 += kPlanThreads * U) {
        int mine = 0, r[U];
        plan_refs(P, p0 + (int64_t)tid * U, 0, r);
#pragma unroll
        for (int k = 0; k < U; ++k) mine += r[k] > 0;
        used += (int)block_sums(mine, 0, s_part, tid).all_a;
    }
    int holes = 0, movers = 0;
    for (int64_t p0 = 0; p0 < P.pages; p0 += kPlanThreads * U) {
        const int64_t first = p0 + (int64_t)tid * U;
        int free = 0, moving = 0, r[U];
        plan_refs(P, first, 0, r);
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const bool in = first + k < used;
            free += in && r[k] <= 0;
            moving += !in && r[k] > 0;
        }
        const Sums s = block_sums(free, moving, s_part, tid);
        int f = holes + (int)s.a, m = movers + (int)s.b;
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const bool in = first + k < used;
            if (in && r[k] <= 0) P.moves[f++].y = (int)(first + k);
            if (!in && r[k] > 0) P.moves[m++].x = (int)(first + k);
        }
        holes += (int)s.all_a;
        movers += (int)s.all_b;
    }
    __syncthreads();
    for (int k = tid; k < movers; k += kPlanThreads) {
        const int4 x = P.moves[k];
        P.moves[k].z = 1 << P.lg;
        P.list[x.x] = x.y;
        P.refs[x.y] = P.refs[x.x];
        P.refs[x.x] = 0;
    }
    if (tid == 0) {
        P.head[0] = movers;
        P.head[1] = used;
    }
}

// The moves of pages, in every array, and with `remap` the table's entries that follow them.  Bound by memory: 16 bytes a
// lane, eight loads in flight, stores past the caches (half a GB moved in a pool 245 us without, 235 with).  A wave takes
// a part of a page at a time: as many parts as give each wave four or so.
__global__ __launch_bounds__(kPageThreads) void k_page_copy(const PagePlan P, int remap) {
    const int lane = threadIdx.x & 63;
    const int64_t waves = (int64_t)gridDim.x * (kPageThreads / 64);
    const int64_t wave = (int64_t)blockIdx.x * (kPageThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int moves = P.head[0];
    if (remap && moves > 0) {
        const int used = P.head[1];
        const int64_t all = (int64_t)P.rows * P.max_pages;
        for (int64_t k = wave * 64 + lane; k < all; k += waves * 64) {
            const int id = P.table[k];
            if (id >= used && id < P.pages) {
                const int to = P.list[id];
                if (plan_page(P, to)) P.table[k] = to;
            }
        }
    }
    const int64_t pages = (int64_t)moves * P.count;
    if (pages == 0) return;
    const int parts = (int)min(max(4 * waves / pages, (int64_t)1), (int64_t)kCopyParts);
    for (int64_t it = wave; it < pages * parts; it += waves) {
        // neighbours in time copy one page's arrays
        const int64_t x = it / parts;
        const int part = (int)(it - x * parts), mv = (int)(x / P.count), a = (int)(x - (int64_t)mv * P.count);
        const int4 m = P.moves[mv];
        const pa_page_array A = P.arrays[a];
        const int64_t head = (int64_t)A.row_bytes << P.lg, page = head * A.heads;
        const char* src = static_cast<const char*>(A.base) + m.x * page;
        char* dst = static_cast<char*>(A.base) + m.y * page;
        const int bytes = m.z * A.row_bytes;  // of a head
        constexpr int U = 8;
        auto move = [&](auto word) __attribute__((always_inline)) {
            typedef decltype(word) W;
            const int per = bytes / (int)sizeof(W), all = per * A.heads;
            const int each = (all + parts * 64 - 1) / (parts * 64) * 64, end = min((part + 1) * each, all);
            const int64_t skip = head - bytes;  // between heads
            for (int x0 = part * each; x0 < end; x0 += 64 * U) {
                W v[U];
                int64_t at[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int k = min(x0 + 64 * u + lane, end - 1);
                    at[u] = (int64_t)sizeof(W) * k + (skip ? skip * (k / per) : 0);
                    v[u] = *reinterpret_cast<const W*>(src + at[u]);
                }
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (x0 + 64 * u + lane < end) __builtin_nontemporal_store(v[u], reinterpret_cast<W*>(dst + at[u]));
            }
        };
        if (bytes % 16 == 0) move(u32x4_d{});  // a head of a page has 16 rows or more
        else move(uint32_t{});
    }
}

// ---------------------------------------------------------------------------------------
// Norms and rotary of the chunks' tokens, into their pages.  A wave per token and four groups of 64 / lpr rows of one
// tensor, a lane holding 16 bytes of a row: the tensor, its weights and the lane's features are the same for all of
// them.  The token's sines and cosines are dealt out over the wave's lanes.  Bound by memory, behind it by
// instructions: 4096 tokens of 56 heads of 128 (117 MB) 24 us; 57 with a workgroup per token whose waves look the
// tensors up, 58 with a workgroup for several tokens, which has too few waves.

struct PageItemDev {
    DraftRow src, out;
    const void* w;
    char* pages;
    int32_t wdt, rotate, heads;
    int32_t wide;  // the weights are of 32 bits or of the rows' type, and can be read 16 bytes at a time
};
struct PageRowsDev {
    PageDev p;
    int32_t dim, count, rot_dim, adt, lpr;
    float eps, interp;
    int64_t angles_sb, angles_sn;
    const void* angles;
    const float* inv_freq;
    int32_t all;                      // tokens
    int32_t first[PA_MAX_ORDER + 2];  // an item's first four groups of rows; of those past the last INT32_MAX
    PageItemDev it[PA_MAX_ORDER + 2];
};

// 16 bytes of a row as E numbers, and E numbers of another type
template <typename T, int E>
__device__ __forceinline__ void page_numbers(u32x4_d raw, float (&x)[E]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = __uint_as_float(raw[e]);
    } else {
        typedef T t2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t word = raw[e];  // a value: a bit cast of the element reads element 0
            const t2 z = __builtin_bit_cast(t2, word);
            x[2 * e] = (float)z[0];
            x[2 * e + 1] = (float)z[1];
        }
    }
}

// the sum over a group of `n` neighbouring lanes, a power of two
__device__ __forceinline__ float page_sum(float x, int n) {
    auto dpp = [](float x, auto ctrl) __attribute__((always_inline)) -> float {
        return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value, 0xf, 0xf, true));
    };
    if (n > 1) x += dpp(x, std::integral_constant<int, 0xb1>());   // neighbours
    if (n > 2) x += dpp(x, std::integral_constant<int, 0x4e>());   // pairs
    if (n > 4) x += dpp(x, std::integral_constant<int, 0x141>());  // the halves of a row of 16, mirrored
    if (n > 8) x += dpp(x, std::integral_constant<int, 0x140>());  // the row, mirrored
    if (n > 16) x += __shfl_xor(x, 16);
    if (n > 32) x += __shfl_xor(x, 32);
    return x;
}

// sin and cos: of an angle that is reduced by Cody and Waite's two parts of 2 pi, by the instructions, which
// are within 2^-20 or so: far less than a 16-bit type's rounding
template <typename T>
__device__ __forceinline__ void page_sincos(float a, float& sn, float& cs) {
    if constexpr (sizeof(T) == 4) {
        sincosf(a, &sn, &cs);
    } else {
        const float q = rintf(a * 0.15915494309189535f);
        const float r = fmaf(-q, -1.7484555e-7f, fmaf(-q, 6.2831855f, a)) * 0.15915494309189535f;
        sn = __builtin_amdgcn_sinf(r);
        cs = __builtin_amdgcn_cosf(r);
    }
}

constexpr int kAppendGroups = 4;

template <typename T>
__global__ __launch_bounds__(kPageThreads) void k_page_append(const PageRowsDev P) {
    constexpr int E = 16 / sizeof(T), U = kAppendGroups;
    __shared__ __align__(16) float s_cos[kPageThreads / 64][256], s_sin[kPageThreads / 64][256];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int k = 0, from = 0;
#pragma unroll
    for (int j = 1; j < PA_MAX_ORDER + 2; ++j)
        if ((int)blockIdx.y >= P.first[j]) {
            k = j;
            from = P.first[j];
        }
    const PageItemDev& I = P.it[k];
    const int group = 64 / P.lpr, h0 = ((int)blockIdx.y - from) * U * group + lane / P.lpr;
    const int x = blockIdx.x * (kPageThreads / 64) + wave;
    if (x >= P.all) return;
    int b, tok;
    if (P.p.packed) {
        tok = x;
        b = page_find(P.p, x, lane);
    } else {
        b = x / P.p.tokens;
        tok = x - b * P.p.tokens;
    }
    const PageRow row = page_row(P.p, b);
    const int i = tok - row.start, pos = row.p0 + i, src_b = P.p.packed ? 0 : b;
    const bool here = i >= 0 && i < row.len;
    if (!here && I.pages) return;
    const int d0 = (lane & (P.lpr - 1)) * E;
    const bool in = d0 < P.dim;
    u32x4_d raw[U];
    const T* const src = I.src.at<T>(src_b, 0) + (int64_t)tok * I.src.sn + d0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        raw[u] = u32x4_d{0u, 0u, 0u, 0u};
        if (here && in && h0 + u * group < I.heads) raw[u] = load16u(src + (h0 + u * group) * I.src.sh);
    }
    float w[E];
#pragma unroll
    for (int e = 0; e < E; ++e) w[e] = 0.f;
    if (I.w && in) {
        const char* const at = static_cast<const char*>(I.w) + d0 * (I.wdt == PA_F32 ? 4 : 2);
        if (!I.wide) {
#pragma unroll
            for (int e = 0; e < E; ++e) w[e] = load_any(I.w, I.wdt, d0 + e);
        } else if (sizeof(T) == 4 || I.wdt != PA_F32) {
            page_numbers<T>(load16u(at), w);
        } else {
            const u32x4_d a = load16u(at), b = load16u(at + 16);
#pragma unroll
            for (int e = 0; e < E; ++e) w[e] = __uint_as_float(e < 4 ? a[e & 3] : b[e & 3]);
        }
    }
    const int64_t place = here ? page_place(P.p, b, pos) : -1;
    if (I.pages && place < 0) return;
    const bool turn = I.rotate && P.rot_dim > 0 && here;
    float cs[E], sn[E];
    if (turn) {
        float *const c = s_cos[wave], *const s = s_sin[wave];
        // the position as the rotary module builds it, rounded to the rows' type
        const float at = round_to<T>(round_to<T>((float)pos) / P.interp);
        for (int p = lane; 2 * p < P.dim; p += 64) {  // a pair of features
            float a = 0.f, a1 = 0.f, s0, c0;
            if (2 * p < P.rot_dim) {
                if (P.angles) {
                    const int64_t from = src_b * P.angles_sb + tok * P.angles_sn + 2 * p;
                    a = load_any(P.angles, P.adt, from);
                    a1 = load_any(P.angles, P.adt, from + 1);
                } else {
                    a = a1 = at * P.inv_freq[p];
                }
            }
            page_sincos<T>(a, s0, c0);
            float s1 = s0, c1 = c0;
            if (__any(a1 != a)) page_sincos<T>(a1, s1, c1);  // usually they turn by one angle
            *reinterpret_cast<float2*>(s + 2 * p) = make_float2(s0, s1);
            *reinterpret_cast<float2*>(c + 2 * p) = make_float2(c0, c1);
        }
        // other lanes of the wave read them: LDS keeps a wave's order, the compiler has to as well
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int e = 0; e < E; e += 4) {
            const int at = in ? d0 + e : 0;
            const float4 x = *reinterpret_cast<const float4*>(c + at), y = *reinterpret_cast<const float4*>(s + at);
            cs[e] = x.x, cs[e + 1] = x.y, cs[e + 2] = x.z, cs[e + 3] = x.w;
            sn[e] = y.x, sn[e + 1] = y.y, sn[e + 2] = y.z, sn[e + 3] = y.w;
        }
    }
    T* out;
    int64_t sh;
    if (I.pages) {
        sh = (int64_t)P.dim << P.p.lg;
        out = reinterpret_cast<T*>(I.pages) + (place >> P.p.lg) * I.heads * sh + (place & ((1 << P.p.lg) - 1)) * P.dim + d0;
    } else {
        sh = I.out.sh;
        out = I.out.at<T>(src_b, 0) + (int64_t)tok * I.out.sn + d0;
    }
    const float rdim = 1.f / (float)P.dim;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        float v[E];
        page_numbers<T>(raw[u], v);
        if (I.w) {
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) ss = fmaf(v[e], v[e], ss);
            const float r = rsqrtf(fmaf(page_sum(ss, P.lpr), rdim, P.eps));
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = v[e] * r * w[e];
        }
        if (turn) {
#pragma unroll
            for (int e = 0; e < E; e += 2) {
                if (d0 + e >= P.rot_dim) continue;  // as it is: a sine of 0 times an infinity is no number
                const float z = v[e] * cs[e] - v[e + 1] * sn[e];
                v[e + 1] = v[e + 1] * cs[e + 1] + v[e] * sn[e + 1];
                v[e] = z;
            }
        }
        u32x4_d y;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (E == 4) y[e] = __float_as_uint(v[e]);
            else y[e] = draft_pack2<T>(v[2 * e], v[2 * e + 1]);
        }
        if (!here) y = u32x4_d{0u, 0u, 0u, 0u};
        if (in && h0 + u * group < I.heads) *reinterpret_cast<u32x4_d*>(out + (h0 + u * group) * sh) = y;
    }
}

// ---------------------------------------------------------------------------------------
// host side

namespace {

// the scratch's parts
size_t plan_scratch(const pa_page_table& t, PagePlan* P) {
    auto whole = [](size_t n) { return (n + 255) & ~size_t(255); };
    char* at = reinterpret_cast<char*>(t.scratch);
    size_t n = 0;
    auto take = [&](size_t bytes) {
        char* p = at ? at + n : nullptr;
        n += whole(bytes);
        return p;
    };
    PagePlan Q;
    if (!P) P = &Q;
    P->head = reinterpret_cast<int32_t*>(take(16));
    P->moves = reinterpret_cast<int4*>(take(std::max<size_t>(t.rows, t.pages / 2 + 1) * sizeof(int4)));
    P->list = reinterpret_cast<int32_t*>(take((size_t)t.pages * 4));
    P->need = reinterpret_cast<int32_t*>(take((size_t)t.rows * 4));
    P->copy = reinterpret_cast<int32_t*>(take((size_t)t.rows * t.max_pages * 4));
    return n;
}

int plan_dev(const pa_page_call* c, PagePlan& P) {
    const pa_page_table& t = c->t;
    if (const int st = page_check(t)) return st;
    if (!t.scratch || (uintptr_t)t.scratch % 16) return PA_EWORKSPACE;
    P.rows = t.rows;
    P.pages = t.pages;
    P.lg = page_lg(t.page_size);
    P.max_pages = t.max_pages;
    P.table = t.table;
    P.counts = t.counts;
    P.refs = t.refs;
    P.fresh = t.fresh;
    P.starts = t.starts;
    P.overflow = t.overflow;
    P.index = c->index;
    P.lengths = c->lengths;
    P.more = c->more;
    plan_scratch(t, &P);
    P.arrays = c->arrays;
    P.count = c->count;
    return PA_OK;
}

}  // namespace

size_t page_scratch(const pa_page_table* t) {
    if (t->rows < 1 || t->pages < 1 || t->max_pages < 1) return 0;
    pa_page_table x = *t;
    x.scratch = nullptr;
    return plan_scratch(x, nullptr);
}

// Workgroups of the copies, four waves each.  Half a GB moved in a pool: 1024 235 us, 512 278, 2048 260; 24 pages of 40
// arrays, partly filled: 256 24 us, 512 17, 1024 18.
constexpr int kCopyGroups = 1024, kStepGroups = 512;
// entries of a table that one workgroup selects
constexpr int64_t kSelectSmall = 8192;

int launch_page_select(const pa_page_call* c, hipStream_t s) {
    PagePlan P;
    if (const int st = plan_dev(c, P)) return st;
    if (!P.index) return PA_EINVAL;
    if ((int64_t)P.rows * P.max_pages <= kSelectSmall) {
        ProfScope ps("page_select", s);
        hipLaunchKernelGGL(k_page_select_all, dim3(1), dim3(kPlanThreads), 0, s, P);
        return PA_OK;
    }
    {
        ProfScope ps("page_select", s);
        hipLaunchKernelGGL(k_page_select, dim3(P.rows), dim3(kPageThreads), 0, s, P);
    }
    ProfScope ps("page_selected", s);
    hipLaunchKernelGGL(k_page_selected, dim3(P.rows), dim3(kPageThreads), 0, s, P);
    return PA_OK;
}

int launch_page_extend(const pa_page_call* c, hipStream_t s) {
    PagePlan P;
    if (const int st = plan_dev(c, P)) return st;
    if (!P.more || P.count < 0 || (P.count > 0 && !P.arrays)) return PA_EINVAL;
    {
        ProfScope ps("page_extend", s);
        hipLaunchKernelGGL(k_page_extend, dim3(1), dim3(kPlanThreads), 0, s, P);
    }
    if (P.count > 0) {
        ProfScope ps("page_copy", s);
        hipLaunchKernelGGL(k_page_copy, dim3(kStepGroups), dim3(kPageThreads), 0, s, P, 0);
    }
    return PA_OK;
}

int launch_page_compact(const pa_page_call* c, hipStream_t s) {
    PagePlan P;
    if (const int st = plan_dev(c, P)) return st;
    if (P.count < 0 || (P.count > 0 && !P.arrays)) return PA_EINVAL;
    {
        ProfScope ps("page_plan", s);
        hipLaunchKernelGGL(k_page_plan, dim3(1), dim3(kPlanThreads), 0, s, P);
    }
    ProfScope ps("page_copy", s);
    hipLaunchKernelGGL(k_page_copy, dim3(kCopyGroups), dim3(kPageThreads), 0, s, P, 1);
    return PA_OK;
}

int launch_page_append(const pa_page_rows* r, hipStream_t s) {
    if (const int st = page_check(r->t)) return st;
    if (r->tokens < 1 || r->dim < 1 || r->count < 1 || r->count > PA_MAX_ORDER + 2) return PA_EINVAL;
    const int T = r->items[0].src.dtype;
    if (!page_dtype(T)) return PA_EINVAL;
    if (!page_dim(r->dim)) return PA_EUNSUPPORTED;
    const bool rotary = r->angles || r->inv_freq;
    if (rotary && (r->rot_dim < 0 || r->rot_dim > r->dim || r->rot_dim % 2 != 0)) return PA_EINVAL;
    if (r->angles && !page_dtype(r->angles_dtype)) return PA_EINVAL;
    if (!r->angles && r->inv_freq && !(r->interp > 0.f)) return PA_EINVAL;
    PageRowsDev P;
    P.p = page_dev(r->t, r->tokens, r->packed != 0);
    P.dim = r->dim;
    P.count = r->count;
    P.rot_dim = rotary ? r->rot_dim : 0;
    P.adt = r->angles_dtype;
    P.eps = r->eps;
    P.interp = r->interp;
    P.angles_sb = r->angles_sb;
    P.angles_sn = r->angles_sn;
    P.angles = r->angles;
    P.inv_freq = r->inv_freq;
    const int E = T == PA_F32 ? 4 : 8;
    P.lpr = 1;
    while (P.lpr * E < r->dim) P.lpr <<= 1;
    int64_t groups = 0;  // four groups of rows each
    for (int k = 0; k < r->count; ++k) {
        const pa_page_item& it = r->items[k];
        if (!it.src.ptr || it.src.heads < 1 || it.src.dtype != T || !it.out.ptr == !it.pages ||
            (it.out.ptr && (it.out.heads != it.src.heads || it.out.dtype != T)) ||
            (it.norm_weight && !page_dtype(it.weight_dtype)))
            return PA_EINVAL;
        if (!page_rows16(it.src) || (it.out.ptr && !page_rows16(it.out)) || (uintptr_t)it.pages % 16) return PA_EUNSUPPORTED;
        PageItemDev& I = P.it[k];
        I.src = page_view(it.src);
        I.out = page_view(it.out);
        I.pages = static_cast<char*>(it.pages);
        I.w = it.norm_weight;
        I.wdt = it.weight_dtype;
        I.rotate = it.rotate;
        I.heads = it.src.heads;
        I.wide = (uintptr_t)it.norm_weight % 16 == 0 && (it.weight_dtype == PA_F32 || it.weight_dtype == T);
        P.first[k] = (int)groups;
        const int rows = kAppendGroups * (64 / P.lpr);
        groups += (I.heads + rows - 1) / rows;
    }
    if (groups > 65535) return PA_EUNSUPPORTED;
    for (int k = r->count; k < PA_MAX_ORDER + 2; ++k) P.first[k] = INT32_MAX;
    const int64_t tokens = (int64_t)r->tokens * (r->packed ? 1 : r->t.rows);
    if (tokens > kPageGroups) return PA_EUNSUPPORTED;
    P.all = (int)tokens;
    const dim3 grid((unsigned)((tokens + kPageThreads / 64 - 1) / (kPageThreads / 64)), (unsigned)groups);
    ProfScope ps("page_append", s);
    if (T == PA_F32) hipLaunchKernelGGL((k_page_append<float>), grid, dim3(kPageThreads), 0, s, P);
    else if (T == PA_F16) hipLaunchKernelGGL((k_page_append<f16>), grid, dim3(kPageThreads), 0, s, P);
    else hipLaunchKernelGGL((k_page_append<bf16>), grid, dim3(kPageThreads), 0, s, P);
    return PA_OK;
}

}  // namespace pa
