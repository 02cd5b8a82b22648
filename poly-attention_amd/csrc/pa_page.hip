// pa_page.hip -- the pages of a paged cache: which row has which (k_page_extend, k_page_select,
// k_page_plan), their copies (k_page_copy), and the norms and rotary of a chunk's tokens into them
// (k_page_append).
//
// A page is free where nothing refers to it, and the free pages are found by a scan in their order: no
// list has to agree with the counts of references, and which page a row gets does not depend on the
// order in which atomics arrive.
#include <algorithm>

#include "pa_draft_partial.h"
#include "pa_page.h"

namespace pa {

constexpr int kPlanThreads = 1024;  // of the kernels of one workgroup
constexpr int kPlanWaves = kPlanThreads / 64;

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
    int32_t* upto;   // [rows]
    int32_t* after;  // [rows]
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
// that ends when enough free pages are found, the writes of the table.
__global__ __launch_bounds__(kPlanThreads) void k_page_extend(const PagePlan P) {
    __shared__ int64_t s_part[kPlanWaves][2];
    __shared__ int s_tail[PA_MAX_PAGE_ROWS];  // the partly filled page that a row is about to write, or -1
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int size = 1 << P.lg;
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
            P.need[b] = want << 3 | flags;
            P.after[b] = after;
            P.upto[b] = clip(needed + s.a + want);
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
    constexpr int U = 4;
    for (int64_t p0 = 0; p0 < P.pages && found < needed; p0 += kPlanThreads * 4 * U) {
        const int64_t first = p0 + (int64_t)tid * 4 * U;
        int r[4 * U];
#pragma unroll
        for (int k = 0; k < 4 * U; ++k) r[k] = first + k < P.pages ? P.refs[first + k] : 1;
        int mine = 0;
#pragma unroll
        for (int k = 0; k < 4 * U; ++k) mine += r[k] == 0;
        const Sums s = block_sums(mine, 0, s_part, tid);
        int64_t at = found + s.a;
#pragma unroll
        for (int k = 0; k < 4 * U; ++k)
            if (r[k] == 0) {
                if (at < needed) P.list[at] = (int)(first + k);
                ++at;
            }
        found += s.all_a;
    }
    __syncthreads();
    // a wave per row
    for (int b = wave; b < P.rows; b += kPlanWaves) {
        int n, m;
        bool past;
        plan_asked(P, b, n, m, past);
        const int need = P.need[b], want = need >> 3;
        const int first = P.upto[b] - want;
        // a row that keeps a page needs the last of those that copied it to have got theirs, and so the others
        const int after = P.after[b];
        const bool ok = m > 0 && (want > 0 ? P.upto[b] <= found : after < 0 || P.upto[after] <= found);
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

// Rows as the beginnings of other rows, in two launches: what the rows become, beside the references; then
// into the table.  One workgroup per row.
__device__ __forceinline__ void select_row(const PagePlan& P, int b, int& old_pages, int& new_count, int& src) {
    src = P.index[b];
    const int size = 1 << P.lg, n = plan_count(P, b);
    old_pages = (n + size - 1) >> P.lg;
    if (src < 0 || src >= P.rows) {
        src = -1;
        new_count = 0;
        return;
    }
    new_count = plan_count(P, src);
    if (P.lengths) new_count = min(new_count, max(P.lengths[b], 0));
}
__global__ __launch_bounds__(kPageThreads) void k_page_select(const PagePlan P) {
    const int b = blockIdx.x, size = 1 << P.lg;
    int old_pages, n, src;
    select_row(P, b, old_pages, n, src);
    const int used = (n + size - 1) >> P.lg, most = max(used, old_pages);
    const int32_t* from = P.table + (int64_t)max(src, 0) * P.max_pages;
    const int32_t* own = P.table + (int64_t)b * P.max_pages;
    int32_t* to = P.copy + (int64_t)b * P.max_pages;
    for (int k = threadIdx.x; k < most; k += kPageThreads) {
        const int was = k < old_pages ? own[k] : -1, is = k < used ? from[k] : -1;
        to[k] = is;
        if (was != is) {
            if (plan_page(P, was)) atomicSub(P.refs + was, 1);
            if (plan_page(P, is)) atomicAdd(P.refs + is, 1);
        }
    }
    if (threadIdx.x == 0) P.need[b] = n;
}
__global__ __launch_bounds__(kPageThreads) void k_page_selected(const PagePlan P) {
    const int b = blockIdx.x, size = 1 << P.lg;
    const int n = P.need[b], old = plan_count(P, b);
    const int most = max((n + size - 1) >> P.lg, (old + size - 1) >> P.lg);
    int32_t* row = P.table + (int64_t)b * P.max_pages;
    const int32_t* from = P.copy + (int64_t)b * P.max_pages;
    for (int k = threadIdx.x; k < most; k += kPageThreads) row[k] = from[k];
    __syncthreads();  // the row's count has been read by every wave: it bounds the loop above
    if (threadIdx.x == 0) {
        P.counts[b] = n;
        P.fresh[b] = 0;
    }
}

// Where the pages in use go: the k-th that lies behind the first `used` places into the k-th free of those.
// One workgroup, two scans of the references.
__global__ __launch_bounds__(kPlanThreads) void k_page_plan(const PagePlan P) {
    __shared__ int64_t s_part[kPlanWaves][2];
    const int tid = threadIdx.x;
    constexpr int U = 16;
    int used = 0;
    for (int64_t p0 = 0; p0 < P.pages; p0 += kPlanThreads * U) {
        int mine = 0;
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int64_t p = p0 + (int64_t)k * kPlanThreads + tid;
            mine += p < P.pages && P.refs[p] > 0;
        }
        used += (int)block_sums(mine, 0, s_part, tid).all_a;
    }
    int holes = 0, movers = 0;
    for (int64_t p0 = 0; p0 < P.pages; p0 += kPlanThreads * U) {
        const int64_t first = p0 + (int64_t)tid * U;
        int free = 0, moving = 0, r[U];
#pragma unroll
        for (int k = 0; k < U; ++k) r[k] = first + k < P.pages ? P.refs[first + k] : 0;
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

// The moves of pages, in every array, a wave for each move, array and head; and with `remap` the table's
// entries that follow them.  Bound by memory: 16 bytes a lane, eight loads in flight.
__global__ __launch_bounds__(kPageThreads) void k_page_copy(const PagePlan P, int remap) {
    const int lane = threadIdx.x & 63;
    const int64_t waves = (int64_t)gridDim.x * (kPageThreads / 64);
    const int64_t wave = (int64_t)blockIdx.x * (kPageThreads / 64) + (threadIdx.x >> 6);
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
    const int64_t items = (int64_t)moves * P.count;
    for (int64_t it = wave; it < items; it += waves) {
        // neighbours in time copy one page's arrays
        const int mv = (int)(it / P.count), a = (int)(it - (int64_t)mv * P.count);
        const int4 m = P.moves[mv];
        const pa_page_array A = P.arrays[a];
        const int64_t head = (int64_t)A.row_bytes << P.lg, page = head * A.heads;
        const char* src = static_cast<const char*>(A.base) + m.x * page;
        char* dst = static_cast<char*>(A.base) + m.y * page;
        const int bytes = m.z * A.row_bytes;  // of a head
        if (A.row_bytes % 16 == 0) {
            constexpr int U = 8;
            const int per = bytes >> 4, all = per * A.heads;
            const int64_t skip = head - bytes;  // between heads
            for (int x0 = 0; x0 < all; x0 += 64 * U) {
                u32x4_d v[U];
                int64_t at[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int x = min(x0 + 64 * u + lane, all - 1);
                    at[u] = 16ll * x + (skip ? skip * (x / per) : 0);
                    v[u] = load16u(src + at[u]);
                }
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (x0 + 64 * u + lane < all) *reinterpret_cast<u32x4_d*>(dst + at[u]) = v[u];
            }
        } else {
            for (int h = 0; h < A.heads; ++h)
                for (int x = lane; x < m.z; x += 64)
                    reinterpret_cast<uint32_t*>(dst + h * head)[x] = reinterpret_cast<const uint32_t*>(src + h * head)[x];
        }
    }
}

// ---------------------------------------------------------------------------------------
// Norms and rotary of the chunks' tokens, into their pages.  A workgroup per token (and, where there are
// few, per tensor), a lane holding 16 bytes of a row: its features are the same in all rows, so the sines
// and cosines are computed once per lane and token.

struct PageItemDev {
    DraftRow src, out;
    const void* w;
    char* pages;
    int32_t wdt, rotate, heads;
};
struct PageRowsDev {
    PageDev p;
    int32_t dim, count, rot_dim, adt, lpr;
    float eps, interp;
    int64_t angles_sb, angles_sn;
    const void* angles;
    const float* inv_freq;
    PageItemDev it[PA_MAX_ORDER + 2];
};

template <typename T>
__global__ __launch_bounds__(kPageThreads) void k_page_append(const PageRowsDev P) {
    constexpr int E = 16 / sizeof(T), U = 2;
    const int tid = threadIdx.x, lane = tid & 63;
    int b = 0, i;
    if (P.p.packed) {
        i = blockIdx.x;
        b = page_find(P.p, i, lane);
    } else {
        b = blockIdx.x / P.p.tokens;
        i = blockIdx.x - b * P.p.tokens;
    }
    const PageRow row = page_row(P.p, b);
    const int tok = i;  // place in the inputs
    i -= row.start;
    const bool here = i >= 0 && i < row.len;
    const int64_t place = here ? page_place(P.p, b, row.p0 + i) : -1;
    const int src_b = P.p.packed ? 0 : b;
    const int sub = tid & (P.lpr - 1), d0 = sub * E;
    const bool in = d0 < P.dim;
    const int per = kPageThreads / P.lpr, first = tid / P.lpr;
    float cs[E], sn[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        cs[e] = 1.f;
        sn[e] = 0.f;
    }
    if (P.rot_dim > 0 && here) {
        float a[E];
        if (P.angles) {
            const int64_t at = src_b * P.angles_sb + tok * P.angles_sn;
#pragma unroll
            for (int e = 0; e < E; ++e)
                a[e] = d0 + e < P.rot_dim ? load_any(P.angles, P.adt, at + d0 + e) : 0.f;
        } else {  // the position as the rotary module builds it, rounded to the rows' type
            const float pos = round_to<T>(round_to<T>((float)(row.p0 + i)) / P.interp);
#pragma unroll
            for (int e = 0; e < E; ++e) a[e] = d0 + e < P.rot_dim ? pos * P.inv_freq[(d0 + e) >> 1] : 0.f;
        }
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            sincosf(a[e], &sn[e], &cs[e]);
            sn[e + 1] = sn[e];
            cs[e + 1] = cs[e];
            // a pair's features usually turn by one angle
            if (a[e + 1] != a[e]) sincosf(a[e + 1], &sn[e + 1], &cs[e + 1]);
        }
    }
    const int64_t head = (int64_t)P.dim << P.p.lg;  // elements between a page's heads
    const int64_t inside = place & ((1 << P.p.lg) - 1), id = place >> P.p.lg;
    for (int k = blockIdx.y; k < P.count; k += gridDim.y) {
        const PageItemDev& I = P.it[k];
        const T* src = I.src.at<T>(src_b, 0) + (int64_t)tok * I.src.sn + d0;
        T* out;
        int64_t sh;
        if (I.pages) {
            if (place < 0) continue;
            out = reinterpret_cast<T*>(I.pages) + id * I.heads * head + inside * P.dim + d0;
            sh = head;
        } else {
            out = I.out.at<T>(src_b, 0) + (int64_t)tok * I.out.sn + d0;
            sh = I.out.sh;
        }
        float w[E];
#pragma unroll
        for (int e = 0; e < E; ++e) w[e] = I.w && in ? load_any(I.w, I.wdt, d0 + e) : 0.f;
        const bool turn = I.rotate && P.rot_dim > 0;
        for (int h0 = first; h0 - first < I.heads; h0 += U * per) {
            u32x4_d raw[U], y[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                raw[u] = u32x4_d{0u, 0u, 0u, 0u};
                if (here && in && h0 + u * per < I.heads) raw[u] = load16u(src + (h0 + u * per) * I.src.sh);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float x[E];
                if constexpr (E == 4) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = __uint_as_float(raw[u][e]);
                } else {
                    typedef T t2 __attribute__((ext_vector_type(2)));
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t word = raw[u][e];  // a value: a bit cast of the element reads element 0
                        const t2 z = __builtin_bit_cast(t2, word);
                        x[2 * e] = (float)z[0];
                        x[2 * e + 1] = (float)z[1];
                    }
                }
                if (I.w) {
                    float ss = 0.f;
#pragma unroll
                    for (int e = 0; e < E; ++e) ss += x[e] * x[e];
                    for (int off = 1; off < P.lpr; off <<= 1) ss += __shfl_xor(ss, off);
                    const float r = rsqrtf(ss / (float)P.dim + P.eps);
#pragma unroll
                    for (int e = 0; e < E; ++e) x[e] = x[e] * r * w[e];
                }
                if (turn) {
#pragma unroll
                    for (int e = 0; e < E; e += 2) {
                        const float z = x[e] * cs[e] - x[e + 1] * sn[e];
                        x[e + 1] = x[e + 1] * cs[e + 1] + x[e] * sn[e + 1];
                        x[e] = z;
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if constexpr (E == 4) y[u][e] = __float_as_uint(x[e]);
                    else y[u][e] = draft_pack2<T>(x[2 * e], x[2 * e + 1]);
                }
                if (!here) y[u] = u32x4_d{0u, 0u, 0u, 0u};
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int h = h0 + u * per;
                if (in && h < I.heads) *reinterpret_cast<u32x4_d*>(out + h * sh) = y[u];
            }
        }
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
    P->upto = reinterpret_cast<int32_t*>(take((size_t)t.rows * 4));
    P->after = reinterpret_cast<int32_t*>(take((size_t)t.rows * 4));
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

// workgroups of the copies: four waves each, the whole card where a pool is compacted; a step's copies are few
// and mostly none
constexpr int kCopyGroups = 2048, kStepGroups = 256;

int launch_page_select(const pa_page_call* c, hipStream_t s) {
    PagePlan P;
    if (const int st = plan_dev(c, P)) return st;
    if (!P.index) return PA_EINVAL;
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

namespace {
bool page_dtype(int d) { return d == PA_F32 || d == PA_F16 || d == PA_BF16; }
bool page_dim(int d) { return d >= 8 && d <= 256 && d % 8 == 0 && (d <= 128 || d % 16 == 0); }
bool page_rows16(const pa_view& v) {
    const int E = v.dtype == PA_F32 ? 4 : 8;
    return (uintptr_t)v.ptr % 16 == 0 && v.sb % E == 0 && v.sh % E == 0 && v.sn % E == 0;
}
DraftRow page_view(const pa_view& v) {
    DraftRow r;
    r.p = static_cast<char*>(v.ptr);
    r.sb = v.sb;
    r.sh = v.sh;
    r.sn = v.sn;
    return r;
}
}  // namespace

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
    }
    const int64_t tokens = (int64_t)r->tokens * (r->packed ? 1 : r->t.rows);
    if (tokens > kPageGroups) return PA_EUNSUPPORTED;
    const dim3 grid((unsigned)tokens, tokens < 512 ? r->count : 1);
    ProfScope ps("page_append", s);
    if (T == PA_F32) hipLaunchKernelGGL((k_page_append<float>), grid, dim3(kPageThreads), 0, s, P);
    else if (T == PA_F16) hipLaunchKernelGGL((k_page_append<f16>), grid, dim3(kPageThreads), 0, s, P);
    else hipLaunchKernelGGL((k_page_append<bf16>), grid, dim3(kPageThreads), 0, s, P);
    return PA_OK;
}

}  // namespace pa
