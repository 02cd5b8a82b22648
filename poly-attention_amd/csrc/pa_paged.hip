// pa_paged.hip -- attention of chunks of new tokens over a paged cache: the join of a tile's units, and the host
// side (kernels: pa_paged_rows.h).
#include <algorithm>

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
    // a maximum that is no number is passed over above, and shows in the sums
    const float t = fmaxf(fmaxf(S.top[0], S.top[1]), fmaxf(S.top[2], S.top[3]));
    sum = 0.f;
    for (int i = 0; i < 4; ++i) y[i] = 0.f;
    for (int w = 0; w < 4; ++w) {
        if (64 * w >= see) break;  // had no position
        const float f = __builtin_amdgcn_exp2f(S.top[w] - t);
        if (f == 0.f) continue;
        sum += S.sum[w] * f;
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
__device__ __forceinline__ void paged_join_tiles(const PagedDev& P, float (*s_red)[6], SlowRow& S) {
    for (int64_t item = blockIdx.x;; item += gridDim.x) {
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

// The tiles of one unit that asked to be formed again.  Units that there are not have any flags.
template <typename T>
__device__ __forceinline__ void paged_again(const PagedDev& P, SlowRow& S) {
    const int64_t all = (int64_t)P.units * P.kv_heads;
    for (int64_t x = blockIdx.x; x < all; x += gridDim.x) {
        if (reinterpret_cast<const uint64_t*>(P.flags)[x] == 0) continue;
        PagedUnit U;
        if (!paged_find<kUnits>(P, x / P.kv_heads, threadIdx.x & 63, U) || U.splits > 1) continue;
        for (int r = U.tile * P.tile; r < min((U.tile + 1) * P.tile, U.rows); ++r)
            paged_slow<T>(P, U, (int)(x % P.kv_heads), r, S);
    }
}
template <typename T>
__global__ __launch_bounds__(kPageThreads) void k_paged_join(const PagedDev P) {
    __shared__ float s_red[kPageThreads][6];
    __shared__ SlowRow s_slow;
    if (P.recs > 0) paged_join_tiles<T>(P, s_red, s_slow);
    paged_again<T>(P, s_slow);
}

// ---------------------------------------------------------------------------------------
// host side

namespace {

bool paged_dtype(int d) { return d == PA_F32 || d == PA_F16 || d == PA_BF16; }
bool paged_dim(int d) { return d >= 8 && d <= 256 && d % 8 == 0 && (d <= 128 || d % 16 == 0); }
bool paged_rows16(const pa_view& v) {
    const int E = v.dtype == PA_F32 ? 4 : 8;
    return (uintptr_t)v.ptr % 16 == 0 && v.sb % E == 0 && v.sh % E == 0 && v.sn % E == 0;
}
DraftRow paged_view(const pa_view& v) {
    DraftRow r;
    r.p = static_cast<char*>(v.ptr);
    r.sb = v.sb;
    r.sh = v.sh;
    r.sn = v.sn;
    return r;
}

constexpr int64_t kPagedCus = 256;
// Units of k_paged_rows: each has its latencies (some 6 us alone), so they are of 64 KB of keys at least, and
// no more than there is room for at once where that leaves them at most 256 KB; beyond, twice as many, which the uneven
// ends of rows fill better.  Measured, us: 32 ragged rows of up to 8192 positions, 32/8 heads of 128, 227 so, 236 with
// three times as many, 247 with up to 512 KB; one row of 65536 116, 129 with up to 128 KB only, 109 with 512; 6 ragged
// chunks behind 5003, 12/4 heads of 128, 111, with 32 KB at least 124, 128 KB 117.
constexpr int64_t kPagedMany = 2, kPagedLarge = 256 * 1024, kPagedSmall = 64 * 1024;
// Units of k_paged_tiles: two chunks at least, and no more than there is room for at once (4 ragged chunks of 512 behind
// 2048, 32/8 heads of 128: 164 us, with twice as many 220; 512 behind 32768: 436 and 491).
constexpr int kTilesFewest = 2;
// Chunks of more query rows per key head than this go to k_paged_tiles, where it applies.  8 rows behind 4096 positions, both
// levels of order 2, 32/8 heads of 128, us: 12 tokens (48 rows at the final level) 67 so and 74 with k_paged_tiles there,
// 16 68 and 75, 24 (96 rows) 96 with k_paged_rows there and 81 so; 16 heads of 64, 40 tokens 89 so and 99.
constexpr int kPagedFewRows = 64;

// What a launch of a level takes: its tiles and their split.
struct PagedPlan {
    int64_t units;  // at most
    int tiles;      // 16-row tiles of a workgroup (few rows)
    size_t records, flags;
};

// many: the launch of k_paged_tiles, or else that of k_paged_rows; both: there is the other one too
PagedPlan paged_plan(const pa_paged* p, bool last, bool many, bool both, PagedDev& P) {
    const int rep = last ? p->heads / p->kv_heads : 1;
    const bool f32 = p->dtype == PA_F32;
    const int D = p->dim <= 64 ? 64 : p->dim <= 128 ? 128 : 256;
    const int64_t rows = (int64_t)p->tokens * rep;  // of a row of the batch, at most
    PagedPlan plan;
    plan.tiles = rows <= 16 ? 1 : f32 ? paged_row_tiles<float>(D) : paged_row_tiles<bf16>(D);
    P.rep = rep;
    P.over = many ? kPagedFewRows : 0;
    P.most = many || !both ? 1 << 30 : kPagedFewRows;
    P.tile = many ? paged_tile_rows(D) : 16 * plan.tiles;
    const int64_t flight = kPagedCus * (many ? (D == 128 ? 1 : 2) : paged_waves(D, plan.tiles));
    P.target = (int)std::max<int64_t>(1, (many ? 1 : kPagedMany) * flight / p->kv_heads);
    const int64_t chunk = (int64_t)kPagedChunk * p->dim * (f32 ? 4 : 2);  // bytes of its keys
    P.target_min = (int)std::max<int64_t>(1, flight / p->kv_heads);
    P.least = many ? 0 : (int)(kPagedLarge / chunk);
    P.fewest = many ? kTilesFewest : (int)std::max<int64_t>(1, kPagedSmall / chunk);
    // tiles of all rows: of chunks of at most P.most rows
    const int64_t each = (std::min<int64_t>(rows, P.most) + P.tile - 1) / P.tile;
    const int64_t tiles = p->packed ? std::min<int64_t>((rows + P.tile - 1) / P.tile + p->t.rows, each * p->t.rows)
                                    : each * p->t.rows;
    // no more units than tiles times the table's chunks
    const int64_t chunks = ((int64_t)p->t.max_pages * p->t.page_size + kPagedChunk - 1) / kPagedChunk;
    plan.units = std::min(tiles + P.target, tiles * chunks);
    // a tile's units are at most twice their chunks over the unit's size where there are two or more
    P.recs = chunks > 1 ? std::min<int64_t>(2 * (int64_t)P.target, tiles * chunks) : 0;
    plan.records = (size_t)P.recs * p->kv_heads * P.tile;
    plan.flags = 8 * (size_t)plan.units * p->kv_heads;
    P.units = (int)std::min<int64_t>(plan.units, 1 << 30);
    // as many rows as the workgroup has threads for (many rows: the units are few), within a tile
    P.lgr = 0;
    while (P.lgr < 4 && (((p->dim >> 2) - 1) >> (8 - P.lgr - 1)) == 0) ++P.lgr;
    return plan;
}

// Whether a level has a launch of many rows beside that of few: where chunks can have them.  The scores' initial value
// is a logsumexp over the scale, so that has to be an ordinary number.
bool paged_many(const pa_paged* p, bool last) {
    const int64_t rows = (int64_t)p->tokens * (last ? p->heads / p->kv_heads : 1);
    return p->dtype != PA_F32 && p->dim <= 128 && p->scale >= 1e-6f && p->scale <= 1e6f && rows > kPagedFewRows;
}

size_t paged_whole(size_t n) { return (n + 255) & ~size_t(255); }
size_t paged_bytes(const PagedPlan& plan, int dim) {
    return paged_whole(plan.records * dim * 4) + paged_whole(plan.records * sizeof(float2)) + paged_whole(plan.flags);
}

}  // namespace

size_t paged_attend_workspace(const pa_paged* p) {
    if (p->kv_heads < 1 || p->heads < 1 || p->tokens < 1 || p->t.rows < 1 || p->t.max_pages < 1 || !paged_dim(p->dim)) return 0;
    PagedDev P;
    size_t n = 16;
    for (int last = 0; last < 2; ++last) {
        // whatever the scale, which says whether there is a launch of many rows
        const size_t a = paged_bytes(paged_plan(p, last, false, true, P), p->dim) +
                         paged_bytes(paged_plan(p, last, true, true, P), p->dim);
        n = std::max(n, std::max(a, paged_bytes(paged_plan(p, last, false, false, P), p->dim)));
    }
    return n;
}

int launch_paged_attend(const pa_paged* p, hipStream_t s) {
    if (const int st = page_check(p->t)) return st;
    if (p->tokens < 1 || p->kv_heads < 1 || p->heads < 1 || p->heads % p->kv_heads != 0 || p->order < 2 ||
        p->order > PA_MAX_ORDER || p->dim < 1 || !paged_dtype(p->dtype))
        return PA_EINVAL;
    if (!paged_dim(p->dim)) return PA_EUNSUPPORTED;
    const int rows = p->packed ? 1 : p->t.rows;
    const int64_t rep = p->heads / p->kv_heads;
    if (p->tokens * rep > (1 << 30)) return PA_EUNSUPPORTED;
    auto view_ok = [&](const pa_view& v, int heads) { return v.ptr && v.heads == heads && v.dtype == p->dtype; };
    if (!p->tickets || p->kv_heads > PA_PAGED_TICKETS / 2) return p->tickets ? PA_EUNSUPPORTED : PA_EINVAL;
    if (!view_ok(p->q, p->heads) || !view_ok(p->out, p->heads)) return PA_EINVAL;
    if (!paged_rows16(p->q) || !paged_rows16(p->out)) return PA_EUNSUPPORTED;
    for (int t = 0; t < p->order; ++t) {
        const pa_paged_level& l = p->levels[t];
        const bool middle = t > 0 && t < p->order - 1;
        if (!l.keys || !l.values || (t < p->order - 1 && !l.lses) || (middle && !view_ok(l.vmul, p->kv_heads)))
            return PA_EINVAL;
        if ((uintptr_t)l.keys % 16 || (uintptr_t)l.values % 16 || (uintptr_t)l.lses % 16 || (middle && !paged_rows16(l.vmul)))
            return PA_EUNSUPPORTED;
    }
    PagedDev P;
    P.p = page_dev(p->t, p->tokens, p->packed != 0);
    P.kv_heads = p->kv_heads;
    P.dim = p->dim;
    P.scale = p->scale;
    P.softclamp = p->softclamp > 0.f ? p->softclamp : 0.f;
    if (!p->workspace || (uintptr_t)p->workspace % 16 != 0 || p->workspace_bytes < paged_attend_workspace(p))
        return PA_EWORKSPACE;
    P.sc = soft_clamp_dev(P.scale, P.softclamp, true);
    for (int last = 0; last < 2; ++last) {
        const bool many = paged_many(p, last);
        if (paged_plan(p, last, false, many, P).units * p->kv_heads > kPageGroups ||
            (many && paged_plan(p, last, true, true, P).units * p->kv_heads > kPageGroups))
            return PA_EUNSUPPORTED;
    }
    for (int t = 0; t < p->order; ++t) {
        const bool last = t == p->order - 1, middle_next = t + 1 < p->order - 1;
        const pa_paged_level& l = p->levels[t];
        P.last = last;
        P.q = paged_view(p->q);
        P.out = paged_view(p->out);
        P.vmul = DraftRow{nullptr, 0, 0, 0};
        if (middle_next) P.vmul = paged_view(p->levels[t + 1].vmul);
        P.keys = static_cast<const char*>(l.keys);
        P.values = static_cast<const char*>(l.values);
        P.bias = t ? p->levels[t - 1].lses : nullptr;
        P.queries = last ? nullptr : static_cast<const char*>(p->levels[t + 1].keys);
        P.next = last ? nullptr : static_cast<char*>(p->levels[t + 1].values);
        P.lses = last ? nullptr : l.lses;
        char* ws = static_cast<char*>(p->workspace);
        auto records = [&](PagedDev& Q, const PagedPlan& plan) {
            Q.ws_o = reinterpret_cast<float*>(ws);
            char* at = ws + paged_whole(plan.records * p->dim * 4);
            Q.ws_s = reinterpret_cast<float2*>(at);
            Q.flags = reinterpret_cast<uint8_t*>(at + paged_whole(plan.records * sizeof(float2)));
            ws += paged_bytes(plan, p->dim);
        };
        const bool many = paged_many(p, last);
        {
            PagedDev A = P;
            const PagedPlan plan = paged_plan(p, last, false, many, A);
            records(A, plan);
            A.tickets = p->tickets;
            // the final level's launch clears the outputs of tokens behind their chunk, too
            const int clear = last ? (int)std::min<int64_t>(((int64_t)p->tokens * rows + 3) / 4, 512) : 0;
            ProfScope ps("paged_rows", s);
            if (p->dtype == PA_F32) launch_paged_rows<float>(A, plan.units, clear, plan.tiles, s);
            else if (p->dtype == PA_F16) launch_paged_rows<f16>(A, plan.units, clear, plan.tiles, s);
            else launch_paged_rows<bf16>(A, plan.units, clear, plan.tiles, s);
        }
        if (many) {
            PagedDev B = P;
            const PagedPlan plan = paged_plan(p, last, true, true, B);
            records(B, plan);
            {
                ProfScope ps("paged_tiles", s);
                if (p->dtype == PA_F16) launch_paged_tiles<f16>(B, plan.units, s);
                else launch_paged_tiles<bf16>(B, plan.units, s);
            }
            const int64_t blocks = ((int64_t)p->tokens * rows * B.rep >> B.lgr) + p->t.rows;
            const dim3 grid((unsigned)std::min<int64_t>(blocks * p->kv_heads, 2048)), block(kPageThreads);
            ProfScope ps("paged_join", s);
            if (p->dtype == PA_F16) hipLaunchKernelGGL((k_paged_join<f16>), grid, block, 0, s, B);
            else hipLaunchKernelGGL((k_paged_join<bf16>), grid, block, 0, s, B);
        }
    }
    return PA_OK;
}

}  // namespace pa
