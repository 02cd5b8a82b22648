// pa_paged.hip -- attention of chunks of new tokens over a paged cache, the host side (kernels: pa_paged_rows.h,
// pa_paged_tiles.h).
#include <algorithm>

#include "pa_paged_join.h"

namespace pa {

template <typename T>
__global__ __launch_bounds__(kPageThreads) void k_paged_join(const PagedDev P) {
    __shared__ float s_red[kPageThreads][6];
    __shared__ SlowRow s_slow;
    if (P.recs > 0) paged_join_tiles<T>(P, blockIdx.x, gridDim.x, s_red, s_slow);
    paged_again<T>(P, blockIdx.x, gridDim.x, s_slow);
}

namespace {

constexpr int64_t kPagedCus = 256;
// Units of k_paged_rows: each has its latencies (some 6 us alone), so they are of 64 KB of keys at least, and
// no more than there is room for at once where that leaves them at most 256 KB; beyond, twice as many, which the uneven
// ends of rows fill better.  Measured, us: 32 ragged rows of up to 8192 positions, 32/8 heads of 128, 227 so, 266 with
// only as many as there is room for, 234 with three times as many, 244 with up to 512 KB; one row of 65536 109, with up to
// 128 KB 119, 512 KB 106.  With 128 KB at least 6 ragged chunks behind 5003, 12/4 heads of 128, 83 and 75 so; fp32
// chunks behind 1111, 8/2 heads of 96, 69 and 63.
constexpr int64_t kPagedMany = 2, kPagedLarge = 256 * 1024, kPagedSmall = 64 * 1024;
// Units of k_paged_tiles: two chunks at least, and no more than there is room for at once (4 ragged chunks of 512 behind
// 2048, 32/8 heads of 128: 171 us, with twice as many 237; 512 behind 32768: 483 and 525; a prompt's 512 among 15 tokens, order
// 3, 16 heads of 64: 150, with four chunks at least 171).
constexpr int kTilesFewest = 2;
// Up to so many workgroups that join tiles share the launch of the few rows', behind those: 512 of them beside 15 rows' tokens
// (order 3, 16 heads of 64) 150 us so, 165 in a launch of their own; beside idle ones (8 rows' 24 tokens behind 2048, 32/8 heads
// of 128) 66 and 61.  More would wait for that launch's registers: 2048 of 4096 tokens behind 4096 658 us so and 640 in their own.
constexpr int kPagedJoins = 1024;
// Chunks of more query rows per key head than this go to k_paged_tiles, where it applies.  8 rows behind 4096 positions, both
// levels of order 2, us: 32/8 heads of 128, 12 tokens (48 rows at the final level) 68 so and 70 with k_paged_tiles there,
// 64 tokens (64 rows at the first) 109 and 118, 24 (96 rows) 97 with k_paged_rows there and 82 so; 16 heads of 64, 40
// tokens 88 so and 98.
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
    P.tile = many ? kTileRows : 16 * plan.tiles;
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
    if (p->kv_heads < 1 || p->heads < 1 || p->tokens < 1 || p->t.rows < 1 || p->t.max_pages < 1 || !page_dim(p->dim)) return 0;
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
        p->order > PA_MAX_ORDER || p->dim < 1 || !page_dtype(p->dtype))
        return PA_EINVAL;
    if (!page_dim(p->dim)) return PA_EUNSUPPORTED;
    const int rows = p->packed ? 1 : p->t.rows;
    const int64_t rep = p->heads / p->kv_heads;
    if (p->tokens * rep > (1 << 30)) return PA_EUNSUPPORTED;
    auto view_ok = [&](const pa_view& v, int heads) { return v.ptr && v.heads == heads && v.dtype == p->dtype; };
    if (!p->tickets || p->kv_heads > PA_PAGED_TICKETS / 2) return p->tickets ? PA_EUNSUPPORTED : PA_EINVAL;
    if (!view_ok(p->q, p->heads) || !view_ok(p->out, p->heads)) return PA_EINVAL;
    if (!page_rows16(p->q) || !page_rows16(p->out)) return PA_EUNSUPPORTED;
    for (int t = 0; t < p->order; ++t) {
        const pa_paged_level& l = p->levels[t];
        const bool middle = t > 0 && t < p->order - 1;
        if (!l.keys || !l.values || (t < p->order - 1 && !l.lses) || (middle && !view_ok(l.vmul, p->kv_heads)))
            return PA_EINVAL;
        if ((uintptr_t)l.keys % 16 || (uintptr_t)l.values % 16 || (uintptr_t)l.lses % 16 || (middle && !page_rows16(l.vmul)))
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
        P.q = page_view(p->q);
        P.out = page_view(p->out);
        P.vmul = DraftRow{nullptr, 0, 0, 0};
        if (middle_next) P.vmul = page_view(p->levels[t + 1].vmul);
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
        PagedDev A = P, B = P;
        const PagedPlan few = paged_plan(p, last, false, many, A);
        records(A, few);
        A.tickets = p->tickets;
        int joins = 0;
        if (many) {
            records(B, paged_plan(p, last, true, true, B));
            const int64_t blocks = ((int64_t)p->tokens * rows * B.rep >> B.lgr) + p->t.rows;
            joins = (int)std::min<int64_t>(blocks * p->kv_heads, 2048);
            {
                ProfScope ps("paged_tiles", s);
                if (p->dtype == PA_F16) launch_paged_tiles<f16>(B, B.units, s);
                else launch_paged_tiles<bf16>(B, B.units, s);
            }
            if (joins > kPagedJoins) {
                ProfScope ps("paged_join", s);
                if (p->dtype == PA_F16) hipLaunchKernelGGL((k_paged_join<f16>), dim3(joins), dim3(kPageThreads), 0, s, B);
                else hipLaunchKernelGGL((k_paged_join<bf16>), dim3(joins), dim3(kPageThreads), 0, s, B);
                joins = 0;
            }
        }
        // the final level's launch clears the outputs of tokens behind their chunk, too
        const int clear = last ? (int)std::min<int64_t>(((int64_t)p->tokens * rows + 3) / 4, 512) : 0;
        ProfScope ps("paged_rows", s);
        if (p->dtype == PA_F32) launch_paged_rows<float>(A, B, few.units, joins, clear, few.tiles, s);
        else if (p->dtype == PA_F16) launch_paged_rows<f16>(A, B, few.units, joins, clear, few.tiles, s);
        else launch_paged_rows<bf16>(A, B, few.units, joins, clear, few.tiles, s);
    }
    return PA_OK;
}

}  // namespace pa
