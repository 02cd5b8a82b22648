// pa_paged.hip -- attention of chunks of new tokens over a paged cache: the join of a tile's units, and the host
// side (kernels: pa_paged_rows.h).
#include <algorithm>

#include "pa_paged.h"

namespace pa {

// A query row of a tile that was split, per workgroup: its units dealt out over parts of the workgroup, four
// features a thread.  The final level's launch also clears the outputs of tokens behind their chunk.
template <typename T>
__global__ __launch_bounds__(kPageThreads) void k_paged_join(const PagedDev P) {
    __shared__ float s_red[kPageThreads][6];
    const int tid = threadIdx.x, lane = tid & 63;
    const int quads = P.dim >> 2;
    int lgq = 0;
    while ((1 << lgq) < quads) ++lgq;                        // at most 64
    const int parts = kPageThreads >> lgq, part = tid >> lgq, d = (tid & ((1 << lgq) - 1)) * 4;
    for (int64_t item = blockIdx.x;; item += gridDim.x) {
        const int hk = (int)(item % P.kv_heads);
        PagedUnit U;
        if (!paged_find<kRows>(P, item / P.kv_heads, lane, U)) break;
        const int live = min(U.splits, (paged_keys(P, U) + U.size * kPagedChunk - 1) / (U.size * kPagedChunk));
        if (U.rec + live > P.recs) continue;  // there are as many as there can be
        const int r = U.at - U.tile * P.tile;
        const int64_t rec = (U.rec * P.kv_heads + hk) * P.tile + r, step = (int64_t)P.kv_heads * P.tile;
        float top = -INFINITY, sum = 0.f;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
        if (d < P.dim) {
            constexpr int N = 4;
            for (int u0 = part; u0 < live; u0 += N * parts) {
                float2 ms[N];
                float4 z[N];
#pragma unroll
                for (int k = 0; k < N; ++k) {
                    const int u = min(u0 + k * parts, live - 1);
                    ms[k] = P.ws_s[rec + u * step];
                    z[k] = *reinterpret_cast<const float4*>(P.ws_o + (rec + u * step) * P.dim + d);
                }
                float t = top;
#pragma unroll
                for (int k = 0; k < N; ++k) t = u0 + k * parts < live ? fmaxf(t, ms[k].x) : t;
                const float f = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - t);
                top = t;
                sum *= f;
                y = make_float4(y.x * f, y.y * f, y.z * f, y.w * f);
#pragma unroll
                for (int k = 0; k < N; ++k) {
                    if (u0 + k * parts >= live || ms[k].x == -INFINITY) continue;
                    const float w = __builtin_amdgcn_exp2f(ms[k].x - top);
                    sum += ms[k].y * w;
                    y = make_float4(fmaf(z[k].x, w, y.x), fmaf(z[k].y, w, y.y), fmaf(z[k].z, w, y.z), fmaf(z[k].w, w, y.w));
                }
            }
        }
        float* const mine = s_red[tid];
        mine[0] = top;
        mine[1] = sum;
        mine[2] = y.x;
        mine[3] = y.y;
        mine[4] = y.z;
        mine[5] = y.w;
        __syncthreads();
        if (part == 0 && d < P.dim) {
            float t = top;
            for (int k = 1; k < parts; ++k) t = fmaxf(t, s_red[(k << lgq) + tid][0]);
            const float f0 = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - t);
            sum *= f0;
            y = make_float4(y.x * f0, y.y * f0, y.z * f0, y.w * f0);
            for (int k = 1; k < parts; ++k) {
                const float* z = s_red[(k << lgq) + tid];
                if (z[0] == -INFINITY) continue;
                const float w = __builtin_amdgcn_exp2f(z[0] - t);
                sum += z[1] * w;
                y = make_float4(fmaf(z[2], w, y.x), fmaf(z[3], w, y.y), fmaf(z[4], w, y.z), fmaf(z[5], w, y.w));
            }
            const PagedTo to = paged_to<T>(P, U, hk, U.at);
            const float inv = 1.f / sum;
            if (to.out) paged_store<T>(to, d, make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv));
            if (d == 0 && to.lse) *to.lse = (t + log2f(sum)) * kLn2;
        }
        __syncthreads();  // s_red is written again
    }
}

// Outputs of tokens behind their chunk: 0.  A wave per token.
template <typename T>
__global__ __launch_bounds__(kPageThreads) void k_paged_clear(const PagedDev P) {
    const int lane = threadIdx.x & 63;
    const int64_t all = (int64_t)P.p.tokens * (P.p.packed ? 1 : P.p.rows), step = (int64_t)gridDim.x * (kPageThreads / 64);
    for (int64_t x = (int64_t)blockIdx.x * (kPageThreads / 64) + (threadIdx.x >> 6); x < all; x += step) {
        int b, i;
        if (P.p.packed) {
            b = 0;
            i = (int)x;
            // the last row that starts at or before it
            int lo = 0, n = P.p.rows;
            while (n > 1) {
                const int half = n >> 1;
                if (P.p.starts[lo + half] <= i) {
                    lo += half;
                    n -= half;
                } else {
                    n = half;
                }
            }
            b = lo;
        } else {
            b = (int)(x / P.p.tokens);
            i = (int)(x - (int64_t)b * P.p.tokens);
        }
        const PageRow r = page_row(P.p, b);
        if (i - r.start >= 0 && i - r.start < r.len) continue;
        const int quads = P.dim >> 2, items = P.kv_heads * P.rep * quads;
        const PagedTo to = {nullptr, nullptr, nullptr};
        for (int k = lane; k < items; k += 64) {
            const int h = k / quads, d = (k - h * quads) * 4;
            PagedTo at = to;
            at.out = reinterpret_cast<char*>(P.out.at<T>(P.p.packed ? 0 : b, h) + (int64_t)i * P.out.sn);
            paged_store<T>(at, d, make_float4(0.f, 0.f, 0.f, 0.f));
        }
    }
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

constexpr int64_t kPagedCus = 256, kPagedMany = 4, kPagedFew = 2, kPagedUnitBytes = 64 * 1024;

// What a level's launch takes: its tiles and their split.
struct PagedPlan {
    int64_t units;  // at most
    int tiles;      // 16-row tiles of a workgroup
    size_t bytes;   // of its records
};

PagedPlan paged_plan(const pa_paged* p, bool last, PagedDev& P) {
    const int rep = last ? p->heads / p->kv_heads : 1;
    const bool f32 = p->dtype == PA_F32;
    const int D = p->dim <= 64 ? 64 : p->dim <= 128 ? 128 : 256;
    const int64_t rows = (int64_t)p->tokens * rep;  // of a row of the batch, at most
    PagedPlan plan;
    plan.tiles = rows <= 16 ? 1 : f32 ? paged_row_tiles<float>(D) : paged_row_tiles<bf16>(D);
    P.rep = rep;
    P.over = 0;
    P.most = 1 << 30;
    P.tile = 16 * plan.tiles;
    const int64_t flight = kPagedCus * paged_waves(D, plan.tiles);
    P.target = (int)std::max<int64_t>(1, kPagedMany * flight / p->kv_heads);
    P.target_min = (int)std::max<int64_t>(1, kPagedFew * flight / p->kv_heads);
    P.least = std::max(1, (int)(kPagedUnitBytes * plan.tiles / ((int64_t)kPagedChunk * p->dim * (f32 ? 4 : 2))));
    const int64_t tiles = p->packed ? (rows + P.tile - 1) / P.tile + p->t.rows : (rows + P.tile - 1) / P.tile * p->t.rows;
    // no more units than tiles times the table's chunks
    const int64_t chunks = ((int64_t)p->t.max_pages * p->t.page_size + kPagedChunk - 1) / kPagedChunk;
    plan.units = std::min(tiles + P.target, tiles * chunks);
    // a tile's units are at most twice their chunks over the unit's size where there are two or more
    P.recs = chunks > 1 ? std::min<int64_t>(2 * (int64_t)P.target, tiles * chunks) : 0;
    plan.bytes = (size_t)P.recs * p->kv_heads * P.tile;  // records
    return plan;
}

size_t paged_bytes(size_t records, int dim) { return ((records * dim * 4 + 255) & ~size_t(255)) + records * sizeof(float2); }

}  // namespace

size_t paged_attend_workspace(const pa_paged* p) {
    if (p->kv_heads < 1 || p->heads < 1 || p->tokens < 1 || p->t.rows < 1 || p->t.max_pages < 1 || !paged_dim(p->dim)) return 0;
    PagedDev P;
    size_t n = 16;
    for (int last = 0; last < 2; ++last) n = std::max(n, paged_bytes(paged_plan(p, last, P).bytes, p->dim));
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
    for (int t = 0; t < p->order; ++t) {
        const bool last = t == p->order - 1;
        const PagedPlan plan = paged_plan(p, last, P);
        if (plan.units * p->kv_heads > kPageGroups) return PA_EUNSUPPORTED;
    }
    for (int t = 0; t < p->order; ++t) {
        const bool last = t == p->order - 1, middle_next = t + 1 < p->order - 1;
        const pa_paged_level& l = p->levels[t];
        const PagedPlan plan = paged_plan(p, last, P);
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
        P.ws_o = static_cast<float*>(p->workspace);
        P.ws_s = reinterpret_cast<float2*>(static_cast<char*>(p->workspace) + ((plan.bytes * p->dim * 4 + 255) & ~size_t(255)));
        {
            ProfScope ps("paged_rows", s);
            if (p->dtype == PA_F32) launch_paged_rows<float>(P, plan.units, plan.tiles, s);
            else if (p->dtype == PA_F16) launch_paged_rows<f16>(P, plan.units, plan.tiles, s);
            else launch_paged_rows<bf16>(P, plan.units, plan.tiles, s);
        }
        if (P.recs > 0) {
            const int64_t items = std::min<int64_t>(P.recs * P.tile, (int64_t)p->tokens * rep * rows) * p->kv_heads;
            const dim3 grid((unsigned)std::min<int64_t>(items, 2048)), block(kPageThreads);
            ProfScope ps("paged_join", s);
            if (p->dtype == PA_F32) hipLaunchKernelGGL((k_paged_join<float>), grid, block, 0, s, P);
            else if (p->dtype == PA_F16) hipLaunchKernelGGL((k_paged_join<f16>), grid, block, 0, s, P);
            else hipLaunchKernelGGL((k_paged_join<bf16>), grid, block, 0, s, P);
        }
    }
    const int64_t tokens = (int64_t)p->tokens * rows;
    const dim3 grid((unsigned)std::min<int64_t>((tokens + 3) / 4, 1024)), block(kPageThreads);
    ProfScope ps("paged_clear", s);
    if (p->dtype == PA_F32) hipLaunchKernelGGL((k_paged_clear<float>), grid, block, 0, s, P);
    else if (p->dtype == PA_F16) hipLaunchKernelGGL((k_paged_clear<f16>), grid, block, 0, s, P);
    else hipLaunchKernelGGL((k_paged_clear<bf16>), grid, block, 0, s, P);
    return PA_OK;
}

}  // namespace pa
