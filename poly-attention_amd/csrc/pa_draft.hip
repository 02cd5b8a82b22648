// pa_draft.hip -- the rest of a drafted step: the join of the units with the tree part
// (k_draft_combine), norms, rotary and draft slots (k_draft_append), the move of the kept nodes
// (k_draft_commit), and the host side of these entry points.
#include <algorithm>

#include "pa_draft_partial.h"

namespace pa {

// ---------------------------------------------------------------------------------------
// One workgroup per (batch row and key head, P.cols columns of the head, up to 64 rows of the final
// level).  First, for all levels at once, the units of the cached positions are joined (a row's
// maximum, sum and the workgroup's columns); then the levels, deepest first: the tree's scores get the
// deeper level's logsumexps, their softmax is joined with the units' and the columns with the tree's
// values.  The levels below the final one have at most 64 rows and are repeated by every row block.
// What bounds it is latency: loads are issued in batches and the next level's scores are loaded before
// this one's are used.  Many rows of a large tree are bound by reading the values from LDS: two rows at once
// and no test per value took 8 rows of 64 nodes of 4 heads (128 columns) from 51 to 41 us; up to 16 nodes
// the shorter code is faster (8.9 against 9.5 us, five nodes).
// Code that runs for the first time waits for its instructions too, and a level's arguments for the
// scalar cache: the score loops are as long as the tree needs (NK), the arguments are read into LDS
// beside the first loads, and nothing divides by a number that is not known before.
constexpr int kDraftBatch = 8;  // units whose records a thread loads together

struct JoinedRow {
    float top, sum;
    float4 acc;
};
__device__ __forceinline__ float exp2_or_0(float x, float top) {
    return x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(x - top);
}
__device__ __forceinline__ void join(JoinedRow& a, float f, float sum, const float4& acc) {
    a.sum += sum * f;
    a.acc.x += acc.x * f;
    a.acc.y += acc.y * f;
    a.acc.z += acc.z * f;
    a.acc.w += acc.w * f;
}
__device__ __forceinline__ void fma4(float4& y, float w, const float4& z) {
    y.x = fmaf(w, z.x, y.x);
    y.y = fmaf(w, z.y, y.y);
    y.z = fmaf(w, z.z, y.z);
    y.w = fmaf(w, z.w, y.w);
}
__device__ __forceinline__ bool finite(const float4& z) {
    return z.x * 0.f + z.y * 0.f + z.z * 0.f + z.w * 0.f == 0.f;
}
__device__ __forceinline__ void raise(JoinedRow& a, float top) {
    const float f = exp2_or_0(a.top, top);
    a.top = top;
    a.sum *= f;
    a.acc = make_float4(a.acc.x * f, a.acc.y * f, a.acc.z * f, a.acc.w * f);
}

template <typename T>
__device__ __forceinline__ float4 load4f(const T* p) {
    if constexpr (sizeof(T) == 4) {
        return *reinterpret_cast<const float4*>(p);
    } else {
        typedef T t4 __attribute__((ext_vector_type(4)));
        const t4 x = *reinterpret_cast<const t4*>(p);
        return make_float4((float)x[0], (float)x[1], (float)x[2], (float)x[3]);
    }
}
template <typename T>
__device__ __forceinline__ void store4f(T* p, const float4& y) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(p) = y;
    } else {
        u32x2_d w;
        w[0] = draft_pack2<T>(y.x, y.y);
        w[1] = draft_pack2<T>(y.z, y.w);
        *reinterpret_cast<u32x2_d*>(p) = w;
    }
}

template <typename T, int NK>
__global__ __launch_bounds__(kDraftThreads) void k_draft_combine(const DraftJoin P) {
    extern __shared__ __align__(16) float smem[];
    __shared__ float s_bias[64], s_top[64], s_inv[64], s_utop[64 * PA_MAX_ORDER], s_usum[64 * PA_MAX_ORDER];
    __shared__ int s_odd[kDraftThreads / 64];
    __shared__ __align__(16) DraftJoinLevel s_lvl[PA_MAX_ORDER];
    const int tid = threadIdx.x;
    const int b = blockIdx.x / P.kv_heads, hk = blockIdx.x % P.kv_heads;
    const int col0 = blockIdx.y << P.lgcols, ncol = min(1 << P.lgcols, P.dim - col0);
    const int last = P.order - 1, low = P.T * last;  // rows of the levels below the final one
    const int r0 = blockIdx.z * 64, frows = min(64, P.T * P.rep - r0);
    const int rows_all = low + frows;
    const int lgq = P.lgcols - 2;                  // a row's items: four columns each
    const int spitch = P.t16 + 4, vpitch = (1 << P.lgcols) + 4;
    float* const s_acc = smem;                     // [rows_all][cols]: the joined units
    float* const s_p = s_acc + (rows_all << P.lgcols);  // [64][spitch]: weights of the tree
    float* s_in = s_p + 64 * spitch;               // [t16][vpitch]: a level's tree values
    float* s_out = s_in + P.t16 * vpitch;          // [t16][vpitch]: its outputs
    float* const s_red = s_in;                     // before the levels: 256 x 6

    const int4 units = P.ws_u[b];
    // Four threads per row take the tree's scores of a level, every fourth one each; a thread's item is a
    // row and four columns.  Both for a level ahead.
    const int row = tid >> 2, sub = tid & 3;
    const int ir = tid >> lgq, id = (tid & ((1 << lgq) - 1)) * 4;
    const float* const scores = P.ws_t + ((int64_t)blockIdx.x * P.rec_rows + row) * P.t16 + sub;
    float s[NK];
    auto load_scores = [&](int t) __attribute__((always_inline)) {
        const int n = t == last ? frows : P.T;
        const float* from = scores + (t * P.T + (t == last ? r0 : 0)) * P.t16;
#pragma unroll
        for (int k = 0; k < NK; ++k) s[k] = row < n && 4 * k < P.t16 ? from[4 * k] : -INFINITY;
    };
    load_scores(0);
    float4 val = make_float4(0.f, 0.f, 0.f, 0.f);
    if (ir < P.T && id < ncol) val = load4f<T>(P.L[0].dv.template at<T>(b, hk) + ir * P.L[0].dv.sn + col0 + id);
    {
        constexpr int W = sizeof(DraftJoinLevel) / 4;
        static_assert(W * PA_MAX_ORDER <= kDraftThreads, "one word per thread");
        if (tid < W * P.order)
            reinterpret_cast<uint32_t*>(s_lvl)[tid] = reinterpret_cast<const uint32_t*>(P.L)[tid];
    }

    {   // the units: an item's are dealt out over `parts` threads where there are few items
        const int64_t urec = (int64_t)P.kv_heads * P.rec_rows;  // records between units
        const int64_t rec0 = ((int64_t)units.x * P.kv_heads + hk) * P.rec_rows;
        const int items = rows_all << lgq;
        int lgp = 0;
        while (lgp < 4 && items << (lgp + 1) <= kDraftThreads && 2 << lgp <= units.y) ++lgp;
        // with parts, a part's items lie in `stride` threads
        const int stride = kDraftThreads >> lgp, part = tid / stride;  // a power of two
        for (int x0 = 0; x0 < items; x0 += stride) {
            const int item = x0 + (tid & (stride - 1)), ra = item >> lgq, d = (item & ((1 << lgq) - 1)) * 4;
            JoinedRow a = {-INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
            if (item < items && d < ncol) {
                const int64_t rec = rec0 + ra + (ra < low ? 0 : r0);
                const float* const from = P.ws_o + col0 + d;
                for (int u = part; u < units.y; u += kDraftBatch << lgp) {
                    float2 ms[kDraftBatch];
                    float4 y[kDraftBatch];
#pragma unroll
                    for (int k = 0; k < kDraftBatch; ++k) {
                        const int64_t at = u + (k << lgp) < units.y ? rec + (int64_t)(u + (k << lgp)) * urec : P.none;
                        ms[k] = P.ws_s[at];
                        y[k] = *reinterpret_cast<const float4*>(from + at * P.dim);
                    }
                    float top = a.top;
#pragma unroll
                    for (int k = 0; k < kDraftBatch; ++k) top = fmaxf(top, ms[k].x);
                    raise(a, top);
#pragma unroll
                    for (int k = 0; k < kDraftBatch; ++k) join(a, exp2_or_0(ms[k].x, top), ms[k].y, y[k]);
                }
            }
            if (lgp) {
                float* r = s_red + tid * 6;
                r[0] = a.top;
                r[1] = a.sum;
                r[2] = a.acc.x;
                r[3] = a.acc.y;
                r[4] = a.acc.z;
                r[5] = a.acc.w;
                __syncthreads();
                if (part == 0 && item < items) {
                    float top = a.top;
                    for (int k = 1; k < 1 << lgp; ++k) top = fmaxf(top, s_red[(tid + k * stride) * 6]);
                    raise(a, top);
                    for (int k = 1; k < 1 << lgp; ++k) {
                        const float* z = s_red + (tid + k * stride) * 6;
                        join(a, exp2_or_0(z[0], top), z[1], make_float4(z[2], z[3], z[4], z[5]));
                    }
                }
            }
            if (part == 0 && item < items && d < ncol) {
                *reinterpret_cast<float4*>(s_acc + (ra << P.lgcols) + d) = a.acc;
                if (d == 0) {
                    s_utop[ra] = a.top;
                    s_usum[ra] = a.sum;
                }
            }
        }
    }
    const uint64_t live = ((uint64_t)(uint32_t)units.w << 32) | (uint32_t)units.z;
    __syncthreads();

    bool odd = false;  // a value of the next level's that is not finite
    for (int t = 0; t <= last; ++t) {
        const DraftJoinLevel& L = s_lvl[t];
        const bool fin = t == last;
        const int rows = fin ? frows : P.T, ra0 = t * P.T, rr = fin ? r0 : 0;
        // the tree's values: v, v * msg, or msg (already in s_in, as the level below left it)
        if (!fin)
            for (int n = ir; n < P.T; n += kDraftThreads >> lgq) {
                if (id >= ncol) break;
                float4 y = val;
                if (n != ir) y = load4f<T>(L.dv.template at<T>(b, hk) + n * L.dv.sn + col0 + id);
                float4* at = reinterpret_cast<float4*>(&s_in[n * vpitch + id]);
                if (t > 0) {
                    const float4 z = *at;
                    y = make_float4(y.x * z.x, y.y * z.y, y.z * z.z, y.w * z.w);
                }
                *at = y;
                if (NK > 4) odd = odd || !finite(y);
            }
        if constexpr (NK > 4) {
            if (t == 0)  // no node: weight 0
                for (int n = P.T + ir; n < ((P.T + 3) & ~3); n += kDraftThreads >> lgq) {
                    *reinterpret_cast<float4*>(&s_in[n * vpitch + id]) = make_float4(0.f, 0.f, 0.f, 0.f);
                    *reinterpret_cast<float4*>(&s_out[n * vpitch + id]) = make_float4(0.f, 0.f, 0.f, 0.f);
                }
            const int any = __any(odd);
            if ((tid & 63) == 0) s_odd[tid >> 6] = any;
            odd = false;
        }
        // maximum and sum over the units and the tree
        const float utop = row < rows ? s_utop[ra0 + row] : -INFINITY;
        float top = utop, sum = 0.f;
        if (t > 0) {
#pragma unroll
            for (int k = 0; k < NK; ++k)  // what a node does not see stays -inf, whatever its logsumexp
                s[k] = s[k] == -INFINITY ? s[k] : s[k] + s_bias[4 * k + sub];
        }
#pragma unroll
        for (int k = 0; k < NK; ++k) top = fmaxf(top, s[k]);
        top = fmaxf(top, __shfl_xor(top, 1));
        top = fmaxf(top, __shfl_xor(top, 2));
#pragma unroll
        for (int k = 0; k < NK; ++k) {
            const float p = exp2_or_0(s[k], top);
            if (row < rows && 4 * k < P.t16) s_p[row * spitch + 4 * k + sub] = p;
            sum += p;
        }
        if (!fin) {
            load_scores(t + 1);
            const DraftJoinLevel& N = s_lvl[t + 1];
            if (t + 1 < last && ir < P.T && id < ncol)
                val = load4f<T>(N.dv.template at<T>(b, hk) + ir * N.dv.sn + col0 + id);
        }
        sum += __shfl_xor(sum, 1);
        sum += __shfl_xor(sum, 2);
        __syncthreads();  // every s_bias has been read
        if (sub == 0) {
            float lse = 0.f;
            if (row < rows) {
                const float f = exp2_or_0(utop, top);
                sum += s_usum[ra0 + row] * f;
                int n = row;
                if (fin) n = (rr + row) % P.T;
                const bool here = (live >> n) & 1;
                s_top[row] = f;
                s_inv[row] = here ? 1.f / sum : 0.f;
                if (!fin && here) lse = top + log2f(sum);
                if (!fin && blockIdx.y == 0 && blockIdx.z == 0) L.lse[b * L.lse_sb + hk * L.lse_sh + row] = lse * kLn2;
            }
            s_bias[row] = lse;
        }
        __syncthreads();
        const int step = kDraftThreads >> lgq;
        auto units_part = [&](int r) __attribute__((always_inline)) -> float4 {
            const float f = s_top[r];
            const float4 u = *reinterpret_cast<const float4*>(s_acc + ((ra0 + r) << P.lgcols) + id);
            return f != 0.f ? make_float4(u.x * f, u.y * f, u.z * f, u.w * f) : make_float4(0.f, 0.f, 0.f, 0.f);
        };
        auto finish = [&](int r, float4 y) __attribute__((always_inline)) {
            // an absent node's row: 0, whatever its query was
            const float inv = s_inv[r];
            y = inv != 0.f ? make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv) : make_float4(0.f, 0.f, 0.f, 0.f);
            if (!fin) *reinterpret_cast<float4*>(&s_out[r * vpitch + id]) = y;
            if (NK > 4) odd = odd || !finite(y);
            if (fin || blockIdx.z == 0) {
                int h = hk, n = r;
                if (fin) {
                    h = (rr + r) / P.T;
                    n = rr + r - h * P.T;
                    h += hk * P.rep;
                }
                store4f<T>(L.out.template at<T>(b, h) + n * L.out.sn + col0 + id, y);
            }
        };
        if (id < ncol) {
            if (NK == 4 || (s_odd[0] | s_odd[1] | s_odd[2] | s_odd[3])) {
                for (int r = ir; r < rows; r += step) {
                    float4 y = units_part(r);
                    for (int k0 = 0; k0 < P.T; k0 += 4) {
                        const float4 p = *reinterpret_cast<const float4*>(&s_p[r * spitch + k0]);
                        const float w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const float4 z = *reinterpret_cast<const float4*>(&s_in[(k0 + k) * vpitch + id]);
                            // what a node does not see (another branch, a slot past the nodes) may hold anything
                            const bool see = w[k] != 0.f;
                            fma4(y, w[k], make_float4(see ? z.x : 0.f, see ? z.y : 0.f, see ? z.z : 0.f, see ? z.w : 0.f));
                        }
                    }
                    finish(r, y);
                }
            } else if (rows <= step) {  // nothing but numbers: no test per value ...
                if (ir < rows) {
                    float4 y = units_part(ir);
                    for (int k0 = 0; k0 < P.T; k0 += 4) {
                        const float4 p = *reinterpret_cast<const float4*>(&s_p[ir * spitch + k0]);
                        const float w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
                        for (int k = 0; k < 4; ++k) fma4(y, w[k], *reinterpret_cast<const float4*>(&s_in[(k0 + k) * vpitch + id]));
                    }
                    finish(ir, y);
                }
            } else {  // ... and two rows take the values together
                for (int r = ir; r < rows; r += 2 * step) {
                    const int r2 = min(r + step, rows - 1);
                    float4 y = units_part(r), y2 = units_part(r2);
                    for (int k0 = 0; k0 < P.T; k0 += 4) {
                        const float4 p = *reinterpret_cast<const float4*>(&s_p[r * spitch + k0]);
                        const float4 p2 = *reinterpret_cast<const float4*>(&s_p[r2 * spitch + k0]);
                        const float w[4] = {p.x, p.y, p.z, p.w}, w2[4] = {p2.x, p2.y, p2.z, p2.w};
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const float4 z = *reinterpret_cast<const float4*>(&s_in[(k0 + k) * vpitch + id]);
                            fma4(y, w[k], z);
                            fma4(y2, w2[k], z);
                        }
                    }
                    finish(r, y);
                    if (r + step < rows) finish(r2, y2);
                }
            }
        }
        __syncthreads();
        float* const done = s_out;  // this level's outputs are the next one's values
        s_out = s_in;
        s_in = done;
    }
}

template <typename T>
void launch_combine(const DraftJoin& P, dim3 grid, size_t lds, hipStream_t s) {
    if (P.t16 == 16) hipLaunchKernelGGL((k_draft_combine<T, 4>), grid, dim3(kDraftThreads), lds, s, P);
    else if (P.t16 == 32) hipLaunchKernelGGL((k_draft_combine<T, 8>), grid, dim3(kDraftThreads), lds, s, P);
    else hipLaunchKernelGGL((k_draft_combine<T, 16>), grid, dim3(kDraftThreads), lds, s, P);
}

// ---------------------------------------------------------------------------------------
// Norms and rotary of a step's nodes into their draft slots.  One workgroup per (node, tensor), a lane
// holding 16 bytes of a row: a lane's features are the same in all its rows, so the sines and cosines
// are computed once per lane (they cost more than the rows), while the first rows are on their way.  Bound by
// that one chain: 32 x 8 nodes of 32 + 3 x 8 heads of 128 take 5.8 us, 5 nodes of 8 heads of 64 5.2.

struct DraftItemDev {
    DraftRow src, out;
    const void* w;
    int32_t wdt, rotate, heads;
};
struct DraftRowsDev {
    int32_t batch, T, dim, count, rot_dim, adt, lpr;
    float eps, interp;
    const int32_t* counts;
    const int32_t* parents;
    int64_t parents_stride, angles_sb, angles_sn;
    const void* angles;
    const float* inv_freq;
    DraftItemDev it[2 * PA_MAX_ORDER];
};

// E values of any of the types from p[i]
template <int E>
__device__ __forceinline__ void load_row(const void* p, int dtype, int64_t i, float (&x)[E]) {
    if (dtype == PA_F32) {
        __builtin_memcpy(x, static_cast<const float*>(p) + i, sizeof(x));
    } else if (dtype == PA_F16) {
        f16 r[E];
        __builtin_memcpy(r, static_cast<const f16*>(p) + i, sizeof(r));
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = to_f(r[e]);
    } else {
        bf16 r[E];
        __builtin_memcpy(r, static_cast<const bf16*>(p) + i, sizeof(r));
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = to_f(r[e]);
    }
}

template <typename T>
__global__ __launch_bounds__(kDraftThreads) void k_draft_append(const DraftRowsDev P) {
    constexpr int E = 16 / sizeof(T), U = 2;  // rows of a thread in flight
    const int tid = threadIdx.x, lane = tid & 63;
    const int b = blockIdx.x / P.T, t = blockIdx.x % P.T;
    const DraftItemDev& I = P.it[blockIdx.y];
    const int sub = tid & (P.lpr - 1), d0 = sub * E;
    const bool in = d0 < P.dim;
    const int per = kDraftThreads / P.lpr, first = tid / P.lpr;  // rows (heads) at a time
    const T* src = I.src.at<T>(b, 0) + t * I.src.sn + d0;
    T* out = I.out.at<T>(b, 0) + t * I.out.sn + d0;
    u32x4_d raw[U];
    auto fetch = [&](int h0) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            raw[u] = u32x4_d{0u, 0u, 0u, 0u};
            if (in && h0 + u * per < I.heads) raw[u] = load16u(src + (h0 + u * per) * I.src.sh);
        }
    };
    fetch(first);
    float w[E], cs[E], sn[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        w[e] = 0.f;
        cs[e] = 1.f;
        sn[e] = 0.f;
    }
    if (I.w && in) load_row<E>(I.w, I.wdt, d0, w);
    const bool turn = I.rotate && P.rot_dim > 0;
    if (turn) {
        float a[E];
        if (P.angles) {
            const int64_t at = b * P.angles_sb + t * P.angles_sn;
            if (d0 + E <= P.rot_dim) {
                load_row<E>(P.angles, P.adt, at + d0, a);
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e)
                    a[e] = d0 + e < P.rot_dim ? load_any(P.angles, P.adt, at + d0 + e) : 0.f;
            }
        } else {  // the position as the rotary module builds it, rounded to the rows' type
            const uint64_t anc = draft_ancestors(P.parents ? P.parents + b * P.parents_stride : nullptr,
                                                 P.T, lane);
            const int depth = __popcll(anc) - 1;
            const int mine = max(0, __shfl(depth, t));
            const float pos = round_to<T>(round_to<T>((float)(P.counts[b] + mine)) / P.interp);
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
    for (int h0 = 0; h0 < I.heads; h0 += U * per) {
        u32x4_d y[U];
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
        }
        fetch(first + h0 + U * per);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int h = first + h0 + u * per;
            if (in && h < I.heads) *reinterpret_cast<u32x4_d*>(out + h * I.out.sh) = y[u];
        }
    }
}

// ---------------------------------------------------------------------------------------
// The kept nodes of a row, from their draft slots to the positions behind the cached ones.

struct DraftCommitDev {
    int32_t batch, kv_heads, slots, capacity, path_len, count, advance;
    const int32_t* path;
    int64_t path_stride;
    const int32_t* kept;
    int32_t* counts;
    int32_t* overflow;
    int32_t* tickets;
    pa_draft_move mv[PA_MAX_MOVES];
};

// entries of row b's path that are moved: up to the first one outside the slots, within the capacity
// (lane i's entry in p)
__device__ __forceinline__ int commit_length(const DraftCommitDev& P, int b, int lane, int& n, int& p, bool& over) {
    p = lane < P.path_len ? P.path[b * P.path_stride + lane] : -1;
    n = min(max(P.counts[b], 0), P.capacity);
    const int want = min(max(P.kept[b], 0), P.path_len);
    const uint64_t outside = __ballot(p < 0 || p >= P.slots);
    const int bad = min(want, outside ? __ffsll((unsigned long long)outside) - 1 : 64);
    over = bad > P.capacity - n;
    return min(bad, P.capacity - n);
}

// `len` rows of every head, four vectors of a thread in flight; lane i of a wave holds the slot of row i
template <typename V>
__device__ __forceinline__ void move_rows(const char* src, char* dst, int64_t sh, int64_t dh, int row_bytes, int len,
                                          int heads, int slot, int tid) {
    const unsigned per = row_bytes / sizeof(V), head = len * per;
    const unsigned all = head * heads;  // at most 64 rows of 1024 vectors and 2^14 heads
    constexpr int U = 4;
    for (unsigned x0 = 0; x0 < all; x0 += U * kDraftThreads) {
        V v[U];
        unsigned h[U], y[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const unsigned x = min(x0 + u * kDraftThreads + tid, all - 1);
            h[u] = x / head;
            y[u] = x - h[u] * head;
            const unsigned i = y[u] / per;
            v[u] = *reinterpret_cast<const V*>(src + h[u] * sh + (int64_t)__shfl(slot, (int)i) * row_bytes +
                                               (y[u] - i * per) * sizeof(V));
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (x0 + u * kDraftThreads + tid < all)
                *reinterpret_cast<V*>(dst + h[u] * dh + y[u] * sizeof(V)) = v[u];
    }
}

// One workgroup per (row, move): 8 rows of 54 buffers 4.9 us, one of 5 4.2 (paths, rows, counts: three dependent
// trips to memory).  With advance the workgroup of a row that draws the last ticket counts the
// kept nodes: by then every other one has read the count, so one launch does both.  The first wave reads it
// for the workgroup: a barrier does not wait for another wave's loads from memory, so a wave that read the
// count for itself might read the advanced one.
__global__ __launch_bounds__(kDraftThreads) void k_draft_commit(const DraftCommitDev P) {
    __shared__ int s_slot[64], s_n, s_len, s_over;
    const int tid = threadIdx.x, b = blockIdx.x;
    if (tid < 64) {
        int at, p;
        bool past;
        const int moved = commit_length(P, b, tid, at, p, past);
        s_slot[tid] = p;
        if (tid == 0) {
            s_n = at;
            s_len = moved;
            s_over = past;
        }
    }
    __syncthreads();  // past it the count has been read: the length in LDS depends on it
    const int n = s_n, len = s_len, slot = s_slot[tid & 63];
    const bool over = s_over;
    const pa_draft_move& M = P.mv[blockIdx.y];
    int done = 0;  // drawn now, looked at after the moves
    // relaxed: nothing that another workgroup wrote is read after it, and this one's read of the count has
    // returned; a release would write the L2 back, at several us
    if (P.advance && tid == 0)
        done = __hip_atomic_fetch_add(P.tickets + b * kTicketStride, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (P.count > 0 && len > 0) {
        const int unit = M.row_bytes % 16 == 0 ? 16 : 4;
        const int64_t bh = (int64_t)b * P.kv_heads;
        const char* src = static_cast<const char*>(M.src) + bh * P.slots * M.row_bytes;
        char* dst = static_cast<char*>(M.dst) + (bh * P.capacity + n) * M.row_bytes;
        const int64_t sh = (int64_t)P.slots * M.row_bytes, dh = (int64_t)P.capacity * M.row_bytes;
        if (unit == 16) move_rows<u32x4_d>(src, dst, sh, dh, M.row_bytes, len, P.kv_heads, slot, tid);
        else move_rows<uint32_t>(src, dst, sh, dh, M.row_bytes, len, P.kv_heads, slot, tid);
    }
    if (P.advance && tid == 0 && done == (int)gridDim.y - 1) {
        P.counts[b] = n + len;
        P.tickets[b * kTicketStride] = 0;
        if (over && P.overflow) *P.overflow = 1;
    }
}

// ---------------------------------------------------------------------------------------
// host side

namespace {

bool draft_dtype(int d) { return d == PA_F32 || d == PA_F16 || d == PA_BF16; }
int draft_size(int dtype) { return dtype == PA_F32 ? 4 : 2; }

// rows of 16-byte aligned starts (E elements); a stride of 0 broadcasts
bool rows16(const pa_view& v) {
    const int E = 16 / draft_size(v.dtype);
    return (uintptr_t)v.ptr % 16 == 0 && v.sb % E == 0 && v.sh % E == 0 && v.sn % E == 0;
}
DraftRow draft_row(const pa_view& v) {
    DraftRow r;
    r.p = static_cast<char*>(v.ptr);
    r.sb = v.sb;
    r.sh = v.sh;
    r.sn = v.sn;
    return r;
}

// head dims: multiples of 8, of 16 above 128 (a lane's features are whole: dim / 16 of the padded dim)
bool draft_dim(int d) { return d >= 8 && d <= 256 && d % 8 == 0 && (d <= 128 || d % 16 == 0); }

// Workgroups of the first launch aimed at, as multiples of those that are in flight together: kDraftMany,
// but kDraftFew where a unit's keys are below kDraftUnitBytes per 16 rows, since a workgroup's start
// and end and its record cost the more the more rows it has.  Behind cold caches: 32 rows of up to 8192
// positions of 128, 32 query rows: 250 us with few, 245 with many; order 3, 8 of up to 2048 of 64, 16 rows: 44 with few,
// 46 with many.  k_draft_wide, 8 x 4096 of 128: as many as are in flight 76, twice as many 81 (64 rows); 90 and 93
// (128 rows).
constexpr int64_t kDraftMany = 4, kDraftFew = 2, kDraftWideMany = 2, kDraftUnitBytes = 64 * 1024, kDraftCus = 256;

// Workgroups of a grid's first dimension, at most: its threads are counted in 32 bits, and a first launch that is
// refused would leave the second one records that nothing has written.
constexpr int64_t kDraftGroups = (int64_t(1) << 32) / kDraftThreads - 1;

// geometry shared by the workspace query and the launch; false where the request is malformed
bool draft_plan(const pa_draft* d, DraftDev& P, int& units, int& tiles) {
    if (d->batch < 1 || d->kv_heads < 1 || d->heads < 1 || d->heads % d->kv_heads != 0) return false;
    if (d->drafts < 1 || d->drafts > PA_MAX_DRAFTS || d->order < 2 || d->order > PA_MAX_ORDER) return false;
    if (d->capacity < 1 || !draft_dim(d->dim) || !draft_dtype(d->levels[0].k.dtype)) return false;
    const int rep = d->heads / d->kv_heads;
    if ((int64_t)rep * d->drafts > (1 << 20)) return false;
    P.batch = d->batch;
    P.kv_heads = d->kv_heads;
    P.T = d->drafts;
    P.dim = d->dim;
    P.order = d->order;
    P.capacity = d->capacity;
    const bool f32 = d->levels[0].k.dtype == PA_F32;
    const int D = d->dim <= 64 ? 64 : d->dim <= 128 ? 128 : 256;
    const int most = d->drafts * rep;
    const int64_t chunks = ((int64_t)d->capacity + kDraftChunk - 1) / kDraftChunk * d->batch;
    // rows of a workgroup: as many as its registers hold
    tiles = most <= 16 ? 1 : std::min(f32 ? draft_row_tiles<float>(D, d->order > 2) : draft_row_tiles<bf16>(D, d->order > 2),
                                              most <= 32 ? 2 : 4);
    const bool wide = draft_wide(D, f32, d->order > 2, most);
    if (wide) tiles = kDraftWideWaves * draft_wide_tiles(D);
    P.row_blocks = (most + 16 * tiles - 1) / (16 * tiles);
    P.rec_rows = d->drafts * (d->order - 1) + most;
    P.t16 = (d->drafts + 15) & ~15;
    const int low = (d->drafts + 16 * tiles - 1) / (16 * tiles);  // blocks of a level below the final one
    const int64_t per = (int64_t)d->kv_heads * (P.row_blocks + (d->order - 1) * low);  // workgroups per unit
    // no more units than the capacity has chunks
    const int64_t flight = kDraftCus * (wide ? 2 : draft_waves(D, tiles, d->order > 2));
    const int64_t target = std::min(std::max<int64_t>(1, (wide ? kDraftWideMany : kDraftMany) * flight / per), chunks);
    P.target = (int)target;
    // as many as are in flight, with half a unit per row that the ends of rows add
    const int64_t few = wide ? flight / per - d->batch / 2 : kDraftFew * flight / per;
    P.target_min = (int)std::min(std::max<int64_t>(1, few), chunks);
    P.least = std::max(1, (int)(kDraftUnitBytes * tiles / ((int64_t)kDraftChunk * d->dim * (f32 ? 4 : 2))));
    units = (int)std::min(target + d->batch, chunks);
    return (int64_t)d->kv_heads * P.row_blocks <= 65535 && (int64_t)d->batch * d->kv_heads <= kDraftGroups &&
           (int64_t)d->batch + units <= kDraftGroups;
}

// the workspace's arrays, and its size
size_t draft_ws(DraftCommon& P, int units, void* base) {
    auto whole = [](size_t n) { return (n + 255) & ~size_t(255); };
    P.none = (int64_t)units * P.kv_heads * P.rec_rows;
    const size_t rec = (size_t)P.none + 1;
    char* at = static_cast<char*>(base);
    P.ws_o = reinterpret_cast<float*>(at);
    size_t n = whole(rec * P.dim * 4);
    P.ws_s = reinterpret_cast<float2*>(at + n);
    n += whole(rec * sizeof(float2));
    P.ws_t = reinterpret_cast<float*>(at + n);
    n += whole((size_t)P.batch * P.kv_heads * P.rec_rows * P.t16 * 4);
    P.ws_u = reinterpret_cast<int4*>(at + n);
    return n + (size_t)P.batch * sizeof(int4);
}

// LDS of the combine with 2^lg columns
size_t combine_lds(const DraftCommon& P, int lg) {
    const int cols = 1 << lg;
    const int rows = P.T * (P.order - 1) + 64;
    const size_t values = 2 * (size_t)P.t16 * (cols + 4);
    return 4 * ((size_t)rows * cols + 64 * (P.t16 + 4) + std::max(values, (size_t)kDraftThreads * 6));
}

}  // namespace

size_t draft_attend_workspace(const pa_draft* d) {
    DraftDev P;
    int units = 0, tiles = 0;
    return draft_plan(d, P, units, tiles) ? draft_ws(P, units, nullptr) : 0;
}

int launch_draft_attend(const pa_draft* d, hipStream_t s) {
    if (d->batch < 1 || d->kv_heads < 1 || d->heads < 1 || d->heads % d->kv_heads != 0 ||
        d->drafts < 1 || d->drafts > PA_MAX_DRAFTS || d->order < 2 || d->order > PA_MAX_ORDER ||
        d->capacity < 1 || d->dim < 1 || !d->counts)
        return PA_EINVAL;
    const int T = d->levels[0].k.dtype;
    if (!draft_dtype(T)) return PA_EINVAL;
    if (!draft_dim(d->dim) || d->capacity > (1 << 30)) return PA_EUNSUPPORTED;  // 32-bit positions, a step ahead
    DraftDev P;
    int units = 0, tiles = 0;
    if (!draft_plan(d, P, units, tiles)) return PA_EUNSUPPORTED;
    if (!d->workspace || (uintptr_t)d->workspace % 16 != 0 ||
        d->workspace_bytes < draft_ws(P, units, d->workspace))
        return PA_EWORKSPACE;
    P.scale = d->scale;
    P.softclamp = d->softclamp > 0.f ? d->softclamp : 0.f;
    P.counts = d->counts;
    P.parents = d->parents;
    P.parents_stride = d->parents_stride;
    const int rep = d->heads / d->kv_heads;
    bool vmul = false;
    DraftJoin J;
    static_cast<DraftCommon&>(J) = P;
    J.rep = rep;
    for (int t = 0; t < d->order; ++t) {
        const pa_draft_level& l = d->levels[t];
        const bool last = t == d->order - 1, middle = t > 0 && !last;
        const int h = last ? d->heads : d->kv_heads;
        auto need = [&](const pa_view& v, bool want, int heads, int dtype) {
            if (!v.ptr) return !want;
            return want && v.heads == heads && v.dtype == dtype;
        };
        if (!need(l.k, true, d->kv_heads, T) || !need(l.v, true, d->kv_heads, T) ||
            !need(l.vmul, middle, d->kv_heads, T) || !need(l.bias, t > 0, d->kv_heads, PA_F32) ||
            !need(l.q, true, h, T) || !need(l.dk, true, d->kv_heads, T) ||
            !need(l.dv, !last, d->kv_heads, T) || !need(l.out, true, h, T) ||
            !need(l.lse, !last, d->kv_heads, PA_F32))
            return PA_EINVAL;
        const pa_view* vecs[7] = {&l.k, &l.v, &l.vmul, &l.q, &l.dk, &l.dv, &l.out};
        for (const pa_view* v : vecs)
            if (v->ptr && !rows16(*v)) return PA_EUNSUPPORTED;
        // a step's offsets are 32-bit: positions at most 2^22 elements apart
        for (const pa_view* v : {&l.k, &l.v, &l.vmul})
            if (v->ptr && (v->sn < 0 || v->sn > (1 << 22))) return PA_EUNSUPPORTED;
        if ((l.bias.ptr && l.bias.sn != 1) || (l.lse.ptr && l.lse.sn != 1)) return PA_EUNSUPPORTED;
        DraftLevelDev& L = P.L[t];
        L.k = draft_row(l.k);
        L.v = draft_row(l.v);
        L.m = draft_row(l.vmul);
        L.bias = draft_row(l.bias);
        L.q = draft_row(l.q);
        L.dk = draft_row(l.dk);
        J.L[t].dv = draft_row(l.dv);
        J.L[t].out = draft_row(l.out);
        J.L[t].lse = static_cast<float*>(l.lse.ptr);
        J.L[t].lse_sb = l.lse.sb;
        J.L[t].lse_sh = l.lse.sh;
        L.rep = last ? rep : 1;
        L.rows = d->drafts * L.rep;
        L.row0 = t * d->drafts;
        vmul = vmul || middle;
    }
    {
        ProfScope ps("draft_partial", s);
        if (tiles >= kDraftWideWaves * draft_wide_tiles(128)) {
            if (T == PA_F16) launch_draft_wide<f16>(P, units, vmul, s);
            else launch_draft_wide<bf16>(P, units, vmul, s);
        } else if (T == PA_F32) launch_draft_partial<float>(P, units, tiles, vmul, s);
        else if (T == PA_F16) launch_draft_partial<f16>(P, units, tiles, vmul, s);
        else launch_draft_partial<bf16>(P, units, tiles, vmul, s);
    }
    // columns per workgroup: few where the grid is small; LDS of two workgroups a CU at least
    const int blocks = (d->drafts * rep + 63) / 64;
    J.lgcols = combine_lds(P, 4) <= 52 * 1024 ? 4 : 3;
    auto groups = [&]() { return (P.dim + (1 << J.lgcols) - 1) >> J.lgcols; };
    while ((1 << J.lgcols) < P.dim && combine_lds(P, J.lgcols + 1) <= 52 * 1024 &&
           (int64_t)P.batch * P.kv_heads * blocks * groups() > 1024)
        ++J.lgcols;
    const size_t lds = combine_lds(P, J.lgcols);
    const dim3 grid(P.batch * P.kv_heads, groups(), blocks);
    ProfScope ps("draft_combine", s);
    if (T == PA_F32) launch_combine<float>(J, grid, lds, s);
    else if (T == PA_F16) launch_combine<f16>(J, grid, lds, s);
    else launch_combine<bf16>(J, grid, lds, s);
    return PA_OK;
}

int launch_draft_append(const pa_draft_rows* r, hipStream_t s) {
    if (r->batch < 1 || r->drafts < 1 || r->drafts > PA_MAX_DRAFTS || r->dim < 1 || r->count < 1 ||
        r->count > 2 * PA_MAX_ORDER)
        return PA_EINVAL;
    const int T = r->items[0].src.dtype;
    if (!draft_dtype(T)) return PA_EINVAL;
    if (!draft_dim(r->dim)) return PA_EUNSUPPORTED;
    const bool rotary = r->angles || r->inv_freq;
    if (rotary && (r->rot_dim < 0 || r->rot_dim > r->dim || r->rot_dim % 2 != 0)) return PA_EINVAL;
    if (r->angles && !draft_dtype(r->angles_dtype)) return PA_EINVAL;
    if (!r->angles && r->inv_freq && (!(r->interp > 0.f) || !r->counts)) return PA_EINVAL;
    DraftRowsDev P;
    const int E = 16 / draft_size(T);
    P.batch = r->batch;
    P.T = r->drafts;
    P.dim = r->dim;
    P.count = r->count;
    P.rot_dim = rotary ? r->rot_dim : 0;
    P.adt = r->angles_dtype;
    P.eps = r->eps;
    P.interp = r->interp;
    P.counts = r->counts;
    P.parents = r->parents;
    P.parents_stride = r->parents_stride;
    P.angles_sb = r->angles_sb;
    P.angles_sn = r->angles_sn;
    P.angles = r->angles;
    P.inv_freq = r->inv_freq;
    P.lpr = 1;
    while (P.lpr * E < r->dim) P.lpr <<= 1;
    for (int k = 0; k < r->count; ++k) {
        const pa_draft_item& it = r->items[k];
        if (!it.src.ptr || !it.out.ptr || it.src.heads < 1 || it.src.dtype != T || it.out.dtype != T ||
            it.out.heads != it.src.heads || (it.norm_weight && !draft_dtype(it.weight_dtype)))
            return PA_EINVAL;
        if (!rows16(it.src) || !rows16(it.out)) return PA_EUNSUPPORTED;
        DraftItemDev& I = P.it[k];
        I.src = draft_row(it.src);
        I.out = draft_row(it.out);
        I.w = it.norm_weight;
        I.wdt = it.weight_dtype;
        I.rotate = it.rotate;
        I.heads = it.src.heads;
    }
    const int64_t nodes = (int64_t)r->batch * r->drafts;
    if (nodes > kDraftGroups) return PA_EUNSUPPORTED;
    const dim3 grid((unsigned)nodes, r->count);
    ProfScope ps("draft_append", s);
    if (T == PA_F32) hipLaunchKernelGGL((k_draft_append<float>), grid, dim3(kDraftThreads), 0, s, P);
    else if (T == PA_F16) hipLaunchKernelGGL((k_draft_append<f16>), grid, dim3(kDraftThreads), 0, s, P);
    else hipLaunchKernelGGL((k_draft_append<bf16>), grid, dim3(kDraftThreads), 0, s, P);
    return PA_OK;
}

int launch_draft_commit(const pa_commit* c, hipStream_t s) {
    if (c->batch < 1 || c->kv_heads < 1 || c->slots < 1 || c->slots > PA_MAX_DRAFTS || c->capacity < 1 ||
        c->count < 0 || c->count > PA_MAX_MOVES || c->path_len < 0 || c->path_len > PA_MAX_DRAFTS ||
        !c->path || !c->kept || !c->counts || (c->advance && !c->tickets))
        return PA_EINVAL;
    if (c->kv_heads > (1 << 14)) return PA_EUNSUPPORTED;  // 32-bit indexes of a row's vectors
    if (c->batch > kDraftGroups) return PA_EUNSUPPORTED;
    DraftCommitDev P;
    P.batch = c->batch;
    P.kv_heads = c->kv_heads;
    P.slots = c->slots;
    P.capacity = c->capacity;
    P.path_len = c->path_len;
    P.path = c->path;
    P.path_stride = c->path_stride;
    P.kept = c->kept;
    P.counts = c->counts;
    P.overflow = c->overflow;
    for (int k = 0; k < c->count; ++k) {
        const pa_draft_move& m = c->moves[k];
        const int a = m.row_bytes % 16 == 0 ? 16 : 4;
        if (!m.src || !m.dst || m.row_bytes < 4 || m.row_bytes > 4096 || m.row_bytes % 4 != 0 || (uintptr_t)m.src % a != 0 ||
            (uintptr_t)m.dst % a != 0)
            return PA_EINVAL;
        P.mv[k] = m;
    }
    P.count = c->count;
    P.advance = c->advance;
    P.tickets = c->tickets;
    if (c->count > 0 || c->advance) {
        ProfScope ps("draft_commit", s);
        hipLaunchKernelGGL(k_draft_commit, dim3(c->batch, std::max(c->count, 1)), dim3(kDraftThreads), 0, s, P);
    }
    return PA_OK;
}

}  // namespace pa
