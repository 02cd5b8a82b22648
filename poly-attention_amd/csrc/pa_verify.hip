// pa_verify.hip -- the walk of drafted tokens against the target's probabilities.
//
// Two launches.  k_verify_stats reads every node's logits once: per chunk of the vocabulary the
// maximum, its first position and the sum of exp(x - max), a chunk held in registers between the
// two.  k_verify_walk runs one workgroup per (row, chunk): each joins the chunks' statistics and
// walks the row's tree for itself (a few values per node; the same result in every workgroup, so
// none waits for another), then takes its chunk of the last node's distribution for the token; the
// workgroup that finishes a row last joins the chunks.
//
// The token is the largest p_i / noise_i: one pass, no cumulative sums, and p's common factor drops
// out.  Only a test of a further child after a rejection needs the residual's sum.  With a draft
// distribution that is a pass over the row.  Without, it is the sum of what no child of the node holds, which the
// statistics keep beside the whole sum, and of the children that are left: sums of positive numbers, where
// 1 - (rejected probabilities) would lose all its digits next to 0.
//
// 32 trees of 16 nodes over 32000 tokens (bf16): 10.8 us for the statistics (3.0 TB/s: 4096 short workgroups),
// 10.4 for the walk (dependent trips to memory).  8 chains of 6 over 128256 (fp32) with the drafts'
// distributions: 6.0 and 13.
#include "pa_draft.h"

namespace pa {

namespace {

constexpr int kVerThreads = 256;
constexpr int kVerChunk = 4096;  // entries of a workgroup: 16 per thread, held in registers
constexpr int kVerSmallNodes = 8, kVerSmallLoads = 2;  // what the single launch takes: 16-byte loads of a row per lane

struct VerifyDev {
    int32_t batch, T, vocab, chunks;
    const void* logits;
    int64_t logits_sb, logits_sn;
    const int64_t* tokens;
    int64_t tokens_stride;
    const int32_t* parents;
    int64_t parents_stride;
    const float* uniforms;
    int64_t uniforms_stride;
    const float* noise;
    int64_t noise_stride;
    const float* temperature;
    const float* probs;
    int64_t probs_sb, probs_sn;
    int32_t* path;
    int32_t* kept;
    int64_t* token;
    float4* stats;       // [B][T][chunks]: maximum, sum, first position of the maximum (as bits), sum without
                         // the tokens of the node's children
    uint64_t* best;      // [B][chunks][2]
    uint32_t* ticket;    // [B][kTicketStride]
};

__device__ __forceinline__ float row_temperature(const VerifyDev& P, int b) {
    if (!P.uniforms) return 0.f;
    const float t = P.temperature ? P.temperature[b] : 1.f;
    return t > 0.f ? t : 0.f;
}

// log2(e) / temperature as a finite number above 0: a difference of logits of 0 stays 0 and one of
// -inf stays -inf where the quotient would be infinite or 0
__device__ __forceinline__ float logit_scale(float temp) {
    return fminf(fmaxf(kLog2e / temp, FLT_MIN), FLT_MAX);
}

// the larger value, the lower position of equals; NaN loses
__device__ __forceinline__ void take_first(float& x, int& i, float y, int j) {
    if (y > x || (y == x && j < i)) {
        x = y;
        i = j;
    }
}

// vector k of thread tid: E entries (16 bytes of T) of its chunk
template <typename T> struct VerVec {
    static constexpr int E = 16 / sizeof(T);
    static constexpr int N = kVerChunk / (kVerThreads * E);
};

// E entries of a row of n at entry i >= 0; what lies past the end is `fill`.  Rows start anywhere (a
// vocabulary need not be a multiple of 8): global loads of 16 bytes may be unaligned.
template <typename T, int E>
__device__ __forceinline__ void load_entries(const T* row, int64_t i, int n, float fill, float (&x)[E]) {
    T raw[E];
    if (i + E <= n) {
        __builtin_memcpy(raw, row + i, sizeof(raw));
#pragma unroll
        for (int k = 0; k < E; ++k) x[k] = to_f(raw[k]);
    } else {
#pragma unroll
        for (int k = 0; k < E; ++k) x[k] = i + k < n ? to_f(row[i + k]) : fill;
    }
}

__device__ __forceinline__ float wave_sum(float x) {
    for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off);
    return x;
}

// lane's node: its parent (-2 past the nodes) and its token (-1 where it is none of the vocabulary)
__device__ __forceinline__ int node_parent(const VerifyDev& P, int b, int lane) {
    return lane >= P.T ? -2 : P.parents ? P.parents[b * P.parents_stride + lane] : lane - 1;
}
__device__ __forceinline__ int node_token(const VerifyDev& P, int b, int lane) {
    const int64_t tok = lane < P.T ? P.tokens[b * P.tokens_stride + lane] : -1;
    return tok >= 0 && tok < P.vocab ? (int)tok : -1;
}

template <typename T>
__global__ __launch_bounds__(kVerThreads) void k_verify_stats(const VerifyDev P) {
    constexpr int E = VerVec<T>::E, N = VerVec<T>::N;
    __shared__ float s_x[4], s_sum[4], s_rest[4];
    __shared__ int s_i[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int chunk = blockIdx.x, t = blockIdx.y, b = blockIdx.z;
    if (chunk == 0 && t == 0 && tid == 0) P.ticket[b * kTicketStride] = 0;  // before the walk's launch begins
    const float temp = row_temperature(P, b);
    // without a draft distribution the walk may take tokens out of p one by one: the node's children, whose loads are
    // on their way before the logits and looked at when the sum is known (0.8 us of 18.4 behind cold caches, 32 trees of 16 over 32000)
    const bool apart = P.uniforms && !P.probs;
    int64_t kid = -1;
    int kid_of = lane - 1;
    if (apart && lane > t && lane < P.T) {
        kid = P.tokens[b * P.tokens_stride + lane];
        if (P.parents) kid_of = P.parents[b * P.parents_stride + lane];
    }
    const T* row = reinterpret_cast<const T*>(P.logits) + b * P.logits_sb + t * P.logits_sn;
    const int i0 = chunk * kVerChunk + tid * E;
    float x[N][E];
    float top = -INFINITY;
    int at = P.vocab;
#pragma unroll
    for (int k = 0; k < N; ++k) load_entries<T, E>(row, i0 + k * kVerThreads * E, P.vocab, -INFINITY, x[k]);
    if (temp > 0.f) {
#pragma unroll
        for (int k = 0; k < N; ++k)
#pragma unroll
            for (int e = 0; e < E; ++e) top = fmaxf(top, x[k][e]);  // NaN loses, and shows in the sum
        for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k)
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (x[k][e] > top) {
                    top = x[k][e];
                    at = i0 + k * kVerThreads * E + e;
                }
        for (int off = 32; off > 0; off >>= 1) take_first(top, at, __shfl_xor(top, off), __shfl_xor(at, off));
    }
    if (lane == 0) {
        s_x[wave] = top;
        s_i[wave] = at;
    }
    __syncthreads();
    top = s_x[0];
    at = s_i[0];
#pragma unroll
    for (int w = 1; w < 4; ++w) take_first(top, at, s_x[w], s_i[w]);
    float sum = 0.f, rest = 0.f;
    if (temp > 0.f) {
        const float c = logit_scale(temp), base = top == -INFINITY ? 0.f : top;
        auto weights = [&]() __attribute__((always_inline)) -> float {
            float y = 0.f;
#pragma unroll
            for (int k = 0; k < N; ++k)
#pragma unroll
                for (int e = 0; e < E; ++e) y += __builtin_amdgcn_exp2f((x[k][e] - base) * c);
            return wave_sum(y);
        };
        sum = rest = weights();
        // a token outside the vocabulary lies in no chunk, or behind the last one's entries
        const uint64_t in = (uint64_t)kid - (uint64_t)chunk * kVerChunk;
        uint64_t kids = __ballot(kid_of == t && in < kVerChunk);
        if (kids) {
            for (; kids; kids &= kids - 1) {
                const int out = __builtin_amdgcn_readlane((int)in, __ffsll((unsigned long long)kids) - 1) - tid * E;
#pragma unroll
                for (int k = 0; k < N; ++k)
#pragma unroll
                    for (int e = 0; e < E; ++e) x[k][e] = out == k * kVerThreads * E + e ? -INFINITY : x[k][e];
            }
            rest = weights();
        }
        if (lane == 0) {
            s_sum[wave] = sum;
            s_rest[wave] = rest;
        }
        __syncthreads();
        sum = s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
        rest = s_rest[0] + s_rest[1] + s_rest[2] + s_rest[3];
    }
    if (tid == 0)
        P.stats[((int64_t)b * P.T + t) * P.chunks + chunk] = make_float4(top, sum, __int_as_float(at), rest);
}

// the residual after `n` rejections of one entry's probability p with draft probability q: inv[k] is
// one over the sum of the k-th residual, 0 where that sum was 0 (p stays as it was)
__device__ __forceinline__ float residual(float p, float q, const float* inv, int n) {
    for (int k = 0; k < n; ++k) p = inv[k] != 0.f ? fmaxf(p - q, 0.f) * inv[k] : p;
    return p;
}

__device__ __forceinline__ uint64_t best_key(float w, float noise, int64_t i) {
    if (!(w > 0.f)) return 0;
    const float key = w / noise;
    if (!(key >= 0.f)) return 0;
    // +1: a key of 0 (underflow) still is a candidate
    return ((uint64_t)(__float_as_uint(key) + 1u) << 32) | (0xffffffffu - (uint32_t)i);
}

__device__ __forceinline__ uint64_t wave_best(uint64_t x) {
    for (int off = 32; off > 0; off >>= 1) {
        const uint64_t y = __shfl_xor((unsigned long long)x, off);
        x = y > x ? y : x;
    }
    return x;
}
__device__ __forceinline__ int64_t best_token(uint64_t key) {
    return key ? (int64_t)(0xffffffffu - (uint32_t)key) : (int64_t)-1;
}

// SMALL: the statistics are formed here, a node per wave at a time, and the walk is the only launch
template <typename T, bool SMALL>
__global__ __launch_bounds__(kVerThreads) void k_verify_walk(const VerifyDev P) {
    constexpr int E = VerVec<T>::E, N = VerVec<T>::N;
    __shared__ float s_top[64], s_inv[64], s_rest[64], s_rinv[64], s_wave[4];
    __shared__ int s_arg[64], s_rej[64];
    __shared__ uint64_t s_best[4][2];
    __shared__ int s_last;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int chunk = blockIdx.x, b = blockIdx.y;
    const float temp = row_temperature(P, b);
    const bool greedy = !(temp > 0.f);
    const float c = greedy ? 0.f : logit_scale(temp);
    const int32_t* parents = P.parents ? P.parents + b * P.parents_stride : nullptr;

    // this chunk's random numbers are in flight over the walk
    const int i0 = chunk * kVerChunk + tid * E;
    float nz[N][E];
    if (!greedy) {
        const float* noise = P.noise + b * P.noise_stride;
#pragma unroll
        for (int k = 0; k < N; ++k) load_entries<float, E>(noise, i0 + k * kVerThreads * E, P.vocab, 1.f, nz[k]);
    }

    // every wave holds the nodes, one per lane, and walks for itself
    const bool node = lane < P.T;
    const int parent = node_parent(P, b, lane), tok = node_token(P, b, lane);
    const float u = node && !greedy ? P.uniforms[b * P.uniforms_stride + lane] : 0.f;
    if constexpr (SMALL) {  // a row in a wave's registers, all rows on their way at once
        constexpr int R = kVerSmallNodes * 64 / kVerThreads;
        float x[R][kVerSmallLoads][E];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int t = min(wave + r * (kVerThreads / 64), P.T - 1);
            const T* from = reinterpret_cast<const T*>(P.logits) + b * P.logits_sb + t * P.logits_sn;
#pragma unroll
            for (int k = 0; k < kVerSmallLoads; ++k) load_entries<T, E>(from, (k * 64 + lane) * E, P.vocab, -INFINITY, x[r][k]);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int t = wave + r * (kVerThreads / 64);
            float top = -INFINITY, sum = 0.f, rest = 0.f;
            int at = P.vocab;
#pragma unroll
            for (int k = 0; k < kVerSmallLoads; ++k)
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (x[r][k][e] > top) {
                        top = x[r][k][e];
                        at = (k * 64 + lane) * E + e;
                    }
            for (int off = 32; off > 0; off >>= 1) take_first(top, at, __shfl_xor(top, off), __shfl_xor(at, off));
            if (!greedy) {
                const float base = top == -INFINITY ? 0.f : top;
                auto weights = [&]() __attribute__((always_inline)) -> float {
                    float y = 0.f;
#pragma unroll
                    for (int k = 0; k < kVerSmallLoads; ++k)
#pragma unroll
                        for (int e = 0; e < E; ++e) y += __builtin_amdgcn_exp2f((x[r][k][e] - base) * c);  // 0 past the end
                    return wave_sum(y);
                };
                sum = rest = weights();
                uint64_t kids = P.probs ? 0 : __ballot(lane > t && parent == t && tok >= 0);
                if (kids) {
                    for (; kids; kids &= kids - 1) {
                        const int out = __builtin_amdgcn_readlane(tok, __ffsll((unsigned long long)kids) - 1) - lane * E;
#pragma unroll
                        for (int k = 0; k < kVerSmallLoads; ++k)
#pragma unroll
                            for (int e = 0; e < E; ++e) x[r][k][e] = out == k * 64 * E + e ? -INFINITY : x[r][k][e];
                    }
                    rest = weights();
                }
            }
            if (t < P.T && lane == 0) {
                s_top[t] = top;
                s_inv[t] = 1.f / sum;
                s_rest[t] = rest;
                s_arg[t] = at;
            }
        }
    } else {  // statistics over the chunks, four threads per node
        const int t = tid >> 2, sub = tid & 3;
        float top = -INFINITY, sum = 0.f, rest = 0.f;
        int at = P.vocab;
        const float4* st = P.stats + ((int64_t)b * P.T + t) * P.chunks;
        if (t < P.T)
#pragma unroll 4
            for (int k = sub; k < P.chunks; k += 4) {
                const float4 x = st[k];
                const float was = top;
                take_first(top, at, x.x, __float_as_int(x.z));
                if (!greedy) {
                    const float f = was == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((was - top) * c),
                                g = x.x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((x.x - top) * c);  // of 0, or NaN
                    sum = sum * f + x.y * g;
                    rest = rest * f + x.w * g;
                }
            }
        for (int off = 1; off < 4; off <<= 1) {
            const float was = top, x = __shfl_xor(top, off), y = __shfl_xor(sum, off), z = __shfl_xor(rest, off);
            take_first(top, at, x, __shfl_xor(at, off));
            if (!greedy) {
                const float f = was == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((was - top) * c),
                            g = x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((x - top) * c);
                sum = sum * f + y * g;
                rest = rest * f + z * g;
            }
        }
        if (t < P.T && sub == 0) {
            s_top[t] = top;
            s_inv[t] = 1.f / sum;
            s_rest[t] = rest;
            s_arg[t] = at;
        }
    }
    const uint64_t live = __ballot(draft_ancestors(parents, P.T, lane) != 0);
    __syncthreads();
    // each node's own probability under its parent, and its weight there (the largest logit's is 1)
    float px = 0.f, qx = 1.f, ex = 0.f;
    if (((live >> lane) & 1) && parent >= 0 && tok >= 0) {
        if (greedy) {
            px = tok == s_arg[parent] ? 1.f : 0.f;
        } else {
            const float x = to_f(reinterpret_cast<const T*>(P.logits)[b * P.logits_sb + parent * P.logits_sn + tok]);
            ex = __builtin_amdgcn_exp2f((x - s_top[parent]) * c);
            px = ex * s_inv[parent];
        }
        if (P.probs) qx = P.probs[b * P.probs_sb + parent * P.probs_sn + tok];
    }

    // the walk: the current node's children in order.  All of it is the same in every wave.
    int cur = 0, kept = live & 1 ? 1 : 0, nrej = 0;  // rejected children of cur
    uint64_t path = kept, rejected = 0;               // kept nodes, rejected children whose token is out of p
    // without probs: children of cur whose token no earlier one has, what those behind this lane's weigh, and the
    // weights that a rejection left
    uint64_t first = 0;
    float behind = 0.f, left = 0.f;
    const T* row = reinterpret_cast<const T*>(P.logits) + b * P.logits_sb;
    const float* qrow = P.probs ? P.probs + b * P.probs_sb : nullptr;
    uint64_t children = kept ? __ballot(((live >> lane) & 1) && parent == 0) : 0;
    while (children) {
        const int t = __ffsll((unsigned long long)children) - 1;
        children &= children - 1;
        float pt = __shfl(px, t);
        const float qt = __shfl(qx, t), ut = __shfl(u, t);
        const int xt = __shfl(tok, t);
        if (nrej > 0) {
            if (P.probs) {
                // the sum of the newest residual, now that a further child needs it
                const float top = s_top[cur], inv = s_inv[cur];
                float part = 0.f;
                float x[2][N][E], q[2][N][E];
                auto fetch = [&](int i, float (&x)[N][E], float (&q)[N][E]) __attribute__((always_inline)) {
#pragma unroll
                    for (int k = 0; k < N; ++k) {
                        const int64_t at = i + (int64_t)k * kVerThreads * E;
                        load_entries<T, E>(row + cur * P.logits_sn, at, P.vocab, -INFINITY, x[k]);
                        load_entries<float, E>(qrow + cur * P.probs_sn, at, P.vocab, 1.f, q[k]);
                    }
                };
                auto add = [&](float (&x)[N][E], float (&q)[N][E]) __attribute__((always_inline)) {
#pragma unroll
                    for (int k = 0; k < N; ++k)
#pragma unroll
                        for (int e = 0; e < E; ++e) {
                            const float p = __builtin_amdgcn_exp2f((x[k][e] - top) * c) * inv;  // 0 past the end
                            part += fmaxf(residual(p, q[k][e], s_rinv, nrej - 1) - q[k][e], 0.f);
                        }
                };
                // two chunks in turn, one on its way
                fetch(tid * E, x[0], q[0]);
                for (int i = tid * E; i - tid * E < P.vocab; i += 2 * kVerChunk) {
                    fetch(i + kVerChunk, x[1], q[1]);
                    add(x[0], q[0]);
                    fetch(i + 2 * kVerChunk, x[0], q[0]);
                    add(x[1], q[1]);
                }
                part = wave_sum(part);
                if (lane == 0) s_wave[wave] = part;
                __syncthreads();
                const float sum = s_wave[0] + s_wave[1] + s_wave[2] + s_wave[3];
                if (tid == 0) s_rinv[nrej - 1] = sum > 0.f ? 1.f / sum : 0.f;
                __syncthreads();
                pt = xt >= 0 ? residual(pt, qt, s_rinv, nrej) : 0.f;
            } else {
                const bool out = __any(((rejected >> lane) & 1) && tok == xt);
                pt = out ? 0.f : __shfl(ex, t) / left;
            }
        }
        if (ut * qt < pt) {
            cur = t;
            ++kept;
            path |= 1ull << t;
            nrej = 0;
            rejected = 0;
            first = 0;
            children = __ballot(((live >> lane) & 1) && parent == t);
        } else if (!greedy) {
            if (P.probs) {
                ++nrej;
            } else if (pt > 0.f) {  // out of p, unless it was all of p
                if (!first) {
                    uint64_t more = __ballot(((live >> lane) & 1) && parent == cur && tok >= 0);
                    behind = 0.f;
                    while (more) {
                        const int j = __ffsll((unsigned long long)more) - 1;
                        first |= 1ull << j;
                        more &= ~__ballot(tok == __builtin_amdgcn_readlane(tok, j));
                        behind += lane < j ? __int_as_float(__builtin_amdgcn_readlane(__float_as_int(ex), j)) : 0.f;
                    }
                }
                // children before t are rejected and out of p, or had no part of it
                const float rest = s_rest[cur] + __int_as_float(__builtin_amdgcn_readlane(__float_as_int(behind), t));
                if (rest > 0x1p-64f) {  // of a weight of 1: what 2^30 tokens hold of it is above fp32's smallest number
                    rejected |= 1ull << t;
                    left = rest;
                    ++nrej;
                }
            }
        }
    }
    if (chunk == 0 && wave == 0) {
        int32_t* to = P.path + (int64_t)b * P.T;
        const uint64_t below = path & ((1ull << lane) - 1);
        if ((path >> lane) & 1) to[__popcll(below)] = lane;
        if (node && lane >= kept) to[lane] = -1;
        if (lane == 0) P.kept[b] = kept;
    }
    if (!kept || greedy) {
        if (chunk == 0 && tid == 0)
            P.token[b] = kept && s_arg[cur] < P.vocab ? (int64_t)s_arg[cur] : (int64_t)-1;
        return;
    }

    // this chunk of the last node's distribution.  With probs the last rejection's residual is taken
    // without its sum (a common factor); `alt` is the candidate before it, for a sum of 0.
    row += cur * P.logits_sn;
    const float top = s_top[cur], inv = s_inv[cur];
    const float* q = P.probs && nrej > 0 ? qrow + cur * P.probs_sn : nullptr;
    const int nout = P.probs ? 0 : nrej;
    if (wave == 0 && ((rejected >> lane) & 1)) s_rej[__popcll(rejected & ((1ull << lane) - 1))] = tok;
    float x[N][E];
#pragma unroll
    for (int k = 0; k < N; ++k) load_entries<T, E>(row, i0 + k * kVerThreads * E, P.vocab, -INFINITY, x[k]);
    __syncthreads();
    uint64_t best = 0, alt = 0;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int i = i0 + k * kVerThreads * E;
        float w[E];
#pragma unroll
        for (int e = 0; e < E; ++e) w[e] = __builtin_amdgcn_exp2f((x[k][e] - top) * c) * inv;  // 0 outside
        if (q) {
            float qj[E];
            load_entries<float, E>(q, i, P.vocab, 1.f, qj);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                w[e] = residual(w[e], qj[e], s_rinv, nrej - 1);
                const uint64_t key = best_key(w[e], nz[k][e], i + e);
                alt = key > alt ? key : alt;
                w[e] = fmaxf(w[e] - qj[e], 0.f);
            }
        }
        for (int r = 0; r < nout; ++r) {
            const int out = s_rej[r] - i;
#pragma unroll
            for (int e = 0; e < E; ++e) w[e] = out == e ? 0.f : w[e];
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const uint64_t key = best_key(w[e], nz[k][e], i + e);
            best = key > best ? key : best;
        }
    }
    best = wave_best(best);
    if (q) alt = wave_best(alt);
    if (lane == 0) {
        s_best[wave][0] = best;
        s_best[wave][1] = alt;
    }
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < 4; ++w) {
            best = s_best[w][0] > best ? s_best[w][0] : best;
            alt = s_best[w][1] > alt ? s_best[w][1] : alt;
        }
        if (P.chunks == 1) {
            P.token[b] = best_token(best ? best : alt);
            return;
        }
        uint64_t* to = P.best + ((int64_t)b * P.chunks + chunk) * 2;
        __hip_atomic_store(to, best, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(to + 1, alt, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        // The stores and the loads below act at the level that all of the GPU shares, so it is enough that the
        // stores have ended before the ticket is drawn; a release would write the L2 back, at several us.
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        const uint32_t n = __hip_atomic_fetch_add(P.ticket + b * kTicketStride, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        s_last = n == (uint32_t)P.chunks - 1;
    }
    if (P.chunks == 1) return;
    __syncthreads();
    if (!s_last || wave != 0) return;
    best = 0;
    alt = 0;
    for (int k = lane; k < P.chunks; k += 64) {
        uint64_t* from = P.best + ((int64_t)b * P.chunks + k) * 2;
        const uint64_t y = __hip_atomic_load(from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const uint64_t z = __hip_atomic_load(from + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        best = y > best ? y : best;
        alt = z > alt ? z : alt;
    }
    best = wave_best(best);
    alt = wave_best(alt);
    if (lane == 0) P.token[b] = best_token(best ? best : alt);
}

int verify_chunks(const pa_verify* v) {
    return (v->vocab + kVerChunk - 1) / kVerChunk;
}

bool verify_sizes(const pa_verify* v) {
    return v->batch >= 1 && v->batch <= 65535 && v->drafts >= 1 && v->drafts <= PA_MAX_DRAFTS &&
           v->vocab >= 1 && v->vocab <= (1 << 30);
}

}  // namespace

size_t draft_verify_workspace(const pa_verify* v) {
    if (!verify_sizes(v)) return 0;
    const size_t chunks = verify_chunks(v), b = v->batch;
    return b * v->drafts * chunks * sizeof(float4) + b * chunks * 16 + b * kTicketStride * 4;
}

int launch_draft_verify(const pa_verify* v, hipStream_t s) {
    if (!verify_sizes(v)) return v->batch > 65535 || v->vocab > (1 << 30) ? PA_EUNSUPPORTED : PA_EINVAL;
    if (v->dtype != PA_F32 && v->dtype != PA_F16 && v->dtype != PA_BF16) return PA_EINVAL;
    if (!v->logits || !v->tokens || !v->path || !v->kept || !v->token || (v->uniforms && !v->noise) ||
        (uintptr_t)v->logits % (v->dtype == PA_F32 ? 4 : 2) != 0)
        return PA_EINVAL;
    if (!v->workspace || (uintptr_t)v->workspace % 16 != 0 || v->workspace_bytes < draft_verify_workspace(v))
        return PA_EWORKSPACE;
    VerifyDev P;
    P.batch = v->batch;
    P.T = v->drafts;
    P.vocab = v->vocab;
    P.chunks = verify_chunks(v);
    P.logits = v->logits;
    P.logits_sb = v->logits_sb;
    P.logits_sn = v->logits_sn;
    P.tokens = v->tokens;
    P.tokens_stride = v->tokens_stride;
    P.parents = v->parents;
    P.parents_stride = v->parents_stride;
    P.uniforms = v->uniforms;
    P.uniforms_stride = v->uniforms_stride;
    P.noise = v->noise;
    P.noise_stride = v->noise_stride;
    P.temperature = v->temperature;
    P.probs = v->uniforms ? v->draft_probs : nullptr;
    P.probs_sb = v->probs_sb;
    P.probs_sn = v->probs_sn;
    P.path = v->path;
    P.kept = v->kept;
    P.token = v->token;
    char* ws = static_cast<char*>(v->workspace);
    P.stats = reinterpret_cast<float4*>(ws);
    ws += (size_t)P.batch * P.T * P.chunks * sizeof(float4);
    P.best = reinterpret_cast<uint64_t*>(ws);
    ws += (size_t)P.batch * P.chunks * 16;
    P.ticket = reinterpret_cast<uint32_t*>(ws);
    // One launch where a row's logits fit the registers of a wave and a wave has two nodes at most (one row of 5
    // nodes over 256 tokens: 13.7 us behind cold caches, 5 else; two launches 17.4).
    const bool small = P.T <= kVerSmallNodes && P.vocab <= 64 * kVerSmallLoads * (v->dtype == PA_F32 ? 4 : 8);
    auto go = [&](auto tag) {
        typedef decltype(tag) T;
        if (small) {
            ProfScope ps("verify_walk", s);
            hipLaunchKernelGGL((k_verify_walk<T, true>), dim3(1, P.batch), dim3(kVerThreads), 0, s, P);
            return;
        }
        {
            ProfScope ps("verify_stats", s);
            hipLaunchKernelGGL((k_verify_stats<T>), dim3(P.chunks, P.T, P.batch), dim3(kVerThreads), 0, s, P);
        }
        ProfScope ps("verify_walk", s);
        hipLaunchKernelGGL((k_verify_walk<T, false>), dim3(P.chunks, P.batch), dim3(kVerThreads), 0, s, P);
    };
    if (v->dtype == PA_F32) go(float{});
    else if (v->dtype == PA_F16) go(f16{});
    else go(bf16{});
    return PA_OK;
}

}  // namespace pa
