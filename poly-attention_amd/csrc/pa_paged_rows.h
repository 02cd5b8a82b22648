// pa_paged_rows.h -- k_paged_rows: a unit of positions for up to 32 query rows of a chunk.
//
// One workgroup per (unit, key head), four waves, each on its own 32 (fp32: 16) positions at a time; nothing
// is shared until the end, so there is no barrier in the loop.  The products and the lane layout are those
// of k_draft_partial: S^T = K Q^T with 16x16 tiles, whose results are the operand of O^T += V^T P^T where
// they lie, the values transposed in registers, weights as two 16-bit numbers.  16 positions lie in one page:
// their page is a scalar, read from a register of 64 of them that is loaded ahead.  Long rows are bound by memory
// (32 of up to 8192 positions, 32/8 heads of 128: 112 to 119 us a level, 5.6 TB/s), short ones by the chain of
// trips: the unit found 1.4 us, pages and queries 1.8, 256 positions of 128 features 5.8, the record 1.9, its ticket 1.1.
#pragma once

#include "pa_paged_join.h"

namespace pa {

// one of a word's numbers, and the word without those that are not finite
template <typename T>
__device__ __forceinline__ float paged_number(uint32_t w, int half) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w);
    else return (float)__builtin_bit_cast(T, (uint16_t)(half ? w >> 16 : w));
}
template <typename T>
__device__ __forceinline__ uint32_t paged_finite(uint32_t w) {
    if constexpr (sizeof(T) == 4) {
        return paged_number<T>(w, 0) * 0.f == 0.f ? w : 0u;
    } else {
        return (paged_number<T>(w, 0) * 0.f == 0.f ? w & 0xffffu : 0u) | (paged_number<T>(w, 1) * 0.f == 0.f ? w & 0xffff0000u : 0u);
    }
}
// keeps a rarely taken branch one
__device__ __forceinline__ void keep_branch_rows() { asm volatile("" ::: "memory"); }

// workgroups: the units', with JOIN `joins` for B's tiles of many rows (whose launch came before), and those that clear outputs
template <typename T, int D, int RT, bool JOIN>
__global__ __launch_bounds__(kPageThreads, paged_waves(D, RT)) void k_paged_rows(const PagedDev P, const PagedDev B, int joins) {
    typedef DraftGeo<T, D> G;
    constexpr int KT = G::KT, KS = G::KS, VE = G::VE, KE = G::KE, CPR = G::CPR, LOADS = KT * KS;
    constexpr int PITCH = D + 4;
    // a query row's fragments stay in registers where those are few
    constexpr bool QLDS = RT * KS * 4 > (G::F32 ? 32 : 16);
    // the waves' outputs meet in NB buffers of 16 rows
    constexpr int OWORDS = 16 * PITCH, QWORDS = QLDS ? RT * KS * 256 : 0, NB = D <= 128 ? 4 : 2;
    // keys pass through LDS (KLDS) where four waves' steps fit
    constexpr bool KLDS = D <= 128;
    constexpr int KWORDS = KLDS ? 4 * G::STEP * CPR * 4 : 0, INWORDS = QWORDS + KWORDS;
    __shared__ __align__(16) float s_o[NB * OWORDS > INWORDS ? NB * OWORDS : INWORDS];  // queries and keys, then these
    u32x4_d* const s_q = reinterpret_cast<u32x4_d*>(s_o);
    __shared__ float s_m[4][16 * RT], s_l[4][16 * RT];
    __shared__ int s_last;

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int main = P.units * P.kv_heads;
    if ((int)blockIdx.x >= main) {
        const int group = blockIdx.x - main;
        if constexpr (JOIN)
            if (group < joins) {
                SlowRow& slow = *reinterpret_cast<SlowRow*>(s_o);
                if (B.recs > 0) paged_join_tiles<T>(B, group, joins, reinterpret_cast<float(*)[6]>(&slow + 1), slow);
                paged_again<T>(B, group, joins, slow);
                return;
            }
        paged_clear<T>(P, group - joins, gridDim.x - main - joins);
        return;
    }
    const int hk = __builtin_amdgcn_readfirstlane(blockIdx.x % P.kv_heads);
    PagedUnit U;
    if (!paged_find<kUnits>(P, blockIdx.x / P.kv_heads, lane, U)) return;
    const int r0 = U.tile * P.tile, nrows = min(P.tile, U.rows - r0), nrt = (nrows + 15) / 16;
    const int begin = U.split * U.size * kPagedChunk;  // below the row's positions, as the unit is one of its
    const int cnt = min(U.size * kPagedChunk, paged_keys(P, U) - begin);
    if (cnt <= 0) return;  // past the tile's last token: the join knows

    auto query = [&](int rt, int s) __attribute__((always_inline)) -> u32x4_d {
        const T* row = paged_query<T>(P, U, hk, min(r0 + 16 * rt + c, U.rows - 1));
        const int d = (KE * 4) * s + KE * g;
        return row && d < P.dim ? load16u(row + d) : u32x4_d{0u, 0u, 0u, 0u};
    };
    u32x4_d qf[QLDS ? 1 : RT][KS], qt[QLDS ? RT * KS / 4 : 1];
    if constexpr (QLDS) {  // a quarter of the fragments per wave
        static_assert(RT * KS % 4 == 0, "four waves");
#pragma unroll
        for (int k = 0; k < RT * KS / 4; ++k) {
            const int f = wave * (RT * KS / 4) + k;
            qt[k] = query(f / KS, f % KS);
        }
    } else {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int s = 0; s < KS; ++s) qf[rt][s] = query(rt, s);
    }
    const int rowb = P.dim * (int)sizeof(T);
    const int inside = (1 << P.p.lg) - 1;
    // the pages of 64 tiles of 16 positions, lane i's the i-th
    const int32_t* const pages = P.p.table + (int64_t)U.b * P.p.max_pages;
    auto load_pages = [&](int o) __attribute__((always_inline)) -> int {
        const int at = min(o + 16 * lane, cnt - 1);
        return pages[(begin + at) >> P.p.lg];
    };
    // Buffers over what is valid of a tile of 16 positions: loads past its end (and at kDraftOut) give 0
    // without touching memory.
    int ids = load_pages(0), ids_next = cnt > 1024 ? load_pages(1024) : 0, block = 0;
    int64_t base[KT];  // of the step's tiles, in positions
    int left[KT];      // positions that are valid; none for a page outside the pool
    auto places = [&](int o) __attribute__((always_inline)) {
        if (o >> 10 != block) {
            block = o >> 10;
            ids = ids_next;
            if (o + 1024 < cnt) ids_next = load_pages((block + 1) << 10);
        }
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            const int id = __builtin_amdgcn_readlane(ids, ((o + 16 * t) >> 4) & 63);
            const bool ok = (unsigned)id < (unsigned)P.p.pages;
            base[t] = paged_base(P, ok ? id : 0, hk) + ((begin + o + 16 * t) & inside);
            left[t] = ok ? min(16, cnt - o - 16 * t) : 0;
        }
    };
    const int ko = KLDS ? (lane % CPR * KE < P.dim ? lane % CPR * 16 : kDraftOut) : 0;
    int kd[KLDS ? 1 : KS];
    if constexpr (!KLDS) {
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int d = (KE * 4) * s + KE * g;
            kd[s] = d < P.dim ? c * rowb + d * (int)sizeof(T) : kDraftOut;
        }
    }
    u32x4_d* const s_k = s_q + QWORDS / 4 + wave * (G::STEP * CPR);
    constexpr int CMASK = CPR < 16 ? CPR - 1 : 15;
    auto chunk = [](int position, int ch) __attribute__((always_inline)) -> int {
        return position * CPR + (ch ^ (position & CMASK));
    };
    const int vo = VE * c < P.dim ? 4 * g * rowb + VE * c * (int)sizeof(T) : kDraftOut;

    u32x4_d kr[LOADS];
    uint32_t v[G::NP][G::VW];
    f32x4_t bz[KT];
    auto load_k = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            constexpr int PER = 64 / CPR;  // positions of a load
            const int t = KLDS ? i * PER / 16 : i / KS;
            const auto rk = draft_buffer(P.keys + base[t] * rowb, left[t] * rowb);
            int off;
            if constexpr (KLDS) off = ko == kDraftOut ? kDraftOut : ko + (i * PER % 16 + lane / CPR) * rowb;
            else off = kd[i % KS];
            kr[i] = __builtin_amdgcn_raw_buffer_load_b128(rk, off, 0, kDraftStream);
        }
    };
    auto load_bias = [&]() __attribute__((always_inline)) {
        if (!P.bias) return;
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            const auto rb = draft_buffer(reinterpret_cast<const char*>(P.bias + base[t]), left[t] > 0 ? 64 : 0);
            bz[t] = __builtin_bit_cast(f32x4_t, __builtin_amdgcn_raw_buffer_load_b128(rb, 16 * g, 0, 0));
        }
    };
    auto load_v = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            const auto rv = draft_buffer(P.values + base[t] * rowb, left[t] * rowb);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                buffer_words<G::VW>(rv, vo == kDraftOut ? kDraftOut : vo + i * rowb, v[4 * t + i]);
        }
    };

    constexpr int STEP = 64 * KT;  // the workgroup's positions per round of steps
    const int first = wave * 16 * KT;
    places(first);
    load_k();
    load_bias();
    load_v();
    if constexpr (QLDS) {
#pragma unroll
        for (int k = 0; k < RT * KS / 4; ++k) s_q[(wave * (RT * KS / 4) + k) * 64 + lane] = qt[k];
        __syncthreads();
    }
    const float sl2 = P.scale * kLog2e, cl2 = P.softclamp * kLog2e;
    const float unclamped = P.softclamp > 0.f ? P.scale / P.softclamp : sl2;
    // the last position that a row sees, and the first tile's least
    int see[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) see[rt] = U.row.p0 + min(r0 + 16 * rt + c, U.rows - 1) / P.rep - begin;
    const int all_see = U.row.p0 + __builtin_amdgcn_readfirstlane(r0 / P.rep) - begin;

    f32x4_t o[RT][VE];
    float m[RT], l[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        m[rt] = -INFINITY;
        l[rt] = 0.f;
#pragma unroll
        for (int j = 0; j < VE; ++j) o[rt][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }

    for (int j0 = first; j0 < cnt; j0 += STEP) {
        f32x4_t bias[KT];
#pragma unroll
        for (int t = 0; t < KT; ++t) bias[t] = bz[t];
        const bool more = j0 + STEP < cnt;
        if constexpr (KLDS) {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) s_k[chunk(i * (64 / CPR) + lane / CPR, lane % CPR)] = kr[i];
            // other lanes of the wave read them: LDS keeps a wave's order, the compiler has to as well
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            if (more) {
                places(j0 + STEP);
                load_k();
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        f32x4_t x[RT][KT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int t = 0; t < KT; ++t) x[rt][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            u32x4_d k[KT];
#pragma unroll
            for (int t = 0; t < KT; ++t) k[t] = KLDS ? s_k[chunk(16 * t + c, 4 * s + g)] : kr[t * KS + s];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                if (rt >= nrt) break;
                const u32x4_d q = QLDS ? s_q[(rt * KS + s) * 64 + lane] : qf[QLDS ? 0 : rt][s];
#pragma unroll
                for (int t = 0; t < KT; ++t) {
                    if constexpr (G::F32) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) x[rt][t] = mma_f32(k[t][j], q[j], x[rt][t]);
                    } else {
                        x[rt][t] = Mma16<T>::run(k[t], q, x[rt][t]);
                    }
                }
            }
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int t = 0; t < KT; ++t) x[rt][t] *= unclamped;
        if (P.softclamp > 0.f) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int t = 0; t < KT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        // tanh(x) = 1 - 2 / (e^2x + 1) to 2^-23 or so absolutely, which 16-bit operands do not see
                        if constexpr (G::F32) x[rt][t][i] = cl2 * tanhf(x[rt][t][i]);
                        else x[rt][t][i] = fmaf(-2.f * cl2, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(2.f * kLog2e * x[rt][t][i]) + 1.f), cl2);
                    }
        }
        if (P.bias) {
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) x[rt][t][i] = fmaf(bias[t][i], kLog2e, x[rt][t][i]);
        }
        bool odd = false;  // a value that is not finite lies among positions that some row does not see
        if (j0 + 16 * KT - 1 > all_see) {  // positions that some row does not see, those past the unit among them
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
                        if (j0 + 16 * t + 4 * g + i > see[rt]) x[rt][t][i] = -INFINITY;
            float none = 0.f;
#pragma unroll
            for (int n = 0; n < G::NP; ++n)
#pragma unroll
                for (int w = 0; w < G::VW; ++w) none = paged_odd<T>(v[n][w], none);
            odd = __any(none != 0.f);
        }
        if (j0 + 16 * KT > cnt) {  // the unit's last positions
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
                        if (j0 + 16 * t + 4 * g + i >= cnt) x[rt][t][i] = -INFINITY;
        }
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (!KLDS) {
            if (more) {
                places(j0 + STEP);
                load_k();
            }
        }
        if (more) load_bias();
        __builtin_amdgcn_sched_barrier(0);
        // probabilities (16-bit types: their leading bits, and the rest); 0 for a tile without rows
        uint32_t pf[RT][4] = {}, pl[RT][4] = {};
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            if (rt >= nrt) break;
            float top = x[rt][0][0];
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) top = fmaxf(top, x[rt][t][i]);
            if (__any(top > m[rt] + draft_tau<T>())) {
                top = fmaxf(top, __shfl_xor(top, 16));
                top = fmaxf(top, __shfl_xor(top, 32));
                const float mn = fmaxf(m[rt], top - draft_lift<T>());
                const float al = mn == m[rt] ? 1.f : __builtin_amdgcn_exp2f(m[rt] - mn);
                m[rt] = mn;
                l[rt] *= al;
#pragma unroll
                for (int j = 0; j < VE; ++j) o[rt][j] *= al;
            }
            const float ms = m[rt] == -INFINITY ? 0.f : m[rt];
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[rt][t][i] = __builtin_amdgcn_exp2f(x[rt][t][i] - ms);
                    l[rt] += x[rt][t][i];
                }
            if constexpr (G::F32) {
#pragma unroll
                for (int i = 0; i < 4; ++i) pf[rt][i] = __float_as_uint(x[rt][0][i]);
            } else {
#pragma unroll
                for (int t = 0; t < KT; ++t) {
                    draft_split2<T>(x[rt][t][0], x[rt][t][1], pf[rt][2 * t], pl[rt][2 * t]);
                    draft_split2<T>(x[rt][t][2], x[rt][t][3], pf[rt][2 * t + 1], pl[rt][2 * t + 1]);
                }
            }
        }
        if (odd) {
            // a weight of 0 times such a value would be no number: they leave the products, and are added to the
            // rows that see them one position after another
            keep_branch_rows();
#pragma unroll
            for (int n = 0; n < G::NP; ++n) {
                float none = 0.f;
#pragma unroll
                for (int w = 0; w < G::VW; ++w) none = paged_odd<T>(v[n][w], none);
                const uint64_t who = __ballot(none != 0.f);
                if (!who) continue;
                for (int g2 = 0; g2 < 4; ++g2) {  // position 16 (n / 4) + 4 g2 + n % 4
                    if (!((who >> (16 * g2)) & 0xffff)) continue;
                    float p[RT];
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) p[rt] = __shfl(x[rt][n / 4][n % 4], 16 * g2 + c);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int j = 0; j < VE; ++j) {
                            const uint32_t word = __shfl(v[n][G::F32 ? j : j / 2], 16 * g2 + 4 * g + i);
                            const float z = paged_number<T>(word, G::F32 ? 0 : j & 1);
#pragma unroll
                            for (int rt = 0; rt < RT; ++rt)
                                if (z * 0.f != 0.f && p[rt] > 0.f) o[rt][j][i] += p[rt] * z;
                        }
                }
#pragma unroll
                for (int w = 0; w < G::VW; ++w) v[n][w] = paged_finite<T>(v[n][w]);
            }
        }
        // O^T += V^T P^T, feature j of every lane's VE per tile
#pragma unroll
        for (int j = 0; j < VE; ++j) {
            if constexpr (G::F32) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
                        if (rt < nrt) o[rt][j] = mma_f32(v[i][j], pf[rt][i], o[rt][j]);
            } else {
                const uint32_t sel = j & 1 ? 0x07060302u : 0x05040100u;
                u32x4_d a;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    a[e] = __builtin_amdgcn_perm(v[2 * e + 1][j / 2], v[2 * e][j / 2], sel);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    if (rt >= nrt) break;
                    const u32x4_d p = {pf[rt][0], pf[rt][1], pf[rt][2], pf[rt][3]};
                    const u32x4_d p2 = {pl[rt][0], pl[rt][1], pl[rt][2], pl[rt][3]};
                    o[rt][j] = Mma16<T>::run(a, p, o[rt][j]);
                    o[rt][j] = Mma16<T>::run(a, p2, o[rt][j]);
                }
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        if (more) load_v();
        __builtin_amdgcn_sched_barrier(0);
    }

    // join the four waves: maxima and sums first, then the outputs
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        l[rt] += __shfl_xor(l[rt], 16);
        l[rt] += __shfl_xor(l[rt], 32);
        if (g == 0) {
            s_m[wave][16 * rt + c] = m[rt];
            s_l[wave][16 * rt + c] = l[rt];
        }
    }
    __syncthreads();
    float f[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        float top = s_m[0][16 * rt + c];
#pragma unroll
        for (int w = 1; w < 4; ++w) top = fmaxf(top, s_m[w][16 * rt + c]);
        f[rt] = m[rt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[rt] - top);
    }
    const bool done = U.splits == 1;
    const PagedRecords<true> R(P, U, hk);
    auto row_sum = [&](int r, float& top) __attribute__((always_inline)) -> float {
        top = s_m[0][r];
        for (int w = 1; w < 4; ++w) top = fmaxf(top, s_m[w][r]);
        float sum = 0.f;
        // a wave without a maximum has a sum of 0, or none where its scores are no numbers
        for (int w = 0; w < 4; ++w)
            sum += s_m[w][r] == -INFINITY ? s_l[w][r] : s_l[w][r] * __builtin_amdgcn_exp2f(s_m[w][r] - top);
        return sum;
    };
    if (!done && !paged_recorded(P, U)) return;
    if (tid < nrows) {
        float top;
        const float sum = row_sum(tid, top);
        if (!done) {
            R.put_sum(U.split * R.step + tid, top, sum);
        } else if (!P.last) {
            const PagedTo to = paged_to<T>(P, U, hk, r0 + tid);
            if (to.lse) *to.lse = (top + log2f(sum)) * kLn2;
        }
    }
    // 16 rows at a time, the waves side by side in NB buffers
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        if (rt >= nrt) break;
#pragma unroll
        for (int w = 0; w < 4; w += NB) {
            if (NB == 4 || wave / NB == w / NB) {
                float* const buf = s_o + (wave % NB) * OWORDS + c * PITCH + 4 * VE * g;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < VE; j += 4) {
                        float4* at = reinterpret_cast<float4*>(buf + VE * i + j);
                        float4 x = w ? *at : make_float4(0.f, 0.f, 0.f, 0.f);
                        x.x += f[rt] * o[rt][j][i];
                        x.y += f[rt] * o[rt][j + 1][i];
                        x.z += f[rt] * o[rt][j + 2][i];
                        x.w += f[rt] * o[rt][j + 3][i];
                        *at = x;
                    }
            }
            __syncthreads();
        }
        const int r = tid >> 4;
        if (16 * rt + r < nrows) {
            float inv = 1.f;
            PagedTo to = {nullptr, nullptr, nullptr};
            if (done) {
                float top;
                inv = 1.f / row_sum(16 * rt + r, top);
                to = paged_to<T>(P, U, hk, r0 + 16 * rt + r);
            }
#pragma unroll
            for (int d = 4 * (tid & 15); d < D; d += 64) {
                if (d >= P.dim) break;
                float4 y = *reinterpret_cast<const float4*>(&s_o[r * PITCH + d]);
#pragma unroll
                for (int k = 1; k < NB; ++k) {
                    const float4 z = *reinterpret_cast<const float4*>(&s_o[k * OWORDS + r * PITCH + d]);
                    y.x += z.x;
                    y.y += z.y;
                    y.z += z.z;
                    y.w += z.w;
                }
                if (!done) {
                    R.put(U.split * R.step + 16 * rt + r, d, y);
                } else if (to.out) paged_store<T>(to, d, make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv));
            }
        }
        if (rt + 1 < RT) __syncthreads();
    }
    if (!done) paged_end<T, RT * D >= 256 ? 4 : RT * D / 64>(P, U, hk, r0, nrows, reinterpret_cast<float(*)[6]>(s_o), s_last);
}

template <typename T, int D>
void launch_paged_rows_d(const PagedDev& P, const PagedDev& B, int64_t units, int joins, int clear, int tiles, hipStream_t s) {
    const dim3 grid((unsigned)(units * P.kv_heads + joins + clear)), block(kPageThreads);
    if constexpr (sizeof(T) == 2 && D <= 128)
        if (joins) {
            hipLaunchKernelGGL((k_paged_rows<T, D, 2, true>), grid, block, 0, s, P, B, joins);
            return;
        }
    if constexpr (paged_row_tiles<T>(D) >= 2)
        if (tiles == 2) {
            hipLaunchKernelGGL((k_paged_rows<T, D, 2, false>), grid, block, 0, s, P, B, joins);
            return;
        }
    hipLaunchKernelGGL((k_paged_rows<T, D, 1, false>), grid, block, 0, s, P, B, joins);
}
template <typename T>
void launch_paged_rows(const PagedDev& P, const PagedDev& B, int64_t units, int joins, int clear, int tiles, hipStream_t s) {
    if (P.dim <= 64) launch_paged_rows_d<T, 64>(P, B, units, joins, clear, tiles, s);
    else if (P.dim <= 128) launch_paged_rows_d<T, 128>(P, B, units, joins, clear, tiles, s);
    else launch_paged_rows_d<T, 256>(P, B, units, joins, clear, tiles, s);
}

}  // namespace pa
