// pa_draft_partial.h -- k_draft_partial: the cached positions of a drafted step.
//
// One workgroup per (unit of positions, key head and block of rows, level), four waves, each on its
// own 32 (fp32: 16) positions at a time; nothing is shared until the end, so there is no barrier in
// the loop.
//
// S^T = K Q^T with 16x16 tiles (A: 16 positions, lane l holds position l % 16; B: 16 rows): lane l =
// 16 g + c gets row c and the positions 4 g .. 4 g + 3 of a tile.  A second product over those
// positions, O^T = V^T P^T, wants from lane l row c and the positions of group g: exactly the
// probabilities it holds, if V^T's operand takes the same positions.  So a lane loads, for its
// group's eight positions (4 g + e of both tiles), the dim / 16 features it owns: 16 lanes cover a
// whole row, and the transposition that the operand needs is inside the lane (one v_perm_b32 for
// two values).  fp32 takes v_mfma_f32_16x16x4_f32, whose operands are single values: no
// transposition at all.  In O^T a lane holds one row, so the running maximum's rescale is one
// factor per lane; it moves only past draft_tau (lazy), so exp2(s - m) is at most 2^8
// (fp16 2^15).
//
// Bound by memory while the rows are few: 32 rows of up to 8192 positions of 128 (163155 in all), 8 key heads of 32
// query rows: 247 us, 5.4 TB/s.
#pragma once

#include <type_traits>

#include "pa_draft.h"

namespace pa {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_d __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_d __attribute__((ext_vector_type(2)));

template <typename T> struct Mma16;
template <> struct Mma16<bf16> {
    typedef __bf16 frag __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x4_t run(u32x4_d a, u32x4_d b, f32x4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(frag, a),
                                                       __builtin_bit_cast(frag, b), c, 0, 0, 0);
    }
};
template <> struct Mma16<f16> {
    typedef _Float16 frag __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x4_t run(u32x4_d a, u32x4_d b, f32x4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(frag, a),
                                                      __builtin_bit_cast(frag, b), c, 0, 0, 0);
    }
};
__device__ __forceinline__ f32x4_t mma_f32(uint32_t a, uint32_t b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a), __uint_as_float(b), c, 0, 0, 0);
}

template <typename T>
__device__ __forceinline__ uint32_t draft_pack2(float lo, float hi) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    typedef T t2 __attribute__((ext_vector_type(2)));
    const f2 v = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, t2));
}
// The probabilities of cached positions as two numbers of the type each, the leading bits (cut off, not rounded) and
// what those leave: 16 bits of a bf16 weight and 22 of an fp16 one, against 8 and 11.  One of them alone was the
// largest error of a 16-bit step (bf16 0.0021 to 0.0025 relative to the output against 0.0017, the rounding of the
// output).  The leading bits are those of a number 2^-12 smaller, so that the rest is above 0: an infinite value then
// gives inf, not inf * 0.
template <typename T>
__device__ __forceinline__ void draft_split2(float a, float b, uint32_t& hi, uint32_t& lo) {
    constexpr float kLess = 1.f - 1.f / 4096.f;
    float ha = a * kLess, hb = b * kLess;
    if constexpr (std::is_same_v<T, bf16>) {
        const uint32_t ia = __float_as_uint(ha), ib = __float_as_uint(hb);
        hi = __builtin_amdgcn_perm(ib, ia, 0x07060302u);
        ha = __uint_as_float(ia & 0xffff0000u);
        hb = __uint_as_float(ib & 0xffff0000u);
    } else {
        const auto h = __builtin_amdgcn_cvt_pkrtz(ha, hb);
        hi = __builtin_bit_cast(uint32_t, h);
        ha = (float)h[0];
        hb = (float)h[1];
    }
    lo = draft_pack2<T>(a - ha, b - hb);
}
// A middle level's values v * msg, two at a time, as two bf16 numbers each whatever the type: word e of hi their
// leading bits, of lo what those leave (16 bits together).  bf16 has fp32's range, where a product of two fp16
// numbers passes fp16's at both ends.  An infinite product leaves its infinity to lo, beside the largest number
// in hi: the rest of an infinity would be inf - inf.
template <typename T>
__device__ __forceinline__ void draft_mul2(uint32_t a, uint32_t b, u32x4_d& hi, u32x4_d& lo, int e) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    typedef T t2 __attribute__((ext_vector_type(2)));
    constexpr float kMost = 0x1.fep127f;  // the largest bf16
    const f2 x = __builtin_convertvector(__builtin_bit_cast(t2, a), f2);
    const f2 y = __builtin_convertvector(__builtin_bit_cast(t2, b), f2);
    const uint32_t i0 = __float_as_uint(__builtin_amdgcn_fmed3f(x[0] * y[0], -kMost, kMost)),
                   i1 = __float_as_uint(__builtin_amdgcn_fmed3f(x[1] * y[1], -kMost, kMost));
    hi[e] = __builtin_amdgcn_perm(i1, i0, 0x07060302u);
    lo[e] = draft_pack2<bf16>(fmaf(x[0], y[0], -__uint_as_float(i0 & 0xffff0000u)),
                              fmaf(x[1], y[1], -__uint_as_float(i1 & 0xffff0000u)));
}

// the weights p + p2 times the values a, of a middle level (middle) a + a2
template <typename T, bool VM>
__device__ __forceinline__ f32x4_t draft_weigh(u32x4_d a, u32x4_d a2, u32x4_d p, u32x4_d p2, f32x4_t o, bool middle) {
    if constexpr (VM)
        if (middle) {
            o = Mma16<bf16>::run(a, p, o);
            o = Mma16<bf16>::run(a2, p, o);
            return Mma16<bf16>::run(a, p2, o);
        }
    o = Mma16<T>::run(a, p, o);
    return Mma16<T>::run(a, p2, o);
}
// as draft_split2, the numbers of the type, of a middle level bf16
template <typename T, bool VM>
__device__ __forceinline__ void draft_weights2(float a, float b, uint32_t& hi, uint32_t& lo, bool middle) {
    if (VM && middle) draft_split2<bf16>(a, b, hi, lo);
    else draft_split2<T>(a, b, hi, lo);
}

__device__ __forceinline__ u32x4_d load16u(const void* p) { return *reinterpret_cast<const u32x4_d*>(p); }

// Fragment geometry of a head dim padded to D: S words of a row's contraction per lane, W words of
// values per lane and position.
template <typename T, int D> struct DraftGeo {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int KT = F32 ? 1 : 2;         // 16-position tiles per step
    static constexpr int NP = 4 * KT;              // a lane's positions per step
    static constexpr int KS = F32 ? D / 16 : D / 32;  // 16-byte loads of a key row per lane
    static constexpr int VE = D / 16;              // features per lane of a value row
    static constexpr int VW = F32 ? VE : VE / 2;   // the same in 32-bit words
    static constexpr int KE = F32 ? 4 : 8;         // elements of a 16-byte load
    static constexpr int CPR = D / KE;             // 16-byte chunks of a row
    static constexpr int STEP = 16 * KT;           // a wave's positions per step
};

// A buffer over the rest of a unit: loads past its end (and at kDraftOut) give 0 without touching memory,
// so neither the last step nor a head dim below D needs a test.  The whole offset goes into the address
// that is checked against the end (a scalar offset need not be).
// They are marked as streaming: a cached position is read once a step, and by the other blocks of rows at
// about the same time.  Behind a kernel that leaves the caches full of its own data that is worth 20 to
// 40% (7 rows of up to 21333 positions 147 -> 91 us, 8 x 2048 of order 3 66 -> 41).
constexpr int kDraftStream = 2;  // nt
constexpr int kDraftOut = 0x7ffffff0;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t draft_buffer(const char* p, int64_t bytes) {
    const int n = bytes <= 0 ? 0 : bytes > 0x40000000 ? 0x40000000 : (int)bytes;
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(p), 0, n, 0x00027000);
}
template <int VW>
__device__ __forceinline__ void buffer_words(__amdgpu_buffer_rsrc_t r, int off, uint32_t (&w)[VW]) {
    if constexpr (VW == 2) {
        const u32x2_d x = __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, kDraftStream);
        w[0] = x[0];
        w[1] = x[1];
    } else {
#pragma unroll
        for (int i = 0; i < VW; i += 4) {
            const u32x4_d x = __builtin_amdgcn_raw_buffer_load_b128(r, off + 4 * i, 0, kDraftStream);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[i + j] = x[j];
        }
    }
}

template <typename T, int D, int RT, bool VM>
__global__ __launch_bounds__(kDraftThreads, draft_waves(D, RT, VM)) void k_draft_partial(const DraftDev P) {
    typedef DraftGeo<T, D> G;
    constexpr int KT = G::KT, KS = G::KS, VE = G::VE, KE = G::KE;
    constexpr int PITCH = D + 4;
    // a query row's fragments stay in registers where those are few
    constexpr bool QLDS = RT * KS * 4 > (G::F32 ? 32 : 16);
    // the waves' outputs meet in NB buffers of 16 rows
    constexpr int OWORDS = 16 * PITCH, QWORDS = QLDS ? RT * KS * 256 : 0, NB = D <= 128 ? 4 : 2;
    // keys pass through LDS (KLDS) where four waves' steps fit
    constexpr bool KLDS = D <= 128;
    constexpr int KWORDS = KLDS ? 4 * G::STEP * G::CPR * 4 : 0, INWORDS = QWORDS + KWORDS;
    __shared__ __align__(16) float s_o[NB * OWORDS > INWORDS ? NB * OWORDS : INWORDS];  // queries and keys, then these
    u32x4_d* const s_q = reinterpret_cast<u32x4_d*>(s_o);
    __shared__ float s_m[4][16 * RT], s_l[4][16 * RT];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int hk = blockIdx.y / P.row_blocks, r0 = (blockIdx.y % P.row_blocks) * 16 * RT;
    const DraftLevelDev L = P.L[blockIdx.z];  // loaded at once, beside the counts
    if (r0 >= L.rows) return;
    const int nrows = min(16 * RT, L.rows - r0);
    const int nrt = (nrows + 15) / 16;
    const bool tree = (int)blockIdx.x < P.batch;  // the first workgroups: a row's drafted tokens
    const int unit = blockIdx.x - P.batch;
    DraftUnits U;
    if (!tree && !draft_units(P, -1, unit, lane, U)) return;
    const int b = tree ? (int)blockIdx.x : U.b;
    const int64_t begin = tree ? 0 : (int64_t)U.place * U.size * kDraftChunk;
    // >= 1: a unit begins inside its row
    const int cnt = tree ? 0 : __builtin_amdgcn_readfirstlane((int)min((int64_t)U.size * kDraftChunk, draft_count(P, b) - begin));

    // the queries: row r of the block is node r % T of the group's head r / T
    auto query = [&](int rt, int s) __attribute__((always_inline)) -> u32x4_d {
        const int r = min(r0 + 16 * rt + c, L.rows - 1);
        const T* row = L.q.at<T>(b, hk * L.rep + r / P.T) + (int64_t)(r % P.T) * L.q.sn;
        const int d = (KE * 4) * s + KE * g;
        return d < P.dim ? load16u(row + d) : u32x4_d{0u, 0u, 0u, 0u};
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
    const bool has_m = VM && L.m.p;
    const char* kb = reinterpret_cast<const char*>(L.k.at<T>(b, hk) + begin * L.k.sn);
    const char* vb = reinterpret_cast<const char*>(L.v.at<T>(b, hk) + begin * L.v.sn);
    const char* mb = has_m ? reinterpret_cast<const char*>(L.m.at<T>(b, hk) + begin * L.m.sn) : nullptr;
    const char* bb = L.bias.p ? reinterpret_cast<const char*>(L.bias.at<float>(b, hk) + begin) : nullptr;
    const int64_t kp = L.k.sn * (int64_t)sizeof(T), vp = L.v.sn * (int64_t)sizeof(T),
                  mp = has_m ? L.m.sn * (int64_t)sizeof(T) : 0;  // bytes between positions
    const int rowb = P.dim * (int)sizeof(T);
    // A lane's offsets inside a step do not change.  Keys: with KLDS a load takes whole rows, 64 / CPR of
    // them, which the wave turns in its own part of LDS (position c, 16-byte chunk 4 s + g; chunks are
    // permuted by the position so that neither side meets bank conflicts); loaded as the operand wants
    // them, 64 bytes of each of 16 rows at a time, they come 8 to 12% slower (32 x 8192: 278 -> 244 us).
    // Values: positions 16 t + 4 g + i.
    constexpr int CPR = G::CPR, LOADS = KT * KS;
    int ko[KLDS ? 1 : KS];
    if constexpr (KLDS) {
        ko[0] = lane % CPR * KE < P.dim ? lane / CPR * (int)kp + lane % CPR * 16 : kDraftOut;
    } else {
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int d = (KE * 4) * s + KE * g;
            ko[s] = d < P.dim ? c * (int)kp + d * (int)sizeof(T) : kDraftOut;
        }
    }
    u32x4_d* const s_k = s_q + QWORDS / 4 + wave * (G::STEP * CPR);
    constexpr int CMASK = CPR < 16 ? CPR - 1 : 15;
    auto chunk = [](int position, int ch) __attribute__((always_inline)) -> int {
        return position * CPR + (ch ^ (position & CMASK));
    };
    const bool vin = VE * c < P.dim;
    const int vo = vin ? 4 * g * (int)vp + VE * c * (int)sizeof(T) : kDraftOut;
    const int mo = vin ? 4 * g * (int)mp + VE * c * (int)sizeof(T) : kDraftOut;

    // One set of registers for the keys and one for the values: the next step's keys are loaded as soon as
    // this step's scores are formed, its values as soon as they have been summed, so that loads are in
    // flight all the time (and twice the waves fit, against two sets).
    u32x4_d kr[LOADS];
    uint32_t v[G::NP][G::VW];
    uint32_t mv[VM ? G::NP : 1][VM ? G::VW : 1];
    uint32_t bz[KT][4];
    auto load_k = [&](int j0) __attribute__((always_inline)) {
        const int left = cnt - j0;  // positions of the unit from here; none past its last step
        const auto rk = draft_buffer(kb + j0 * kp, left > 0 ? (left - 1) * kp + rowb : 0);
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
            kr[i] = __builtin_amdgcn_raw_buffer_load_b128(
                rk, KLDS ? ko[0] + i * (64 / CPR) * (int)kp : ko[KLDS ? 0 : i % KS] + i / KS * 16 * (int)kp, 0, kDraftStream);
    };
    auto load_bias = [&](int j0) __attribute__((always_inline)) {
        if (!bb) return;
        const auto rb = draft_buffer(bb + 4ll * j0, 4ll * (cnt - j0));
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                bz[t][i] = __builtin_amdgcn_raw_buffer_load_b32(rb, 16 * g + 64 * t + 4 * i, 0, 0);
    };
    auto load_v = [&](int j0) __attribute__((always_inline)) {
        const int left = cnt - j0;
        const auto rv = draft_buffer(vb + j0 * vp, left > 0 ? (left - 1) * vp + rowb : 0);
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                buffer_words<G::VW>(rv, vo + (16 * t + i) * (int)vp, v[4 * t + i]);
        if constexpr (VM)
            if (has_m) {
                const auto rm = draft_buffer(mb + j0 * mp, left > 0 ? (left - 1) * mp + rowb : 0);
#pragma unroll
                for (int t = 0; t < KT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        buffer_words<G::VW>(rm, mo + (16 * t + i) * (int)mp, mv[4 * t + i]);
            }
    };

    constexpr int STEP = 64 * KT;  // the workgroup's positions per round of steps
    const int first = wave * 16 * KT;
    // the first step is on its way before the queries are needed (a tree's workgroup has none)
    load_k(first);
    load_bias(first);
    load_v(first);
    if constexpr (QLDS) {
#pragma unroll
        for (int k = 0; k < RT * KS / 4; ++k) s_q[(wave * (RT * KS / 4) + k) * 64 + lane] = qt[k];
        __syncthreads();
    }
    const float sl2 = P.scale * kLog2e, cl2 = P.softclamp * kLog2e;
    const float unclamped = P.softclamp > 0.f ? P.scale / P.softclamp : sl2;

    if (tree) {  // 16 drafted keys per wave
        if (blockIdx.x + blockIdx.y + blockIdx.z == 0 && wave == 3) draft_none(P, lane);
        if (16 * wave >= P.T) return;
        const uint64_t anc = draft_ancestors(P.parents ? P.parents + b * P.parents_stride : nullptr, P.T, lane);
        const uint32_t anc_lo = (uint32_t)anc, anc_hi = (uint32_t)(anc >> 32);
        const T* row = L.dk.at<T>(b, hk) + min(16 * wave + c, P.T - 1) * L.dk.sn;
        u32x4_d kf[KS];
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int d = (KE * 4) * s + KE * g;
            kf[s] = d < P.dim ? load16u(row + d) : u32x4_d{0u, 0u, 0u, 0u};
        }
        if (blockIdx.y == 0 && blockIdx.z == 0 && wave == 0) {  // for the join
            const uint64_t live = __ballot(anc != 0);
            draft_units(P, b, 0, lane, U);
            if (lane == 0) P.ws_u[b] = make_int4(U.first, U.number, (int)(uint32_t)live, (int)(live >> 32));
        }
        float* to = P.ws_t + (((int64_t)b * P.kv_heads + hk) * P.rec_rows + L.row0 + r0) * P.t16;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            if (rt >= nrt) break;
            f32x4_t a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const u32x4_d q = QLDS ? s_q[(rt * KS + s) * 64 + lane] : qf[QLDS ? 0 : rt][s];
                if constexpr (G::F32) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) a = mma_f32(kf[s][j], q[j], a);
                } else {
                    a = Mma16<T>::run(kf[s], q, a);
                }
            }
            const int r = r0 + 16 * rt + c;
            const uint64_t sees = ((uint64_t)__shfl(anc_hi, r % P.T) << 32) | __shfl(anc_lo, r % P.T);
            f32x4_t y;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = a[i] * unclamped;
                y[i] = (sees >> (16 * wave + 4 * g + i)) & 1 ? (P.softclamp > 0.f ? cl2 * tanhf(x) : x) : -INFINITY;
            }
            if (16 * rt + c < nrows)
                *reinterpret_cast<f32x4_t*>(to + (int64_t)(16 * rt + c) * P.t16 + 16 * wave + 4 * g) = y;
        }
        return;
    }

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
        if constexpr (KLDS) {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) s_k[chunk(i * (64 / CPR) + lane / CPR, lane % CPR)] = kr[i];
            // other lanes of the wave read them: LDS keeps a wave's order, the compiler has to as well
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            load_k(j0 + STEP);
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
                    for (int i = 0; i < 4; ++i) x[rt][t][i] = cl2 * tanhf(x[rt][t][i]);
        }
        if (bb) {
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
                        x[rt][t][i] = fmaf(__uint_as_float(bz[t][i]), kLog2e, x[rt][t][i]);
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
        if constexpr (!KLDS) load_k(j0 + STEP);
        load_bias(j0 + STEP);
        __builtin_amdgcn_sched_barrier(0);
        // probabilities (16-bit types: their leading bits, and the rest); 0 for a tile without rows, whose test would
        // else keep the scores alive beside them (52 spilled registers with four tiles)
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
                    draft_weights2<T, VM>(x[rt][t][0], x[rt][t][1], pf[rt][2 * t], pl[rt][2 * t], has_m);
                    draft_weights2<T, VM>(x[rt][t][2], x[rt][t][3], pf[rt][2 * t + 1], pl[rt][2 * t + 1], has_m);
                }
            }
        }
        // O^T += V^T P^T, feature j of every lane's VE per tile
#pragma unroll
        for (int j = 0; j < VE; ++j) {
            if constexpr (G::F32) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t a = v[i][j];
                    if constexpr (VM)
                        if (has_m) a = __float_as_uint(__uint_as_float(a) * __uint_as_float(mv[i][j]));
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
                        if (rt < nrt) o[rt][j] = mma_f32(a, pf[rt][i], o[rt][j]);
                }
            } else {
                const uint32_t sel = j & 1 ? 0x07060302u : 0x05040100u;
                u32x4_d a, a2 = {0u, 0u, 0u, 0u};
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    a[e] = __builtin_amdgcn_perm(v[2 * e + 1][j / 2], v[2 * e][j / 2], sel);
                if constexpr (VM)
                    if (has_m) {
                        // one rounding of the product was most of a middle level's error
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t y = __builtin_amdgcn_perm(mv[2 * e + 1][j / 2], mv[2 * e][j / 2], sel);
                            draft_mul2<T>(a[e], y, a, a2, e);
                        }
                    }
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    if (rt >= nrt) break;
                    const u32x4_d p = {pf[rt][0], pf[rt][1], pf[rt][2], pf[rt][3]};
                    const u32x4_d p2 = {pl[rt][0], pl[rt][1], pl[rt][2], pl[rt][3]};
                    o[rt][j] = draft_weigh<T, VM>(a, a2, p, p2, o[rt][j], has_m);
                }
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        load_v(j0 + STEP);
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
    const int64_t rec = ((int64_t)unit * P.kv_heads + hk) * P.rec_rows + L.row0 + r0;
    if (tid < nrows) {
        float top = s_m[0][tid], sum = 0.f;
        for (int w = 1; w < 4; ++w) top = fmaxf(top, s_m[w][tid]);
        for (int w = 0; w < 4; ++w)
            sum += s_m[w][tid] == -INFINITY ? 0.f : s_l[w][tid] * __builtin_amdgcn_exp2f(s_m[w][tid] - top);
        P.ws_s[rec + tid] = make_float2(top, sum);
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
        if (16 * rt + r < nrows)
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
                *reinterpret_cast<float4*>(P.ws_o + (rec + 16 * rt + r) * P.dim + d) = y;
            }
        if (rt + 1 < RT) __syncthreads();
    }
}

inline dim3 draft_partial_grid(const DraftDev& P, int units) {
    return dim3(P.batch + units, P.kv_heads * P.row_blocks, P.order);
}

template <typename T, int D, int RT>
void launch_draft_partial_rt(const DraftDev& P, int units, bool vmul, hipStream_t s) {
    if (vmul) hipLaunchKernelGGL((k_draft_partial<T, D, RT, true>), draft_partial_grid(P, units), dim3(kDraftThreads), 0, s, P);
    else hipLaunchKernelGGL((k_draft_partial<T, D, RT, false>), draft_partial_grid(P, units), dim3(kDraftThreads), 0, s, P);
}

template <typename T, int D>
void launch_draft_partial_d(const DraftDev& P, int units, int tiles, bool vmul, hipStream_t s) {
    constexpr int most = draft_row_tiles<T>(D, false), most_m = draft_row_tiles<T>(D, true);
    if (tiles == 1) return launch_draft_partial_rt<T, D, 1>(P, units, vmul, s);
    if constexpr (most >= 2)
        if (tiles == 2) return launch_draft_partial_rt<T, D, 2>(P, units, vmul, s);
    if constexpr (most_m >= 4)  // a middle level's alone
        hipLaunchKernelGGL((k_draft_partial<T, D, 4, true>), draft_partial_grid(P, units), dim3(kDraftThreads), 0, s, P);
}

template <typename T>
void launch_draft_partial(const DraftDev& P, int units, int tiles, bool vmul, hipStream_t s) {
    if (P.dim <= 64) launch_draft_partial_d<T, 64>(P, units, tiles, vmul, s);
    else if (P.dim <= 128) launch_draft_partial_d<T, 128>(P, units, tiles, vmul, s);
    else launch_draft_partial_d<T, 256>(P, units, tiles, vmul, s);
}

}  // namespace pa
