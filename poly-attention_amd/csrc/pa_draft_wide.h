// pa_draft_wide.h -- k_draft_wide: the cached positions of a drafted step with many rows.
//
// k_draft_partial gives each wave positions of its own and all rows of the block, and what it does once
// per wave and position (the keys' way through LDS, the values' transposition) with many rows leaves no
// room for a second wave per SIMD.  Here the four waves of a workgroup hold rows of their own, up to 16 RT
// each, and all of them take all positions of the unit from LDS.
//
// The products and the lane layout are those of k_draft_partial (S^T = K Q^T, O^T += V^T P^T, 16x16
// tiles).  Keys and values go from memory to LDS directly, NS stages of SP positions in a ring, one
// barrier per stage; V^T's operand comes from transposing reads (ds_read_b64_tr_b16).  A row of 16-byte
// chunks is stored with its chunks permuted by the position (chunk ch at ch ^ position), so that 16
// positions' equal chunks lie on different banks for both kinds of reads.  A wave holds whole rows: the
// results go to their records from registers, and nothing is joined.
//
// Bound by neither the loads nor the products alone but by how far they overlap, at two waves per SIMD.
// 8 x 4096 positions of 128, 8 key heads, behind cold caches: 64 rows 76 us (loads alone 62; k_draft_partial 94),
// 128 rows 89 (71), 256 rows in two blocks 143 (91).  With one product per weight and value instead of two (weights
// rounded to the type): 73, 86 and 131; at that stage, loads not marked as streaming: 135 us for 128 rows; a row
// tile's number tested inside the loop, which keeps LDS reads from running ahead of it: 166 us for 256 rows, 155
// without; eight waves with 256 rows: 154.
#pragma once

#include <type_traits>

#include "pa_draft_partial.h"
#include "pa_mfma.h"

namespace pa {

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// as dma16, marked as streaming
__device__ __forceinline__ void dma16_nt(srd_t srd, uint32_t lds, uint32_t voff) {
    lds = __builtin_amdgcn_readfirstlane(lds);
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 4\n\tbuffer_load_dwordx4 %0, %2, 0 offen nt lds"
                 :
                 : "v"(voff), "s"(lds), "s"(srd)
                 : "memory", "m0");
}
// as dma16, 4 bytes a lane
__device__ __forceinline__ void dma4(srd_t srd, uint32_t lds, uint32_t voff) {
    lds = __builtin_amdgcn_readfirstlane(lds);
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 4\n\tbuffer_load_dword %0, %2, 0 offen lds"
                 :
                 : "v"(voff), "s"(lds), "s"(srd)
                 : "memory", "m0");
}
#pragma clang diagnostic pop

template <typename T, int D, bool VM>
__global__ __launch_bounds__(64 * kDraftWideWaves, 2) void k_draft_wide(const DraftDev P) {
    constexpr int RT = draft_wide_tiles(D), NW = kDraftWideWaves;
    constexpr int KS = D / 32, VE = D / 16;  // key steps of 32 features, output tiles of 16
    constexpr int CPR = D / 8, CMASK = CPR < 16 ? CPR - 1 : 15;
    constexpr int SP = D <= 64 ? 64 : 32;          // positions of a stage
    constexpr int NS = VM ? 3 : 4;                 // stages; 72 or 64 KB: two workgroups per CU
    constexpr int TILE = SP * CPR * 16;            // bytes of a stage's keys (values, multipliers)
    constexpr int LOADS = TILE / (1024 * NW);      // 16-byte loads of a lane per tile
    constexpr int TILES = VM ? 3 : 2;
    static_assert(LOADS * 1024 * NW == TILE, "whole loads");
    __shared__ __align__(16) char s_tile[NS][TILES][TILE];
    __shared__ __align__(16) float s_bias[NS][NW][64];  // a copy per wave: equal loads in all of them

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int hk = blockIdx.y / P.row_blocks, b0 = (blockIdx.y % P.row_blocks) * 16 * NW * RT;
    const DraftLevelDev L = P.L[P.order - 1 - blockIdx.z];  // the level of most rows first
    if (b0 >= L.rows) return;
    const int brows = min(16 * NW * RT, L.rows - b0);
    const int wrows = 16 * ((brows + 16 * NW - 1) / (16 * NW));  // a wave's rows, at most ...
    const int r0 = b0 + wave * wrows;
    const int nrows = min(wrows, b0 + brows - r0);               // ... and the rows it has (none: <= 0)
    const int nrt = nrows > 0 ? (nrows + 15) / 16 : 0;
    const bool tree = (int)blockIdx.x < P.batch;
    const int unit = blockIdx.x - P.batch;
    DraftUnits U;
    if (!tree && !draft_units(P, -1, unit, lane, U)) return;
    const int b = tree ? (int)blockIdx.x : U.b;
    const int64_t begin = tree ? 0 : (int64_t)U.place * U.size * kDraftChunk;
    const int cnt = tree ? 0 : __builtin_amdgcn_readfirstlane((int)min((int64_t)U.size * kDraftChunk, draft_count(P, b) - begin));

    u32x4_d qf[RT][KS];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int r = min(r0 + 16 * rt + c, L.rows - 1);
        const T* row = L.q.at<T>(b, hk * L.rep + r / P.T) + (int64_t)(r % P.T) * L.q.sn;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int d = 32 * s + 8 * g;
            qf[rt][s] = d < P.dim ? load16u(row + d) : u32x4_d{0u, 0u, 0u, 0u};
        }
    }
    const float sl2 = P.scale * kLog2e, cl2 = P.softclamp * kLog2e;
    const float unclamped = P.softclamp > 0.f ? P.scale / P.softclamp : sl2;

    if (tree) {  // a wave's rows against all drafted keys
        if (blockIdx.x + blockIdx.y + blockIdx.z == 0 && wave == 3) draft_none(P, lane);
        const uint64_t anc = draft_ancestors(P.parents ? P.parents + b * P.parents_stride : nullptr, P.T, lane);
        const uint32_t anc_lo = (uint32_t)anc, anc_hi = (uint32_t)(anc >> 32);
        if (blockIdx.y == 0 && blockIdx.z == 0 && wave == 0) {  // for the join
            const uint64_t live = __ballot(anc != 0);
            draft_units(P, b, 0, lane, U);
            if (lane == 0) P.ws_u[b] = make_int4(U.first, U.number, (int)(uint32_t)live, (int)(live >> 32));
        }
        float* to = P.ws_t + (((int64_t)b * P.kv_heads + hk) * P.rec_rows + L.row0 + r0) * P.t16;
        for (int k0 = 0; k0 < P.T; k0 += 16) {
            const T* row = L.dk.at<T>(b, hk) + min(k0 + c, P.T - 1) * L.dk.sn;
            u32x4_d kf[KS];
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const int d = 32 * s + 8 * g;
                kf[s] = d < P.dim ? load16u(row + d) : u32x4_d{0u, 0u, 0u, 0u};
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                if (rt >= nrt) break;
                f32x4_t a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = 0; s < KS; ++s) a = Mma16<T>::run(kf[s], qf[rt][s], a);
                const int n = (r0 + 16 * rt + c) % P.T;
                const uint64_t sees = ((uint64_t)__shfl(anc_hi, n) << 32) | __shfl(anc_lo, n);
                f32x4_t y;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float x = a[i] * unclamped;
                    y[i] = (sees >> (k0 + 4 * g + i)) & 1 ? (P.softclamp > 0.f ? cl2 * tanhf(x) : x) : -INFINITY;
                }
                if (16 * rt + c < nrows)
                    *reinterpret_cast<f32x4_t*>(to + (int64_t)(16 * rt + c) * P.t16 + k0 + 4 * g) = y;
            }
        }
        return;
    }

    const bool has_m = VM && L.m.p, has_b = L.bias.p;
    const char* kb = reinterpret_cast<const char*>(L.k.at<T>(b, hk) + begin * L.k.sn);
    const char* vb = reinterpret_cast<const char*>(L.v.at<T>(b, hk) + begin * L.v.sn);
    const char* mb = has_m ? reinterpret_cast<const char*>(L.m.at<T>(b, hk) + begin * L.m.sn) : vb;
    const char* bb = has_b ? reinterpret_cast<const char*>(L.bias.at<float>(b, hk) + begin) : vb;
    const int64_t kp = L.k.sn * (int64_t)sizeof(T), vp = L.v.sn * (int64_t)sizeof(T),
                  mp = has_m ? L.m.sn * (int64_t)sizeof(T) : 0;  // bytes between positions
    const int rowb = P.dim * (int)sizeof(T);
    // lane l of load i of a wave fills slot (NW i + wave) 64 + l of the tile
    int pos[LOADS], col[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int slot = (NW * i + wave) * 64 + lane;
        pos[i] = slot / CPR;
        const int ch = (slot % CPR) ^ (pos[i] & CMASK);
        col[i] = ch * 8 < P.dim ? ch * 16 : kDraftOut;
    }
    const uint32_t tile0 = lds_addr(&s_tile[0][0][0]) + wave * 1024, bias0 = lds_addr(&s_bias[0][0][0]) + wave * 256;
    // what is loaded does not pass the unit's end: such loads give 0 without touching memory
    auto bytes = [](int64_t n) __attribute__((always_inline)) -> uint32_t {
        return n <= 0 ? 0u : n > 0x40000000 ? 0x40000000u : (uint32_t)n;
    };
    auto load = [&](int st) __attribute__((always_inline)) {
        const int64_t j0 = (int64_t)st * SP, left = cnt - j0;
        const uint32_t at = tile0 + (st % NS) * (TILES * TILE);
        auto tile = [&](const char* p, int64_t pitch, uint32_t to, bool there = true) __attribute__((always_inline)) {
            const srd_t r = make_srd(p + j0 * pitch, bytes(there && left > 0 ? (left - 1) * pitch + rowb : 0));
#pragma unroll
            for (int i = 0; i < LOADS; ++i)
                dma16_nt(r, to + i * (1024 * NW), col[i] == kDraftOut ? kDraftOut : pos[i] * (int)pitch + col[i]);
        };
        tile(kb, kp, at);
        tile(vb, vp, at + TILE);
        if constexpr (VM) tile(mb, mp, at + 2 * TILE, has_m);
        dma4(make_srd(bb + 4 * j0, has_b ? bytes(4 * left) : 0u), bias0 + (st % NS) * (256 * NW), lane < SP ? 4 * lane : kDraftOut);
    };
    constexpr int OPS = TILES * LOADS + 1;  // loads of a wave per stage

    const int stages = (cnt + SP - 1) / SP;
    for (int st = 0; st < NS - 1; ++st) load(st);

    // NR: the wave's tiles, a compile-time number (a test per tile keeps the reads of LDS from running ahead)
    // and whether the level is a middle one, for the same reason
    auto run = [&](auto tiles, auto middle) __attribute__((always_inline)) {
        constexpr int NR = decltype(tiles)::value;
        constexpr bool MID = decltype(middle)::value;
        f32x4_t o[NR + 1][VE];
        float m[NR + 1], l[NR + 1];
#pragma unroll
        for (int rt = 0; rt < NR; ++rt) {
            m[rt] = -INFINITY;
            l[rt] = 0.f;
#pragma unroll
            for (int j = 0; j < VE; ++j) o[rt][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        }
        for (int st = 0; st < stages; ++st) {
            wait_vmcnt<(NS - 2) * OPS>();  // this wave's loads of the stage ...
            lds_barrier();                 // ... and everyone's; the stage before it has been read
            load(st + NS - 1);
            if constexpr (NR == 0) continue;
            const char* const tk = s_tile[st % NS][0];
            const char* const tv = s_tile[st % NS][1];
            const char* const tm = s_tile[st % NS][TILES - 1];
            const float* const tb = s_bias[st % NS][wave];
#pragma unroll
            for (int p0 = 0; p0 < SP; p0 += 32) {
                const int j0 = st * SP + p0;
                if (p0 > 0 && j0 >= cnt) break;
                f32x4_t x[NR + 1][2];
#pragma unroll
                for (int rt = 0; rt < NR; ++rt)
#pragma unroll
                    for (int t = 0; t < 2; ++t) x[rt][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    u32x4_d k[2];
#pragma unroll
                    for (int t = 0; t < 2; ++t)
                        k[t] = *reinterpret_cast<const u32x4_d*>(tk + ((p0 + 16 * t + c) * CPR + ((4 * s + g) ^ (c & CMASK))) * 16);
#pragma unroll
                    for (int rt = 0; rt < NR; ++rt) {
#pragma unroll
                        for (int t = 0; t < 2; ++t) x[rt][t] = Mma16<T>::run(k[t], qf[rt][s], x[rt][t]);
                    }
                }
                f32x4_t z[2];  // 0 without a bias
#pragma unroll
                for (int t = 0; t < 2; ++t)
                    z[t] = *reinterpret_cast<const f32x4_t*>(tb + p0 + 16 * t + 4 * g) * kLog2e;
                if (P.softclamp > 0.f) {
#pragma unroll
                    for (int rt = 0; rt < NR; ++rt)
#pragma unroll
                        for (int t = 0; t < 2; ++t)
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                x[rt][t][i] = fmaf(cl2, tanhf(x[rt][t][i] * unclamped), z[t][i]);
                } else {
#pragma unroll
                    for (int rt = 0; rt < NR; ++rt)
#pragma unroll
                        for (int t = 0; t < 2; ++t)
#pragma unroll
                            for (int i = 0; i < 4; ++i) x[rt][t][i] = fmaf(x[rt][t][i], unclamped, z[t][i]);
                }
                if (j0 + 32 > cnt) {  // the unit's last positions
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int rt = 0; rt < NR; ++rt)
                                if (j0 + 16 * t + 4 * g + i >= cnt) x[rt][t][i] = -INFINITY;
                }
                u32x4_d pf[NR + 1], pl[NR + 1];  // leading bits and the rest
#pragma unroll
                for (int rt = 0; rt < NR; ++rt) {
                    float top = x[rt][0][0];
#pragma unroll
                    for (int t = 0; t < 2; ++t)
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
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            x[rt][t][i] = __builtin_amdgcn_exp2f(x[rt][t][i] - ms);
                            l[rt] += x[rt][t][i];
                        }
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            uint32_t hi, lo;
                            draft_weights2<T, MID>(x[rt][t][2 * i], x[rt][t][2 * i + 1], hi, lo, MID);
                            pf[rt][2 * t + i] = hi;
                            pl[rt][2 * t + i] = lo;
                        }
                }
                // O^T += V^T P^T, features 16 j + c; lane L of a group of 16 reads position L / 4, columns 4 (L % 4)
                const int vrow = 4 * g + (c >> 2), vch = (c >> 1) & 1, vlow = (c & 1) * 8;
                auto turned = [&](const char* from, int j) __attribute__((always_inline)) -> u32x4_d {
                    u32x4_d a;
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        const u32x2_t w = lds_read_tr(from + ((p0 + 16 * t + vrow) * CPR + ((2 * j + vch) ^ (vrow & CMASK))) * 16 + vlow);
                        a[2 * t] = w[0];
                        a[2 * t + 1] = w[1];
                    }
                    return a;
                };
#pragma unroll
                for (int j = 0; j < VE; ++j) {
                    u32x4_d a = turned(tv, j), a2 = {0u, 0u, 0u, 0u};
                    if constexpr (MID) {
                        const u32x4_d y = turned(tm, j), x1 = a;
#pragma unroll
                        for (int e = 0; e < 4; ++e) draft_mul2<T>(x1[e], y[e], a, a2, e);
                    }
#pragma unroll
                    for (int rt = 0; rt < NR; ++rt) o[rt][j] = draft_weigh<T, MID>(a, a2, pf[rt], pl[rt], o[rt][j], MID);
                }
            }
        }
        wait_vmcnt<0>();  // no load is on its way to LDS when the workgroup ends

        const int64_t rec = ((int64_t)unit * P.kv_heads + hk) * P.rec_rows + L.row0 + r0;
#pragma unroll
        for (int rt = 0; rt < NR; ++rt) {
            l[rt] += __shfl_xor(l[rt], 16);
            l[rt] += __shfl_xor(l[rt], 32);
            const int r = 16 * rt + c;
            if (r >= nrows) continue;
            if (g == 0) P.ws_s[rec + r] = make_float2(m[rt], l[rt]);  // without a maximum 0, or no number
#pragma unroll
            for (int j = 0; j < VE; ++j)
                if (16 * j + 4 * g < P.dim) *reinterpret_cast<f32x4_t*>(P.ws_o + (rec + r) * P.dim + 16 * j + 4 * g) = o[rt][j];
        }
    };
    auto level = [&](auto middle) __attribute__((always_inline)) {
        if (nrt == 0) run(std::integral_constant<int, 0>{}, middle);
        else if (nrt == 1) run(std::integral_constant<int, 1>{}, middle);
        else if (RT == 2 || nrt == 2) run(std::integral_constant<int, 2>{}, middle);
        else run(std::integral_constant<int, RT>{}, middle);
    };
    if constexpr (VM) {
        if (has_m) return level(std::true_type{});
    }
    level(std::false_type{});
}

template <typename T, int D>
void launch_draft_wide_d(const DraftDev& P, int units, bool vmul, hipStream_t s) {
    const dim3 grid = draft_partial_grid(P, units), block(64 * kDraftWideWaves);
    if (vmul) hipLaunchKernelGGL((k_draft_wide<T, D, true>), grid, block, 0, s, P);
    else hipLaunchKernelGGL((k_draft_wide<T, D, false>), grid, block, 0, s, P);
}

template <typename T>
void launch_draft_wide(const DraftDev& P, int units, bool vmul, hipStream_t s) {
    if (P.dim <= 64) launch_draft_wide_d<T, 64>(P, units, vmul, s);
    else launch_draft_wide_d<T, 128>(P, units, vmul, s);
}

}  // namespace pa
