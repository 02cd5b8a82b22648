// pa_paged_tiles.h -- k_paged_tiles: a unit of positions for a tile of many query rows (16-bit types, head dims to 128).
//
// A wave holds 32 QB rows, and the workgroup's waves share tiles of 64 positions, which travel from memory to LDS
// directly, four stages in a ring, filled and waited for in pairs.  S^T = K Q^T with 32x32x16 tiles; a lane has one
// query row of each block, so the softmax state is a scalar, and the probabilities are the operand of
// O^T += V^T P^T where they lie (pa_mfma.h); V^T comes from transposing reads.  16 positions lie in one
// page: the loads of a wave go to one page each, whose number is a scalar from a register of 64 that is
// loaded ahead.
//
// A wave works on two blocks of 32 x 32 scores at once, one's products beside the other's exponentials: two blocks of
// rows at head dim 64, where each fragment read from LDS feeds two products; two of positions at 128, eight waves of 32
// rows, since two blocks of rows there pass 256 registers, and copies between the two halves of the register file took
// a quarter of the time.  4096 tokens behind 4096, 32/8 heads of 128, the final level: 672 us so, 500 with eight waves, 450
// (910 TFLOP/s) with the fragments read and the loads sent where they are now: between products that wait for one another.
// No maximum is taken per tile: the probabilities are formed against the running one, and a tile whose sums
// say that it was passed by far, or a row that has none yet, is formed again (kTileCap).  Scores get the logsumexp
// of the level below as the products' initial value.
//
// What a level leaves in the cache is kept, and read by every later token: its weights enter the products as two numbers of the
// operands' type, as in k_paged_rows, so that it does not depend on how many tokens a chunk has. The final level's weights are
// rounded once, and divided by the sum of the rounded ones: of a row's many weights each is off by at most half a step, and the
// output, 2^-9 off by its own rounding in bf16, 1.2 to 1.4 times as far off as that alone (fp16 the same). 4096 tokens behind
// 4096, 32/8 heads of 128: 631 us so, 800 with two numbers at the final level too, 587 with one at both, which left the cached
// values 1.4 times as far off, at each level anew.
#pragma once

#include <type_traits>

#include "pa_mfma.h"
#include "pa_paged.h"

namespace pa {

constexpr int kTileKeys = 64, kTileStages = 4;
constexpr float kTileCap = 8192.f;  // of a lane's sum of a tile's probabilities

// waves of a workgroup, and 32-row blocks of a wave
constexpr int paged_tile_waves(int D) { return D == 128 ? 8 : 4; }
constexpr int paged_tile_blocks(int D) { return 8 / paged_tile_waves(D); }

template <typename T, int D, bool SOFTCLAMP, bool BIAS, bool LAST>
__global__ __launch_bounds__(64 * paged_tile_waves(D), 2) void k_paged_tiles(const PagedDev P) {
    constexpr int NW = paged_tile_waves(D), QB = paged_tile_blocks(D), NT = 64 * NW;
    using M = Mma<T>;
    typedef typename M::frag frag;
    constexpr int BN = kTileKeys, CPR = D / 8, NL = BN * CPR / NT, NSTG = kTileStages;
    constexpr int ELEMS = BN * D;
    // fp16's smallest numbers are near: its weights are held 2^7 times larger
    constexpr float LIFT = draft_lift<T>();
    __shared__ __attribute__((aligned(16))) T sK[NSTG * ELEMS];
    __shared__ __attribute__((aligned(16))) T sV[NSTG * ELEMS];
    __shared__ __attribute__((aligned(16))) float sBraw[NSTG][BN];
    __shared__ __attribute__((aligned(16))) float sBw[NW][2][BN];  // a wave's, of a pair of tiles, in the scores' unit

    const int tid = threadIdx.x, lane = tid & 63, w = wave_id();
    const int hh = lane >> 5, col = lane & 31;
    const int hk = __builtin_amdgcn_readfirstlane(blockIdx.x % P.kv_heads);
    // eight of them, whatever the waves; 0 too where there is no unit, so that the join looks for none
    auto flag = [&](bool any) __attribute__((always_inline)) {
        if (lane < 8 / NW) *paged_flag(P, w + NW * lane) = any;
    };
    PagedUnit U;
    if (!paged_find<kUnits>(P, blockIdx.x / P.kv_heads, lane, U)) return flag(false);
    const int begin = U.split * U.size * kPagedChunk;
    const int cnt = min(U.size * kPagedChunk, paged_keys(P, U) - begin);
    if (cnt <= 0) return flag(false);  // past the tile's last token: the join knows
    const int r0 = U.tile * P.tile + w * 32 * QB, rend = min((U.tile + 1) * P.tile, U.rows);

    constexpr bool TWO = !LAST;  // numbers of the type that a weight is in its product
    struct Weights {
        u32x4_t hi[2], lo[TWO ? 2 : 1];
    };
    frag qf[QB][D / 16];
    f32x16_t o[QB][D / 32];
    float m[QB], l[QB];
    int see[QB];  // the last position that a row sees, from the unit's first
#pragma unroll
    for (int u = 0; u < QB; ++u) {
        const int r = min(r0 + 32 * u + col, U.rows - 1);  // rows past the end repeat the last one
        const T* row = paged_query<T>(P, U, hk, r);
        const T* from = row ? row : reinterpret_cast<const T*>(P.keys);
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
            const int d = c * 16 + 8 * hh;
            u32x4_t raw = *reinterpret_cast<const u32x4_t*>(from + (d < P.dim ? d : 0));
            if (!row || d >= P.dim) raw = u32x4_t{0u, 0u, 0u, 0u};
            qf[u][c] = __builtin_bit_cast(frag, raw);
        }
#pragma unroll
        for (int x = 0; x < D / 32; ++x) o[u][x] = zero16();
        m[u] = -INFINITY;
        l[u] = 0.f;
        see[u] = U.row.p0 + r / P.rep - begin;
    }
    const int all_see = U.row.p0 + __builtin_amdgcn_readfirstlane(min(r0, U.rows - 1) / P.rep) - begin;
    const int last_see = U.row.p0 + __builtin_amdgcn_readfirstlane(min(min(r0 + 32 * QB, rend) - 1, U.rows - 1) / P.rep) - begin;

    // the pages of 64 blocks of 16 positions, lane i's the i-th
    const int32_t* const pages = P.p.table + (int64_t)U.b * P.p.max_pages;
    const int inside = (1 << P.p.lg) - 1;
    auto load_pages = [&](int at) __attribute__((always_inline)) -> int {
        return pages[(begin + min(at + 16 * lane, cnt - 1)) >> P.p.lg];
    };
    int ids = load_pages(0), ids_next = cnt > 1024 ? load_pages(1024) : 0, block = 0;
    // these loads are the only ones that the compiler sees: retire them before the first direct one
#pragma unroll
    for (int u = 0; u < QB; ++u)
#pragma unroll
        for (int c = 0; c < D / 16; ++c) qf[u][c] = opaque(qf[u][c]);
    ids = opaque(ids);
    ids_next = opaque(ids_next);

    const int rowb = P.dim * 2;
    // a thread's 16-byte chunks of a tile, n * NT + tid: row p / CPR, chunk p % CPR permuted by the row
    auto swz_key = [](int r) __attribute__((always_inline)) -> int {
        if (D == 64) {
            const int v = (r >> 1) & 7;
            return ((v & 1) << 2) | (v & 2) | ((v >> 2) & 1);
        }
        return r & 15;
    };
    auto swz_val = [](int r) __attribute__((always_inline)) -> int { return D == 64 ? 2 * (r & 3) : 4 * (r & 3); };
    uint32_t offk[NL], offv[NL];
#pragma unroll
    for (int n = 0; n < NL; ++n) {
        const int p = n * NT + tid, r = p / CPR, ph = p % CPR;
        const int ck = ph ^ swz_key(r), cv = ph ^ swz_val(r);
        offk[n] = ck * 8 < P.dim ? (r & 15) * rowb + ck * 16 : kDraftOut;
        offv[n] = cv * 8 < P.dim ? (r & 15) * rowb + cv * 16 : kDraftOut;
    }
    const uint32_t lds_k = lds_addr(sK), lds_v = lds_addr(sV), lds_b = lds_addr(&sBraw[0][0]);
    auto turn_page = [&](int j0) __attribute__((always_inline)) {
        if (j0 >> 10 == block) return;
        block = j0 >> 10;
        ids = ids_next;
        if (j0 + 1024 < cnt) ids_next = load_pages((block + 1) << 10);
    };
    // a wave's part n of NL of a tile's loads; 0 past the unit's end
    auto issue_part = [&](int j0, int stage, int n) __attribute__((always_inline)) {
        const uint32_t kd = lds_k + (uint32_t)(stage * ELEMS * 2), vd = lds_v + (uint32_t)(stage * ELEMS * 2);
        const int j = j0 + ((n * NT + w * 64) / CPR & ~15);  // the block of 16 that the wave's rows lie in
        const int id = __builtin_amdgcn_readlane(ids, (j >> 4) & 63);
        const bool ok = (unsigned)id < (unsigned)P.p.pages;
        const int64_t at = (paged_base(P, ok ? id : 0, hk) + ((begin + j) & inside)) * rowb;
        const uint32_t bytes = ok && j < cnt ? min(16, cnt - j) * rowb : 0;
        dma16(make_srd(P.keys + at, bytes), kd + (uint32_t)((n * NT + w * 64) * 16), offk[n]);
        dma16(make_srd(P.values + at, bytes), vd + (uint32_t)((n * NT + w * 64) * 16), offv[n]);
        if (BIAS && n == NL - 1 && w < 4) {
            const int j = j0 + 16 * w;  // a quarter of the tile's
            const int id = __builtin_amdgcn_readlane(ids, (j >> 4) & 63);
            const bool ok = (unsigned)id < (unsigned)P.p.pages;
            const int64_t at = paged_base(P, ok ? id : 0, hk) + ((begin + j) & inside);
            if (lane < 4)
                dma16(make_srd(P.bias + at, ok && j < cnt ? 64 : 0), lds_b + (uint32_t)(stage * BN * 4 + w * 64), 16 * lane);
        }
    };
    auto issue = [&](int j0, int stage) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < NL; ++n) issue_part(j0, stage, n);
    };

    int koff[D / 16];  // rows col (+ 32 kb), chunk 2c + hh
#pragma unroll
    for (int c = 0; c < D / 16; ++c) koff[c] = col * D + (((2 * c + hh) ^ swz_key(col)) * 8);
    int voff[D / 32];  // rows 4 hh + j / 4 (+ 16 t2 + 8 u + 32 kb), columns 32 x + col
    {
        const int g = lane >> 4, j = lane & 15, r = 4 * (g >> 1) + (j >> 2);
#pragma unroll
        for (int x = 0; x < D / 32; ++x) {
            const int ch = 4 * x + 2 * (g & 1) + ((j & 3) >> 1);
            voff[x] = r * D + ((ch ^ swz_val(r)) * 8) + 4 * (j & 1);
        }
    }

    const float sl2 = SOFTCLAMP ? 1.f : P.scale * kLog2e;        // what a score counts in log2 units
    const float bmul = SOFTCLAMP ? kLog2e : 1.f / P.scale;       // a logsumexp in the scores' unit
    const int ntl = (cnt + BN - 1) / BN;
    // steps of 32 positions; a wave without rows only keeps the barriers
    const int nact = r0 >= rend || last_see < 0 ? 0 : min((cnt + 31) / 32, last_see / 32 + 1);
    issue(0, 0);
    if (ntl > 1) issue(BN, 1);

    float odd = 0.f;  // no number: a value that is not finite lies among those that some row does not see
    // positions that a row of block u does not see, and those past the unit
    auto mask = [&](f32x16_t& s, int u, int j0) __attribute__((always_inline)) {
        const int lim = min(see[u], cnt - 1) - j0 - 4 * hh;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (8 * (i / 4) + (i % 4) > lim) s[i] = -INFINITY;
    };
    auto top = [&](const f32x16_t& s) __attribute__((always_inline)) -> float {
        float q[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 16; ++i) q[i & 3] = fmaxf(q[i & 3], s[i]);
        return xhalf_max(fmaxf(fmaxf(q[0], q[1]), fmaxf(q[2], q[3]))) * sl2 - LIFT;
    };
    auto clamp = [&](f32x16_t& s, const float* bias) __attribute__((always_inline)) {
        if constexpr (SOFTCLAMP)
            soft_clamp16<true>(s, P, [&](int g) __attribute__((always_inline)) {
                if (!BIAS) return make_float4(0.f, 0.f, 0.f, 0.f);
                return *reinterpret_cast<const float4*>(bias + 8 * g);
            });
    };
    // rows that have no maximum yet take the step's
    auto begin_rows = [&](const f32x16_t& s, int u) __attribute__((always_inline)) {
        if (__any(m[u] == -INFINITY)) {
            keep_branch();
            const float t = top(s);
            if (m[u] == -INFINITY) m[u] = t;
        }
    };
    // four probabilities of a block of rows into the packed operands and the sums
    auto four = [&](const f32x16_t& s, int i, float msub, Weights& pk, float (&lts)[4]) __attribute__((always_inline)) {
        const int a = 4 * i;
        const float p0 = fast_exp2(fmaf(s[a], sl2, -msub)), p1 = fast_exp2(fmaf(s[a + 1], sl2, -msub));
        const float p2 = fast_exp2(fmaf(s[a + 2], sl2, -msub)), p3 = fast_exp2(fmaf(s[a + 3], sl2, -msub));
        uint32_t w0, w1;
        if constexpr (TWO) {
            uint32_t r0, r1;
            draft_split2<T>(p0, p1, w0, r0);
            draft_split2<T>(p2, p3, w1, r1);
            pk.lo[a / 8][(a % 8) / 2] = r0;
            pk.lo[a / 8][(a % 8) / 2 + 1] = r1;
        } else {
            w0 = pack2<T>(p0, p1);
            w1 = pack2<T>(p2, p3);
        }
        pk.hi[a / 8][(a % 8) / 2] = w0;
        pk.hi[a / 8][(a % 8) / 2 + 1] = w1;
        if constexpr (LAST) {  // the weights as the products take them
            lts[(2 * i) % 4] = sum_pair<T>(w0, lts[(2 * i) % 4]);
            lts[(2 * i + 1) % 4] = sum_pair<T>(w1, lts[(2 * i + 1) % 4]);
        } else {
            lts[0] += p0;
            lts[1] += p1;
            lts[2] += p2;
            lts[3] += p3;
        }
    };
    auto without = [](float x) __attribute__((always_inline)) -> float { return x == -INFINITY ? 0.f : x; };
    // the rare path of a block whose sums passed the cap
    auto again = [&](const f32x16_t& s, int u, float lt, Weights& pk) __attribute__((always_inline)) {
        if (__any(!(lt <= kTileCap))) {
            keep_branch();
            const float mn = fmaxf(m[u], top(s));
            const float al = mn > m[u] ? fast_exp2(m[u] - mn) : 1.f;
            l[u] *= al;
#pragma unroll
            for (int x = 0; x < D / 32; ++x)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[u][x][i] *= al;
            m[u] = mn;
            float lts[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 4; ++i) four(s, i, without(mn), pk, lts);
            lt = (lts[0] + lts[1]) + (lts[2] + lts[3]);
        }
        l[u] += lt;
    };
    constexpr int NK = D / 16, NV = 2 * (D / 32);  // products of 32 x 32 scores, and of their part of the averages
    auto load_key = [&](frag (&kf)[NK], int stage, int kb, int c) __attribute__((always_inline)) {
        kf[c] = ld_frag<T>(sK + stage * ELEMS + kb * 32 * D + koff[c]);
    };
    auto load_keys = [&](frag (&kf)[NK], int stage, int kb) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < NK; ++c) load_key(kf, stage, kb, c);
    };
    auto load_value = [&](frag (&vf)[2][D / 32], int stage, int kb, int i) __attribute__((always_inline)) {
        const int t2 = i / (D / 32), x = i % (D / 32);
        const T* base = sV + stage * ELEMS + (kb * 32 + 16 * t2) * D + voff[x];
        const u32x2_t lo = lds_read_tr(base), hi = lds_read_tr(base + 8 * D);
        const u32x4_t v4 = {lo[0], lo[1], hi[0], hi[1]};
        vf[t2][x] = __builtin_bit_cast(frag, v4);
    };
    auto check_values = [&](const frag (&vf)[2][D / 32]) __attribute__((always_inline)) {
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2)
#pragma unroll
            for (int x = 0; x < D / 32; ++x) {
                const u32x4_t v4 = __builtin_bit_cast(u32x4_t, vf[t2][x]);
#pragma unroll
                for (int e = 0; e < 4; ++e) odd = paged_odd<T>(v4[e], odd);
            }
    };
    auto first_scores = [&](const float* bias) __attribute__((always_inline)) -> f32x16_t {
        f32x16_t init = zero16();
        if (BIAS && !SOFTCLAMP) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float4 bb = *reinterpret_cast<const float4*>(bias + 8 * g);
                init[4 * g] = bb.x;
                init[4 * g + 1] = bb.y;
                init[4 * g + 2] = bb.z;
                init[4 * g + 3] = bb.w;
            }
        }
        return init;
    };
    // Two blocks of 32 x 32 scores, of two blocks of rows (QB 2) or of positions: one's products run beside the other's
    // exponentials.  (A) scores of the first; (B) scores of the second, probabilities of the first; (C) averages of
    // the first, probabilities of the second; (D) averages of the second.  Each fragment is read from LDS when the one that it
    // follows in its registers has gone into a product: the next step's first keys (k0) in (D), with MORE.
    // (A) has no exponentials beside it, but the loads of the next pair of tiles (side), whose addresses are a good many scalar
    // instructions.
    auto step = [&](int stage, int kb, int j0, frag (&k0)[NK], auto MORE, auto side) __attribute__((always_inline)) {
        constexpr int R1 = QB - 1;  // the second one's rows ...
        const int kb1 = QB == 2 ? kb : 1, j1 = QB == 2 ? j0 : j0 + 32;  // ... and positions
        const float* const bias = &sBw[w][stage & 1][4 * hh];
        const bool edge = j0 + (QB == 2 ? 31 : 63) > all_see || j0 + (QB == 2 ? 32 : 64) > cnt;
        frag k1[QB == 2 ? 1 : NK];
        f32x16_t s0 = first_scores(bias + 32 * kb);
#pragma unroll
        for (int c = 0; c < NK; ++c) {
            s0 = M::run(k0[c], qf[0][c], s0);
            side(c);
        }
        if constexpr (QB == 1) {
            __builtin_amdgcn_sched_barrier(0);
            load_keys(k1, stage, 1);
        }
        f32x16_t s1 = first_scores(bias + 32 * kb1);
        clamp(s0, bias + 32 * kb);
        if (edge) {
            keep_branch();
            mask(s0, 0, j0);
        }
        begin_rows(s0, 0);
        __builtin_amdgcn_sched_barrier(0);
        Weights pk0, pk1;
        frag v0[2][D / 32], v1[QB == 2 ? 1 : 2][D / 32];
        static_assert(NK == NV, "a fragment of the values takes the place of one of the keys");
        float lt;
        {
            const float msub = without(m[0]);
            float lts[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < NK; ++i) {
                s1 = M::run(QB == 2 ? k0[i] : k1[QB == 2 ? 0 : i], qf[R1][i], s1);
                load_value(v0, stage, kb, i);
                if (i % (NK / 4) == 0) four(s0, i / (NK / 4), msub, pk0, lts);
                __builtin_amdgcn_sched_barrier(0);
            }
            lt = (lts[0] + lts[1]) + (lts[2] + lts[3]);
        }
        again(s0, 0, lt, pk0);
        clamp(s1, bias + 32 * kb1);
        if (edge) {
            keep_branch();
            check_values(v0);
            mask(s1, R1, j1);
        }
        begin_rows(s1, R1);
        __builtin_amdgcn_sched_barrier(0);
        {
            const float msub = without(m[R1]);
            float lts[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int t2 = i / (D / 32), x = i % (D / 32);
                o[0][x] = M::run(v0[t2][x], __builtin_bit_cast(frag, pk0.hi[t2]), o[0][x]);
                if constexpr (TWO) o[0][x] = M::run(v0[t2][x], __builtin_bit_cast(frag, pk0.lo[t2]), o[0][x]);
                if constexpr (QB == 1) load_value(v1, stage, 1, i);
                if (i % (NV / 4) == 0) four(s1, i / (NV / 4), msub, pk1, lts);
                __builtin_amdgcn_sched_barrier(0);
            }
            lt = (lts[0] + lts[1]) + (lts[2] + lts[3]);
        }
        again(s1, R1, lt, pk1);
        if constexpr (QB == 1) {
            if (edge) {
                keep_branch();
                check_values(v1);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int t2 = i / (D / 32), x = i % (D / 32);
            const frag v = QB == 2 ? v0[t2][x] : v1[QB == 2 ? 0 : t2][x];
            o[R1][x] = M::run(v, __builtin_bit_cast(frag, pk1.hi[t2]), o[R1][x]);
            if constexpr (TWO) o[R1][x] = M::run(v, __builtin_bit_cast(frag, pk1.lo[t2]), o[R1][x]);
            if constexpr (MORE) load_key(k0, QB == 2 && !kb ? stage : stage + 1, QB == 2 ? !kb : 0, i);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    // pairs of tiles, a barrier each: both have landed, and the pair before has been read
    int t = 0;
    auto pair = [&]() __attribute__((always_inline)) {
        wait_vmcnt<0>();
        lds_barrier();
        turn_page((t + 2) * BN);  // a pair's tiles lie in one block of 1024
    };
    for (; 2 * t < nact; t += 2) {
        pair();
        const int st = t & 3;
        const int j0 = t * BN, left = nact - 2 * t;  // 32-position steps of this pair, and further ones
        auto next = [&](int c) __attribute__((always_inline)) {
            constexpr int PER = NK / (2 * NL);  // products between two parts
            if (c % PER != PER - 1) return;
            const int n = c / PER % NL, u = c / (PER * NL);
            __builtin_amdgcn_sched_barrier(0);
            issue_part((t + 2 + u) * BN, (st ^ 2) + u, n);
            __builtin_amdgcn_sched_barrier(0);
        };
        auto none = [](int) __attribute__((always_inline)) {};
        if (BIAS)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int j = j0 + BN * k + lane;
                sBw[w][k][lane] = j < cnt ? sBraw[st + k][lane] * bmul : -INFINITY;
            }
        const std::true_type more;
        const std::false_type last;
        frag k0[NK];
        load_keys(k0, st, 0);
        step(st, 0, j0, k0, more, next);  // the keys of a step that there is not are read in vain
        if constexpr (QB == 1) {
            if (left > 2) step(st + 1, 0, j0 + 64, k0, last, none);
        } else {
            if (left > 1) step(st, 1, j0 + 32, k0, more, none);
            if (left > 2) step(st + 1, 0, j0 + 64, k0, more, none);
            if (left > 3) step(st + 1, 1, j0 + 96, k0, last, none);
        }
    }
    for (; t < ntl; t += 2) {  // the same barriers in every wave
        pair();
        issue((t + 2) * BN, (t & 3) ^ 2);
        issue((t + 3) * BN, ((t & 3) ^ 2) + 1);
    }
    wait_vmcnt<0>();  // the loads past the end

    const bool any = __any(odd != 0.f);
    flag(U.splits == 1 && any);
    if (U.splits > 1 && !paged_recorded(P, U)) return;
    const PagedRecords<false> R(P, U, hk);
#pragma unroll
    for (int u = 0; u < QB; ++u) {
        const int r = r0 + 32 * u + col;
        const float sum = xhalf_sum(l[u]);
        if (r >= rend) continue;
        if (U.splits > 1) {
            const int at = U.split * R.step + r - U.tile * P.tile;
            if (hh == 0) R.put_sum(at, m[u], any ? NAN : sum);
#pragma unroll
            for (int x = 0; x < D / 32; ++x)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int d = x * 32 + 8 * g + 4 * hh;
                    if (d < P.dim)
                        R.put(at, d, make_float4(o[u][x][4 * g], o[u][x][4 * g + 1], o[u][x][4 * g + 2], o[u][x][4 * g + 3]));
                }
            continue;
        }
        const PagedTo to = paged_to<T>(P, U, hk, r);
        if (hh == 0 && to.lse) *to.lse = (m[u] + log2f(sum)) * kLn2;
        if (!to.out) continue;
        const float inv = 1.f / sum;
#pragma unroll
        for (int x = 0; x < D / 32; ++x)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int d = x * 32 + 8 * g + 4 * hh;
                if (d < P.dim)
                    paged_store<T>(to, d, make_float4(o[u][x][4 * g] * inv, o[u][x][4 * g + 1] * inv, o[u][x][4 * g + 2] * inv,
                                                      o[u][x][4 * g + 3] * inv));
            }
    }
}

template <typename T, int D, bool SOFTCLAMP>
void launch_paged_tiles_d(const PagedDev& P, int64_t units, hipStream_t s) {
    const dim3 grid((unsigned)(units * P.kv_heads)), block(64 * paged_tile_waves(D));
    if (P.last) hipLaunchKernelGGL((k_paged_tiles<T, D, SOFTCLAMP, true, true>), grid, block, 0, s, P);
    else if (P.bias) hipLaunchKernelGGL((k_paged_tiles<T, D, SOFTCLAMP, true, false>), grid, block, 0, s, P);
    else hipLaunchKernelGGL((k_paged_tiles<T, D, SOFTCLAMP, false, false>), grid, block, 0, s, P);
}
template <typename T>
void launch_paged_tiles(const PagedDev& P, int64_t units, hipStream_t s) {
    if (P.dim <= 64) {
        if (P.softclamp > 0.f) launch_paged_tiles_d<T, 64, true>(P, units, s);
        else launch_paged_tiles_d<T, 64, false>(P, units, s);
    } else {
        if (P.softclamp > 0.f) launch_paged_tiles_d<T, 128, true>(P, units, s);
        else launch_paged_tiles_d<T, 128, false>(P, units, s);
    }
}

}  // namespace pa
