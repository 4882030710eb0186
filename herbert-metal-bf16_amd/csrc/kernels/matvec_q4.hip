// matvec_q4.hip -- y[m][n] = x[m][k] . W^T over weights of 4 bits in the
// layout of q4.hip, for up to 16 rows of x: a decode step's projections
// (ROWS 0), and the routed experts of a decode batch over moe_sort's tiles of
// up to 16 rows (ROWS 1: x rows gathered through the list, y in sorted order;
// 2: x in sorted order, y rows scattered through the list).
//
//   y[m][n] = sum over groups g of s[n][g] * (sum over k in g of (q - 8) x)
//
// The codes never become scaled weights: a bf16 of 16 + q is one and-or of a
// rotated word (two codes each), the MFMA sums (16 + q) x exactly in its
// products, and starts from the sum of -24 x, an MFMA with a constant operand
// that the row tiles of a wave share.  The group's scale then multiplies the
// f32 sum of 16 rows x 16 columns.  Sums are f32 throughout; Out rounds once.
// (The sums pass through 24 x and 31 x: an infinite x, or a group's sum of
// those past f32's range, gives NaN.)
//
// Bound by the codes' bytes: K N / 2 and 2 K N / GROUP for the scales.
// Measured against them at the 7.0 TB/s that a streaming read reaches (a
// launch's own 2.4 us in both): 2560 to 151936 in groups of 32 at 1 row 34.4
// us of 33.7, at 4 rows 36.8; 17408 to 5120 in groups of 128 at 1 row 11.3 of
// 9.0, at 16 rows 18.3; 4096 to 2560 at 1 row 3.5 of 3.2.  The case at 16 rows
// runs 160 workgroups of 32 W rows: 96 of the 256 CUs have none, and each of
// the others reads all of x (557 KB) for 287 KB of codes and scales.  16 W rows
// a wave (320 workgroups) take 28 us there, 64 (80 workgroups) 26.  K in four
// parts over four times the workgroups took 13.9 us before the 2.5 or more of a
// second launch that adds the parts: some 2 us less in all, for a workspace;
// not built.  A second stage of loads in registers changed nothing (the waves
// of a CU cover each other's latency).  Half of the VALU's issue is in use at
// 4 rows: 28 of some 60 instructions a tile make the codes bf16.
#include "hb_common.h"

constexpr u32 K = HB_K, N = HB_N, GROUP = HB_GROUP, OUT = HB_OUT, MV = HB_MV_M;
constexpr u32 KT = (K + 127) / 128, NT = (N + 15) / 16, TILES = KT * NT, GPT = 128 / GROUP, SPG = GROUP / 32;
constexpr u64 CODES = (u64)TILES * 1024, BLOB = CODES + (u64)((NT + 3) / 4) * KT * 128 * GPT;
constexpr u32 RT = HB_RT, SPLIT = HB_SPLIT, WAVES = HB_WAVES, U = HB_UNROLL, ROWS = HB_ROWS, TOPK = HB_TOPK;
constexpr bool SWI = OUT == 3;
constexpr u32 NOUT = SWI ? N / 2 : N;
constexpr u32 OT = SWI ? RT / 2 : RT;                    // output tiles of a wave
constexpr u32 ONT = SWI ? NT / 2 : NT;                   // output tiles
constexpr u32 NBLK = (ONT + OT - 1) / OT, GPW = WAVES / SPLIT;
constexpr u32 NWG = (NBLK + GPW - 1) / GPW;
// Every wave's tiles of K are whole rounds of U.
constexpr bool WHOLE = KT % (SPLIT * U) == 0;
static_assert(K % 8 == 0 && (!SWI || (RT % 2 == 0 && N % 32 == 0)), "shape");
static_assert(WAVES % SPLIT == 0 && MV >= 1 && MV <= 16, "waves");

#define HB_INLINE2 __attribute__((always_inline))
// At most 256 registers: the compiler then keeps the MFMAs' sums in VGPRs,
// where the scales multiply them, and not in AGPRs.
#define HB_VGPR_FORM __attribute__((amdgpu_waves_per_eu(2)))

typedef u32x4 chunk_t __attribute__((aligned(2)));

// The scales of a row's groups in a tile.
template <u32 groups>
struct Scales {
    typedef u16 type;
};
template <>
struct Scales<2> {
    typedef u32 type;
};
template <>
struct Scales<4> {
    typedef u32x2 type;
};
typedef Scales<GPT>::type scales_t;
HB_DEV float scale_of(u16 s, u32) { return bf16_to_f32(s); }
HB_DEV float scale_of(u32 s, u32 g) { return g ? bf16_hi(s) : bf16_lo(s); }
HB_DEV float scale_of(u32x2 s, u32 g) { return scale_of(g < 2 ? s.x : s.y, g & 1u); }

HB_DEV f32x4 mfma(u32x4 x, bf16x8 w, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), w, c, 0, 0, 0);
}

// A word's codes as bf16 16 + q, the MFMA's B operand.  `mask` and `base`
// are 0x00780078 and 0x41804180 in registers: an and-or takes no literal.
HB_DEV bf16x8 codes(u32 w, u32 mask, u32 base) {
    u32x4 a;
#pragma unroll
    for (u32 i = 0; i < 4; i++) a[i] = (__builtin_amdgcn_alignbit(w, w, 4 * i) & mask) | base;
    return __builtin_bit_cast(bf16x8, a);
}

// Out of the sum of y[row][n].
HB_DEV void store(void* yv, u64 row, u32 n, float v) {
    const u64 at = row * NOUT + n;
    if (OUT == 1) {
        ((float*)yv)[at] = v;
    } else {
        u16* y = (u16*)yv + at;
        *y = (u16)pack_bf16x2(OUT == 2 ? bf16_to_f32(*y) + v : v, 0.0f);
    }
}

// LDS bytes of a wave: its x tile, then its parts of the sums (rows_of_w).
template <u32 M>
struct Lds {
    static constexpr u32 REP = M <= 4 ? 4 : M <= 8 ? 2 : 1, TG = RT < REP ? RT : REP, C = 16 / TG;
    static constexpr u32 X = C * 256, P = SPLIT > 1 || SWI ? RT * M * 64 : 0, BYTES = X > P ? X : P;
};

// Workgroup `wg` of a matrix: `cols` <= M columns, column c from x row
// xrow(c) into y row yrow(c).
//
// The MFMA's 16 x rows hold C = 16 / TG of them TG times over, so that the
// quads of lanes all have the sums of a tile's 16 W rows and each quad keeps
// one of TG tiles: a set of TG tiles takes one load of scales and one
// register of sums for each of a lane's x rows.
template <u32 M, typename XRow, typename YRow>
HB_DEV void rows_of_w(const unsigned char* __restrict__ W, const u16* __restrict__ x, void* yv, unsigned char* lds, u32 wg,
                      u32 cols, XRow xrow, YRow yrow) {
    constexpr u32 TG = Lds<M>::TG, SETS = RT / TG, C = Lds<M>::C, AR = M < 4 ? M : 4;
    constexpr u32 XI = ((M < C ? M : C) + 3) / 4;  // loads of four x rows
    static_assert(RT % TG == 0 && M <= C, "tiles in whole sets");
    const u32 tid = threadIdx.x, lane = tid & 63u, col = lane & 15u, quad = lane >> 4;
    const u32 wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const u32 sp = wave % SPLIT, gi = wave / SPLIT;
    const u32 mine = quad * TG / 4;     // the lane's tile of a set
    const u32 row0 = (4 * quad) % C;    // its x rows: row0 .. + AR - 1
    // x comes in whole 256-byte lines of a row, four rows a load, and turns
    // into the MFMA's operand through a tile of the wave's own in LDS, its
    // 16-byte chunks at chunk ^ row, so that reads of one chunk of 16 rows
    // meet no bank twice.  (Loaded as the operand, 64 bytes of 16 rows at a
    // time, x took most of the time at 16 rows: 17408 to 5120 21 us.)
    // Columns past the rows repeat the last one and are never stored.
    u32x4* const xt = (u32x4*)(lds + wave * Lds<M>::BYTES);
    const u16* xp[XI];
#pragma unroll
    for (u32 i = 0; i < XI; i++) {
        const u32 c = 4 * i + quad;
        xp[i] = x + xrow(c < cols ? c : cols - 1) * K;
    }
    const u16* scales = (const u16*)(W + CODES);
    const u32 blk = wg * GPW + gi;
    // Tile r of the wave; past the last they repeat it and are never stored.
    auto tile = [&](u32 r) HB_INLINE2 -> u32 {
        const u32 o = blk * OT + r % OT;
        return (o < ONT ? o : ONT - 1) + (r / OT) * ONT;
    };
    u32 tn[RT];
    const scales_t* sn[SETS];
#pragma unroll
    for (u32 r = 0; r < RT; r++) tn[r] = tile(r) * KT;
#pragma unroll
    for (u32 g = 0; g < SETS; g++) {
        const u32 t = tile(g * TG + mine);
        sn[g] = (const scales_t*)scales + (u64)(t / 4) * KT * 64 + (t % 4) * 16 + col;
    }
    const u32 kt0 = sp * KT / SPLIT, kt1 = (sp + 1) * KT / SPLIT;
    const bf16x8 b24 = __builtin_bit_cast(bf16x8, u32x4{0xC1C0C1C0u, 0xC1C0C1C0u, 0xC1C0C1C0u, 0xC1C0C1C0u});
    u32 mask = 0x00780078u, one = 0x41804180u;
    asm("" : "+v"(mask), "+v"(one));
    float acc[SETS][AR];
#pragma unroll
    for (u32 g = 0; g < SETS; g++)
#pragma unroll
        for (u32 i = 0; i < AR; i++) acc[g][i] = 0.0f;

    // U tiles of K in flight as registers; past kt1 the last one's codes again
    // with zeros for x and the scales.
    auto inside = [&](u32 kt, u32 u) HB_INLINE2 { return WHOLE || u == 0 || kt + u < kt1; };
    struct Stage {
        u32x4 w[U][RT], x[U][XI];
        scales_t s[U][SETS];
    };
    auto load = [&](Stage& t, u32 kt) HB_INLINE2 {
#pragma unroll
        for (u32 u = 0; u < U; u++) {
            const u32 q = inside(kt, u) ? kt + u : kt1 - 1;
#pragma unroll
            for (u32 r = 0; r < RT; r++)
                t.w[u][r] = __builtin_nontemporal_load((const u32x4*)(W + (u64)(tn[r] + q) * 1024) + lane);
#pragma unroll
            for (u32 g = 0; g < SETS; g++) t.s[u][g] = sn[g][(u64)q * 64];
#pragma unroll
            for (u32 i = 0; i < XI; i++) {
                const u32 k = q * 128 + 8 * col;
                t.x[u][i] = *(const chunk_t*)(xp[i] + (K % 128 == 0 || k < K ? k : 0));
            }
        }
    };
    auto add = [&](const Stage& t, u32 kt) HB_INLINE2 {
#pragma unroll
        for (u32 u = 0; u < U; u++) {
            // The wave's own tile: its LDS accesses run in program order.
            const bool in = inside(kt, u), in_k = in && (K % 128 == 0 || (kt + u) * 128 + 8 * col < K);
            u32x4 xf[4];
#pragma unroll
            for (u32 i = 0; i < XI; i++) {
                const u32 c = 4 * i + quad;
                xt[c * 16 + (col ^ c)] = in_k ? t.x[u][i] : u32x4{0, 0, 0, 0};
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (u32 j = 0; j < 4; j++) {
                const u32 c = col % C < 4 * XI ? col % C : 0;
                xf[j] = xt[c * 16 + ((4 * j + quad) ^ c)];
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (u32 g = 0; g < GPT; g++) {
                f32x4 base = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (u32 j = g * SPG; j < (g + 1) * SPG; j++) base = mfma(xf[j], b24, base);
#pragma unroll
                for (u32 e = 0; e < SETS; e++) {
                    f32x4 c[TG];
#pragma unroll
                    for (u32 r = 0; r < TG; r++) {
                        c[r] = base;
#pragma unroll
                        for (u32 j = g * SPG; j < (g + 1) * SPG; j++)
                            c[r] = mfma(xf[j], codes(t.w[u][e * TG + r][j], mask, one), c[r]);
                    }
                    const float sc = in ? scale_of(t.s[u][e], g) : 0.0f;
#pragma unroll
                    for (u32 i = 0; i < AR; i++) {
                        float v = c[0][i];
#pragma unroll
                        for (u32 r = 1; r < TG; r++) v = mine == r ? c[r][i] : v;
                        acc[e][i] = __builtin_fmaf(sc, v, acc[e][i]);
                    }
                }
            }
        }
    };
    for (u32 kt = kt0; kt < kt1; kt += U) {
        Stage a;
        load(a, kt);
        add(a, kt);
    }

    // A lane holds W row `col` of tile `mine` of each set for x rows row0 ..
    auto put = [&](u32 r, u32 c, u32 nr, float v, float up) HB_INLINE2 {
        const u32 o = blk * OT + r, n = o * 16 + nr;
        if (o >= ONT || c >= cols || n >= NOUT) return;
        if (SWI) {
            float h;
            swiglu_n<1>(&v, &up, &h);
            v = h;
        }
        store(yv, yrow(c), n, v);
    };
    if constexpr (SPLIT == 1 && !SWI) {
#pragma unroll
        for (u32 g = 0; g < SETS; g++)
#pragma unroll
            for (u32 i = 0; i < AR; i++) put(g * TG + mine, row0 + i, col, acc[g][i], 0.0f);
    } else {
        // A split's parts, and the gate and up rows, meet in LDS; the parts
        // are added in wave order: [wave][tile][x row][W row].
        auto at = [&](u32 w, u32 r, u32 c) HB_INLINE2 -> float& { return ((float*)(lds + w * Lds<M>::BYTES))[r * M * 16 + c]; };
#pragma unroll
        for (u32 g = 0; g < SETS; g++)
#pragma unroll
            for (u32 i = 0; i < AR; i++)
                if (row0 + i < M) at(wave, g * TG + mine, (row0 + i) * 16 + col) = acc[g][i];
        __syncthreads();
        const u32 need = cols * 16;
        for (u32 it = sp * 64 + lane; it < OT * need; it += SPLIT * 64) {
            const u32 r = it / need, c = it % need;
            float v = at(gi * SPLIT, r, c), up = SWI ? at(gi * SPLIT, r + OT, c) : 0.0f;
#pragma unroll
            for (u32 q = 1; q < SPLIT; q++) {
                v += at(gi * SPLIT + q, r, c);
                if (SWI) up += at(gi * SPLIT + q, r + OT, c);
            }
            put(r, c / 16, c % 16, v, up);
        }
    }
}

#if HB_ROWS == 0
extern "C" __global__ __launch_bounds__(64 * WAVES) HB_VGPR_FORM void HB_NAME(const unsigned char* __restrict__ W,
                                                                                const u16* __restrict__ x, void* yv,
                                                                                u32 rows) {
    __shared__ u32x4 lds[WAVES * Lds<MV>::BYTES / 16];
    rows_of_w<MV>(W, x, yv, (unsigned char*)lds, blockIdx.x, rows < MV ? rows : MV, [](u32 c) -> u64 { return c; },
                  [](u32 c) -> u64 { return c; });
}
#else
extern "C" __global__ __launch_bounds__(64 * WAVES) HB_VGPR_FORM void HB_NAME(
    const u32* __restrict__ state, const unsigned char* __restrict__ W, const u16* __restrict__ x, void* yv,
    const u32* __restrict__ list, const u32* __restrict__ tiles, u32 m_launch) {
    constexpr u32 BYTES = Lds<4>::BYTES > Lds<MV>::BYTES ? Lds<4>::BYTES : Lds<MV>::BYTES;
    __shared__ u32x4 lds[WAVES * BYTES / 16];
    const u32 m = rows_of_state(state, m_launch), pairs = m * TOPK, t = blockIdx.x / NWG;
    if (t >= tiles[0]) return;
    const u32 expert = tiles[1 + 3 * t], first = tiles[2 + 3 * t];
    u32 cols = tiles[3 + 3 * t];
    if (expert >= HB_E || first >= pairs) return;
    cols = cols < MV ? cols : MV;
    cols = cols < pairs - first ? cols : pairs - first;
    if (cols == 0) return;
    auto xrow = [&](u32 c) -> u64 {
        if (ROWS != 1) return first + c;
        const u32 r = list[first + c] / TOPK;
        return r < m ? r : m - 1;
    };
    auto yrow = [&](u32 c) -> u64 {
        if (ROWS == 1) return first + c;
        const u32 r = list[first + c];
        return r < pairs ? r : pairs - 1;
    };
    // Most tiles of a decode batch have few rows.
    if (cols <= 4)
        rows_of_w<4>(W + expert * BLOB, x, yv, (unsigned char*)lds, blockIdx.x % NWG, cols, xrow, yrow);
    else
        rows_of_w<MV>(W + expert * BLOB, x, yv, (unsigned char*)lds, blockIdx.x % NWG, cols, xrow, yrow);
}
#endif
