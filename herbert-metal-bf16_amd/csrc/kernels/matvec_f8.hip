// matvec_f8.hip -- y[m][n] = x[m][k] . W^T over an 8-bit matrix (f8.h) for up
// to 16 rows of bf16 x, quantised as they are loaded: a decode step's
// projections (ROWS 0), and the routed experts of a decode batch over
// moe_sort's tiles of up to 16 rows (ROWS 1: x rows gathered through the list,
// y in sorted order; 2: x in sorted order, y rows scattered through the list).
//
//   y[m][n] = sum over blocks b of 128 K of sx[m][b] sw[n / 128][b] *
//             (sum over k in b of qx qw)
//
// A block of 16 x rows by 16 W rows is one v_mfma_f32_16x16x128_f8f6f4, whose
// f32 sums the two scales multiply: x is its first operand, so that a lane has
// one W row's sums for four x rows.  How the MFMA orders K does not matter as
// long as both operands have it alike: a lane takes the 16-byte chunks q and
// q + 4 of its row's 128, q its quad of lanes, so that a load instruction
// reads 64 bytes of 16 rows and a pair of them whole lines.
//
// x comes in whole 256-byte lines, four rows a load; the 16 lanes of a row
// find its block's scale and codes, which turn into the operand through a tile
// of the wave's own in LDS, 16-byte chunks at chunk ^ row.
#include "f8.h"

constexpr u32 K = HB_K, N = HB_N, OUT = HB_OUT, MV = HB_MV_M;
constexpr u32 KT = f8_blocks(K), NT = (N + 15) / 16;
constexpr u64 MATRIX = f8_matrix_bytes(K, N);
constexpr u32 RT = HB_RT, SPLIT = HB_SPLIT, WAVES = HB_WAVES, U = HB_UNROLL, ROWS = HB_ROWS, TOPK = HB_TOPK;
constexpr bool SWI = OUT == 3;
constexpr u32 NOUT = SWI ? N / 2 : N;
constexpr u32 OT = SWI ? RT / 2 : RT;                    // output tiles of a wave
constexpr u32 ONT = SWI ? NT / 2 : NT;                   // output tiles
constexpr u32 NBLK = (ONT + OT - 1) / OT, GPW = WAVES / SPLIT;
constexpr u32 NWG = (NBLK + GPW - 1) / GPW;
constexpr u32 SC = SWI ? 2 : 1;                          // W scales of a wave's K tile
// Every wave's tiles of K are whole rounds of U.
constexpr bool WHOLE = KT % (SPLIT * U) == 0;
static_assert(K % 16 == 0 && (!SWI || (RT % 2 == 0 && N % 256 == 0)) && (RT & (RT - 1)) == 0 && RT <= 8, "shape");
static_assert(WAVES % SPLIT == 0 && MV >= 1 && MV <= 16, "waves");

#define HB_INLINE2 __attribute__((always_inline))
// At most 256 registers: the compiler then keeps the MFMAs' sums in VGPRs,
// where the scales multiply them, and not in AGPRs.
#define HB_VGPR_FORM __attribute__((amdgpu_waves_per_eu(2)))

typedef u32x4 chunk_t __attribute__((aligned(2)));

HB_DEV i32x8 operand(u32x4 a, u32x4 b) {
    return i32x8{(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w};
}
// No scale operands: the plain product.
HB_DEV f32x4 mfma(i32x8 x, i32x8 w) { return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, w, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0); }

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

// LDS bytes of a wave: its x tile (codes of XI * 4 rows, 16 scales), then its
// parts of the sums.
template <u32 M>
struct Lds {
    static constexpr u32 XI = (M + 3) / 4;
    static constexpr u32 X = XI * 512 + 64, P = SPLIT > 1 || SWI ? RT * M * 64 : 0, BYTES = X > P ? X : P;
};

// Workgroup `wg` of a matrix: `cols` <= M columns, column c from x row
// xrow(c) into y row yrow(c).
template <u32 M, typename XRow, typename YRow>
HB_DEV void rows_of_w(const unsigned char* __restrict__ W, const u16* __restrict__ x, void* yv, unsigned char* lds, u32 wg,
                      u32 cols, XRow xrow, YRow yrow) {
    constexpr u32 XI = Lds<M>::XI, AR = M < 4 ? M : 4;
    const u32 tid = threadIdx.x, lane = tid & 63u, col = lane & 15u, quad = lane >> 4;
    const u32 wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const u32 sp = wave % SPLIT, gi = wave / SPLIT;
    u32x4* const xt = (u32x4*)(lds + wave * Lds<M>::BYTES);
    float* const xs = (float*)(xt + XI * 32);
    // Columns past the rows repeat the last one and are never stored.
    const u16* xp[XI];
#pragma unroll
    for (u32 i = 0; i < XI; i++) {
        const u32 c = 4 * i + quad;
        xp[i] = x + xrow(c < cols ? c : cols - 1) * K;
    }
    const u32 blk = wg * GPW + gi;
    // Tile r of the wave; past the last they repeat it and are never stored.
    auto tile = [&](u32 r) HB_INLINE2 -> u32 {
        const u32 o = blk * OT + r % OT;
        return (o < ONT ? o : ONT - 1) + (r / OT) * ONT;
    };
    const unsigned char* wp[RT];
#pragma unroll
    for (u32 r = 0; r < RT; r++) {
        const u32 n = tile(r) * 16 + col;
        wp[r] = W + (u64)(n < N ? n : N - 1) * K + 16 * quad;
    }
    // A wave's tiles lie within one block of 128 rows (two with gate and up).
    const float* sp_w[SC];
#pragma unroll
    for (u32 c = 0; c < SC; c++) sp_w[c] = (const float*)(W + (u64)N * K) + (u64)(tile(c * OT) / 8) * KT;
    const u32 kt0 = sp * KT / SPLIT, kt1 = (sp + 1) * KT / SPLIT;
    float acc[RT][AR];
#pragma unroll
    for (u32 r = 0; r < RT; r++)
#pragma unroll
        for (u32 i = 0; i < AR; i++) acc[r][i] = 0.0f;

    // U tiles of K in flight as registers; past kt1 the last one again, not
    // added.
    auto inside = [&](u32 kt, u32 u) HB_INLINE2 { return WHOLE || u == 0 || kt + u < kt1; };
    struct Stage {
        u32x4 w[U][RT][2], x[U][XI];
        float s[U][SC];
    };
    auto load = [&](Stage& t, u32 kt) HB_INLINE2 {
#pragma unroll
        for (u32 u = 0; u < U; u++) {
            const u32 q = inside(kt, u) ? kt + u : kt1 - 1;
#pragma unroll
            for (u32 r = 0; r < RT; r++)
#pragma unroll
                for (u32 h = 0; h < 2; h++) {
                    const bool in = K % 128 == 0 || q * 128 + h * 64 + 16 * quad < K;
                    t.w[u][r][h] = __builtin_nontemporal_load((const u32x4*)(in ? wp[r] + q * 128 + h * 64 : wp[r]));
                    if (!in) t.w[u][r][h] = u32x4{0, 0, 0, 0};
                }
#pragma unroll
            for (u32 c = 0; c < SC; c++) t.s[u][c] = sp_w[c][q];
#pragma unroll
            for (u32 i = 0; i < XI; i++) {
                const u32 k = q * 128 + 8 * col;
                const bool in = K % 128 == 0 || k < K;
                t.x[u][i] = *(const chunk_t*)(xp[i] + (in ? k : 0));
                if (!in) t.x[u][i] = u32x4{0, 0, 0, 0};
            }
        }
    };
    auto add = [&](const Stage& t, u32 kt) HB_INLINE2 {
#pragma unroll
        for (u32 u = 0; u < U; u++) {
            // The wave's own tile: its LDS accesses run in program order.
#pragma unroll
            for (u32 i = 0; i < XI; i++) {
                const u32 c = 4 * i + quad;
                const F8Scale s = f8_scale(f8_max_lanes(f8_max8(t.x[u][i])));
                ((u32x2*)xt)[c * 16 + ((col / 2) ^ (c & 7u)) * 2 + col % 2] = f8_codes8(t.x[u][i], s.inv);
                if (col == 0) xs[c] = s.s;
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            const u32 c = col < 4 * XI ? col : 0;
            const i32x8 xf = operand(xt[c * 8 + (quad ^ (c & 7u))], xt[c * 8 + ((quad + 4) ^ (c & 7u))]);
            const f32x4 sx = *(const f32x4*)(xs + (quad < XI ? 4 * quad : 0));
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            float sc[SC][AR];
#pragma unroll
            for (u32 j = 0; j < SC; j++)
#pragma unroll
                for (u32 i = 0; i < AR; i++) sc[j][i] = sx[i] * t.s[u][j];
#pragma unroll
            for (u32 r = 0; r < RT; r++) {
                const f32x4 v = mfma(xf, operand(t.w[u][r][0], t.w[u][r][1]));
#pragma unroll
                for (u32 i = 0; i < AR; i++) {
                    const float sum = __builtin_fmaf(sc[r / OT][i], v[i], acc[r][i]);
                    acc[r][i] = inside(kt, u) ? sum : acc[r][i];
                }
            }
        }
    };
    for (u32 kt = kt0; kt < kt1; kt += U) {
        Stage a;
        load(a, kt);
        add(a, kt);
    }

    // A lane holds W row `col` of each tile for x rows 4 quad ..
    auto put = [&](u32 r, u32 c, u32 nr, float v, float up) HB_INLINE2 {
        const u32 o = blk * OT + r, n = o * 16 + nr;
        if (o >= ONT || c >= cols || n >= NOUT) return;
        if (SWI) v = f8_swiglu(v, up);
        store(yv, yrow(c), n, v);
    };
    if constexpr (SPLIT == 1 && !SWI) {
#pragma unroll
        for (u32 r = 0; r < RT; r++)
#pragma unroll
            for (u32 i = 0; i < AR; i++) put(r, 4 * quad + i, col, acc[r][i], 0.0f);
    } else {
        // A split's parts, and the gate and up rows, meet in LDS; the parts
        // are added in wave order: [wave][tile][x row][W row].
        auto at = [&](u32 w, u32 r, u32 c) HB_INLINE2 -> float& { return ((float*)(lds + w * Lds<M>::BYTES))[r * M * 16 + c]; };
#pragma unroll
        for (u32 r = 0; r < RT; r++)
#pragma unroll
            for (u32 i = 0; i < AR; i++)
                if (4 * quad + i < M) at(wave, r, (4 * quad + i) * 16 + col) = acc[r][i];
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
        rows_of_w<4>(W + expert * MATRIX, x, yv, (unsigned char*)lds, blockIdx.x % NWG, cols, xrow, yrow);
    else
        rows_of_w<MV>(W + expert * MATRIX, x, yv, (unsigned char*)lds, blockIdx.x % NWG, cols, xrow, yrow);
}
#endif
