// matvec_f8.hip -- y[m][n] = x[m][k] . W^T over an 8-bit matrix (f8.h) for up
// to 16 rows of bf16 x, quantised as they are loaded: a decode step's
// projections (ROWS 0), and the routed experts of a decode batch over
// moe_sort's tiles of up to 16 rows (ROWS 1: x rows gathered through the list,
// y in sorted order; 2: x in sorted order, y rows scattered through the list).
//
//   y[m][n] = sum over blocks b of 128 K of sx[m][b] sw[n / 128][b] *
//             (sum over k in b of qx qw)
//
// A block of 16 x rows by 16 W rows is four v_mfma_f32_16x16x32_bf16 of the codes
// as bf16 (f8.h: sums in f32, and the loads of W still bound the kernel), whose
// sums the two scales multiply: x is the first operand, so that a lane has one W
// row's sums for four x rows.  How the MFMA orders K does not matter as long as
// both operands have it alike: a lane takes the 16-byte chunks q and q + 4 of
// its row's 128, q its quad of lanes.
//
// Each wave loads its own W rows and x rows straight into LDS
// (buffer_load_dwordx4 ... lds), HB_UNROLL tiles of 128 K ahead, with no barrier
// in its loop: whole lines of 8 W rows and of 4 x rows a load.  (W loaded as the
// operand, 64 bytes of 16 rows at a time, reached 4.4 TB/s; now 2560 to 151936
// at 4 rows 64 us, 6.1 TB/s, and a short matrix its launch, 4096 to 2560 4.7.)  The 16 lanes of an
// x row find its block's scale and codes, which go back to LDS as the operand;
// chunks stand at chunk ^ row there, and W's at chunk ^ row >> 1.
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
static_assert(K % 16 == 0 && (!SWI || (RT % 2 == 0 && N % 256 == 0)) && (RT & (RT - 1)) == 0 && RT <= 8, "shape");
static_assert(WAVES % SPLIT == 0 && MV >= 1 && MV <= 16, "waves");

#define HB_INLINE2 __attribute__((always_inline))
// At most 256 registers: the compiler then keeps the MFMAs' sums in VGPRs,
// where the scales multiply them, and not in AGPRs.
#define HB_VGPR_FORM __attribute__((amdgpu_waves_per_eu(2)))
// A wave's loads but the last n landed, its LDS accesses done.
#define WAIT_LOADS(n) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(n) : "memory")
#define WAIT_LDS() asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory")

HB_DEV i32x8 operand(u32x4 a, u32x4 b) {
    return i32x8{(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w};
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

// A DPP control: quad_perm [i, i, i, i].
template <int ctrl>
struct Perm {
    static constexpr int value = ctrl;
};

// LDS bytes of a wave: U stages of its W and x tiles, the codes of its x tile
// and their scales, then in the same place its parts of the sums.
template <u32 M>
struct Lds {
    static constexpr u32 XI = (M + 3) / 4, STAGE = RT * 2048 + XI * 1024, X = U * STAGE + XI * 512 + 64;
    static constexpr u32 P = SPLIT > 1 || SWI ? RT * M * 64 : 0, BYTES = X > P ? X : P;
};

// Workgroup `wg` of a matrix: `cols` <= M columns, column c from x row
// xrow(c) into y row yrow(c).
template <u32 M, typename XRow, typename YRow>
HB_DEV void rows_of_w(const unsigned char* __restrict__ W, const u16* __restrict__ x, void* yv, unsigned char* lds, u32 wg,
                      u32 cols, XRow xrow, YRow yrow) {
    constexpr u32 XI = Lds<M>::XI, AR = M < 4 ? M : 4, STAGE = Lds<M>::STAGE, NL = RT * 2 + XI;
    const u32 tid = threadIdx.x, lane = tid & 63u, col = lane & 15u, quad = lane >> 4;
    const u32 wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const u32 sp = wave % SPLIT, gi = wave / SPLIT;
    unsigned char* const mine = lds + wave * Lds<M>::BYTES;
    u32x4* const xt = (u32x4*)(mine + U * STAGE);
    float* const xs = (float*)(xt + XI * 32);
    const u32 blk = wg * GPW + gi;
    const u32 tile0 = blk * OT < ONT ? blk * OT : ONT - 1;  // the wave's first output tile
    // A block's rows: past the matrix's end a load gives zeros without a memory
    // access, as do a short last tile's chunks past K (both at `AWAY`).
    constexpr u32 AWAY = 0x80000000u;
    __amdgpu_buffer_rsrc_t rw[SC];
#pragma unroll
    for (u32 c = 0; c < SC; c++) {
        const u64 row = tile0 * 16 + (u64)c * NOUT, left = ((u64)N - row) * K;
        rw[c] = __builtin_amdgcn_make_buffer_rsrc((void*)(W + row * K), (short)0, (int)(left < 0x7fffffffu ? left : 0x7fffffffu), 0x00020000);
    }
    const __amdgpu_buffer_rsrc_t rx = __builtin_amdgcn_make_buffer_rsrc((void*)x, (short)0, 0x7fffffff, 0x00020000);
    const u32 wr = lane / 8, wc = lane % 8 ^ (wr >> 1);  // of a load's 8 rows; an odd load's chunk is wc ^ 4
    const u32 woff = wr * K;
    // Columns past the rows repeat the last one and are never stored.
    u32 xoff[XI];
#pragma unroll
    for (u32 i = 0; i < XI; i++) {
        const u32 c = 4 * i + quad;
        xoff[i] = (u32)xrow(c < cols ? c : cols - 1) * (K * 2) + col * 16;
    }
    // A wave's tiles lie within one block of 128 rows (two with gate and up).
    const float* sp_w[SC];
#pragma unroll
    for (u32 c = 0; c < SC; c++) sp_w[c] = (const float*)(W + (u64)N * K) + (u64)((tile0 + c * ONT) / 8) * KT;
    const u32 kt0 = sp * KT / SPLIT, kt1 = (sp + 1) * KT / SPLIT;
    float acc[RT][AR];
#pragma unroll
    for (u32 r = 0; r < RT; r++)
#pragma unroll
        for (u32 i = 0; i < AR; i++) acc[r][i] = 0.0f;

    typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
    // Loads of K tile kt into stage st: past kt1 of nothing, so that every
    // round has as many.
    auto load = [&](u32 kt, u32 st) HB_INLINE2 {
        const u32 at = (u32)(u64)(lds_u32x4*)(mine + st * STAGE);
        const bool in = kt < kt1;
#pragma unroll
        for (u32 q = 0; q < RT * 2; q++) {
            const u32 r = q / 2, chunk = q & 1u ? wc ^ 4u : wc;
            u32 off = woff + chunk * 16 + ((r % OT) * 16 + (q & 1u) * 8) * K;
            if (!in || (K % 128 != 0 && kt == KT - 1 && chunk * 16 >= K % 128)) off = AWAY;
            asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, %3 offen nt lds"
                         :: "s"(at + q * 1024), "v"(off), "s"(rw[r / OT]), "s"(in ? kt * 128 : 0) : "memory");
        }
#pragma unroll
        for (u32 i = 0; i < XI; i++) {
            u32 off = xoff[i];
            if (!in || (K % 128 != 0 && kt == KT - 1 && col * 8 >= K % 128)) off = AWAY;
            asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                         :: "s"(at + RT * 2048 + i * 1024), "v"(off), "s"(rx), "s"(in ? kt * 256 : 0) : "memory");
        }
    };
#pragma unroll
    for (u32 u = 0; u < U; u++) load(kt0 + u, u);
    u32 st = 0;
    for (u32 kt = kt0; kt < kt1; kt++) {
        float sw[SC];
#pragma unroll
        for (u32 c = 0; c < SC; c++) sw[c] = sp_w[c][kt];
        WAIT_LOADS((U - 1) * NL);
        const u32x4* sW = (const u32x4*)(mine + st * STAGE);
        const u32x4* sX = sW + RT * 128;
        i32x8 wf[RT];
        u32x4 xv[XI];
#pragma unroll
        for (u32 r = 0; r < RT; r++)
            wf[r] = operand(sW[r * 128 + col * 8 + (quad ^ (col >> 1))], sW[r * 128 + col * 8 + ((quad + 4) ^ (col >> 1))]);
#pragma unroll
        for (u32 i = 0; i < XI; i++) xv[i] = sX[i * 64 + lane];
        // Read: the stage is free.
        WAIT_LDS();
        load(kt + U, st);
        st = st + 1 == U ? 0 : st + 1;
        // The wave's own tile: its LDS accesses run in program order.
        // One division for all loads: lane col of a row of lanes has the group
        // of load col % 4, and the quads of lanes hand the reciprocals round.
        u32 top = 0;
#pragma unroll
        for (u32 i = 0; i < XI; i++) {
            const u32 t = f8_max_lanes(f8_max8(xv[i]));
            top = i == 0 || col % 4 == i ? t : top;
        }
        const F8Scale s = f8_scale(top);
        if (col < XI) xs[4 * col + quad] = s.s;
        auto codes = [&](u32 i, auto perm) HB_INLINE2 {
            const u32 c = 4 * i + quad;
            const float inv = XI == 1 ? s.inv
                                      : __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, s.inv),
                                                                                              decltype(perm)::value, 0xf, 0xf, true));
            ((u32x2*)xt)[c * 16 + ((col / 2) ^ (c & 7u)) * 2 + col % 2] = f8_codes8(xv[i], inv);
        };
        codes(0, Perm<0x00>{});
        if constexpr (XI > 1) codes(1, Perm<0x55>{});
        if constexpr (XI > 2) codes(2, Perm<0xAA>{});
        if constexpr (XI > 3) codes(3, Perm<0xFF>{});
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        const u32 c = col < 4 * XI ? col : 0;
        const F8Wide xf = f8_wide(operand(xt[c * 8 + (quad ^ (c & 7u))], xt[c * 8 + ((quad + 4) ^ (c & 7u))]));
        const f32x4 sx = *(const f32x4*)(xs + (quad < XI ? 4 * quad : 0));
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        float sc[SC][AR];
#pragma unroll
        for (u32 j = 0; j < SC; j++)
#pragma unroll
            for (u32 i = 0; i < AR; i++) sc[j][i] = sx[i] * sw[j];
#pragma unroll
        for (u32 r = 0; r < RT; r++) {
            const f32x4 v = f8_product(xf, f8_wide(wf[r]));
#pragma unroll
            for (u32 i = 0; i < AR; i++) acc[r][i] = __builtin_fmaf(sc[r / OT][i], v[i], acc[r][i]);
        }
    }
    WAIT_LOADS(0);  // before the parts take the stages' place

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
