// gemm_f8.hip -- Y[m][n] = X[m][k] . W^T of 8-bit operands (f8.h): X f8 rows,
// W an f8 matrix, f32 sums, one rounding at the output as Out says; dense rows
// (ROWS 0), and the routed experts over moe_sort's tiles of BM rows (1: X rows
// gathered through the list, Y in sorted order; 2: X in sorted order, Y rows
// scattered through the list).
//
//   Y[m][n] = sum over blocks b of 128 K of sx[m][b] sw[n / 128][b] *
//             (sum over k in b of qx qw)
//
// A block's products of 16 W rows and 16 X rows are one
// v_mfma_f32_16x16x128_f8f6f4 from zero.  W is its first operand, so that a
// lane has four columns n of one row m: the row's scale is the lane's, W's is
// one for all of the fragment, and their product adds the four sums to the
// accumulators with an fma each, 16 cycles of VALU beside the MFMA's 32.  Its
// sums come out some 2^-16 off, little beside the half step of 2^-8 of a bf16
// output; an f32 output, and any that the caller asks f32 sums for, takes the
// bf16 products of f8.h in its place (HB_WIDE), at half the rate.
//
// X and W tiles of 128 K go straight into LDS (buffer_load_dwordx4 ... lds)
// through HB_STAGES stages, 16-byte chunks XORed by row >> 1 so that the
// fragments' reads meet no bank twice; a lane takes the chunks q and q + 4 of
// its row, q its quad (both operands alike, so the order of K within the MFMA
// does not matter).  X's scales of eight K tiles at a time go the same way into
// one of two places, 32 bytes a row; W's, all of a tile's blocks, are read once.
//
// 8192 x 34816 x 5120: 1260 us in the mean of 40 launches, 1180 to 1210 at the
// least, 2.32 to 2.47 PFLOP/s (the library's product under one scale for all 1059);
// the MFMAs are busy for 60% of it, the scales' fmas and the barrier a K tile hold
// the rest; with f32 sums 2470.  509 x 7001 x 5008 in f32 by bf16 products: 47 us
// with x quantised, one tile on each of 220 CUs, and each wave converts its own
// fragments (96 for 32 products a K tile and wave): W's by the four waves that
// share them, X's by two.
//
// Out::Swiglu: W holds [gate (N / 2) | up (N / 2)] rows; a tile covers 128
// features, a wave's first fragments their gate rows and its others the up
// rows, so a lane has both sums of a feature.  h = rne(g * sigmoid(g) * u) in
// bf16 and at once quantised: the 128 features are one group of an f8 row,
// whose largest is met over the waves in LDS.
//
// Constants: HB_K, HB_N (W rows), HB_OUT (0 bf16, 1 f32, 2 residual, 3
// SwiGLU), HB_ROWS, HB_TOPK, HB_E, HB_TILES (what the table holds), HB_BM,
// HB_BN, HB_WM, HB_WN, HB_STAGES, HB_BAND, HB_KSPLIT, HB_WIDE.  Bindings: state,
// W, X, Y, list, tiles; then the rows the launch was sized for.
#include "f8.h"

constexpr u32 K = HB_K, N = HB_N;
constexpr int OUT = HB_OUT, ROWS = HB_ROWS;
constexpr u32 TOPK = HB_TOPK, BM = HB_BM, BN = HB_BN, WM = HB_WM, WN = HB_WN;
constexpr u32 NWV = WM * WN, NTH = 64 * NWV, NS = HB_STAGES, KSP = HB_KSPLIT;
constexpr u32 FM = 16, FR = 4;                           // a block of FM x FM: sums a lane
constexpr u32 TM = BM / WM, TN = BN / WN, IM = TM / FM, IN = TN / FM;
constexpr bool SWI = OUT == 3;
constexpr u32 KB = f8_blocks(K), KBP = (KB + 63) / 64 * 64, NB = f8_blocks(N), NOUT = SWI ? N / 2 : N, BF = SWI ? BN / 2 : BN;
constexpr u32 NTILES = (NOUT + BF - 1) / BF;
constexpr u64 XROW = f8_row_bytes(K), HROW = f8_row_bytes(NOUT), MATRIX = f8_matrix_bytes(K, N);
constexpr u32 XST = BM * 8, WST = BN * 8;                 // 16-byte chunks of a stage
constexpr u32 NXL = XST / 64, NWL = WST / 64;             // wave loads of a stage
constexpr u32 XLMAX = (NXL + NWV - 1) / NWV, WLMAX = (NWL + NWV - 1) / NWV;
constexpr u32 LMIN = NXL / NWV + NWL / NWV;               // loads a stage of every wave
constexpr u32 NSL = BM / 32, SLMAX = (NSL + NWV - 1) / NWV;  // wave loads of eight K tiles' X scales
constexpr u32 SWR = SWI ? 2 : BN % 128 == 0 ? BN / 128 : (BN + 127) / 128 + (128 % BN != 0);  // W's blocks of a tile
constexpr u32 LDS = NS * (XST + WST) + BM * 4 + SWR * KBP / 4;  // 16-byte chunks: stages, scales
// Outputs of two bytes whose rows are whole chunks leave through LDS, a row
// (and a chunk between them, so that the rows' banks differ) at EPIROW bytes.
constexpr u32 EPIROW = BN * 2 + 16;
constexpr bool EPI_LDS = OUT == 0 && NOUT % 8 == 0 && BM * EPIROW <= 160 * 1024;
constexpr u32 EPI = EPI_LDS ? BM * EPIROW / 16 : 0;
constexpr u32 LROWS = NWV * 8;                            // rows between a wave's loads
#ifndef HB_SCHED
#define HB_SCHED 0
#endif
constexpr bool AHEAD = HB_SCHED == 1;
#ifndef HB_WIDE
#define HB_WIDE 0
#endif
// The W row of a tile's row r, from the tile's first column on: a wave's gate
// rows stand before the up rows of the same features.
constexpr u32 w_row(u32 r) {
    return SWI ? (r % TN >= TN / 2 ? NOUT : 0) + r / TN * (TN / 2) + r % TN % (TN / 2) : r;
}
// Its rows LROWS apart lie as far from each other wherever they start.
static_assert(!SWI || LROWS % TN == 0 || (TN / 2) % LROWS == 0, "SwiGLU rows of a wave's loads");
static_assert(LROWS % 16 == 0, "the rows of a wave's loads share their swizzle");
static_assert((NS - 2) * LMIN < 64, "vmcnt");
static_assert(!AHEAD || (NS == 2 && IN >= 4), "fragments ahead: two stages, four fragments of W a wave");
static_assert(K % 16 == 0 && BM % 32 == 0 && BN % 16 == 0 && TM % FM == 0 && TN % FM == 0, "tile");
static_assert(!SWI || (BN == 256 && IN % 2 == 0 && N % 256 == 0 && KSP == 1 && ROWS != 2), "SwiGLU");
static_assert(KSP == 1 || (OUT == 1 && ROWS == 0), "split K: f32 partial sums");
static_assert(NS >= 2 && NS <= 4, "stages");

#define HB_INLINE __attribute__((always_inline))
#define WAIT_VM(n) __builtin_amdgcn_s_waitcnt((((n) & 15) | (((n) >> 4) << 14) | (7 << 4) | (15 << 8)))
// This wave's LDS accesses done, then the workgroup barrier; not
// __syncthreads(), which would also wait for the stages in flight.
#define STAGE_BARRIER() asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory")

// Four columns n .. n + 3 of row `yrow`.
HB_DEV void store4(void* Yv, u64 yrow, u32 n, f32x4 v) {
    typedef f32x4 loose4 __attribute__((aligned(4)));
    typedef u32x2 loose2 __attribute__((aligned(2)));
    const u64 at = yrow * NOUT + n;
    if (N % 4 == 0 || n + 4 <= NOUT) {
        if constexpr (OUT == 1) {
            *(loose4*)((float*)Yv + at) = v;
        } else {
            loose2* p = (loose2*)((u16*)Yv + at);
            if constexpr (OUT == 2) {
                const u32x2 o = *p;
                v += f32x4{bf16_lo(o.x), bf16_hi(o.x), bf16_lo(o.y), bf16_hi(o.y)};
            }
            *p = u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
        }
        return;
    }
#pragma unroll
    for (u32 e = 0; e < 4; e++) {
        if (n + e >= NOUT) return;
        if constexpr (OUT == 1) {
            ((float*)Yv)[at + e] = v[e];
        } else {
            u16* p = (u16*)Yv + at + e;
            *p = (u16)pack_bf16x2(OUT == 2 ? bf16_to_f32(*p) + v[e] : v[e], 0.0f);
        }
    }
}

extern "C" __global__ __launch_bounds__(NTH) void HB_NAME(const u32* __restrict__ state, const unsigned char* __restrict__ W,
                                                            const unsigned char* __restrict__ X, void* __restrict__ Yv,
                                                            const u32* __restrict__ list, const u32* __restrict__ tiles,
                                                            u32 m_launch) {
    __shared__ u32x4 lds[LDS > EPI ? LDS : EPI];
    u32x4* const sXa = lds;
    u32x4* const sWa = lds + NS * XST;
    u32x4* const sscale = sWa + NS * WST;                // X's scales: [place][row][K tile of eight]
    float* const wscale = (float*)(sscale + 2 * BM * 2);
    const u32 tid = threadIdx.x, lane = tid & 63u;
    const u32 wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const u32 wm = wave % WM, wn = wave / WM;

    // The tile: its first row (dense row or sorted pair), its rows, its
    // column tile, its expert.
    u32 g = blockIdx.x, row0, rows, gn, expert = 0;
    const u32 m = rows_of_state(state, m_launch), pairs = m * TOPK;
    const u32 part = KSP > 1 ? g % KSP : 0;
    if constexpr (KSP > 1) g /= KSP;
    if constexpr (ROWS == 0) {
        // Each XCD takes a contiguous range of tiles: bands of HB_BAND row
        // tiles, each walked over every column tile.
        g = xcd_remap(g, gridDim.x / KSP);
        const u32 mb = (m + BM - 1) / BM;
        constexpr u32 PER = HB_BAND * NTILES;
        const u32 full = mb / HB_BAND;
        u32 gm;
        if (g < full * PER) {
            const u32 idx = g % PER;
            gm = (g / PER) * HB_BAND + idx % HB_BAND;
            gn = idx / HB_BAND;
        } else {
            const u32 rem = mb - full * HB_BAND, idx = g - full * PER;
            if (rem == 0) return;
            gm = full * HB_BAND + idx % rem;
            gn = idx / rem;
        }
        if (gm >= mb || gn >= NTILES) return;
        row0 = gm * BM;
        rows = m - row0 < BM ? m - row0 : BM;
    } else {
        // The table's tiles alone, no more than it has room for and the launch
        // has workgroups, each XCD a contiguous range of them.
        u32 held = tiles[0];
        held = held < HB_TILES ? held : HB_TILES;
        held = held < m_launch * TOPK ? held : m_launch * TOPK;
        const u32 total = held * NTILES, per = (total + 7) / 8, i = g >> 3;
        if (i >= per) return;
        g = (g & 7u) * per + i;
        if (g >= total) return;
        const u32 t = g / NTILES;
        gn = g % NTILES;
        expert = tiles[1 + 3 * t];
        row0 = tiles[2 + 3 * t];
        rows = tiles[3 + 3 * t];
        if (expert >= HB_E || row0 >= pairs) return;
        rows = rows < BM ? rows : BM;
        rows = rows < pairs - row0 ? rows : pairs - row0;
        if (rows == 0) return;
    }
    const u32 n0 = gn * BF;

    // Row r of an experts' tile in X.
    auto x_row = [&](u32 r) HB_INLINE -> u32 {
        if constexpr (ROWS == 1) {
            const u32 pr = list[row0 + r] / TOPK;
            return pr < m ? pr : m - 1;
        }
        return row0 + r;
    };
    // W's block of 128 rows that fragment i of wave wn stands in, of the tile's.
    const u32 nb0 = n0 / 128;
    auto w_block = [&](u32 i) HB_INLINE -> u32 {
        if constexpr (SWI) return i >= IN / 2 ? 1u : 0u;
        if constexpr (BN % 128 == 0 && 128 % TN == 0) return wn * TN / 128;  // one for all i
        return (n0 + wn * TN + i * FM) / 128 - nb0;
    };

    // This wave's loads of a stage, wave loads wave, wave + NWV, ..: LDS slot p
    // of the operand's stage holds (row p / 8, chunk p % 8 ^ row >> 1), so that a
    // lane's chunk is the same in each (LROWS is a multiple of 16), and its rows
    // LROWS apart: one address a lane and constants.  Rows past the operand's end
    // lie past its resource's range, an experts' tile's rows past its own are put there:
    // zeros without a memory access.  (The scalar offset, which the range
    // check takes off the range, stays within a row.)
    constexpr u32 AWAY = 0x80000000u;
    const u32 lr = wave * 8 + lane / 8, cc = (lane % 8) ^ ((lr >> 1) & 7u);
    u32 xoff[ROWS == 0 ? 1 : XLMAX], soff[SLMAX];
#pragma unroll
    for (u32 i = 0; i < (ROWS == 0 ? 1 : XLMAX); i++) {
        const u32 r = lr + LROWS * i;
        xoff[i] = ROWS == 0 ? (u32)((row0 + r) * XROW) + cc * 16 : r < rows ? (u32)(x_row(r) * XROW) + cc * 16 : AWAY;
    }
    const u32 woff = (w_row(lr) + n0) * K + cc * 16;
#pragma unroll
    for (u32 i = 0; i < SLMAX; i++) {
        const u32 r = (wave + NWV * i) * 32 + lane / 2;
        soff[i] = ROWS == 0 || r < rows ? (u32)((ROWS == 0 ? row0 + r : x_row(r)) * XROW) + K + (lane % 2) * 16 : AWAY;
    }
    const u64 xbytes = (u64)(ROWS == 2 ? m_launch * TOPK : m_launch) * XROW;
    const __amdgpu_buffer_rsrc_t rX = __builtin_amdgcn_make_buffer_rsrc((void*)X, (short)0, (int)xbytes, 0x00020000);
    const __amdgpu_buffer_rsrc_t rW =
        __builtin_amdgcn_make_buffer_rsrc((void*)(W + expert * MATRIX), (short)0, (int)((u64)N * K), 0x00020000);
    typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
    auto lds_addr = [&](u32x4* p) HB_INLINE -> u32 { return (u32)(u64)(lds_u32x4*)p; };
    // The last K tile may be short: its chunks past K are zeros.
    auto cut = [&](u32 kt, u32 off) HB_INLINE -> u32 {
        if constexpr (K % 128 == 0) return off;
        return kt == KB - 1 && cc * 16 >= K % 128 ? AWAY : off;
    };
    const u32 kt0 = part * KB / KSP, kt1 = (part + 1) * KB / KSP;
    auto load_scales = [&](u32 c) HB_INLINE {
#pragma unroll
        for (u32 i = 0; i < SLMAX; i++) {
            if (NSL % NWV && wave + NWV * i >= NSL) continue;
            asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                         :: "s"(lds_addr(&sscale[(c & 1u) * BM * 2 + (wave + NWV * i) * 64])), "v"(soff[i]), "s"(rX),
                            "s"(c * 32) : "memory");
        }
    };
    auto load_x = [&](u32 kt, u32 st) HB_INLINE {
        // The scales first, so that they have landed when the tile has.
        if (kt % 8 == 0 || kt == kt0) load_scales(kt / 8);
        const u32 xo = cut(kt, xoff[0]);
#pragma unroll
        for (u32 i = 0; i < XLMAX; i++) {
            if (NXL % NWV && wave + NWV * i >= NXL) continue;
            asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                         :: "s"(lds_addr(&sXa[st * XST + (wave + NWV * i) * 64])),
                            "v"(ROWS == 0 ? xo + i * LROWS * (u32)XROW : cut(kt, xoff[ROWS == 0 ? 0 : i])), "s"(rX),
                            "s"(kt * 128) : "memory");
        }
    };
    // W's loads first, first + step, ..
    auto load_w = [&](u32 kt, u32 st, u32 first, u32 step) HB_INLINE {
        const u32 wo = cut(kt, woff);
#pragma unroll
        for (u32 i = first; i < WLMAX; i += step) {
            if (NWL % NWV && wave + NWV * i >= NWL) continue;
            asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                         :: "s"(lds_addr(&sWa[st * WST + (wave + NWV * i) * 64])), "v"(wo + w_row(LROWS * i) * K), "s"(rW),
                            "s"(kt * 128) : "memory");
        }
    };
    auto load_tile = [&](u32 kt, u32 st) HB_INLINE {
        load_x(kt, st);
        load_w(kt, st, 0, 1);
    };

    float acc[IN][IM][FR];
#pragma unroll
    for (u32 i = 0; i < IN; i++)
#pragma unroll
        for (u32 j = 0; j < IM; j++)
#pragma unroll
            for (u32 e = 0; e < FR; e++) acc[i][j][e] = 0.0f;
    const u32 fr = lane % FM, fc = lane / FM, fsw = (fr >> 1) & 7u;
    const u32 wbase = (wn * TN + fr) * 8, xbase = (wm * TM + fr) * 8;
    typedef i32x8 Fragment;
    auto fragment = [&](const u32x4* p) HB_INLINE -> Fragment {
        const u32x4 a = p[fc ^ fsw], b = p[(fc + 4) ^ fsw];
        return i32x8{(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w};
    };
#if HB_WIDE
    typedef F8Wide Operand;
    auto operand_of = [&](const Fragment& f) HB_INLINE -> Operand { return f8_wide(f); };
#else
    typedef Fragment Operand;
    auto operand_of = [&](const Fragment& f) HB_INLINE -> Operand { return f; };
#endif
    typedef float block_t __attribute__((ext_vector_type(FR)));

    float sx[IM];
    Operand xf[IM];
    auto read_x = [&](u32 kt, u32 st) HB_INLINE {
        const u32x4* sX = sXa + st * XST + xbase;
        const float* sc = (const float*)(sscale + (kt / 8 & 1u) * BM * 2) + (wm * TM + fr) * 8 + (kt & 7u);
#pragma unroll
        for (u32 j = 0; j < IM; j++) {
            xf[j] = operand_of(fragment(sX + j * FM * 8));
            sx[j] = sc[j * FM * 8];
        }
    };
    float last_sw = 0.0f;
    auto product_of = [&](const Operand& w, const Operand& x) HB_INLINE -> block_t {
#if HB_WIDE
        return f8_product(w, x);
#else
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, block_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
#endif
    };
    auto add = [&](u32 i, u32 j, const block_t& t, float s) HB_INLINE {
#pragma unroll
        for (u32 e = 0; e < FR; e++) {
            acc[i][j][e] = __builtin_fmaf(s, t[e], acc[i][j][e]);
            // Here and not later: the compiler would let blocks wait in
            // registers and add them behind the next barrier.
            if (AHEAD) asm volatile("" : "+v"(acc[i][j][e]));
        }
    };
    // W's scales of the tile's blocks, a row of them KBP places apart, the same
    // way; past a row's end come the next one's or zeros.
    const __amdgpu_buffer_rsrc_t rS = __builtin_amdgcn_make_buffer_rsrc((void*)(W + expert * MATRIX + (u64)N * K), (short)0,
                                                                        (int)(NB * KB * 4), 0x00020000);
    auto w_scales = [&]() HB_INLINE {
#pragma unroll
        for (u32 i = 0; i < (SWR * (KBP / 64) + NWV - 1) / NWV; i++) {
            const u32 q = wave + NWV * i, r = q / (KBP / 64), part64 = q % (KBP / 64);
            if (r >= SWR) continue;
            u32 b = nb0 + (SWI ? r * (NOUT / 128) : r);
            b = b < NB ? b : NB - 1;
            asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dword %1, %2, 0 offen lds"
                         :: "s"(lds_addr((u32x4*)(wscale + q * 64))), "v"((b * KB + part64 * 64 + lane) * 4), "s"(rS) : "memory");
        }
    };

    if constexpr (AHEAD) {
        // One barrier a K tile, before its last LAST fragments of W: by then a
        // wave holds those, so that the tile's stage is free for tile kt + 2,
        // and tile kt + 1 has landed, so that X's fragments of it and W's first
        // one are read while the last MFMAs run.
        constexpr u32 LAST = IN / 4;
        w_scales();
        load_tile(kt0, 0);
        if (kt0 + 1 < kt1) {
            load_tile(kt0 + 1, 1);
            WAIT_VM(LMIN);
        } else {
            WAIT_VM(0);
        }
        STAGE_BARRIER();
        Fragment xa[IM], xb[IM], first;
        float sa[IM], sb[IM];
        auto ready = [&](u32 kt, u32 st, Fragment (&x)[IM], float (&sc)[IM]) HB_INLINE {
            const u32x4* sX = sXa + st * XST + xbase;
            const float* c = (const float*)(sscale + (kt / 8 & 1u) * BM * 2) + (wm * TM + fr) * 8 + (kt & 7u);
            first = fragment(sWa + st * WST + wbase);
#pragma unroll
            for (u32 j = 0; j < IM; j++) {
                x[j] = fragment(sX + j * FM * 8);
                sc[j] = c[j * FM * 8];
            }
        };
        auto step = [&](u32 kt, u32 st, Fragment (&x)[IM], float (&sc)[IM], Fragment (&xn)[IM], float (&sn)[IM]) HB_INLINE {
            const u32x4* sW = sWa + st * WST + wbase;
            Fragment w[IN];
            Operand xo[IM];
#pragma unroll
            for (u32 j = 0; j < IM; j++) xo[j] = operand_of(x[j]);
            w[0] = first;
            float sw = wscale[w_block(0) * KBP + kt];
            block_t t[2];
#pragma unroll
            for (u32 i = 0; i < IN; i++) {
                if (i + 1 < IN - LAST) w[i + 1] = fragment(sW + (i + 1) * FM * 8);
                if (i + 1 == IN - LAST) {
#pragma unroll
                    for (u32 q = IN - LAST; q < IN; q++) w[q] = fragment(sW + q * FM * 8);
                }
                if (i == IN - LAST) {
                    WAIT_VM(0);
                    STAGE_BARRIER();
                    if (kt + 2 < kt1) load_tile(kt + 2, st);
                    ready(kt + 1, 1 - st, xn, sn);  // past the last tile: of a stage that nobody uses
                }
                if (!(BN % 128 == 0 && 128 % TN == 0 && !SWI) && i) sw = wscale[w_block(i) * KBP + kt];
                const Operand wo = operand_of(w[i]);
#pragma unroll
                for (u32 j = 0; j < IM; j++) {
                    const u32 q = i * IM + j;
                    t[q % 2] = product_of(wo, xo[j]);
                    if (q) {
                        const u32 p = q - 1;
                        // Two MFMAs, then the eight fmas of the two before them
                        // (8192 x 34816 x 5120: 1183 us, one by one in the
                        // order written 1257, left to the compiler 1180 to 1210).
                        __builtin_amdgcn_sched_group_barrier(0x8, 2, 0);
                        __builtin_amdgcn_sched_group_barrier(0x2, 8, 0);
                        add(p / IM, p % IM, t[p % 2], sc[p % IM] * (p / IM == i ? sw : last_sw));
                    }
                }
                last_sw = sw;
            }
            add(IN - 1, IM - 1, t[(IN * IM - 1) % 2], sc[IM - 1] * sw);
        };
        ready(kt0, 0, xa, sa);
        u32 kt = kt0;
#pragma unroll 1
        for (; kt + 1 < kt1; kt += 2) {
            step(kt, 0, xa, sa, xb, sb);
            step(kt + 1, 1, xb, sb, xa, sa);
        }
        if (kt < kt1) step(kt, 0, xa, sa, xb, sb);
        STAGE_BARRIER();
    } else {
        // W's scales and tiles 0 .. NS - 2 in flight, the first landed.
        w_scales();
#pragma unroll
        for (u32 t = 0; t + 1 < NS; t++)
            if (kt0 + t < kt1) load_tile(kt0 + t, t);
        if (kt0 + NS - 1 <= kt1) WAIT_VM((NS - 2) * LMIN);
        else WAIT_VM(0);
        STAGE_BARRIER();
        u32 st = 0;
        // As a loop for few tiles too: unrolled whole, 16 waves miss the
        // instruction cache (1024 rows, 1024 to 4096 SwiGLU: 27 us, 14 as one).
#pragma unroll 1
        for (u32 kt = kt0; kt < kt1; kt++) {
            // Tile kt + NS - 1 into the stage that tile kt - 1 used: every wave
            // has passed the barrier after its last read of it.
            const bool more = kt + NS - 1 < kt1;
            if (more) load_tile(kt + NS - 1, st == 0 ? NS - 1 : st - 1);
            const u32x4* sW = sWa + st * WST + wbase;
            read_x(kt, st);
#pragma unroll
            for (u32 i = 0; i < IN; i++) {
                const Operand wf = operand_of(fragment(sW + i * FM * 8));
                const float sw = wscale[w_block(i) * KBP + kt];
#pragma unroll
                for (u32 j = 0; j < IM; j++) add(i, j, product_of(wf, xf[j]), sx[j] * sw);
            }
            // Tile kt + 1 landed: at most the loads of the tiles after it are in
            // flight.
            if (more) WAIT_VM((NS - 2) * LMIN);
            else WAIT_VM(0);
            STAGE_BARRIER();
            st = st + 1 == NS ? 0 : st + 1;
        }
    }

    if constexpr (KSP > 1) Yv = (float*)Yv + (u64)part * m_launch * N;  // this part's slab
    if constexpr (SWI) {
        // h of the lane's features, rounded; the largest of each row over the
        // lane's, its column's other quads, and the waves of WN.
        constexpr u32 NR = FR / 4;  // runs of four features a block
        u32* const tops = (u32*)lds;
        u32x2 h[IN > 1 ? IN / 2 : 1][IM][NR];
#pragma unroll
        for (u32 j = 0; j < IM; j++) {
            u32 top = 0;
#pragma unroll
            for (u32 i = 0; i < IN / 2; i++)
#pragma unroll
                for (u32 q = 0; q < NR; q++) {
                    float hr[4];
#pragma unroll
                    for (u32 e = 0; e < 4; e++) hr[e] = f8_swiglu(acc[i][j][4 * q + e], acc[i + IN / 2][j][4 * q + e]);
                    h[i][j][q] = u32x2{pack_bf16x2(hr[0], hr[1]), pack_bf16x2(hr[2], hr[3])};
                    top = f8_max2(top, f8_max2(h[i][j][q].x & 0x7fff7fffu, h[i][j][q].y & 0x7fff7fffu));
                }
#pragma unroll
            for (u32 x = FM; x < 64; x *= 2) top = f8_max2(top, (u32)__shfl_xor((int)top, x, 64));
            top = f8_max2(top, top >> 16) & 0xffffu;
            if (fc == 0) tops[wn * BM + wm * TM + j * FM + fr] = top;
        }
        STAGE_BARRIER();
#pragma unroll
        for (u32 j = 0; j < IM; j++) {
            const u32 ml = wm * TM + j * FM + fr;
            u32 top = 0;
#pragma unroll
            for (u32 q = 0; q < WN; q++) top = tops[q * BM + ml] > top ? tops[q * BM + ml] : top;
            if (ml >= rows) continue;
            const F8Scale s = f8_scale(top);
            unsigned char* y = (unsigned char*)Yv + (u64)(row0 + ml) * HROW;
#pragma unroll
            for (u32 i = 0; i < IN / 2; i++)
#pragma unroll
                for (u32 q = 0; q < NR; q++)
                    *(u32*)(y + n0 + wn * (TN / 2) + i * FM + q * 8 + 4 * fc) =
                        f8_codes2<true>(h[i][j][q].y, s.inv, f8_codes2<false>(h[i][j][q].x, s.inv, 0));
            if (wn == 0 && fc == 0) *(float*)(y + NOUT + 4 * gn) = s.s;
        }
        return;
    }
    auto y_row = [&](u32 r) HB_INLINE -> u32 {
        if constexpr (ROWS == 2) {
            const u32 p = list[row0 + r];
            return p < pairs ? p : pairs - 1;
        }
        return row0 + r;
    };
    if constexpr (EPI_LDS) {
        // Past the barrier behind the last tile.
        unsigned char* const t = (unsigned char*)lds;
#pragma unroll
        for (u32 j = 0; j < IM; j++)
#pragma unroll
            for (u32 i = 0; i < IN; i++)
#pragma unroll
                for (u32 q = 0; q < FR / 4; q++)
                    *(u32x2*)(t + (wm * TM + j * FM + fr) * EPIROW + (wn * TN + i * FM + q * 8 + 4 * fc) * 2) =
                        u32x2{pack_bf16x2(acc[i][j][4 * q], acc[i][j][4 * q + 1]), pack_bf16x2(acc[i][j][4 * q + 2], acc[i][j][4 * q + 3])};
        STAGE_BARRIER();
        constexpr u32 CPR = BN / 8;
        typedef u32x4 loose_chunk __attribute__((aligned(2)));  // Y may start at any element
        for (u32 c = tid; c < BM * CPR; c += NTH) {
            const u32 r = c / CPR, n = n0 + c % CPR * 8;
            if (r >= rows || n >= NOUT) continue;
            const u32x4 v = *(const u32x4*)(t + r * EPIROW + c % CPR * 16);
            __builtin_nontemporal_store(v, (loose_chunk*)((u16*)Yv + (u64)y_row(r) * NOUT + n));
        }
        return;
    }
#pragma unroll
    for (u32 j = 0; j < IM; j++) {
        const u32 ml = wm * TM + j * FM + fr;
        if (ml >= rows) continue;
        const u32 yrow = y_row(ml);
#pragma unroll
        for (u32 i = 0; i < IN; i++)
#pragma unroll
            for (u32 q = 0; q < FR / 4; q++) {
                const u32 n = n0 + wn * TN + i * FM + q * 8 + 4 * fc;
                const float* v = &acc[i][j][4 * q];
                if (n < NOUT) store4(Yv, yrow, n, f32x4{v[0], v[1], v[2], v[3]});
            }
    }
}
