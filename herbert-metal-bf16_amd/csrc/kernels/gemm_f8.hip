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
// accumulators with an fma each, 16 cycles of VALU beside the MFMA's 32.
//
// X and W tiles of 128 K go straight into LDS (buffer_load_dwordx4 ... lds)
// through HB_STAGES stages, 16-byte chunks XORed by row >> 1 so that the
// fragments' reads meet no bank twice; a lane takes the chunks q and q + 4 of
// its row, q its quad (both operands alike, so the order of K within the MFMA
// does not matter).  X's scales of eight K tiles at a time go the same way into
// one of two places, 32 bytes a row; W's, all of a tile's blocks, are read once.
//
// Out::Swiglu: W holds [gate (N / 2) | up (N / 2)] rows; a tile covers 128
// features, a wave's first fragments their gate rows and its others the up
// rows, so a lane has both sums of a feature.  h = rne(g * sigmoid(g) * u) in
// bf16 and at once quantised: the 128 features are one group of an f8 row,
// whose largest is met over the waves in LDS.
//
// Constants: HB_K, HB_N (W rows), HB_OUT (0 bf16, 1 f32, 2 residual, 3
// SwiGLU), HB_ROWS, HB_TOPK, HB_E, HB_BM, HB_BN, HB_WM, HB_WN, HB_STAGES,
// HB_BAND, HB_KSPLIT.  Bindings: state, W, X, Y, list, tiles; then the rows
// the launch was sized for.
#include "f8.h"

constexpr u32 K = HB_K, N = HB_N;
constexpr int OUT = HB_OUT, ROWS = HB_ROWS;
constexpr u32 TOPK = HB_TOPK, BM = HB_BM, BN = HB_BN, WM = HB_WM, WN = HB_WN;
constexpr u32 NWV = WM * WN, NTH = 64 * NWV, NS = HB_STAGES, KSP = HB_KSPLIT;
constexpr u32 TM = BM / WM, TN = BN / WN, IM = TM / 16, IN = TN / 16;
constexpr bool SWI = OUT == 3;
constexpr u32 KB = f8_blocks(K), NB = f8_blocks(N), NOUT = SWI ? N / 2 : N, BF = SWI ? BN / 2 : BN;
constexpr u32 NTILES = (NOUT + BF - 1) / BF;
constexpr u64 XROW = f8_row_bytes(K), HROW = f8_row_bytes(NOUT), MATRIX = f8_matrix_bytes(K, N);
constexpr u32 XST = BM * 8, WST = BN * 8;                 // 16-byte chunks of a stage
constexpr u32 NXL = XST / 64, NWL = WST / 64;             // wave loads of a stage
constexpr u32 XLMAX = (NXL + NWV - 1) / NWV, WLMAX = (NWL + NWV - 1) / NWV;
constexpr u32 LMIN = NXL / NWV + NWL / NWV;               // loads a stage of every wave
constexpr u32 NSL = BM / 32, SLMAX = (NSL + NWV - 1) / NWV;  // wave loads of eight K tiles' X scales
constexpr u32 SWR = SWI ? 2 : BN % 128 == 0 ? BN / 128 : (BN + 127) / 128 + (128 % BN != 0);  // W's blocks of a tile
static_assert(K % 16 == 0 && BM % 32 == 0 && BN % 16 == 0 && TM % 16 == 0 && TN % 16 == 0, "tile");
static_assert(!SWI || (BN == 256 && IN % 2 == 0 && N % 256 == 0 && KSP == 1 && ROWS != 2), "SwiGLU");
static_assert(KSP == 1 || (OUT == 1 && ROWS == 0 && N % 4 == 0), "split K: f32 partial sums");
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
    __shared__ u32x4 lds[NS * (XST + WST)];
    __shared__ u32x4 sscale[2 * BM * 2];   // X's scales: [place][row][K tile of eight]
    __shared__ float wscale[SWR * KB];
    u32x4* const sXa = lds;
    u32x4* const sWa = lds + NS * XST;
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
        // The table's tiles alone, each XCD a contiguous range of them.
        const u32 total = tiles[0] * NTILES, per = (total + 7) / 8, i = g >> 3;
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

    // Row r of the tile in X, and the W row of its row r; past N the last one.
    auto x_row = [&](u32 r) HB_INLINE -> u32 {
        if constexpr (ROWS == 1) {
            const u32 pr = list[row0 + r] / TOPK;
            return pr < m ? pr : m - 1;
        }
        return row0 + r;
    };
    auto w_row = [&](u32 r) HB_INLINE -> u32 {
        if constexpr (SWI) {
            const u32 t = r % TN, i = t / 16, up = i >= IN / 2 ? 1u : 0u;
            return up * NOUT + n0 + (r / TN) * (TN / 2) + (i - up * (IN / 2)) * 16 + t % 16;
        }
        return n0 + r < N ? n0 + r : N - 1;
    };
    // W's block of 128 rows that fragment i of wave wn stands in, of the tile's.
    const u32 nb0 = n0 / 128;
    auto w_block = [&](u32 i) HB_INLINE -> u32 {
        if constexpr (SWI) return i >= IN / 2 ? 1u : 0u;
        return (n0 + wn * TN + i * 16) / 128 - nb0;
    };

    // This wave's loads of a stage: LDS slot p of the operand's stage holds
    // (row p / 8, chunk p % 8 ^ row >> 1).  Rows past the tile's at an offset
    // past the resource's range: zeros without a memory access.
    constexpr u32 AWAY = 0x80000000u;
    u32 xoff[XLMAX], woff[WLMAX], soff[SLMAX];
#pragma unroll
    for (u32 i = 0; i < XLMAX; i++) {
        const u32 p = (wave + NWV * i) * 64 + lane, r = p / 8, cc = (p % 8) ^ ((r >> 1) & 7u);
        xoff[i] = r < rows ? (u32)(x_row(r) * XROW) + cc * 16 : AWAY;
    }
#pragma unroll
    for (u32 i = 0; i < WLMAX; i++) {
        const u32 p = (wave + NWV * i) * 64 + lane, r = p / 8, cc = (p % 8) ^ ((r >> 1) & 7u);
        woff[i] = r < BN ? w_row(r) * K + cc * 16 : AWAY;
    }
#pragma unroll
    for (u32 i = 0; i < SLMAX; i++) {
        const u32 p = (wave + NWV * i) * 64 + lane, r = p / 2;
        soff[i] = r < rows ? (u32)(x_row(r) * XROW) + K + (p % 2) * 16 : AWAY;
    }
    const u64 xbytes = (u64)(ROWS == 2 ? m_launch * TOPK : m_launch) * XROW;
    const __amdgpu_buffer_rsrc_t rX = __builtin_amdgcn_make_buffer_rsrc((void*)X, (short)0, (int)xbytes, 0x00020000);
    const __amdgpu_buffer_rsrc_t rW =
        __builtin_amdgcn_make_buffer_rsrc((void*)(W + expert * MATRIX), (short)0, (int)((u64)N * K), 0x00020000);
    typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
    auto lds_addr = [&](u32x4* p) HB_INLINE -> u32 { return (u32)(u64)(lds_u32x4*)p; };
    // The last K tile may be short: its chunks past K are zeros.
    auto cut = [&](u32 kt, u32 i, u32 off) HB_INLINE -> u32 {
        if constexpr (K % 128 == 0) return off;
        const u32 p = (wave + NWV * i) * 64 + lane, r = p / 8, cc = (p % 8) ^ ((r >> 1) & 7u);
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
    auto load_tile = [&](u32 kt, u32 st) HB_INLINE {
        // The scales first, so that they have landed when the tile has.
        if (kt % 8 == 0 || kt == kt0) load_scales(kt / 8);
#pragma unroll
        for (u32 i = 0; i < XLMAX; i++) {
            if (NXL % NWV && wave + NWV * i >= NXL) continue;
            asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                         :: "s"(lds_addr(&sXa[st * XST + (wave + NWV * i) * 64])), "v"(cut(kt, i, xoff[i])), "s"(rX),
                            "s"(kt * 128) : "memory");
        }
#pragma unroll
        for (u32 i = 0; i < WLMAX; i++) {
            if (NWL % NWV && wave + NWV * i >= NWL) continue;
            asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                         :: "s"(lds_addr(&sWa[st * WST + (wave + NWV * i) * 64])), "v"(cut(kt, i, woff[i])), "s"(rW),
                            "s"(kt * 128) : "memory");
        }
    };

    f32x4 acc[IN][IM];
#pragma unroll
    for (u32 i = 0; i < IN; i++)
#pragma unroll
        for (u32 j = 0; j < IM; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const u32 fr = lane & 15u, fc = lane >> 4, fsw = (fr >> 1) & 7u;
    const u32 wbase = (wn * TN + fr) * 8, xbase = (wm * TM + fr) * 8;
    auto fragment = [&](const u32x4* p) HB_INLINE -> i32x8 {
        const u32x4 a = p[fc ^ fsw], b = p[(fc + 4) ^ fsw];
        return i32x8{(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w};
    };

    // Prologue: tiles 0 .. NS - 2 in flight, W's scales into LDS.
#pragma unroll
    for (u32 t = 0; t + 1 < NS; t++)
        if (kt0 + t < kt1) load_tile(kt0 + t, t);
    {
        const float* ws = (const float*)(W + expert * MATRIX + (u64)N * K);
        for (u32 i = tid; i < SWR * KB; i += NTH) {
            u32 b = SWI ? (i / KB) * (NOUT / 128) + nb0 : nb0 + i / KB;
            b = b < NB ? b : NB - 1;
            wscale[i] = ws[(u64)b * KB + i % KB];
        }
    }
    WAIT_VM(0);
    STAGE_BARRIER();

    u32 st = 0;
    for (u32 kt = kt0; kt < kt1; kt++) {
        // Tile kt + NS - 1 into the stage that tile kt - 1 used: every wave
        // has passed the barrier after its last read of it.
        const bool more = kt + NS - 1 < kt1;
        if (more) load_tile(kt + NS - 1, st == 0 ? NS - 1 : st - 1);
        const u32x4* sX = sXa + st * XST + xbase;
        const u32x4* sW = sWa + st * WST + wbase;
        const float* sc = (const float*)(sscale + (kt / 8 & 1u) * BM * 2) + (wm * TM + fr) * 8 + (kt & 7u);
        float sx[IM];
        i32x8 b[IM];
#pragma unroll
        for (u32 j = 0; j < IM; j++) {
            b[j] = fragment(sX + j * 128);
            sx[j] = sc[j * 128];
        }
#pragma unroll
        for (u32 i = 0; i < IN; i++) {
            const i32x8 a = fragment(sW + i * 128);
            const float sw = wscale[w_block(i) * KB + kt];
#pragma unroll
            for (u32 j = 0; j < IM; j++) {
                const f32x4 t = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b[j], f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
                const float s = sx[j] * sw;
#pragma unroll
                for (u32 e = 0; e < 4; e++) acc[i][j][e] = __builtin_fmaf(s, t[e], acc[i][j][e]);
            }
        }
        // Tile kt + 1 landed: at most the loads of the tiles after it are in
        // flight.
        if (more) WAIT_VM((NS - 2) * LMIN);
        else WAIT_VM(0);
        STAGE_BARRIER();
        st = st + 1 == NS ? 0 : st + 1;
    }

    if constexpr (KSP > 1) Yv = (float*)Yv + (u64)part * m_launch * N;  // this part's slab
    if constexpr (SWI) {
        // h of the lane's features, rounded; the largest of each row over the
        // lane's, its column's other quads, and the waves of WN.
        u32* const tops = (u32*)lds;
        u32x2 h[IN > 1 ? IN / 2 : 1][IM];
#pragma unroll
        for (u32 j = 0; j < IM; j++) {
            u32 top = 0;
#pragma unroll
            for (u32 i = 0; i < IN / 2; i++) {
                float gr[4], ur[4], hr[4];
#pragma unroll
                for (u32 e = 0; e < 4; e++) gr[e] = acc[i][j][e], ur[e] = acc[i + IN / 2][j][e];
                swiglu_n<4>(gr, ur, hr);
                h[i][j] = u32x2{pack_bf16x2(hr[0], hr[1]), pack_bf16x2(hr[2], hr[3])};
                top = f8_max2(top, f8_max2(h[i][j].x & 0x7fff7fffu, h[i][j].y & 0x7fff7fffu));
            }
#pragma unroll
            for (u32 x = 16; x < 64; x *= 2) top = f8_max2(top, (u32)__shfl_xor((int)top, x, 64));
            top = f8_max2(top, top >> 16) & 0xffffu;
            if (fc == 0) tops[wn * BM + wm * TM + j * 16 + fr] = top;
        }
        STAGE_BARRIER();
#pragma unroll
        for (u32 j = 0; j < IM; j++) {
            const u32 ml = wm * TM + j * 16 + fr;
            u32 top = 0;
#pragma unroll
            for (u32 q = 0; q < WN; q++) top = tops[q * BM + ml] > top ? tops[q * BM + ml] : top;
            if (ml >= rows) continue;
            const F8Scale s = f8_scale(top);
            unsigned char* y = (unsigned char*)Yv + (u64)(row0 + ml) * HROW;
#pragma unroll
            for (u32 i = 0; i < IN / 2; i++)
                *(u32*)(y + n0 + wn * (TN / 2) + i * 16 + 4 * fc) = f8_codes2<true>(h[i][j].y, s.inv, f8_codes2<false>(h[i][j].x, s.inv, 0));
            if (wn == 0 && fc == 0) *(float*)(y + NOUT + 4 * gn) = s.s;
        }
        return;
    }
#pragma unroll
    for (u32 j = 0; j < IM; j++) {
        const u32 ml = wm * TM + j * 16 + fr;
        if (ml >= rows) continue;
        u32 yrow = row0 + ml;
        if constexpr (ROWS == 2) {
            const u32 s = list[row0 + ml];
            yrow = s < pairs ? s : pairs - 1;
        }
#pragma unroll
        for (u32 i = 0; i < IN; i++) {
            const u32 n = n0 + wn * TN + i * 16 + 4 * fc;
            if (n < NOUT) store4(Yv, yrow, n, acc[i][j]);
        }
    }
}
