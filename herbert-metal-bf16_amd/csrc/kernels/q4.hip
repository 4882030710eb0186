// q4.hip -- weights of 4 bits: quantised from bf16 (HB_OP 1), laid out from
// codes and scales in row order (2), read back as bf16 (3).
//
// A row's elements stand in groups of GROUP along K, the last one may be
// short: element = (q - 8) * s, q of 0..15, s the group's bf16 scale.
// The layout is what the matvec's MFMAs read: tiles of 16 rows x 128 K, K
// fastest, each 1 KiB of codes: lane l of a wave takes 16 bytes, its word j
// the 8 codes of row l % 16 at K 32 j + 8 (l / 16) of the tile, one MFMA
// step's operand.  In a word, element e stands at bits 4 (e / 2) (+ 16 for odd
// e), all rotated left by 3, so that a rotation by 4 i and a mask leave
// elements 2 i and 2 i + 1 in the top mantissa bits of two bf16.  After the
// last tile's codes the scales, for each four row tiles and 128 K
// [row 0..63][group].  Rows past N and elements past K hold the code 8, their
// scales 0.
//
// All three are bound by the bf16 side's bytes, read and written at what a
// copy reaches (5.4 TB/s): 5120 x 34816 in groups of 32, 457 MB, quantised in
// 86 us and read back in 83, each alone over several matrices; in turn, as the
// case of both has them, 110 and 72, 176 for the pair (likely as part of the
// read back's 356 MB of writes leave the last-level cache under the launch that
// follows); 256 matrices of 2048 x 1024, 604 MB, laid out in 114.  A wave
// handles a tile, 16 bytes of bf16 a lane in four passes of 4 rows x 256
// bytes, their loads in flight at once (one after the other: 131); divisions
// and float extremes cost more than the bytes (144), hence the reciprocal and
// the packed halves.
#include "hb_common.h"

constexpr u32 K = HB_K, N = HB_N, GROUP = HB_GROUP;
constexpr u32 KT = (K + 127) / 128, NT = (N + 15) / 16, TILES = KT * NT;
constexpr u32 GPT = 128 / GROUP;        // groups of a tile
constexpr u32 GROUPS = (K + GROUP - 1) / GROUP;  // of a row
constexpr u64 CODES = (u64)TILES * 1024, BLOB = CODES + (u64)((NT + 3) / 4) * KT * 128 * GPT;  // bytes of a matrix
static_assert(K % 8 == 0, "K a multiple of 8");
static_assert(GROUP == 32 || GROUP == 64 || GROUP == 128, "groups of 32, 64 or 128");

// Tensors may start at any element.
typedef u32x4 chunk_t __attribute__((aligned(2)));

typedef u32 word_t __attribute__((aligned(2)));
// The low halves of a word's bytes, side by side.
HB_DEV u32 halves(u32 b) {
    b &= 0x0f0f0f0fu;
    b = (b | b >> 4) & 0x00ff00ffu;
    return (b | b >> 8) & 0xffffu;
}

// Word of chunk ch (8 elements) of row `row` within a tile's 256 words.
HB_DEV u32 word_at(u32 row, u32 ch) { return ((ch & 3u) * 16 + row) * 4 + (ch >> 2); }
// Scale of group g of row n in the K tile kt.
HB_DEV u64 scale_at(u32 n, u32 kt, u32 g) { return ((u64)(n / 64 * KT + kt) * 64 + n % 64) * GPT + g; }
HB_DEV u32 rotl(u32 v, u32 s) { return __builtin_amdgcn_alignbit(v, v, 32 - s); }

#if HB_OP == 1
typedef short s16x2 __attribute__((ext_vector_type(2)));
HB_DEV u32 word(u32x4 v, u32 i) { return v[i]; }

template <u32 ctrl>
HB_DEV s16x2 lane_max(s16x2 v) {
    const int b = __builtin_bit_cast(int, v);
    return __builtin_elementwise_max(v, __builtin_bit_cast(s16x2, __builtin_amdgcn_update_dpp(b, b, ctrl, 0xf, 0xf, true)));
}

// The codes q + 8 of eight elements in their places, q = w / s to the nearest
// whole number of -8..7, ties to even.
HB_DEV u32 group_codes(u32x4 v, float s) {
    u32 nw = 0;
    if (!(__builtin_fabsf(s) > 0x1p-100f)) {
        // A scale near the subnormals, or of zero, where all codes are 8.
#pragma unroll 1
        for (u32 e = 0; e < 8; e++) {
            const u32 half = v[e / 2] >> (16 * (e & 1)) & 0xffffu;
            const float q = s == 0.0f ? 0.0f : __builtin_rintf(__fdiv_rn(bf16_to_f32(half), s));
            nw |= (u32)(int)(__builtin_amdgcn_fmed3f(q, -8.0f, 7.0f) + 8.0f) << (4 * (e / 2) + 16 * (e & 1));
        }
        return nw;
    }
    // w / s by the reciprocal, corrected once by its exact remainder.  w and s
    // have 8 bits each, so a quotient that is no half lies 2^-11 or more from
    // the next one, and where it is one the correction gives it exactly.
    // Adding 2^23 + 8 rounds to a whole number in the low bits, ties to even as
    // 8 is even; the words' other bits sum to a constant.
    const float r = __builtin_amdgcn_rcpf(s);
    constexpr u32 MAGIC = 0x4B000000u;
    nw = 0;
#pragma unroll
    for (u32 e = 0; e < 8; e++) nw -= MAGIC << (4 * (e / 2) + 16 * (e & 1));
#pragma unroll
    for (u32 e = 0; e < 8; e++) {
        const float w = e & 1 ? bf16_hi(v[e / 2]) : bf16_lo(v[e / 2]);
        float q = w * r;
        q = __builtin_fmaf(__builtin_fmaf(-s, q, w), r, q);
        const float z = __builtin_amdgcn_fmed3f(q, -8.0f, 7.0f) + 8388616.0f;
        nw += __builtin_bit_cast(u32, z) << (4 * (e / 2) + 16 * (e & 1));
    }
    return nw;
}
#endif

#if HB_OP == 1 || HB_OP == 2
extern "C" __global__ __launch_bounds__(256) void HB_NAME(const u16* __restrict__ src,
#if HB_OP == 2
                                                            const u16* __restrict__ scales,
#endif
                                                            unsigned char* __restrict__ dst, u32 count) {
    __shared__ u32 words[4][256];
    const u32 lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const u64 id = (u64)blockIdx.x * 4 + wave, all = (u64)count * TILES;
    const bool live = id < all;
    const u64 mat = live ? id / TILES : 0;
    const u32 tile = live ? (u32)(id % TILES) : 0, nt = tile / KT, kt = tile % KT;
    unsigned char* blob = dst + mat * BLOB;
    u16* sc = (u16*)(blob + CODES);
    const u32 ch = lane & 15u, k = kt * 128 + ch * 8;
    // All loads in flight at once; past N and K some element's instead.
#if HB_OP == 1
    u32x4 vs[4];
#else
    u32 vs[4], ss[4];
#endif
#pragma unroll
    for (u32 i = 0; i < 4; i++) {
        const u32 n = nt * 16 + 4 * i + (lane >> 4);
        const u64 row = mat * N + (n < N ? n : N - 1);
#if HB_OP == 1
        vs[i] = *(const chunk_t*)(src + row * K + (k < K ? k : 0));
#else
        vs[i] = *(const word_t*)(src + (row * K + (k < K ? k : 0)) / 4);
        ss[i] = scales[row * GROUPS + (k < K ? k : 0) / GROUP];
#endif
    }
#pragma unroll
    for (u32 i = 0; i < 4; i++) {
        const u32 row = 4 * i + (lane >> 4), n = nt * 16 + row;
        const bool in = live && n < N && k < K;
        u32 nw = 0x88888888u;
#if HB_OP == 1
        const u32x4 v = in ? vs[i] : u32x4{0, 0, 0, 0};
        // bf16 bits order as their values do, the positive ones as signed
        // halves and all of them without their sign: the group's largest of
        // both, in the low and the high half of one word.
        s16x2 hi = {-32768, -32768}, size = {0, 0};
#pragma unroll
        for (u32 e = 0; e < 4; e++) {
            hi = __builtin_elementwise_max(hi, __builtin_bit_cast(s16x2, word(v, e)));
            size = __builtin_elementwise_max(size, __builtin_bit_cast(s16x2, word(v, e) & 0x7fff7fffu));
        }
        s16x2 far = {hi.x > hi.y ? hi.x : hi.y, size.x > size.y ? size.x : size.y};
        far = lane_max<0xB1>(far);  // quad_perm [1, 0, 3, 2], [2, 3, 0, 1]
        far = lane_max<0x4E>(far);
        if (GROUP >= 64) far = lane_max<0x141>(far);   // row_half_mirror
        if (GROUP == 128) far = lane_max<0x140>(far);  // row_mirror
        // s = the element of largest size (the positive one of two) / -8,
        // which loses bits only among the subnormals; a group with a NaN or
        // an infinity stands for NaN.
        const u32 top = (u16)far.y;
        const bool bad = top >= 0x7f80u;
        const float eighth = bf16_to_f32(far.x == far.y ? top : top | 0x8000u) * -0.125f;
        const u32 sb = bad ? 0x7fc0u : pack_bf16x2(eighth, 0.0f);
        const float s = bf16_to_f32(sb);
        if (!bad && top != 0) nw = group_codes(v, s);
        if (live && ch % (GROUP / 8) == 0) sc[scale_at(n, kt, ch / (GROUP / 8))] = n < N && k < K ? (u16)sb : 0;
#else
        // Row order: byte b of a row holds element 2 b in its low half.
        if (in) nw = halves(vs[i]) | halves(vs[i] >> 4) << 16;
        if (live && ch % (GROUP / 8) == 0) sc[scale_at(n, kt, ch / (GROUP / 8))] = in ? (u16)ss[i] : 0;
#endif
        words[wave][word_at(row, ch)] = rotl(nw, 3);
    }
    // The scales of the rows that a last group of four tiles lacks.
    if (live && nt == NT - 1 && NT % 4 != 0)
        for (u32 i = lane; i < (4 - NT % 4) * 16 * GPT; i += 64) sc[scale_at(NT * 16, kt, 0) + i] = 0;
    __syncthreads();
    if (live) ((u32x4*)(blob + (u64)tile * 1024))[lane] = ((u32x4*)words[wave])[lane];
}

#elif HB_OP == 3
extern "C" __global__ __launch_bounds__(256) void HB_NAME(const unsigned char* __restrict__ src,
                                                            u16* __restrict__ dst, u32 count) {
    const u32 lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const u64 id = (u64)blockIdx.x * 4 + wave;
    if (id >= (u64)count * TILES) return;
    const u64 mat = id / TILES;
    const u32 tile = (u32)(id % TILES), nt = tile / KT, kt = tile % KT;
    const unsigned char* blob = src + mat * BLOB;
    const u32* words = (const u32*)(blob + (u64)tile * 1024);
    const u16* sc = (const u16*)(blob + CODES);
    const u32 ch = lane & 15u, k = kt * 128 + ch * 8;
#pragma unroll
    for (u32 i = 0; i < 4; i++) {
        const u32 row = 4 * i + (lane >> 4), n = nt * 16 + row;
        if (n >= N || k >= K) continue;
        const u32 nw = rotl(words[word_at(row, ch)], 29);
        const float s = bf16_to_f32(sc[scale_at(n, kt, ch / (GROUP / 8))]);
        u32x4 o;
#pragma unroll
        for (u32 e = 0; e < 4; e++)
            o[e] = pack_bf16x2((float)((int)(nw >> (4 * e) & 15u) - 8) * s, (float)((int)(nw >> (16 + 4 * e) & 15u) - 8) * s);
        *(chunk_t*)(dst + (mat * N + n) * K + k) = o;
    }
}
#endif
