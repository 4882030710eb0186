// f8.hip -- bf16 quantised to 8-bit floating point (f8.h) and read back:
// HB_OP 1 rows of activations, 2 a weight matrix, 3 and 4 the same back to
// bf16, q * s rounded once.
// The copy bounds all four: a matrix's block stays in registers between its
// largest and its codes, so that W is read once.  5120 x 34816 there and back
// 196 us, 5.5 TB/s (a 4 GiB copy reads and writes at 4.6 to 5.4); rows of a short
// block are the launch (57 of 5008 there and back 8 us).
// Constants: HB_OP, HB_K, HB_N (a matrix's rows).
#include "f8.h"

constexpr u32 K = HB_K, N = HB_N, KB = f8_blocks(K), NB = f8_blocks(N);
constexpr u64 ROW = f8_row_bytes(K), MATRIX = f8_matrix_bytes(K, N);
static_assert(K % 16 == 0, "K a multiple of 16");

// Tensors may start at any element.
typedef u32x4 chunk_t __attribute__((aligned(2)));

#if HB_OP == 1
// 16 lanes a group, 8 elements a lane; a wave's four groups one after the
// other along the rows.
extern "C" __global__ __launch_bounds__(256) void HB_NAME(const u16* __restrict__ x, unsigned char* __restrict__ q, u32 m) {
    const u32 l = threadIdx.x & 15u;
    const u64 g = (u64)blockIdx.x * 16 + (threadIdx.x >> 4);
    const u64 row = g / KB;
    const u32 kb = (u32)(g % KB), k = kb * 128 + 8 * l;
    if (row >= m) return;  // all 16 lanes of a group
    u32x4 v = {0, 0, 0, 0};
    if (K % 128 == 0 || k < K) v = *(const chunk_t*)(x + row * K + k);
    const F8Scale s = f8_scale(f8_max_lanes(f8_max8(v)));
    unsigned char* out = q + row * ROW;
    if (K % 128 == 0 || k < K) *(u32x2*)(out + k) = f8_codes8(v, s.inv);
    if (l == 0) *(float*)(out + K + 4 * kb) = s.s;
}

#elif HB_OP == 2
// A workgroup a block of 128 x 128: 16 rows of 256 bytes a pass, eight passes
// in registers.
extern "C" __global__ __launch_bounds__(256) void HB_NAME(const u16* __restrict__ w, unsigned char* __restrict__ q, u32 m) {
    (void)m;
    __shared__ u32 tops[4];
    const u32 l = threadIdx.x & 15u, r = threadIdx.x >> 4;
    const u32 kb = blockIdx.x % KB, b = blockIdx.x / KB, nb = b % NB, mat = b / NB;
    const u32 k = kb * 128 + 8 * l;
    const u16* src = w + (u64)mat * N * K;
    unsigned char* dst = q + mat * MATRIX;
    const bool in_k = K % 128 == 0 || k < K;
    u32x4 v[8];
    u32 top = 0;
#pragma unroll
    for (u32 i = 0; i < 8; i++) {
        const u32 n = nb * 128 + i * 16 + r;
        v[i] = u32x4{0, 0, 0, 0};
        if (in_k && (N % 128 == 0 || n < N)) v[i] = *(const chunk_t*)(src + (u64)n * K + k);
    }
#pragma unroll
    for (u32 i = 0; i < 8; i++) top = f8_max2(top, f8_max8(v[i]));
    top = f8_max_lanes(top);
    // A wave's four rows of lanes, then the four waves.
#pragma unroll
    for (u32 i = 16; i < 64; i *= 2) {
        const u32 o = (u32)__shfl_xor((int)top, i, 64);
        top = o > top ? o : top;
    }
    if ((threadIdx.x & 63u) == 0) tops[threadIdx.x >> 6] = top;
    __syncthreads();
#pragma unroll
    for (u32 i = 0; i < 4; i++) top = tops[i] > top ? tops[i] : top;
    const F8Scale s = f8_scale(top);
#pragma unroll
    for (u32 i = 0; i < 8; i++) {
        const u32 n = nb * 128 + i * 16 + r;
        if (in_k && (N % 128 == 0 || n < N)) *(u32x2*)(dst + (u64)n * K + k) = f8_codes8(v[i], s.inv);
    }
    if (threadIdx.x == 0) *(float*)(dst + (u64)N * K + 4 * ((u64)nb * KB + kb)) = s.s;
}

#else
// 16 codes a thread.
typedef float f32x2 __attribute__((ext_vector_type(2)));
HB_DEV u32 back2(u32 codes, bool high, float s) {
    const f32x2 v = high ? __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true) : __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false);
    return pack_bf16x2(v.x * s, v.y * s);
}

extern "C" __global__ __launch_bounds__(256) void HB_NAME(const unsigned char* __restrict__ q, u16* __restrict__ x, u32 m) {
    constexpr u32 CPR = K / 16;  // chunks a row
    const u64 i = (u64)blockIdx.x * 256 + threadIdx.x;
    const u64 row = i / CPR;
    const u32 k = (u32)(i % CPR) * 16;
    if (row >= (u64)m * (HB_OP == 3 ? 1 : N)) return;
    const unsigned char* codes;
    float s;
    if (HB_OP == 3) {
        codes = q + row * ROW;
        s = *(const float*)(codes + K + 4 * (k / 128));
    } else {
        const unsigned char* mat = q + row / N * MATRIX;
        const u32 n = (u32)(row % N);
        codes = mat + (u64)n * K;
        s = *(const float*)(mat + (u64)N * K + 4 * ((u64)(n / 128) * KB + k / 128));
    }
    const u32x4 c = *(const u32x4*)(codes + k);
    u32x4 lo, hi;
    lo.x = back2(c.x, false, s), lo.y = back2(c.x, true, s), lo.z = back2(c.y, false, s), lo.w = back2(c.y, true, s);
    hi.x = back2(c.z, false, s), hi.y = back2(c.z, true, s), hi.z = back2(c.w, false, s), hi.w = back2(c.w, true, s);
    *(chunk_t*)(x + row * K + k) = lo;
    *(chunk_t*)(x + row * K + k + 8) = hi;
}
#endif
