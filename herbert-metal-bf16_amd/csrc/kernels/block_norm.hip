// block_norm.hip -- what stands between two blocks, in one pass over the rows:
//
//   u  = y, or RMSNorm(y) with the block's own post norm (POST)
//   v  = u, or gate * u: sigmoid of a row's gate (GATE 1) or of an element's
//        (2), or a channel's factor as it is (3)
//   xo = rne(a x + b v), a and b the layer's scales (SCALES) or 1
//   h  = rne(RMSNorm(xo) w_pre), the next block's input (PRE)
//
// RMSNorm(t) w = t / sqrt(mean(t^2) + eps) * w, w + 1 for PLUS1.  Everything
// between is f32; xo and h are rounded once each, and the pre norm reads xo
// as it is stored.
//
// A workgroup a row, its elements held in registers from the first load to
// the last store: bound by x, y and an element gate read once and xo and h
// written once, and for a few rows by one memory latency and two reductions.
// Measured: 2048 rows of 5120 with both norms 18.5 us, 4.5 TB/s where a copy
// reaches 5.4; 57 rows of 2560 with an element gate 2.6, 1 row 2.4, of which
// a launch alone is 2.3.
#include "hb_common.h"

constexpr u32 D = HB_D, THREADS = HB_THREADS, WAVES = THREADS / 64;
constexpr bool POST = HB_POST, PRE = HB_PRE, SCALES = HB_SCALES;
constexpr u32 GATE = HB_GATE;
constexpr u32 CELLS = (D + 7) / 8, CPT = (CELLS + THREADS - 1) / THREADS;
constexpr u32 TAIL = D % 8;  // elements of a row's last, short chunk

typedef u32x4 chunk_t __attribute__((aligned(2)));

// Elements 8 c .. +7 of a row of D, zeros past its end.
HB_DEV u32x4 load8(const u16* p, u32 c) {
    u32x4 v = {0, 0, 0, 0};
    if (TAIL == 0 || c < D / 8) {
        v = *(const chunk_t*)(p + 8 * c);
    } else {
#pragma unroll
        for (u32 e = 0; e < TAIL; e++) v[e / 2] |= (u32)p[8 * c + e] << (16 * (e & 1));
    }
    return v;
}
HB_DEV void store8(u16* p, u32 c, u32x4 v) {
    if (TAIL == 0 || c < D / 8) {
        *(chunk_t*)(p + 8 * c) = v;
    } else {
#pragma unroll
        for (u32 e = 0; e < TAIL; e++) p[8 * c + e] = (u16)(v[e / 2] >> (16 * (e & 1)));
    }
}
HB_DEV float at(u32x4 v, u32 e) { return e & 1 ? bf16_hi(v[e / 2]) : bf16_lo(v[e / 2]); }

HB_DEV float block_sum(float v, float* red) {
    v = butterfly_sum(v);
    if (WAVES == 1) return v;
    if ((threadIdx.x & 63u) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = red[0];
#pragma unroll
    for (u32 i = 1; i < WAVES; i++) s += red[i];
    return s;
}
HB_DEV float inv_rms(float ss) {
    return __fdiv_rn(1.0f, __fsqrt_rn(ss * (1.0f / (float)D) + __uint_as_float((u32)HB_EPS)));
}

extern "C" __global__ __launch_bounds__(THREADS) void HB_NAME(const u16* x, const u16* y, u16* xo,
#if HB_PRE
                                                                u16* h,
#endif
#if HB_POST
                                                                const u16* w_post,
#endif
#if HB_GATE
                                                                const u16* gate,
#endif
#if HB_SCALES
                                                                const float* scales,
#endif
#if HB_PRE
                                                                const u16* w_pre,
#endif
                                                                u32 rows) {
    __shared__ float red[2][WAVES];
    const u32 r = blockIdx.x, t = threadIdx.x;
    if (r >= rows) return;
    const u64 base = (u64)r * D;
    u32x4 xv[CPT], yv[CPT], gv[CPT], pv[CPT], nv[CPT];
#pragma unroll
    for (u32 i = 0; i < CPT; i++) {
        const u32 c = t + THREADS * i;
        xv[i] = yv[i] = gv[i] = pv[i] = nv[i] = u32x4{0, 0, 0, 0};
        if (CELLS % THREADS != 0 && c >= CELLS) continue;
        yv[i] = load8(y + base, c);
        xv[i] = load8(x + base, c);
#if HB_GATE == 2
        gv[i] = load8(gate + base, c);
#elif HB_GATE == 3
        gv[i] = load8(gate, c);
#endif
#if HB_POST
        pv[i] = load8(w_post, c);
#endif
#if HB_PRE
        nv[i] = load8(w_pre, c);
#endif
    }
    float a = 1.0f, b = 1.0f;
#if HB_SCALES
    a = scales[0], b = scales[1];
#endif
    float g = 1.0f;
#if HB_GATE == 1
    g = hb_sigmoid(bf16_to_f32(gate[r]));
#endif
    float inv = 1.0f;
    if (POST) {
        float ss = 0.0f;
#pragma unroll
        for (u32 i = 0; i < CPT; i++)
#pragma unroll
            for (u32 e = 0; e < 8; e++) ss = __builtin_fmaf(at(yv[i], e), at(yv[i], e), ss);
        inv = inv_rms(block_sum(ss, red[0]));
    }
    float ss = 0.0f;
#pragma unroll
    for (u32 i = 0; i < CPT; i++) {
        const u32 c = t + THREADS * i;
        if (CELLS % THREADS != 0 && c >= CELLS) continue;
        float o[8];
#pragma unroll
        for (u32 e = 0; e < 8; e++) {
            float v = at(yv[i], e);
            if (POST) v = (v * inv) * (HB_PLUS1 ? at(pv[i], e) + 1.0f : at(pv[i], e));
            if (GATE == 1) v = v * g;
            if (GATE == 2) v = v * hb_sigmoid(at(gv[i], e));
            if (GATE == 3) v = v * at(gv[i], e);
            o[e] = SCALES ? a * at(xv[i], e) + b * v : at(xv[i], e) + v;
        }
#pragma unroll
        for (u32 e = 0; e < 4; e++) xv[i][e] = pack_bf16x2(o[2 * e], o[2 * e + 1]);
        store8(xo + base, c, xv[i]);
        if (PRE)
#pragma unroll
            for (u32 e = 0; e < 8; e++)
                if (TAIL == 0 || c < D / 8 || e < TAIL) ss = __builtin_fmaf(at(xv[i], e), at(xv[i], e), ss);
    }
#if HB_PRE
    inv = inv_rms(block_sum(ss, red[1]));
#pragma unroll
    for (u32 i = 0; i < CPT; i++) {
        const u32 c = t + THREADS * i;
        if (CELLS % THREADS != 0 && c >= CELLS) continue;
        u32x4 o;
#pragma unroll
        for (u32 e = 0; e < 4; e++) {
            const float w0 = HB_PLUS1 ? at(nv[i], 2 * e) + 1.0f : at(nv[i], 2 * e);
            const float w1 = HB_PLUS1 ? at(nv[i], 2 * e + 1) + 1.0f : at(nv[i], 2 * e + 1);
            o[e] = pack_bf16x2((at(xv[i], 2 * e) * inv) * w0, (at(xv[i], 2 * e + 1) * inv) * w1);
        }
        store8(h + base, c, o);
    }
#endif
}
