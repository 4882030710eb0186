// route_topk.hip -- routing to experts: per row, of the scores s of E experts,
//
//   p = softmax(s) or sigmoid(s),  c = p, or p + bias
//   groups of E / G consecutive experts: a group's score its largest c, or the
//     sum of its two largest; the TG groups of largest score stay
//   the TOPK experts of largest c in them, ties to the lowest index
//   w = p, or p / (the sum of the chosen p), times a factor
//
// written as route_qwen's rows are: route[r][i] = expert, in increasing order,
// route[r][TOPK + i] = the f32 bits of its weight, here not rounded to bf16.
// A score of NaN or -inf masks its expert: p = 0, and it is chosen, as are
// those of groups that do not stay, only where fewer than TOPK others are
// left, the lowest index first, with weight 0.
//
// What decides between experts is held in 64 bits, so that the choice does not
// hang on how an exponential rounds: without a bias the scores themselves order
// the experts; with one, or for sums of two, c in f64.
//
// A wave a row; lane l holds experts l P .. l P + P - 1, sorted, and pops its
// first when it is chosen, so that each choice looks at one key a lane: the
// wave's largest high word, and its largest low word only where several lanes
// share the high one.
// One row is the launch (3.7 us from the host); many rows are their instructions
// (8192 rows of 256 sigmoids in f32, groups 4 of 8: 12.2 us a pass, where the
// scores alone take 1.3 from memory): 857 vector instructions a wave, most of
// them in the choices, each a maximum over the wave, and in the keys' order; the
// f64 sigmoids are 2.7 us of it (with the scores in their place 10.9 of 13.6).
// Constants: HB_E, HB_TOPK, HB_SIGMOID, HB_BIAS, HB_GROUPS, HB_TOP_GROUPS,
// HB_GROUP_TOP, HB_RENORM, HB_F32 (scores f32, else bf16), HB_SCALE (f32 bits).
#include "hb_common.h"

constexpr u32 E = HB_E, TOPK = HB_TOPK, G = HB_GROUPS, TG = HB_TOP_GROUPS, GT = HB_GROUP_TOP;
constexpr bool SIGMOID = HB_SIGMOID, BIAS = HB_BIAS, RENORM = HB_RENORM, F32 = HB_F32;
constexpr u32 P = (E + 63) / 64, S = E / G;
constexpr bool GROUPED = G > 1 && TG < G;
constexpr bool KEY64 = BIAS || (GROUPED && GT == 2);
constexpr u32 lanes_a_group() {
    u32 l = 64;
    while (l * G > 64) l /= 2;
    return l;
}
constexpr u32 L = lanes_a_group();
static_assert(E >= 1 && E <= 1024 && TOPK >= 1 && TOPK <= 32 && E % G == 0 && G <= 64 && TG <= G && TOPK <= TG * S, "shape");

#define HB_INF __builtin_inff()

HB_DEV u32 lane_u32(u32 v, u32 l) { return (u32)__builtin_amdgcn_readlane((int)v, (int)l); }
// The wave's largest word.
HB_DEV u32 wave_max(u32 v) {
#define HB_DPP_MAX(ctrl)                                                                       \
    do {                                                                                       \
        const u32 o = (u32)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, 0xf, 0xf, true);       \
        v = o > v ? o : v;                                                                     \
    } while (0)
    HB_DPP_MAX(0x128);  // row_ror:8
    HB_DPP_MAX(0x124);  // row_ror:4
    HB_DPP_MAX(0x4E);   // quad_perm [2,3,0,1]
    HB_DPP_MAX(0xB1);   // quad_perm [1,0,3,2]
#undef HB_DPP_MAX
    const u32 a = lane_u32(v, 0), b = lane_u32(v, 16), c = lane_u32(v, 32), d = lane_u32(v, 48);
    const u32 ab = a > b ? a : b, cd = c > d ? c : d;
    return ab > cd ? ab : cd;
}
// Words in the order of the floats, zeros of both signs alike.
HB_DEV u32 ordered(float f) {
    const u32 b = __builtin_bit_cast(u32, f + 0.0f);
    return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}
HB_DEV float unordered(u32 k) { return __builtin_bit_cast(float, k ^ (k >> 31 ? 0x80000000u : 0xffffffffu)); }
HB_DEV u64 ordered(double f) {
    const u64 b = __builtin_bit_cast(u64, f + 0.0);
    return b ^ (b >> 63 ? ~0ull : 1ull << 63);
}
HB_DEV double shuffled(double v, u32 mask) {
    const u64 b = __builtin_bit_cast(u64, v);
    const u32 lo = (u32)__shfl_xor((int)(u32)b, mask, 64), hi = (u32)__shfl_xor((int)(u32)(b >> 32), mask, 64);
    return __builtin_bit_cast(double, (u64)hi << 32 | lo);
}
HB_DEV double larger(double a, double b) { return a > b ? a : b; }
HB_DEV double smaller(double a, double b) { return a < b ? a : b; }

// Below every score's key (ordered(-inf) is 0x007fffff): an expert that is
// masked or whose group is out, and a lane's places past the last expert.
constexpr u32 OUT = 1, NONE = 0;

HB_DEV float score(const void* s, u64 at) { return F32 ? ((const float*)s)[at] : bf16_to_f32(((const u16*)s)[at]); }

extern "C" __global__ __launch_bounds__(256) void HB_NAME(const void* __restrict__ scores, u32* __restrict__ route,
#if HB_BIAS
                                                            const float* __restrict__ bias,
#endif
                                                            u32 rows) {
    const u32 lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const u32 r = blockIdx.x * 4 + wave;
    __shared__ double held[GROUPED ? 4 * E : 1];
    if (r >= rows) return;  // a whole wave; nothing below joins waves
    const u64 base = (u64)r * E;

    float v[P];
    u32 hi[P], lo[P], at[P];
    bool live[P];
    if constexpr (E == 64 * P && (P & (P - 1)) == 0 && P > 1) {
        if constexpr (F32) {
            typedef float vec __attribute__((ext_vector_type(P)));
            typedef vec loose __attribute__((aligned(4)));
            const vec t = *(const loose*)((const float*)scores + base + lane * P);
#pragma unroll
            for (u32 p = 0; p < P; p++) v[p] = t[p];
        } else {
            typedef u16 vec __attribute__((ext_vector_type(P)));
            typedef vec loose __attribute__((aligned(2)));
            const vec t = *(const loose*)((const u16*)scores + base + lane * P);
#pragma unroll
            for (u32 p = 0; p < P; p++) v[p] = bf16_to_f32(t[p]);
        }
    } else {
#pragma unroll
        for (u32 p = 0; p < P; p++) v[p] = lane * P + p < E ? score(scores, base + lane * P + p) : -HB_INF;
    }
#pragma unroll
    for (u32 p = 0; p < P; p++) {
        live[p] = v[p] > -HB_INF;
        at[p] = lane * P + p;
    }

    // The row's largest score and the sum of the exponentials, where needed.
    float mx = -HB_INF, sum = 0.0f;
    if constexpr (!SIGMOID && (KEY64 || !RENORM)) {
        u32 top = 0;
#pragma unroll
        for (u32 p = 0; p < P; p++) {
            const u32 k = live[p] ? ordered(v[p]) : 0u;
            top = k > top ? k : top;
        }
        top = wave_max(top);
        mx = top ? unordered(top) : 0.0f;
        if constexpr (!RENORM) {
#pragma unroll
            for (u32 p = 0; p < P; p++) sum += live[p] ? hb_expf(v[p] == mx ? 0.0f : v[p] - mx) : 0.0f;
            sum = butterfly_sum(sum);
        }
    }
    double c[KEY64 || GROUPED ? P : 1];
    if constexpr (KEY64) {
        if constexpr (SIGMOID) {
#pragma unroll
            for (u32 p = 0; p < P; p++) c[p] = 1.0 / (1.0 + exp(-(double)v[p]));
        } else {
            double all = 0.0;
#pragma unroll
            for (u32 p = 0; p < P; p++) {
                c[p] = live[p] ? exp(v[p] == mx ? 0.0 : (double)v[p] - (double)mx) : 0.0;
                all += c[p];
            }
#pragma unroll
            for (u32 i = 32; i >= 1; i >>= 1) all += shuffled(all, i);
            if (all > 0.0) {
#pragma unroll
                for (u32 p = 0; p < P; p++) c[p] /= all;
            }
        }
#if HB_BIAS
#pragma unroll
        for (u32 p = 0; p < P; p++) {
            c[p] += lane * P + p < E ? (double)bias[lane * P + p] : 0.0;
            live[p] = live[p] && c[p] > -(double)HB_INF;
        }
#endif
    } else if constexpr (GROUPED) {
#pragma unroll
        for (u32 p = 0; p < P; p++) c[p] = (double)v[p];
    }

    if constexpr (GROUPED) {
        // L lanes a group look over its experts through LDS (the wave's own,
        // whose accesses run in program order).
        double* const mine = held + wave * E;
#pragma unroll
        for (u32 p = 0; p < P; p++)
            if (lane * P + p < E) mine[lane * P + p] = live[p] ? c[p] : -(double)HB_INF;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        const u32 g = lane / L, sub = lane % L;
        double one = -(double)HB_INF, two = one;
        if (g < G) {
            for (u32 i = sub; i < S; i += L) {
                const double k = mine[g * S + i];
                if (GT == 2) two = larger(two, smaller(one, k));
                one = larger(one, k);
            }
        }
#pragma unroll
        for (u32 i = L / 2; i >= 1; i >>= 1) {
            const double o = shuffled(one, i);
            if (GT == 2) two = larger(larger(two, shuffled(two, i)), smaller(one, o));
            one = larger(one, o);
        }
        const double total = GT == 2 && two > -(double)HB_INF ? one + two : one;
        const u64 tb = __builtin_bit_cast(u64, total);
        u32 before = 0;
#pragma unroll
        for (u32 j = 0; j < G; j++) {
            const u64 ob = (u64)lane_u32((u32)(tb >> 32), j * L) << 32 | lane_u32((u32)tb, j * L);
            const double o = __builtin_bit_cast(double, ob);
            before += o > total || (o == total && j < g) ? 1u : 0u;
        }
        const u64 stay = __ballot(g < G && before < TG);
#pragma unroll
        for (u32 p = 0; p < P; p++) {
            const u32 e = lane * P + p < E ? lane * P + p : E - 1;
            live[p] = live[p] && (stay >> (e / S * L) & 1u);
        }
    }

#pragma unroll
    for (u32 p = 0; p < P; p++) {
        if constexpr (KEY64) {
            const u64 k = ordered(c[p]);
            hi[p] = live[p] ? (u32)(k >> 32) : OUT;
            lo[p] = live[p] ? (u32)k : 0u;
        } else {
            hi[p] = live[p] ? ordered(v[p]) : OUT;
            lo[p] = 0;
        }
        if (E != 64 * P && lane * P + p >= E) hi[p] = NONE, lo[p] = 0;
    }
    // The lane's keys in falling order, equal ones as they stand.
#pragma unroll
    for (u32 round = 0; round < P; round++) {
#pragma unroll
        for (u32 p = round & 1u; p + 1 < P; p += 2) {
            const bool swap = hi[p + 1] > hi[p] || (KEY64 && hi[p + 1] == hi[p] && lo[p + 1] > lo[p]);
            const u32 h = hi[p], l = lo[p], a = at[p];
            hi[p] = swap ? hi[p + 1] : h;
            hi[p + 1] = swap ? h : hi[p + 1];
            lo[p] = swap ? lo[p + 1] : l;
            lo[p + 1] = swap ? l : lo[p + 1];
            at[p] = swap ? at[p + 1] : a;
            at[p + 1] = swap ? a : at[p + 1];
        }
    }

    u32 chosen[TOPK], expert = 0;
    bool counts = false;  // lane i: choice i is of a live expert
#pragma unroll
    for (u32 i = 0; i < TOPK; i++) {
        const u32 top = wave_max(hi[0]);
        u64 who = __ballot(hi[0] == top);
        if (KEY64 && (who & (who - 1))) {
            const u32 low = wave_max(hi[0] == top ? lo[0] : 0u);
            who = __ballot(hi[0] == top && lo[0] == low);
        }
        const u32 winner = (u32)__builtin_ctzll(who);
        chosen[i] = lane_u32(at[0], winner);
        if (lane == i) {
            expert = chosen[i];
            counts = top > OUT;
        }
        if (lane == winner) {
#pragma unroll
            for (u32 p = 0; p + 1 < P; p++) {
                hi[p] = hi[p + 1];
                lo[p] = lo[p + 1];
                at[p] = at[p + 1];
            }
            hi[P - 1] = NONE;
            lo[P - 1] = 0;
        }
    }

    // Lane i has choice i.
    const bool has = lane < TOPK && counts;
    const float s = has ? score(scores, base + expert) : -HB_INF;
    // e^(s - mx).  A difference of -60 rounded to f32 would leave the exponential
    // 2e-6 off: its rest goes in by the first term.
    auto relative = [&]() __attribute__((always_inline)) {
        const float d = s == mx ? 0.0f : s - mx, back = d - s, rest = (s - (d - back)) + (-mx - back);
        const float e = has ? hb_expf(d) : 0.0f;
        return has && s != mx && e > 0.0f ? __builtin_fmaf(e, rest, e) : e;
    };
    auto largest = [&]() __attribute__((always_inline)) -> float {  // of the chosen ones' scores
        const u32 top = wave_max(has ? ordered(s) : 0u);
        return top ? unordered(top) : 0.0f;
    };
    float p, total = 0.0f;
    if constexpr (SIGMOID) {
        p = has ? hb_sigmoid(s) : 0.0f;
        if constexpr (RENORM) total = butterfly_sum(p);
        // 1 / (1 + e^-s) is subnormal below -87 and 0 from -88.73 on, where e^s,
        // the same to f32, is not; and where all chosen lie far below 0 their
        // weights come from e^s / (1 + e^s) over e^largest.  Both are rare, and a
        // row without them pays for neither (8192 rows of 256: 0.5 us of 13.6).
        const bool far = has && s < -87.0f;
        if (__builtin_expect(__ballot(far || (RENORM && total < 0.00390625f)) != 0, 0)) {
            p = far ? hb_expf(s) : p;
            if constexpr (RENORM) {
                mx = largest();
                if (mx < 0.0f) p = has ? relative() / (1.0f + hb_expf(s)) : 0.0f;
                total = butterfly_sum(p);
            }
        }
    } else {
        if constexpr (RENORM) mx = largest();  // the chosen ones alone, over their own sum
        p = relative();
        if constexpr (RENORM) total = butterfly_sum(p);
        else p = sum > 0.0f ? p / sum : 0.0f;
    }
    if constexpr (RENORM) p = p / (total > 0.0f ? total : 1.0f);  // no branch: all p are 0 beside a sum of 0
    p *= __builtin_bit_cast(float, (u32)HB_SCALE);
    u32 rank = 0;
#pragma unroll
    for (u32 j = 0; j < TOPK; j++) rank += chosen[j] < expert ? 1u : 0u;
    if (lane < TOPK) {
        u32* o = route + (u64)r * 2 * TOPK;
        o[rank] = expert;
        o[TOPK + rank] = __builtin_bit_cast(u32, p);
    }
}
